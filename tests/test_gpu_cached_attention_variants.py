"""cached_attention in each of the ways in which its rows and keys are shared out."""
import pytest
import torch

import titans_core as tc
from cache_cases import FORMATS, check_two_numbers, filled, gen, seen_by

pytestmark = pytest.mark.gpu


def queries(dev, B, H, T, d, dtype):
    return torch.randn(B, T, H, d, generator=gen(dev, 9), device=dev).to(dtype).transpose(1, 2)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,H,heads,d,n", [(2, 1, 4, 4, 64, 300), (2, 40, 4, 4, 64, 300), (16, 200, 4, 4, 64, 300),
                                             (12, 200, 8, 8, 128, 260), (2, 40, 2, 2, 64, 3000), (2, 40, 2, 2, 128, 3000),
                                             (60, 40, 4, 4, 64, 300), (60, 40, 4, 4, 128, 300)])
def test_probabilities_keep_their_bits(dev, B, T, H, heads, d, n, dtype, fmt):
    """Few rows or many, beside many sequences or few: the result's rounding is the only one of its size."""
    lens = [n - 7 * (b % 16) for b in range(B)]
    c, table, lengths = filled(dev, B, heads, d, 32, lens, dtype, fmt)
    q = queries(dev, B, H, T, d, dtype)
    out = tc.cached_attention(q, c, table, lengths, None, 4)
    news = [min(T, length) for length in lens]
    check_two_numbers(out, q, c, table, lens, news, seen_by(B, T, lens, news, None, 4))
