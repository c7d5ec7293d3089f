"""TitanMAC.decode on caches in 8 bits, against its layers on the rows that the caches hold."""
import math

import pytest
import torch

import titans_core as tc
from cache_cases import seen_by
from test_gpu_decoding import close, model

pytestmark = pytest.mark.gpu


def by_rows(m, ids, state, table, window):
    """Logits of ids by the model's layers, each of which attends to the keys and values that its cache holds, in 64 bits."""
    B, T = ids.shape
    Np, n = state.n_persistent, state.n_persistent + T
    x = torch.cat([m.persistent_tokens.expand(B, -1, -1), m.embed_tokens(ids) + m.embed_positions.weight[:T]], 1)
    mask = seen_by(1, n, [n], [n], window, Np)[0].to(ids.device)
    for layer, cache in zip(m.layers, state.caches):
        k, v = tc.cache_read(cache, table, state.lengths, n, dtype=torch.float32)
        H, d = k.shape[1], k.shape[3]
        q = layer.attention.qkv_proj(layer.norm_attn(x))[..., :H * d].view(B, n, H, d).transpose(1, 2)
        z = (q.double().unsqueeze(-2) * k.double().unsqueeze(2)).sum(-1) / math.sqrt(d)
        p = torch.softmax(z.masked_fill(~mask, -math.inf), -1)
        o = (p.unsqueeze(-1) * v.double().unsqueeze(2)).sum(-2).float()
        x = x + layer.attention.out_proj(o.transpose(1, 2).reshape(B, n, H * d))
        x = x + layer.mlp(layer.norm_mlp(x))
    return m.lm_head(m.norm(x[:, Np:]))


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("parts", [(60,), (30, 1, 29)])
def test_decode_is_its_layers_on_what_is_held(dev, parts, fmt):
    m = model(dev)
    ids = torch.randint(0, 211, (2, 60), device=dev)
    state = m.new_decode_state(2, fmt=fmt, page=16)
    got, at = [], 0
    for n in parts:
        got.append(m.decode(ids[:, at:at + n], state))
        at += n
    got = torch.cat(got, 1)
    window = m.config.window_size
    with torch.no_grad():
        assert close(got, by_rows(m, ids, state, state.table, window), torch.float32)
        # the bound tells mistakes from rounding: another window, another sequence's rows, values in the keys' place
        assert not close(got, by_rows(m, ids, state, state.table, window + 1), torch.float32)
        assert not close(got, by_rows(m, ids, state, state.table.flip(0), window), torch.float32)
        c = state.caches[0]
        state.caches[0] = tc.KVCache(c.v, c.k, c.d_head, c.v_scale, c.k_scale)
        assert not close(got, by_rows(m, ids, state, state.table, window), torch.float32)
