"""Refusals, argument errors, shapes under tracing and dispatch of the key/value cache's operators, on the CPU."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import titans_core as tc
from titans_core.kernels import _lib
from titans_core.kernels import kv_cache as kc

FAKE = 1 << 20
B, H, T, D = 2, 3, 4, 40


def parts(dtype=torch.bfloat16, fmt=None, page=16):
    c = tc.KVCache.new(5, H, D, page=page, dtype=dtype, fmt=fmt, device="cpu")
    x = torch.zeros(B, H, T, D, dtype=dtype)
    return c, x, torch.zeros(B, 2, dtype=torch.int32), torch.full((B,), T, dtype=torch.int32)


def calls(c, x, table, lengths, **kw):
    return {"write": lambda: tc.cache_write(x, x, c, table, lengths, **kw),
            "read": lambda: tc.cache_read(c, table, lengths, 5, dtype=x.dtype),
            "keep": lambda: tc.cache_keep(c, table, lengths, torch.zeros(B, 2, dtype=torch.int32), T),
            "attend": lambda: tc.cached_attention(x, c, table, lengths, **kw)}


def refused(error, text, names=("write", "read", "keep", "attend"), args=None, **kw):
    made = calls(*(args or parts()), **kw)
    for name in names:
        with pytest.raises(error, match=text):
            made[name]()


def test_new():
    c = tc.KVCache.new(5, H, D, page=32, fmt="e4m3", device="cpu")
    assert c.k.shape == (5, H, 32, 48) and c.k.dtype == torch.float8_e4m3fn and c.d_head == D
    assert c.k_scale.shape == (5, H, 32) and c.v_scale.dtype == torch.float32
    assert tc.KVCache.new(1, 1, 64, dtype=torch.float16, device="cpu").v_scale is None
    for kw in ({"page": 24}, {"page": 8}, {"d_head": 0}, {"d_head": 129}, {"n_pages": 0}, {"n_heads": 0}, {"fmt": "int4"}):
        with pytest.raises(ValueError, match="KVCache"):
            tc.KVCache.new(**{"n_pages": 2, "n_heads": 2, "d_head": 64, "device": "cpu", **kw})
    with pytest.raises(TypeError, match="dtype"):
        tc.KVCache.new(2, 2, 64, dtype=torch.float64, device="cpu")


def test_refusals():
    c, x, table, lengths = parts()
    refused(RuntimeError, "GPU")
    refused(TypeError, "int32", args=(c, x, table.long(), lengths))
    refused(TypeError, "int32", args=(c, x, table, lengths.long()))
    refused(TypeError, "int32", ("write", "attend"), counts=lengths.long())
    refused(ValueError, "counts must be", ("write", "attend"), counts=lengths[:1])
    refused(ValueError, "table must be", args=(c, x, table[:1], lengths))
    refused(ValueError, "table must be", args=(c, x, table[0], lengths))
    refused(ValueError, "table must be", args=(c, x, table[:, :0], lengths))
    refused(ValueError, "(lengths|table) must be", args=(c, x, table, lengths[:1]))
    refused(TypeError, "does not hold", args=(c, x.half(), table, lengths), names=("write", "read", "attend"))
    refused(TypeError, "unsupported dtype", args=(c, x.double(), table, lengths), names=("write", "read", "attend"))
    refused(ValueError, "(d_head|heads)", args=(c, x[..., :32], table, lengths), names=("write", "attend"))
    refused(ValueError, "heads", args=(c, x[:, :2], table, lengths), names=("write", "attend"))
    across = c.k.transpose(0, 1).contiguous().transpose(0, 1)
    for error, text, bad in ((ValueError, "alike", (c.k, c.v[:, :, :, :32], D)), (ValueError, "alike", (c.k[0], c.v[0], D)),
                             (ValueError, "pages of", (c.k, c.v, 50)), (ValueError, "contiguous", (across, c.v, D)),
                             (ValueError, "pages of", (c.k[:, :, :8], c.v[:, :, :8], D)), (ValueError, "pages of", (c.k, c.v, 0)),
                             (ValueError, "pages of", (c.k[:0], c.v[:0], D)), (TypeError, "dtype", (c.k.double(), c.v.double(), D)),
                             (RuntimeError, "devices", (c.k, c.v.to("meta"), D))):
        with pytest.raises(error, match=text):
            tc.KVCache(*bad)
    for fmt in ("int8", "e4m3"):
        q = parts(fmt=fmt)[0]
        for bad in (None, q.v_scale.half(), q.v_scale[:, :2], q.v_scale.transpose(0, 1).contiguous().transpose(0, 1)):
            with pytest.raises(ValueError, match="need k_scale"):
                tc.KVCache(q.k, q.v, D, q.k_scale, bad)
        assert tc.KVCache(q.k, q.v, D, q.k_scale, q.v_scale).v_scale is q.v_scale
    with pytest.raises(AttributeError):
        c.k = c.v
    with pytest.raises(ValueError, match="k and v must be"):
        tc.cache_write(x, x.half(), c, table, lengths)
    with pytest.raises(ValueError, match="k and v must be"):
        tc.cache_write(x[0], x[0], c, table, lengths)
    with pytest.raises(ValueError, match="n_positions"):
        tc.cache_read(c, table, lengths, -1)
    path = torch.zeros(B, 2, dtype=torch.int32)
    for bad, n in ((path.long(), T), (path[0], T), (path, 1), (path, 65), (path, -1)):
        with pytest.raises(ValueError, match="cache_keep"):
            tc.cache_keep(c, table, lengths, bad, n)
    with pytest.raises(ValueError, match="q must be"):
        tc.cached_attention(x[0], c, table, lengths)
    for kw in ({"window_size": -1}, {"n_persistent": -1}):
        with pytest.raises(ValueError, match="negative"):
            tc.cached_attention(x, c, table, lengths, **kw)
    tree = torch.zeros(B, T, dtype=torch.int64)
    for bad in (tree.int(), tree[:1], tree[:, :2], tree[0, :2]):
        with pytest.raises(ValueError, match="tree must be"):
            tc.cached_attention(x, c, table, lengths, tree=bad)
    long = torch.zeros(B, H, 65, D, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="up to 64"):
        tc.cached_attention(long, c, table, lengths, tree=torch.zeros(65, dtype=torch.int64))
    one = torch.zeros(1, dtype=torch.bfloat16)
    huge = one.expand(B, H, 1 << 26, D)
    refused(ValueError, "2\\^26", args=(c, huge, table, lengths), names=("write", "attend"))
    with pytest.raises(ValueError, match="2\\^26"):
        tc.cache_read(c, table, lengths, 1 << 26)
    with pytest.raises(ValueError, match="2\\^26"):
        tc.cached_attention(one.expand(1 << 20, H, 64, D), c, table[:1].expand(1 << 20, 2), lengths[:1].expand(1 << 20))


def test_no_gradient():
    c, x, table, lengths = parts()
    y = x.clone().requires_grad_()
    for name in ("write", "attend"):
        with pytest.raises(NotImplementedError, match="no gradient"):
            calls(c, y, table, lengths)[name]()
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        tc.cached_attention(y, c, table, lengths)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        c, x, table, lengths = parts(fmt="int8")
        assert tc.cache_write(x, x, c, table, lengths) is None
        k, v = tc.cache_read(c, table, lengths, 7, dtype=torch.float16)
        assert k.shape == v.shape == (B, H, 7, D) and k.dtype == torch.float16
        assert tc.cache_keep(c, table, lengths, table, T) is None
        assert tc.cached_attention(x, c, table, lengths, 5, 2).shape == (B, H, T, D)


class Record:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name) or 0


def test_dispatch(monkeypatch):
    """Plain calls go to the library at once; a trace records the registered ops; forward mode is refused."""
    rec = Record()
    monkeypatch.setattr(_lib, "lib", lambda: rec)
    monkeypatch.setattr(_lib, "require_device", lambda *t, what: t[0].device)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 0)
    kc._workspace.cache_clear()
    args = parts()
    for name, call in calls(*args).items():
        call()
    assert [c for c in rec.calls if "workspace" not in c] == ["tmac_cache_write", "tmac_cache_read", "tmac_cache_keep",
                                                               "tmac_cached_attn"]
    version = args[0].k._version
    calls(*args)["write"]()
    assert args[0].k._version == version + 1
    from torch.fx.experimental.proxy_tensor import make_fx
    c, x, table, lengths = args
    graph = make_fx(lambda q: tc.cached_attention(q, c, table, lengths, 5))(x)
    assert "titanmac.cached_attention" in graph.code
    del rec.calls[:]
    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
        tc.cached_attention(fwAD.make_dual(x.float(), x.float()), tc.KVCache(c.k.float(), c.v.float(), D), table, lengths)
    assert not rec.calls
    kc._workspace.cache_clear()


FIELDS = ("d_k", "d_v", "d_k_scale", "d_v_scale", "d_table", "d_lengths", "d_counts", "n_pages", "table_stride", "n_heads",
          "page", "pitch", "d_head", "max_pages", "format", "dtype")


def c_arg(**kw):
    """A cache whose numbers are in order; nothing is read at its addresses."""
    a = {"d_k": FAKE, "d_v": FAKE, "d_k_scale": FAKE, "d_v_scale": FAKE, "d_table": FAKE, "d_lengths": FAKE,
         "d_counts": 0, "n_pages": 10, "table_stride": 4, "n_heads": 3, "page": 16, "pitch": 48, "d_head": 40,
         "max_pages": 4, "format": 1, "dtype": 1, **kw}
    return kc._CACHE_ARG(*(a[n] or 0 for n in FIELDS))


BAD = [({"d_k": None}, -1), ({"d_v": None}, -1), ({"d_table": None}, -1), ({"d_lengths": None}, -1),
       ({"d_k_scale": None}, -1), ({"d_v_scale": None}, -1), ({"dtype": 3}, -4), ({"format": 3}, -4), ({"format": -1}, -4),
       ({"page": 8}, -2), ({"page": 24}, -2), ({"page": 512}, -2), ({"pitch": 40}, -2), ({"pitch": 64}, -2),
       ({"d_head": 0}, -2), ({"d_head": 129, "pitch": 144}, -2), ({"n_heads": 0}, -2), ({"n_pages": 0}, -2),
       ({"n_pages": 1 << 31}, -2), ({"max_pages": 0}, -2), ({"max_pages": (1 << 26) + 1}, -2), ({"table_stride": 3}, -2),
       ({"d_k": FAKE + 8}, -5), ({"d_v_scale": FAKE + 4}, -5), ({"d_table": FAKE + 2}, -5), ({"d_lengths": FAKE + 1}, -5),
       ({"d_counts": FAKE + 2}, -5)]


def test_argument_errors(lib):
    st = (ctypes.c_int64 * 3)(1, 1, 1)
    n = ctypes.c_size_t(0)

    def write(c, k=FAKE, ks=st, v=FAKE, vs=st, b=2, t=5):
        return lib.tmac_cache_write(c, k, ks, v, vs, b, t, None)

    def read(c, k=FAKE, v=FAKE, b=2, t=5):
        return lib.tmac_cache_read(c, k, v, b, t, None)

    def keep(c, path=FAKE, stride=4, a=4, b=2, t=5):
        return lib.tmac_cache_keep(c, path, stride, a, b, t, None)

    def attn(c, q=FAKE, qs=st, tree=None, ts=0, out=FAKE, ws=FAKE, nb=1 << 40, b=2, t=5, h=6, w=10, np=2):
        return lib.tmac_cached_attn(c, q, qs, tree, ts, out, ws, nb, b, t, h, w, np, 1.0, None)

    def size(c, b=2, t=5, h=6, w=10, np=2, to=ctypes.byref(n)):
        return lib.tmac_cached_attn_workspace(c, b, t, h, w, np, to)

    for f in (write, read, keep, attn, size):
        assert f(None) == -1
        for kw, want in BAD:
            assert f(c_arg(**kw)) == want, (f, kw)
        assert f(c_arg(), b=-1) == -2 and f(c_arg(), t=-1) == -2
        assert f(c_arg(), b=0) == 0
    for f in (write, read, attn):
        assert f(c_arg(), t=0) == 0 and f(c_arg(), t=(1 << 26)) == -2
    assert keep(c_arg(), a=0) == 0
    for kw in ({"k": None}, {"ks": None}, {"v": None}, {"vs": None}):
        assert write(c_arg(), **kw) == -1
    for kw in ({"k": None}, {"v": None}):
        assert read(c_arg(), **kw) == -1
    for kw, want in (({"path": None}, -1), ({"a": 6}, -2), ({"t": 65}, -2), ({"stride": 3}, -2), ({"b": 40000}, -2)):
        assert keep(c_arg(), **kw) == want
    for kw, want in (({"q": None}, -1), ({"qs": None}, -1), ({"out": None}, -1), ({"h": 5}, -2), ({"h": 0}, -2),
                     ({"w": -1}, -8), ({"np": -1}, -8), ({"tree": FAKE, "t": 65}, -2), ({"tree": FAKE, "ts": 4}, -2)):
        assert attn(c_arg(), **kw) == want, kw
    assert size(c_arg(), to=None) == -1 and size(c_arg(), h=5) == -2 and size(c_arg(), w=-1) == -8
    # few rows over a long axis need a workspace
    long = {"max_pages": 4096, "table_stride": 4096}
    assert size(c_arg(**long), t=1, w=1 << 30) == 0 and n.value > 0
    need = n.value
    for kw, want in (({"ws": None}, -6), ({"nb": need - 1}, -6), ({"ws": FAKE + 8}, -5)):
        assert attn(c_arg(**long), t=1, w=1 << 30, **kw) == want
    # the window bounds what a row sees, and with it the workspace
    assert size(c_arg(**long), t=1, w=500) == 0 and n.value == 0


def config(**kw):
    return tc.TitanMACConfig(**{**dict(vocab_size=20, d_model=32, n_heads=2, n_layers=1, d_ff=32, max_seq_len=16,
                                       n_persistent=0, window_size=4, use_block_sparse=False), **kw})


def test_decoding_refusals():
    for kw, text in (({"use_block_sparse": True}, "use_block_sparse"), ({"causal": False}, "causal"),
                     ({"use_neural_memory": True}, "neural memory")):
        with pytest.raises(ValueError, match=text):
            tc.TitanMAC(config(**kw)).new_decode_state(1)
    m = tc.TitanMAC(config()).eval()
    for args in ((0,), (1, 0), (1, 17)):
        with pytest.raises(ValueError, match="max_tokens"):
            m.new_decode_state(*args)
    with pytest.raises(ValueError, match="fmt"):
        m.new_decode_state(1, fmt="int4")
    state = m.new_decode_state(2, 10)
    ids = torch.zeros(2, 11, dtype=torch.long)
    with pytest.raises(ValueError, match="do not fit"):
        m.decode(ids, state)
    assert state.used == 0 and state.lengths.tolist() == [0, 0]
    with pytest.raises(ValueError, match="2 sequences"):
        m.decode(ids[:1], state)
    for bad in (torch.ones(2), torch.ones(3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="counts"):
            m.decode(ids[:, :3], state, counts=bad)
    for bad in (torch.ones(3), torch.ones(2, 2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="tree"):
            m.decode(ids[:, :3], state, tree=bad)
    with pytest.raises(RuntimeError, match="no draft"):
        state.keep(torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU"):
        m.decode(ids[:, :3], state)
    state = m.new_decode_state(2, 10)
    assert m.decode(ids[:, :0], state).shape == (2, 0, 20)
    with pytest.raises(ValueError, match="generate"):
        m.generate(ids[:, :0], 3)
    c, t, n = state.caches[0], state.table, state.lengths
    for attention, text in ((tc.WindowedAttention(config(attention_dropout=0.1)).train(), "dropout"),
                            (tc.WindowedAttention(config(causal=False)), "causal")):
        with pytest.raises(ValueError, match=text):
            attention.forward_cached(torch.zeros(2, 1, 32), c, t, n)
    block = tc.TitanBlock(config(use_block_sparse=True))
    with pytest.raises(ValueError, match="use_block_sparse"):
        block.forward_cached(torch.zeros(1, 1, 32), None, None, None)


def test_pools_without_versions():
    """Pools made in inference mode have no version to move on; those beside them do."""
    with torch.inference_mode():
        a = torch.zeros(2, H, 16, 48, dtype=torch.bfloat16)
    b = torch.zeros(2, H, 16, 48, dtype=torch.bfloat16)
    for k, v in ((a, a.clone()), (a, b), (b, a)):
        at = b._version
        kc._changed(tc.KVCache(k, v, D))
        assert b._version == at + (k is b or v is b)
