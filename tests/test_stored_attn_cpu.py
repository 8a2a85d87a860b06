"""Attention to stored keys and values without a GPU: the C ABI's refusals (no
kernel is launched), the Python layer's checks, and the references against
finite differences and against each other."""
import ctypes
import math

import pytest
import torch

from tests import _attn_ref as ref

P = ctypes.c_void_p
FAKE = 0x10000  # never dereferenced: every call below fails its host-side checks first


def _view(data=FAKE, sb=1 << 16, st=1 << 12, sh=128):
    from b200_gemm import _lib
    return _lib.AttnView(data, sb, st, sh)


def _cache(**kw):
    from b200_gemm import _lib
    c = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, num_pages=8, page_size=64, kv_heads=2, block_table=FAKE,
             table_stride=4, max_pages=4)
    c.update(kw)
    return _lib.KvCache(*c.values())


def test_write_refusals():
    from b200_gemm import _lib
    f = _lib.load().b200_kv_cache_write

    def call(k=None, v=None, cache=None, lens=FAKE, batch=2, new=1, d=128):
        return f(k or _view(), v or _view(), cache or _cache(), P(lens), None, batch, new, d, None)

    bad = _lib.B200_ERR_INVALID_ARG
    assert call(d=64) == bad
    assert call(batch=-1) == bad
    assert call(new=-1) == bad
    assert call(lens=None) == bad
    assert call(cache=_cache(page_size=48)) == bad
    assert call(cache=_cache(num_pages=-1)) == bad
    assert call(cache=_cache(k_scale=None)) == bad
    assert call(cache=_cache(block_table=None)) == bad
    assert call(cache=_cache(table_stride=3)) == bad
    assert call(k=_view(data=None)) == bad
    assert call(v=_view(sb=64)) == bad                       # entries overlap
    assert call(k=_view(data=FAKE + 8)) == _lib.B200_ERR_ALIGNMENT
    assert call(k=_view(sh=130)) == _lib.B200_ERR_ALIGNMENT
    assert call(cache=_cache(k=FAKE + 8)) == _lib.B200_ERR_ALIGNMENT
    assert call(cache=_cache(num_pages=1 << 26, page_size=64)) == _lib.B200_ERR_TOO_LARGE
    assert call(batch=1 << 17) == _lib.B200_ERR_TOO_LARGE
    assert call(batch=0) == _lib.B200_OK
    assert call(new=0) == _lib.B200_OK


def test_cache_attn_refusals():
    from b200_gemm import _lib
    lib = _lib.load()

    def call(q=None, cache=None, lens=FAKE, o=None, batch=2, q_len=1, heads=4, d=128, scale=0.1):
        return lib.b200_cache_attn(q or _view(), cache or _cache(), P(lens), None, o or _view(), batch, q_len, heads, d,
                                   scale, None, 0, None)

    bad = _lib.B200_ERR_INVALID_ARG
    assert call(d=64) == bad
    assert call(heads=3) == bad
    assert call(cache=_cache(kv_heads=0)) == bad
    assert call(q_len=-1) == bad
    assert call(lens=None) == bad
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert call(scale=scale) == bad
    assert call(cache=_cache(page_size=8)) == bad
    assert call(o=_view(data=FAKE + 4)) == _lib.B200_ERR_ALIGNMENT
    assert call(q=_view(st=1 << 40), q_len=2) == _lib.B200_ERR_TOO_LARGE
    assert call(batch=0) == _lib.B200_OK
    n = ctypes.c_size_t(7)
    assert lib.b200_cache_attn_workspace_bytes(2, 1, 3, _cache(), ctypes.byref(n)) == bad
    assert lib.b200_cache_attn_workspace_bytes(2, 0, 4, _cache(), ctypes.byref(n)) == _lib.B200_OK and n.value == 0


def test_cross_attn_refusals():
    from b200_gemm import _lib
    lib = _lib.load()

    def call(q=None, k=None, v=None, o=None, batch=2, q_len=4, kv_len=5, heads=4, kv_heads=2, d=128, scale=0.1, lse=None,
             lens=None):
        return lib.b200_cross_attn_bf16(q or _view(), k or _view(), v or _view(), P(lens), o or _view(), P(lse), batch, q_len,
                                        kv_len, heads, kv_heads, d, scale, None, 0, None)

    bad = _lib.B200_ERR_INVALID_ARG
    assert call(d=256) == bad
    assert call(heads=5) == bad
    assert call(kv_heads=0) == bad
    assert call(kv_len=-1) == bad
    assert call(scale=0.0) == bad
    assert call(k=_view(data=None)) == bad
    assert call(q=_view(st=100)) == bad
    assert call(q=_view(st=132)) == _lib.B200_ERR_ALIGNMENT
    assert call(v=_view(data=FAKE + 2)) == _lib.B200_ERR_ALIGNMENT
    assert call(lse=FAKE + 2) == _lib.B200_ERR_ALIGNMENT
    assert call(lens=FAKE + 1) == _lib.B200_ERR_ALIGNMENT
    assert call(kv_len=1 << 31) == _lib.B200_ERR_TOO_LARGE
    assert call(q_len=0) == _lib.B200_OK
    assert call(heads=0, kv_heads=0) == _lib.B200_OK
    n = ctypes.c_size_t(7)
    assert lib.b200_cross_attn_workspace_bytes(2, 4, -1, 4, 2, ctypes.byref(n)) == bad


def test_cross_attn_backward_refusals():
    from b200_gemm import _lib
    lib = _lib.load()

    def call(q=None, dv=None, o=None, lse=FAKE, lens=None, batch=2, q_len=4, kv_len=5, heads=4, kv_heads=2, d=128, scale=0.1,
             ws=FAKE, n=1 << 20):
        x = _view()
        return lib.b200_cross_attn_bwd_bf16(q or x, x, x, o or x, x, P(lse), P(lens), x, x, dv or x, batch, q_len, kv_len,
                                            heads, kv_heads, d, scale, P(ws), n, None)

    bad = _lib.B200_ERR_INVALID_ARG
    assert call(d=64) == bad
    assert call(heads=3) == bad
    assert call(kv_len=-1) == bad
    assert call(scale=math.nan) == bad
    assert call(lse=None) == bad
    assert call(ws=None) == bad
    assert call(n=256 + 2 * 4 * 8 * 128 - 1) == bad
    assert call(q=_view(data=None)) == bad
    assert call(dv=_view(sh=64)) == bad
    assert call(o=_view(data=FAKE + 8)) == _lib.B200_ERR_ALIGNMENT
    assert call(ws=FAKE + 16) == _lib.B200_ERR_ALIGNMENT
    assert call(lens=FAKE + 2) == _lib.B200_ERR_ALIGNMENT
    assert call(kv_len=1 << 31) == _lib.B200_ERR_TOO_LARGE
    assert call(batch=0) == _lib.B200_OK
    assert call(q_len=0, kv_len=0) == _lib.B200_OK
    n = ctypes.c_size_t(0)
    assert lib.b200_cross_attn_bwd_workspace_bytes(2, -1, 5, 4, 2, ctypes.byref(n)) == bad
    assert lib.b200_cross_attn_bwd_workspace_bytes(2, 5, -1, 4, 2, ctypes.byref(n)) == bad
    assert lib.b200_cross_attn_bwd_workspace_bytes(2, 5, 5, 4, 3, ctypes.byref(n)) == bad
    assert lib.b200_cross_attn_bwd_workspace_bytes(2, 5, 1 << 31, 4, 2, ctypes.byref(n)) == _lib.B200_ERR_TOO_LARGE


def test_status_text():
    from b200_gemm import _lib
    assert b"out of range" in _lib.load().b200_gemm_strerror(_lib.B200_ERR_BAD_INDEX)


def test_python_checks_on_cpu():
    import b200_gemm
    x = torch.zeros((1, 2, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        b200_gemm.cross_attn(x, x, x)
    with pytest.raises(TypeError, match="bfloat16"):
        b200_gemm.cross_attn(x.float(), x, x)
    with pytest.raises(TypeError, match="bfloat16"):
        b200_gemm.cache_attn(x.half(), x, x, x, x, x, x)
    with pytest.raises(ValueError, match="CUDA"):
        b200_gemm.kv_cache_write(x, x, x, x, x, x, x, x)


def test_python_none_and_other_types_are_refused():
    """None for a tensor raises (never crashes), in every place that can be reached without a GPU."""
    import b200_gemm
    x = torch.zeros((1, 2, 2, 128), dtype=torch.bfloat16)
    for args in ((None, x, x), (x, None, x), (x, x, None), (3, x, x), ([1], x, x)):
        with pytest.raises((TypeError, ValueError)):
            b200_gemm.cross_attn(*args)
    for i in range(8):
        args = [x] * 8
        args[i] = None
        with pytest.raises((TypeError, ValueError)):
            b200_gemm.kv_cache_write(*args)
    for i in range(7):
        args = [x] * 7
        args[i] = None
        with pytest.raises((TypeError, ValueError)):
            b200_gemm.cache_attn(*args)
    for i in range(6):
        args = [x] * 6
        args[i] = None
        with pytest.raises((TypeError, ValueError)):
            b200_gemm.cross_attn_backward(*args)


def test_power_scale():
    assert ref.power_scale(0.0) == 2.0 ** -100
    assert ref.power_scale(448.0) == 1.0
    assert ref.power_scale(448.0 * (1 + 2.0 ** -40)) == 2.0
    assert ref.power_scale(224.0) == 0.5


def test_reference_gradients_against_differences():
    """The reference's formulas against central differences of its own output."""
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(s, generator=g, dtype=torch.float64) for s in
                   ((2, 3, 4, 128), (2, 5, 2, 128), (2, 5, 2, 128), (2, 3, 4, 128)))
    lens = torch.tensor([5, 2])
    r = ref.cross_attn(q, k, v, lens, 0.09, do)

    def loss(a, b, c):
        return float((ref.cross_attn(a, b, c, lens, 0.09)["out"][0] * do).sum())

    for name, x, args in (("dq", q, lambda y: (y, k, v)), ("dk", k, lambda y: (q, y, v)), ("dv", v, lambda y: (q, k, y))):
        d = torch.randn(x.shape, generator=g, dtype=torch.float64)
        h = 1e-5
        diff = (loss(*args(x + h * d)) - loss(*args(x - h * d))) / (2 * h)
        # Central differences: h^2 / 6 times a third derivative of order one, and 2^-52 / h of rounding.
        assert abs(diff - float((r[name][0] * d).sum())) < 1e-7 * (1 + abs(diff))
