"""GPU tests of attention to stored keys and values: the 8-bit cache's write
(bit for bit), attention over it, cross attention; against 64-bit references
with derived bounds (tests/_attn_ref.py).  Covers lengths of zero and one,
pages that end inside a tile, ragged batches, grouped heads, strided operands,
NaN behind the last key, offsets past 32 bits, other streams, captured graphs,
and a decoder layer that runs them with the library's GEMM."""
import math

import pytest
import torch

import b200_gemm
from tests import _attn_ref as ref

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _randn(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(torch.bfloat16)


def _pool(g, batch, kv_heads, page, most, spare=2):
    """An empty cache of random bytes (NaN codes among them), wild scales, and a shuffled block table; on the CPU."""
    per = max(1, -(-most // page))
    pages = batch * per + spare
    codes = [torch.randint(0, 256, (pages, kv_heads, page, 128), generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn)
             for _ in range(2)]
    scales = [torch.exp2(torch.randint(-30, 30, (pages, kv_heads), generator=g).float()) for _ in range(2)]
    table = torch.randperm(pages, generator=g)[:batch * per].view(batch, per).to(torch.int32)
    return codes[0], codes[1], scales[0], scales[1], table


def _filled(g, lens, kv_heads, page, most=None):
    """A cache whose sequences of `lens` tokens were written from normal values, on the CPU."""
    most = max([1, *lens]) if most is None else most
    kc, vc, ks, vs, table = _pool(g, len(lens), kv_heads, page, most)
    k, v = (_randn(g, len(lens), most, kv_heads, 128) for _ in range(2))
    lens = torch.tensor(lens, dtype=torch.int32)
    kc, vc, ks, vs = _write_fast(k, v, kc, vc, ks, vs, table, lens)
    return [kc, vc, ks, vs, table, lens]


def _write_fast(k, v, kc, vc, ks, vs, table, lens):
    """Fresh sequences into the cache, a page at a time (scales of 2^-7 to 2^-5, whatever the values)."""
    page = kc.shape[2]
    for x, codes, scale in ((k, kc, ks), (v, vc, vs)):
        for b, n in enumerate(lens.tolist()):
            for i in range(-(-n // page)):
                p, m = int(table[b, i]), min(page, n - i * page)
                s = 2.0 ** (-7 + (i + b) % 3)
                vals = (x[b, i * page:i * page + m].transpose(0, 1).float() / s).clamp(-448, 448)
                codes[p, :, :m] = vals.to(torch.float8_e4m3fn)
                scale[p] = s
    return kc, vc, ks, vs


def _on(ts):
    return [t.to(DEV) for t in ts]


def _same(a, b):
    """Bit for bit, NaN codes equal to NaN codes."""
    a, b = a.cpu(), b.cpu()
    if a.dtype == torch.float8_e4m3fn:
        a, b = a.float(), b.float()
    return torch.equal(torch.nan_to_num(a, nan=1e9), torch.nan_to_num(b, nan=1e9)) and torch.equal(a.isnan(), b.isnan())


def _within(got, want, bound, what=""):
    got = got.double().cpu()
    assert torch.equal(got.isfinite(), want.isfinite()), f"{what}: infinities or NaN differ"
    err = torch.where(want.isfinite(), (got - want).abs(), 0.0)
    assert bool((err <= bound + 1e-30).all()), f"{what}: error {float((err / (bound + 1e-30)).max()):.3f} x the bound"


def _ok():
    torch.cuda.synchronize()
    assert b200_gemm.check_status() == 0


# --- kv_cache_write -----------------------------------------------------------


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("case", [
    # (new_max, lengths with the new tokens, new lengths or None, kv_heads)
    (1, [1, 2, 17, 64, 65, 129], None, 3),
    (5, [5, 6, 16, 33, 130, 259], None, 2),
    (300, [300, 301, 417], None, 1),
    (150, [150, 7, 64, 0, 200], [150, 7, 1, 0, 33], 2),
], ids=["step", "five", "prompt", "ragged"])
def test_write_bit_for_bit(page, case):
    new_max, lens, fresh, kv_heads = case
    g = torch.Generator().manual_seed(page + new_max)
    kc, vc, ks, vs, table = _pool(g, len(lens), kv_heads, page, max(lens) + page)
    lens = torch.tensor(lens, dtype=torch.int32)
    fresh = None if fresh is None else torch.tensor(fresh, dtype=torch.int32)
    # Magnitudes over many powers of two, so that scales grow in some pages and not in others.
    k, v = (_randn(g, len(lens), new_max, kv_heads, 128) *
            torch.exp2(torch.randint(-20, 12, (len(lens), new_max, kv_heads, 1), generator=g)).to(torch.bfloat16)
            for _ in range(2))
    want = ref.cache_write(k, v, kc, vc, ks, vs, table, lens, fresh)
    got = _on([kc, vc, ks, vs])
    b200_gemm.kv_cache_write(*_on([k, v]), *got, table.to(DEV), lens.to(DEV), new_lens=None if fresh is None else fresh.to(DEV))
    _ok()
    for name, a, b in zip(("k", "v", "k scale", "v scale"), got, want):
        assert _same(a, b), name


def test_write_token_by_token_grows_scales():
    """60 appends of one token each, ever larger values: every page's codes are rounded to its growing scale."""
    g = torch.Generator().manual_seed(3)
    kc, vc, ks, vs, table = _pool(g, 2, 2, 16, 64)
    got = _on([kc, vc, ks, vs])
    want = (kc, vc, ks, vs)
    for i in range(60):
        k, v = (_randn(g, 2, 1, 2, 128, scale=1.2 ** i) for _ in range(2))
        lens = torch.tensor([i + 1, i + 3], dtype=torch.int32)
        want = ref.cache_write(k, v, *want, table, lens)
        b200_gemm.kv_cache_write(*_on([k, v]), *got, table.to(DEV), lens.to(DEV))
    _ok()
    for a, b in zip(got, want):
        assert _same(a, b)


def test_write_special_values():
    """Zeros (scale 2^-100), NaN (kept, outside the scale), infinities (largest code), bf16's smallest and largest."""
    g = torch.Generator().manual_seed(4)
    kc, vc, ks, vs, table = _pool(g, 1, 1, 16, 16)
    top = torch.finfo(torch.bfloat16).max
    rows = [torch.zeros(128), torch.full((128,), math.nan), torch.full((128,), 2.0 ** -133), torch.full((128,), -0.0)]
    for extra in ([], [torch.full((128,), 448.0)], [torch.full((128,), 450.0)], [torch.full((128,), top)],
                  [torch.full((128,), 1.0).index_fill(0, torch.tensor([3, 7]), math.inf)]):
        x = torch.stack(rows + extra).view(1, -1, 1, 128).to(torch.bfloat16)
        lens = torch.tensor([x.shape[1]], dtype=torch.int32)
        want = ref.cache_write(x, -x, kc, vc, ks, vs, table, lens)
        got = _on([kc, vc, ks, vs])
        b200_gemm.kv_cache_write(*_on([x, -x]), *got, table.to(DEV), lens.to(DEV))
        _ok()
        for a, b in zip(got, want):
            assert _same(a, b)


def test_write_strided_inputs_and_long_tables():
    """k and v as views of a fused projection, heads before tokens, a table with a longer row pitch."""
    g = torch.Generator().manual_seed(5)
    kc, vc, ks, vs, table = _pool(g, 3, 2, 32, 100)
    lens = torch.tensor([40, 100, 39], dtype=torch.int32)
    qkv = _randn(g, 3, 39, 8, 128)
    bhsd = _randn(g, 3, 2, 39, 128)
    wide = torch.full((3, 11), -7, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    k, v = qkv[:, :, 4:6], bhsd.transpose(1, 2)
    want = ref.cache_write(k, v, kc, vc, ks, vs, table, lens)
    got = _on([kc, vc, ks, vs])
    b200_gemm.kv_cache_write(qkv.to(DEV)[:, :, 4:6], bhsd.to(DEV).transpose(1, 2), *got, wide.to(DEV)[:, :table.shape[1]],
                             lens.to(DEV))
    _ok()
    for a, b in zip(got, want):
        assert _same(a, b)


def test_write_out_of_range_is_reported_and_not_written():
    g = torch.Generator().manual_seed(6)
    kc, vc, ks, vs, table = _pool(g, 5, 1, 16, 32)
    table[1, 1] = kc.shape[0]    # past the last page
    table[2, 1] = -1
    lens = torch.tensor([20, 20, 20, 33, 1], dtype=torch.int32)  # 33 > 2 pages of 16
    fresh = torch.tensor([2, 2, 2, 2, 2], dtype=torch.int32)     # 2 new of 1
    k, v = (_randn(g, 5, 2, 1, 128) for _ in range(2))
    want = ref.cache_write(k[:1], v[:1], kc, vc, ks, vs, table[:1], lens[:1])
    got = _on([kc, vc, ks, vs])
    b200_gemm.kv_cache_write(*_on([k, v]), *got, table.to(DEV), lens.to(DEV), new_lens=fresh.to(DEV))
    torch.cuda.synchronize()
    with pytest.raises(b200_gemm.B200GemmError, match="out of range"):
        b200_gemm.check_status()
    assert b200_gemm.check_status() == 0  # reported once
    for a, b in zip(got, want):
        assert _same(a, b)


# --- cache_attn -------------------------------------------------------------------


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("shape", [(1, 4, 4), (1, 8, 2), (1, 32, 1), (1, 6, 2), (3, 4, 2), (5, 16, 2), (9, 8, 1)],
                         ids=lambda s: "x".join(map(str, s)))
def test_cache_attn_lengths(page, shape):
    t, h, kv = shape
    g = torch.Generator().manual_seed(page * 100 + t * 10 + h)
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000]
    cache = _filled(g, lens, kv, page)
    q = _randn(g, len(lens), t, h, 128)
    out = b200_gemm.cache_attn(q.to(DEV), *_on(cache))
    _ok()
    want, bound = ref.cache_attn(q, *cache)
    _within(out, want, bound, f"page {page} {shape}")


def test_cache_attn_ragged_queries_and_scale():
    g = torch.Generator().manual_seed(11)
    lens, fresh = [200, 50, 3, 0, 77], [6, 1, 3, 0, 0]
    cache = _filled(g, lens, 2, 32)
    q = _randn(g, 5, 6, 4, 128)
    for i, m in enumerate(fresh):
        q[i, m:] = math.nan  # padding may hold anything; its rows become zeros
    out = b200_gemm.cache_attn(q.to(DEV), *_on(cache), new_lens=torch.tensor(fresh, dtype=torch.int32, device=DEV), scale=0.05)
    _ok()
    want, bound = ref.cache_attn(q, *cache, fresh, 0.05)
    _within(out, want, bound)
    assert all(not bool(out[i, m:].any()) for i, m in enumerate(fresh))


def test_cache_attn_query_magnitudes_and_page_scales():
    """Rows of q from 2^-60 to 2^20 and value scales from 2^-90 to 2^90 in one sequence: nothing over- or underflows."""
    g = torch.Generator().manual_seed(12)
    cache = _filled(g, [150, 150, 150], 1, 16)
    kc, vc, ks, vs, table, lens = cache
    q = _randn(g, 3, 1, 1, 128)
    q[0] *= 2.0 ** -60
    q[1] *= 2.0 ** 20
    ks[table[1].long()] *= 2.0 ** -20
    for i, p in enumerate(table[2].tolist()):
        vs[p] = 2.0 ** (-90 + 20 * i)
    out = b200_gemm.cache_attn(q.to(DEV), *_on(cache))
    _ok()
    want, bound = ref.cache_attn(q, *cache)
    _within(out, want, bound)


def test_cache_attn_zero_value_pages_keep_their_weight():
    """A page of zeros holds scale 2^-100: its keys still count in the softmax."""
    g = torch.Generator().manual_seed(13)
    kc, vc, ks, vs, table = _pool(g, 1, 1, 16, 48)
    k, v = (_randn(g, 1, 48, 1, 128) for _ in range(2))
    v[:, 16:32] = 0
    lens = torch.tensor([48], dtype=torch.int32)
    cache = _on([kc, vc, ks, vs])
    b200_gemm.kv_cache_write(*_on([k, v]), *cache, table.to(DEV), lens.to(DEV))
    q = _randn(g, 1, 1, 1, 128)
    out = b200_gemm.cache_attn(q.to(DEV), *cache, table.to(DEV), lens.to(DEV))
    _ok()
    want, bound = ref.cache_attn(q, *[c.cpu() for c in cache], table, lens)
    assert float(cache[3][int(table[0, 1]), 0]) == 2.0 ** -100
    _within(out, want, bound)


def test_cache_attn_strides_and_out():
    g = torch.Generator().manual_seed(14)
    cache = _filled(g, [70, 200], 2, 64)
    qkv = _randn(g, 2, 2, 12, 128)
    want, bound = ref.cache_attn(qkv[:, :, :8], *cache)
    buf = torch.full((2, 8, 2, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    out = buf.transpose(1, 2)
    got = b200_gemm.cache_attn(qkv.to(DEV)[:, :, :8], *_on(cache), out=out)
    _ok()
    assert got is out
    _within(out, want, bound)


def test_cache_attn_repeats_bit_for_bit_and_splits():
    """Few heads, long sequences: segments are cut over many CTAs and joined in a fixed order."""
    g = torch.Generator().manual_seed(15)
    cache = _filled(g, [5000, 1, 7777], 1, 64)
    q = _randn(g, 3, 1, 4, 128)
    dev = _on(cache)
    outs = [b200_gemm.cache_attn(q.to(DEV), *dev) for _ in range(5)]
    _ok()
    want, bound = ref.cache_attn(q, *cache)
    _within(outs[0], want, bound)
    assert all(torch.equal(outs[0], o) for o in outs)


def test_cache_attn_large_batch():
    """More sequences than threads of a CTA, most of them short."""
    g = torch.Generator().manual_seed(16)
    lens = [(i * 37) % 90 for i in range(700)]
    cache = _filled(g, lens, 1, 16)
    q = _randn(g, len(lens), 1, 2, 128)
    out = b200_gemm.cache_attn(q.to(DEV), *_on(cache))
    _ok()
    want, bound = ref.cache_attn(q, *cache)
    _within(out, want, bound)


@pytest.mark.parametrize("shape", [(1, 4, 4), (1, 32, 1), (5, 16, 2), (9, 8, 1)], ids=lambda s: "x".join(map(str, s)))
def test_cache_attn_short_sequences_under_a_wide_table(shape):
    """The table has room for 64 times the tokens there are; entries of no page hold -1 and are not read."""
    t, h, kv = shape
    g = torch.Generator().manual_seed(70 + h)
    lens = [0, 1, 31, 32, 33, 64, 0, 300, 1000, 0]
    cache = _filled(g, lens, kv, 32)
    wide = torch.full((len(lens), 2000), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        wide[i, :-(-n // 32)] = cache[4][i, :-(-n // 32)]
    cache[4] = wide
    q = _randn(g, len(lens), t, h, 128)
    out = b200_gemm.cache_attn(q.to(DEV), *_on(cache))
    _ok()
    want, bound = ref.cache_attn(q, *cache)
    _within(out, want, bound)


@pytest.mark.parametrize("shape", [(1, 8, 2), (6, 8, 1)], ids=lambda s: "x".join(map(str, s)))
def test_cache_attn_long_and_short_side_by_side(shape):
    """Workers that hold the end of a long sequence, several short ones and the start of the next; up to 48 rows."""
    t, h, kv = shape
    g = torch.Generator().manual_seed(80 + h)
    lens = [9000, 0, 3, 40, 12345, 1, 0, 700, 16000]
    cache = _filled(g, lens, kv, 128)
    q = _randn(g, len(lens), t, h, 128)
    out = b200_gemm.cache_attn(q.to(DEV), *_on(cache))
    _ok()
    want, bound = ref.cache_attn(q, *cache)
    _within(out, want, bound)


def test_cache_attn_sequences_that_share_pages():
    """A common prefix stored once: the same pages in several rows of the table."""
    g = torch.Generator().manual_seed(90)
    cache = _filled(g, [200, 180, 64], 2, 32)
    cache[4][1, :2] = cache[4][0, :2]
    cache[4][2, :2] = cache[4][0, :2]
    q = _randn(g, 3, 1, 8, 128)
    out = b200_gemm.cache_attn(q.to(DEV), *_on(cache))
    _ok()
    want, bound = ref.cache_attn(q, *cache)
    _within(out, want, bound)


def test_cache_attn_offsets_past_32_bits():
    """A cache of 4.5 GB each for K and V, the sequence's pages at its far end."""
    g = torch.Generator().manual_seed(17)
    pages, kv, page = 34500, 8, 128
    kc, vc = (torch.empty((pages, kv, page, 128), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.zeros((pages, kv), device=DEV) for _ in range(2))
    assert kc.numel() > 1 << 32
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    lens = torch.tensor([300], dtype=torch.int32)
    k, v = (_randn(g, 1, 300, kv, 128) for _ in range(2))
    b200_gemm.kv_cache_write(*_on([k, v]), kc, vc, ks, vs, table.to(DEV), lens.to(DEV))
    q = _randn(g, 1, 1, 16, 128)
    out = b200_gemm.cache_attn(q.to(DEV), kc, vc, ks, vs, table.to(DEV), lens.to(DEV))
    _ok()
    pick = table[0].long().to(DEV)
    near = [kc.view(torch.uint8)[pick].cpu().view(torch.float8_e4m3fn), vc.view(torch.uint8)[pick].cpu().view(torch.float8_e4m3fn),
            ks[pick].cpu(), vs[pick].cpu(), torch.arange(3, dtype=torch.int32).view(1, 3), lens]
    want, bound = ref.cache_attn(q, *near)
    _within(out, want, bound)


def test_cache_attn_bad_pages_are_reported():
    g = torch.Generator().manual_seed(18)
    cache = _filled(g, [100, 100], 1, 32)
    good = ref.cache_attn(torch.ones((2, 1, 1, 128), dtype=torch.bfloat16), *cache)
    cache[4][0, 1] = 10 ** 6
    q = torch.ones((2, 1, 1, 128), dtype=torch.bfloat16, device=DEV)
    out = b200_gemm.cache_attn(q, *_on(cache))
    torch.cuda.synchronize()
    with pytest.raises(b200_gemm.B200GemmError, match="out of range"):
        b200_gemm.check_status()
    _within(out[1:], good[0][1:], good[1][1:])  # the other sequence is right
    cache[4][0, 1] = 0
    cache[5][0] = 10 ** 6  # longer than its table
    b200_gemm.cache_attn(q, *_on(cache))
    torch.cuda.synchronize()
    with pytest.raises(b200_gemm.B200GemmError, match="out of range"):
        b200_gemm.check_status()
    assert b200_gemm.check_status() == 0


@pytest.mark.parametrize("length", [-(1 << 31), -(1 << 31) + 5, -1, (1 << 31) - 1, 65])
def test_cache_lengths_far_out_of_range(length):
    """Differences of such lengths wrap around in 32 bits: nothing is written, both calls report, the other sequence is right."""
    g = torch.Generator().manual_seed(20)
    cache = _filled(g, [40, 40], 2, 16, most=64)
    dev = _on(cache)
    k = _randn(g, 2, 10, 2, 128)
    lens = torch.tensor([length, 40], dtype=torch.int32)
    b200_gemm.kv_cache_write(*_on([k, k]), *dev[:5], lens.to(DEV))
    torch.cuda.synchronize()
    with pytest.raises(b200_gemm.B200GemmError, match="out of range"):
        b200_gemm.check_status()
    want = ref.cache_write(k[1:], k[1:], *cache[:4], cache[4][1:], lens[1:])
    assert all(_same(a, b) for a, b in zip(dev[:4], want))
    q = _randn(g, 2, 1, 4, 128)
    out = b200_gemm.cache_attn(q.to(DEV), *dev[:5], lens.to(DEV))
    torch.cuda.synchronize()
    with pytest.raises(b200_gemm.B200GemmError, match="out of range"):
        b200_gemm.check_status()
    near = [d.cpu() for d in dev[:4]]
    value, bound = ref.cache_attn(q[1:], *near, cache[4][1:], lens[1:])
    _within(out[1:], value, bound)


def test_cache_refusals():
    g = torch.Generator().manual_seed(19)
    kc, vc, ks, vs, table, lens = _on(_filled(g, [20], 2, 16))
    q = torch.zeros((1, 1, 4, 128), dtype=torch.bfloat16, device=DEV)
    k = torch.zeros((1, 1, 2, 128), dtype=torch.bfloat16, device=DEV)
    attn, write = b200_gemm.cache_attn, b200_gemm.kv_cache_write
    with pytest.raises(TypeError):
        attn(q, kc.view(torch.uint8), vc, ks, vs, table, lens)
    with pytest.raises(TypeError):
        attn(q, kc, vc, ks, vs, table.long(), lens)
    with pytest.raises(TypeError):
        attn(q, kc, vc, ks, vs, table, lens.long())
    with pytest.raises(TypeError):
        attn(q, kc, vc, ks, vs, table, None)
    for i in range(7):
        args = [q, kc, vc, ks, vs, table, lens]
        args[i] = None
        with pytest.raises(TypeError):
            attn(*args)
        with pytest.raises(TypeError):
            write(k, k, *args[1:]) if i else write(None, k, *args[1:])
    with pytest.raises(ValueError):
        attn(q[:, :, :3], kc, vc, ks, vs, table, lens)
    with pytest.raises(ValueError):
        attn(q, kc[:, :, :8], vc[:, :, :8], ks, vs, table, lens)
    with pytest.raises(ValueError):
        attn(q, kc, vc, ks[:, :1], vs, table, lens)
    with pytest.raises(ValueError):
        attn(q, kc, vc, ks, vs, table.cpu(), lens)
    with pytest.raises(ValueError):
        attn(q, kc, vc, ks, vs, table, lens, scale=-1.0)
    with pytest.raises(ValueError):
        attn(q.expand(1, 2, 4, 128), kc, vc, ks, vs, table, lens)
    with pytest.raises(ValueError):
        attn(q, kc, vc, ks, vs, table, lens, out=q[:, :, :2])
    with pytest.raises(ValueError):
        attn(q, kc, vc, ks, vs, table, lens, out=q)
    with pytest.raises(ValueError):
        write(k, k[:, :, :1], kc, vc, ks, vs, table, lens)
    with pytest.raises(ValueError):
        write(q, q, kc, vc, ks, vs, table, lens)  # four heads into a cache of two
    with pytest.raises(ValueError):
        write(k, k, kc, vc, ks, vs, table, lens.repeat(2))
    empty = torch.zeros((0, 1, 4, 128), dtype=torch.bfloat16, device=DEV)
    assert attn(empty, kc, vc, ks, vs, table[:0], lens[:0]).shape == empty.shape
    _ok()


# --- cross_attn ----------------------------------------------------------------------


def _cross_inputs(seed, b, t, n, h, kv):
    g = torch.Generator().manual_seed(seed)
    return _randn(g, b, t, h, 128), _randn(g, b, n, kv, 128), _randn(g, b, n, kv, 128)


def _spoil(x, lens):
    """What lies behind the keys of each entry: NaN and infinities."""
    for i, m in enumerate(lens):
        x[i, m:] = math.nan
        x[i, m:, :, ::3] = math.inf
    return x


def _cross_check(q, k, v, lens=None, scale=None, **kw):
    dev_lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    out, lse = b200_gemm.cross_attn(*_on([q, k, v]), kv_lens=dev_lens, scale=scale, return_lse=True, **kw)
    _ok()
    want = ref.cross_attn(q, k, v, lens, 128 ** -0.5 if scale is None else scale)
    _within(out, *want["out"], "out")
    _within(lse, *want["lse"], "lse")
    return out


@pytest.mark.parametrize("heads", [(2, 2), (8, 2), (3, 1)], ids=["mha", "gqa", "mqa"])
@pytest.mark.parametrize("n", [1, 63, 64, 65, 127, 128, 129, 300, 777])
@pytest.mark.parametrize("t", [1, 5, 16, 33, 65, 128, 129, 257, 300])
def test_cross_attn_lengths(t, n, heads):
    _cross_check(*_cross_inputs(t * 1000 + n, 2, t, n, *heads))


@pytest.mark.parametrize("t", [1, 7, 100, 200, 600])
def test_cross_attn_ragged_sources(t):
    """Lengths on the device, an empty source, NaN and infinities behind every source."""
    lens = [0, 1, 100, 128, 129, 383, 384]
    q, k, v = _cross_inputs(t, len(lens), t, 384, 4, 2)
    _cross_check(q, _spoil(k, lens), _spoil(v, lens), lens)


@pytest.mark.parametrize("t", [1, 4, 100, 200])
@pytest.mark.parametrize("lens", [[0, 1, 31, 32, 33, 4000, 8999, 9000], [0, 0, 1, 0, 5, 130, 0, 0]], ids=["mixed", "short"])
def test_cross_attn_ragged_long_sources(t, lens):
    """Few rows per key/value head: workers or parts along the keys, most of which have no keys of a short source."""
    q, k, v = _cross_inputs(t + len(lens), len(lens), t, 9000, 8 if t < 100 else 2, 2 if t < 100 else 1)
    _cross_check(q, _spoil(k, lens), _spoil(v, lens), lens)


@pytest.mark.parametrize("batch,heads", [(12, (16, 4)), (40, (8, 8))], ids=["few entries", "many entries"])
@pytest.mark.parametrize("t", [100, 300])
def test_cross_attn_more_work_than_sms(t, batch, heads):
    """Several CTAs per SM, entries of many and of no keys among them."""
    lens = [(i * 211) % 501 for i in range(batch)]
    lens[-1] = 500
    q, k, v = _cross_inputs(t + batch, batch, t, 500, *heads)
    _cross_check(q, _spoil(k, lens), _spoil(v, lens), lens)


@pytest.mark.parametrize("t", [1, 150])
def test_cross_attn_lengths_are_clamped(t):
    q, k, v = _cross_inputs(t + 7, 3, t, 100, 2, 2)
    lens = torch.tensor([-5, 100, 1 << 30], dtype=torch.int32, device=DEV)
    out = b200_gemm.cross_attn(*_on([q, k, v]), kv_lens=lens)
    _ok()
    want = ref.cross_attn(q, k, v, [0, 100, 100])
    _within(out, *want["out"])


@pytest.mark.parametrize("t", [1, 9, 150])
def test_cross_attn_no_keys(t):
    q, k, v = _cross_inputs(t, 2, t, 0, 4, 2)
    out, lse = b200_gemm.cross_attn(*_on([q, k, v]), return_lse=True)
    _ok()
    assert not bool(out.any()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("t", [3, 140])
def test_cross_attn_strides_scale_and_out(t):
    """q with heads before tokens, k and v as views of one fused projection, out strided."""
    g = torch.Generator().manual_seed(t)
    q, kv = _randn(g, 2, 4, t, 128).transpose(1, 2), _randn(g, 2, 200, 2, 2, 128)
    want = ref.cross_attn(q, kv[:, :, 0], kv[:, :, 1], None, 0.11)
    buf = torch.full((2, t, 6, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    d = kv.to(DEV)
    got = b200_gemm.cross_attn(q.to(DEV), d[:, :, 0], d[:, :, 1], scale=0.11, out=buf[:, :, 1:5])
    _ok()
    _within(got, *want["out"])
    assert bool((buf[:, :, 0] == 7.0).all()) and bool((buf[:, :, 5] == 7.0).all())


def test_cross_attn_growing_scores():
    """Keys that score higher and higher: the running maximum keeps moving."""
    for t in (2, 130):
        q, k, v = _cross_inputs(t, 1, t, 900, 2, 2)
        k = (k.float() * torch.linspace(0.2, 3.0, 900).view(1, 900, 1, 1)).to(torch.bfloat16)
        _cross_check(q, k, v)


@pytest.mark.parametrize("t", [1, 130])
@pytest.mark.parametrize("n", [1, 64, 128, 1000])
def test_cross_attn_lse_of_equal_keys(t, n):
    """q = 0: every key weighs exactly 1 and the sum is n; log2, its product with ln 2 and the parts' weights add less than
    2^-20 (1 + lse)."""
    q, k, v = _cross_inputs(t + n, 1, t, n, 2, 2)
    q.zero_()
    out, lse = b200_gemm.cross_attn(*_on([q, k, v]), return_lse=True)
    _ok()
    assert float((lse.double().cpu() - math.log(n)).abs().max()) <= 2.0 ** -20 * (1 + math.log(n))
    _within(out, *ref.cross_attn(q, k, v)["out"])


def test_cross_attn_agrees_with_flash_attn_on_square_shapes():
    """The same function: both within the bound of the exact result (their key tiles may be added in another order)."""
    for n in (384, 512):
        q, k, v = _cross_inputs(21 + n, 2, n, n, 4, 2)
        want = ref.cross_attn(q, k, v)["out"]
        _within(b200_gemm.cross_attn(*_on([q, k, v])), *want, "cross")
        _within(b200_gemm.flash_attn(*_on([q, k, v]), causal=False), *want, "flash")
    _ok()


def test_cross_attn_long_source():
    q, k, v = _cross_inputs(22, 1, 1, 20000, 2, 1)
    a = _cross_check(q, k, v)
    b = b200_gemm.cross_attn(*_on([q, k, v]))
    assert torch.equal(a, b)


def test_cross_refusals():
    q, k, v = (t.to(DEV) for t in _cross_inputs(0, 2, 3, 5, 4, 2))
    f = b200_gemm.cross_attn
    with pytest.raises(ValueError):
        f(q, k, v[:, :4])
    with pytest.raises(ValueError):
        f(q, k[:1], v[:1])
    with pytest.raises(ValueError):
        f(q[:, :, :3], k, v)
    with pytest.raises(TypeError):
        f(q, k.half(), v.half())
    with pytest.raises(TypeError):
        f(q, k, v, kv_lens=torch.ones(2, device=DEV))
    with pytest.raises(ValueError):
        f(q, k, v, kv_lens=torch.ones(3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        f(q, k[:1].expand(2, 5, 2, 128), v)
    with pytest.raises(ValueError):
        f(q, k, v, scale=0.0)
    with pytest.raises(ValueError):
        f(q[..., :64], k[..., :64], v[..., :64])
    with pytest.raises(ValueError):
        f(q, k, v, out=q[:, :2])
    with pytest.raises(ValueError):
        f(q, k, v, out=q)
    assert f(q[:, :0], k, v).shape == (2, 0, 4, 128)
    _ok()


# --- cross_attn_backward ---------------------------------------------------------------


def _grad_check(q, k, v, do, lens=None, scale=None, dev=None):
    dq, dk, dv, ddo = _on([q, k, v, do]) if dev is None else dev
    dev_lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    out, lse = b200_gemm.cross_attn(dq, dk, dv, kv_lens=dev_lens, scale=scale, return_lse=True)
    grads = b200_gemm.cross_attn_backward(ddo, dq, dk, dv, out, lse, kv_lens=dev_lens, scale=scale)
    _ok()
    want = ref.cross_attn(q, k, v, lens, 128 ** -0.5 if scale is None else scale, do)
    for name, got in zip(("dq", "dk", "dv"), grads):
        _within(got, *want[name], name)
    return grads


@pytest.mark.parametrize("heads", [(2, 2), (8, 2), (3, 1)], ids=["mha", "gqa", "mqa"])
@pytest.mark.parametrize("n", [1, 64, 127, 128, 129, 300, 640])
@pytest.mark.parametrize("t", [1, 5, 64, 127, 128, 129, 300, 520])
def test_backward_lengths(t, n, heads):
    q, k, v = _cross_inputs(t * 1000 + n + 1, 2, t, n, *heads)
    _grad_check(q, k, v, _randn(torch.Generator().manual_seed(t + n), *q.shape))


@pytest.mark.parametrize("t", [1, 100, 300])
def test_backward_ragged_sources(t):
    """Lengths on the device, an empty source, NaN and infinities behind every source; dk and dv are 0 there."""
    lens = [0, 1, 100, 128, 129, 383, 384]
    q, k, v = _cross_inputs(t + 50, len(lens), t, 384, 4, 2)
    do = _randn(torch.Generator().manual_seed(t), *q.shape)
    dq, dk, dv = _grad_check(q, _spoil(k, lens), _spoil(v, lens), do, lens)
    assert not bool(dq[0].any())
    for i, m in enumerate(lens):
        assert not bool(dk[i, m:].any()) and not bool(dv[i, m:].any())


@pytest.mark.parametrize("batch,heads", [(12, (16, 8)), (40, (6, 6))], ids=["few entries", "many entries"])
def test_backward_more_items_than_sms(batch, heads):
    """Every CTA takes several items, of many and of no tiles."""
    lens = [(i * 211) % 301 for i in range(batch)]
    lens[-1] = 300
    q, k, v = _cross_inputs(batch, batch, 200, 300, *heads)
    do = _randn(torch.Generator().manual_seed(batch), *q.shape)
    dq, dk, dv = _grad_check(q, _spoil(k, lens), _spoil(v, lens), do, lens)
    for i, m in enumerate(lens):
        assert not bool(dk[i, m:].any()) and not bool(dv[i, m:].any())


@pytest.mark.parametrize("shape", [(1, 700, 500, 8, 1), (1, 60, 3500, 4, 2), (2, 1300, 40, 4, 1), (3, 200, 5000, 4, 2),
                                   (3, 500, 1100, 12, 1), (1, 1, 2000, 8, 2), (4, 2000, 1, 2, 1)],
                         ids=lambda s: "x".join(map(str, s)))
def test_backward_few_long_items(shape):
    """Fewer items than SMs, each with many tiles: many query rows per key tile, or many keys per query tile."""
    b, t, n, h, kv = shape
    lens = None if b == 1 else [n, n // 3, 1, 0][:b]
    q, k, v = _cross_inputs(n, b, t, n, h, kv)
    do = _randn(torch.Generator().manual_seed(t), *q.shape)
    if lens is not None:
        k, v = _spoil(k, lens), _spoil(v, lens)
    first = _grad_check(q, k, v, do, lens)
    assert all(torch.equal(a, c) for a, c in zip(first, _grad_check(q, k, v, do, lens)))


def test_backward_strides_and_scale():
    g = torch.Generator().manual_seed(61)
    q, kv = _randn(g, 2, 4, 200, 128).transpose(1, 2), _randn(g, 2, 150, 2, 2, 128)
    do = _randn(g, 2, 200, 6, 128)[:, :, 1:5]
    d = kv.to(DEV)
    _grad_check(q, kv[:, :, 0], kv[:, :, 1], do, None, 0.07, (q.to(DEV), d[:, :, 0], d[:, :, 1], do.to(DEV)))


def test_backward_empty_sides():
    for t, n in ((0, 130), (130, 0)):
        q, k, v = _cross_inputs(t, 2, t, n, 4, 2)
        q, k, v = _on([q, k, v])
        out, lse = b200_gemm.cross_attn(q, k, v, return_lse=True)
        grads = b200_gemm.cross_attn_backward(torch.ones_like(out), q, k, v, out, lse)
        _ok()
        assert all(a.shape == b.shape and not bool(a.any()) for a, b in zip(grads, (q, k, v)))


def test_backward_repeats_bit_for_bit():
    q, k, v = _on(_cross_inputs(62, 2, 700, 900, 8, 2))
    do = _randn(torch.Generator().manual_seed(63), *q.shape).to(DEV)
    out, lse = b200_gemm.cross_attn(q, k, v, return_lse=True)
    first = b200_gemm.cross_attn_backward(do, q, k, v, out, lse)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(first, b200_gemm.cross_attn_backward(do, q, k, v, out, lse)))
    _ok()


def test_backward_refusals():
    q, k, v = _on(_cross_inputs(0, 2, 3, 5, 4, 2))
    out, lse = b200_gemm.cross_attn(q, k, v, return_lse=True)
    f = b200_gemm.cross_attn_backward
    with pytest.raises(ValueError):
        f(out[:, :2], q, k, v, out, lse)
    with pytest.raises(ValueError):
        f(out[:, :1].expand(2, 3, 4, 128), q, k, v, out, lse)  # a broadcast gradient is materialised by its owner
    for i in range(6):
        args = [out, q, k, v, out, lse]
        args[i] = None
        with pytest.raises(TypeError):
            f(*args)
    with pytest.raises(TypeError):
        f(out, q, k, v, out, lse.double())
    with pytest.raises(ValueError):
        f(out, q, k, v, out, lse.transpose(1, 2))
    with pytest.raises(ValueError):
        f(out, q, k, v[:, :4], out, lse)
    with pytest.raises(ValueError):
        f(out, q, k, v, out, lse, scale=math.nan)
    _ok()


def test_backward_workspace_is_checked():
    """Few gradient tiles: the fp32 sums of their parts are in the workspace, and one byte less is refused."""
    import ctypes

    from b200_gemm import _lib
    lib = _lib.load()
    q, k, v = _on(_cross_inputs(66, 1, 600, 900, 4, 1))
    out, lse = b200_gemm.cross_attn(q, k, v, return_lse=True)
    do = torch.ones_like(q)
    need = ctypes.c_size_t(0)
    assert lib.b200_cross_attn_bwd_workspace_bytes(1, 600, 900, 4, 1, ctypes.byref(need)) == _lib.B200_OK
    plain = 256 + 2 * 4 * 4 * 640  # counters, and two floats per padded query row
    assert need.value > plain
    ws = torch.empty(need.value, dtype=torch.uint8, device=DEV)
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]

    def view(t):
        return ctypes.byref(_lib.AttnView(t.data_ptr(), *t.stride()[:3]))

    def call(n):
        return lib.b200_cross_attn_bwd_bf16(view(q), view(k), view(v), view(out), view(do), lse.data_ptr(), None, *map(view, grads),
                                            1, 600, 900, 4, 1, 128, 128 ** -0.5, ws.data_ptr(), n, None)

    torch.cuda.synchronize()
    for n in (need.value - 1, plain, plain - 1, 0):
        assert call(n) == _lib.B200_ERR_INVALID_ARG
    torch.cuda.synchronize()
    assert all(bool((t == 7.0).all()) for t in grads)
    assert call(need.value) == _lib.B200_OK
    _ok()
    assert all(torch.equal(a, b) for a, b in zip(grads, b200_gemm.cross_attn_backward(do, q, k, v, out, lse)))


def test_training_step_captured_and_on_another_stream():
    """Forward and backward in a captured graph, replayed with new inputs, and on a side stream."""
    g = torch.Generator().manual_seed(64)
    q, k, v = _cross_inputs(65, 2, 150, 200, 4, 2)
    lens = [200, 70]
    dev = _on([q, k, v, _randn(g, *q.shape)])
    dev_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def step(**kw):
        out, lse = b200_gemm.cross_attn(*dev[:3], kv_lens=dev_lens, return_lse=True, **kw)
        return out, *b200_gemm.cross_attn_backward(dev[3], *dev[:3], out, lse, kv_lens=dev_lens, **kw)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        new = [_randn(g, *t.shape) for t in dev]
        for d, x in zip(dev, new):
            d.copy_(x)
        graph.replay()
        graph.replay()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        on_side = step(stream=side)
        torch.cuda.current_stream().wait_stream(side)
        _ok()
        want = ref.cross_attn(*new[:3], lens, dout=new[3])
        for name, a, b in zip(("out", "dq", "dk", "dv"), got, on_side):
            _within(a, *want[name], name)
            assert torch.equal(a, b)


# --- streams, graphs, together -----------------------------------------------------------


def test_other_stream_and_captured_graphs():
    """Two captured graphs with workspaces of their own, replayed in turn with new inputs, and calls on a side stream."""
    g = torch.Generator().manual_seed(31)
    caches = [_filled(g, [900, 333], 2, 32), _filled(g, [64, 2000], 2, 32)]
    qs = [_randn(g, 2, 1, 8, 128) for _ in range(2)]
    cross = _cross_inputs(32, 2, 1, 1500, 8, 2)
    side = torch.cuda.Stream()
    dev, graphs, outs = [_on(c) for c in caches], [], []
    dq, dx = [q.to(DEV) for q in qs], _on(cross)
    b200_gemm.cache_attn(dq[0], *dev[0])
    b200_gemm.cross_attn(*dx)
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((b200_gemm.cache_attn(dq[i], *dev[i]), b200_gemm.cross_attn(dq[i], dx[1], dx[2])))
        graphs.append(graph)
    for step in range(3):
        new = [_randn(g, 2, 1, 8, 128) for _ in range(2)]
        for i in range(2):
            dq[i].copy_(new[i])
        for i in (0, 1, 0, 1):
            graphs[i].replay()
        side.wait_stream(torch.cuda.current_stream())
        on_side = b200_gemm.cache_attn(dq[0], *dev[0], stream=side), b200_gemm.cross_attn(dq[0], dx[1], dx[2], stream=side)
        torch.cuda.current_stream().wait_stream(side)
        _ok()
        for i in range(2):
            want, bound = ref.cache_attn(new[i], *caches[i])
            _within(outs[i][0], want, bound)
            _within(outs[i][1], *ref.cross_attn(new[i], cross[1], cross[2])["out"])
        assert torch.equal(on_side[0], outs[0][0]) and torch.equal(on_side[1], outs[0][1])


def test_calls_on_two_streams_at_once():
    """Forward, backward and cache calls of two streams beside each other, each as when alone."""
    g = torch.Generator().manual_seed(51)
    sets = []
    for i in range(2):
        q, k, v = _on(_cross_inputs(52 + i, 2, 300 + 200 * i, 700, 8, 2))
        cache = _on(_filled(g, [3000, 10 + i, 9000], 1, 64))
        sets.append((q, k, v, torch.randn_like(q), cache, _randn(g, 3, 1, 8, 128).to(DEV), torch.randn_like(q[:, :1])))

    def run(s, stream):
        q, k, v, do, cache, dq, few = s
        out, lse = b200_gemm.cross_attn(q, k, v, return_lse=True, stream=stream)
        return [out, lse, *b200_gemm.cross_attn_backward(do, q, k, v, out, lse, stream=stream),
                b200_gemm.cache_attn(dq, *cache, stream=stream), b200_gemm.cross_attn(few, k, v, stream=stream)]

    alone = [run(s, None) for s in sets]
    _ok()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(sets):
            got[i].append(run(s, streams[i]))
    _ok()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(alone[i], r))


def test_decoder_layer_steps():
    """Five tokens, one after the other, through projections (gemm), the cache, attention over it and cross attention,
    against the same in 64 bits on the operands each step saw."""
    g = torch.Generator().manual_seed(41)
    B, H, KV, E = 3, 4, 2, 256
    wqkv = _randn(g, (H + 2 * KV) * 128, E, scale=E ** -0.5).to(DEV)
    wo, wq = _randn(g, E, H * 128, scale=0.04).to(DEV), _randn(g, H * 128, E, scale=0.06).to(DEV)
    enc = _randn(g, B, 90, 2, KV, 128).to(DEV)
    enc_lens = torch.tensor([90, 17, 0], dtype=torch.int32, device=DEV)
    kc, vc, ks, vs, table = _on(_pool(g, B, KV, 16, 64))
    lens = torch.tensor([0, 14, 31], dtype=torch.int32, device=DEV)
    past = _randn(g, B, 31, KV, 128).to(DEV), _randn(g, B, 31, KV, 128).to(DEV)
    b200_gemm.kv_cache_write(*past, kc, vc, ks, vs, table, lens, new_lens=lens)
    x = _randn(g, B, E).to(DEV)
    for _ in range(5):
        lens += 1
        qkv = b200_gemm.matmul(x, wqkv).view(B, 1, H + 2 * KV, 128)
        q, k, v = qkv[:, :, :H], qkv[:, :, H:H + KV], qkv[:, :, H + KV:]
        b200_gemm.kv_cache_write(k, v, kc, vc, ks, vs, table, lens)
        a = b200_gemm.cache_attn(q, kc, vc, ks, vs, table, lens)
        y = b200_gemm.gemm(a.view(B, H * 128), wo, beta=1.0, c=x)
        q2 = b200_gemm.matmul(y, wq).view(B, 1, H, 128)
        c = b200_gemm.cross_attn(q2, enc[:, :, 0], enc[:, :, 1], kv_lens=enc_lens)
        x = b200_gemm.gemm(c.view(B, H * 128), wo, beta=1.0, c=y)
        _ok()
        want, bound = ref.cache_attn(q.cpu(), kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), table.cpu(), lens.cpu())
        _within(a, want, bound, "cache")
        _within(c, *ref.cross_attn(q2.cpu(), enc[:, :, 0].cpu(), enc[:, :, 1].cpu(), enc_lens.cpu())["out"], "cross")
        got = kc.cpu(), ks.cpu()
        for b in range(B):  # the newest keys are in the cache, within half a step of e4m3 (2^-4, or 2^-10 s below 2^-6 s)
            n = int(lens[b])
            for h in range(KV):
                last = ref.cache_values(*got, table[b].cpu(), n, h)[-1]
                s = float(got[1][int(table[b, (n - 1) // 16]), h])
                new = k[b, 0, h].double().cpu()
                assert bool(((last - new).abs() <= torch.clamp(new.abs() * 2.0 ** -4, min=2.0 ** -10 * s)).all())
