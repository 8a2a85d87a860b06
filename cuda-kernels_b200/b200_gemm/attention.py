"""Attention to stored keys and values, through the C ABI (include/b200_gemm.h): a paged key/value cache in 8
bits, attention of the newest tokens over it, and cross attention to an encoder's states.  The reference's attention
operator (flash_attn/flash_attn.cpp:16-30) has one length for queries and keys and keeps no state; `flash_attn` in
ops.py is its counterpart, and these stand beside it.

One decoder layer of a serving step, with x the new tokens' activations and `gemm` the projections:

    kv_cache_write(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens)
    a = cache_attn(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens)
    c = cross_attn(q2, enc_k, enc_v, kv_lens=enc_lens)

Every tensor is on one CUDA device; calls run on torch's current stream of that device or on `stream`.  With `stream`,
outputs and workspaces come from that stream's memory pool; ordering the inputs before it and the outputs after it is
the caller's.  All calls can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._lib import B200GemmError

HEAD_DIM = 128
PAGE_SIZES = (16, 32, 64, 128)


def _view(name: str, t: torch.Tensor, heads: int | None = None) -> _lib.AttnView:
    """A [batch, tokens, heads, 128] bf16 CUDA tensor as a b200_attn_view."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be a bfloat16 torch.Tensor")
    if not t.is_cuda or t.dim() != 4:
        raise ValueError(f"{name} must be a 4-D CUDA tensor [batch, tokens, heads, {HEAD_DIM}]")
    if t.shape[3] != HEAD_DIM:
        raise ValueError(f"{name} must have head_dim {HEAD_DIM}, got {t.shape[3]}")
    if heads is not None and t.shape[2] != heads:
        raise ValueError(f"{name} must have {heads} heads, got {t.shape[2]}")
    sb, st, sh, sd = t.stride()
    if t.numel() > 0:
        if sd != 1:
            raise ValueError(f"{name} must be contiguous in its last dimension, got strides {t.stride()}")
        for extent, stride in zip(t.shape, (sb, st, sh)):
            if extent > 1 and (stride < HEAD_DIM or stride % 8 != 0):
                raise ValueError(f"{name}'s strides must be multiples of 8, at least {HEAD_DIM} (expanded tensors are "
                                 f"not taken), got {t.stride()}")
    return _lib.AttnView(t.data_ptr(), sb, st, sh)


def _lens(name: str, t: torch.Tensor | None, batch: int, device: torch.device) -> int | None:
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 torch.Tensor")
    if t.device != device or t.shape != (batch,) or (batch > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous [{batch}] tensor on {device}")
    return t.data_ptr()


def _cache(k_cache, v_cache, k_scale, v_scale, block_table, batch: int, device: torch.device) -> _lib.KvCache:
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float8_e4m3fn:
            raise TypeError(f"{name} must be a float8_e4m3fn torch.Tensor")
        if t.dim() != 4 or t.shape[3] != HEAD_DIM or t.shape[2] not in PAGE_SIZES or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous [num_pages, kv_heads, page_size, {HEAD_DIM}] with page_size in "
                             f"{PAGE_SIZES}, got {tuple(t.shape)}")
    pages, kv_heads, page, _ = k_cache.shape
    if v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
            raise TypeError(f"{name} must be a float32 torch.Tensor")
        if t.shape != (pages, kv_heads) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous [{pages}, {kv_heads}], got {tuple(t.shape)}")
    if not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32:
        raise TypeError("block_table must be an int32 torch.Tensor")
    if block_table.dim() != 2 or block_table.shape[0] != batch or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be row-major [{batch}, max_pages], got {tuple(block_table.shape)}")
    if not (k_cache.device == v_cache.device == k_scale.device == v_scale.device == block_table.device == device):
        raise ValueError("the cache, its scales and the block table must be on the device of the other tensors")
    rows, most = block_table.shape
    stride = block_table.stride(0) if rows > 1 else most
    if stride < most:
        raise ValueError("block_table's rows overlap")
    return _lib.KvCache(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, page,
                        kv_heads, block_table.data_ptr(), stride, most)


def _scale(scale: float | None) -> float:
    if scale is None:
        return HEAD_DIM ** -0.5
    scale = float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def _on(device: torch.device, stream: torch.cuda.Stream | None, call):
    """call(stream handle, allocate) with `device` current; allocate(shape, dtype) gives memory whose use on the call's
    stream is ordered (and which may also be used on the stream that was current)."""
    index = device.index
    if stream is None and index == torch.cuda.current_device():
        return call(torch.cuda.current_stream().cuda_stream,
                    lambda shape, dtype: torch.empty(shape, dtype=dtype, device=device))
    with torch.cuda.device(index):
        if stream is None:
            stream = torch.cuda.current_stream(device)
        elif stream.device != device:
            raise ValueError(f"stream is on {stream.device}, the tensors on {device}")
        current = torch.cuda.current_stream(device)

        def allocate(shape, dtype):
            with torch.cuda.stream(stream):
                t = torch.empty(shape, dtype=dtype, device=device)
            if stream != current:
                t.record_stream(current)
            return t

        return call(stream.cuda_stream, allocate)


def _check(rc: int, what: str) -> None:
    if rc != _lib.B200_OK:
        raise B200GemmError(rc, what)


def _workspace(allocate, nbytes: int):
    """(tensor to keep alive, 256-byte aligned pointer or None): torch's allocations are 512-byte aligned."""
    if nbytes == 0:
        return None, None
    ws = allocate((nbytes,), torch.uint8)
    assert ws.data_ptr() % 256 == 0
    return ws, ws.data_ptr()


def kv_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                   v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                   new_lens: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> None:
    """Append new keys and values to the paged 8-bit cache, in place (b200_kv_cache_write).

    k, v: bf16 [batch, new_max, kv_heads, 128], any strides that keep the last dimension contiguous.
    k_cache, v_cache: float8_e4m3fn [num_pages, kv_heads, page_size, 128], page_size 16, 32, 64 or 128; k_scale, v_scale:
    float32 [num_pages, kv_heads]; a value is code * scale.  block_table: int32 [batch, max_pages], place j of sequence b
    is slot j % page_size of page block_table[b, j // page_size].  seq_lens: int32 [batch], lengths with the new tokens;
    new_lens: int32 [batch], how many of them are new (default: new_max).

    A page's scale is the smallest power of two >= 2**-100 that brings its values within 448; it grows while the page
    fills (codes already there are rounded to it) and starts afresh when slot 0 is written.  No page may belong to two
    sequences of one call.  Lengths or pages out of range leave their sequence unwritten and are raised by
    check_status()."""
    cache_heads = k_cache.shape[1] if isinstance(k_cache, torch.Tensor) and k_cache.dim() == 4 else None
    kk, vv = _view("k", k, cache_heads), _view("v", v, cache_heads)
    if v.shape != k.shape or v.device != k.device:
        raise ValueError("k and v must have the same shape and device")
    batch, new_max = k.shape[:2]
    cache = _cache(k_cache, v_cache, k_scale, v_scale, block_table, batch, k.device)
    if seq_lens is None:
        raise TypeError("seq_lens must be an int32 torch.Tensor")
    lens, fresh = _lens("seq_lens", seq_lens, batch, k.device), _lens("new_lens", new_lens, batch, k.device)
    lib = _lib.load()
    rc = _on(k.device, stream, lambda s, _: lib.b200_kv_cache_write(kk, vv, cache, lens, fresh, batch, new_max, HEAD_DIM, s))
    _check(rc, f"kv_cache_write batch={batch} new_max={new_max} kv_heads={k.shape[2]}")


@functools.lru_cache(maxsize=256)
def _cache_attn_workspace(index: int, batch: int, q_len: int, heads: int, pages: int, page: int, kv_heads: int,
                          most: int) -> int:
    """Workspace bytes for these sizes on the current device (`index`)."""
    n = ctypes.c_size_t(0)
    sizes = _lib.KvCache(None, None, None, None, pages, page, kv_heads, None, most, most)
    _check(_lib.load().b200_cache_attn_workspace_bytes(batch, q_len, heads, sizes, ctypes.byref(n)), "cache_attn workspace")
    return n.value


def cache_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
               block_table: torch.Tensor, seq_lens: torch.Tensor, *, new_lens: torch.Tensor | None = None,
               scale: float | None = None, out: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Attention of each sequence's newest tokens over the cache of kv_cache_write (b200_cache_attn).

    q: bf16 [batch, q_len, heads, 128], heads a multiple of kv_heads (query head h reads key/value head
    h // (heads // kv_heads)).  seq_lens: lengths with the new tokens, which are already in the cache; new_lens: how many
    of q's tokens a sequence has (default: q_len).  Query t is at place seq_lens - new_lens + t and attends to the places
    up to its own.  Rows past new_lens and rows that see nothing are 0.  scale defaults to 128 ** -0.5."""
    qq = _view("q", q)
    batch, q_len, heads, _ = q.shape
    cache = _cache(k_cache, v_cache, k_scale, v_scale, block_table, batch, q.device)
    kv_heads = cache.kv_heads
    if (heads > 0 and kv_heads == 0) or (kv_heads > 0 and heads % kv_heads != 0):
        raise ValueError(f"the number of query heads ({heads}) must be a multiple of the cache's ({kv_heads})")
    if seq_lens is None:
        raise TypeError("seq_lens must be an int32 torch.Tensor")
    lens, fresh = _lens("seq_lens", seq_lens, batch, q.device), _lens("new_lens", new_lens, batch, q.device)
    scale = _scale(scale)
    if out is not None:
        _check_out(out, q)
    lib = _lib.load()

    def call(s, allocate):
        o = out if out is not None else allocate(q.shape, torch.bfloat16)
        n = _cache_attn_workspace(q.device.index, batch, q_len, heads, cache.num_pages, cache.page_size, kv_heads,
                                  cache.max_pages) if q.numel() else 0
        ws, ptr = _workspace(allocate, n)
        rc = lib.b200_cache_attn(qq, cache, lens, fresh, _view("out", o), batch, q_len, heads, HEAD_DIM, scale, ptr, n, s)
        _check(rc, f"cache_attn batch={batch} q_len={q_len} heads={heads} kv_heads={kv_heads}")
        return o

    return _on(q.device, stream, call)


def _check_out(out: torch.Tensor, q: torch.Tensor) -> None:
    _view("out", out)
    if out.shape != q.shape or out.device != q.device:
        raise ValueError(f"out must be {tuple(q.shape)} on {q.device}, got {tuple(out.shape)} on {out.device}")


def _cross_shapes(q, k, v):
    batch, q_len, heads, _ = q.shape
    if k.shape != v.shape or k.shape[0] != batch or not (k.device == v.device == q.device):
        raise ValueError("k and v must have the same shape, and q's batch and device")
    kv_len, kv_heads = k.shape[1:3]
    if (heads > 0 and kv_heads == 0) or (kv_heads > 0 and heads % kv_heads != 0):
        raise ValueError(f"the number of query heads ({heads}) must be a multiple of the key/value heads ({kv_heads})")
    return batch, q_len, kv_len, heads, kv_heads


@functools.lru_cache(maxsize=256)
def _cross_attn_workspace(index: int, batch: int, q_len: int, kv_len: int, heads: int, kv_heads: int) -> int:
    """Workspace bytes for these sizes on the current device (`index`)."""
    n = ctypes.c_size_t(0)
    _check(_lib.load().b200_cross_attn_workspace_bytes(batch, q_len, kv_len, heads, kv_heads, ctypes.byref(n)),
           "cross_attn workspace")
    return n.value


def cross_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, kv_lens: torch.Tensor | None = None,
               scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False,
               stream: torch.cuda.Stream | None = None):
    """Cross attention softmax(scale q k^T) v to an encoder's states of another length (b200_cross_attn_bf16).

    q: bf16 [batch, q_len, heads, 128]; k, v: bf16 [batch, kv_len, kv_heads, 128], heads a multiple of kv_heads; any strides
    that keep the last dimension contiguous (a fused projection's views, [batch, heads, tokens, 128] storage).  kv_lens:
    int32 [batch], keys of each entry (default: kv_len); what lies behind them is not used.  An entry without keys gives 0.
    return_lse=True returns (out, lse) with lse float32 [batch, heads, q_len], the natural log of the softmax denominator
    (-inf without keys), which cross_attn_backward takes.  scale defaults to 128 ** -0.5."""
    qq, kk, vv = _view("q", q), _view("k", k), _view("v", v)
    batch, q_len, kv_len, heads, kv_heads = _cross_shapes(q, k, v)
    lens = _lens("kv_lens", kv_lens, batch, q.device)
    scale = _scale(scale)
    if out is not None:
        _check_out(out, q)
    lib = _lib.load()

    def call(s, allocate):
        o = out if out is not None else allocate(q.shape, torch.bfloat16)
        lse = allocate((batch, heads, q_len), torch.float32) if return_lse else None
        n = _cross_attn_workspace(q.device.index, batch, q_len, kv_len, heads, kv_heads)
        ws, ptr = _workspace(allocate, n)
        rc = lib.b200_cross_attn_bf16(qq, kk, vv, lens, _view("out", o), lse.data_ptr() if return_lse else None, batch, q_len,
                                      kv_len, heads, kv_heads, HEAD_DIM, scale, ptr, n, s)
        _check(rc, f"cross_attn batch={batch} q_len={q_len} kv_len={kv_len} heads={heads} kv_heads={kv_heads}")
        return (o, lse) if return_lse else o

    return _on(q.device, stream, call)


def cross_attn_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                        lse: torch.Tensor, *, kv_lens: torch.Tensor | None = None, scale: float | None = None,
                        stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv) of cross_attn (b200_cross_attn_bwd_bf16), bf16, shaped like q, k and v.

    out and lse are what cross_attn(..., return_lse=True) gave for the same q, k, v, kv_lens and scale; dout is the gradient
    of out.  dk and dv are summed over the query heads of a group and 0 behind an entry's keys.  The sums run in a fixed
    order: equal inputs give equal bits."""
    views = [_view(name, t) for name, t in (("q", q), ("k", k), ("v", v), ("out", out), ("dout", dout))]
    batch, q_len, kv_len, heads, kv_heads = _cross_shapes(q, k, v)
    for name, t in (("out", out), ("dout", dout)):
        if t.shape != q.shape or t.device != q.device:
            raise ValueError(f"{name} must be {tuple(q.shape)} on {q.device}, got {tuple(t.shape)} on {t.device}")
    if not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32:
        raise TypeError("lse must be a float32 torch.Tensor")
    if lse.shape != (batch, heads, q_len) or lse.device != q.device or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous [{batch}, {heads}, {q_len}] on {q.device}, got {tuple(lse.shape)}")
    lens = _lens("kv_lens", kv_lens, batch, q.device)
    scale = _scale(scale)
    lib = _lib.load()

    def call(s, allocate):
        grads = [allocate(t.shape, torch.bfloat16) for t in (q, k, v)]
        n = ctypes.c_size_t(0)
        _check(lib.b200_cross_attn_bwd_workspace_bytes(batch, q_len, heads, ctypes.byref(n)), "cross_attn_backward workspace")
        ws, ptr = _workspace(allocate, n.value)
        outs = [_view(name, t) for name, t in zip(("dq", "dk", "dv"), grads)]
        rc = lib.b200_cross_attn_bwd_bf16(*views, lse.data_ptr(), lens, *outs, batch, q_len, kv_len, heads, kv_heads, HEAD_DIM,
                                          scale, ptr, n.value, s)
        _check(rc, f"cross_attn_backward batch={batch} q_len={q_len} kv_len={kv_len} heads={heads} kv_heads={kv_heads}")
        return tuple(grads)

    return _on(q.device, stream, call)
