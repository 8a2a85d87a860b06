"""Attention to stored keys and values, through the C ABI (include/b200_gemm.h): a paged key/value cache in 8
bits, attention of the newest tokens over it, and cross attention to an encoder's states.  The reference's attention
operator (flash_attn/flash_attn.cpp:16-30) has one length for queries and keys and keeps no state; `flash_attn` in
ops.py is its counterpart, and these stand beside it.

One decoder layer of a serving step, with x the new tokens' activations and `gemm` the projections:

    kv_cache_write(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens)
    a = cache_attn(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens)
    c = cross_attn(q2, enc_k, enc_v, kv_lens=enc_lens)

The checks and the calls are in flash_attn/stored_attn.cpp.  Every tensor is on one CUDA device; calls run on torch's
current stream of that device or on `stream`.  With `stream`, outputs and workspaces come from that stream's memory pool;
ordering the inputs before it and the outputs after it is the caller's.  All calls can be captured into a CUDA graph.
"""
from __future__ import annotations

import torch

from .binding import load_stored_attn_binding

_ext = None


def _binding():
    global _ext
    if _ext is None:
        _ext = load_stored_attn_binding()
    return _ext


def _stream(stream: torch.cuda.Stream | None):
    return None if stream is None else (stream.stream_id, stream.device_index)


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
    sequences of one call or stand twice in one.  Lengths or pages out of range leave their sequence unwritten and are raised by
    check_status()."""
    _binding().kv_cache_write(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens, _stream(stream))


def cache_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
               block_table: torch.Tensor, seq_lens: torch.Tensor, *, new_lens: torch.Tensor | None = None,
               scale: float | None = None, out: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Attention of each sequence's newest tokens over the cache of kv_cache_write (b200_cache_attn).

    q: bf16 [batch, q_len, heads, 128], heads a multiple of kv_heads (query head h reads key/value head
    h // (heads // kv_heads)).  seq_lens: lengths with the new tokens, which are already in the cache; new_lens: how many
    of q's tokens a sequence has (default: q_len).  Query t is at place seq_lens - new_lens + t and attends to the places
    up to its own.  Rows past new_lens and rows that see nothing are 0.  scale defaults to 128 ** -0.5.  out, if given, is shaped like q
    and does not share q's memory."""
    return _binding().cache_attn(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens, scale, out,
                                 _stream(stream))


def cross_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, kv_lens: torch.Tensor | None = None,
               scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False,
               stream: torch.cuda.Stream | None = None):
    """Cross attention softmax(scale q k^T) v to an encoder's states of another length (b200_cross_attn_bf16).

    q: bf16 [batch, q_len, heads, 128]; k, v: bf16 [batch, kv_len, kv_heads, 128], heads a multiple of kv_heads; any strides
    that keep the last dimension contiguous (a fused projection's views, [batch, heads, tokens, 128] storage).  kv_lens:
    int32 [batch], keys of each entry (default: kv_len); what lies behind them is not used.  An entry without keys gives 0.
    return_lse=True returns (out, lse) with lse float32 [batch, heads, q_len], the natural log of the softmax denominator
    (-inf without keys), which cross_attn_backward takes.  scale defaults to 128 ** -0.5.  out, if given, is shaped like q
    and shares no memory with the inputs."""
    o, lse = _binding().cross_attn(q, k, v, kv_lens, scale, out, return_lse, _stream(stream))
    return (o, lse) if return_lse else o


def cross_attn_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                        lse: torch.Tensor, *, kv_lens: torch.Tensor | None = None, scale: float | None = None,
                        stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv) of cross_attn (b200_cross_attn_bwd_bf16), bf16, shaped like q, k and v.

    out and lse are what cross_attn(..., return_lse=True) gave for the same q, k, v, kv_lens and scale; dout is the gradient
    of out.  dk and dv are summed over the query heads of a group and 0 behind an entry's keys.  The sums run in a fixed
    order: equal inputs give equal bits."""
    return _binding().cross_attn_backward(dout, q, k, v, out, lse, kv_lens, scale, _stream(stream))
