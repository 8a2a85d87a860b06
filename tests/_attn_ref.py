"""64-bit references of attention to stored keys and values, on the CPU, and the
error bounds the tests hold the kernels to.

Rounding to a type is off by at most finfo(type).eps / 2 of the value: 2^-8 for
bf16, 2^-11 for fp16, 2^-4 for e4m3.  Bounds, with A = sum_j p_j |v_j|:
  * P is rounded once (bf16, or fp16 over the 8-bit cache) before the product
    with V and the denominator is not: 2^-8 A or 2^-11 A;
  * scores are fp32 sums of 128 exact products, off by at most
    128 * 2^-24 * sum |q_d k_d| * scale, and P by that relative share; exp2 and
    the sums over keys add less than 2^-18.  Their sum E, from the row's
    largest sum |q_d k_d|: E A;
  * the output is rounded once: 2^-8 |o|."""
from __future__ import annotations

import math

import torch

def attend(q, k, v, seen, scale):
    """One head in 64 bits: q [t, 128], k, v [n, 128], seen [t, n].  (o, lse, p, a = p |v|, E [t, 1])."""
    t, n = q.shape[0], k.shape[0]
    if n == 0 or t == 0:
        z = torch.zeros(t, 128, dtype=torch.float64)
        return z, torch.full((t,), -math.inf, dtype=torch.float64), torch.zeros(t, n, dtype=torch.float64), z.clone(), z[:, :1]
    x = (q.double() @ k.double().T) * scale
    most = torch.where(seen, q.double().abs() @ k.double().abs().T, 0.0).amax(1, keepdim=True) * scale
    err = 2.0 ** -17 * most + 2.0 ** -18
    x = torch.where(seen, x, -math.inf)
    lse = torch.logsumexp(x, 1)
    p = torch.exp(x - torch.where(lse == -math.inf, 0.0, lse).unsqueeze(1))
    return p @ v.double(), lse, p, p @ v.double().abs(), err


def cache_values(codes, scale, table, n, head):
    """The first n places of one sequence and head of the cache, in 64 bits."""
    page = codes.shape[2]
    pages = table[:-(-n // page)].long()
    x = codes[pages, head].double() * scale[pages, head].double().view(-1, 1, 1)
    return x.reshape(-1, 128)[:n]


def cache_attn(q, k_cache, v_cache, k_scale, v_scale, table, seq_lens, new_lens=None, scale=128 ** -0.5):
    """(output, bound) of cache_attn, [batch, q_len, heads, 128] in 64 bits."""
    b, t, h, _ = q.shape
    kv = k_cache.shape[1]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for i in range(b):
        n = int(seq_lens[i])
        m = t if new_lens is None else int(new_lens[i])
        place = torch.arange(n - m, n)
        for j in range(kv):
            k, v = (cache_values(c, s, table[i], n, j) for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
            seen = torch.arange(n).view(1, n) <= place.view(m, 1)
            for e in range(j * (h // kv), (j + 1) * (h // kv)):
                o, _, _, a, err = attend(q[i, :m, e], k, v, seen, scale)
                out[i, :m, e] = o
                bound[i, :m, e] = (2.0 ** -11 + err) * a + 2.0 ** -8 * o.abs()
    return out, bound


def cross_attn(q, k, v, kv_lens=None, scale=128 ** -0.5, dout=None):
    """Output, log-sum-exp, gradients (with dout) in 64 bits, and their bounds: {name: (value, bound)}."""
    b, t, h, _ = q.shape
    n, kv = k.shape[1:3]
    def z(*s):
        return torch.zeros(*s, dtype=torch.float64)
    r = {"out": (z(b, t, h, 128), z(b, t, h, 128)), "lse": (torch.full((b, h, t), -math.inf, dtype=torch.float64), z(b, h, t))}
    if dout is not None:
        r |= {"dq": (z(b, t, h, 128), z(b, t, h, 128)), "dk": (z(*k.shape), z(*k.shape)), "dv": (z(*k.shape), z(*k.shape))}
    for i in range(b):
        m = n if kv_lens is None else min(max(int(kv_lens[i]), 0), n)
        for e in range(h):
            j = e // (h // kv)
            qh, kh, vh = q[i, :, e].double(), k[i, :m, j].double(), v[i, :m, j].double()
            o, lse, p, a, err = attend(qh, kh, vh, torch.ones(t, m, dtype=torch.bool), scale)
            o_bound = (2.0 ** -8 + err) * a + 2.0 ** -8 * o.abs()
            r["out"][0][i, :, e], r["out"][1][i, :, e] = o, o_bound
            r["lse"][0][i, e], r["lse"][1][i, e] = lse, err[:, 0] + 2.0 ** -20 * lse.abs().nan_to_num(posinf=0.0)
            if dout is None or m == 0:
                continue
            # P = exp(x - lse) anew: off by E from the scores and E from
            # the stored lse.  delta = sum_d dO O takes the rounded O.  dS is
            # rounded once, as P is for dV; each sum is fp32 (2^-12 covers
            # up to 4096 terms' 2^-24 each); each gradient is rounded once.
            do = dout[i, :, e].double()
            dp, delta = do @ vh.T, (do * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            d_delta = (do.abs() * o_bound).sum(1, keepdim=True)
            d_dp = 2.0 ** -17 * (do.abs() @ vh.abs().T)  # 128 products in fp32
            ds_bound = 2.0 ** -8 * ds.abs() + 2 * err * ds.abs() + p * (d_delta + d_dp) * (1 + 2 * err)
            p_bound = (2.0 ** -8 + 2 * err) * p
            tail = 2.0 ** -12
            dq, dk, dv = scale * ds @ kh, scale * ds.T @ qh, p.T @ do
            r["dq"][0][i, :, e] = dq
            r["dq"][1][i, :, e] = scale * (ds_bound + tail * ds.abs()) @ kh.abs()
            r["dk"][0][i, :m, j] += dk
            r["dk"][1][i, :m, j] += scale * (ds_bound + tail * ds.abs()).T @ qh.abs()
            r["dv"][0][i, :m, j] += dv
            r["dv"][1][i, :m, j] += (p_bound + tail * p).T @ do.abs()
    for name in ("dq", "dk", "dv") if dout is not None else ():
        r[name][1].add_(2.0 ** -8 * r[name][0].abs())
    return r


def power_scale(amax: float) -> float:
    """The smallest power of two >= 2^-100 with amax <= 448 s."""
    s = 2.0 ** -100
    while amax > 448.0 * s:
        s *= 2.0
    return s


def cache_write(k, v, k_cache, v_cache, k_scale, v_scale, table, seq_lens, new_lens=None):
    """kv_cache_write page by page, on copies: (k_cache, v_cache, k_scale, v_scale).  Exact: all values are powers of
    two times bf16 numbers, so the kernel has to give the same codes and scales."""
    outs = []
    for x, codes, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        codes, scale = codes.clone(), scale.clone()
        page = codes.shape[2]
        for b in range(x.shape[0]):
            n = int(seq_lens[b])
            m = x.shape[1] if new_lens is None else int(new_lens[b])
            at = n - m
            while at < n:
                stop = min(n, (at // page + 1) * page)
                p, lo = int(table[b, at // page]), at % page
                for h in range(x.shape[2]):
                    vals = x[b, at - (n - m):stop - (n - m), h].double()
                    fin = vals[~vals.isnan()].abs()
                    # An infinity counts as bf16's largest value.
                    s = power_scale(min(float(fin.max()), torch.finfo(torch.bfloat16).max) if fin.numel() else 0.0)
                    if lo:
                        s = max(s, float(scale[p, h]))
                        if s != float(scale[p, h]):
                            old = codes[p, h, :lo].double() * (float(scale[p, h]) / s)
                            codes[p, h, :lo] = old.float().to(torch.float8_e4m3fn)
                    codes[p, h, lo:lo + stop - at] = (vals / s).clamp(-448.0, 448.0).float().to(torch.float8_e4m3fn)
                    scale[p, h] = s
                at = stop
        outs.append((codes, scale))
    return outs[0][0], outs[1][0], outs[0][1], outs[1][1]
