"""Attention to stored keys and values: what is timed of it, in plain torch and through this library.

Four operators, as a decoder with a key/value cache and an encoder's states uses them:

  write  kv_cache_write: new keys and values into a paged e4m3 cache, one scale per (page, key/value head)
  cache  cache_attn: attention of the newest tokens over that cache
  cross  cross_attn: attention to an encoder's bf16 states of another length, one token to long prompts
  train  cross_attn and cross_attn_backward: output and gradients of the same

The scale of a page and head is the smallest power of two (2^-100 at least) that brings every value of the page within
e4m3's 448.  It only grows while a page fills, and codes already in the page are rounded again to the new scale; a page
whose first slot is written starts afresh.
"""
import math
import os
import sys

import torch

own = False

D = 128  # head dimension


def _ops():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-kernels_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import b200_gemm
    return b200_gemm


def listed():
    return [
        # A serving step of 48 requests: each appends one token.
        {"name": "write-step", "op": "write", "batch": 48, "new": 1, "new_min": 1, "kv_heads": 8, "page": 32,
         "len_min": 17, "len": 4000},
        # Six ragged prompts of a padded batch enter the cache.
        {"name": "write-prompts", "op": "write", "batch": 6, "new": 2500, "new_min": 700, "kv_heads": 8, "page": 64,
         "len_min": 2500, "len": 2600},
        # One user's next token: latency.
        {"name": "cache-one", "op": "cache", "batch": 1, "q": 1, "heads": 32, "kv_heads": 8, "page": 64,
         "len_min": 1000, "len": 1000},
        # A full serving batch with contexts of every length.
        {"name": "cache-batch", "op": "cache", "batch": 64, "q": 1, "heads": 32, "kv_heads": 8, "page": 64,
         "len_min": 100, "len": 8192},
        # Two long documents: few rows, a long axis.
        {"name": "cache-long", "op": "cache", "batch": 2, "q": 1, "heads": 64, "kv_heads": 8, "page": 128,
         "len_min": 100001, "len": 131072},
        # Five drafted tokens are verified at once, a key/value head per query head, small pages.
        {"name": "cache-verify", "op": "cache", "batch": 24, "q": 5, "heads": 16, "kv_heads": 16, "page": 16,
         "len_min": 5, "len": 2999},
        # One translation's next token: latency.
        {"name": "cross-one", "op": "cross", "batch": 1, "q": 1, "heads": 16, "kv_heads": 16, "len_min": 777, "len": 777},
        # The decoder step of 32 requests over sources of every length.
        {"name": "cross-step", "op": "cross", "batch": 32, "q": 1, "heads": 16, "kv_heads": 16, "len_min": 200,
         "len": 2000},
        # Prompts of a padded batch against padded sources.
        {"name": "cross-prompt", "op": "cross", "batch": 8, "q": 333, "heads": 16, "kv_heads": 16, "len_min": 600,
         "len": 1500},
        # Long documents on both sides, grouped heads.
        {"name": "cross-long", "op": "cross", "batch": 2, "q": 4096, "heads": 32, "kv_heads": 8, "len_min": 7001,
         "len": 8192},
        # A training step of sentence pairs, one of them with an empty source.
        {"name": "train-pairs", "op": "train", "batch": 8, "q": 500, "heads": 16, "kv_heads": 16, "len_min": 0,
         "len": 1333},
        # A training step of a long pair, grouped heads.
        {"name": "train-long", "op": "train", "batch": 1, "q": 4096, "heads": 32, "kv_heads": 8, "len_min": 4096,
         "len": 4096},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["write", "cache", "cross", "train"])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8] if kv_heads <= 4 else [1, 2, 4])
    if op == "write":
        new = rng.choice([1, 1, log(2, 2500)])
        batch = log(1, max(1, min(128, 16000 // new)))
        last = log(new, max(new, min(16000, 200000 // batch)))
        return {"op": op, "batch": batch, "new": new, "new_min": rng.randint(1, new), "kv_heads": kv_heads,
                "page": rng.choice([16, 32, 64, 128]), "len_min": rng.randint(new, last), "len": last}
    if op == "cache":
        batch = log(1, 96)
        last = log(8, min(131072, 400000 // batch))
        return {"op": op, "batch": batch, "q": rng.choice([1, 1, 1, log(2, 8)]), "heads": heads, "kv_heads": kv_heads,
                "page": rng.choice([16, 32, 64, 128]), "len_min": rng.randint(8, last), "len": last}
    if op == "cross" and rng.random() < 0.4:
        batch = log(1, 64)
        last = log(1, 4000)
        return {"op": op, "batch": batch, "q": 1, "heads": heads, "kv_heads": kv_heads, "len_min": rng.randint(0, last),
                "len": last}
    batch = log(1, 8)
    q = log(2, 4096)
    last = log(1, max(1, min(8192, (1 << 28) // (batch * heads * q))))
    return {"op": op, "batch": batch, "q": q, "heads": heads, "kv_heads": kv_heads, "len_min": rng.randint(0, last),
            "len": last}


def _spread(n, lo, hi):
    """n lengths from hi down to lo, evenly."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def work(case):
    b, kv = case["batch"], case["kv_heads"]
    if case["op"] == "write":
        new = _spread(b, case["new_min"], case["new"])
        pages = sum(-(-n // case["page"]) for n in new)
        # k and v read in bf16, written in 8 bits; a scale for each page begun.
        return {"bytes": 2.0 * (sum(new) * kv * D * 3 + pages * kv * 4), "flops": 4.0 * sum(new) * kv * D}
    lens = _spread(b, case["len_min"], case["len"])
    rows = b * case["q"] * case["heads"]
    if case["op"] == "cache":
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2.0 * (sum(lens) * kv * D + pages * kv * 4) + 4.0 * pages + 4.0 * rows * D,
                "flops": 4.0 * sum(lens) * case["q"] * case["heads"] * D}
    scores = float(sum(lens)) * case["q"] * case["heads"]
    if case["op"] == "cross":
        return {"bytes": 4.0 * sum(lens) * kv * D + 4.0 * rows * D + 4.0 * rows, "flops": 4.0 * scores * D}
    # q, k, v, dout read; out, lse, dq, dk, dv written (dk and dv whole, masked places too).
    return {"bytes": 4.0 * sum(lens) * kv * D + 4.0 * b * case["len"] * kv * D + 8.0 * rows * D + 4.0 * rows,
            "flops": 14.0 * scores * D}


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _keys(g, *shape):
    """Keys with a few strong channels per head, as trained projections have them."""
    gain = torch.exp(0.5 * _normal(g, 1, 1, shape[2], D))
    return (_normal(g, *shape) * gain).to(torch.bfloat16)


def _shuffled(g, values):
    t = torch.tensor(values, dtype=torch.int32, device="cuda")
    return t[torch.randperm(len(values), generator=g, device="cuda")]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    b, kv = case["batch"], case["kv_heads"]
    if case["op"] in ("cross", "train"):
        q, h, n = case["q"], case["heads"], case["len"]
        state = {"op": case["op"], "q": _normal(g, b, q, h, D).to(torch.bfloat16), "k": _keys(g, b, n, kv, D),
                 "v": _normal(g, b, n, kv, D).to(torch.bfloat16),
                 "lens": _shuffled(g, _spread(b, case["len_min"], n))}
        if case["op"] == "train":
            state["dout"] = (_normal(g, b, q, h, D) * 0.1).to(torch.bfloat16)
        return state
    page = case["page"]
    lens = _shuffled(g, _spread(b, case["len_min"], case["len"]))
    per = -(-case["len"] // page)
    pages = b * per + 3
    # Pages in no order; some belong to nobody.  What nobody wrote holds any bytes, NaN codes among them.
    table = torch.randperm(pages, generator=g, device="cuda")[:b * per].view(b, per).to(torch.int32)
    k_cache, v_cache = (torch.randint(0, 256, (pages, kv, page, D), generator=g, device="cuda", dtype=torch.uint8)
                        .view(torch.float8_e4m3fn) for _ in range(2))
    k_scale, v_scale = (torch.exp2(torch.randint(-9, -4, (pages, kv), generator=g, device="cuda").float())
                        for _ in range(2))
    state = {"op": case["op"], "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale,
             "table": table, "lens": lens}
    # What the cache holds already: values near a page's largest at 1 to 4.
    held = lens
    if case["op"] == "write":
        new = torch.minimum(_shuffled(g, _spread(b, case["new_min"], case["new"])), lens)
        state |= {"new": new, "k": _keys(g, b, case["new"], kv, D), "v": _normal(g, b, case["new"], kv, D).to(torch.bfloat16)}
        held = lens - new
    slot = torch.arange(per * page, device="cuda").view(1, per, 1, page, 1)
    there = slot < held.view(b, 1, 1, 1, 1)
    for cache in (k_cache, v_cache):
        x = (_normal(g, b, per, kv, page, D) * 96.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        raw = cache.view(torch.uint8)
        raw[table.long()] = torch.where(there, x, raw[table.long()])
    if case["op"] == "cache":
        state["q"] = _normal(g, b, case["q"], case["heads"], D).to(torch.bfloat16)
    return state


def _power(amax):
    """The smallest power of two s >= 2^-100 with amax <= 448 s."""
    m, e = torch.frexp(amax)  # amax = m 2^e, 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, -100).clamp(min=-100))


def _write(s):
    page = s["k_cache"].shape[2]
    k = s["k"]
    b, t, kv, _ = k.shape
    new, first = s["new"].long(), (s["lens"] - s["new"]).long()
    # Padding repeats its sequence's last token: it lands where that token does.
    step = torch.minimum(torch.arange(t, device=k.device).view(1, t), new.view(b, 1) - 1)
    pos = first.view(b, 1) + step
    where = torch.gather(s["table"].long(), 1, pos // page)  # page of each token [b, t]
    slot = pos % page
    begun = torch.gather(s["table"].long(), 1, (first // page).view(b, 1)).view(b)  # the page that may hold more
    older = torch.arange(page, device=k.device).view(1, page) < (first % page).view(b, 1)
    for x, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        x = torch.gather(x.float(), 1, step.view(b, t, 1, 1).expand(b, t, kv, D))
        amax = torch.nan_to_num(x.abs(), nan=0.0).amax(3)  # [b, t, kv]
        most = torch.zeros_like(scale).scatter_reduce_(0, where.reshape(-1, 1).expand(-1, kv), amax.view(b * t, kv), "amax")
        base = torch.zeros_like(scale)
        was = scale[begun]
        base[begun] = torch.where((first % page > 0).view(b, 1), was, 0.0)
        now = torch.maximum(base, _power(most))
        scale[where.reshape(-1)] = now[where.reshape(-1)]
        codes = cache.view(torch.uint8)
        held = cache[begun].float() * (was / now[begun]).view(b, kv, 1, 1)
        codes[begun] = torch.where(older.view(b, 1, page, 1), held.to(torch.float8_e4m3fn).view(torch.uint8), codes[begun])
        fresh = (x / now[where].unsqueeze(3)).to(torch.float8_e4m3fn)
        codes[where.reshape(-1), :, slot.reshape(-1)] = fresh.view(torch.uint8).view(b * t, kv, D)
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _attend(q, k, v, seen):
    """q [b, kv, rows, D], k and v [b, kv, n, D] in 32 bits; seen [b, 1, rows or 1, n].  Output, log-sum-exp and P."""
    s = (q @ k.transpose(2, 3)).mul_(D ** -0.5).masked_fill_(~seen, -math.inf)
    top = s.amax(3, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(3, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    return p @ v, (top + total.log()).squeeze(3), p


def _rows(x, kv):
    """[b, t, heads, D] -> [b, kv, group * t, D] in 32 bits."""
    b, t, h, _ = x.shape
    return x.float().view(b, t, kv, h // kv, D).permute(0, 2, 3, 1, 4).reshape(b, kv, h // kv * t, D)


def _unrows(x, t):
    """[b, kv, group * t, ...] -> [b, t, heads, ...]."""
    b, kv, r = x.shape[:3]
    x = x.view(b, kv, r // t, t, *x.shape[3:])
    return x.permute(0, 3, 1, 2, *range(4, x.dim())).reshape(b, t, kv * (r // t), *x.shape[4:])


def _cache(s):
    q, table = s["q"], s["table"].long()
    b, t, h, _ = q.shape
    kv, page = s["k_cache"].shape[1:3]
    n = table.shape[1] * page
    place = torch.arange(n, device=q.device)
    there = place.view(1, n) < s["lens"].view(b, 1)
    k, v = ((c[table].float() * m[table].view(b, -1, kv, 1, 1)).transpose(1, 2).reshape(b, kv, n, D)
            .masked_fill_(~there.view(b, 1, n, 1), 0.0) for c, m in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
    last = s["lens"].view(b, 1) - t + torch.arange(t, device=q.device)  # the place of each query [b, t]
    seen = (place.view(1, 1, n) <= last.view(b, t, 1)).repeat(1, h // kv, 1)
    o, _, _ = _attend(_rows(q, kv), k, v, seen.unsqueeze(1))
    return _unrows(o, t).to(torch.bfloat16)


def _cross(s):
    q, k, v = s["q"], s["k"], s["v"]
    b, t, h, _ = q.shape
    n, kv = k.shape[1:3]
    there = torch.arange(n, device=q.device).view(1, n) < s["lens"].view(b, 1)
    kf, vf = (x.float().transpose(1, 2).masked_fill(~there.view(b, 1, n, 1), 0.0) for x in (k, v))
    qf = _rows(q, kv)
    o, lse, p = _attend(qf, kf, vf, there.view(b, 1, 1, n))
    out, lse = _unrows(o, t).to(torch.bfloat16), _unrows(lse, t).transpose(1, 2).contiguous()
    if s["op"] == "cross":
        return out, lse
    do = _rows(s["dout"], kv)
    dv = p.transpose(2, 3) @ do
    ds = (do @ vf.transpose(2, 3)).sub_((do * o).sum(3, keepdim=True)).mul_(p).mul_(D ** -0.5)
    dq = _unrows(ds @ kf, t)
    dk = ds.transpose(2, 3) @ qf
    return (out, lse, dq.to(torch.bfloat16), dk.transpose(1, 2).contiguous().to(torch.bfloat16),
            dv.transpose(1, 2).contiguous().to(torch.bfloat16))


def run(state):
    s = state
    if own:
        ops = _ops()
        if s["op"] == "write":
            ops.kv_cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lens"],
                               new_lens=s["new"])
            return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
        if s["op"] == "cache":
            return ops.cache_attn(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lens"])
        out, lse = ops.cross_attn(s["q"], s["k"], s["v"], kv_lens=s["lens"], return_lse=True)
        if s["op"] == "cross":
            return out, lse
        return out, lse, *ops.cross_attn_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, kv_lens=s["lens"])
    return {"write": _write, "cache": _cache, "cross": _cross, "train": _cross}[s["op"]](s)


def _exact_write(s):
    """Token by token of the definition, a page at a time, in 64 bits."""
    page = s["k_cache"].shape[2]
    lens, new, table = s["lens"].tolist(), s["new"].tolist(), s["table"].tolist()
    outs = []
    for x, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        codes, scales = cache.double(), scale.double()
        for b, (n, m) in enumerate(zip(lens, new)):
            at = n - m
            while at < n:
                stop = min(n, (at // page + 1) * page)
                p, lo = table[b][at // page], at % page
                vals = x[b, at - (n - m):stop - (n - m)].double().transpose(0, 1)  # [kv, tokens, D]
                top = vals.abs().nan_to_num(nan=0.0).amax((1, 2))
                need = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp(min=-100.0))
                need = torch.where(need * 224.0 >= top, need / 2, need)  # log2 next to a border
                need = torch.where(need * 448.0 < top, need * 2, need).clamp(min=2.0 ** -100)
                grown = torch.maximum(need, scales[p]) if lo else need
                if lo:
                    codes[p, :, :lo] = (codes[p, :, :lo] * (scales[p] / grown).view(-1, 1, 1)).to(torch.float8_e4m3fn).double()
                codes[p, :, lo:lo + stop - at] = (vals / grown.view(-1, 1, 1)).to(torch.float8_e4m3fn).double()
                scales[p] = grown
                at = stop
        outs.append((codes, scales))
    return outs[0][0], outs[1][0], outs[0][1], outs[1][1]


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "write":
        return _exact_write(s) if sum(s["new"].tolist()) // case["page"] + case["batch"] < 4000 else None
    q = s["q"]
    b, t, h, _ = q.shape
    train, lens = s["op"] == "train", s["lens"].tolist()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((b, h, t), -math.inf, dtype=torch.float64, device=q.device)
    kv = case["kv_heads"]
    if train:
        dq = torch.zeros_like(out)
        dk, dv = (torch.zeros(s["k"].shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for i in range(b):
        n = lens[i]
        if n == 0:
            continue
        for j in range(kv):
            if s["op"] == "cache":
                pages = s["table"][i, :-(-n // case["page"])].long()
                k, v = ((c[pages, j].double() * m[pages, j].double().view(-1, 1, 1)).reshape(-1, D)[:n]
                        for c, m in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
            else:
                k, v = s["k"][i, :n, j].double(), s["v"][i, :n, j].double()
            for e in range(j * (h // kv), (j + 1) * (h // kv)):
                x = torch.einsum("td,nd->tn", q[i, :, e].double(), k) / math.sqrt(D)
                if s["op"] == "cache":
                    x[torch.arange(n, device=q.device) > torch.arange(n - t, n, device=q.device).view(t, 1)] = -math.inf
                lse[i, e] = torch.logsumexp(x, 1)
                p = torch.exp(x - lse[i, e].view(t, 1))
                o = torch.einsum("tn,nd->td", p, v)
                out[i, :, e] = o
                if train:
                    do = s["dout"][i, :, e].double()
                    dp = torch.einsum("td,nd->tn", do, v)
                    dx = p * (dp - torch.einsum("td,td->t", do, o).view(t, 1)) / math.sqrt(D)
                    dq[i, :, e] = torch.einsum("tn,nd->td", dx, k)
                    dk[i, :n, j] += torch.einsum("tn,td->nd", dx, q[i, :, e].double())
                    dv[i, :n, j] += torch.einsum("tn,td->nd", p, do)
    if s["op"] == "cache":
        return out
    return (out, lse, dq, dk, dv) if train else (out, lse)
