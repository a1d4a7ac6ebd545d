"""Attention and the 4-bit cache in 64 bits, from their formulas, with bounds of
what the kernels' roundings can add up to."""
from __future__ import annotations

import numpy as np
import torch

EPS16 = 2.0 ** -11  # half a step of fp16, relative to the value
EPS32 = 2.0 ** -24


def randn(shape, seed, device, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(torch.float16).to(device)


def softmax_pv(s, v, vabs=None, serr=0.0):
    """(out, bound) of softmax(s) @ v for one head, s [rows, keys] in 64 bits with
    -inf at masked places, v [keys, dim]; vabs: |what a probability is multiplied
    by as fp16|, where that is not v itself; serr: error bound of s.

    Bound, relative to the row's maximum (p <= 1, l = sum p >= 1): each p (times a
    scale) is rounded to fp16 once: EPS16 of it, or half of fp16's least step
    (2^-25 where the largest scale is brought to 1 or more) where it is subnormal;
    each p is off by exp(2 serr) - 1 and by the fp32 exponential and sums (a few
    EPS32 per key of a running sum: 2^-18 covers the lengths tested); the result is
    rounded to fp16 once, whose least step is 2^-24."""
    vabs = v.abs() if vabs is None else vabs
    m = s.amax(dim=1, keepdim=True).clamp(min=-1e300)
    p = torch.exp(s - m)
    l = p.sum(dim=1, keepdim=True).clamp(min=1e-300)
    out = (p @ v) / l
    visible = torch.isfinite(s).to(torch.float64)
    bound = (EPS16 * (p @ vabs) + 2.0 ** -25 * vabs.max() * visible.sum(1, keepdim=True)) / l
    bound += (2.1 * serr + 2.0 ** -18) * ((p @ (v.abs() + vabs)) / l)
    return out, bound + EPS16 * (out.abs() + bound) + 2.0 ** -25


def score_error(q, k, scale):
    """Bound of the fp32 score's error over one head's rows: fp16 products are exact
    in fp32, their sum and the scalings are off by EPS32 a step."""
    mag = (q.abs() @ k.abs().t()).max() * scale
    return float(mag) * (q.shape[1] + 8) * EPS32


def attention(q, k, v, spans, scale):
    """out, bound [tokens, heads, dim] and the rows that are written, of packed causal
    attention over spans = [(begin, end), ...]."""
    q, k, v = (t.to(torch.float64) for t in (q, k, v))
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    rows = torch.zeros(q.shape[0], dtype=torch.bool, device=q.device)
    per = q.shape[1] // k.shape[1]
    for b, e in spans:
        if e <= b:
            continue
        rows[b:e] = True
        later = torch.ones((e - b, e - b), dtype=torch.bool, device=q.device).triu(1)
        for h in range(q.shape[1]):
            kk, vv = k[b:e, h // per], v[b:e, h // per]
            s = (q[b:e, h] @ kk.t() * scale).masked_fill(later, -torch.inf)
            out[b:e, h], bound[b:e, h] = softmax_pv(s, vv, None,
                                                    score_error(q[b:e, h], kk, scale))
    return out, bound, rows


def quantize4(x, group):
    """(codes uint8, scale, offset) of fp16 numpy x [.., dim], fp32 arithmetic step by step."""
    x = x.astype(np.float32).reshape(*x.shape[:-1], -1, group)
    low, high = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        scale = ((high - low) / np.float32(15)).astype(np.float16)
        s = scale.astype(np.float32)
        offset = (low + np.float32(8) * s).astype(np.float16)
        n = np.rint((x - offset.astype(np.float32)) / s) + np.float32(8)
        n = np.where(s > 0, np.clip(n, 0, 15), 8).astype(np.uint8)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    scale[bad] = offset[bad] = np.nan
    return np.where(bad, 8, n).reshape(*x.shape[:-2], -1), scale[..., 0], offset[..., 0]


def pack4(codes, keys):
    """Bytes of rows of codes [.., dim] in the cache's order."""
    if keys:
        d = codes.shape[-1]
        order = [32 * j + 8 * g + i for g in range(4) for j in range(d // 32) for i in range(8)]
        codes = codes[..., order]
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def cache_values(cache, keys):
    """(values, |scale * (code - 8)|) fp64 [pages, kv_heads, page_size, dim] of a cache."""
    codes = (cache.k_codes if keys else cache.v_codes).to(torch.int64)
    scales = (cache.k_scales if keys else cache.v_scales).to(torch.float64)
    n = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    d = n.shape[-1]
    if keys:
        place = torch.empty(d, dtype=torch.int64)
        for at, ch in enumerate(32 * j + 8 * g + i for g in range(4) for j in range(d // 32)
                                for i in range(8)):
            place[ch] = at
        n = n[..., place.to(n.device)]
    of = torch.arange(d, device=n.device) // cache.group
    part = scales[..., of, 0] * (n - 8)
    return scales[..., of, 1] + part, part.abs()


def attention_kv4(q, cache, table, lens, scale):
    """out, bound [seqs, heads, dim] of one token per sequence over the cache."""
    k, kpart = cache_values(cache, True)
    v, vpart = cache_values(cache, False)
    q = q.to(torch.float64)
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    per, size = q.shape[1] // cache.kv_heads, cache.page_size
    for i in range(q.shape[0]):
        n = max(0, min(int(lens[i]), table.shape[1] * size))
        t = torch.arange(n, device=q.device)
        page = table[i].to(torch.int64)[t // size]
        ok = (page >= 0) & (page < cache.pages)
        page, t = page[ok], t[ok]
        if page.numel() == 0:
            continue
        for h in range(cache.kv_heads):
            kk, vv, vp = k[page, h, t % size], v[page, h, t % size], vpart[page, h, t % size]
            qq = q[i, h * per: (h + 1) * per]
            # the score is summed as codes times scale plus offset times the query's sum
            mag = kk.abs() + 2 * kpart[page, h, t % size]
            o, b = softmax_pv(qq @ kk.t() * scale, vv, vp, score_error(qq, mag, scale) * 2)
            out[i, h * per: (h + 1) * per], bound[i, h * per: (h + 1) * per] = o, b
    return out, bound


def assert_within(got, out, bound, what=""):
    """|got - out| <= bound everywhere, and got finite."""
    got = got.to(torch.float64)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - out).abs() - bound
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, (f"{what}: {int((over > 0).sum())} of {over.numel()} values past their "
                        f"bound, the worst by {worst}")
