"""The paged 4-bit cache in service, from its definitions: pages and slots in whole numbers,
page keys and scores in 64 bits (exact), attention of chunks in 64 bits with a bound of what
the kernel's roundings can add up to."""
from __future__ import annotations

import numpy as np
import torch

from attention_ref import EPS16, EPS32, cache_values, softmax_pv

SUB16 = 2.0 ** -24  # fp16's least step


def ceil_div(a, b):
    return -(-a // b)


def extend(new, lens, table, free, count, page, tokens):
    """slots, starts, lens, count, table (lists) of kv4_extend."""
    most = len(table[0]) * page if table else 0
    table = [list(r) for r in table]
    count = max(0, min(count, len(free)))
    slots, starts, after = [-1] * tokens, [0], []
    at = wanted = taken = 0
    for i, (m, n) in enumerate(zip(new, lens)):
        m, n = max(m, 0), max(0, min(n, most))
        begin, at = at, at + m
        starts.append(min(at, tokens))
        fits = at <= tokens and n + m <= most
        need = ceil_div(n + m, page) - ceil_div(n, page) if fits else 0
        first, wanted = wanted, wanted + need
        if not fits or (need and wanted > count):
            after.append(n)
            continue
        for f in range(need):
            table[i][ceil_div(n, page) + f] = free[count - 1 - first - f]
            taken = first + f + 1
        for j in range(m):
            p = table[i][(n + j) // page]
            slots[begin + j] = p * page + (n + j) % page if p >= 0 else -1
        after.append(n + m)
    return slots, starts, after, count - taken, table


def trim(keep, lens, table, free, count, page):
    """lens, count, free (lists) of kv4_trim."""
    most = len(table[0]) * page if table else 0
    free, gone, after = list(free), [], []
    count = max(0, min(count, len(free)))
    for i, (m, n) in enumerate(zip(keep, lens)):
        n = max(0, min(n, most))
        m = min(max(m, 0), n)
        gone += table[i][ceil_div(m, page): ceil_div(n, page)]
        after.append(m)
    for f, p in enumerate(gone[::-1]):
        if count + f < len(free):
            free[count + f] = p
    return after, min(count + len(gone), len(free)), free


def codes8(x):
    """(codes, scale) of numpy fp64 x [n, dim]: the least power of two with codes in +-127."""
    ok = np.isfinite(x).all(1)
    top = np.abs(np.where(ok[:, None], x, 0)).max(1)
    scale = np.zeros_like(top)
    for i in range(len(top)):
        if ok[i] and top[i] > 0:
            e = -100
            while 127 * 2.0 ** e < top[i]:
                e += 1
            scale[i] = 2.0 ** e
    with np.errstate(all="ignore"):
        codes = np.rint(x / scale[:, None])
    codes = np.where((scale > 0)[:, None], codes, 0)
    return codes, np.where(ok, scale, np.nan)


def page_key(cache, page, count):
    """(codes [kv_heads, dim], scale [kv_heads]) of a page's first `count` tokens."""
    sub = type(cache)(*(t[page: page + 1] for t in (cache.k_codes, cache.v_codes, cache.k_scales,
                                                    cache.v_scales)))
    k = cache_values(sub, True)[0][0, :, :count]
    return codes8((k.sum(dim=1) / count).cpu().numpy())


def select(q, codes, scales, table, lens, keep, page, pages):
    """(chosen [seqs][kv_heads][keep], lens) of kv4_select; q fp16 tensor, codes and scales
    numpy, the rest lists."""
    kv_heads = codes.shape[1]
    per = q.shape[1] // kv_heads
    qq = q.cpu().numpy().astype(np.float64)
    chosen, left = [], []
    for i, n in enumerate(lens):
        n = max(0, min(n, len(table[i]) * page))
        have = ceil_div(n, page)
        left.append(n if have <= keep else n - (have - keep) * page)
        rows = []
        for h in range(kv_heads):
            cols = list(range(have))
            if have > keep:
                with np.errstate(all="ignore"):
                    code, scale = codes8(qq[i, h * per: (h + 1) * per].sum(0)[None])
                if np.isnan(scale[0]):
                    code = code * 0
                score = []
                for c in range(have - 1):
                    p = table[i][c]
                    s = -np.inf if not 0 <= p < pages else \
                        float((codes[p, h].astype(np.float64) * code[0]).sum() * scales[p, h])
                    score.append(-np.inf if np.isnan(s) else s)
                cols = sorted(sorted(range(have - 1), key=lambda c: (-score[c], c))[: keep - 1])
                cols.append(have - 1)
            rows.append([table[i][c] for c in cols] + [-1] * (keep - len(cols)))
        chosen.append(rows)
    return chosen, left


def chunks(q, cache, table, lens, starts, scale):
    """out, bound [tokens, heads, dim] and the rows that are written.

    Keys and values enter as fp16 halves of the cache's values x = o + s (n - 8): rounded
    once, EPS16 |x|, or where the half is subnormal half of fp16's least step, SUB16 of x;
    halving a subnormal scale or offset is off by as much, the scale's times up to 8."""
    k, _ = cache_values(cache, True)
    v, _ = cache_values(cache, False)
    q = q.to(torch.float64)
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    rows = torch.zeros(q.shape[0], dtype=torch.bool, device=q.device)
    per, size = q.shape[1] // cache.kv_heads, cache.page_size
    lost = lambda x: EPS16 * x.abs() + 10 * SUB16  # noqa: E731
    for i, n in enumerate(lens):
        n = max(0, min(n, table.shape[1] * size))
        b, e = starts[i], starts[i + 1]
        if e <= b:
            continue
        rows[b:e] = True
        t = torch.arange(n, device=q.device)
        page = table[i].to(torch.int64)[t // size]
        ok = (page >= 0) & (page < cache.pages)
        page, t = page[ok], t[ok]
        see = t[None, :] <= n - (e - b) + torch.arange(e - b, device=q.device)[:, None]
        if page.numel() == 0:
            continue
        for h in range(cache.kv_heads):
            kk, vv = k[page, h, t % size], v[page, h, t % size]
            for g in range(h * per, (h + 1) * per):
                qq = q[b:e, g]
                s = (qq @ kk.t() * scale).masked_fill(~see, -torch.inf)
                mag = qq.abs() @ kk.abs().t() * scale
                serr = qq.abs() @ lost(kk).t() * scale + mag * (q.shape[2] + 8) * EPS32
                serr = float(serr.masked_fill(~see, 0).max())
                o, bd = softmax_pv(s, vv, None, serr)
                m = s.amax(dim=1, keepdim=True).clamp(min=-1e300)
                p = torch.exp(s - m)
                bd = bd + p @ lost(vv) / p.sum(1, keepdim=True).clamp(min=1e-300) * 1.001
                out[b:e, g], bound[b:e, g] = o, bd
    return out, bound, rows
