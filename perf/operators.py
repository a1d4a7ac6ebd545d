"""The operators between a decoder layer's linear layers, and the work a program gives them.

  attention      causal attention of whole prompts, several sequences of any
                 lengths packed into one row matrix, grouped heads
  kv4            keys and values written into a paged cache of 4-bit codes and
                 read back
  attention_kv4  attention of one new token per sequence over that cache
  experts        a mixture-of-experts layer for the few tokens of a decode step

Where `own` is false, run() computes them from their formulas with elementary
torch operations in 32 bits; where it is true, it makes the package's calls.
Inputs have the distributions the path meets: N(0, 1) activations with 0.5% of
the channels 20 times larger, int8 weights over the whole range, queries whose
scores spread over a few units, keys with a few large channels.

  listed()             the named cases
  draw(rng)            another case of the same ranges
  prepare(case, seed)  what a program holds before the call
  run(state)           one pass
  work(case)           bytes and operations the pass cannot do without
  exact(case, seed)    the outputs in 64 bits from the definitions
"""
from __future__ import annotations

import math

import torch

own = False

QMAX = 127.0


def listed():
    return [
        # A long prompt alone: the head counts of an 8B model's layer.  Matrix
        # rate is what counts.
        dict(name="prompt_8192", kind="attention", lens="8192", heads=32, kv_heads=8, dim=128),
        # A batch of prompts as a server packs them: lengths from one token to
        # a few thousand, none of them whole tiles.
        dict(name="prompts_ragged", kind="attention", lens="1,2047,333,17,640,1001", heads=32,
             kv_heads=8, dim=128),
        # Equal short prompts of a small model: one key head per query head,
        # heads of 64.
        dict(name="prompts_8x512_dim64", kind="attention", lens="512,512,512,512,512,512,512,512",
             heads=16, kv_heads=16, dim=64),
        # The shortest ordinary prompt: launch latency.
        dict(name="prompt_61", kind="attention", lens="61", heads=32, kv_heads=8, dim=128),
        # A prompt's keys and values going into the cache.
        dict(name="kv4_prompt_8192", kind="kv4", tokens=8192, kv_heads=8, dim=128, page=64,
             group=32, pages=256),
        # The new tokens of a decode batch going into the cache: latency.
        dict(name="kv4_24_tokens", kind="kv4", tokens=24, kv_heads=8, dim=128, page=16, group=128,
             pages=256),
        # One sequence with a short context: latency.
        dict(name="decode_1x777", kind="attention_kv4", lens="777", heads=32, kv_heads=8, dim=128,
             page=16, group=64),
        # One sequence with a very long context: all the chip on one row.
        dict(name="decode_1x131072", kind="attention_kv4", lens="131072", heads=32, kv_heads=8,
             dim=128, page=64, group=32),
        # A batch with contexts of every length, the head counts of a 70B model.
        dict(name="decode_48_ragged", kind="attention_kv4",
             lens=",".join(str(1 + (i * 4211 + 977) % 8192) for i in range(48)), heads=64,
             kv_heads=8, dim=128, page=64, group=32),
        # One token through a layer of 8 large experts: two experts' weights.
        dict(name="experts_1_of_8", kind="experts", tokens=1, hidden=4096, inter=14336, experts=8,
             topk=2),
        # A decode batch through the same layer: every expert's weights.
        dict(name="experts_16_of_8", kind="experts", tokens=16, hidden=4096, inter=14336, experts=8,
             topk=2),
        # A few tokens through many small experts: latency and many short tiles.
        dict(name="experts_5_of_64", kind="experts", tokens=5, hidden=2048, inter=1408, experts=64,
             topk=6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# (query heads, key heads, width of a head)
_HEADS = [(32, 8, 128), (64, 8, 128), (16, 16, 64), (32, 32, 128), (8, 1, 128), (12, 4, 64),
          (40, 8, 128)]
# expert layers: (experts, topk, hidden, inter)
_EXPERT_LAYERS = [(8, 2, 4096, 14336), (64, 6, 7168, 2048), (64, 6, 2048, 1408), (16, 2, 4096, 6400)]


def draw(rng):
    kind = rng.choice(["attention", "attention", "kv4", "attention_kv4", "attention_kv4",
                       "experts", "experts"])
    if kind == "experts":
        e, t, h, i = rng.choice(_EXPERT_LAYERS)
        return dict(kind=kind, tokens=rng.randint(1, 16), hidden=h, inter=i, experts=e, topk=t)
    heads, kv_heads, dim = rng.choice(_HEADS)
    if kind == "attention":
        seqs = _log(rng, 1, 16)
        # the widest layout costs what the largest listed prompt does
        most = int(math.sqrt(8192.0 ** 2 * 32 * 128 / (heads * dim * seqs)))
        lens = [_log(rng, 1, min(most, 8192)) for _ in range(seqs)]
        return dict(kind=kind, lens=",".join(map(str, lens)), heads=heads, kv_heads=kv_heads,
                    dim=dim)
    page = rng.choice([16, 32, 64, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= dim])
    if kind == "kv4":
        tokens = _log(rng, 1, 8192 * 8 * 128 // (max(kv_heads, 8) * dim))
        return dict(kind=kind, tokens=tokens, kv_heads=kv_heads, dim=dim, page=page, group=group,
                    pages=-(-tokens // page) + rng.randint(1, 64))
    seqs = _log(rng, 1, 48)
    most = min(131072, 131072 * 8 * 128 // (kv_heads * dim * seqs))
    lens = [_log(rng, 1, most) for _ in range(seqs)]
    return dict(kind=kind, lens=",".join(map(str, lens)), heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, group=group)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

class _Inputs:
    def __init__(self, seed):
        self.dev = torch.device("cuda:0")
        self.gen = torch.Generator(device=self.dev)
        self.gen.manual_seed(int(seed) * 6151 + 29)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device=self.dev)

    def uniform(self, lo, hi, *shape):
        return torch.rand(shape, generator=self.gen, device=self.dev) * (hi - lo) + lo

    def int8(self, *shape):
        return torch.randint(-127, 128, shape, generator=self.gen, device=self.dev,
                             dtype=torch.int8)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device=self.dev)

    def activations(self, m, k):
        x = self.normal(m, k)
        x[:, self.order(k)[: round(0.005 * k)]] *= 20.0
        return x.to(torch.float16)

    def keys(self, tokens, heads, dim):
        """Keys: each head has a few channels that are large in every token."""
        x = self.normal(tokens, heads, dim)
        x[:, :, self.order(dim)[: dim // 32]] *= 4.0
        return x.to(torch.float16)

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.dev)


def _lens(case):
    return [int(v) for v in case["lens"].split(",")]


def prepare(case, seed):
    g, kind = _Inputs(seed), case["kind"]
    st = dict(case=case)
    if kind == "attention":
        # one matrix from the layer's fused projection; q, k and v are columns of it
        h, kh, d, lens = case["heads"], case["kv_heads"], case["dim"], _lens(case)
        t = sum(lens)
        qkv = g.normal(t, (h + 2 * kh) * d)
        qkv[:, : h * d] *= 2.0
        qkv = qkv.to(torch.float16)
        st["q"] = qkv[:, : h * d].unflatten(1, (h, d))
        st["k"] = qkv[:, h * d: (h + kh) * d].unflatten(1, (kh, d))
        st["v"] = qkv[:, (h + kh) * d:].unflatten(1, (kh, d))
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        st["starts"] = g.ints(starts)
    elif kind == "kv4":
        t, kh, d = case["tokens"], case["kv_heads"], case["dim"]
        page, pages = case["page"], case["pages"]
        st["k"], st["v"] = g.keys(t, kh, d), g.normal(t, kh, d).to(torch.float16)
        # the tokens fill whole pages of a pool in any order
        at = torch.arange(t, device=g.dev)
        st["slots"] = (g.order(pages)[at // page] * page + at % page).to(torch.int32)
        st["cache"] = _empty_cache(pages, kh, page, d, case["group"], g.dev)
    elif kind == "attention_kv4":
        h, kh, d, page, lens = (case["heads"], case["kv_heads"], case["dim"], case["page"],
                                _lens(case))
        per = -(-max(lens) // page)  # columns of the block table
        pages = sum(-(-n // page) for n in lens) + 3
        st["q"] = (g.normal(len(lens), h, d) * 2.0).to(torch.float16)
        st["cache"] = _empty_cache(pages, kh, page, d, case["group"], g.dev)
        for at in range(0, pages, 4096):  # in pieces: a long cache is large in 32 bits
            n = min(4096, pages - at)
            ids = (torch.arange(n * page, device=g.dev) + at * page)
            _write(st["cache"], ids, g.keys(n * page, kh, d),
                   g.normal(n * page, kh, d).to(torch.float16))
        pool, table, used = g.order(pages).tolist(), [], 0
        for n in lens:
            own_pages = -(-n // page)
            table.append(pool[used: used + own_pages] + [-1] * (per - own_pages))
            used += own_pages
        st["table"], st["lens"] = g.ints(table), g.ints(lens)
    else:
        t, h, i, e = case["tokens"], case["hidden"], case["inter"], case["experts"]
        # weight scales that leave both products' outputs of the order of 1
        st.update(x=g.activations(t, h), logits=g.normal(t, e), s=g.uniform(0.5, 2.0, e, h),
                  wgu=g.int8(e, 2 * i, h), sgu=g.uniform(3e-5, 3e-4, e, 2 * i),
                  s2=g.uniform(0.5, 2.0, e, i), wd=g.int8(e, h, i),
                  sd=g.uniform(3e-5, 3e-4, e, h))
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(st):
    kind = st["case"]["kind"]
    if own:
        return _call(st)
    if kind == "attention":
        return _attention(st["q"], st["k"], st["v"], st["starts"], max(_lens(st["case"])))
    if kind == "kv4":
        _write(st["cache"], st["slots"], st["k"], st["v"])
        return _read(st["cache"], st["slots"])
    if kind == "attention_kv4":
        return _attention_kv4(st["q"], st["cache"], st["table"], st["lens"])
    return _experts(st["x"], st["logits"], st["s"], st["wgu"], st["sgu"], st["s2"], st["wd"],
                    st["sd"], st["case"]["topk"])


def _call(st):
    import optimized_rocwmma_samples_amd as w8a8

    kind = st["case"]["kind"]
    if kind == "attention":
        return w8a8.attention(st["q"], st["k"], st["v"], st["starts"])
    if kind == "experts":
        return w8a8.moe_ffn_decode(st["x"], st["logits"], st["s"], st["wgu"], st["sgu"], st["wd"],
                                   st["sd"], st["case"]["topk"], st["s2"])
    cache = st.get("handle")
    if cache is None:  # the handle a program makes when it allocates its cache
        c = st["cache"]
        cache = st["handle"] = w8a8.KV4Cache(c["k_codes"], c["v_codes"], c["k_scales"],
                                             c["v_scales"])
    if kind == "kv4":
        w8a8.kv4_store(st["k"], st["v"], st["slots"], cache)
        return w8a8.kv4_load(cache, st["slots"])
    return w8a8.attention_kv4(st["q"], cache, st["table"], st["lens"])


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _attention(q, k, v, starts, longest):
    """out[t, h] = sum_j p[j] v[j], p = softmax over the tokens j <= t of t's own
    sequence of q[t, h] . k[j] / sqrt(dim); sequences padded to one length."""
    tokens, heads, dim = q.shape
    kv_heads, seqs = k.shape[1], starts.numel() - 1
    pos = torch.arange(longest, device=q.device)
    rows = (starts[:-1, None] + pos).clamp(max=tokens - 1)

    def padded(x, per):  # [tokens, n * per, dim] -> [seqs * n, per * longest, dim]
        n = x.shape[1] // per
        x = x[rows].to(torch.float32).unflatten(2, (n, per)).permute(0, 2, 3, 1, 4)
        return x.reshape(seqs * n, per * longest, dim)

    per = heads // kv_heads
    s = torch.bmm(padded(q, per) * (1.0 / math.sqrt(dim)),
                  padded(k, 1).transpose(1, 2).contiguous())
    s = s.view(seqs * kv_heads, per, longest, longest)
    s.masked_fill_(pos[None, :] > pos[:, None], -math.inf)
    s -= s.amax(dim=-1, keepdim=True)
    s.exp_()
    total = s.sum(dim=-1, keepdim=True)
    o = torch.bmm(s.view(seqs * kv_heads, per * longest, longest), padded(v, 1))
    o = o.view(seqs, kv_heads, per, longest, dim) / total.view(seqs, kv_heads, per, longest, 1)
    t = torch.arange(tokens, device=q.device)
    seq = torch.searchsorted(starts, t, right=True) - 1
    return o[seq, :, :, t - starts[seq]].reshape(tokens, heads, dim).to(torch.float16)


# The cache: per page and key head, page-size rows of dim / 2 bytes of codes, the even
# channel of a pair in the low half of its byte, and rows of dim / group (scale, offset)
# pairs in fp16.  A value is offset + scale * (code - 8).  The rows of keys hold the
# channels in the order [4][dim / 32][8]: channel 32 j + 8 g + i at place (g, j, i).

def _empty_cache(pages, kv_heads, page, dim, group, dev):
    codes = lambda: torch.zeros((pages, kv_heads, page, dim // 2), dtype=torch.uint8,  # noqa: E731
                                device=dev)
    scales = lambda: torch.zeros((pages, kv_heads, page, dim // group, 2),  # noqa: E731
                                 dtype=torch.float16, device=dev)
    return dict(k_codes=codes(), v_codes=codes(), k_scales=scales(), v_scales=scales())


def _quantize4(x, group):
    """(codes [.., dim], scales [.., dim / group, 2]) of fp16 x [.., dim]."""
    x = x.to(torch.float32).unflatten(-1, (-1, group))
    low, high = x.amin(dim=-1, keepdim=True), x.amax(dim=-1, keepdim=True)
    scale = ((high - low) / 15.0).to(torch.float16)
    offset = (low + 8.0 * scale.to(torch.float32)).to(torch.float16)
    # 64 bits: a quotient next to a half goes to the side it is on
    at = torch.round((x.double() - offset.double()) / scale.double()) + 8.0
    codes = torch.where(scale > 0, at.clamp(0, 15), 8.0)
    return codes.to(torch.uint8).flatten(-2), torch.cat([scale, offset], dim=-1)


def _rows(cache, slots):
    """Index of the rows of all heads of these slots."""
    kv_heads, page = cache["k_codes"].shape[1:3]
    slots = slots.to(torch.int64)
    return (slots // page)[:, None], torch.arange(kv_heads, device=slots.device), \
        (slots % page)[:, None]


def _write(cache, slots, k, v):
    at, dim = _rows(cache, slots), k.shape[-1]
    group = dim // cache["k_scales"].shape[3]
    codes, cache["k_scales"][at] = _quantize4(k, group)
    codes = codes.unflatten(-1, (dim // 32, 4, 8)).transpose(-3, -2).flatten(-3)
    cache["k_codes"][at] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    codes, cache["v_scales"][at] = _quantize4(v, group)
    cache["v_codes"][at] = codes[..., 0::2] | (codes[..., 1::2] << 4)


def _values(codes, scales, keys):
    """fp32 [.., dim] of rows of codes and scales."""
    n = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    dim = n.shape[-1]
    if keys:
        n = n.unflatten(-1, (4, dim // 32, 8)).transpose(-3, -2).flatten(-3)
    n = n.to(torch.float32).unflatten(-1, (scales.shape[-2], -1))
    scales = scales.to(torch.float32)
    return (scales[..., 1:] + scales[..., :1] * (n - 8.0)).flatten(-2)


def _read(cache, slots):
    at = _rows(cache, slots)
    return tuple(_values(cache[c + "_codes"][at], cache[c + "_scales"][at], c == "k")
                 .to(torch.float16) for c in "kv")


def _attention_kv4(q, cache, table, lens):
    """Attention of one token per sequence over the first lens[s] tokens of the
    pages in its row of the table; a sequence of no tokens gives zeros."""
    seqs, heads, dim = q.shape
    kv_heads, page = cache["k_codes"].shape[1:3]
    pages = table.clamp(min=0).to(torch.int64)

    def gathered(c):  # [seqs, kv_heads, columns * page, dim]
        x = _values(cache[c + "_codes"][pages], cache[c + "_scales"][pages], c == "k")
        return x.transpose(1, 2).reshape(seqs * kv_heads, -1, dim)

    qs = q.to(torch.float32).view(seqs * kv_heads, heads // kv_heads, dim) / math.sqrt(dim)
    s = torch.bmm(qs, gathered("k").transpose(1, 2).contiguous())
    s = s.view(seqs, heads, -1)
    none = torch.arange(s.shape[-1], device=q.device) >= lens[:, None]
    s.masked_fill_(none[:, None, :], -math.inf)
    s = torch.exp(s - s.amax(dim=-1, keepdim=True).clamp(min=-3e38))
    total = s.sum(dim=-1, keepdim=True)
    o = torch.bmm(s.view(seqs * kv_heads, heads // kv_heads, -1), gathered("v"))
    o = o.view(seqs, heads, dim) / torch.where(total > 0, total, 1.0)
    return o.to(torch.float16)


def _quantize8(p):
    """(whole numbers in -127..127, scale) of rows p, as the package's quantizer."""
    r = p.abs().amax(dim=-1, keepdim=True) / QMAX
    inv = torch.where(r > 0, 1.0 / r, 0.0)
    return torch.clamp(torch.round(p * inv), -QMAX, QMAX), r


def _experts(x, logits, s, wgu, sgu, s2, wd, sd, topk):
    """For each token and each of its topk experts e (the largest logits, the lower
    index first among equals), with q(.) the quantizer of a row:
      g, u = dequant(q(x * s[e]) . wgu[e]^T),  a = g / (1 + exp(-g)) * u * s2[e]
      out  = sum over its experts of softmax(logits)[e] * dequant(q(a) . wd[e]^T)"""
    tokens, inter = x.shape[0], wd.shape[2]
    logits = logits.to(torch.float32)
    top = torch.exp(logits - logits.amax(dim=1, keepdim=True))
    top = top / top.sum(dim=1, keepdim=True)
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :topk]
    weight, ids = top.gather(1, ids), ids.flatten()
    xq, r = _quantize8((x.to(torch.float32)[:, None, :] * s[ids].view(tokens, topk, -1)).flatten(0, 1))
    gu = torch.bmm(wgu[ids].to(torch.float32), xq[:, :, None])[:, :, 0] * r * sgu[ids]
    g, u = gu[:, :inter], gu[:, inter:]
    a, r = _quantize8(g / (1.0 + torch.exp(-g)) * u * s2[ids])
    y = torch.bmm(wd[ids].to(torch.float32), a[:, :, None])[:, :, 0] * r * sd[ids]
    return (y.view(tokens, topk, -1) * weight[:, :, None]).sum(dim=1).to(torch.float16)


# ---------------------------------------------------------------------------
# What a pass cannot do without: each input read once, each output written once
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "attention":
        h, kh, d, lens = case["heads"], case["kv_heads"], case["dim"], _lens(case)
        # two products over the keys j <= t of each token t
        return dict(bytes=sum(lens) * 4 * (h + kh) * d + 4 * (len(lens) + 1),
                    flops=4.0 * h * d * sum(n * (n + 1) // 2 for n in lens))
    if kind == "kv4":
        t, row = case["tokens"], case["kv_heads"] * case["dim"]
        # keys and values in; codes, scales out; codes, scales in; values out
        return dict(bytes=t * (8 * row + 2 * (row + 8 * row // case["group"]) + 4),
                    flops=16.0 * t * row)
    if kind == "attention_kv4":
        h, kh, d, lens = case["heads"], case["kv_heads"], case["dim"], _lens(case)
        return dict(bytes=sum(lens) * kh * (d + 8 * d // case["group"]) + len(lens) * 4 * h * d
                    + 4 * sum(1 + -(-n // case["page"]) for n in lens),
                    flops=4.0 * h * d * sum(lens))
    t, h, i, e, top = (case[v] for v in ("tokens", "hidden", "inter", "experts", "topk"))
    used = e * (1.0 - (1.0 - top / e) ** t)  # experts that some token is routed to
    return dict(bytes=used * (3 * h * i + 4 * (3 * i + 2 * h)) + 4 * t * h + 4 * t * e,
                flops=6.0 * t * top * h * i)


# ---------------------------------------------------------------------------
# The same outputs in 64 bits, sequence by sequence and expert by expert
# ---------------------------------------------------------------------------

def _f64(t):
    return t.to(torch.float64)


def _exact_attention(st):
    q, k, v = st["q"], st["k"], st["v"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    per, at = q.shape[1] // k.shape[1], 0
    for n in _lens(st["case"]):
        later = torch.ones((n, n), dtype=torch.bool, device=q.device).triu(1)
        for h in range(q.shape[1]):
            kh, vh = _f64(k[at: at + n, h // per]), _f64(v[at: at + n, h // per])
            s = _f64(q[at: at + n, h]) @ kh.t() / math.sqrt(q.shape[2])
            s[later] = -math.inf
            out[at: at + n, h] = torch.softmax(s, dim=1) @ vh
        at += n
    return out


def _exact_kv4(st):
    outs = []
    for x in (st["k"], st["v"]):
        x = _f64(x).unflatten(-1, (-1, st["case"]["group"]))
        low, high = x.min(dim=-1, keepdim=True)[0], x.max(dim=-1, keepdim=True)[0]
        step = _f64(((high - low) / 15).to(torch.float16))
        mid = _f64((low + 8 * step).to(torch.float16))
        n = torch.round((x - mid) / torch.where(step > 0, step, 1.0)).clamp(-8, 7)
        outs.append((mid + step * n).flatten(-2))
    return tuple(outs)


def _exact_rows(cache, c, pages):
    """fp64 [kv_heads, len(pages) * page, dim] of one sequence's keys or values."""
    codes, scales = cache[c + "_codes"][pages].to(torch.int32), _f64(cache[c + "_scales"][pages])
    dim, groups = codes.shape[-1] * 2, scales.shape[-2]
    ch = torch.arange(dim, device=codes.device)
    place = ch if c == "v" else ch // 8 % 4 * (dim // 4) + ch // 32 * 8 + ch % 8
    n = codes[..., place // 2] >> (place % 2 * 4) & 15
    of = ch // (dim // groups)
    x = scales[..., of, 1] + scales[..., of, 0] * (_f64(n) - 8)
    return x.transpose(0, 1).flatten(1, 2)


def _exact_attention_kv4(st):
    q, lens, page = st["q"], _lens(st["case"]), st["case"]["page"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    kv_heads = st["case"]["kv_heads"]
    for i, n in enumerate(lens):
        pages = st["table"][i, : -(-n // page)].to(torch.int64)
        k, v = (_exact_rows(st["cache"], c, pages)[:, :n] for c in "kv")
        s = _f64(q[i]).view(kv_heads, -1, q.shape[2]) @ k.transpose(1, 2) / math.sqrt(q.shape[2])
        out[i] = (torch.softmax(s, dim=2) @ v).flatten(0, 1)
    return out


def _exact_quantize8(p):
    r = p.abs().max(dim=1, keepdim=True)[0] / QMAX
    return torch.round(p / torch.where(r > 0, r, 1.0)).clamp(-QMAX, QMAX), r


def _exact_experts(st):
    x, case = _f64(st["x"]), st["case"]
    p = torch.softmax(_f64(st["logits"]), dim=1)
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    weights, ids = torch.topk(p, case["topk"], dim=1)
    for e in range(case["experts"]):
        tok, slot = torch.nonzero(ids == e, as_tuple=True)
        if tok.numel() == 0:
            continue
        q, r = _exact_quantize8(x[tok] * _f64(st["s"][e]))
        g, u = (q @ _f64(st["wgu"][e]).t() * r * _f64(st["sgu"][e])).chunk(2, dim=1)
        q, r = _exact_quantize8(g * torch.sigmoid(g) * u * _f64(st["s2"][e]))
        y = q @ _f64(st["wd"][e]).t() * r * _f64(st["sd"][e])
        out.index_add_(0, tok, y * weights[tok, slot][:, None])
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "kv4": _exact_kv4,
            "attention_kv4": _exact_attention_kv4, "experts": _exact_experts}[case["kind"]](st)
