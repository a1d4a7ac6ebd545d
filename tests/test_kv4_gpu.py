"""The 4-bit cache: rows in and out bit for bit, and the attention of single
tokens over it against the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

WIDTHS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


def _ref():
    import attention_ref
    return attention_ref


def _zeros(w8a8, gpu, pages, kv_heads, dim, page, group):
    import torch
    c = w8a8.KV4Cache.empty(pages, kv_heads, dim, page, group, gpu)
    for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales):
        t.fill_(119 if t.dtype == torch.uint8 else 5.0)
    return c


def _filled(w8a8, gpu, pages, kv_heads, dim, page, group, seed, spread=1.0):
    """A cache whose every slot holds something."""
    import torch
    R = _ref()
    c = _zeros(w8a8, gpu, pages, kv_heads, dim, page, group)
    n = pages * page
    k = R.randn((n, kv_heads, dim), seed, gpu)
    k[..., 1] *= 6
    w8a8.kv4_store(k, R.randn((n, kv_heads, dim), seed + 1, gpu, spread),
                   torch.arange(n, dtype=torch.int32, device=gpu), c)
    return c


@pytest.mark.parametrize("dim,group", WIDTHS)
@pytest.mark.parametrize("tokens,page", [(1, 16), (37, 32), (130, 64)])
def test_store_and_load(w8a8, gpu, dim, group, tokens, page):
    import torch
    R = _ref()
    heads, pages = 3, 5
    rng = np.random.default_rng(dim + group + tokens)
    c = _zeros(w8a8, gpu, pages, heads, dim, page, group)
    before = [t.cpu().numpy().copy() for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales)]
    qkv = R.randn((tokens, (2 * heads + 1) * dim), tokens, gpu, 3.0)
    k = qkv[:, : heads * dim].unflatten(1, (heads, dim))
    v = qkv[:, heads * dim: 2 * heads * dim].unflatten(1, (heads, dim))
    k[0, 0, :] = 2.5            # a group of equal values
    v[0, 1, :] = -0.0
    v[tokens - 1, 2, 5] = 6e4   # a wide range
    v[tokens - 1, 2, 6] = -6e4
    k[tokens - 1, 1, :] = k[tokens - 1, 1, :] * 2.0 ** -18  # subnormal steps
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    if tokens > 4:
        slots[2], slots[3] = -1, pages * page  # outside the cache: skipped
    w8a8.kv4_store(k, v, torch.from_numpy(slots).to(gpu), c)
    got = [t.cpu().numpy() for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales)]
    for side, x in enumerate((k, v)):
        x = x.cpu().numpy()
        codes, scale, offset = R.quantize4(x, group)
        for t, slot in enumerate(slots):
            if 0 <= slot < pages * page:
                at = (slot // page, slice(None), slot % page)
                before[side][at] = R.pack4(codes[t], side == 0)
                before[2 + side][at] = np.stack([scale[t], offset[t]], -1)
    for g, b in zip(got, before):
        assert np.array_equal(g.view(np.uint8), b.view(np.uint8))
    # back out: half(offset + scale * (code - 8)), rows outside left alone
    out = tuple(torch.full((tokens, heads, dim), 9.0, dtype=torch.float16, device=gpu)
                for _ in "kv")
    assert w8a8.kv4_load(c, torch.from_numpy(slots).to(gpu), out=out) is not None
    live = torch.from_numpy((slots >= 0) & (slots < pages * page)).to(gpu)
    s = torch.from_numpy(slots.astype(np.int64)).to(gpu)[live]
    for keys, o in ((True, out[0]), (False, out[1])):
        want = R.cache_values(c, keys)[0][s // page, :, s % page].to(torch.float32)
        assert torch.equal(o[live], want.to(torch.float16))
        assert (o[~live] == 9).all()


@pytest.mark.parametrize("dim,group", WIDTHS)
def test_store_keeps_half_a_step(w8a8, gpu, dim, group):
    # what comes back is within half a step of what went in, plus the roundings of
    # the offset, of the step (7.5 steps away at most) and of the value
    import torch
    R = _ref()
    n, heads = 64, 2
    c = _zeros(w8a8, gpu, 4, heads, dim, 16, group)
    k, v = R.randn((n, heads, dim), 3, gpu, 5.0), R.randn((n, heads, dim), 4, gpu, 0.01)
    slots = torch.arange(n, dtype=torch.int32, device=gpu)
    w8a8.kv4_store(k, v, slots, c)
    for x, y, scales in zip((k, v), w8a8.kv4_load(c, slots), (c.k_scales, c.v_scales)):
        step = scales.transpose(1, 2).reshape(n, heads, dim // group, 2)[..., 0].double()
        step = step.repeat_interleave(group, dim=2)
        big = x.double().abs().amax()
        slack = 2 * R.EPS16 * big + 9 * R.EPS16 * step + 2.0 ** -23
        assert ((x.double() - y.double()).abs() <= step / 2 + slack).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_store_of_a_nonfinite_group(w8a8, gpu, value):
    import torch
    R = _ref()
    c = _zeros(w8a8, gpu, 2, 2, 128, 16, 32)
    k, v = R.randn((3, 2, 128), 5, gpu), R.randn((3, 2, 128), 6, gpu)
    slots = torch.tensor([0, 20, 31], dtype=torch.int32, device=gpu)
    w8a8.kv4_store(k, v, slots, c)
    ko, vo = w8a8.kv4_load(c, slots)
    k[1, 0, 40] = value
    w8a8.kv4_store(k, v, slots, c)
    kn, vn = w8a8.kv4_load(c, slots)
    assert torch.isnan(kn[1, 0, 32:64]).all()
    ko[1, 0, 32:64] = kn[1, 0, 32:64] = 0
    assert torch.equal(kn, ko) and torch.equal(vn, vo)


def _table(pool_pages, cols, seqs, seed, gpu):
    import torch
    rng = np.random.default_rng(seed)
    t = np.stack([rng.permutation(pool_pages)[:cols] for _ in range(seqs)]).astype(np.int32)
    return torch.from_numpy(t).to(gpu)


@pytest.mark.parametrize("dim,group", WIDTHS)
@pytest.mark.parametrize("page,lens", [(16, [1]), (16, [15, 16, 17, 0, 63]), (32, [64, 65, 200]),
                                       (64, [1, 127, 128, 129]), (128, [700, 3])])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (17, 1)])
def test_decode_lengths(w8a8, gpu, dim, group, page, lens, heads, kv_heads):
    import torch
    R = _ref()
    cols = max(1, -(-max(lens) // page))
    c = _filled(w8a8, gpu, cols + 3, kv_heads, dim, page, group, dim + page)
    table = _table(cols + 3, cols, len(lens), len(lens), gpu)
    q = R.randn((len(lens), heads, dim), heads, gpu, 2.0)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    out, bound = R.attention_kv4(q, c, table, lens, dim ** -0.5)
    for ws in ("auto", None):
        got = w8a8.attention_kv4(q, c, table, n, workspace=ws)
        R.assert_within(got, out, bound, f"workspace {ws}")
        for i, length in enumerate(lens):
            assert length or (got[i] == 0).all()


@pytest.mark.parametrize("dim,group,heads,kv_heads", [(128, 32, 32, 8), (64, 64, 4, 4),
                                                      (128, 128, 64, 2), (128, 64, 8, 8)])
def test_decode_long(w8a8, gpu, dim, group, heads, kv_heads):
    import torch
    R = _ref()
    lens = [5000, 1, 8191, 0, 3333]
    page = 64
    c = _filled(w8a8, gpu, 140, kv_heads, dim, page, group, 77)
    table = _table(140, 128, len(lens), 5, gpu)
    q = R.randn((len(lens), heads, dim), 6, gpu, 2.0)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    got = w8a8.attention_kv4(q, c, table, n)
    out, bound = R.attention_kv4(q, c, table, lens, dim ** -0.5)
    R.assert_within(got, out, bound)
    assert torch.equal(got, w8a8.attention_kv4(q, c, table, n))  # no order changes it


@pytest.mark.parametrize("spread", [1e-3, 0.05, 3000.0])
def test_decode_small_and_large_values(w8a8, gpu, spread):
    import torch
    R = _ref()
    c = _filled(w8a8, gpu, 20, 2, 128, 32, 32, 7, spread)
    table = _table(20, 12, 2, 5, gpu)
    lens = [380, 77]
    q = R.randn((2, 8, 128), 6, gpu, 0.5)
    got = w8a8.attention_kv4(q, c, table, torch.tensor(lens, dtype=torch.int32, device=gpu))
    out, bound = R.attention_kv4(q, c, table, lens, 128 ** -0.5)
    # the least normal fp16 is the floor of a result's precision
    R.assert_within(got, out, bound)


def test_decode_scales_that_grow_along_the_context(w8a8, gpu):
    # values a million times larger at the end than at the start, and back
    import torch
    R = _ref()
    n = 512
    for order in (1, -1):
        c = _zeros(w8a8, gpu, 8, 1, 128, 64, 32)
        v = R.randn((n, 1, 128), 3, gpu)
        v *= (2.0 ** torch.linspace(-12, 8, n, device=gpu)[::1])[:, None, None].to(torch.float16)
        if order < 0:
            v = v.flip(0)
        w8a8.kv4_store(R.randn((n, 1, 128), 2, gpu), v.contiguous(),
                       torch.arange(n, dtype=torch.int32, device=gpu), c)
        q = R.randn((1, 4, 128), 6, gpu, 0.5)
        table = torch.arange(8, dtype=torch.int32, device=gpu)[None]
        got = w8a8.attention_kv4(q, c, table, torch.tensor([n], dtype=torch.int32, device=gpu))
        out, bound = R.attention_kv4(q, c, table, [n], 128 ** -0.5)
        R.assert_within(got, out, bound)


def test_decode_what_is_masked_does_not_reach(w8a8, gpu):
    # NaN scales and any codes behind a sequence's end, in pages that are not its own
    # and under page numbers outside the cache
    import torch
    R = _ref()
    c = _filled(w8a8, gpu, 10, 2, 128, 16, 32, 7)
    lens = [21, 0, 40]
    table = torch.tensor([[0, 1, 9, 9], [9, 9, 9, 9], [2, -5, 3, 10]], dtype=torch.int32,
                         device=gpu)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    q = R.randn((3, 8, 128), 6, gpu, 2.0)
    want = w8a8.attention_kv4(q, c, table, n)
    out, bound = R.attention_kv4(q, c, table, lens, 128 ** -0.5)
    R.assert_within(want, out, bound)
    assert (want[1] == 0).all()
    for s in (c.k_scales, c.v_scales):
        s[9] = float("nan")
        s[1, :, 5:] = float("inf")
        s[3, :, 8:] = float("nan")
    for ws in ("auto", None):
        assert torch.equal(w8a8.attention_kv4(q, c, table, n, workspace=ws),
                           want if ws else w8a8.attention_kv4(q, c, table, n, workspace=None))
        R.assert_within(w8a8.attention_kv4(q, c, table, n, workspace=ws), out, bound)
    # lengths outside the table count as its ends; a page of NaN that is seen shows
    c.k_scales[9] = c.v_scales[9] = 1.0
    n2 = torch.tensor([21, -7, 40], dtype=torch.int32, device=gpu)
    assert torch.equal(w8a8.attention_kv4(q, c, table, n2), want)
    c.v_scales[0, 1, 3] = float("nan")
    got = w8a8.attention_kv4(q, c, table, n)
    assert torch.isnan(got[0, 4:]).all() and torch.equal(got[0, :4], want[0, :4])
    assert torch.equal(got[1:], want[1:])


def test_decode_length_past_the_table(w8a8, gpu):
    import torch
    R = _ref()
    c = _filled(w8a8, gpu, 6, 1, 64, 16, 64, 3)
    table = _table(6, 4, 2, 3, gpu)
    q = R.randn((2, 2, 64), 6, gpu)
    got = w8a8.attention_kv4(q, c, table, torch.tensor([2 ** 31 - 1, 64], dtype=torch.int32,
                                                       device=gpu))
    out, bound = R.attention_kv4(q, c, table, [64, 64], 0.125)
    R.assert_within(got, out, bound)


def test_decode_strides_out_and_graph(w8a8, gpu):
    import torch
    R = _ref()
    c = _filled(w8a8, gpu, 40, 2, 128, 16, 32, 9)
    wide = _table(40, 30, 4, 1, gpu)
    table = wide[:, 2:27]
    qkv = R.randn((4, 12 * 128), 3, gpu)
    q = qkv[:, : 8 * 128].unflatten(1, (8, 128))
    n = torch.tensor([400, 1, 333, 16], dtype=torch.int32, device=gpu)
    buf = torch.full((4, 10 * 128), 7.0, dtype=torch.float16, device=gpu)
    out = buf[:, : 8 * 128].unflatten(1, (8, 128))
    w8a8.attention_kv4(q, c, table, n, out=out)
    ref, bound = R.attention_kv4(q, c, table, n.tolist(), 128 ** -0.5)
    R.assert_within(out, ref, bound)
    assert (buf[:, 8 * 128:] == 7).all()
    ws = torch.empty(max(1, w8a8.attention_kv4_workspace_size(4, 8, 2, 128, 25 * 16)),
                     dtype=torch.uint8, device=gpu)
    kn, vn = R.randn((4, 2, 128), 71, gpu), R.randn((4, 2, 128), 72, gpu)
    place = (n - 1).to(torch.int64)
    slots = (table.gather(1, (place // 16)[:, None])[:, 0] * 16 + place % 16).to(torch.int32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):  # a decode step: the new token stored, then attended to
        w8a8.kv4_store(kn, vn, slots, c)
        w8a8.attention_kv4(q, c, table, n, out=out, workspace=ws)
    for i in range(3):
        kn.copy_(R.randn((4, 2, 128), 80 + i, gpu))
        ws.fill_(255)  # what an earlier user left in it
        g.replay()
        torch.cuda.synchronize()
        ref, bound = R.attention_kv4(q, c, table, n.tolist(), 128 ** -0.5)
        R.assert_within(out, ref, bound, f"replay {i}")


def test_long_cache_offsets(w8a8, gpu):
    # a cache whose codes lie past 2^32 bytes from its start
    import torch
    R = _ref()
    pages, page, heads, dim = 600, 1024, 128, 128
    c = w8a8.KV4Cache.empty(pages, heads, dim, page, 128, gpu)
    assert c.k_codes.numel() > 2 ** 32
    t = torch.tensor([pages * page - 2, pages * page - 1, 0, 1], dtype=torch.int32, device=gpu)
    for x in (c.k_scales, c.v_scales):
        x[0], x[pages - 1] = 0, 0
    k, v = R.randn((4, heads, dim), 1, gpu), R.randn((4, heads, dim), 2, gpu)
    w8a8.kv4_store(k, v, t, c)
    ko, vo = w8a8.kv4_load(c, t)
    codes, scale, offset = R.quantize4(v[0, 127:].cpu().numpy(), 128)
    want = (offset.astype(np.float32)[..., None]
            + scale.astype(np.float32)[..., None] * (codes.astype(np.float32) - 8)[:, :])
    assert np.array_equal(vo[0, 127:].cpu().numpy(), want.reshape(1, dim).astype(np.float16))
    q = R.randn((1, heads, dim), 3, gpu)
    sub = w8a8.KV4Cache(c.k_codes[-1:], c.v_codes[-1:], c.k_scales[-1:], c.v_scales[-1:])
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=gpu)
    n = torch.tensor([1024], dtype=torch.int32, device=gpu)
    got = w8a8.attention_kv4(q, c, table, n)
    out, bound = R.attention_kv4(q, sub, torch.zeros_like(table), [1024], dim ** -0.5)
    R.assert_within(got, out, bound)


def test_prompt_then_token(w8a8, gpu):
    """A layer's step as a server runs it: the prompt's attention and its keys and
    values stored, then a token stored and attended to from the cache."""
    import torch
    R = _ref()
    heads, kv_heads, dim, page, n = 8, 2, 128, 16, 75
    hidden = heads * dim
    g = torch.Generator().manual_seed(3)
    wq = torch.randint(-127, 128, ((heads + 2 * kv_heads) * dim, hidden), generator=g,
                       dtype=torch.int8).to(gpu)
    sw = (torch.rand(wq.shape[0], generator=g) * 1e-4 + 1e-4).to(gpu)
    s = torch.ones(hidden, device=gpu)
    x = R.randn((n + 1, hidden), 1, gpu)
    qkv, _, _ = w8a8.fused_sq_gemm(x, s, wq, sw)
    q = qkv[:, :hidden].unflatten(1, (heads, dim))
    k = qkv[:, hidden: hidden + kv_heads * dim].unflatten(1, (kv_heads, dim))
    v = qkv[:, hidden + kv_heads * dim:].unflatten(1, (kv_heads, dim))
    prompt = w8a8.attention(q[:n], k[:n], v[:n],
                            torch.tensor([0, n], dtype=torch.int32, device=gpu))
    out, bound, _ = R.attention(q[:n], k[:n], v[:n], [(0, n)], dim ** -0.5)
    R.assert_within(prompt, out, bound)
    c = w8a8.KV4Cache.empty(9, kv_heads, dim, page, 32, gpu)
    table = torch.tensor([[3, 1, 8, 0, 5]], dtype=torch.int32, device=gpu)
    at = torch.arange(n + 1, device=gpu)
    slots = (table[0].to(torch.int64)[at // page] * page + at % page).to(torch.int32)
    w8a8.kv4_store(k[:n], v[:n], slots[:n], c)
    w8a8.kv4_store(k[n:], v[n:], slots[n:], c)
    got = w8a8.attention_kv4(q[n:], c, table, torch.tensor([n + 1], dtype=torch.int32, device=gpu))
    ref, bound = R.attention_kv4(q[n:], c, table, [n + 1], dim ** -0.5)
    R.assert_within(got, ref, bound)
    # and on into the next projection
    wo = torch.randint(-127, 128, (hidden, hidden), generator=g, dtype=torch.int8).to(gpu)
    y, _, _ = w8a8.fused_sq_gemm(got.flatten(1), s, wo, sw[:hidden].contiguous())
    assert torch.isfinite(y).all()


def _check_decode(w8a8, gpu, c, table, lens, heads, seed, spread=2.0):
    """Attention over the cache with and without a workspace against the formula."""
    import torch
    R = _ref()
    q = R.randn((len(lens), heads, c.head_dim), seed, gpu, spread)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    out, bound = R.attention_kv4(q, c, table, lens, c.head_dim ** -0.5)
    for ws in ("auto", None):
        got = w8a8.attention_kv4(q, c, table, n, workspace=ws)
        R.assert_within(got, out, bound, f"workspace {ws}")


@pytest.mark.parametrize("dim,group", WIDTHS)
@pytest.mark.parametrize("page,lens", [(16, [15, 16, 17, 0, 63, 64]), (64, [1, 127, 128, 129]),
                                       (128, [700, 3])])
@pytest.mark.parametrize("heads,kv_heads", [(8, 1), (5, 1), (16, 2), (18, 3), (32, 2), (36, 1)])
def test_decode_heads_of_a_key_head(w8a8, gpu, dim, group, page, lens, heads, kv_heads):
    # 5, 6 and 8 query heads a key head take half of a product's columns twice; 16 all of
    # them; 36 three units, the last of four heads
    cols = -(-max(lens) // page)
    c = _filled(w8a8, gpu, cols + 3, kv_heads, dim, page, group, dim + page + heads)
    table = _table(cols + 3, cols, len(lens), heads, gpu)
    _check_decode(w8a8, gpu, c, table, lens, heads, heads + 1)


@pytest.mark.parametrize("dim,group,heads,kv_heads", [(128, 32, 64, 8), (128, 64, 40, 8),
                                                      (128, 128, 8, 1), (64, 32, 12, 2)])
def test_decode_long_contexts_of_5_to_8_heads(w8a8, gpu, dim, group, heads, kv_heads):
    lens = [4999, 1, 8192, 0, 3333, 64]
    c = _filled(w8a8, gpu, 140, kv_heads, dim, 64, group, 78)
    _check_decode(w8a8, gpu, c, _table(140, 128, len(lens), 6, gpu), lens, heads, 7)


@pytest.mark.parametrize("seqs,heads,kv_heads,dim,group", [(130, 8, 1, 128, 32),
                                                           (130, 6, 2, 64, 64),
                                                           (300, 32, 8, 128, 64),
                                                           (300, 64, 8, 64, 32)])
def test_decode_many_sequences(w8a8, gpu, seqs, heads, kv_heads, dim, group):
    # more sequences than lanes; more units than waves, and more heads to join than blocks
    rng = np.random.default_rng(seqs + heads)
    lens = [int(v) for v in rng.integers(0, 250, seqs)]
    lens[:3] = [256, 0, 1]
    c = _filled(w8a8, gpu, 40, kv_heads, dim, 32, group, seqs)
    _check_decode(w8a8, gpu, c, _table(40, 8, seqs, seqs, gpu), lens, heads, 9)


def test_ends_of_fp16_read_back_finite(w8a8, gpu):
    # groups that reach 65504: the step and the offset are rounded to fp16, so the last code
    # may stand for more, and a finite group reads back finite all the same
    import torch
    R = _ref()
    c = _zeros(w8a8, gpu, 2, 2, 128, 16, 32)
    g = torch.Generator().manual_seed(1)
    x = torch.rand((6, 2, 128), generator=g)
    low = torch.tensor([0.0, -65504.0, -65504.0, 60000.0, -65504.0, 32768.0])[:, None, None]
    high = torch.tensor([65504.0, 65504.0, -34772.0, 65504.0, 0.0, 65504.0])[:, None, None]
    x = low + (high - low) * x
    x[..., 0::32], x[..., 1::32] = low.expand(6, 2, 4), high.expand(6, 2, 4)
    x = x.to(torch.float16).to(gpu)
    assert torch.isfinite(x).all()
    slots = torch.arange(6, dtype=torch.int32, device=gpu) + 5
    w8a8.kv4_store(x, x.flip(2).contiguous(), slots, c)
    k, v = w8a8.kv4_load(c, slots)
    whole = R.cache_values(c, True)[0][0, :, 5:11].transpose(0, 1)
    assert (whole.abs() >= 65520).any()  # what the codes stand for: past fp16
    for got, want in ((k, x), (v, x.flip(2))):
        assert torch.isfinite(got).all()
        # half a step of 8736 at the most, and the roundings of step and offset
        assert ((got.double() - want.double()).abs() <= 4368 + 15 * 8 + 16).all()
    # and attended to: a context of one such token is its values
    table = torch.zeros((1, 1), dtype=torch.int32, device=gpu)
    q = R.randn((1, 4, 128), 6, gpu)
    for t in range(6):
        d = w8a8.KV4Cache.empty(1, 2, 128, 16, 32, gpu)
        w8a8.kv4_store(x[t:t + 1] * 0, x[t:t + 1], torch.zeros(1, dtype=torch.int32, device=gpu), d)
        _, want = w8a8.kv4_load(d, torch.zeros(1, dtype=torch.int32, device=gpu))
        got = w8a8.attention_kv4(q, d, table, torch.ones(1, dtype=torch.int32, device=gpu))
        assert torch.isfinite(got).all()
        err = (got[0].view(2, 2, 128).double() - want[0, :, None].double()).abs()
        # p is 1: the scale of the centred code is rounded once as fp16, the result once
        assert (err <= 2.0 ** -11 * 8 * 8736 + 2.0 ** -11 * 65504).all()
    # cut by runs, whose parts a second launch joins: 256 such tokens
    d = w8a8.KV4Cache.empty(16, 1, 128, 16, 32, gpu)
    many = x[:1, :1].expand(256, 1, 128).contiguous()
    w8a8.kv4_store(many * 0, many, torch.arange(256, dtype=torch.int32, device=gpu), d)
    got = w8a8.attention_kv4(q[:, :2], d, torch.arange(16, dtype=torch.int32, device=gpu)[None],
                             torch.tensor([256], dtype=torch.int32, device=gpu))
    assert torch.isfinite(got).all() and float(got.max()) >= 65504 - 2.0 ** -11 * 8 * 8736


def test_cache_whose_tensors_move_is_refused(w8a8, gpu):
    # the handle knows where its tensors lay: calls must not write where they no longer are
    import torch
    c = _filled(w8a8, gpu, 3, 2, 64, 16, 32, 5)
    with pytest.raises(AttributeError):
        c.k_codes = torch.zeros_like(c.k_codes)
    kv = _ref().randn((2, 2, 64), 1, gpu)
    slots = torch.tensor([3, 40], dtype=torch.int32, device=gpu)
    table = torch.tensor([[0, 1], [2, 0]], dtype=torch.int32, device=gpu)
    q, n = _ref().randn((2, 4, 64), 2, gpu), torch.tensor([20, 9], dtype=torch.int32, device=gpu)
    want = w8a8.attention_kv4(q, c, table, n)
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        t = getattr(c, name)
        keep = t.data
        t.data = t.clone()
        for call in (lambda: w8a8.kv4_store(kv, kv, slots, c), lambda: w8a8.kv4_load(c, slots),
                     lambda: w8a8.attention_kv4(q, c, table, n)):
            with pytest.raises(ValueError, match="KV4Cache"):
                call()
        assert torch.equal(w8a8.attention_kv4(
            q, w8a8.KV4Cache(c.k_codes, c.v_codes, c.k_scales, c.v_scales), table, n), want)
        t.data = keep
    assert torch.equal(w8a8.attention_kv4(q, c, table, n), want)
