"""Attention of several new tokens per sequence over the 4-bit cache against the formula in
64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import paged_ref as P
from test_kv4_gpu import WIDTHS, _filled, _table
from test_kv4_pages_gpu import ints

pytestmark = pytest.mark.gpu


def starts_of(news, first=0):
    return (np.concatenate([[0], np.cumsum(news)]) + first).tolist()


def check(w8a8, gpu, c, table, lens, news, heads, seed, spread=2.0, first=0, behind=0,
          max_new=None):
    """The rows of the sequences against the formula, the others left as they were."""
    import attention_ref as R
    import torch
    starts = starts_of(news, first)
    tokens = starts[-1] + behind
    q = R.randn((tokens, heads, c.head_dim), seed, gpu, spread)
    out, bound, rows = P.chunks(q, c, table, lens, starts, c.head_dim ** -0.5)
    got = torch.full_like(q, 7.0)
    w8a8.attention_kv4_chunks(q, c, table, ints(lens, gpu), ints(starts, gpu), out=got,
                              max_new=max_new)
    R.assert_within(got[rows], out[rows], bound[rows])
    assert (got[~rows] == 7).all()
    again = torch.full_like(q, 7.0)
    w8a8.attention_kv4_chunks(q, c, table, ints(lens, gpu), ints(starts, gpu), out=again,
                              max_new=max_new)
    assert torch.equal(got, again)  # no order changes it
    return q, got


@pytest.mark.parametrize("dim,group", WIDTHS)
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (17, 1), (40, 8)])
@pytest.mark.parametrize("page,lens,news", [
    (16, [1], [1]), (16, [17, 40, 31, 5], [3, 1, 31, 5]), (32, [200, 64, 129], [5, 33, 1]),
    (64, [300], [77]), (128, [131, 1, 127], [2, 1, 127])])
def test_chunks(w8a8, gpu, dim, group, heads, kv_heads, page, lens, news):
    cols = P.ceil_div(max(lens), page) + 1
    c = _filled(w8a8, gpu, cols + 3, kv_heads, dim, page, group, dim + page)
    table = _table(cols + 3, cols, len(lens), len(lens), gpu)
    check(w8a8, gpu, c, table, lens, news, heads, heads)


@pytest.mark.parametrize("dim,group,heads,kv_heads", [(128, 32, 32, 8), (64, 64, 4, 4),
                                                      (128, 128, 8, 1), (128, 64, 12, 4),
                                                      (64, 32, 16, 2)])
@pytest.mark.parametrize("lens,news", [([3000], [8]), ([2500, 64, 1, 4001], [1, 64, 1, 5]),
                                       ([1500, 900], [300, 900]), ([700], [700]),
                                       ([4096, 130], [129, 128])])
def test_chunks_long(w8a8, gpu, dim, group, heads, kv_heads, lens, news):
    c = _filled(w8a8, gpu, 70, kv_heads, dim, 64, group, 77)
    table = _table(70, 64, len(lens), 5, gpu)
    check(w8a8, gpu, c, table, lens, news, heads, 6)
    check(w8a8, gpu, c, table, lens, news, heads, 6, max_new=max(news))
    # a bound that does not hold costs time, not rows
    check(w8a8, gpu, c, table, lens, news, heads, 6, max_new=1)
    check(w8a8, gpu, c, table, lens, news, heads, 6, max_new=20)


@pytest.mark.parametrize("dim,group", WIDTHS)
@pytest.mark.parametrize("heads,kv_heads", [(8, 1), (10, 2), (16, 8), (34, 2), (3, 3)])
@pytest.mark.parametrize("lens,news", [([600], [600]), ([701, 5, 900], [513, 5, 400]),
                                       ([1000, 1000], [577, 260]), ([131, 650], [130, 519])])
def test_chunks_of_many_rows(w8a8, gpu, dim, group, heads, kv_heads, lens, news):
    # sequences of more than 512 rows a key head: first new tokens at any place of a key tile
    c = _filled(w8a8, gpu, 70, kv_heads, dim, 16, group, dim + heads)
    table = _table(70, 63, len(lens), heads, gpu)
    check(w8a8, gpu, c, table, lens, news, heads, 3)


def test_chunks_many_sequences(w8a8, gpu):
    # more sequences than lanes, empty ones among them, more units than blocks
    rng = np.random.default_rng(3)
    for seqs, kv_heads, most in ((150, 1, 300), (200, 4, 90)):
        lens = [int(v) for v in rng.integers(1, most, seqs)]
        news = [int(rng.integers(0, min(n, 9) + 1)) for n in lens]
        news[3] = lens[3] = 40
        c = _filled(w8a8, gpu, 60, kv_heads, 64, 16, 32, seqs)
        table = _table(60, P.ceil_div(most, 16), seqs, seqs, gpu)
        check(w8a8, gpu, c, table, lens, news, 2 * kv_heads, 9)


def test_chunks_rows_of_no_sequence(w8a8, gpu):
    # rows before the first and behind the last sequence; lengths that make no sense; more new
    # tokens than there are, whose first rows see nothing
    c = _filled(w8a8, gpu, 20, 2, 128, 16, 32, 5)
    table = _table(20, 6, 5, 8, gpu)
    _, got = check(w8a8, gpu, c, table, [50, 0, -9, 2 ** 31 - 1, 4], [9, 3, 2, 7, 11], 4, 1,
                   first=5, behind=6)
    starts = starts_of([9, 3, 2, 7, 11], 5)
    assert (got[starts[1]: starts[3]] == 0).all() and (got[starts[4]: starts[4] + 7] == 0).all()


def test_chunks_nothing(w8a8, gpu):
    import torch
    c = _filled(w8a8, gpu, 3, 2, 64, 16, 32, 5)
    q = torch.ones((4, 4, 64), dtype=torch.float16, device=gpu)
    none = torch.empty((2, 0), dtype=torch.int32, device=gpu)
    got = w8a8.attention_kv4_chunks(q, c, none, ints([5, 5], gpu), ints([0, 3, 4], gpu))
    assert (got == 0).all()
    bad = torch.full((2, 9), -1, dtype=torch.int32, device=gpu)
    got = w8a8.attention_kv4_chunks(q, c, bad, ints([140, 144], gpu), ints([0, 3, 4], gpu))
    assert (got == 0).all()
    out = torch.full_like(q, 3.0)
    w8a8.attention_kv4_chunks(q, c, bad, ints([9, 9], gpu), ints([2, 2, 2], gpu), out=out)
    w8a8.attention_kv4_chunks(q[:0], c, bad, ints([9, 9], gpu), ints([0, 0, 0], gpu), out=out[:0])
    w8a8.attention_kv4_chunks(q, c, bad[:0], ints([], gpu), ints([0], gpu), out=out)
    assert (out == 3).all()


def test_chunks_starts_out_of_order(w8a8, gpu):
    # starts outside the rows or not ascending: counted as the nearer end, none where they fall
    import torch
    c = _filled(w8a8, gpu, 8, 1, 64, 16, 32, 5)
    table = _table(8, 4, 3, 1, gpu)
    q = torch.ones((10, 2, 64), dtype=torch.float16, device=gpu)
    a = w8a8.attention_kv4_chunks(q, c, table, ints([20, 30, 40], gpu), ints([-4, 6, 2, 99], gpu),
                                  out=torch.zeros_like(q))
    b = w8a8.attention_kv4_chunks(q, c, table[:1], ints([20], gpu), ints([0, 6], gpu),
                                  out=torch.zeros_like(q))
    assert torch.equal(a[:2], b[:2])
    d = w8a8.attention_kv4_chunks(q, c, table[2:], ints([40], gpu), ints([2, 10], gpu),
                                  out=torch.zeros_like(q))
    assert torch.equal(a[6:], d[6:])


@pytest.mark.parametrize("news", [[6, 20], [40, 90], [61, 140]])
def test_chunks_what_is_masked_does_not_reach(w8a8, gpu, news):
    # NaN behind a row's position, in pages that are not its own and outside the cache
    import torch
    c = _filled(w8a8, gpu, 24, 2, 128, 16, 32, 7)
    lens = [61, 150]
    table = torch.full((2, 12), 23, dtype=torch.int32, device=gpu)
    table[0, :4], table[1, :10] = ints([0, 1, 2, 3], gpu), ints([4, 5, -1, 7, 8, 24, 9, 10, 11, 12],
                                                                gpu)
    for s in (c.k_scales, c.v_scales):
        s[23] = float("nan")
        s[3, :, 13:] = float("inf")
        s[12, :, 6:] = float("nan")
    q, want = check(w8a8, gpu, c, table, lens, news, 8, 4)
    # a value of NaN at some new token: seen by its own and later rows, in its group only
    starts = starts_of(news)
    for at in (lens[1] - news[1], lens[1] - news[1] // 2, lens[1] - 1, 33 if news[1] < 100 else 0):
        d = w8a8.KV4Cache(*(t.clone() for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales)))
        page = int(table[1, at // 16])
        if not 0 <= page < c.pages:
            continue
        d.v_scales[page, 1, at % 16, 2] = float("nan")
        got = w8a8.attention_kv4_chunks(q, d, table, ints(lens, gpu), ints(starts, gpu))
        sees = torch.zeros(got.shape, dtype=torch.bool, device=gpu)
        first = starts[1] + max(0, at - (lens[1] - news[1]))
        sees[first:, 4:, 64:96] = True
        assert torch.isnan(got[sees]).all() and torch.equal(got[~sees], want[~sees])
        # and a key of NaN: in all of the row
        d.v_scales.copy_(c.v_scales)
        d.k_scales[page, 0, at % 16, 1] = float("nan")
        got = w8a8.attention_kv4_chunks(q, d, table, ints(lens, gpu), ints(starts, gpu))
        sees[:] = False
        sees[first:, :4] = True
        assert torch.isnan(got[sees]).all() and torch.equal(got[~sees], want[~sees])


@pytest.mark.parametrize("spread,qs", [(1e-3, 0.5), (0.05, 8.0), (3000.0, 0.5)])
def test_chunks_small_and_large_values(w8a8, gpu, spread, qs):
    c = _filled(w8a8, gpu, 20, 2, 128, 32, 32, 7, spread)
    check(w8a8, gpu, c, _table(20, 12, 2, 5, gpu), [380, 77], [9, 50], 8, 6, qs)


def test_chunks_of_exact_values(w8a8, gpu):
    # whole keys and values of -8 .. 7: the cache and the fp16 operands hold them exactly, so
    # only probabilities are rounded
    import attention_ref as R
    import torch
    for dim, group, heads, kv_heads in ((128, 32, 8, 2), (64, 64, 4, 4), (128, 128, 16, 1)):
        c = w8a8.KV4Cache.empty(12, kv_heads, dim, 32, group, gpu)
        g = torch.Generator().manual_seed(dim + group)
        kv = torch.randint(-8, 8, (2, 12 * 32, kv_heads, dim), generator=g).to(torch.float16)
        kv[..., 0::32], kv[..., 1::32] = -8, 7
        kv = kv.to(gpu)
        w8a8.kv4_store(kv[0], kv[1], torch.arange(384, dtype=torch.int32, device=gpu), c)
        table = torch.arange(12, dtype=torch.int32, device=gpu)[None]
        q = R.randn((50, heads, dim), 3, gpu, 0.2)
        got = w8a8.attention_kv4_chunks(q, c, table, ints([370], gpu), ints([0, 50], gpu))
        per = heads // kv_heads
        k, v = kv[:, :370].to(torch.float64)
        later = torch.arange(370, device=gpu)[None] > 320 + torch.arange(50, device=gpu)[:, None]
        for h in range(heads):
            qq, kk = q[:, h].to(torch.float64), k[:, h // per]
            s = (qq @ kk.t() * dim ** -0.5).masked_fill(later, -torch.inf)
            out, bound = R.softmax_pv(s, v[:, h // per], None, R.score_error(qq, kk, dim ** -0.5))
            R.assert_within(got[:, h], out, bound)


def test_chunks_ends_of_fp16(w8a8, gpu):
    # groups that reach 65504, whose last code stands for more: finite
    import torch
    c = w8a8.KV4Cache.empty(16, 2, 128, 16, 32, gpu)
    x = torch.rand((256, 2, 128), generator=torch.Generator().manual_seed(1)) * 65504
    x[..., 0::32], x[..., 1::32] = 0, 65504
    x = x.to(torch.float16).to(gpu)
    w8a8.kv4_store(x * 0, x, torch.arange(256, dtype=torch.int32, device=gpu), c)
    table = torch.arange(16, dtype=torch.int32, device=gpu)[None]
    for n, new in ((1, 1), (256, 5), (256, 256)):
        _, got = check(w8a8, gpu, c, table, [n], [new], 4, 2)
        assert torch.isfinite(got).all()
    w8a8.kv4_store(x * 0, x * 0 + 65504, torch.arange(256, dtype=torch.int32, device=gpu), c)
    _, got = check(w8a8, gpu, c, table, [256], [200], 4, 2)
    assert (got == 65504).all()
    # and keys of that size
    w8a8.kv4_store(x, x * 0 + 1, torch.arange(256, dtype=torch.int32, device=gpu), c)
    _, got = check(w8a8, gpu, c, table, [256], [3], 4, 2, 1e-3)
    assert torch.isfinite(got).all()


def test_chunks_infinite_queries(w8a8, gpu):
    # an infinity or NaN in a query stays in its own row and head
    import torch
    import attention_ref as R
    c = _filled(w8a8, gpu, 12, 2, 64, 16, 32, 7)
    table = _table(12, 10, 1, 5, gpu)
    q = R.randn((40, 6, 64), 1, gpu)
    args = (c, table, ints([150], gpu), ints([0, 40], gpu))
    want = w8a8.attention_kv4_chunks(q, *args)
    for at, value in (((3, 1, 5), float("nan")), ((39, 5, 0), float("inf"))):
        bad = q.clone()
        bad[at] = value
        got = w8a8.attention_kv4_chunks(bad, *args)
        rest = torch.ones(got.shape, dtype=torch.bool, device=gpu)
        rest[at[0], at[1]] = False
        assert torch.equal(got[rest], want[rest])
    bad = q.clone()
    bad[3, 1, 5] = float("nan")
    assert torch.isnan(w8a8.attention_kv4_chunks(bad, *args)[3, 1]).all()


def test_chunks_strides_streams_and_graph(w8a8, gpu):
    import attention_ref as R
    import torch
    c = _filled(w8a8, gpu, 40, 2, 128, 16, 32, 9)
    table = _table(40, 30, 3, 1, gpu)[:, 2:28]
    news, lens = [4, 1, 70], [400, 33, 90]
    starts, n = ints(starts_of(news), gpu), ints(lens, gpu)
    qkv = R.randn((75, 12 * 128), 3, gpu)
    q = qkv[:, : 8 * 128].unflatten(1, (8, 128))
    buf = torch.full((75, 10 * 128), 7.0, dtype=torch.float16, device=gpu)
    out = buf[:, : 8 * 128].unflatten(1, (8, 128))
    ref, bound, _ = P.chunks(q, c, table, lens, starts_of(news), 128 ** -0.5)
    w8a8.attention_kv4_chunks(q, c, table, n, starts, out=out)
    R.assert_within(out, ref, bound)
    assert (buf[:, 8 * 128:] == 7).all()
    size = w8a8.attention_kv4_chunks_workspace_size(c, 3, 75, 8, 26, 70)
    ws = torch.empty(size, dtype=torch.uint8, device=gpu)
    with pytest.raises(w8a8.W8A8Error, match="workspace"):
        w8a8.attention_kv4_chunks(q, c, table, n, starts, workspace=ws[:-1], max_new=70)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = w8a8.attention_kv4_chunks(q, c, table, n, starts)
    s.synchronize()
    assert torch.equal(got, out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w8a8.attention_kv4_chunks(q, c, table, n, starts, out=out, workspace=ws, max_new=70)
    for i in range(3):
        qkv.copy_(R.randn((75, 12 * 128), 80 + i, gpu))
        n.copy_(ints([400 - i, 33 + i, 90 - 5 * i], gpu))
        ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        ref, bound, _ = P.chunks(q, c, table, n.tolist(), starts_of(news), 128 ** -0.5)
        R.assert_within(out, ref, bound, f"replay {i}")


def test_chunks_of_one_token_are_decode(w8a8, gpu):
    import attention_ref as R
    import torch
    c = _filled(w8a8, gpu, 70, 4, 128, 64, 32, 2)
    lens = [4000, 1, 777, 0]
    table = _table(70, 64, 4, 3, gpu)
    q = R.randn((4, 16, 128), 1, gpu, 2.0)
    a = w8a8.attention_kv4(q, c, table, ints(lens, gpu))
    b = w8a8.attention_kv4_chunks(q, c, table, ints(lens, gpu), ints([0, 1, 2, 3, 4], gpu))
    _, one = R.attention_kv4(q, c, table, lens, 128 ** -0.5)
    _, two, _ = P.chunks(q, c, table, lens, [0, 1, 2, 3, 4], 128 ** -0.5)
    assert ((a.double() - b.double()).abs() <= one + two).all() and torch.isfinite(b).all()


def test_a_server(w8a8, gpu):
    """As a server runs them: prompts taken in by chunks, pages handed out on the device, keys
    and values stored, chunks attended to; then tokens decoded over the pages that suit them."""
    import attention_ref as R
    import torch
    heads, kv_heads, dim, page, seqs = 8, 2, 128, 16, 3
    c = w8a8.KV4Cache.empty(64, kv_heads, dim, page, 32, gpu)
    keys = w8a8.KV4PageKeys.empty(c)
    table = torch.full((seqs, 20), -1, dtype=torch.int32, device=gpu)
    lens = torch.zeros(seqs, dtype=torch.int32, device=gpu)
    free = torch.randperm(64, generator=torch.Generator().manual_seed(2)).to(torch.int32).to(gpu)
    count = ints([64], gpu)
    want_lens = [0] * seqs
    for step, new in enumerate([[70, 33, 0], [64, 1, 120], [1, 1, 1], [1, 1, 1], [90, 1, 5]]):
        tokens = sum(new)
        qkv = R.randn((tokens, (heads + 2 * kv_heads) * dim), step, gpu)
        q, k, v = (t.unflatten(1, (-1, dim)) for t in
                   qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), dim=1))
        slots, starts, lens, count = w8a8.kv4_extend(ints(new, gpu), lens, table, free, count, page,
                                                     tokens)
        w8a8.kv4_store(k, v, slots, c)
        w8a8.kv4_summarize(c, keys, table, lens, starts, tokens)
        want_lens = [a + b for a, b in zip(want_lens, new)]
        assert lens.tolist() == want_lens and (slots >= 0).all()
        ref, bound, rows = P.chunks(q, c, table, want_lens, starts.tolist(), dim ** -0.5)
        got = w8a8.attention_kv4_chunks(q, c, table, lens, starts)
        assert rows.all()
        R.assert_within(got, ref, bound, f"step {step}")
        if max(new) == 1:
            pages, left = w8a8.kv4_select(q, keys, table, lens, 4, page)
            chosen, n = P.select(q, keys.codes.cpu().numpy(), keys.scales.cpu().numpy(),
                                 table.tolist(), want_lens, 4, page, 64)
            assert pages.tolist() == chosen and left.tolist() == n
            got = w8a8.attention_kv4(q, c, pages, left)
            per = heads // kv_heads
            for h in range(kv_heads):
                ref, bound = R.attention_kv4(q, c, pages[:, h], n, dim ** -0.5)
                at = slice(h * per, (h + 1) * per)
                R.assert_within(got[:, at], ref[:, at], bound[:, at])
    # the first sequence ends, the second gives up its last 20 tokens
    lens, count = w8a8.kv4_trim(ints([0, 17, 10 ** 6], gpu), lens, table, free, count, page)
    want_lens = [0, 17, want_lens[2]]
    assert lens.tolist() == want_lens
    assert int(count) == 64 - sum(P.ceil_div(n, page) for n in want_lens)
    held = [p for i, n in enumerate(want_lens) for p in table[i, : P.ceil_div(n, page)].tolist()]
    assert sorted(held + free[: int(count)].tolist()) == list(range(64))
