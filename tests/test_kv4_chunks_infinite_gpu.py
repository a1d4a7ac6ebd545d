"""Attention of chunks over groups whose scale or offset is an infinity: they count as NaN, to the
rows that see them, by each of the ways a sequence can go.  And of queries with infinities, whose
softmax is NaN."""
from __future__ import annotations

import pytest

from test_kv4_chunks_gpu import starts_of
from test_kv4_gpu import _filled, _table
from test_kv4_pages_gpu import ints

pytestmark = pytest.mark.gpu


# units of 32 rows, of 64, and keys and values unpacked first
@pytest.mark.parametrize("dim,group", [(128, 32), (128, 128), (64, 32)])
@pytest.mark.parametrize("news", [[4, 3], [40, 90], [61, 140]])
@pytest.mark.parametrize("part,value", [(0, float("inf")), (1, float("inf")), (1, -float("inf"))])
def test_infinite_groups_are_nan(w8a8, gpu, dim, group, news, part, value):
    # part 0: the scale, 1: the offset
    import attention_ref as R
    import torch
    heads, kv_heads, lens = 8, 2, [61, 400]
    per = heads // kv_heads
    c = _filled(w8a8, gpu, 30, kv_heads, dim, 16, group, 7)
    table, starts = _table(30, 26, 2, 5, gpu), starts_of(news)
    q = R.randn((starts[-1], heads, dim), 1, gpu)

    def run(cache):
        return w8a8.attention_kv4_chunks(q, cache, table, ints(lens, gpu), ints(starts, gpu))
    want, first = run(c), lens[1] - news[1]
    assert torch.isfinite(want).all()
    last = dim // group - 1
    for at in (0, first - 1, first, first + news[1] // 2, lens[1] - 1):
        page = int(table[1, at // 16])
        places = (table == page).nonzero().tolist()
        rows = torch.zeros(starts[-1], dtype=torch.bool, device=gpu)
        for i, col in places:  # the page may be in the other sequence as well
            t = col * 16 + at % 16
            if t < lens[i]:
                rows[starts[i] + max(0, t - (lens[i] - news[i])): starts[i + 1]] = True
        for keys in (True, False):
            d = w8a8.KV4Cache(*(t.clone() for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales)))
            (d.k_scales if keys else d.v_scales)[page, 1, at % 16, last, part] = value
            nan = torch.zeros(want.shape, dtype=torch.bool, device=gpu)
            nan[rows, per:, (0 if keys else last * group):] = True
            got = run(d)
            assert torch.isnan(got[nan]).all(), (at, keys)
            assert torch.equal(got[~nan], want[~nan]), (at, keys)


@pytest.mark.parametrize("news,lens", [([4, 3], [61, 2]), ([40, 90], [40, 700]), ([9, 140], [5, 140])])
def test_infinite_queries_are_nan(w8a8, gpu, news, lens):
    # all scores -infinity among them, which is what unseen keys have as well; a row that sees
    # no key gives zeros all the same
    import attention_ref as R
    import torch
    heads, kv_heads, dim = 8, 2, 128
    c = w8a8.KV4Cache.empty(50, kv_heads, dim, 16, 32, gpu)
    k = R.randn((800, kv_heads, dim), 1, gpu).abs() + 1
    w8a8.kv4_store(k, R.randn(k.shape, 2, gpu), torch.arange(800, dtype=torch.int32, device=gpu), c)
    table, starts = _table(50, 46, 2, 5, gpu), starts_of(news)
    q = R.randn((starts[-1], heads, dim), 3, gpu)

    def run(q):
        return w8a8.attention_kv4_chunks(q, c, table, ints(lens, gpu), ints(starts, gpu))
    want = run(q)
    assert torch.isfinite(want).all()
    bad, nan = q.clone(), torch.zeros(want.shape, dtype=torch.bool, device=gpu)
    for i, (row, head, channel, value) in enumerate([
            (0, 0, 0, float("-inf")), (1, 3, 127, float("inf")), (starts[1], 5, 64, float("-inf")),
            (starts[1] + 1, 7, 31, float("-inf")), (starts[-1] - 1, 4, 9, float("-inf")),
            (starts[-1] - 1, 2, 77, float("inf"))]):
        bad[row, head, channel] = value
        s = 0 if row < starts[1] else 1
        nan[row, head] = lens[s] - news[s] + row - starts[s] >= 0
    got = run(bad)
    assert torch.isnan(got[nan]).all() and torch.equal(got[~nan], want[~nan])
