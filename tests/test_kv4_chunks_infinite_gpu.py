"""Attention of chunks over groups whose scale or offset is an infinity: they count as NaN, to the
rows that see them, by each of the ways a sequence can go."""
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
