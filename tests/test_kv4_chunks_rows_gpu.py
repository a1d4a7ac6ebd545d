"""Attention of chunks whose rows lie far apart: strides that pass 32 bits within a tile of rows."""
from __future__ import annotations

import pytest

import paged_ref as P
from test_kv4_gpu import _filled, _table
from test_kv4_pages_gpu import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("news", [[150], [3, 9, 138]])
def test_rows_past_32_bits(w8a8, gpu, news):
    # 2^25 values from row to row: row 64 of a tile lies 2^32 bytes behind its first
    import attention_ref as R
    import torch
    heads, dim, stride, rows = 8, 128, 2 ** 25, sum(news)
    lens = [n + 100 * i + 50 for i, n in enumerate(news)]
    starts = [sum(news[:i]) for i in range(len(news) + 1)]
    c = _filled(w8a8, gpu, 40, 2, dim, 16, 32, 3)
    table = _table(40, P.ceil_div(max(lens), 16), len(news), 5, gpu)
    near = R.randn((rows, heads, dim), 1, gpu)
    ref, bound, _ = P.chunks(near, c, table, lens, starts, dim ** -0.5)
    size = (rows - 1) * stride + heads * dim
    wide = [torch.empty(size, dtype=torch.float16, device=gpu).as_strided(
        (rows, heads, dim), (stride, dim, 1)) for _ in range(2)]
    wide[0].copy_(near)
    args = c, table, ints(lens, gpu), ints(starts, gpu)
    got = w8a8.attention_kv4_chunks(wide[0], *args, out=wide[1])
    R.assert_within(got, ref, bound)
    assert torch.equal(got, w8a8.attention_kv4_chunks(near, *args))
    del wide, got
    torch.cuda.empty_cache()
