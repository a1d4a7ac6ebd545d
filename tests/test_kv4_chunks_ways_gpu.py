"""Attention of chunks whose sequences go either way, unpacked first or where they are used: in
batches of many, in one captured launch after another, with strides, in runs of whole units."""
from __future__ import annotations

import numpy as np
import pytest

import paged_ref as P
from test_kv4_chunks_gpu import check, starts_of
from test_kv4_gpu import _filled, _table
from test_kv4_pages_gpu import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,longs", [(64, [0, 63]), (65, [64]), (150, [1, 63, 64, 127, 149])])
def test_long_ones_among_many(w8a8, gpu, seqs, longs):
    # up to 64 sequences and more; long ones at the ends of 64
    lens = [1 + 37 * i % 290 for i in range(seqs)]
    news = [min(n, i % 4) for i, n in enumerate(lens)]
    for x, i in enumerate(longs):
        lens[i], news[i] = 300 - 7 * x, 140 + 11 * x
    c = _filled(w8a8, gpu, 60, 2, 64, 16, 32, seqs)
    check(w8a8, gpu, c, _table(60, 19, seqs, seqs, gpu), lens, news, 8, 9)


def test_ways_in_a_graph(w8a8, gpu):
    # one captured call replayed while sequences change their ways and the workspace holds anything
    import attention_ref as R
    import torch
    c = _filled(w8a8, gpu, 80, 2, 128, 64, 32, 9)
    table = _table(80, 20, 4, 1, gpu)
    tokens = 700
    q, out = (torch.zeros((tokens, 8, 128), dtype=torch.float16, device=gpu) for _ in range(2))
    n, starts = ints([0] * 4, gpu), ints([0] * 5, gpu)
    ws = torch.empty(w8a8.attention_kv4_chunks_workspace_size(c, 4, tokens, 8, 20),
                     dtype=torch.uint8, device=gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w8a8.attention_kv4_chunks(q, c, table, n, starts, out=out, workspace=ws)
    for i, (lens, news) in enumerate([([900, 1280, 33, 500], [300, 1, 3, 200]),
                                      ([901, 5, 34, 0], [1, 5, 1, 0]),
                                      ([1, 1280, 0, 640], [1, 500, 0, 140]),
                                      ([1000, 1000, 1000, 1000], [129, 128, 200, 130])]):
        q.copy_(R.randn(q.shape, 80 + i, gpu))
        n.copy_(ints(lens, gpu))
        starts.copy_(ints(starts_of(news), gpu))
        ws.fill_(255 if i % 2 else 127)
        out.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        ref, bound, rows = P.chunks(q, c, table, lens, starts_of(news), 128 ** -0.5)
        R.assert_within(out[rows], ref[rows], bound[rows], f"replay {i}")
        assert (out[~rows] == 7).all()


@pytest.mark.parametrize("page", [16, 1024])
def test_long_with_strides(w8a8, gpu, page):
    import attention_ref as R
    import torch
    c = _filled(w8a8, gpu, 4096 // page, 2, 128, page, 64, 9)
    cols = 2048 // page
    table = _table(4096 // page, 2 * cols, 2, 1, gpu)[:, cols // 2: cols // 2 + cols]
    news, lens = [350, 171], [2048, 171]
    qkv = R.randn((521, 14 * 128), 3, gpu)
    q = qkv[:, 128: 11 * 128].unflatten(1, (10, 128))
    buf = torch.full((521, 12 * 128), 7.0, dtype=torch.float16, device=gpu)
    out = buf[:, 128: 11 * 128].unflatten(1, (10, 128))
    w8a8.attention_kv4_chunks(q, c, table, ints(lens, gpu), ints(starts_of(news), gpu), out=out)
    ref, bound, _ = P.chunks(q, c, table, lens, starts_of(news), 128 ** -0.5)
    R.assert_within(out, ref, bound)
    assert (buf[:, :128] == 7).all() and (buf[:, 11 * 128:] == 7).all()


@pytest.mark.parametrize("seqs,kv_heads,most,new", [(24, 8, 256, 5), (24, 8, 1000, 4), (90, 2, 500, 1),
                                                    (16, 8, 768, 9), (3, 1, 260, 40),
                                                    (70, 8, 130, 2)])
def test_short_units(w8a8, gpu, seqs, kv_heads, most, new):
    # a run a unit and equal runs, at the batches where one becomes the other
    lens = (most - np.arange(seqs) * 3 % 50).tolist()
    c = _filled(w8a8, gpu, 80, kv_heads, 128, 16, 32, seqs)
    check(w8a8, gpu, c, _table(80, P.ceil_div(most, 16), seqs, 3, gpu), lens, [new] * seqs,
          8 * kv_heads, 2)
