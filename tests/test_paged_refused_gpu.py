"""Sequences that get no places, told apart on the device, and pages that sequences share."""
from __future__ import annotations

import pytest

import paged_ref as P
from test_kv4_pages_gpu import ints

pytestmark = pytest.mark.gpu


def test_refused_sequences_in_a_step(w8a8, gpu):
    # a captured step; which sequences find places changes from replay to replay
    import attention_ref as R
    import torch
    heads, kv_heads, dim, page, seqs, tokens = 8, 2, 128, 16, 4, 48
    c = w8a8.KV4Cache.empty(16, kv_heads, dim, page, 32, gpu)
    keys = w8a8.KV4PageKeys.empty(c)
    fill = R.randn((256, kv_heads, dim), 1, gpu)
    table = torch.full((seqs, 3), -1, dtype=torch.int32, device=gpu)
    free, new, before, count = (ints(x, gpu) for x in (range(8), [0] * 4, [0] * 4, [0]))
    qkv = R.randn((tokens, (heads + 2 * kv_heads) * dim), 1, gpu)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in
               qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), dim=1))
    out = torch.zeros((tokens, heads, dim), dtype=torch.float16, device=gpu)
    ws = torch.empty(w8a8.attention_kv4_chunks_workspace_size(c, seqs, tokens, heads, 3) + 1,
                     dtype=torch.uint8, device=gpu)

    def step():
        slots, starts, after, left = w8a8.kv4_extend(new, before, table, free, count, page, tokens)
        refused = (new > 0) & (after == before)
        seen = torch.where(refused, 0, after)
        w8a8.kv4_store(k, v, slots, c)
        w8a8.kv4_summarize(c, keys, table, seen, starts, tokens)
        w8a8.attention_kv4_chunks(q, c, table, seen, starts, out=out, workspace=ws)
        return refused, after, starts, left, seen
    step()  # (no sequence has tokens: loads what a first call loads)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for i, (news, lens, pages, refuse) in enumerate([
            ([20, 16, 1, 0], [10, 16, 20, 30], 3, [0, 0, 0, 0]),
            ([20, 16, 1, 0], [10, 16, 20, 30], 1, [0, 1, 0, 0]),    # too few pages
            ([20, 6, 1, 0], [10, 10, 16, 30], 1, [0, 0, 1, 0]),
            ([3, 25, 2, 5], [10, 30, 16, 30], 3, [0, 1, 0, 0]),     # the table's columns
            ([20, 16, 13, 2], [10, 16, 20, 30], 4, [0, 0, 1, 1])]):  # the step's rows
        w8a8.kv4_store(fill, fill, torch.arange(256, dtype=torch.int32, device=gpu), c)
        keys.codes.fill_(77)
        table[:] = -1
        held = 0
        for s, n in enumerate(lens):  # its pages, from the end of the pool
            for col in range(P.ceil_div(n, page)):
                table[s, col] = 15 - held
                held += 1
        new.copy_(ints(news, gpu))
        before.copy_(ints(lens, gpu))
        count.copy_(ints([pages], gpu))
        out.fill_(7)
        ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        refused, after, starts, left, seen = got
        assert refused.tolist() == [bool(x) for x in refuse], i
        assert after.tolist() == [n if r else n + m for n, m, r in zip(lens, news, refuse)]
        at = starts.tolist()
        want = [0 if r else n + m for n, m, r in zip(lens, news, refuse)]
        assert seen.tolist() == want
        ref, bound, rows = P.chunks(q, c, table, want, at, dim ** -0.5)
        R.assert_within(out[rows], ref[rows], bound[rows], f"step {i}")
        assert (out[~rows] == 7).all()
        touched = set()
        for s, r in enumerate(refuse):
            if r:
                assert (out[at[s]: at[s + 1]] == 0).all()
            elif news[s]:
                touched |= set(table[s, lens[s] // page: P.ceil_div(want[s], page)].tolist())
        untouched = sorted(set(range(16)) - touched)
        assert (keys.codes[untouched] == 77).all() and not (keys.codes[sorted(touched)] == 77).all()


def test_shared_prefix(w8a8, gpu):
    # three sequences behind one prefix of two pages: trimmed to the prefix at the least, each
    # gives back its own pages, and all of them come back once
    import torch
    page = 16
    table = torch.full((3, 6), -1, dtype=torch.int32, device=gpu)
    table[:, 0], table[:, 1] = 9, 4
    free = ints([0, 1, 2, 3, 5, 6, 7, 8, -1, -1], gpu)
    lens, count = ints([32] * 3, gpu), ints([8], gpu)
    _, _, lens, count = w8a8.kv4_extend(ints([40, 1, 33], gpu), lens, table, free, count, page, 74)
    assert lens.tolist() == [72, 33, 65] and int(count) == 1
    lens, count = w8a8.kv4_trim(ints([32, 40, 50], gpu), lens, table, free, count, page)
    assert lens.tolist() == [32, 33, 50] and int(count) == 5
    lens, count = w8a8.kv4_trim(ints([32] * 3, gpu), lens, table, free, count, page)
    assert int(count) == 8 and sorted(free[:8].tolist()) == [0, 1, 2, 3, 5, 6, 7, 8]
