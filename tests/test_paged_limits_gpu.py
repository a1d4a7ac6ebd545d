"""The ends of what the paged 4-bit cache in service allows: caches past 2^32 bytes, more long
sequences than are unpacked, two calls at once, another device's current stream."""
from __future__ import annotations

import pytest

import paged_ref as P
from test_kv4_gpu import _filled, _table
from test_kv4_pages_gpu import ints

pytestmark = pytest.mark.gpu


def _head(w8a8, c, h, pages=slice(None)):
    """A cache of one key head of some pages."""
    return w8a8.KV4Cache(*(t[pages, h: h + 1].contiguous() for t in
                           (c.k_codes, c.v_codes, c.k_scales, c.v_scales)))


def test_cache_past_32_bits(w8a8, gpu):
    import attention_ref as R
    import torch
    pages, page, heads, dim = 600, 1024, 128, 128
    c = w8a8.KV4Cache.empty(pages, heads, dim, page, 128, gpu)
    assert c.k_codes.numel() > 2 ** 32
    for x in (c.k_scales, c.v_scales):
        x[0], x[pages - 2:] = 0, 0
    at = torch.arange(700, dtype=torch.int32, device=gpu) + (pages - 1) * page - 40
    k, v = R.randn((700, heads, dim), 1, gpu), R.randn((700, heads, dim), 2, gpu)
    w8a8.kv4_store(k, v, at, c)
    # the sequence's pages are the last two; its first 984 tokens are zeros
    table = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device=gpu)
    n = ints([2 * page - 364], gpu)
    tail = _head(w8a8, c, 127, slice(pages - 2, pages))
    near = torch.tensor([[0, 1]], dtype=torch.int32, device=gpu)
    for new in (3, 40, 600):  # by each of the ways
        q = R.randn((new, heads, dim), new, gpu)
        starts = ints([0, new], gpu)
        got = w8a8.attention_kv4_chunks(q, c, table, n, starts)
        out, bound, _ = P.chunks(q[:, 127:], tail, near, [int(n)], [0, new], dim ** -0.5)
        R.assert_within(got[:, 127:], out, bound)
    keys = w8a8.KV4PageKeys.empty(c)
    w8a8.kv4_summarize(c, keys, table, n, ints([0, 700], gpu), 700)
    codes, scale = P.page_key(tail, 1, int(n) - page)
    assert (keys.codes[-1, 127].cpu().numpy() == codes[0]).all()
    assert float(keys.scales[-1, 127]) == scale[0]


def test_more_long_sequences_than_are_unpacked(w8a8, gpu):
    # room for 32768 unpacked tokens of 64 key heads: the third sequence goes the other way
    import attention_ref as R
    import torch
    heads, dim, page, length, new = 64, 128, 64, 15000, 520
    per = P.ceil_div(length, page)
    c = _filled(w8a8, gpu, per, heads, dim, page, 32, 5)
    table = torch.stack([torch.randperm(per, generator=torch.Generator().manual_seed(i))
                         for i in range(3)]).to(torch.int32).to(gpu)
    q = R.randn((3 * new, heads, dim), 1, gpu, 2.0)
    lens, starts = [length, length - 33, length - 1], [0, new, 2 * new, 3 * new]
    got = w8a8.attention_kv4_chunks(q, c, table, ints(lens, gpu), ints(starts, gpu))
    for h in (0, 63):
        out, bound, _ = P.chunks(q[:, h: h + 1], _head(w8a8, c, h), table, lens, starts, dim ** -0.5)
        R.assert_within(got[:, h: h + 1], out, bound)


def test_two_at_once(w8a8, gpu):
    # chunks of one cache from two streams, each with its own workspace; selections beside them
    import attention_ref as R
    import torch
    c = _filled(w8a8, gpu, 80, 2, 128, 64, 32, 3)
    keys = w8a8.KV4PageKeys.empty(c)
    table = _table(80, 40, 2, 5, gpu)
    w8a8.kv4_summarize(c, keys, torch.arange(80, dtype=torch.int32, device=gpu)[None],
                       ints([5120], gpu), ints([0, 5120], gpu), 5120)
    args = [(R.randn((sum(new), 8, 128), s, gpu), ints(lens, gpu), ints([0, new[0], sum(new)], gpu))
            for s, lens, new in ((3, [2560, 77], [300, 5]), (4, [1000, 2000], [1, 700]))]

    def run(q, n, starts):
        return (w8a8.attention_kv4_chunks(q, c, table, n, starts),
                *w8a8.kv4_select(q[:2], keys, table, n, 7, 64))
    want = [run(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(10):
        for i, a in enumerate(args):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(*a))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for g in got[i] for x, y in zip(g, want[i]))


def test_a_graph_of_all(w8a8, gpu):
    # a server's whole step captured: pages, store, page keys, selection and both attentions
    import attention_ref as R
    import torch
    heads, kv_heads, dim, page, seqs = 8, 2, 128, 16, 3
    c = w8a8.KV4Cache.empty(64, kv_heads, dim, page, 32, gpu)
    keys = w8a8.KV4PageKeys.empty(c)
    table = torch.full((seqs, 20), -1, dtype=torch.int32, device=gpu)
    n, count, free = ints([0] * seqs, gpu), ints([64], gpu), torch.arange(64, dtype=torch.int32,
                                                                          device=gpu)
    new, tokens = ints([2, 1, 2], gpu), 5
    qkv = R.randn((tokens, (heads + 2 * kv_heads) * dim), 1, gpu)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in
               qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), dim=1))
    slots, starts = ints([0] * tokens, gpu), ints([0] * (seqs + 1), gpu)
    out = torch.zeros((tokens, heads, dim), dtype=torch.float16, device=gpu)
    one = torch.zeros((seqs, heads, dim), dtype=torch.float16, device=gpu)
    pages, left = torch.zeros((seqs, kv_heads, 3), dtype=torch.int32, device=gpu), ints([0] * 3, gpu)
    ws = [torch.empty(max(1, b), dtype=torch.uint8, device=gpu) for b in (
        w8a8.attention_kv4_chunks_workspace_size(c, seqs, tokens, heads, 20),
        w8a8.kv4_select_workspace_size(seqs, kv_heads, 20, 3),
        w8a8.attention_kv4_workspace_size(seqs, heads, kv_heads, dim, 3 * page))]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w8a8.kv4_extend(new, n, table, free, count, page, tokens, out=(slots, starts, n, count))
        w8a8.kv4_store(k, v, slots, c)
        w8a8.kv4_summarize(c, keys, table, n, starts, tokens)
        w8a8.attention_kv4_chunks(q, c, table, n, starts, out=out, workspace=ws[0])
        w8a8.kv4_select(q[:seqs], keys, table, n, 3, page, out=(pages, left), workspace=ws[1])
        w8a8.attention_kv4(q[:seqs], c, pages, left, out=one, workspace=ws[2])
    lens, want = [0] * seqs, [[-1] * 20 for _ in range(seqs)]
    stack, free_count = list(range(64)), 64
    for i in range(40):
        qkv.copy_(R.randn(qkv.shape, 30 + i, gpu))
        for w in ws:
            w.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        s, b, lens, free_count, want = P.extend([2, 1, 2], lens, want, stack, free_count, page, 5)
        assert slots.tolist() == s and starts.tolist() == b and n.tolist() == lens
        assert table.tolist() == want and count.tolist() == [free_count]
        ref, bound, _ = P.chunks(q, c, table, lens, b, dim ** -0.5)
        R.assert_within(out, ref, bound, f"replay {i}")
        chosen, m = P.select(q[:seqs], keys.codes.cpu().numpy(), keys.scales.cpu().numpy(), want,
                             lens, 3, page, 64)
        assert pages.tolist() == chosen and left.tolist() == m
        for h in range(kv_heads):
            at = slice(4 * h, 4 * h + 4)
            ref, bound = R.attention_kv4(q[:seqs], c, pages[:, h], m, dim ** -0.5)
            R.assert_within(one[:, at], ref[:, at], bound[:, at])
