"""Pages of the 4-bit cache handed out and taken back on the device, against whole numbers
on the host."""
from __future__ import annotations

import numpy as np
import pytest

import paged_ref as P

pytestmark = pytest.mark.gpu


def ints(v, gpu):
    import torch
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def state(rng, seqs, most, page, cols, spare):
    """Lengths, a table and a stack as a server has them."""
    lens = [int(v) for v in rng.integers(0, most + 1, seqs)]
    pool = [int(v) for v in rng.permutation(sum(P.ceil_div(n, page) for n in lens) + spare)]
    table, at = [], 0
    for n in lens:
        mine = P.ceil_div(n, page)
        table.append(pool[at: at + mine] + [-7] * (cols - mine))
        at += mine
    return lens, table, pool[at:] + [-9] * at, len(pool) - at


def check_extend(w8a8, gpu, new, lens, table, free, count, page, tokens):
    import torch
    want = P.extend(new, lens, table, free, count, page, tokens)
    t = ints(table, gpu).view(len(lens), -1)
    args = (ints(new, gpu), ints(lens, gpu), t, ints(free, gpu), ints([count], gpu))
    got = w8a8.kv4_extend(*args, page, tokens)
    for g, w in zip((*got, t), (want[0], want[1], want[2], [want[3]], want[4])):
        assert torch.equal(g, ints(w, gpu).view(g.shape))
    assert args[1].tolist() == lens and args[4].tolist() == [count]  # the inputs stay
    assert args[3].tolist() == free
    # and over the lengths and the count themselves
    t2 = ints(table, gpu).view(len(lens), -1)
    lens2, count2 = ints(lens, gpu), ints([count], gpu)
    out = (torch.full_like(got[0], 5), torch.full_like(got[1], 5), lens2, count2)
    w8a8.kv4_extend(args[0], lens2, t2, args[3], count2, page, tokens, out=out)
    for g, w in zip((*out, t2), (*got, t)):
        assert torch.equal(g, w)
    return got, t


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("seqs,most,new_most", [(1, 0, 1), (1, 200, 100), (7, 90, 40),
                                                (64, 300, 1), (65, 500, 70), (300, 40, 5)])
@pytest.mark.parametrize("spare", [0.0, 0.5, 1.5])
def test_extend(w8a8, gpu, page, seqs, most, new_most, spare):
    rng = np.random.default_rng(page + seqs + int(10 * spare))
    new = [int(v) for v in rng.integers(0, new_most + 1, seqs)]
    cols = P.ceil_div(most + new_most, page) + 1
    # enough pages for all of the new tokens, or for about half
    lens, table, free, count = state(rng, seqs, most, page, cols,
                                     int(spare * (sum(new) / page + seqs)))
    check_extend(w8a8, gpu, new, lens, table, free, count, page, sum(new))


def test_extend_refuses(w8a8, gpu):
    # rows past `tokens`, columns past the table, too few pages, and those behind them
    table = [[3, -1, -1], [4, 5, 6], [-1] * 3, [-1] * 3, [7, -1, -1], [-1] * 3]
    lens, new = [16, 40, 0, 0, 9, 0], [1, 9, 49, 33, 7, 20]
    free = [10, 11, 12, 13, 14, 15]
    for count in range(7):
        for tokens in (0, 1, 58, 59, 60, 98, 99, 119, 130):
            check_extend(w8a8, gpu, new, lens, table, free, count, 16, tokens)
    # numbers that make no sense count as the nearer end
    check_extend(w8a8, gpu, [-5, 3, 2 ** 31 - 1, 1], [-3, 2 ** 31 - 1, 5, 5],
                 [[1, 2], [3, 4], [5, 6], [7, -1]], free, 100, 16, 40)
    check_extend(w8a8, gpu, [1, 1], [0, 16], [[-1, -1], [2, -1]], free, -4, 16, 2)
    # a page that is none gives no slot
    check_extend(w8a8, gpu, [3, 18], [5, 5], [[-1, -1], [-1, -1]], [1, -3], 2, 16, 21)


def test_extend_nothing(w8a8, gpu):
    check_extend(w8a8, gpu, [0, 0], [5, 0], [[1], [-1]], [2], 1, 16, 4)
    import torch
    got = w8a8.kv4_extend(ints([], gpu), ints([], gpu),
                          torch.empty((0, 3), dtype=torch.int32, device=gpu), ints([1], gpu),
                          ints([1], gpu), 16, 3)
    assert [g.tolist() for g in got] == [[-1, -1, -1], [0], [], [1]]


@pytest.mark.parametrize("seqs,most,new", [(3, 100, 9000), (1500, 60, 12), (2100, 30, 1),
                                           (1024, 64, 33)])
def test_extend_large(w8a8, gpu, seqs, most, new):
    # more sequences than a block has threads, more tokens than one block takes
    rng = np.random.default_rng(seqs)
    fresh = [int(v) for v in rng.integers(0, new + 1, seqs)]
    for spare in (0.6, 2):
        lens, table, free, count = state(rng, seqs, most, 16, P.ceil_div(most + new, 16),
                                         int(spare * (sum(fresh) / 16 + seqs / 2)))
        check_extend(w8a8, gpu, fresh, lens, table, free, count, 16, sum(fresh) + 5)


def check_trim(w8a8, gpu, keep, lens, table, free, count, page):
    import torch
    after, left, stack = P.trim(keep, lens, table, free, count, page)
    t, f, n, c = ints(table, gpu), ints(free, gpu), ints(lens, gpu), ints([count], gpu)
    got = w8a8.kv4_trim(ints(keep, gpu), n, t, f, c, page)
    assert got[0].tolist() == after and got[1].tolist() == [left] and f.tolist() == stack
    assert n.tolist() == lens and c.tolist() == [count] and t.tolist() == table
    f2 = ints(free, gpu)
    w8a8.kv4_trim(ints(keep, gpu), n, t, f2, c, page, out=(n, c))
    assert n.tolist() == after and c.tolist() == [left] and torch.equal(f, f2)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("seqs,most,cols", [(1, 30, 3), (9, 200, 13), (70, 100, 9), (1300, 50, 4),
                                            (300, 700, 60)])
def test_trim(w8a8, gpu, page, seqs, most, cols):
    rng = np.random.default_rng(seqs + page)
    lens, table, free, count = state(rng, seqs, most, page, cols, 11)
    for keep in ([0] * seqs, lens, [max(0, n - int(d)) for n, d in
                                    zip(lens, rng.integers(0, 40, seqs))],
                 [int(v) for v in rng.integers(-3, most + 50, seqs)]):
        check_trim(w8a8, gpu, keep, lens, table, free, count, page)


def test_trim_past_the_stack(w8a8, gpu):
    # what the stack has no room for is dropped, and nothing written behind it
    check_trim(w8a8, gpu, [0, 5], [40, 60], [[1, 2, 3, 9], [4, 5, 6, 7]], [8, -1, -1, -1], 1, 16)
    check_trim(w8a8, gpu, [0, 5], [2 ** 31 - 1, -4], [[1, 2, 3, 9], [4, 5, 6, 7]], [8] * 9, 50, 16)


@pytest.mark.parametrize("seqs,new", [(40, 30), (3, 5000)])
def test_trim_restores_what_extend_took(w8a8, gpu, seqs, new):
    import torch
    rng = np.random.default_rng(seqs)
    lens, table, free, count = state(rng, seqs, 300, 16, 20 + new // 16, seqs * new // 16 + seqs)
    t, f, n, c = ints(table, gpu), ints(free, gpu), ints(lens, gpu), ints([count], gpu)
    fresh = ints([int(v) for v in rng.integers(0, new, seqs)], gpu)
    _, _, n2, c2 = w8a8.kv4_extend(fresh, n, t, f, c, 16, int(fresh.sum()))
    assert torch.equal(n2, n + fresh) and int(c2) < count
    n3, c3 = w8a8.kv4_trim(n, n2, t, f, c2, 16)
    assert torch.equal(n3, n) and torch.equal(c3, c) and f.tolist() == free


def test_tables_with_a_row_stride(w8a8, gpu):
    import torch
    rng = np.random.default_rng(1)
    lens, table, free, count = state(rng, 20, 100, 16, 9, 40)
    new = [int(v) for v in rng.integers(0, 30, 20)]
    want = P.extend(new, lens, table, free, count, 16, sum(new))
    wide = torch.full((20, 14), 77, dtype=torch.int32, device=gpu)
    wide[:, 3:12] = ints(table, gpu)
    got = w8a8.kv4_extend(ints(new, gpu), ints(lens, gpu), wide[:, 3:12], ints(free, gpu),
                          ints([count], gpu), 16, sum(new))
    assert got[0].tolist() == want[0] and wide[:, 3:12].tolist() == want[4]
    assert (wide[:, :3] == 77).all() and (wide[:, 12:] == 77).all()


def test_a_decode_loop_in_a_graph(w8a8, gpu):
    # a step after a step, replayed over its own lengths and count; now and then some
    # sequences end and their pages come back
    import torch
    rng = np.random.default_rng(5)
    seqs, page = 33, 16
    lens, table, free, count = state(rng, seqs, 40, page, 12, 90)
    t, f, n, c = ints(table, gpu), ints(free, gpu), ints(lens, gpu), ints([count], gpu)
    one, slots = ints([1] * seqs, gpu), ints([0] * seqs, gpu)
    starts, keep = ints([0] * (seqs + 1), gpu), n.clone()
    step, back = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(step):
        w8a8.kv4_extend(one, n, t, f, c, page, seqs, out=(slots, starts, n, c))
    with torch.cuda.graph(back):
        w8a8.kv4_trim(keep, n, t, f, c, page, out=(n, c))
    for i in range(12):
        step.replay()
        torch.cuda.synchronize()
        want, _, lens, count, table = P.extend([1] * seqs, lens, table, free, count, page, seqs)
        assert slots.tolist() == want and n.tolist() == lens and c.tolist() == [count]
        assert t.tolist() == table
        if i % 4 == 3:
            keep.copy_(ints([0 if (s + i) % 5 == 0 else 10 ** 6 for s in range(seqs)], gpu))
            back.replay()
            torch.cuda.synchronize()
            lens, count, free = P.trim(keep.tolist(), lens, table, free, count, page)
            assert n.tolist() == lens and c.tolist() == [count] and f.tolist() == free


def test_on_another_stream(w8a8, gpu):
    import torch
    rng = np.random.default_rng(9)
    lens, table, free, count = state(rng, 50, 300, 16, 30, 200)
    new = [int(v) for v in rng.integers(0, 60, 50)]
    want = P.extend(new, lens, table, free, count, 16, sum(new))
    t, args = ints(table, gpu), (ints(new, gpu), ints(lens, gpu))
    f, c = ints(free, gpu), ints([count], gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = w8a8.kv4_extend(*args, t, f, c, 16, sum(new))
    s.synchronize()
    assert got[0].tolist() == want[0] and t.tolist() == want[4]
