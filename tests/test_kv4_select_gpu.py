"""Page keys, the pages that suit a query, and attention over a block table for each key
head: whole numbers equal, attention against the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import paged_ref as P
from test_kv4_gpu import WIDTHS, _filled, _table
from test_kv4_pages_gpu import ints

pytestmark = pytest.mark.gpu


def keys_of(w8a8, c, fill=99):
    k = w8a8.KV4PageKeys.empty(c)
    k.codes.fill_(fill)
    k.scales.fill_(float(fill))
    return k


def check_summary(w8a8, gpu, c, table, lens, news):
    """Page keys of the touched pages, the others left as they were; the keys."""
    import torch
    keys = keys_of(w8a8, c)
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    n, s = ints(lens, gpu), ints(starts, gpu)
    w8a8.kv4_summarize(c, keys, table, n, s, starts[-1])
    codes, scales = np.full(keys.codes.shape, 99.0), np.full(keys.scales.shape, 99.0)
    for i, (length, new) in enumerate(zip(lens, news)):
        if new == 0 or length <= 0:
            continue
        length = min(length, table.shape[1] * c.page_size)
        for col in range(max(length - new, 0) // c.page_size, P.ceil_div(length, c.page_size)):
            p = int(table[i, col])
            if 0 <= p < c.pages:
                codes[p], scales[p] = P.page_key(c, p, min(c.page_size, length - col * c.page_size))
    assert np.array_equal(keys.codes.cpu().numpy(), codes)
    assert np.array_equal(keys.scales.cpu().numpy(), scales.astype(np.float32), equal_nan=True)
    pages = torch.arange(c.pages, dtype=torch.int32, device=gpu)
    want = keys.codes.float() * keys.scales[..., None]
    assert torch.equal(torch.nan_to_num(w8a8.kv4_page_keys(keys, pages), 7),
                       torch.nan_to_num(want, 7))
    return keys


@pytest.mark.parametrize("dim,group", WIDTHS)
@pytest.mark.parametrize("page,lens,news", [
    (16, [1], [1]), (16, [16, 17, 40, 0, 5], [16, 1, 33, 0, 0]),
    (64, [130, 64, 63], [130, 2, 63]), (1024, [1500, 1], [700, 1]),
    (32, [5, 90], [9, 400])])  # more new tokens than there are: all of them
def test_summarize(w8a8, gpu, dim, group, page, lens, news):
    cols = P.ceil_div(max(lens), page) + 1
    heads = 3
    c = _filled(w8a8, gpu, cols * len(lens) + 2, heads, dim, page, group, dim + page)
    rng = np.random.default_rng(page)
    table = ints(rng.permutation(c.pages)[: cols * len(lens)].reshape(len(lens), cols), gpu)
    check_summary(w8a8, gpu, c, table, lens, news)


def test_summarize_many_sequences(w8a8, gpu):
    rng = np.random.default_rng(4)
    lens = [int(v) for v in rng.integers(0, 70, 150)]
    news = [int(rng.integers(0, n + 1)) for n in lens]
    c = _filled(w8a8, gpu, 150 * 5, 2, 64, 16, 32, 8)
    check_summary(w8a8, gpu, c, ints(np.arange(750).reshape(150, 5), gpu), lens, news)


def test_summarize_special_values(w8a8, gpu):
    # equal keys (a code of 127 or of a power of two), zeros, subnormals, the ends of fp16, NaN
    import torch
    c = _filled(w8a8, gpu, 9, 2, 64, 16, 32, 3)
    k = torch.zeros((9, 16, 2, 64), dtype=torch.float16, device=gpu)
    k[1] = 1.0
    k[2] = 127 / 128
    k[3] = 2.0 ** -24
    k[4] = 65504.0
    k[5, :, :, 3] = -65504.0
    k[6, 4, 1, 40] = float("nan")
    k[7, :8], k[7, 8:] = 3.0, -3.0
    k[8, :, :, :] = 0.5 + 2.0 ** -9  # halves between two codes
    flat = k.view(144, 2, 64)
    w8a8.kv4_store(flat, flat, torch.arange(144, dtype=torch.int32, device=gpu), c)
    keys = check_summary(w8a8, gpu, c, ints([list(range(9))], gpu), [144], [144])
    assert torch.isnan(keys.scales[6, 1]) and not torch.isnan(keys.scales[6, 0])
    assert (keys.scales[0] == 0).all() and (keys.scales[7] == 0).all()
    # pages outside the cache are passed over
    table = ints([[0, -1, 9, 2 ** 31 - 1, 3]], gpu)
    check_summary(w8a8, gpu, c, table, [80], [80])


def check_select(w8a8, gpu, q, keys, table, lens, keep, page):
    import torch
    want, left = P.select(q, keys.codes.cpu().numpy(), keys.scales.cpu().numpy(), table.tolist(),
                          lens, keep, page, keys.pages)
    got, n = w8a8.kv4_select(q, keys, table, ints(lens, gpu), keep, page)
    assert n.tolist() == left
    assert torch.equal(got, ints(want, gpu).view(got.shape))
    return got, n


def random_keys(w8a8, gpu, pages, heads, dim, seed, levels=128):
    """Page keys of few different values, so that scores are equal now and then."""
    import torch
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-levels + 1, levels, (pages, heads, dim), generator=g).to(torch.int8)
    scales = 2.0 ** torch.randint(-9, -6, (pages, heads), generator=g).float()
    return w8a8.KV4PageKeys(codes.to(gpu), scales.to(gpu))


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (128, 8, 2), (128, 17, 1), (64, 6, 2)])
@pytest.mark.parametrize("page,lens,keep", [(16, [0, 1, 16, 17, 160, 250], 4), (16, [900, 33], 1),
                                            (32, [3000, 64, 97], 2), (64, [5, 100], 300),
                                            (64, [64 * 40, 64 * 39 + 1], 39)])
def test_select(w8a8, gpu, dim, heads, kv_heads, page, lens, keep):
    from attention_ref import randn
    cols = P.ceil_div(max(lens), page)
    keys = random_keys(w8a8, gpu, cols + 7, kv_heads, dim, page + keep)
    table = _table(cols + 7, cols, len(lens), keep, gpu)
    q = randn((len(lens), heads, dim), dim + heads, gpu, 2.0)
    check_select(w8a8, gpu, q, keys, table, lens, keep, page)


@pytest.mark.parametrize("levels", [1, 2, 128])
def test_select_long_and_equal(w8a8, gpu, levels):
    # thousands of pages, all equal, of few values, and of many
    from attention_ref import randn
    page, cols = 16, 5000
    keys = random_keys(w8a8, gpu, cols, 2, 64, 3, levels)
    table = _table(cols, cols, 3, 4, gpu)
    q = randn((3, 4, 64), 5, gpu)
    for keep in (1, 64, 777, 4999):
        check_select(w8a8, gpu, q, keys, table, [16 * 5000, 16 * 1300 + 3, 16 * 778], keep, page)


def test_select_special_values(w8a8, gpu):
    # page keys of NaN and of zeros, pages outside, queries of zeros, infinities and NaN, and
    # sums that only 64 bits hold
    import torch
    keys = random_keys(w8a8, gpu, 30, 2, 64, 1)
    keys.scales[3, 0] = float("nan")
    keys.scales[4] = 0
    keys.codes[5] = 0
    table = torch.arange(30, dtype=torch.int32, device=gpu).repeat(6, 1)
    table[:, 7], table[:, 9], table[1, 29] = -1, 30, -5
    q = torch.randn((6, 8, 64), generator=torch.Generator().manual_seed(2)).to(torch.float16)
    q[1] = 0
    q[2, 0, 5] = float("inf")
    q[3, 6, 5] = float("nan")
    q[4, :, :] = 60000.0
    q[5, 0], q[5, 1], q[5, 2] = 65504.0, 2.0 ** -24, -65504.0
    q = q.to(gpu)
    for keep in (1, 5, 28, 29):
        check_select(w8a8, gpu, q, keys, table, [480, 480, 480, 480, 470, 465], keep, 16)


def test_select_strides_out_and_graph(w8a8, gpu):
    import torch
    from attention_ref import randn
    keys = random_keys(w8a8, gpu, 80, 2, 128, 8)
    wide = torch.stack([torch.randperm(80, generator=torch.Generator().manual_seed(i))
                        for i in range(3)]).to(torch.int32).to(gpu)
    table = wide[:, 5:65]
    qkv = randn((3, 12 * 128), 1, gpu)
    q = qkv[:, 128: 9 * 128].unflatten(1, (8, 128))
    lens = [960, 431, 16]
    want, left = check_select(w8a8, gpu, q, keys, table, lens, 9, 16)
    out = (torch.zeros_like(want), torch.zeros_like(left))
    n = ints(lens, gpu)
    ws = torch.empty(w8a8.kv4_select_workspace_size(3, 2, 60, 9), dtype=torch.uint8, device=gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w8a8.kv4_select(q, keys, table, n, 9, 16, out=out, workspace=ws)
    for i in range(3):
        qkv.copy_(randn((3, 12 * 128), 20 + i, gpu))
        ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        want, left = check_select(w8a8, gpu, q, keys, table, lens, 9, 16)
        assert torch.equal(out[0], want) and torch.equal(out[1], left)
    # tables of many columns need a workspace
    wide = table[:1].expand(3, 60).repeat(1, 100)
    assert w8a8.kv4_select_workspace_size(3, 2, 6000, 9) >= 3 * 2 * 6000 * 4
    with pytest.raises(w8a8.W8A8Error, match="workspace"):
        w8a8.kv4_select(q, keys, wide, n, 9, 16, workspace=None)
    check_select(w8a8, gpu, q, keys, wide, [16 * 5999, 431, 16], 9, 16)


def attention_by_head(q, c, tables, lens):
    """out, bound of attention with a table for each key head."""
    import attention_ref as R
    import torch
    out, bound = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    per = q.shape[1] // c.kv_heads
    for h in range(c.kv_heads):
        o, b = R.attention_kv4(q, c, tables[:, h], lens, c.head_dim ** -0.5)
        out[:, h * per: (h + 1) * per] = o[:, h * per: (h + 1) * per]
        bound[:, h * per: (h + 1) * per] = b[:, h * per: (h + 1) * per]
    return out, bound


@pytest.mark.parametrize("dim,group", WIDTHS)
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (36, 2)])
@pytest.mark.parametrize("page,lens", [(16, [1, 0, 40, 96]), (64, [640, 5])])
def test_attention_with_a_table_for_each_head(w8a8, gpu, dim, group, heads, kv_heads, page, lens):
    import torch
    import attention_ref as R
    c = _filled(w8a8, gpu, 25, kv_heads, dim, page, group, dim + heads)
    cols = P.ceil_div(max(lens), page)
    tables = _table(25, cols, len(lens) * kv_heads, heads, gpu).view(len(lens), kv_heads, cols)
    tables[0, 0, 0] = -1
    q = R.randn((len(lens), heads, dim), 5, gpu, 2.0)
    out, bound = attention_by_head(q, c, tables, lens)
    for ws in ("auto", None):
        got = w8a8.attention_kv4(q, c, tables, ints(lens, gpu), workspace=ws)
        R.assert_within(got, out, bound, f"workspace {ws}")
    # one table for all heads, given for each: bit for bit the same
    same = tables[:, :1].expand(-1, kv_heads, -1).contiguous()
    assert torch.equal(w8a8.attention_kv4(q, c, same, ints(lens, gpu)),
                       w8a8.attention_kv4(q, c, tables[:, 0].contiguous(), ints(lens, gpu)))
