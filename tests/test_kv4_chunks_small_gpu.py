"""Attention of chunks over small keys and values, whose scales and offsets are subnormal in fp16.

A value x = o + s (n - 8) enters as twice half(s (n - 8) / 2 + half(o / 2)).  s (n - 8) / 2 is
exact inside.  half(o / 2) is off by 2^-25 where o is an odd number of steps of 2^-24 below 2^-13,
else exact.  The sum is rounded to 2^-11 of itself or, where it is subnormal, to 2^-25.  So x is
off by 2^-11 |x| + 2 (2^-25 + 2^-25), two steps of 2^-24, where paged_ref.chunks allows ten."""
from __future__ import annotations

import pytest

import paged_ref as P
from test_kv4_gpu import _table
from test_kv4_pages_gpu import ints

pytestmark = pytest.mark.gpu


def _case(w8a8, gpu, monkeypatch, k, v, q, lens, news, page, group):
    import attention_ref as R
    import torch
    monkeypatch.setattr(P, "SUB16", P.SUB16 / 5)
    dim, pages = k.shape[2], k.shape[0] // page
    c = w8a8.KV4Cache.empty(pages, k.shape[1], dim, page, group, gpu)
    w8a8.kv4_store(k, v, torch.arange(k.shape[0], dtype=torch.int32, device=gpu), c)
    table = _table(pages, P.ceil_div(max(lens), page), len(lens), 5, gpu)
    starts = [sum(news[:i]) for i in range(len(news) + 1)]
    out, bound, _ = P.chunks(q, c, table, lens, starts, dim ** -0.5)
    got = w8a8.attention_kv4_chunks(q, c, table, ints(lens, gpu), ints(starts, gpu))
    R.assert_within(got, out, bound)


# few keys, so that errors do not average out, and many; units of 32 and 64 rows, unpacked first
LENS, NEWS = [1, 2, 5, 40, 700, 640], [1, 1, 3, 40, 600, 1]


@pytest.mark.parametrize("dim,group", [(128, 32), (64, 64), (128, 128)])
@pytest.mark.parametrize("spread", [1e-3, 1e-4, 1e-5, 1e-6])
def test_small_values(w8a8, gpu, monkeypatch, dim, group, spread):
    import attention_ref as R
    k, v = R.randn((768, 2, dim), 1, gpu), R.randn((768, 2, dim), 2, gpu, spread)
    q = R.randn((sum(NEWS), 8, dim), 3, gpu)
    _case(w8a8, gpu, monkeypatch, k, v, q, LENS, NEWS, 32, group)


@pytest.mark.parametrize("heads", [8, 80])  # units of 32 rows, and of 64
@pytest.mark.parametrize("dim,group", [(128, 32), (64, 64)])
@pytest.mark.parametrize("spread", [1e-3, 1e-4, 1e-5, 1e-6])
def test_small_keys(w8a8, gpu, heads, dim, group, spread):
    # One new token behind one other, whose values are 7 and -8, and queries of one channel: the
    # result is 7 - 15 / (1 + exp(s0 - s1)), whose slope is at most 15 / 4 and whose error of the
    # scores is that of two key values.  Probabilities are rounded to 2^-11 of themselves or to
    # 2^-25, 15 times of them at the most; fp32 steps add up to less than 2^-18.
    import attention_ref as R
    import torch
    seqs, kv_heads, per = 48, 2, heads // 2
    c = w8a8.KV4Cache.empty(seqs, kv_heads, dim, 16, group, gpu)
    slots = torch.arange(seqs * 16, dtype=torch.int32, device=gpu)
    k = R.randn((seqs, 16, kv_heads, dim), 1, gpu, spread)
    v = torch.full_like(k, 7.0)
    v[:, 1] = -8
    w8a8.kv4_store(k.flatten(0, 1), v.flatten(0, 1), slots, c)
    assert torch.equal(w8a8.kv4_load(c, slots)[1].view_as(v), v)
    size, scale = 6e4 if spread < 1e-3 else 1.5e4, dim ** -0.5
    q = torch.zeros((seqs, heads, dim), dtype=torch.float16, device=gpu)
    x = torch.zeros((seqs, heads, 2), dtype=torch.float64, device=gpu)
    values = R.cache_values(c, True)[0]
    for i in range(seqs):
        for h in range(heads):
            ch = (3 * i + 7 * h) % dim
            q[i, h, ch] = size
            x[i, h] = values[i, h // per, :2, ch]
    got = w8a8.attention_kv4_chunks(q, c, torch.arange(seqs, dtype=torch.int32, device=gpu)[:, None],
                                    ints([2] * seqs, gpu), ints(range(seqs + 1), gpu))
    size = float(q.max())
    p = torch.sigmoid((x[..., 0] - x[..., 1]) * size * scale)
    want = 7 * p - 8 * (1 - p)
    off = R.EPS16 * x.abs().sum(-1) + 2 * 2 * P.SUB16
    bound = 15 / 4 * off * size * scale + (R.EPS16 + 2.0 ** -18) * (7 * p + 8 * (1 - p)) + 2.0 ** -21
    bound = bound + R.EPS16 * (want.abs() + bound)
    R.assert_within(got, want[..., None].expand(got.shape), bound[..., None].expand(got.shape))
