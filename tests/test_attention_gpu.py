"""Causal attention of packed prompts against the formula in 64 bits."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


def _ref():
    import attention_ref
    return attention_ref


def _inputs(tokens, heads, kv_heads, dim, seed, gpu, spread=2.0):
    """q, k, v as columns of one projection's output."""
    R = _ref()
    qkv = R.randn((tokens, (heads + 2 * kv_heads) * dim), seed, gpu)
    q = qkv[:, : heads * dim].unflatten(1, (heads, dim))
    q *= spread
    k = qkv[:, heads * dim: (heads + kv_heads) * dim].unflatten(1, (kv_heads, dim))
    v = qkv[:, (heads + kv_heads) * dim:].unflatten(1, (kv_heads, dim))
    return q, k, v


def _starts(lens, gpu, first=0):
    import torch
    at = [first]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=gpu), list(zip(at[:-1], at[1:]))


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (8, 1, 128), (3, 3, 128), (10, 2, 64)])
@pytest.mark.parametrize("lens", [[1], [7], [31, 32, 33], [63, 64, 65, 0, 1], [127, 128, 129],
                                  [0, 300, 2], [515], [1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 257]])
def test_packed_lengths(w8a8, gpu, heads, kv_heads, dim, lens):
    R = _ref()
    q, k, v = _inputs(sum(lens), heads, kv_heads, dim, 11 * len(lens) + heads, gpu)
    starts, spans = _starts(lens, gpu)
    got = w8a8.attention(q, k, v, starts)
    out, bound, _ = R.attention(q, k, v, spans, dim ** -0.5)
    R.assert_within(got, out, bound, f"lens {lens}")


def test_long_prompt_and_many_heads(w8a8, gpu):
    R = _ref()
    q, k, v = _inputs(2049, 32, 8, 128, 5, gpu)
    starts, spans = _starts([2049], gpu)
    got = w8a8.attention(q, k, v, starts)
    out, bound, _ = R.attention(q, k, v, spans, 128 ** -0.5)
    R.assert_within(got, out, bound)


def test_many_sequences(w8a8, gpu):
    # more sequences than a wave has lanes, most of them a token or none
    R = _ref()
    lens = [(i * 7) % 4 if i % 50 else 140 for i in range(201)]
    q, k, v = _inputs(sum(lens), 4, 4, 64, 9, gpu)
    starts, spans = _starts(lens, gpu)
    got = w8a8.attention(q, k, v, starts)
    out, bound, rows = R.attention(q, k, v, spans, 0.125)
    assert rows.all()
    R.assert_within(got, out, bound)


@pytest.mark.parametrize("scale", [1e-3, 0.7, 30.0])
def test_scale(w8a8, gpu, scale):
    # from a flat softmax to one that is a single key almost everywhere
    R = _ref()
    q, k, v = _inputs(200, 4, 2, 128, 3, gpu)
    starts, spans = _starts([200], gpu)
    got = w8a8.attention(q, k, v, starts, scale=scale)
    out, bound, _ = R.attention(q, k, v, spans, scale)
    R.assert_within(got, out, bound)


def test_growing_scores_rescale(w8a8, gpu):
    # each key scores higher than those before it: the running maximum moves at every tile
    import torch
    R = _ref()
    n, dim = 400, 64
    q = torch.ones((n, 1, dim), dtype=torch.float16, device=gpu)
    k = (torch.arange(n, device=gpu) / 8.0).to(torch.float16)[:, None, None].expand(n, 1, dim)
    k = k.contiguous()
    v = R.randn((n, 1, dim), 4, gpu)
    for kk in (k, k.flip(0).contiguous()):
        starts, spans = _starts([n], gpu)
        got = w8a8.attention(q, kk, v, starts)
        out, bound, _ = R.attention(q, kk, v, spans, dim ** -0.5)
        R.assert_within(got, out, bound)


def test_rows_outside_the_sequences_stay(w8a8, gpu):
    import torch
    R = _ref()
    q, k, v = _inputs(300, 4, 2, 128, 21, gpu)
    wide = torch.full((300, 4 * 128 + 64), 7.0, dtype=torch.float16, device=gpu)
    out = wide[:, : 4 * 128].unflatten(1, (4, 128))
    starts, spans = _starts([70, 0, 100], gpu, first=13)
    assert w8a8.attention(q, k, v, starts, out=out) is out
    ref, bound, rows = R.attention(q, k, v, spans, 128 ** -0.5)
    assert (out[~rows] == 7).all() and (wide[:, 4 * 128:] == 7).all()
    R.assert_within(out[rows], ref[rows], bound[rows])


def test_starts_past_the_rows_count_as_their_ends(w8a8, gpu):
    import torch
    R = _ref()
    q, k, v = _inputs(150, 2, 1, 64, 2, gpu)
    starts = torch.tensor([-40, 60, 100000, 2 ** 31 - 1], dtype=torch.int32, device=gpu)
    got = w8a8.attention(q, k, v, starts)
    ref, bound, rows = R.attention(q, k, v, [(0, 60), (60, 150)], 0.125)
    assert rows.all()
    R.assert_within(got, ref, bound)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("at", [0, 1, 30, 64, 100, 149])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_comes_later_does_not_reach_a_token(w8a8, gpu, dim, at, value):
    # a non-finite key and value at one token: the tokens before it, and the other
    # sequences, keep their results bit for bit; the tokens from it on see it
    import torch
    q, k, v = _inputs(220, 2, 1, dim, 8, gpu)
    starts, _ = _starts([150, 70], gpu)
    want = w8a8.attention(q, k, v, starts)
    v[at, :, 3] = value
    got = w8a8.attention(q, k, v, starts)
    clean = torch.ones(220, dtype=torch.bool, device=gpu)
    clean[at:150] = False
    assert torch.equal(got[clean], want[clean])
    assert not torch.isfinite(got[at:150, :, 3]).any()
    others = [c for c in range(dim) if c != 3]
    assert torch.equal(got[..., others], want[..., others])
    k[at, :, 5] = value
    got = w8a8.attention(q, k, v, starts)
    assert torch.equal(got[clean], want[clean])


def test_empty_calls(w8a8, gpu):
    import torch
    q = torch.empty((0, 4, 64), dtype=torch.float16, device=gpu)
    got = w8a8.attention(q, q, q, torch.zeros(3, dtype=torch.int32, device=gpu))
    assert got.shape == (0, 4, 64)
    q, k, v = _inputs(5, 4, 4, 64, 8, gpu)
    out = torch.full((5, 4, 64), 3.0, dtype=torch.float16, device=gpu)
    w8a8.attention(q, k, v, torch.zeros(1, dtype=torch.int32, device=gpu), out=out)
    w8a8.attention(q, k, v, torch.full((4,), 5, dtype=torch.int32, device=gpu), out=out)
    torch.cuda.synchronize()
    assert (out == 3).all()


def test_graph_replays_and_other_streams(w8a8, gpu):
    import torch
    q, k, v = _inputs(333, 8, 2, 128, 31, gpu)
    starts, _ = _starts([200, 133], gpu)
    want = w8a8.attention(q, k, v, starts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = w8a8.attention(q, k, v, starts)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w8a8.attention(q, k, v, starts, out=out)
    for i in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        # new contents in the same buffers, other sequences among them
        q.copy_(_inputs(333, 8, 2, 128, 50 + i, gpu)[0])
        starts[1] = 100 + i
        want = w8a8.attention(q, k, v, starts)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,lens", [(2, [700, 33]), (64, [1100])])
def test_values_at_the_ends_of_fp16(w8a8, gpu, dim, heads, lens):
    # a result is a mean of the values: those of 65504 cannot make an infinity, whatever the
    # rounded probabilities add up to
    import torch
    R = _ref()
    n = sum(lens)
    q, k, v = _inputs(n, heads, 1, dim, 41, gpu)
    v[..., 0::4], v[..., 1::4] = 65504.0, -65504.0
    starts, spans = _starts(lens, gpu)
    got = w8a8.attention(q, k, v, starts)
    out, bound, _ = R.attention(q, k, v, spans, dim ** -0.5)
    assert float(out.max()) > 65503.9 and float(out.min()) < -65503.9
    R.assert_within(got, out, bound)
    # an infinite value is seen as one
    v[20, 0, 2] = math.inf
    got = w8a8.attention(q, k, v, starts)
    assert (got[20:lens[0], :, 2] == math.inf).all()
    v[20, 0, 6] = math.nan
    got = w8a8.attention(q, k, v, starts)
    assert torch.isnan(got[20:lens[0], :, 6]).all() and torch.isfinite(got[..., 0]).all()


def test_long_offsets(w8a8, gpu):
    # rows that lie past 2^31 values and 2^32 bytes from the tensors' starts
    import torch
    R = _ref()
    tokens, width, n = 40000, 65536, 300
    qkv = torch.empty((tokens, width), dtype=torch.float16, device=gpu)
    assert (tokens - n) * width > 2 ** 31
    q, k, v, out = (qkv[:, at:at + h * 64].unflatten(1, (h, 64))
                    for at, h in ((0, 4), (1024, 2), (2048, 2), (3200, 4)))
    small = [R.randn((n, t.shape[1], 64), s, gpu) for s, t in ((1, q), (2, k), (3, v))]
    for t, x in zip((q, k, v), small):
        t[-n:] = x
    out[-n - 1] = 7.0
    starts = torch.tensor([tokens - n, tokens - 77, tokens], dtype=torch.int32, device=gpu)
    w8a8.attention(q, k, v, starts, out=out)
    ref, bound, _ = R.attention(*small, [(0, n - 77), (n - 77, n)], 0.125)
    R.assert_within(out[-n:], ref, bound)
    assert (out[-n - 1] == 7).all()
