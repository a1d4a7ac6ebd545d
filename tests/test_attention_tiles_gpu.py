"""Causal attention at the call sizes that take each of its four tile shapes: few blocks and
many, heads of 64 and 128, with sequences that end inside, at and past a tile."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim,lens", [
    (2, 128, [257, 64, 1]), (96, 128, [129, 127, 640, 31, 33]), (96, 128, [1100]),
    (2, 64, [257, 64, 1, 700]), (2, 64, [128, 60, 3]), (96, 64, [129, 127, 640, 31, 33]),
    (96, 64, [1100])])
def test_tiles(w8a8, gpu, heads, dim, lens):
    import attention_ref as R
    import torch
    n = sum(lens)
    q, k, v = R.randn((n, heads, dim), 1, gpu), R.randn((n, 2, dim), 2, gpu), \
        R.randn((n, 2, dim), 3, gpu)
    at = [0]
    for length in lens:
        at.append(at[-1] + length)
    starts = torch.tensor(at, dtype=torch.int32, device=gpu)
    got = w8a8.attention(q, k, v, starts)
    out, bound, rows = R.attention(q, k, v, list(zip(at[:-1], at[1:])), dim ** -0.5)
    assert rows.all()
    R.assert_within(got, out, bound)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [1, 96])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_masked_values_at_every_tile_shape(w8a8, gpu, dim, heads, value):
    import torch
    import attention_ref as R
    q, k, v = (R.randn((900, h, dim), s, gpu) for s, h in ((1, heads), (2, 1), (3, 1)))
    starts = torch.tensor([0, 900], dtype=torch.int32, device=gpu)
    want = w8a8.attention(q, k, v, starts)
    for at in (0, 95, 127, 500, 899):
        w = v.clone()
        w[at, 0, 3] = value
        got = w8a8.attention(q, k, w, starts)
        assert torch.equal(got[:at], want[:at])
        assert not torch.isfinite(got[at:, :, 3]).any()
        others = [c for c in range(dim) if c != 3]
        assert torch.equal(got[..., others], want[..., others])
