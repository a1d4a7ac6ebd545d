"""Causal attention with infinite scores: a key whose score is -inf has no weight, wherever
it lies, and a row without any finite score is NaN."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("at", [0, 31, 32, 64, 100, 149])
def test_key_of_no_weight(w8a8, gpu, dim, at):
    # row `at` starts a wave's rows or ends them: its own key, the first it meets, is out
    import attention_ref as R
    import torch
    q, k, v = (R.randn((150, 1, dim), s, gpu) for s in (1, 2, 3))
    q[..., 5] = q[..., 5].abs() + 0.5
    starts = torch.tensor([0, 150], dtype=torch.int32, device=gpu)
    k[at, 0, 5] = -math.inf
    got = w8a8.attention(q, k, v, starts)
    # the same without the key: token `at` keeps its own row out of sight of all
    keep = torch.arange(150, device=gpu) != at
    s = (q[:, 0].double() @ torch.where(keep[:, None], k[:, 0], 0).double().t()) * dim ** -0.5
    s.masked_fill_(torch.ones_like(s, dtype=torch.bool).triu(1) | ~keep, -math.inf)
    serr = R.score_error(q[:, 0].double(), torch.where(keep[:, None], k[:, 0], 0).double(),
                         dim ** -0.5)
    first = 1 if at == 0 else 0  # token 0 sees nothing else
    out, bound = R.softmax_pv(s[first:], v[:, 0].double(), serr=serr)
    R.assert_within(got[first:, 0], out, bound)
    if at == 0:
        assert torch.isnan(got[0]).all()


def test_no_finite_score_and_plus_infinity(w8a8, gpu):
    import attention_ref as R
    import torch
    q, k, v = (R.randn((70, 2, 64), s, gpu) for s in (4, 5, 6))
    starts = torch.tensor([0, 70], dtype=torch.int32, device=gpu)
    want = w8a8.attention(q, k, v, starts)
    q[40, 1, 0] = math.inf  # scores of both signs: no softmax
    got = w8a8.attention(q, k, v, starts)
    assert torch.isnan(got[40, 1]).all()
    got[40, 1] = want[40, 1]
    assert torch.equal(got, want)
