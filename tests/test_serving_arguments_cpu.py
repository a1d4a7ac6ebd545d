"""Shapes and strides that the Python calls of attention, the 4-bit cache and the expert
layer of few tokens refuse before anything is launched (their checks need no GPU)."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import optimized_rocwmma_samples_amd as W  # noqa: E402


@pytest.fixture(autouse=True)
def _loaded():
    W._torch()


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def test_row_strides():
    assert W._heads3d("q", half(5, 4, 64)) == 256
    assert W._heads3d("q", half(5, 640)[:, :256].unflatten(1, (4, 64))) == 640
    # one row: whatever stride it carries
    assert W._heads3d("q", half(9, 4, 64)[::9]) == 256
    assert W._heads3d("q", half(1, 64)[:, None].expand(1, 1, 64)) == 64
    assert W._row_stride("x", 1, 0, 64) == 64 and W._row_stride("x", 2, 80, 64) == 80


@pytest.mark.parametrize("t", [half(1, 2, 64).expand(3, 2, 64),            # stride 0
                               half(4 * 128 + 64).as_strided((4, 2, 64), (64, 64, 1))])
def test_overlapping_rows(t):
    with pytest.raises(ValueError, match="overlap"):
        W._heads3d("k", t)


def test_overlapping_rows_2d():
    with pytest.raises(ValueError, match="overlap"):
        W._row_stride("x", 3, 0, 64)


@pytest.mark.parametrize("t", [half(5, 64), half(5, 4, 64).float(), half(5, 64, 4).transpose(1, 2),
                               half(4, 5, 64).transpose(0, 1), half(5, 4, 128)[..., ::2]])
def test_layouts(t):
    with pytest.raises(ValueError):
        W._heads3d("q", t)


def test_workspaces():
    W._workspace_on("auto", torch.device("cpu"))
    W._workspace_on(None, torch.device("cpu"))
    W._workspace_on(torch.zeros(8), torch.device("cpu"))
    with pytest.raises(ValueError, match="contiguous"):
        W._workspace_on(torch.zeros(8)[::2], torch.device("cpu"))
    with pytest.raises(ValueError, match="device tensors"):
        W._workspace_on(torch.zeros(8), torch.device("meta"))


def test_row_strides_past_32_bits():
    # the library takes strides in 32 bits: 2^32 + 256 must not become 256
    far = 2 ** 32 + 256
    t = torch.empty_strided((2, 4, 64), (far, 64, 1), dtype=torch.float16, device="meta")
    with pytest.raises(ValueError, match="row stride"):
        W._heads3d("k", t)
    with pytest.raises(ValueError, match="row stride"):
        W._row_stride("block_table", 2, 2 ** 32 + 16, 16)
    assert W._row_stride("x", 2, 2 ** 32 - 8, 256) == 2 ** 32 - 8
    assert W._row_stride("x", 1, far, 256) == 256  # one row: never read


@pytest.mark.parametrize("dim,group", [(128, 48), (128, 100), (64, 128), (64, 0), (96, 64)])
def test_cache_groups_that_do_not_divide_the_head(dim, group):
    # 128 channels in groups of 48 are not two groups of 64
    with pytest.raises(ValueError, match="group"):
        W.KV4Cache.empty(2, 2, dim, 16, group, device="meta")
