"""Filters given as one value per row, before they reach the kernels (no GPU)."""
import pytest
import torch

from nerf_amd import ops

CPU = torch.device("cpu")


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_top_k_of_every_whole_type(dtype):
    info = torch.iinfo(dtype)
    k = torch.tensor([0, 1, 50, info.max, info.min], dtype=dtype)
    scalar, rows = ops._per_row(k, "top_k", torch.int32, k.shape, CPU)
    assert scalar == 0 and rows.dtype == torch.int32 and rows.is_contiguous()
    want = [0, 1, 50, min(info.max, 2 ** 31 - 1)]
    assert rows[:4].tolist() == want and int(rows[4]) <= 0               # 0 and less: all


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.bool, torch.complex64])
def test_top_k_that_is_not_a_count(dtype):
    with pytest.raises(TypeError, match="top_k: expected whole numbers"):
        ops._per_row(torch.ones(3, dtype=dtype), "top_k", torch.int32, torch.Size([3]), CPU)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.int64])
def test_other_filters_as_f32(dtype):
    _, rows = ops._per_row(torch.ones(3, dtype=dtype), "top_p", torch.float32, torch.Size([3]), CPU)
    assert rows.dtype == torch.float32 and rows.tolist() == [1.0] * 3
