"""Sizes that do not fit the 32-bit arguments of the C entry points are refused, not taken modulo 2^32 (tensors without storage; no GPU)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from nerf_amd import ops

BIG = [2 ** 31, 2 ** 32 + 5]


@pytest.mark.parametrize("size", BIG)
def test_sample_logits(size):
    with FakeTensorMode():
        u = torch.empty((1, 1), device="cuda")
        with pytest.raises(ValueError, match=f"logits: rows of {size}"):
            ops.sample_logits(torch.empty((1, size), dtype=torch.bfloat16, device="cuda"), 1, u=u)
        with pytest.raises(ValueError, match=f"n_samples: {size}"):
            ops.sample_logits(torch.empty((1, 100), device="cuda"), size, u=u.expand(1, size))


@pytest.mark.parametrize("size", BIG)
def test_lookup(size):
    with FakeTensorMode():
        ids = torch.empty((1,), dtype=torch.int64, device="cuda")
        wide = torch.empty((1, size), dtype=torch.bfloat16, device="cuda")
        with pytest.raises(ValueError, match=f"table: rows of {size}"):
            ops.lookup_fwd(wide, ids)
        with pytest.raises(ValueError, match=f"g_out: rows of {size}"):
            ops.lookup_bwd(wide, ids, 4)
