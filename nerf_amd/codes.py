"""Learned codes: one vector per training image, video frame or hashed grid corner, looked up by index and trained with the
network (no counterpart in the reference, whose encodings are all fixed).

`CodeTable` stands beside `positional_encoding.Embedder`: `codes(ids)` -> [*ids.shape, dim], differentiable w.r.t. its rows.
render.run_network(..., codes=...) appends one code per ray to the direction channels; raybatch's samplers say which image
each ray of a batch comes from.  The kernels are nrf_lookup_fwd and nrf_lookup_bwd."""
import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops


class _LookupFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, padding_idx, out_dtype):
        ctx.save_for_backward(ids)
        ctx.cfg = (table.shape[0], scale, padding_idx, table.dtype)
        return ops.lookup_fwd(table, ids, scale, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (ids,) = ctx.saved_tensors
        n_rows, scale, padding_idx, dtype = ctx.cfg
        return ops.lookup_bwd(g, ids, n_rows, scale, padding_idx, dtype), None, None, None, None


def lookup(table, ids, scale=1.0, padding_idx=None, out_dtype=None):
    """scale * table[ids] with the gradient w.r.t. `table` (reverse mode; forward mode is refused); see ops.lookup_fwd / ops.lookup_bwd
    for types and shapes."""
    if forward_ad.unpack_dual(table).tangent is not None:       # the kernel's output would lose the tangent
        raise NotImplementedError("lookup: no forward-mode derivative (jvp)")
    if padding_idx is not None and not 0 <= padding_idx < table.shape[0]:
        raise ValueError(f"padding_idx {padding_idx} is outside the table's {table.shape[0]} rows")
    if table.requires_grad and torch.is_grad_enabled():
        return _LookupFunction.apply(table, ids, float(scale), padding_idx, out_dtype)
    return ops.lookup_fwd(table, ids, scale, out_dtype)


class CodeTable(nn.Module):
    """num_codes learned vectors of `dim` elements.  padding_idx: a row that starts at zero and receives no gradient."""

    def __init__(self, num_codes, dim, scale=1.0, padding_idx=None, init_std=0.01, dtype=torch.float32, out_dtype=None):
        super().__init__()
        if num_codes < 1 or dim < 1:
            raise ValueError(f"CodeTable needs at least one code of one element, got {num_codes} x {dim}")
        if padding_idx is not None and not 0 <= padding_idx < num_codes:
            raise ValueError(f"padding_idx {padding_idx} is outside the table's {num_codes} rows")
        self.num_codes, self.dim = int(num_codes), int(dim)
        self.scale, self.padding_idx, self.out_dtype = float(scale), padding_idx, out_dtype
        self.weight = nn.Parameter(torch.empty((num_codes, dim), dtype=dtype))
        nn.init.normal_(self.weight, std=init_std)
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].zero_()

    def forward(self, ids):
        return lookup(self.weight, ids, self.scale, self.padding_idx, self.out_dtype)

    def extra_repr(self):
        return f"{self.num_codes}, {self.dim}, scale={self.scale}, padding_idx={self.padding_idx}"
