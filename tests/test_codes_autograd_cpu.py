"""What codes.lookup does about derivatives and the padding row that it does not offer, with a plain lookup in the kernel's place (no GPU)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from nerf_amd import codes, ops


@pytest.fixture
def plain(monkeypatch):
    """Like the kernel, the stand-in makes a tensor that autograd knows nothing of."""
    def lookup_fwd(table, ids, scale=1.0, out_dtype=None):
        with torch.no_grad():
            return fwd_ad.unpack_dual(table).primal.detach()[ids] * scale

    def lookup_bwd(g, ids, n_rows, scale=1.0, padding_idx=None, dtype=None):
        out = torch.zeros(n_rows, g.shape[-1]).index_add_(0, ids, g * scale)
        if padding_idx is not None:
            out[padding_idx] = 0
        return out
    monkeypatch.setattr(ops, "lookup_fwd", lookup_fwd)
    monkeypatch.setattr(ops, "lookup_bwd", lookup_bwd)


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_derivatives_are_refused(plain, requires_grad):
    table, ids = torch.randn(5, 3, requires_grad=requires_grad), torch.tensor([1, 4])
    with fwd_ad.dual_level():
        dual = fwd_ad.make_dual(table, torch.ones(5, 3))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError), match="forward|jvp"):
                codes.lookup(dual, ids)


def test_reverse_mode_and_none(plain):
    table, ids = torch.randn(5, 3, requires_grad=True), torch.tensor([1, 4, 4])
    out = codes.lookup(table, ids, 2.0, padding_idx=1)
    out.sum().backward()
    assert torch.equal(out, 2.0 * table[ids]) and table.grad.tolist() == [[0.0] * 3] * 4 + [[4.0] * 3]
    with torch.no_grad():
        assert not codes.lookup(table, ids).requires_grad
    assert not codes.lookup(table.detach(), ids).requires_grad
    with fwd_ad.dual_level():                                   # a level alone makes no table a dual one
        assert torch.equal(codes.lookup(table, ids), table[ids])


@pytest.mark.parametrize("padding_idx", [5, -1, 1 << 40])
@pytest.mark.parametrize("grad", [False, True])
def test_a_padding_row_outside_the_table_is_refused_before_the_backward_pass(plain, padding_idx, grad):
    with pytest.raises(ValueError, match="outside the table's 5 rows"):
        codes.lookup(torch.randn(5, 3, requires_grad=grad), torch.tensor([1]), padding_idx=padding_idx)
