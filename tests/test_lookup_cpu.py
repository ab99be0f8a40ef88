"""Code tables without a GPU: what nrf_lookup_* and their wrappers refuse, before anything is launched."""
import ctypes as C

import pytest
import torch

from nerf_amd import _lib

NULL = C.c_void_p(0)
P = C.c_void_p(4096)          # never read: every call below is refused first


def msg():
    return _lib.lib().nrf_last_error_string().decode()


def fwd(table=P, stride=8, dtype=0, n_rows=4, dim=8, ids=P, i64=1, n=3, out=P, out_dtype=0):
    return _lib.lib().nrf_lookup_fwd(table, stride, dtype, n_rows, dim, ids, i64, n, 1.0, out, out_dtype, NULL)


def bwd(g=P, stride=8, g_dtype=0, ids=P, n=3, n_rows=4, dim=8, pad=-1, grad=P, dtype=0, ws=P):
    return _lib.lib().nrf_lookup_bwd(g, stride, g_dtype, ids, 1, n, n_rows, dim, 1.0, pad, grad, dtype, ws, NULL)


@pytest.mark.parametrize("kw,code,text", [
    (dict(table=NULL), 1, "null"), (dict(ids=NULL), 1, "null"), (dict(out=NULL), 1, "null"),
    (dict(stride=7), 1, "stride"), (dict(dim=0), 1, "dim"), (dict(n=-1), 1, "n -1"), (dict(n_rows=-1), 1, "n_rows"),
    (dict(dtype=3), 1, "dtype"), (dict(out_dtype=-1), 1, "dtype"),
    (dict(dtype=1, out_dtype=2), 2, "type"), (dict(dtype=0, out_dtype=1), 2, "type"),
    (dict(dim=32769, stride=32769), 2, "dim at most"), (dict(n=2 ** 31), 2, "2^31"), (dict(n_rows=2 ** 31), 2, "2^31"),
    (dict(n=2 ** 30, dim=8), 2, "2^33"),
])
def test_forward_refusals(kw, code, text):
    assert fwd(**kw) == code
    assert text in msg()


@pytest.mark.parametrize("kw,code,text", [
    (dict(g=NULL), 1, "null"), (dict(ids=NULL), 1, "null"), (dict(grad=NULL), 1, "null"), (dict(ws=NULL, n=100000), 1, "null"),
    (dict(ws=C.c_void_p(4097)), 1, "aligned"), (dict(stride=7), 1, "stride"), (dict(dim=0), 1, "dim"), (dict(n=-1), 1, "n -1"),
    (dict(dtype=1, g_dtype=2), 2, "type"), (dict(dtype=0, g_dtype=1), 2, "type"), (dict(dtype=9), 1, "dtype"),
    (dict(dim=32769, stride=32769), 2, "dim at most"), (dict(n=2 ** 31), 2, "2^31"), (dict(n_rows=2 ** 31 - 1), 2, "2^31"),
    (dict(n_rows=2 ** 30), 2, "n_rows * dim"),
])
def test_gradient_refusals(kw, code, text):
    assert bwd(**kw) == code
    assert text in msg()


def test_nothing_to_do_launches_nothing():
    assert fwd(n=0, ids=NULL, out=NULL, table=NULL) == 0
    assert bwd(n_rows=0, grad=NULL) == 0


def test_workspace_sizes():
    f = _lib.lib().nrf_lookup_bwd_workspace_bytes
    assert f(0, 10, 4) >= 0 and f(4096, 5000, 32) == f(16384, 5000, 32) == 0         # up to 16384 tokens: no sort, no workspace
    assert f(-1, 10, 4) == -1 and f(10, 10, 0) == -1 and f(10, 10, 32769) == -1 and f(2 ** 31, 10, 1) == -1
    # pairs of (id, position), twice for more than one pass, and two partial sums a tile: within a small multiple of the input
    for n, rows, dim in ((17000, 5000, 32), (9000, 50000, 300), (786432, 200, 33), (2097152, 524288, 2), (16384, 131072, 4096)):
        assert n * 8 <= f(n, rows, dim) <= n * 24 + n * dim * 4 + (1 << 24)


def test_python_refusals():
    from nerf_amd import ops
    from nerf_amd.codes import CodeTable
    ids = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.lookup_fwd(torch.zeros(4, 8), ids)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.lookup_bwd(torch.zeros(3, 8), ids, 4)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        CodeTable(4, 8)(ids)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.lookup_fwd([[0.0]], ids)
    for bad in (dict(num_codes=0, dim=4), dict(num_codes=4, dim=0), dict(num_codes=4, dim=4, padding_idx=4),
                dict(num_codes=4, dim=4, padding_idx=-1)):
        with pytest.raises(ValueError):
            CodeTable(**bad)
