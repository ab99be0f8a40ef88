"""What nrf_sample_logits and its wrapper refuse, before anything is launched (no GPU)."""
import ctypes as C

import pytest
import torch

from nerf_amd import _lib

NULL = C.c_void_p(0)
P = C.c_void_p(4096)          # never read: every call below is refused first


def call(logits=P, stride=100, dtype=0, rows=4, size=100, draws=2, t=1.0, k=0, p=1.0, m=0.0, tv=NULL, kv=NULL, pv=NULL, mv=NULL, u=P,
         ids=P, prob=P, ws=P):
    return _lib.lib().nrf_sample_logits(logits, stride, dtype, rows, size, draws, t, k, p, m, tv, kv, pv, mv, u, ids, prob, ws, NULL)


@pytest.mark.parametrize("kw,code,text", [
    (dict(logits=NULL), 1, "null"), (dict(u=NULL), 1, "null"), (dict(ids=NULL), 1, "null"), (dict(prob=NULL), 1, "null"),
    (dict(dtype=3), 1, "dtype"), (dict(rows=-1), 1, "n_rows"), (dict(size=0), 1, "size 0"), (dict(draws=-1), 1, "n_draws"),
    (dict(stride=-1), 1, "stride"), (dict(t=-0.5), 1, "temperature"), (dict(t=float("inf")), 1, "temperature"),
    (dict(t=float("nan")), 1, "temperature"), (dict(p=float("nan")), 1, "top_p"), (dict(m=1.5), 1, "min_p"),
    (dict(m=float("nan")), 1, "min_p"), (dict(size=2 ** 28 + 1), 2, "2^28"), (dict(rows=2 ** 21 + 1), 2, "2^21"),
    (dict(rows=2 ** 20, draws=2 ** 11), 2, "2^31"), (dict(size=70000, ws=NULL), 1, "workspace"),
    (dict(size=70000, ws=C.c_void_p(4100)), 1, "aligned"),
])
def test_refusals(kw, code, text):
    assert call(**kw) == code
    assert text in _lib.lib().nrf_last_error_string().decode()


def test_nothing_to_draw_launches_nothing():
    assert call(rows=0, logits=NULL) == 0
    assert call(draws=0, ids=NULL) == 0


def test_python_refuses_cpu_tensors():
    from nerf_amd.sampling import sample_logits
    with pytest.raises(RuntimeError, match="GPU tensor"):
        sample_logits(torch.zeros(2, 5))
    with pytest.raises(TypeError, match="torch.Tensor"):
        sample_logits([0.0])


def test_workspace_sizes():
    f = _lib.lib().nrf_sample_logits_workspace_bytes
    assert f(1, 2048, 1) == 0 and f(4096, 131072, 1) == 0 and f(0, 70000, 1) == 0 and f(-1, 70000, 1) == 0
    assert f(2, 70000, 1) == 2 * f(1, 640000, 1) == 2 * f(1, 3000, 500) > 0 and f(1, 70000, 1) % 16 == 0
