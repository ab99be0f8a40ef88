"""Where top-p cuts long rows whose mass lies in very many very small entries.  The rows stand in falling order, so that u = 1 names the
last kept entry, the cut itself, and u = 0 the first, whose prob is 1 / (kept mass).

The host adds in 80 bits.  The device adds masses in f64 (sums taken in parts: some 2^-53 S, SUMS below with room) of which a histogram
holds each to 2^-42 or better (MASSES).  A cut is the same on both sides as long as no running sum of the host's lies so near to p S,
which every case asks for before it looks at the device's answer."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SUMS, MASSES = 2e-15, 2.0 ** -41
P32 = lambda p: float(np.float32(p))  # noqa: E731


def cut_of(x, p, t):
    """How many of the entries of a falling row top-p keeps, and their mass (host)."""
    run = np.cumsum(np.exp((x.astype(np.longdouble) - x[0]) / t))
    want = P32(p) * run[-1]
    n = 1 + int(np.searchsorted(run, want, side="left"))
    assert n < len(x) and min(run[n - 1] - want, want - run[n - 2] if n > 1 else 1) > (SUMS + MASSES) * run[-1]
    return n, float(run[n - 1])


def drawn_ends(x, p, t, rows=1, n=2):
    from nerf_amd import ops
    u = torch.zeros(rows, n, device="cuda")
    u[:, 1::2] = 1.0
    ids, prob = ops.sample_logits(x.reshape(1, -1).expand(rows, -1), n, t, 0, p, 0.0, u)
    assert (ids[:, ::2] == 0).all() and (ids[:, 1::2] == ids[:, 1:2]).all() and (ids[:, 1] == ids[0, 1]).all()
    return int(ids[0, 1]), float(prob[0, 0])


# rows: few (split over blocks), many (a block each); sizes: one word of the histogram holds the row, and more than that
@pytest.mark.parametrize("V,rows,t", [(640000, 1, 0.7), (640000, 200, 0.7), (1 << 22, 1, 0.7), (5000001, 1, 0.05), (1 << 22, 66, 0.7)])
def test_normal_rows(V, rows, t):
    x = -np.sort(-np.random.RandomState(V).normal(size=V).astype(np.float32) * np.float32(2.5 if t > 0.1 else 0.15))
    t = P32(t)
    for p in (0.9, 0.99, 0.9999, 0.999999):
        n, mass = cut_of(x, p, t)
        last, first = drawn_ends(torch.from_numpy(x).cuda(), p, t, rows)
        assert last == n - 1, (p, last, n - 1)
        assert abs(first * mass - 1.0) <= 2.0 ** -24 * 1.001


# One entry at 0, all others at `low`, in sizes at which the tail weighs some percent of the peak or less.  Kept are the peak and the
# others j with 1 + j e < p (1 + (V - 1) e): a closed form.
@pytest.mark.parametrize("V,rows,low,p", [
    (1 << 28, 1, -22.875, 0.99), (1 << 28, 1, -23.625, 0.99), ((1 << 26) + 11, 1, -19.0, 0.995), (1 << 24, 1, -26.0, 0.99995),
    (1 << 22, 1, -30.0, 0.9999999), (1 << 22, 3, -12.0, 0.6), (1 << 23, 70, -20.0, 0.995), (1000003, 1, -25.0, 0.99999),
    (1000003, 300, -25.0, 0.99999)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_peak_and_a_flat_tail(V, rows, low, p, dtype):
    x = torch.full((V,), low, device="cuda", dtype=dtype)
    x[0] = 0.0
    e = math.exp(low)
    others = (P32(p) * (1.0 + (V - 1) * e) - 1.0) / e
    # the sums' error in entries, and what an error of e does to the closed form: (1 - p) / e of it
    assert 0 < others < V - 1 and abs(others - round(others)) > (SUMS * (1.0 + V * e) + MASSES * (1.0 - p)) / e + 1e-3
    others = math.ceil(others)
    last, first = drawn_ends(x, p, 1.0, rows)
    assert last == others, (last, others)
    assert abs(first * (1.0 + others * e) - 1.0) <= 2.0 ** -24 * 1.001


@pytest.mark.parametrize("t", [1e-3, 0.02, 1.0])
def test_narrow_rows(t):
    """All values within a few temperatures of the largest, many times each."""
    V, t = 3000001, P32(t)
    steps = np.random.RandomState(3).randint(0, 200, V)
    x = -np.sort(steps).astype(np.float32) * np.float32(t * 0.05)
    x = -np.sort(-x)
    for p in (0.3, 0.9, 0.999):
        n, mass = cut_of(x, p, t)
        last, first = drawn_ends(torch.from_numpy(x).cuda(), p, t)
        assert last == n - 1, (p, last, n - 1)
        assert abs(first * mass - 1.0) <= 2.0 ** -24 * 1.001


@pytest.mark.parametrize("R,V", [(2, 5000), (1, 70001), (140, 70001)])
def test_temperatures_and_logits_at_the_ends_of_f32(R, V):
    """Bins without an order of mass (differences beyond f32's range), masses that underflow within a bin, and +inf."""
    from test_gpu_sample_logits import check
    rng = np.random.RandomState(V)
    u = torch.from_numpy(rng.rand(R, 4).astype(np.float32)).cuda()
    row = torch.from_numpy(rng.uniform(-3.0, 3.0, (1, V)).astype(np.float32)).cuda()
    wide = (row * 1e38).expand(R, V)
    for t in (3e38, 1e38, 4e36, 1.0):
        check(wide, u, t=t, p=0.9)
        check(wide, u, t=t, k=V // 2, p=0.7)
    for t in (1e-2, 1e-4, 1e-20, 1e-44):
        check(row.expand(R, V), u, t=t, p=0.9)
        check(row.expand(R, V), u, t=t, k=V // 2, p=0.999)
    inf = row.clone()
    inf[0, ::2] = math.inf
    for f in (dict(p=0.9), dict(k=V // 3, p=0.3), dict(k=V - 5), dict(p=0.0)):
        check(inf.expand(R, V), u, t=0.7, **f)
