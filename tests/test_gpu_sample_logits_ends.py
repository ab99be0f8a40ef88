"""The last thing that can be drawn: u = 1 (and what is clamped to it) names the last kept entry that has mass, wherever the row's
masses end.  Indices have to equal those of test_gpu_sample_logits' reference (f64, host).  prob is rounded once to f32: half a step is
2^-24 of a value in the normal range and 2^-150 (half of the least denormal) below it, where the small ends of these rows lie."""
import numpy as np
import pytest
import torch

from test_gpu_sample_logits import reference

pytestmark = pytest.mark.gpu

ENDS = [1.0, 2.0, float("inf"), 1.0 - 2.0 ** -24, 0.5, 0.0]


def check(x, u, t=1.0, k=0, p=1.0, m=0.0):
    from nerf_amd import ops
    ids, prob = ops.sample_logits(x, u.shape[-1], t, k, p, m, u)
    t, p, m = (float(np.float32(v)) for v in (t, p, m))
    xs, us, ids, prob = x.double().cpu().numpy(), u.cpu().numpy(), ids.cpu().numpy(), prob.double().cpu().numpy()
    for r in range(x.shape[0]):
        ri, rp = reference(xs[r], us[r], t, k, p, m)
        assert (ids[r] == ri).all(), (r, ids[r][ids[r] != ri], ri[ids[r] != ri], us[r][ids[r] != ri])
        assert (np.abs(prob[r] - rp) <= rp * 2.0 ** -24 * 1.001 + 2.0 ** -150).all(), (r, np.abs(prob[r] - rp).max())


def rows_with_empty_ends(R, V, rng):
    """Normal rows whose last tiles of 1024 entries are masked, some of the tiles before them too; row 0 ends with one tiny mass."""
    x = rng.normal(size=(R, V)).astype(np.float32) * 2.5
    for r in range(R):
        end = V - int(rng.randint(1, V // 2048 + 1)) * 1024 - int(rng.randint(1024))
        x[r, end:] = -np.inf
        for q in rng.randint(0, max(1, end // 1024), 5):
            x[r, q * 1024:(q + 1) * 1024] = -np.inf
    x[0, V - 3000:] = -np.inf
    x[0, V - 3000] = x[0].max() - 60.0                   # 1e-26 of the largest: no running sum moves by it
    return x


# both forms of long rows, with many draws and with few (split: 640000 and 150000; a block a row: 40000 and 20011)
@pytest.mark.parametrize("R,V,n", [(1, 640000, 6), (3, 640000, 30), (2, 150000, 500), (200, 40000, 6), (100, 20011, 40)])
def test_rows_whose_last_tiles_hold_nothing(R, V, n):
    rng = np.random.RandomState(V + n)
    x = torch.from_numpy(rows_with_empty_ends(R, V, rng)).cuda()
    u = rng.rand(R, n).astype(np.float32)
    u[:, :6] = ENDS
    u = torch.from_numpy(u).cuda()
    for f in (dict(), dict(t=0.3), dict(m=1e-3), dict(p=0.999, t=2.0)):
        check(x, u, **f)
        check(x.bfloat16(), u, **f)


@pytest.mark.parametrize("R,V,n", [(1, 640000, 6), (2, 150000, 500), (200, 40000, 6)])
def test_tiles_that_top_p_cuts_away(R, V, n):
    """Large logits first, small ones behind: whole tiles at the end are cut, or have less mass than min_p asks for."""
    rng = np.random.RandomState(V)
    x = rng.normal(size=(R, V)).astype(np.float32)
    x[:, V // 3:] -= 9.0
    x = torch.from_numpy(x).cuda()
    u = rng.rand(R, n).astype(np.float32)
    u[:, :6] = ENDS
    u = torch.from_numpy(u).cuda()
    for f in (dict(p=0.9), dict(p=0.99, t=1.3), dict(k=V // 4), dict(m=1e-4)):
        check(x, u, **f)


@pytest.mark.parametrize("V", [1, 63, 700, 1500, 2048, 3000])
def test_the_end_of_short_rows_and_of_lists(V):
    rng = np.random.RandomState(V)
    x = rng.normal(size=(30, V)).astype(np.float32) * 2.5
    x[1::2, V - V // 3:] = -np.inf
    x = torch.from_numpy(x).cuda()
    u = torch.tensor([ENDS] * 30).cuda()
    for f in (dict(), dict(k=200), dict(p=0.9), dict(m=0.02), dict(k=1000, p=0.99, m=1e-3)):
        check(x, u, **f)


@pytest.mark.parametrize("R,V,n", [(6, 5, 3), (6, 700, 3), (6, 1500, 17), (6, 2048, 3), (6, 4483, 3), (200, 40000, 3), (2, 150000, 30)])
def test_the_first_entry_with_mass_however_small(R, V, n):
    """u = 0: a mass far below a rounding of the sums, at the row's first entry, with the largest close behind it or far."""
    rng = np.random.RandomState(V)
    u = rng.rand(R, n).astype(np.float32)
    u[:, :2] = [0.0, -1.0]
    u = torch.from_numpy(u).cuda()
    for down in (40.0, 300.0, 650.0):
        x = rng.uniform(-900.0, -800.0, (R, V)).astype(np.float32)       # no mass at all
        for r in range(R):
            peak = int(rng.randint(1, V)) if r % 3 == 2 else 1 + r % min(V - 1, 4)
            x[r, peak] = 0.0
            x[r, int(rng.randint(0, peak))] = -down
        for f in (dict(), dict(k=2), dict(k=5), dict(k=V // 2), dict(k=min(V, 300))):
            check(torch.from_numpy(x).cuda(), u, **f)


@pytest.mark.parametrize("V", [12, 700, 3000])
@pytest.mark.parametrize("L", [2, 3, 4, 5, 8, 12])
def test_lists_that_begin_with_a_small_mass(V, L):
    """All places of a small mass and the largest in a list of L entries, the others without mass."""
    pairs = [(i, j) for j in range(1, L) for i in range(j)]
    x = np.full((len(pairs), V), -900.0, np.float32)
    x[:, :L] = -800.0
    for r, (i, j) in enumerate(pairs):
        x[r, i], x[r, j] = -200.0 - r, 0.0
    u = torch.tensor([[0.0, -3.0, 2.0 ** -24, 0.5, 1.0]] * len(pairs)).cuda()
    check(torch.from_numpy(x).cuda(), u, k=L)
