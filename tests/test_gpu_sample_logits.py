"""nrf_sample_logits against the definition in 64 bits on the host.  Indices have to be equal: both sides carry masses and running
sums in f64, whose roundings (1e-15 of a sum) are met by a random u with a probability below 1e-9 a draw.  prob is rounded once to
f32 (2^-24), from masses whose error is far below that."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def reference(x, u, t, k, p, m):
    """One row in f64: (ids, prob)."""
    n = len(u)
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any() or not np.isfinite(t) or t < 0 or np.isnan(p) or np.isnan(m):
        return np.full(n, -1), np.zeros(n)
    order = np.lexsort((np.arange(len(x)), -x))
    z = x[order]
    with np.errstate(all="ignore"):
        e = np.where(z == z[0], 1.0, np.exp((z - z[0]) / t) if t > 0 else 0.0)
    keep = len(x) if k <= 0 else min(k, len(x))
    if t == 0:
        keep = 1
    e = e[:keep]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(e)[:-1]])
        e = e[:max(1, int(np.sum(before < p * np.sum(e))))]
    e = e * (e >= min(m, 1.0))
    full = np.zeros(len(x))
    full[order[:len(e)]] = e
    cum = np.cumsum(full)
    uc = np.clip(np.where(np.isnan(u), 0, u).astype(np.float64), 0, 1)
    ids = np.searchsorted(cum, uc * cum[-1], side="right")
    ids = np.minimum(ids, np.nonzero(full)[0][-1])
    prob = full[ids] / cum[-1]
    return np.where(np.isnan(u), -1, ids), np.where(np.isnan(u), 0, prob)


def check(x, u, got=None, t=1.0, k=0, p=1.0, m=0.0):
    """x [R, V], u [R, n] GPU tensors; filters: numbers or per-row tensors."""
    from nerf_amd import ops
    ids, prob = got if got is not None else ops.sample_logits(x, u.shape[-1], t, k, p, m, u)
    assert ids.dtype == torch.int64 and prob.dtype == torch.float32 and ids.shape == prob.shape == u.shape
    xs, us, ids, prob = x.double().cpu().numpy(), u.cpu().numpy(), ids.cpu().numpy(), prob.cpu().numpy()
    row = lambda v, r: float(v[r]) if torch.is_tensor(v) else float(np.float32(v))  # noqa: E731
    for r in range(x.shape[0]):
        ri, rp = reference(xs[r], us[r], row(t, r), int(row(k, r)), row(p, r), row(m, r))
        bad = np.nonzero(ids[r] != ri)[0]
        assert not len(bad), (r, bad[:5], ids[r][bad[:5]], ri[bad[:5]], us[r][bad[:5]])
        assert (np.abs(prob[r] - rp) <= rp * 2.0 ** -24 * 1.001).all(), (r, np.abs(prob[r] - rp).max())


def make(kind, R, V, rng):
    x = rng.normal(size=(R, V)).astype(np.float32) * 2.5
    if kind == "errors":
        x = np.log((x * 0.04) ** 2 + 1e-6).astype(np.float32)
    elif kind == "ties":
        x = np.round(x)                                                  # a dozen values
    elif kind == "flat":
        x[:] = 0.25
    elif kind == "two":
        x = (x > 1.0).astype(np.float32) * 3.0 - 1.0
    elif kind == "masked":
        x[rng.rand(R, V) < 0.9] = -np.inf
        x[0] = -np.inf                                                   # nothing left
        x[-1, rng.randint(V)] = np.nan
    elif kind == "outlier":
        x[:, V // 2] = 3e38
        x[:, V // 3] = -3e38
        x[:, V // 4] = 2.9e38
    elif kind == "narrow":
        x = (1.0 + rng.randint(0, 1 << 20, (R, V)) * 2.0 ** -23).astype(np.float32)   # within one step of the first histogram
    return torch.from_numpy(np.ascontiguousarray(x, np.float32))


FILTERS = [dict(), dict(k=1), dict(k=40), dict(p=0.9), dict(m=0.05), dict(k=3000, p=0.95), dict(t=0.0), dict(t=0.25, k=100, p=0.5, m=0.1),
           dict(p=0.0), dict(t=1e-3), dict(t=30.0, p=0.999), dict(k=2500), dict(k=2500, p=0.9999, m=1e-4, t=3.0)]


@pytest.mark.parametrize("kind", ["normal", "errors", "ties", "flat", "two", "masked", "outlier", "narrow"])
@pytest.mark.parametrize("R,V", [(3, 1), (5, 2), (9, 65), (4, 1001), (3, 2048), (3, 2049), (2, 20011)])
def test_filters(kind, R, V):
    rng = np.random.RandomState(V)
    x = make(kind, R, V, rng).cuda()
    for f in FILTERS:
        u = torch.from_numpy(rng.rand(R, 5).astype(np.float32)).cuda()
        check(x, u, **f)


@pytest.mark.parametrize("kind", ["normal", "errors", "flat", "two", "masked", "outlier", "narrow"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("R,V,n", [(1, 131072, 1), (2, 100003, 40), (18, 65537, 3), (200, 4099, 2), (3, 2500, 300), (70, 30000, 20), (3, 65536, 2), (6, 131072, 1)])
def test_long_rows(kind, dtype, R, V, n):
    rng = np.random.RandomState(V + n)
    x = make(kind, R, V, rng)
    if dtype == "f16":
        x = x.clamp(-6e4, 6e4)
    x = x.to(TYPES[dtype]).cuda()
    for f in (dict(), dict(k=50, p=0.9, m=0.02, t=0.8), dict(p=0.97, t=0.5), dict(k=3000, p=0.9, t=2.0), dict(t=0.0)):
        u = torch.from_numpy(rng.rand(R, n).astype(np.float32)).cuda()
        check(x, u, **f)


@pytest.mark.parametrize("R,V,n", [(1, 640000, 4096), (20, 40000, 300)])
def test_an_error_map_and_many_draws(R, V, n):
    rng = np.random.RandomState(1)
    x = make("errors", R, V, rng).cuda()
    u = torch.from_numpy(rng.rand(R, n).astype(np.float32)).cuda()
    for f in (dict(t=0.5, p=0.95), dict(), dict(m=0.01), dict(k=V // 3)):
        check(x, u, **f)


def test_top_k_of_rows_that_hold_fewer():
    """Masks that leave fewer entries than k: none, one, fewer and more than the list; both forms of long rows."""
    rng = np.random.RandomState(6)
    for V, rows in ((16550, 7), (140000, 3), (140000, 7)):
        x = rng.normal(size=(rows, V)).astype(np.float32) * 2.5
        for r, left in enumerate((1, 0, 300, 1200, 2048, 2049, 5000)[:rows]):
            x[r, rng.permutation(V)[left:]] = -np.inf
        for k, n in ((536, 70), (1500, 3), (1400, 1)):
            u = torch.from_numpy(rng.rand(rows, n).astype(np.float32)).cuda()
            check(torch.from_numpy(x).cuda(), u, k=k, t=0.7)
            check(torch.from_numpy(x).cuda().half(), u, k=k, p=0.9)


def test_filters_of_each_row():
    rng = np.random.RandomState(4)
    for R, V in ((40, 700), (40, 5000)):
        x = make("normal", R, V, rng).cuda()
        col = lambda v, t=torch.float32: torch.tensor(v, dtype=t).cuda()  # noqa: E731
        t, p, m = rng.rand(R) * 2, rng.rand(R) * 1.2, rng.rand(R) * 0.2
        k = rng.randint(-3, V + 10, R)
        t[0], t[1], t[2], t[3] = 0.0, -1.0, np.inf, np.nan
        p[4], p[5], m[6], m[7] = np.nan, -0.5, np.nan, 7.0
        u = torch.from_numpy(rng.rand(R, 6).astype(np.float32)).cuda()
        check(x, u, t=col(t), k=col(k, torch.int64), p=col(p), m=col(m))
        check(x, u, t=col(t), k=5, p=0.7, m=col(m))


def test_numbers_at_the_ends_and_values_that_are_not_finite():
    from nerf_amd import ops
    for V in (7, 3000):
        x = torch.zeros(2, V).cuda()
        x[0, 1] = x[0, V - 2] = float("inf")
        x[1, 0] = x[1, V - 1] = -float("inf")
        x[1, 3] = float("nan")
        u = torch.tensor([[0.0, 1.0, 0.49999, 0.5, -1.0, 2.0, float("nan")]] * 2).cuda()
        for f in (dict(), dict(p=0.9), dict(k=2), dict(t=0.0)):
            check(x, u, **f)
        ids, prob = ops.sample_logits(x, 7, u=u)
        assert ids[0].tolist() == [1, V - 2, 1, V - 2, 1, V - 2, -1] and prob[0].tolist() == [0.5] * 6 + [0.0]
        assert ids[1, 0] == 1 and ids[1, 1] == V - 2                     # the masked ends are never drawn


def test_shapes_and_strides():
    from nerf_amd import ops
    rng = np.random.RandomState(6)
    base = make("normal", 12, 4003, rng).cuda()
    u = torch.from_numpy(rng.rand(12, 3).astype(np.float32)).cuda()
    check(base[:, 1:2999], u, k=30)
    check(base.t()[:12].contiguous().t()[:12], u, p=0.8)                 # column stride 12
    check(base[:1].expand(12, 4003), u)                                  # one row for all
    three = base.reshape(3, 4, 4003)
    ids, prob = ops.sample_logits(three, 3, 0.7, torch.full((3, 4), 20).cuda(), 0.9, u=u.reshape(3, 4, 3))
    check(base, u, got=(ids.reshape(12, 3), prob.reshape(12, 3)), t=0.7, k=20, p=0.9)
    one = ops.sample_logits(base[0], 3, u=u[0])
    check(base[:1], u[:1], got=(one[0][None], one[1][None]))
    assert ops.sample_logits(base[:0], 3)[0].shape == (0, 3) and ops.sample_logits(base, 0)[0].shape == (12, 0)
    ids, prob = ops.sample_logits(base, 1000)                            # numbers of its own
    assert int(ids.min()) >= 0 and int(ids.max()) < 4003 and float(prob.min()) > 0


def test_refusals():
    from nerf_amd import ops
    x = torch.zeros(4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="temperature"):
        ops.sample_logits(x, 1, temperature=-1.0)
    with pytest.raises(RuntimeError, match="temperature"):
        ops.sample_logits(x, 1, temperature=float("inf"))
    with pytest.raises(RuntimeError, match="min_p"):
        ops.sample_logits(x, 1, min_p=1.5)
    with pytest.raises(RuntimeError, match="top_p"):
        ops.sample_logits(x, 1, top_p=float("nan"))
    with pytest.raises(ValueError, match="one value per row"):
        ops.sample_logits(x, 1, top_p=torch.ones(3, device="cuda"))
    with pytest.raises(RuntimeError, match="expected a tensor on"):
        ops.sample_logits(x, 1, top_p=torch.ones(4))
    with pytest.raises(ValueError, match="u: expected"):
        ops.sample_logits(x, 2, u=torch.zeros(4, 1, device="cuda"))
    with pytest.raises(TypeError, match="float32"):
        ops.sample_logits(x.double(), 1)
    with pytest.raises(ValueError, match="V >= 1"):
        ops.sample_logits(x[:, :0], 1)


def test_another_stream_and_captured_graphs():
    from nerf_amd import ops
    rng = np.random.RandomState(9)
    cases = [(make("normal", 6, 50000, rng).cuda(), torch.rand(6, 3, device="cuda"), dict(top_k=60, top_p=0.9)),
             (make("errors", 1, 300000, rng).cuda(), torch.rand(1, 500, device="cuda"), dict(top_p=0.9)),
             (make("normal", 300, 900, rng).cuda(), torch.rand(300, 2, device="cuda"), dict(min_p=0.1))]
    for x, u, f in cases:
        run = lambda: ops.sample_logits(x, u.shape[1], u=u, **f)  # noqa: E731,B023
        want = run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = run()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                res = run()
            graphs.append((g, res))
        for _ in range(3):
            u.copy_(torch.rand_like(u))
            x.copy_(x.roll(1, -1))
            for g, _ in graphs:
                g.replay()
            torch.cuda.synchronize()
            want = run()
            for _, res in graphs:
                assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])


def test_rows_far_apart_and_odd_addresses():
    """Row offsets beyond 2^31 elements; 16-bit rows that begin at odd elements."""
    from nerf_amd import ops
    rng = np.random.RandomState(11)
    base = torch.zeros(2 ** 31 + 80000, dtype=torch.bfloat16, device="cuda")
    for V in (900, 5000, 70001):
        x = base.as_strided((3, V), (2 ** 30, 1), 3)
        x.copy_(make("normal", 3, V, rng).bfloat16())
        u = torch.from_numpy(rng.rand(3, 4).astype(np.float32)).cuda()
        for f in (dict(), dict(k=20, p=0.9), dict(p=0.8)):
            check(x, u, **f)
    del base
    x = make("normal", 3, 3001, rng).half().cuda()[:, 1:]
    check(x, torch.rand(3, 5, device="cuda"), k=9)
    check(x[:, :1001], torch.rand(3, 5, device="cuda"))


def test_values_near_the_ends_of_the_range():
    from nerf_amd import ops
    rng = np.random.RandomState(13)
    tiny = torch.from_numpy((rng.randint(-400, 400, (4, 3000)) * 1.4e-45).astype(np.float32)).cuda()     # denormal logits
    u = torch.from_numpy(rng.rand(4, 6).astype(np.float32)).cuda()
    for f in (dict(), dict(k=7), dict(p=0.5), dict(t=1e-38, k=2000), dict(t=1e-38, p=0.9)):
        check(tiny, u, **f)
        check(tiny[:, :900], u, **f)
    zeros = torch.zeros(2, 2500, device="cuda")
    zeros[:, ::2] = -0.0                                                 # equal values, whatever their sign
    check(zeros, u[:2], k=100)
    check(zeros, u[:2], t=0.0)
    assert ops.sample_logits(zeros, 1, temperature=0.0)[0].tolist() == [[0], [0]]


def test_top_k_among_equal_values_and_many_draws():
    """The groups' bound lets every entry through: the histogram and the first k by index."""
    rng = np.random.RandomState(14)
    x = torch.full((1, 70001), 0.5, device="cuda")
    x[0, 60000:] = 0.25
    for n in (3, 700):
        u = torch.from_numpy(rng.rand(1, n).astype(np.float32)).cuda()
        for f in (dict(k=50), dict(k=1400, p=0.7), dict(k=60500), dict(k=60500, p=0.999)):
            check(x, u, **f)
