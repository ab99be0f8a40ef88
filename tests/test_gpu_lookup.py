"""Code tables: nrf_lookup_fwd / nrf_lookup_bwd (ops, codes.CodeTable) against the formulas in 64 bits.

Tolerances count roundings.  Forward: one f32 product (2^-24) and one rounding to the output type (half a step).  Gradient: a
sum of n terms in f32 in any order is off by at most (n - 1) 2^-24 sum|g| to first order; n 2^-24 bounds that with the scale's
product; then half a step of the table's type.  f16 results below its normal range are off by at most half of 2^-24."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def half_step(t):
    return torch.finfo(t).eps / 2


def make_ids(kind, n, V, rng):
    if kind == "one":
        ids = np.full(n, V // 2)
    elif kind == "runs":
        ids = np.repeat(rng.randint(0, V, n // 192 + 1), 192)[:n]
    elif kind == "zipf":
        ids = np.minimum(np.exp(rng.rand(n) * np.log(V + 1.0)).astype(np.int64) - 1, V - 1)
    elif kind == "sorted":
        ids = np.sort(rng.randint(0, V, n))
    else:
        ids = rng.randint(0, V, n)
    return torch.from_numpy(ids.astype(np.int64))


def check_fwd(table, ids, scale, out):
    V = table.shape[0]
    want = table.double().cpu()[ids.cpu().clamp(0, max(V - 1, 0)).long()] * scale
    bad = ((ids < 0) | (ids >= V)).cpu()
    got = out.double().cpu()
    assert out.shape == (*ids.shape, table.shape[1])
    assert torch.isnan(got[bad]).all() and not torch.isnan(got[~bad]).any()
    tol = want.abs() * (2.0 ** -24 + half_step(out.dtype)) * (1 + 1e-6) + TINY[out.dtype]
    assert ((got - want).abs() <= tol)[~bad].all()


def check_bwd(g, ids, V, scale, pad, grad):
    """(the sums in 64 bits on the host)"""
    D = g.shape[-1]
    flat, gd = ids.reshape(-1).cpu().long(), g.reshape(-1, D).double().cpu()
    live = (flat >= 0) & (flat < V)
    if pad is not None:
        live &= flat != pad
    want, mass, count = torch.zeros(V, D, dtype=torch.float64), torch.zeros(V, D, dtype=torch.float64), torch.zeros(V, 1, dtype=torch.float64)
    want.index_add_(0, flat[live], gd[live])
    mass.index_add_(0, flat[live], gd[live].abs())
    count.index_add_(0, flat[live], torch.ones(int(live.sum()), 1, dtype=torch.float64))
    want, mass = want * scale, mass * abs(scale)
    tol = (count * 2.0 ** -24 * mass + half_step(grad.dtype) * want.abs()) * (1 + 1e-3) + TINY[grad.dtype]
    d = (grad.double().cpu() - want).abs()
    assert grad.shape == (V, D) and (d <= tol).all(), (float((d - tol).max()), float(d.max()))


# n, V, D: one token, one column, odd sizes, rows that are not 16-byte multiples, wide rows, sizes around the sorts' borders
SHAPES = [(1, 1, 1), (1, 7, 48), (3, 2, 5), (64, 100, 32), (65, 100, 33), (1000, 3, 27), (4097, 300, 8), (300, 70000, 4),
          (900, 100000, 4), (1024, 4097, 9), (2440, 9464, 8), (4096, 50000, 3), (8056, 195952, 5), (6000, 700, 65), (5000, 1, 8), (70000, 3, 1), (30000, 1000, 7),
          (200000, 1 << 20, 1), (9000, (1 << 20) + 1, 2), (150000, 1025, 4), (300001, 600000, 2), (4100, 5000, 33), (16384, 1025, 12), (16385, 1500, 16), (20000, 5, 2), (50001, 4096, 3), (33, 1000, 4096), (40, 9, 1111), (2, 3, 32768),
          (17, 50000, 40), (2000, 1, 512), (4095, 2049, 1), (4096, 3000, 258), (9000, 2, 4100), (12000, 5000, 515), (16383, 524288, 12),
          (16384, 1000, 64), (16384, 20000, 1), (300, 1, 32767), (3000, 4000, 1700), (100, 1 << 21, 5), (70000, 900, 36)]


@pytest.mark.parametrize("n,V,D", SHAPES)
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one"])
def test_forward_and_gradient(n, V, D, kind):
    from nerf_amd import ops
    rng = np.random.RandomState(n + V + D)
    ids = make_ids(kind, n, V, rng).cuda()
    table = torch.from_numpy(rng.normal(size=(V, D)).astype(np.float32)).cuda()
    g = torch.from_numpy(rng.normal(size=(n, D)).astype(np.float32)).cuda()
    check_fwd(table, ids, 0.75, ops.lookup_fwd(table, ids, 0.75))
    grad = ops.lookup_bwd(g, ids, V, 0.75)
    check_bwd(g, ids, V, 0.75, None, grad)
    assert torch.equal(grad, ops.lookup_bwd(g, ids.int(), V, 0.75))       # the same bits again, from 32-bit ids


@pytest.mark.parametrize("t,o", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("n,V,D", [(1, 4, 64), (777, 50, 33), (5000, 900, 24), (20000, 1 << 19, 2), (130, 60, 2056), (9001, 3000, 5), (8000, 70, 8), (15000, 3001, 36), (9000, 40, 2056), (9000, 40, 2057)])
def test_sixteen_bit_tables(t, o, n, V, D):
    from nerf_amd import ops
    rng = np.random.RandomState(D)
    ids = make_ids("zipf", n, V, rng).cuda()
    table = torch.from_numpy(rng.normal(size=(V, D)).astype(np.float32)).cuda().to(TYPES[t])
    out = ops.lookup_fwd(table, ids, 5.5, TYPES[o])
    assert out.dtype == TYPES[o]
    check_fwd(table, ids, 5.5, out)
    g = torch.from_numpy(rng.normal(size=(n, D)).astype(np.float32)).cuda().to(TYPES[o])
    grad = ops.lookup_bwd(g, ids, V, 5.5, dtype=TYPES[t])
    assert grad.dtype == TYPES[t]
    check_bwd(g, ids, V, 5.5, None, grad)


@pytest.mark.parametrize("n", [500, 15000, 40000])
def test_ids_outside_the_table_and_the_padding_row(n):
    from nerf_amd import ops
    rng = np.random.RandomState(3)
    V, D = 40, 20
    ids = torch.from_numpy(rng.randint(-3, V + 4, n)).cuda()
    ids[7], ids[11], ids[13] = 2 ** 40, -2 ** 62, 2 ** 32 + 1            # would alias rows if cut to 32 bits
    table = torch.randn(V, D, device="cuda")
    check_fwd(table, ids, 1.0, ops.lookup_fwd(table, ids))
    g = torch.randn(n, D, device="cuda")
    g[(ids < 0) | (ids >= V)] = float("nan")                             # what takes no part may hold anything
    check_bwd(g, ids, V, 1.0, None, ops.lookup_bwd(g, ids, V))
    g[ids == 5] = float("inf")
    check_bwd(g, ids, V, 1.0, 5, ops.lookup_bwd(g, ids, V, padding_idx=5))
    allout = torch.full((n,), -1, device="cuda")
    assert torch.isnan(ops.lookup_fwd(table, allout)).all()
    assert (ops.lookup_bwd(g, allout, V) == 0).all()


def test_no_tokens_no_rows():
    from nerf_amd import ops
    none = torch.empty((0,), dtype=torch.int64, device="cuda")
    table = torch.randn(5, 3, device="cuda")
    assert ops.lookup_fwd(table, none).shape == (0, 3)
    assert torch.equal(ops.lookup_bwd(torch.empty(0, 3, device="cuda"), none, 5), torch.zeros(5, 3, device="cuda"))
    ids = torch.tensor([[0, 1]], device="cuda")
    assert torch.isnan(ops.lookup_fwd(table[:0], ids)).all()
    assert ops.lookup_bwd(torch.randn(1, 2, 3, device="cuda"), ids, 0).shape == (0, 3)


def test_strides_alignment_and_shapes():
    from nerf_amd import ops
    rng = np.random.RandomState(5)
    base = torch.from_numpy(rng.normal(size=(90, 131)).astype(np.float32)).cuda()
    ids = torch.from_numpy(rng.randint(0, 90, (6, 7))).cuda()
    for table in (base[:, :64], base[:, 1:65], base[:, 2:34], base.t()[:90, :32], base[:1].expand(90, 131), base[3:4, :8].bfloat16(),
                  base[:, :64].bfloat16()[:, 1:33], base.half()[:, 3:], base[:, 5:6]):
        check_fwd(table, ids, 2.0, ops.lookup_fwd(table, ids, 2.0))
    wide = torch.from_numpy(rng.normal(size=(6, 7, 131)).astype(np.float32)).cuda()
    for g in (wide[..., :64], wide[..., 1:65], wide[..., 2:34], wide.transpose(0, 1).contiguous().transpose(0, 1),
              wide[:1, :1].expand(6, 7, 131), wide[..., 3:35].bfloat16(), wide.half()[..., 1:], wide[..., 5:6]):
        check_bwd(g, ids, 90, 2.0, None, ops.lookup_bwd(g, ids, 90, 2.0))
    # ids with strides of their own
    t = ids.t()
    assert torch.equal(ops.lookup_fwd(base, t), ops.lookup_fwd(base, t.contiguous()))


def test_values_that_are_not_finite_stay_in_their_rows():
    from nerf_amd import ops
    table = torch.randn(6, 10, device="cuda")
    table[2, 3], table[4, 1] = float("inf"), float("nan")
    out = ops.lookup_fwd(table, torch.tensor([2, 0, 4], device="cuda"), 2.0)
    torch.testing.assert_close(out, table[[2, 0, 4]] * 2.0, rtol=0, atol=0, equal_nan=True)
    g = torch.ones(3, 10, device="cuda")
    g[1] = float("inf")
    grad = ops.lookup_bwd(g, torch.tensor([2, 0, 4], device="cuda"), 6)
    assert torch.isinf(grad[0]).all() and torch.isfinite(grad[1:]).all()


def test_gradient_of_many_tokens_on_few_rows():
    """Runs that cover thousands of tiles (the join), among short ones."""
    from nerf_amd import ops
    rng = np.random.RandomState(8)
    n, V, D = 786432, 200, 33
    ids = make_ids("runs", n, V, rng)
    ids[:400000] = 17
    ids = ids.cuda()
    g = torch.from_numpy(rng.normal(size=(n, D)).astype(np.float32)).cuda()
    grad = ops.lookup_bwd(g, ids, V)
    check_bwd(g, ids, V, 1.0, None, grad)
    assert torch.equal(grad, ops.lookup_bwd(g, ids, V))


@pytest.mark.parametrize("kind", ["zipf", "one"])
def test_gradient_of_a_large_table(kind):
    """2^28 elements: the sort of 16384 tokens beside the zeros; compared row by row on the GPU, in f64."""
    from nerf_amd import ops
    rng = np.random.RandomState(12)
    n, V, D = 16384, 131072, 2048
    ids = make_ids(kind, n, V, rng).cuda()
    g = torch.from_numpy(rng.normal(size=(n, D)).astype(np.float32)).cuda().bfloat16()
    grad = ops.lookup_bwd(g, ids, V, 0.5)
    rows, inverse, count = torch.unique(ids, return_inverse=True, return_counts=True)
    want = torch.zeros(len(rows), D, dtype=torch.float64, device="cuda").index_add_(0, inverse, g.double()) * 0.5
    mass = torch.zeros(len(rows), D, dtype=torch.float64, device="cuda").index_add_(0, inverse, g.double().abs()) * 0.5
    tol = (count[:, None] * 2.0 ** -24 * mass + 2.0 ** -8 * want.abs()) * (1 + 1e-3)
    assert ((grad[rows].double() - want).abs() <= tol).all()
    grad[rows] = 0
    assert int((grad != 0).sum()) == 0
    assert torch.equal(ops.lookup_bwd(g, ids, V, 0.5)[rows], ops.lookup_bwd(g, ids, V, 0.5)[rows])


def test_offsets_beyond_32_bits():
    from nerf_amd import ops
    V, D = 540000, 4096                                                  # 2.2e9 elements
    table = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([V - 1, 0, 530000, V - 1, 524288], device="cuda")
    rows = torch.randn(5, D, device="cuda").bfloat16()
    rows[3] = rows[0]
    table[ids] = rows
    assert torch.equal(ops.lookup_fwd(table, ids), rows)
    del table
    for n in (5, 5000):                                                  # with and without the sort
        many = ids.repeat(n // 5)
        g = rows.repeat(n // 5, 1)
        grad = ops.lookup_bwd(g, many, V)
        want = torch.zeros(V, dtype=torch.float64)
        want.index_add_(0, many.cpu(), g[:, -1].double().cpu())
        tol = 2.0 ** -8 * want.abs() + n * 2.0 ** -24 * want.abs()
        assert ((grad[:, -1].double().cpu() - want).abs() <= tol * 1.001).all()
        assert int((grad != 0).any(1).sum()) == 4
        del grad
    # gradients whose rows lie far apart
    wide = torch.randn(2 ** 30 * 2 + 64, device="cuda", dtype=torch.bfloat16).as_strided((3, 40), (2 ** 30, 1))
    check_bwd(wide, ids[:3] % 7, 7, 1.0, None, ops.lookup_bwd(wide, ids[:3] % 7, 7))


def test_autograd_and_differences():
    from nerf_amd.codes import CodeTable
    torch.manual_seed(0)
    codes = CodeTable(12, 6, scale=3.0, padding_idx=4).cuda()
    assert (codes.weight[4] == 0).all()
    ids = torch.tensor([[1, 4, 1], [11, 0, 1]], device="cuda")
    w = torch.randn(2, 3, 6, device="cuda")
    loss = (codes(ids) * w).sum()
    loss.backward()
    check_bwd(w, ids, 12, 3.0, 4, codes.weight.grad)
    # the loss is linear in the table: a difference over a step of one is its derivative, but for the sums' rounding
    with torch.no_grad():
        for r, c in ((1, 2), (11, 5), (7, 0)):
            l0 = (codes(ids).double() * w.double()).sum()
            codes.weight[r, c] += 1.0
            l1 = (codes(ids).double() * w.double()).sum()
            codes.weight[r, c] -= 1.0
            assert abs(float(l1 - l0) - float(codes.weight.grad[r, c])) < 1e-4
    # a gradient of shared values: every token has the same one (an expanded tensor)
    codes.weight.grad = None
    codes(ids).sum().backward()
    assert torch.equal(codes.weight.grad[1], torch.full((6,), 9.0, device="cuda"))
    assert (codes.weight.grad[4] == 0).all()
    with torch.no_grad():
        assert not codes(ids).requires_grad


@pytest.mark.parametrize("n", [700, 12000, 20000])
def test_another_stream_and_a_captured_training_step(n):
    from nerf_amd.codes import lookup
    rng = np.random.RandomState(2)
    table = torch.from_numpy(rng.normal(size=(300, 24)).astype(np.float32)).cuda().requires_grad_()
    ids = make_ids("zipf", n, 300, rng).cuda()
    w = torch.from_numpy(rng.normal(size=(n, 24)).astype(np.float32)).cuda()

    def step():
        out = lookup(table, ids, 0.5)
        return out, torch.autograd.grad(out, table, w)[0]

    out0, grad0 = (v.detach().clone() for v in step())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out1, grad1 = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out0, out1) and torch.equal(grad0, grad1)
    del out1, grad1
    graphs = []
    for _ in range(2):                       # two captured graphs, replayed in turn: nothing shared between them
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        graphs.append((graph, res))
    for k in range(3):
        with torch.no_grad():
            table.add_(0.25)
            w.mul_(-0.5)
            ids.copy_(ids.roll(1))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        out, grad = step()
        for _, res in graphs:
            assert torch.equal(res[0], out) and torch.equal(res[1], grad), k


def test_refusals():
    from nerf_amd import ops
    from nerf_amd.codes import lookup
    table, ids = torch.zeros(4, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.lookup_fwd(table, ids.float())
    with pytest.raises(RuntimeError, match="ids: expected a tensor on"):
        ops.lookup_fwd(table, ids.cpu())
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.lookup_fwd(table.double(), ids)
    with pytest.raises(TypeError, match="out_dtype"):
        ops.lookup_fwd(table, ids, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="dim >= 1"):
        ops.lookup_fwd(table[0], ids)
    with pytest.raises(RuntimeError, match="dim at most"):
        ops.lookup_fwd(torch.zeros(1, 40000, device="cuda"), ids)
    g = torch.zeros(3, 8, device="cuda")
    with pytest.raises(ValueError, match="g_out: expected"):
        ops.lookup_bwd(g[:2], ids, 4)
    with pytest.raises(TypeError, match="does not go with"):
        ops.lookup_bwd(g.half(), ids, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="padding_idx"):
        ops.lookup_bwd(g, ids, 4, padding_idx=4)
    # ids changed between forward and backward: autograd's own check speaks
    t = table.requires_grad_()
    out = lookup(t, ids)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
