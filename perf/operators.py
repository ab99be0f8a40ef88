"""What is measured of the operators that choose a training batch and look up its learned codes: drawing indices from rows of
logits (`sample_logits`), the rows of a code table (`lookup`) and the table's gradient (`lookup_bwd`).

`own` chooses who computes: False = plain torch operations, True = this framework's kernels."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}

# What a case may cost at most (the largest listed ones): values looked up, values of a dense gradient, logits, draws.
MOST_LOOKED_UP, MOST_TABLE, MOST_LOGITS, MOST_DRAWS = 1 << 26, 1 << 29, 1 << 25, 1 << 16


def listed():
    return [
        # the code of the one image a viewer renders
        dict(name="code of one image", op="lookup", n=1, rows=100, dim=48, type="f32", scale=1.0, ids="uniform"),
        # one code for each ray of a training batch drawn over 100 images
        dict(name="codes of a ray batch", op="lookup", n=4096, rows=100, dim=32, type="f32", scale=1.0, ids="uniform"),
        # the eight corners around each of 262144 points in one level of a hashed feature grid
        dict(name="features of grid corners", op="lookup", n=2097152, rows=524288, dim=2, type="f32", scale=1.0, ids="uniform"),
        # wide 16-bit rows for a long sequence of tokens, scaled by the root of their width
        dict(name="rows of a token batch", op="lookup", n=16384, rows=131072, dim=4096, type="bf16", scale=64.0, ids="zipf"),
        # gradient of the codes of a ray batch: few rows, each met by about 40 rays
        dict(name="gradient, ray batch", op="lookup_bwd", n=4096, rows=100, dim=32, type="f32", scale=1.0, ids="uniform"),
        # gradient of per-frame codes looked up for every sample point of a batch (4096 rays of 192), an odd width
        dict(name="gradient, sample points", op="lookup_bwd", n=786432, rows=200, dim=33, type="f32", scale=1.0, ids="runs"),
        # gradient of one level of a hashed feature grid
        dict(name="gradient, grid corners", op="lookup_bwd", n=2097152, rows=524288, dim=2, type="f32", scale=1.0, ids="uniform"),
        # gradient of a wide 16-bit table: most of its rows are zero, a few are met by very many tokens
        dict(name="gradient, token batch", op="lookup_bwd", n=16384, rows=131072, dim=4096, type="bf16", scale=64.0, ids="zipf"),
        # the pixels of a training batch, drawn by the error map of one 800 x 800 image
        dict(name="pixels by an error map", op="sample_logits", rows=1, size=640000, draws=4096, type="f32",
             logits="errors", filters="scalar", temperature=0.5, top_k=0, top_p=0.95, min_p=0.0),
        # the next token of one sequence
        dict(name="one token", op="sample_logits", rows=1, size=131072, draws=1, type="bf16", logits="normal",
             filters="scalar", temperature=0.8, top_k=50, top_p=0.9, min_p=0.02),
        # the next tokens of a full batch, each sequence with filters of its own
        dict(name="tokens of a batch", op="sample_logits", rows=256, size=131072, draws=1, type="bf16", logits="normal",
             filters="rows", temperature=1.0, top_k=1000, top_p=0.95, min_p=0.01),
        # one class for each of many short rows, an odd length, only a temperature
        dict(name="classes of many rows", op="sample_logits", rows=4096, size=1001, draws=1, type="f32", logits="normal",
             filters="scalar", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_bwd", "sample_logits"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "sample_logits":
        size = _log_int(rng, 1, 640000)
        rows = _log_int(rng, 1, max(1, min(4096, MOST_LOGITS // size)))
        return dict(op=op, rows=rows, size=size, draws=_log_int(rng, 1, max(1, min(4096, MOST_DRAWS // rows))), type=kind,
                    logits=rng.choice(["errors", "normal", "masked"]), filters=rng.choice(["scalar", "rows"]),
                    temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]), top_k=rng.choice([0, 0, 1, _log_int(rng, 1, size)]),
                    top_p=rng.choice([1.0, 1.0, round(rng.uniform(0.05, 0.999), 3)]),
                    min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]))
    dim = _log_int(rng, 1, 4096)
    n = _log_int(rng, 1, min(1 << 21, MOST_LOOKED_UP // dim))
    rows = _log_int(rng, 1, min(1 << 19, (MOST_TABLE if op == "lookup_bwd" else 2 * MOST_TABLE) // dim))
    return dict(op=op, n=n, rows=rows, dim=dim, type=kind, scale=rng.choice([1.0, 0.125, round(math.sqrt(dim), 3)]),
                ids=rng.choice(["uniform", "zipf", "runs"]))


def _ids(case, gen):
    n, rows = case["n"], case["rows"]
    if case["ids"] == "zipf":       # frequencies that fall as 1 / rank: token ids, pixels of a bright object
        r = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
        return (torch.exp(r * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
    ids = torch.randint(0, rows, (n,), generator=gen, device="cuda")
    if case["ids"] == "runs":       # one id for each ray, repeated for its 192 sample points
        ids = ids[: (n + 191) // 192].repeat_interleave(192)[:n]
    return ids


def _logits(case, gen):
    shape = (case["rows"], case["size"])
    if case["logits"] == "errors":  # the log of squared colour errors, which spread over many decades
        e = torch.randn(shape, generator=gen, device="cuda") * 0.1
        x = torch.log(e * e + 1e-6)
    else:
        x = torch.randn(shape, generator=gen, device="cuda") * 2.5
    if case["logits"] == "masked":  # entries that may not be drawn; about one row in 20 has none that may
        hole = torch.rand(shape, generator=gen, device="cuda") < torch.rand((shape[0], 1), generator=gen, device="cuda") * 1.05
        x = x.masked_fill(hole, -math.inf)
    return x.to(DTYPES[case["type"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = DTYPES.get(case["type"])
    if case["op"] == "sample_logits":
        rows, size = case["rows"], case["size"]
        state = dict(case=case, logits=_logits(case, gen),
                     u=torch.rand((rows, case["draws"]), generator=gen, device="cuda"))
        t, k, p, m = case["temperature"], case["top_k"], case["top_p"], case["min_p"]
        if case["filters"] == "rows":
            f = lambda: torch.rand(rows, generator=gen, device="cuda")  # noqa: E731
            state.update(temperature=t * (0.5 + f()), top_k=(k * (0.5 + f())).round().int().clamp(0, size),
                         top_p=(1.0 - (1.0 - p) * 2.0 * f()).clamp(0.01, 1.0), min_p=m * 2.0 * f())
        else:
            state.update(temperature=t, top_k=k, top_p=p, min_p=m)
        return state
    state = dict(case=case, ids=_ids(case, gen))
    if case["op"] == "lookup":
        state["table"] = torch.randn((case["rows"], case["dim"]), generator=gen, device="cuda", dtype=torch.float32).to(kind)
    else:
        state["g"] = (torch.randn((case["n"], case["dim"]), generator=gen, device="cuda") * 0.01).to(kind)
    return state


def run(state):
    case = state["case"]
    if case["op"] == "lookup":
        return _run_lookup(case, state["table"], state["ids"])
    if case["op"] == "lookup_bwd":
        return _run_lookup_bwd(case, state["g"], state["ids"])
    return _run_sample(state)


def _run_lookup(case, table, ids):
    if own:
        from nerf_amd import ops
        return ops.lookup_fwd(table, ids, scale=case["scale"])
    return (table[ids].float() * case["scale"]).to(table.dtype)


def _run_lookup_bwd(case, g, ids):
    if own:
        from nerf_amd import ops
        return ops.lookup_bwd(g, ids, case["rows"], scale=case["scale"])
    grad = torch.zeros((case["rows"], case["dim"]), device=g.device, dtype=torch.float32)
    grad.index_add_(0, ids, g.float())
    return (grad * case["scale"]).to(g.dtype)


def _run_sample(s):
    case = s["case"]
    if own:
        from nerf_amd import ops
        return ops.sample_logits(s["logits"], case["draws"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                 min_p=s["min_p"], u=s["u"])
    x = s["logits"].float()
    rows, size = x.shape
    col = lambda v, t: v.to(t)[:, None] if torch.is_tensor(v) else torch.full((rows, 1), v, device=x.device, dtype=t)  # noqa: E731
    t, p, m = (col(s[k], torch.float32).double() for k in ("temperature", "top_p", "min_p"))
    k = col(s["top_k"], torch.int64)
    k = torch.where(k <= 0, size, k)
    k = torch.where(t == 0, 1, k)                                    # greedy: the first maximum alone
    # masses in 64 bits: an index is exact only if the running sums around it are
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    e = torch.exp((x.double() - top.double()) / t)
    e = torch.where(x == top, 1.0, e)
    e = torch.where(x == -math.inf, 0.0, e)
    if case["temperature"] == 0 or case["top_k"] > 0 or case["top_p"] < 1 or case["min_p"] > 0:
        # kept: a prefix of the entries in falling order, ties in the order of their index
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices
        es = e.gather(-1, order)
        rank = torch.arange(size, device=x.device)
        es_k = torch.where(rank < k, es, 0.0)
        cum = torch.cumsum(es_k, -1)
        before = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], -1)
        keep = (rank < k) & ((p >= 1) | (before < p * cum[:, -1:])) & (es >= m)
        keep |= rank == 0
        e = e * torch.zeros_like(keep).scatter_(-1, order, keep)
    cum = torch.cumsum(e, -1)
    total = cum[:, -1:].contiguous()
    ids = torch.searchsorted(cum, s["u"].double() * total, right=True)
    last = torch.where(e > 0, torch.arange(size, device=x.device), 0).amax(-1, keepdim=True)
    ids = torch.minimum(ids, last)
    prob = e.gather(-1, ids) / total
    ids = torch.where(total > 0, ids, -1)
    return ids, torch.where(total > 0, prob, 0.0).float()


def work(case):
    if case["op"] == "sample_logits":
        n = case["rows"] * case["size"]
        # each logit: a difference, a scaling, an exponential, a sum
        return dict(bytes=n * SIZE[case["type"]] + case["rows"] * case["draws"] * 16, flops=4 * n)
    values, size = case["n"] * case["dim"], SIZE[case["type"]]
    table = case["rows"] * case["dim"]
    if case["op"] == "lookup":
        return dict(bytes=min(values, table) * size + values * size + case["n"] * 8, flops=values)
    return dict(bytes=values * size + table * size + case["n"] * 8, flops=values)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lookup":
        return torch.mul(s["table"].double(), case["scale"]).index_select(0, s["ids"])
    if case["op"] == "lookup_bwd":
        # differences of one running sum over the tokens in the order of their ids
        order = torch.argsort(s["ids"], stable=True)
        ends = torch.searchsorted(s["ids"][order], torch.arange(case["rows"] + 1, device="cuda"))
        out = []
        for lo in range(0, case["dim"], 512):
            run_ = torch.cumsum(s["g"][:, lo:lo + 512].double()[order], 0)
            run_ = torch.cat([torch.zeros_like(run_[:1]), run_])
            out.append((run_[ends[1:]] - run_[ends[:-1]]) * case["scale"])
        return torch.cat(out, 1)
    # row by row on the host: sort the masses, cut, walk the distribution
    rows, size = s["logits"].shape
    if rows * size > 1 << 23:
        return None
    x = s["logits"].double().cpu().numpy()
    u = s["u"].double().cpu().numpy()
    host = lambda v: np.broadcast_to(v.float().cpu().numpy().astype(np.float64) if torch.is_tensor(v) else np.float64(np.float32(v)), (rows,))  # noqa: E731
    t, k, p, m = (host(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    prob = np.zeros(u.shape)
    for r in range(rows):
        if not np.any(x[r] > -np.inf):
            continue
        order = np.lexsort((np.arange(size), -x[r]))
        z = x[r][order]
        if t[r] == 0:
            z = z[:1]
        e = np.exp((z - z[0]) / t[r]) if t[r] > 0 else np.ones(1)
        if k[r] > 0:
            e = e[:int(k[r])]
        if p[r] < 1:
            run_ = np.cumsum(e)
            e = e[:1 + int(np.searchsorted(run_, p[r] * run_[-1], side="left"))]
        e = e[:max(1, int(np.sum(e >= m[r])))]
        full = np.zeros(size)
        full[order[:len(e)]] = e
        cdf = np.cumsum(full) / np.sum(e)
        at = np.searchsorted(cdf, u[r], side="right")
        at = np.minimum(at, np.max(np.nonzero(full)[0]))
        prob[r] = full[at] / np.sum(e)
    return None, torch.from_numpy(prob)
