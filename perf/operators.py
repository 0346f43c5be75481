"""Cases of the framework's training operators on tensors and row tables, to be timed and compared:

  norm    gradients.global_norm              one 2-norm over many gradient tensors
  clip    gradients.clip_by_global_norm      the same, and the gradients scaled to a largest norm
  lookup  row_table.lookup_rows              scaled rows of a table by integer id
  grad    row_table.lookup_rows_backward     the gradient of that table, and which rows it touched
  step    surfel.SparseGaussianAdam.step     row-masked Adam on gradients clipped by their global norm

`own` chooses between the framework's operators and their plain form in elementary torch
operations.  Inputs live on the GPU and are made from the seed alone.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
WIDTHS = (3, 3, 1, 2, 4)                 # floats per splat: position, colour, opacity, scales, rotation
LRS = (0.00016, 0.0025, 0.05, 0.005, 0.001)
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BETA1, BETA2, EPS = 0.9, 0.999, 1e-15
LARGEST = 1.1e9                          # bytes of the largest listed case


def listed():
    return [
        # a map just started (one keyframe's points kept): the call's own latency
        {"name": "norm splats 1000", "op": "norm", "layout": "splats", "n": 1000},
        # the gradients of a deep network beside the map: 144 tensors, 805 MB of bfloat16
        {"name": "norm network 24x2048", "op": "norm", "layout": "network", "layers": 24, "width": 2048, "dtype": "bf16"},
        # a map at the reference's operating point, ragged by one splat
        {"name": "clip splats 299999", "op": "clip", "layout": "splats", "n": 299999, "max_norm": 1.0},
        # bfloat16 gradients clipped into the float32 gradients that the optimiser reads
        {"name": "clip network 10x2048", "op": "clip", "layout": "network", "layers": 10, "width": 2048, "dtype": "bf16", "max_norm": 1.0},
        # one token's row while serving
        {"name": "lookup one token", "op": "lookup", "n": 1, "rows": 32768, "cols": 2048, "dtype": "bf16", "ids": "power", "scale": 45.25},
        # a batch of tokens while training
        {"name": "lookup 16381 tokens", "op": "lookup", "n": 16381, "rows": 32768, "cols": 2048, "dtype": "bf16", "ids": "power", "scale": 45.25},
        # every splat of a map reads the affine colour row (3 x 4) of the keyframe that owns it
        {"name": "lookup keyframe rows", "op": "lookup", "n": 1000000, "rows": 80, "cols": 12, "dtype": "fp32", "ids": "owners", "scale": 1.0},
        # the few splats of a new keyframe and their colour offsets: the call's own latency
        {"name": "grad 300 splats", "op": "grad", "n": 300, "rows": 77, "cols": 3, "dtype": "fp32", "ids": "owners", "scale": 1.0},
        # the training batch's backward pass; frequent tokens own many positions
        {"name": "grad 16381 tokens", "op": "grad", "n": 16381, "rows": 32768, "cols": 2048, "dtype": "bf16", "ids": "power", "scale": 45.25},
        # few rows, each the sum over thousands of splats
        {"name": "grad keyframe rows", "op": "grad", "n": 1000000, "rows": 80, "cols": 12, "dtype": "fp32", "ids": "owners", "scale": 1.0},
        # the optimiser's step of a small map
        {"name": "step splats 2000", "op": "step", "n": 2000, "max_norm": 1.0},
        # ... and of the map of the headline workload
        {"name": "step splats 1000000", "op": "step", "n": 1000000, "max_norm": 1.0},
    ]


def _between(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["norm", "clip", "lookup", "grad", "step"])
        case = {"op": op}
        if op in ("norm", "clip"):
            case["layout"] = rng.choice(["splats", "network"])
            if case["layout"] == "splats":
                case["n"] = _between(rng, 200, 5000000)
            else:
                case["layers"] = rng.randint(1, 10 if op == "clip" else 24)
                case["width"] = _between(rng, 64, 2048)
                case["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
            if op == "clip":
                case["max_norm"] = rng.choice([0.01, 1.0, 1.0, 1e6])
        elif op == "step":
            case["n"] = _between(rng, 200, 2000000)
            case["max_norm"] = rng.choice([0.01, 1.0, 1.0, 1e6])
        else:
            case["ids"] = rng.choice(["power", "uniform", "owners"])
            if case["ids"] == "owners":      # splats and their keyframes' rows
                case.update(n=_between(rng, 200, 1000000), rows=_between(rng, 2, 2000), cols=_between(rng, 1, 64), dtype="fp32", scale=1.0)
            else:                            # tokens and a wide table
                case.update(n=_between(rng, 1, 32768), rows=_between(rng, 500, 65536), cols=_between(rng, 32, 4096),
                            dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
                if rng.random() < 0.6:
                    case["cols"] = max(32, case["cols"] // 64 * 64)
                case["scale"] = round(math.sqrt(case["cols"]), 3)
        if work(case)["bytes"] <= 0.9 * LARGEST:
            return case


def _shapes(case):
    """[(shape, dtype)] of the gradient tensors of a norm or clip case."""
    if case["layout"] == "splats":
        return [((case["n"], w), "fp32") for w in WIDTHS]
    w, dt = case["width"], case["dtype"]
    return ([((w, w), dt)] * 4 + [((w,), "fp32")] * 2) * case["layers"]


def _ids(case, gen):
    n, rows = case["n"], case["rows"]
    if case["ids"] == "power":           # a few ids are frequent, most are rare
        u = torch.rand(n, device=DEV, generator=gen, dtype=torch.float64)
        return (rows * u ** 4).long().clamp_(0, rows - 1)
    rand = torch.randint(0, rows, (n,), device=DEV, generator=gen)
    if case["ids"] == "uniform":
        return rand
    # splats are appended keyframe by keyframe; some change their owner later, some have none (-1)
    mine = torch.arange(n, device=DEV) * rows // n
    u = torch.rand(n, device=DEV, generator=gen)
    return torch.where(u < 0.01, torch.full_like(mine, -1), torch.where(u < 0.2, rand, mine))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def rand(shape, dtype="fp32", scale=1.0):
        return (torch.randn(shape, device=DEV, generator=gen) * scale).to(DTYPES[dtype])

    op = case["op"]
    st = {"op": op, "case": case}
    if op in ("norm", "clip"):
        st["grads"] = [rand(s, d, 0.02) for s, d in _shapes(case)]
        if op == "clip":
            st["out"] = [torch.empty(s, device=DEV) for s, _ in _shapes(case)]
    elif op in ("lookup", "grad"):
        st["ids"] = _ids(case, gen)
        if op == "lookup":
            st["table"] = rand((case["rows"], case["cols"]), case["dtype"], 0.02)
        else:
            st["grad"] = rand((case["n"], case["cols"]), case["dtype"], 0.02)
    else:
        n = case["n"]
        st["visible"] = torch.rand(n, device=DEV, generator=gen) < 0.7
        st["params"] = [rand((n, w)) for w in WIDTHS]
        grads = [rand((n, w), scale=0.02) for w in WIDTHS]
        st["exp_avg"] = [rand((n, w), scale=0.01) for w in WIDTHS]
        st["exp_avg_sq"] = [rand((n, w), scale=0.01).square_().add_(1e-8) for w in WIDTHS]
        for p, g in zip(st["params"], grads):
            p.grad = g
        if own:                          # the optimiser that a training program keeps
            from vings_mono_amd.surfel import SparseGaussianAdam
            opt = SparseGaussianAdam([{"params": [p], "lr": lr} for p, lr in zip(st["params"], LRS)], lr=0.0, eps=EPS)
            for p, m, v in zip(st["params"], st["exp_avg"], st["exp_avg_sq"]):
                opt.state[p] = {"step": torch.tensor(0.0), "exp_avg": m, "exp_avg_sq": v}
            st["opt"] = opt
    return st


def _plain_norm(grads):
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def run(st):
    op, case = st["op"], st["case"]
    if own:
        from vings_mono_amd import gradients, row_table
        if op == "norm":
            return gradients.global_norm(st["grads"])
        if op == "clip":
            norm = gradients.clip_by_global_norm(st["grads"], case["max_norm"], out=st["out"])
            return {"norm": norm, "out": st["out"]}
        if op == "lookup":
            return row_table.lookup_rows(st["table"], st["ids"], scale=case["scale"])
        if op == "grad":
            rows, touched = row_table.lookup_rows_backward(st["grad"], st["ids"], case["rows"], scale=case["scale"])
            return {"rows": rows, "touched": touched}
        norm = st["opt"].step(st["visible"], case["n"], max_norm=case["max_norm"])
        return {"norm": norm, "params": st["params"], "exp_avg": st["exp_avg"], "exp_avg_sq": st["exp_avg_sq"]}

    if op == "norm":
        return _plain_norm(st["grads"])
    if op == "clip":
        norm = _plain_norm(st["grads"])
        coef = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        for g, o in zip(st["grads"], st["out"]):
            o.copy_(g.float() * coef)
        return {"norm": norm, "out": st["out"]}
    if op == "lookup":
        ids, table = st["ids"], st["table"]
        found = (ids >= 0) & (ids < case["rows"])
        rows = table[torch.where(found, ids, torch.zeros_like(ids))].float() * case["scale"]
        return torch.where(found[:, None], rows, torch.zeros_like(rows)).to(table.dtype)
    if op == "grad":
        ids, grad, rows = st["ids"], st["grad"], case["rows"]
        at = torch.where((ids >= 0) & (ids < rows), ids, torch.full_like(ids, rows))     # one row more for those without
        total = torch.zeros((rows + 1, case["cols"]), device=DEV).index_add_(0, at, grad.float())
        touched = torch.zeros(rows + 1, dtype=torch.bool, device=DEV)
        touched[at] = True
        return {"rows": (total[:rows] * case["scale"]).to(grad.dtype), "touched": touched[:rows].clone()}
    seen = st["visible"][:, None]
    grads = [torch.where(seen, p.grad, torch.zeros_like(p.grad)) for p in st["params"]]
    norm = _plain_norm(grads)
    coef = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    seen = seen & torch.isfinite(norm)
    for p, g, m, v, lr in zip(st["params"], grads, st["exp_avg"], st["exp_avg_sq"], LRS):
        g = g * coef
        m.copy_(torch.where(seen, BETA1 * m + (1 - BETA1) * g, m))
        v.copy_(torch.where(seen, BETA2 * v + (1 - BETA2) * g * g, v))
        p.copy_(torch.where(seen, p - lr * m / (v.sqrt() + EPS), p))
    return {"norm": norm, "params": st["params"], "exp_avg": st["exp_avg"], "exp_avg_sq": st["exp_avg_sq"]}


def _distinct(case):
    """Expected number of table rows that the ids of a case name."""
    n, rows = case["n"], case["rows"]
    if case["ids"] == "power":
        p = np.diff((np.arange(rows + 1) / rows) ** 0.25)
    else:
        p = np.full(rows, 1.0 / rows)
    return float(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12))).sum())


def work(case):
    """Bytes and operations of one pass: every input once, every output once."""
    op = case["op"]
    if op in ("norm", "clip"):
        sizes = [(math.prod(s), DTYPES[d].itemsize) for s, d in _shapes(case)]
        n = sum(k for k, _ in sizes)
        read = sum(k * b for k, b in sizes)
        return {"bytes": read + (4 * n if op == "clip" else 0), "flops": (3 if op == "clip" else 2) * n}
    if op == "step":
        n = case["n"] * sum(WIDTHS) * 0.7
        return {"bytes": 7 * 4 * n + case["n"], "flops": 16 * n}
    size = DTYPES[case["dtype"]].itemsize * case["cols"]
    if op == "lookup":
        return {"bytes": 8 * case["n"] + size * (_distinct(case) + case["n"]), "flops": case["n"] * case["cols"]}
    return {"bytes": 8 * case["n"] + size * (case["n"] + case["rows"]) + case["rows"], "flops": case["n"] * case["cols"]}


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    st = prepare(case, seed)
    op = case["op"]

    def length(parts):
        return torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(x.double()) for x in parts]))

    if op == "norm":
        return length(st["grads"])
    if op == "clip":
        norm = length(st["grads"])
        factor = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
        return {"norm": norm, "out": [g.double() * factor for g in st["grads"]]}
    if op == "lookup":
        ids = st["ids"]
        out = torch.zeros((case["n"], case["cols"]), dtype=torch.float64, device=DEV)
        good = ((ids >= 0) & (ids < case["rows"])).nonzero()[:, 0]
        out[good] = st["table"].index_select(0, ids[good]).double() * case["scale"]
        return out
    if op == "grad":
        # ids in order, running sums of their rows, and the differences of those at the ids' ends
        ids, order = torch.sort(st["ids"])
        run_sum = torch.cat([torch.zeros((1, case["cols"]), dtype=torch.float64, device=DEV),
                             st["grad"][order].double().cumsum(0)])
        names = torch.arange(case["rows"], device=DEV)
        first, last = torch.searchsorted(ids, names), torch.searchsorted(ids, names, right=True)
        return {"rows": (run_sum[last] - run_sum[first]) * case["scale"], "touched": last > first}
    keep = st["visible"].nonzero()[:, 0]
    norm = length([p.grad[keep] for p in st["params"]])
    factor = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    res = {"norm": norm, "params": [], "exp_avg": [], "exp_avg_sq": []}
    for p, m, v, lr in zip(st["params"], st["exp_avg"], st["exp_avg_sq"], LRS):
        p, g, m, v = p.detach().double(), p.grad.double(), m.double(), v.double()
        g = g[keep] * factor
        m[keep] = BETA1 * m[keep] + (1 - BETA1) * g
        v[keep] = BETA2 * v[keep] + (1 - BETA2) * g ** 2
        p[keep] = p[keep] - lr * m[keep] / (v[keep].sqrt() + EPS)
        for key, value in (("params", p), ("exp_avg", m), ("exp_avg_sq", v)):
            res[key].append(value)
    return res
