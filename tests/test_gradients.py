"""Global gradient norm, clipping and the clipped row-masked Adam step against their formulas in
float64.

Tolerances (u = 2^-24, half a float32 step; h_t = eps/2 of the result's type): a norm is a sum of
exact squares in 64 bits, rounded once: 2 u.  A clipped gradient carries the norm's rounding, the
coefficient's and its own product's: 3 u + h_t, and half of float16's smallest step below its
normal range."""
import ctypes
import math
import threading

import pytest
import torch

from vings_mono_amd import _lib, gradients, harness, surfel, synth

DEV = "cuda:0"
U = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
gpu = pytest.mark.gpu


def rand(shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def norm64(tensors, kind=2.0):
    flat = torch.cat([t.detach().reshape(-1).double().cpu() for t in tensors])
    if kind == 2.0:
        return float(flat.square().sum().sqrt())
    return float(flat.abs().max()) if flat.numel() else 0.0


LISTS = {
    "one": [((1,), torch.float32)],
    "odd": [((7, 3), torch.float32), ((5,), torch.bfloat16), ((0, 4), torch.float32), ((1, 1), torch.float16)],
    "chunk edges": [((n,), t) for n in (2047, 2048, 2049, 4096) for t in HALF],
    "splats": [((12345, w), torch.float32) for w in (3, 3, 1, 2, 4)],
    "one workgroup": [((30719,), torch.float32), ((2047,), torch.bfloat16)],      # 16 chunks: its most
    "two workgroups": [((30719,), torch.float32), ((2049,), torch.bfloat16)],
    "16 tensors": [((5000 + i,), torch.bfloat16) for i in range(16)],             # the short table
    "17 tensors": [((5000 + i,), torch.bfloat16) for i in range(17)],
    "112 tensors": [((100 + i,), torch.float32) for i in range(112)],             # one clipping launch
    "113 tensors": [((100 + i,), torch.float16) for i in range(113)],
    "161 tensors": [((3000 + i,), torch.float32) for i in range(161)],            # two norm launches
    "many": [((17 + 13 * i,), (torch.bfloat16, torch.float32, torch.float16)[i % 3]) for i in range(389)],
    "long": [((3000001,), torch.bfloat16), ((1500007,), torch.float32)],
}


def make(name, scale=1.0):
    return [rand(s, t, seed=i, scale=scale) for i, (s, t) in enumerate(LISTS[name])]


@gpu
@pytest.mark.parametrize("kind", [2.0, float("inf")])
@pytest.mark.parametrize("name", list(LISTS))
def test_norm(name, kind):
    ts = make(name)
    got = gradients.global_norm(ts, kind)
    assert got.shape == () and got.dtype == torch.float32 and got.device == ts[0].device
    want = norm64(ts, kind)
    assert abs(float(got) - want) <= 2 * U * want
    assert torch.equal(got, gradients.global_norm(ts, kind))


@gpu
@pytest.mark.parametrize("kind", [2.0, float("inf")])
@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("where", ["in place", "own type", "float32"])
def test_clip(name, kind, where):
    ts = make(name, scale=0.5)
    before = [t.clone() for t in ts]
    want = norm64(before, kind)
    max_norm = 0.3 * want
    out = {"in place": None, "own type": [torch.empty_like(t) for t in ts],
           "float32": [torch.empty_like(t, dtype=torch.float32) for t in ts]}[where]
    norm = gradients.clip_by_global_norm(ts, max_norm, kind, out=out)
    assert abs(float(norm) - want) <= 2 * U * want
    coef = min(1.0, max_norm / (want + 1e-6))
    for b, t, o in zip(before, ts, ts if out is None else out):
        if out is not None:
            assert torch.equal(b, t)
        ref = b.double() * coef
        floor = 2.0 ** -25 if o.dtype == torch.float16 else 0.0
        assert ((o.double() - ref).abs() <= ref.abs() * (3 * U + HALF[o.dtype]) + floor).all()


@gpu
def test_short_gradients_stay_bit_for_bit():
    ts = make("splats") + make("odd")
    before = [t.clone() for t in ts]
    versions = [t._version for t in ts]
    gradients.clip_by_global_norm(ts, 1e9)
    assert all(torch.equal(a, b) for a, b in zip(before, ts))
    assert all(t._version > v for t, v in zip(ts, versions))
    out = [torch.full_like(t, 7.0) for t in ts]
    gradients.clip_by_global_norm(ts, float("inf"), out=out)
    assert all(torch.equal(a, b) for a, b in zip(before, out))


@gpu
def test_some_in_place_and_some_not():
    ts = make("splats")
    before = [t.clone() for t in ts]
    out = [ts[0], torch.empty_like(ts[1]), ts[2], torch.empty_like(ts[3]), ts[4]]
    gradients.clip_by_global_norm(ts, 1.0, out=out)
    alone = [torch.empty_like(t) for t in ts]
    gradients.clip_by_global_norm(before, 1.0, out=alone)
    assert all(torch.equal(a, b) for a, b in zip(out, alone))
    assert torch.equal(ts[1], before[1]) and torch.equal(ts[3], before[3])


@gpu
def test_two_threads_on_two_streams():
    """No state is shared between calls: each thread gets the bits of a solitary call."""
    lists = [make("splats"), make("many")]
    want = [gradients.global_norm(ts) for ts in lists]
    torch.cuda.synchronize()
    got = [[], []]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got[k].append(gradients.global_norm(lists[k]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert len(got[k]) == 50 and all(torch.equal(g, want[k]) for g in got[k])


@gpu
def test_zero_norm_and_zero_max_norm():
    ts = [torch.zeros(5000, device=DEV)]
    assert float(gradients.clip_by_global_norm(ts, 1.0)) == 0.0 and not ts[0].any()
    ts = make("splats")
    gradients.clip_by_global_norm(ts, 0.0)
    assert not any(t.any() for t in ts)
    empty = [torch.empty(0, device=DEV), torch.empty((0, 3), device=DEV)]
    assert float(gradients.global_norm(empty)) == 0.0
    assert float(gradients.clip_by_global_norm(empty, 1.0)) == 0.0


@gpu
@pytest.mark.parametrize("n", [4097, 300000])
@pytest.mark.parametrize("scale", [1e30, 1e-30, 1e-42])
def test_extreme_magnitudes(n, scale):
    """Squares that leave float32's range on either side do not leave the sum's."""
    t = rand((n,), seed=3, scale=scale)
    want = norm64([t])
    # (a norm in float32's subnormal range is rounded to 2^-149)
    assert abs(float(gradients.global_norm([t])) - want) <= 2 * U * want + 2.0 ** -149
    out = [torch.empty_like(t)]
    gradients.clip_by_global_norm([t], scale, out=out)
    coef = min(1.0, scale / (want + 1e-6))
    ref = t.double() * coef
    # the coefficient's float32 rounding of max_norm is one more u
    assert ((out[0].double() - ref).abs() <= ref.abs() * (5 * U) + 2.0 ** -149).all()


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("n", [100, 100000])
@pytest.mark.parametrize("kind", [2.0, float("inf")])
def test_not_finite(bad, n, kind):
    t = rand((n,), seed=1)
    t[n // 2] = bad
    norm = float(gradients.global_norm([t], kind))
    assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
    with pytest.raises(_lib.VingsError, match="not finite"):
        p = torch.nn.Parameter(torch.zeros(n, device=DEV))
        p.grad = t
        gradients.clip_grad_norm_([p], 1.0, kind, error_if_nonfinite=True)
    out = torch.empty_like(t)
    gradients.clip_by_global_norm([t], 1.0, kind, out=[out])
    if math.isnan(bad):
        assert torch.isnan(out).all()
    else:
        assert torch.isnan(out[n // 2]) and not out[: n // 2].any() and not out[n // 2 + 1:].any()


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("shift", [1, 2, 3, 5])
def test_views_at_any_element(dtype, shift):
    """Tensors that start inside a larger one; what lies around them is left alone."""
    base = rand((40000,), dtype, seed=9)
    keep = base.clone()
    t = base[shift:shift + 30011]
    out_base = torch.full((40000,), 3.0, device=DEV)
    out = out_base[shift + 1:shift + 1 + 30011]
    want = norm64([t])
    assert abs(float(gradients.global_norm([t])) - want) <= 2 * U * want
    gradients.clip_by_global_norm([t], 1.0, out=[out])
    ref = t.double() / (want + 1e-6)
    assert ((out.double() - ref).abs() <= ref.abs() * 4 * U).all()
    assert (out_base[:shift + 1] == 3).all() and (out_base[shift + 1 + 30011:] == 3).all()
    gradients.clip_by_global_norm([t], 1.0)
    assert torch.equal(base[:shift], keep[:shift]) and torch.equal(base[shift + 30011:], keep[shift + 30011:])
    ref = keep[shift:shift + 30011].double() / (want + 1e-6)
    floor = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert ((t.double() - ref).abs() <= ref.abs() * (3 * U + HALF[dtype]) + floor).all()


@gpu
def test_dense_orders_other_than_row_major():
    a = rand((64, 33, 5), seed=4).permute(2, 0, 1)
    b = rand((31, 77), torch.bfloat16, seed=5).t()
    want = norm64([a, b])
    assert abs(float(gradients.global_norm([a, b])) - want) <= 2 * U * want
    ra = a.double() / (want + 1e-6)
    out = [torch.empty_like(a), torch.empty_like(b, dtype=torch.float32)]
    gradients.clip_by_global_norm([a, b], 1.0, out=out)
    assert ((out[0].double() - ra).abs() <= ra.abs() * 4 * U).all()
    gradients.clip_by_global_norm([a, b], 1.0)
    assert torch.equal(a, out[0])


@gpu
def test_a_tensor_of_more_than_2_to_the_31_elements():
    n = (1 << 31) + 4099
    t = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    t[0], t[1 << 31], t[-1] = 3.0, 4.0, 12.0
    assert float(gradients.global_norm([t])) == 13.0
    gradients.clip_by_global_norm([t], 6.5)
    # 0.5 is the coefficient up to the 1e-6: a relative 8e-8, far below bfloat16's half step
    assert [float(t[i]) for i in (0, 1 << 31, n - 1)] == [1.5, 2.0, 6.0]


@gpu
def test_parameters():
    ps = [torch.nn.Parameter(rand((50, 3), seed=i)) for i in range(3)] + [torch.nn.Parameter(rand((4,)))]
    for i, p in enumerate(ps[:3]):
        p.grad = rand((50, 3), seed=10 + i)
    before = [p.grad.clone() for p in ps[:3]]
    want = norm64(before)
    norm = gradients.clip_grad_norm_(iter(ps + ps), 0.5)       # given twice: counted once
    assert abs(float(norm) - want) <= 2 * U * want
    for p, b in zip(ps, before):
        ref = b.double() * 0.5 / (want + 1e-6)
        assert ((p.grad.double() - ref).abs() <= ref.abs() * 4 * U).all()
    assert float(gradients.clip_grad_norm_([ps[3]], 1.0)) == 0.0
    assert abs(float(gradients.clip_grad_norm_(ps[0], 1e9)) - norm64([ps[0].grad])) <= 2 * U * want


@gpu
def test_refusals_on_the_device():
    a, b = rand((64,)), rand((64, 8))
    clip = gradients.clip_by_global_norm
    for call in (lambda: gradients.global_norm([]),
                 lambda: gradients.global_norm([a.double()]),
                 lambda: gradients.global_norm([a, b[:, :3]]),
                 lambda: gradients.global_norm([a.cpu()]),
                 lambda: gradients.global_norm([a, a.cpu()]),
                 lambda: gradients.global_norm([a[:1].expand(64)]),
                 lambda: gradients.global_norm([b.to_sparse()]),
                 lambda: gradients.global_norm([a], 3.0),
                 lambda: clip([a], -1.0),
                 lambda: clip([a], float("nan")),
                 lambda: clip([a], 1.0, out=[a, a]),
                 lambda: clip([a], 1.0, out=[b]),
                 lambda: clip([a], 1.0, out=[a.bfloat16()]),
                 lambda: clip([a, a], 1.0),
                 lambda: clip([b, b[:2]], 1.0),
                 lambda: clip([a[:32], a[16:48]], 1.0, out=[torch.empty_like(a[:32]), a[32:64]]),
                 lambda: clip([a[:32]], 1.0, out=[a[8:40]]),
                 lambda: clip([b], 1.0, out=[torch.empty((8, 64), device=DEV).t()])):
        with pytest.raises(_lib.VingsError):
            call()


@gpu
def test_other_stream_and_replayed_graph():
    ts = make("splats") + make("many")
    out = [torch.empty_like(t) for t in ts]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n1 = gradients.global_norm(ts)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(n1, gradients.global_norm(ts))
    gradients.clip_by_global_norm(ts, 1.0, out=out)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        norm = gradients.clip_by_global_norm(ts, 1.0, out=out)
    with torch.cuda.graph(other, pool=graph.pool()):
        big = gradients.global_norm(ts, float("inf"))
    for seed in range(4):
        for i, t in enumerate(ts):
            t.copy_(rand(t.shape, t.dtype, seed=100 * seed + i, scale=seed + 0.5))
        graph.replay()
        other.replay()
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.empty_like(t) for t in ts]
        assert torch.equal(norm, gradients.clip_by_global_norm(ts, 1.0, out=eager))
        assert torch.equal(big, gradients.global_norm(ts, float("inf")))
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


# ---------------------------------------------------------------------------
# the clipped row-masked Adam step
# ---------------------------------------------------------------------------
def adam_state(n, widths, seed=0, offset=0):
    def arr(w, k, scale):
        flat = rand((n * w + offset,), seed=1000 * seed + 10 * w + k, scale=scale)
        return flat[offset:].view(n, w)
    ps = [arr(w, 0, 1.0) for w in widths]
    gs = [arr(w, 1, 0.05) for w in widths]
    ms = [arr(w, 2, 0.01) for w in widths]
    vs = [arr(w, 3, 0.01).square_() for w in widths]
    vis = (torch.rand(n, generator=torch.Generator().manual_seed(seed)) < 0.6).to(DEV)
    return ps, gs, ms, vs, vis


def optimizer(ps, gs, ms, vs, lrs=None, **group_extra):
    params = [torch.nn.Parameter(p.clone() if p.storage_offset() == 0 else p) for p in ps]
    opt = surfel.SparseGaussianAdam(
        [dict({"params": [p], "lr": (lrs or [0.01] * 99)[i], "name": str(i)}, **group_extra)
         for i, p in enumerate(params)], lr=0.0, eps=1e-15)
    for p, g, m, v in zip(params, gs, ms, vs):
        p.grad = g
        opt.state[p] = {"step": torch.tensor(0.0), "exp_avg": m.clone() if m.storage_offset() == 0 else m,
                        "exp_avg_sq": v.clone() if v.storage_offset() == 0 else v}
    return opt, params


def check_step(before, after, vis, coef, lr, b1=0.9, b2=0.999, eps=1e-15):
    """Reference in float64 with the update's own float32 constants.  Errors, S = |b1 m| +
    |(1-b1) g'|: the gradient carries 3 u (norm, coefficient, product), the first moment 6 u S, the
    second (all terms positive) 12 u of itself, the step 6 u for its root, quotient and products."""
    f = lambda x: float(torch.tensor(x, dtype=torch.float32))
    one_b1, one_b2 = f(1.0 - b1), f(1.0 - b2)
    p, g, m, v = (x.double() for x in before)
    g = g * coef
    m2 = f(b1) * m + one_b1 * g
    v2 = f(b2) * v + one_b2 * g * g
    size = (f(b1) * m).abs() + (one_b1 * g).abs()
    step = f(lr) / (v2.sqrt() + f(eps))
    p2 = p - step * m2
    seen = vis[:, None].expand_as(p)
    for got, want, old, tol in ((after[1], m2, before[2], 6 * U * size), (after[2], v2, before[3], 12 * U * v2),
                                (after[0], p2, before[0], U * p2.abs() + step * (6 * U * size + 12 * U * m2.abs()))):
        assert ((got.double() - want).abs() <= tol)[seen].all()
        assert torch.equal(got[~seen], old[~seen])


@gpu
@pytest.mark.parametrize("n,widths,offset", [(1, (3, 3, 1, 2, 4), 0), (3, (1,), 0), (1023, (3, 3, 1, 2, 4), 0),
                                             (20001, (3, 3, 1, 2, 4), 0), (777, (5, 7, 12, 64, 129), 0),
                                             (777, (3, 1, 4, 6), 1), (50, tuple(range(1, 20)), 0)])
@pytest.mark.parametrize("share", [0.2, 5.0])
def test_clipped_step(n, widths, offset, share):
    ps, gs, ms, vs, vis = adam_state(n, widths, seed=n, offset=offset)
    before = [tuple(x.clone() for x in t) for t in zip(ps, gs, ms, vs)]
    want = norm64([g[vis] for g in gs]) if vis.any() else 0.0
    max_norm = share * want if want else 1.0
    coef = min(1.0, max_norm / (want + 1e-6))
    opt, params = optimizer(ps, gs, ms, vs)
    norm = opt.step(vis, n, max_norm=max_norm)
    assert abs(float(norm) - want) <= 2 * U * want
    for p, b in zip(params, before):
        st = opt.state[p]
        assert torch.equal(p.grad, b[1])                       # the gradients are not written
        check_step(b, (p.detach(), st["exp_avg"], st["exp_avg_sq"]), vis, coef, 0.01)


@gpu
def test_step_without_need_to_clip_is_the_plain_step():
    """One step: the two differ by their factors 1 - beta alone, float32(1) - float32(0.999) being
    1.3e-5 off and float32(1) - float32(0.9) 2.4e-7, and by the roundings counted in check_step."""
    data = adam_state(30011, (3, 3, 1, 2, 4), seed=2)
    a, pa = optimizer(*data[:4])
    b, pb = optimizer(*data[:4])
    vis = data[4]
    assert a.step(vis, 30011) is None
    b.step(vis, 30011, max_norm=1e9)
    for x, y, g in zip(pa, pb, data[1]):
        ma, mb = a.state[x]["exp_avg"], b.state[y]["exp_avg"]
        va, vb = a.state[x]["exp_avg_sq"], b.state[y]["exp_avg_sq"]
        assert ((ma - mb).abs() <= 2.5e-7 * 0.1 * g.abs() + 8 * U * (ma.abs() + 0.2 * g.abs())).all()
        assert ((va - vb).abs() <= 1.4e-5 * 0.001 * g * g + 8 * U * va).all()
        assert torch.equal(x[~vis], y[~vis]) and not torch.equal(x[vis], y.detach()[vis] + 1)


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_step_of_a_gradient_that_is_not_finite(bad):
    data = adam_state(5000, (3, 1), seed=3)
    vis = data[4]
    row = int(vis.nonzero()[7])
    data[1][0][row, 1] = bad
    opt, ps = optimizer(*data[:4])
    before = [p.detach().clone() for p in ps]
    norm = float(opt.step(vis, 5000, max_norm=1.0))
    assert not math.isfinite(norm)
    assert all(torch.equal(p, b) for p, b in zip(ps, before))
    assert all(torch.equal(opt.state[p]["exp_avg"], m) for p, m in zip(ps, data[2]))
    # ... but not if it lies in a row that is not stepped
    vis = vis.clone()
    vis[row] = False
    assert math.isfinite(float(opt.step(vis, 5000, max_norm=1.0)))
    assert not torch.equal(ps[0], before[0])
    assert torch.equal(ps[0][row], before[0][row])


@gpu
def test_step_groups_with_their_own_constants():
    n = 4000
    ps, gs, ms, vs, vis = adam_state(n, (3, 2, 4), seed=5)
    params = [torch.nn.Parameter(p.clone()) for p in ps]
    extra = [dict(betas=(0.9, 0.999), eps=1e-15), dict(betas=(0.5, 0.9), eps=1e-3), dict(betas=(0.9, 0.999), eps=1e-15)]
    opt = surfel.SparseGaussianAdam([dict(params=[p], lr=0.1 * (i + 1), **e) for i, (p, e) in enumerate(zip(params, extra))],
                                    lr=0.0, eps=1e-15)
    for p, g, m, v in zip(params, gs, ms, vs):
        p.grad = g
        opt.state[p] = {"step": torch.tensor(0.0), "exp_avg": m.clone(), "exp_avg_sq": v.clone()}
    want = norm64([g[vis] for g in gs])
    opt.step(vis, n, max_norm=0.5)
    coef = min(1.0, 0.5 / (want + 1e-6))
    for i, p in enumerate(params):
        st = opt.state[p]
        b1, b2 = extra[i]["betas"]
        check_step((ps[i], gs[i], ms[i], vs[i]), (p.detach(), st["exp_avg"], st["exp_avg_sq"]), vis, coef,
                   0.1 * (i + 1), b1, b2, extra[i]["eps"])


@gpu
def test_step_edges_and_refusals():
    ps, gs, ms, vs, vis = adam_state(100, (3, 1), seed=6)
    opt, params = optimizer(ps, gs, ms, vs)
    before = [p.detach().clone() for p in params]
    none = torch.zeros_like(vis)
    assert float(opt.step(none, 100, max_norm=1.0)) == 0.0
    assert all(torch.equal(a, b) for a, b in zip(params, before))
    with pytest.raises(_lib.VingsError):
        opt.step(vis, 99, max_norm=1.0)
    with pytest.raises(_lib.VingsError):
        opt.step(vis, 100, max_norm=-1.0)
    with pytest.raises(_lib.VingsError):
        opt.step(vis, 100, max_norm=float("nan"))
    moment = opt.state[params[0]]["exp_avg"]
    for wrong in (moment.double(), moment[:50], moment.cpu()):
        opt.state[params[0]]["exp_avg"] = wrong
        with pytest.raises(_lib.VingsError):
            opt.step(vis, 100, max_norm=1.0)
    opt.state[params[0]]["exp_avg"] = moment
    guard = torch.tensor([11], dtype=torch.int32, device=DEV)
    norm = opt.step(vis, 100, guard=(guard.data_ptr(), 10), max_norm=1.0)       # does not fit: dropped
    assert float(norm) > 0 and all(torch.equal(a, b) for a, b in zip(params, before))
    opt.step(vis, 100, guard=(guard.data_ptr(), 11), max_norm=1.0)
    assert not torch.equal(params[0], before[0])
    for p in params:
        p.grad = None
    assert float(opt.step(vis, 100, max_norm=1.0)) == 0.0
    empty, _ = optimizer([torch.empty((0, 3), device=DEV)], [torch.empty((0, 3), device=DEV)],
                         [torch.empty((0, 3), device=DEV)], [torch.empty((0, 3), device=DEV)])
    assert float(empty.step(torch.empty(0, dtype=torch.bool, device=DEV), 0, max_norm=1.0)) == 0.0


@gpu
def test_step_on_more_than_2_to_the_31_elements():
    w = 64
    n = (1 << 31) // w + 3
    p = torch.zeros((n, w), device=DEV)
    g = torch.zeros((n, w), device=DEV)
    m, v = torch.zeros((n, w), device=DEV), torch.zeros((n, w), device=DEV)
    vis = torch.zeros(n, dtype=torch.bool, device=DEV)
    vis[0], vis[n - 2] = True, True
    g[0, 0], g[n - 2, w - 1], g[n - 1, 5] = 3.0, 4.0, 100.0
    par = torch.nn.Parameter(p)
    opt = surfel.SparseGaussianAdam([{"params": [par], "lr": 0.1}], lr=0.0, eps=1e-15)
    opt.state[par] = {"step": torch.tensor(0.0), "exp_avg": m, "exp_avg_sq": v}
    par.grad = g
    assert float(opt.step(vis, n, max_norm=1e9)) == 5.0
    # 0.1 rounded to float32, and the product
    assert float(m[0, 0]) == pytest.approx(0.3, rel=2 * U) and float(m[n - 2, w - 1]) == pytest.approx(0.4, rel=2 * U)
    assert int((m != 0).sum()) == 2 and int((par.detach() != 0).sum()) == 2


@gpu
@pytest.mark.parametrize("n,w", [((1 << 31) - 8000, 1), ((1 << 31) - 1, 1), ((1 << 30) + 1, 2), (715827890, 3)])
def test_step_of_narrow_rows_by_64_bit_indexes(n, w):
    """Four consecutive elements lie in up to four rows; every row keeps its own visibility."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("60 GB of free memory")
    p, g, m, v = (torch.zeros((n, w), device=DEV) for _ in range(4))
    vis = torch.zeros(n, dtype=torch.bool, device=DEV)
    ends = [(0, (0, 2, 3, 5, 7)), (n - 9, (0, 1, 3, 6, 8))]
    for first, rows in ends:
        g[first:first + 9] = 1.0
        for r in rows:
            vis[first + r] = True
    par = torch.nn.Parameter(p)
    opt = surfel.SparseGaussianAdam([{"params": [par], "lr": 0.1}], lr=0.0, eps=1e-15)
    opt.state[par] = {"step": torch.tensor(0.0), "exp_avg": m, "exp_avg_sq": v}
    par.grad = g
    norm = opt.step(vis, n, max_norm=1e9)
    assert float(norm) == pytest.approx((10 * w) ** 0.5, rel=2 * U)
    for first, rows in ends:
        for t in (par.detach(), m, v):
            moved = (t[first:first + 9] != 0).cpu()
            assert torch.equal(moved, torch.tensor([r in rows for r in range(9)])[:, None].expand(9, w))
    assert int((m[9:n - 9] != 0).sum()) == 0


@gpu
def test_step_of_more_rows_than_31_bits_is_refused():
    opt, _ = optimizer(*adam_state(100, (3, 1), seed=6)[:4])
    with pytest.raises(_lib.VingsError):
        opt.step(torch.zeros((1 << 31) + 4, dtype=torch.bool, device=DEV), (1 << 31) + 4, max_norm=1.0)


@gpu
def test_captured_step():
    data = adam_state(20000, (3, 3, 1, 2, 4), seed=8)
    vis = data[4]
    a, pa = optimizer(*data[:4])
    b, pb = optimizer(*data[:4])
    for p, q in zip(pa, pb):
        q.grad = q.grad.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    state0 = [x.detach().clone() for p in pa for x in (p, a.state[p]["exp_avg"], a.state[p]["exp_avg_sq"])]
    with torch.cuda.graph(graph):
        norm = a.step(vis, 20000, max_norm=0.7)
    for x, y in zip([x for p in pa for x in (p, a.state[p]["exp_avg"], a.state[p]["exp_avg_sq"])], state0):
        assert torch.equal(x, y)                               # capturing runs nothing
    for k in range(3):
        for p, q in zip(pa, pb):
            p.grad.copy_(rand(p.shape, seed=50 + k, scale=0.1 * k + 0.01))
            q.grad.copy_(p.grad)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, b.step(vis, 20000, max_norm=0.7))
        for p, q in zip(pa, pb):
            assert torch.equal(p, q) and torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])


def _mapper(max_grad_norm):
    raw = synth.make_splats(2000, 160, 96)
    return harness.SurfelMapper(raw, DEV, max_grad_norm=max_grad_norm), raw


@gpu
def test_mapper_view_steps_clip():
    """The autograd, the fused and the captured view step under one max_grad_norm."""
    intr = synth.intrinsic_for(160, 96)
    c2w = torch.eye(4, device=DEV)
    plain, raw = _mapper(None)
    with torch.no_grad():
        gtp = harness.render({k: v.to(DEV) for k, v in synth.perturb_splats(raw).items()}, c2w, intr)
    gt = lambda: {"rgb": gtp["rgb"].clone(), "depth": gtp["depth"].clone(), "depth_cov": torch.ones_like(gtp["depth"])}
    plain.train_view(c2w, intr, gt())
    assert plain.last_grad_norm is None
    loose, _ = _mapper(1e9)
    loose.train_view(c2w, intr, gt())
    full = float(loose.last_grad_norm)
    assert full > 0
    tight, _ = _mapper(full / 8)
    tight.train_view(c2w, intr, gt())
    # (two backward passes of one view differ by the order of the blend's float atomics: 1e-4 as
    # in the parity tests)
    assert abs(float(tight.last_grad_norm) - full) <= 1e-4 * full
    for k in plain.NAMES:
        ma = plain.optimizer.state[plain.params[k]]["exp_avg"].double()
        mb = tight.optimizer.state[tight.params[k]]["exp_avg"].double()
        assert float((ma / 8 - mb).norm()) <= 2e-4 * float(ma.norm()) / 8
    settings = harness.view_settings(torch.eye(4, device=DEV), intr)
    fused, _ = _mapper(full / 8)
    graphed, _ = _mapper(full / 8)
    gf, gg = gt(), gt()
    R = torch.eye(3)
    for _ in range(4):
        fused.fused_view(settings, intr, gf, R)
        graphed.fused_view_graphed("kf", settings, intr, gg, R)
        nf, ng = float(fused.last_grad_norm), float(graphed.last_grad_norm)
        assert nf > 0 and abs(nf - ng) <= 1e-2 * nf


@gpu
def test_a_dropped_step_reports_no_norm():
    """The gradients of a step that its guard drops are incomplete, or another step's: their norm is
    none of this step's.  Infinity says so, as the norm of every skipped step is not finite."""
    ps, gs, ms, vs, vis = adam_state(5000, (3, 1), seed=16)
    opt, params = optimizer(ps, gs, ms, vs)
    guard = torch.tensor([11], dtype=torch.int32, device=DEV)
    first = float(opt.step(vis, 5000, guard=(guard.data_ptr(), 11), max_norm=1.0))
    assert math.isfinite(first) and first > 0
    before = [x.clone() for p in params for x in (p.detach(), *list(opt.state[p].values())[1:])]
    assert float(opt.step(vis, 5000, guard=(guard.data_ptr(), 10), max_norm=1.0)) == math.inf
    after = [x for p in params for x in (p.detach(), *list(opt.state[p].values())[1:])]
    assert all(torch.equal(x, y) for x, y in zip(before, after))
    gs[0][int(vis.nonzero()[0]), 0] = float("nan")               # ... whatever they hold
    assert float(opt.step(vis, 5000, guard=(guard.data_ptr(), 10), max_norm=1.0)) == math.inf


@gpu
def test_a_dropped_view_step_reports_no_norm():
    """The same of a captured view whose instances outgrew its graph, behind a step of another view."""
    intr = synth.intrinsic_for(256, 160)
    raw = synth.make_splats(5000, 256, 160, n_views=2, seed=72)
    mapper = harness.SurfelMapper(raw, DEV, max_grad_norm=0.1)
    views = []
    for c2w in synth.window_poses(2):
        w2c = torch.linalg.inv(c2w).to(DEV)
        with torch.no_grad():
            pr = harness.render({k: v.to(DEV) for k, v in synth.perturb_splats(raw).items()}, w2c, intr)
        gt = {"rgb": pr["rgb"].clone(), "depth": pr["depth"].clone(), "depth_cov": torch.ones_like(pr["depth"])}
        views.append((harness.view_settings(w2c, intr), gt, w2c[:3, :3].cpu()))
    step = lambda k: mapper.fused_view_graphed(k, views[k][0], intr, views[k][1], views[k][2], k)
    step(0), step(1)
    ent = mapper._view_graphs[0]
    assert ent["D"] > 8000
    ent["D"] = 64
    step(0)                                                      # captured with too little room: dropped
    torch.cuda.synchronize()
    assert int(ent["count"][2]) > ent["capacity"]
    assert float(mapper.last_grad_norm) == math.inf
    step(1)
    assert 0 < float(mapper.last_grad_norm) < math.inf
    step(0)                                                      # repeated, and captured with room
    assert 0 < float(mapper.last_grad_norm) < math.inf


@gpu
def test_step_counts_as_written():
    """Parameters and moments that autograd saved before a clipped step are noticed in the backward pass."""
    ps, gs, ms, vs, vis = adam_state(100, (3, 1), seed=6)
    opt, params = optimizer(ps, gs, ms, vs)
    arrays = [t for p in params for t in (p, opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"])]
    versions = [t._version for t in arrays]
    product = params[0] * params[0]
    opt.step(vis, 100, max_norm=1.0)
    assert all(t._version > v for t, v in zip(arrays, versions))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()


@gpu
def test_fused_and_captured_view_steps_apply_the_clipped_gradient():
    """Their moments, not only the norm they report: this Adam moves parameters alike whatever the
    gradients' scale.  From equal maps the moments of a step on g * c are c and c^2 times those on g;
    two backward passes differ by 1e-4 of their norm (the order of the blend's atomics), here an
    eighth and a 64th are told from 1.  The captured step (second call) starts from maps that
    moved apart by such differences; without the coefficient its first moments would be 4.7 times
    those of the eager one."""
    intr = synth.intrinsic_for(160, 96)
    raw = synth.make_splats(2000, 160, 96)
    eye = torch.eye(4, device=DEV)
    with torch.no_grad():
        gtp = harness.render({k: v.to(DEV) for k, v in synth.perturb_splats(raw).items()}, eye, intr)
    settings, R = harness.view_settings(eye, intr), torch.eye(3)

    def mapper(max_norm):
        gt = {"rgb": gtp["rgb"].clone(), "depth": gtp["depth"].clone(), "depth_cov": torch.ones_like(gtp["depth"])}
        return harness.SurfelMapper(raw, DEV, max_grad_norm=max_norm), gt

    def moments(m, k):
        st = m.optimizer.state[m.params[k]]
        return st["exp_avg"].double(), st["exp_avg_sq"].double()

    def near(a, b, tol):
        assert float(b.norm()) > 0 and float((a - b).norm()) <= tol * float(b.norm())

    loose, gt = mapper(1e9)
    loose.fused_view(settings, intr, gt, R)
    full = float(loose.last_grad_norm)
    coef = (full / 8) / (full + 1e-6)
    fused, gf = mapper(full / 8)
    graphed, gg = mapper(full / 8)
    fused.fused_view(settings, intr, gf, R)
    graphed.fused_view_graphed("kf", settings, intr, gg, R)
    for m in (fused, graphed):
        for k in m.NAMES:
            (a1, a2), (b1, b2) = moments(m, k), moments(loose, k)
            near(a1, coef * b1, 1e-2)
            near(a2, coef * coef * b2, 2e-2)
    fused.fused_view(settings, intr, gf, R)
    graphed.fused_view_graphed("kf", settings, intr, gg, R)
    assert graphed._view_graphs["kf"]["graph"] is not None
    for k in fused.NAMES:
        (a1, a2), (b1, b2) = moments(graphed, k), moments(fused, k)
        near(a1, b1, 0.1)
        near(a2, b2, 0.2)


def test_compact_exchange_refuses_clipping():
    class Reducer:
        world, compact, n = 2, True, 4
    mapper = harness.SurfelMapper.__new__(harness.SurfelMapper)
    mapper.max_grad_norm = 1.0
    with pytest.raises(_lib.VingsError, match="compact"):
        mapper.fused_view(None, None, None, None, reducer=Reducer())


@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=gpu)])
def test_forward_mode_tangents_are_refused(device):
    """They would be lost: kernels that take addresses see the values alone."""
    fwd = torch.autograd.forward_ad
    with fwd.dual_level():
        for leaf in (False, True):
            plain = torch.ones(4, device=device)
            dual = fwd.make_dual(torch.ones(4, device=device, requires_grad=leaf), plain.clone())
            calls = [lambda: gradients.global_norm([plain, dual]), lambda: gradients.global_norm(dual),
                     lambda: gradients.clip_by_global_norm([dual], 1.0)]
            if device != "cpu":                      # (there the gradients are refused before the results)
                calls.append(lambda: gradients.clip_by_global_norm([plain], 1.0, out=[dual]))
            for call in calls:
                with pytest.raises(_lib.VingsError, match="tangent"):
                    call()
                with torch.no_grad(), pytest.raises(_lib.VingsError, match="tangent"):
                    call()


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.VingsError):
        gradients.global_norm([torch.ones(3)])
    with pytest.raises(_lib.VingsError):
        gradients.clip_by_global_norm([torch.ones(3)], 1.0)
    with pytest.raises(_lib.VingsError):
        gradients.global_norm([])
    with pytest.raises(_lib.VingsError):
        gradients.global_norm(torch.ones(2), 3.0)


# ---------------------------------------------------------------------------
# argument checks of the C entry points: they fail before the first HIP call
# ---------------------------------------------------------------------------
host_only = pytest.mark.skipif(torch.cuda.is_available(), reason="host-only argument checks")
FAKE = 0x10000


def _list(values, kind):
    return (kind * len(values))(*values)


def _clip(ins, outs, numels, types, out_types, kind=0, max_norm=1.0, norm=FAKE, ws=FAKE, ws_bytes=1 << 20):
    P = lambda v: _list(v, ctypes.c_void_p)
    return _lib.lib().vings_grad_clip(len(ins), P(ins), P(outs), _list(numels, ctypes.c_int64), _list(types, ctypes.c_int),
                                      _list(out_types, ctypes.c_int), kind, max_norm, norm, ws, ws_bytes, None)


def _error():
    return _lib.lib().vings_last_error().decode()


@host_only
def test_clip_arguments():
    ok = dict(ins=[FAKE * 2], outs=[FAKE * 4], numels=[100], types=[0], out_types=[0])
    for change, text in ((dict(kind=2), "norm kind"), (dict(max_norm=-1.0), "max_norm"),
                         (dict(max_norm=float("nan")), "max_norm"), (dict(norm=None), "null pointer"),
                         (dict(types=[7]), "element type"), (dict(numels=[-1]), "sizes"),
                         (dict(ins=[None]), "null pointer"), (dict(outs=[None]), "null pointer"),
                         (dict(out_types=[1]), "own type"), (dict(ins=[FAKE * 2 + 2]), "alignment"),
                         (dict(ws_bytes=0), "too small"), (dict(ws=FAKE + 4), "8-byte"),
                         (dict(outs=[FAKE * 2 + 8]), "overlaps")):
        assert _clip(**{**ok, **change}) != 0 and text in _error(), change
    two = dict(ins=[FAKE * 2, FAKE * 4], outs=[FAKE * 2, FAKE * 2 + 64], numels=[100, 100], types=[0, 0], out_types=[0, 0])
    assert _clip(**two) != 0 and "overlaps" in _error()
    # widening in place: the output is longer than its input's memory
    assert _clip([FAKE * 2], [FAKE * 2], [100], [1], [0]) != 0 and "overlaps" in _error()


@host_only
def test_norm_workspace_grows_with_the_list():
    f = _lib.lib().vings_grad_norm_workspace_bytes
    size = lambda numels: f(len(numels), _list(numels, ctypes.c_int64))
    assert size([0, 0]) >= 0 and size([10]) >= 8
    assert size([1 << 30]) == 8 * 1024                     # one launch: 1024 partial results at most
    assert size([100] * 1000) >= 8 * 7


@host_only
def test_clipped_step_arguments():
    L = _lib.lib()
    one = lambda x, t=ctypes.c_void_p: _list([x], t)
    F = ctypes.c_float

    def call(n=1, p=FAKE, g=FAKE, width=3, vis=FAKE, N=5, max_norm=1.0, norm=FAKE, ws=FAKE, ws_bytes=1 << 20):
        return L.vings_sparse_adam_clipped(n, one(p), one(g), one(FAKE), one(FAKE), one(width, ctypes.c_int), one(0.1, F),
                                           one(0.9, F), one(0.999, F), one(1e-15, F), vis, N, max_norm, norm, ws, ws_bytes,
                                           None, 0, None)
    for change, text in ((dict(n=0), "groups"), (dict(n=65), "groups"), (dict(N=-1), "sizes"), (dict(max_norm=-0.5), "max_norm"),
                         (dict(norm=None), "null pointer"), (dict(ws=None), "null pointer"), (dict(ws=FAKE + 4), "8-byte"),
                         (dict(ws_bytes=8), "too small"), (dict(vis=None), "null pointer"), (dict(width=0), "widths"),
                         (dict(g=None), "group pointers"), (dict(p=FAKE + 2), "4-byte")):
        assert call(**change) != 0 and text in _error(), change
