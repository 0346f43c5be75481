"""Scaled row lookup, its gradient by sorted ids, and a run of both with the clipped row-masked
step, against their formulas in float64.

Tolerances (u = 2^-24, h_t = eps/2 of the result's type): the lookup's product u + h_t.  A row of
the gradient is a float32 sum whose longest chain of additions is at most 64 inside a lane group,
8 in the scan over the groups, one per partial row that a lane group of the join adds and 8 in the
join's tree.  Partial rows: a piece of the sorted form holds 16 ids or more and at least four
groups share them, a tile of the few-rows form holds one id of the row or more and at least
sixteen groups share them, so a group adds count / 16 + 1 at most: (82 + count / 16) u of the sum
of magnitudes, then u for the scale and h_t; float16 adds half its smallest step."""
import threading

import pytest
import torch

from vings_mono_amd import _lib, gradients, row_table, surfel

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}
gpu = pytest.mark.gpu


def rand(shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def make_ids(n, rows, how, seed=0, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed + 77)
    if how == "uniform":
        ids = torch.randint(0, rows, (n,), generator=g)
    elif how == "one":
        ids = torch.full((n,), rows // 2)
    elif how == "power":
        ids = (rows * torch.rand(n, generator=g) ** 6).long().clamp(0, rows - 1)
    elif how == "sorted":
        ids = torch.arange(n) * rows // max(n, 1)
    elif how == "none":
        ids = torch.full((n,), -1)
    else:                                        # ids that name no row among the others
        ids = torch.randint(-2, rows + 2, (n,), generator=g)
        ids[::7] = -(2 ** 31) if dtype == torch.int32 else -(2 ** 62)
        ids[3::11] = 2 ** 31 - 1 if dtype == torch.int32 else 2 ** 40 + 1
    return ids.to(dtype).to(DEV)


def lookup64(table, ids, scale):
    found = (ids >= 0) & (ids < table.shape[0])
    out = table.double().new_zeros(tuple(ids.shape) + (table.shape[1],))
    out[found] = table.double()[ids[found].long()] * scale
    return out


def backward64(grad, ids, rows, padding=None):
    """(sums, sums of magnitudes, counts) by the definition, unscaled."""
    ids = ids.reshape(-1).long()
    g = grad.reshape(ids.numel(), -1).double()
    keep = (ids >= 0) & (ids < rows)
    if padding is not None:
        keep &= ids != padding
    count = torch.bincount(ids[keep], minlength=rows)
    g = g[keep][torch.argsort(ids[keep], stable=True)]
    add = lambda x: torch.segment_reduce(x, "sum", lengths=count, initial=0.0)
    return add(g), add(g.abs()), count


def check_backward(grad, ids, rows, scale, got, touched, padding=None):
    total, size, count = backward64(grad, ids, rows, padding)
    f = float(torch.tensor(scale, dtype=torch.float32))
    ref = total * f
    tol = (82 + count[:, None] / 16) * U * size * abs(f) + (U + HALF[got.dtype]) * ref.abs()
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert got.shape == ref.shape
    assert ((got.double() - ref).abs() <= tol).all()
    assert not got[count == 0].any()
    assert torch.equal(touched.bool(), count > 0)


SHAPES = [(1, 1, 1), (1, 5, 4), (5, 3, 3), (64, 7, 8), (300, 77, 3), (1000, 80, 12), (1025, 300, 130), (4097, 513, 33),
          (333, 1000, 257), (77, 50, 513), (40, 33, 2048), (16384, 90, 5), (2000, 40, 1030)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,cols", SHAPES)
def test_lookup(n, rows, cols, dtype):
    table = rand((rows, cols), dtype, seed=n)
    for id_type in (torch.int64, torch.int32):
        for how in ("uniform", "strays", "none"):
            ids = make_ids(n, rows, how, dtype=id_type)
            for scale in (1.0, 11.3137):
                out = row_table.lookup_rows(table, ids, scale=scale)
                ref = lookup64(table, ids, float(torch.tensor(scale, dtype=torch.float32)))
                floor = 2.0 ** -25 if dtype == torch.float16 else 0.0
                assert out.dtype == dtype and out.shape == ref.shape
                assert ((out.double() - ref).abs() <= ref.abs() * (U + HALF[dtype]) + floor).all()


@gpu
@pytest.mark.parametrize("how", ["uniform", "one", "power", "sorted", "none", "strays"])
@pytest.mark.parametrize("n,rows,cols", SHAPES + [(16385, 70000, 8), (50001, 300, 9), (200003, 80, 12), (70000, 3, 2),
                                                  (20000, 5, 640), (30000, 60000, 20), (3000, 255, 4), (3000, 256, 4),
                                                  (90001, 1999, 64), (1024, 4095, 16), (1025, 4095, 3), (5000, 4096, 16),
                                                  (40000, 257, 60), (2600, 700, 68), (32768, 5000, 12),
                                                  (32769, 5000, 12), (9000, 70000, 24), (17000, 4097, 300)])
def test_backward(n, rows, cols, how):
    dtype = TYPES[(n + cols) % 3]
    id_type = (torch.int64, torch.int32)[(n + rows) % 2]
    grad = rand((n, cols), dtype, seed=cols, scale=0.1)
    ids = make_ids(n, rows, how, dtype=id_type)
    for out_type in {dtype, torch.float32}:
        out = torch.full((rows, cols), 9.0, dtype=out_type, device=DEV)
        got, touched = row_table.lookup_rows_backward(grad, ids, rows, scale=0.75, out=out)
        assert got is out
        check_backward(grad, ids, rows, 0.75, got, touched)
    again, t2 = row_table.lookup_rows_backward(grad, ids, rows, scale=0.75)
    first, _ = row_table.lookup_rows_backward(grad, ids, rows, scale=0.75)
    assert torch.equal(again, first) and torch.equal(t2, touched)


@gpu
@pytest.mark.parametrize("how", ["uniform", "one", "strays"])
@pytest.mark.parametrize("n,rows,cols", [(n, r, c) for n in (131071, 131072, 131073, 300001)
                                         for r, c in ((5000, 8), (70000, 5), (4000, 72))] + [(4300001, 70000, 5)])
def test_sort_by_tiles(n, rows, cols, how):
    """Up to 64 tiles of 2048 ids and above; 4 300 001 ids are two rounds of the scan."""
    grad, ids = rand((n, cols), seed=cols), make_ids(n, rows, how)
    out = torch.full((rows, cols), 9.0, device=DEV)
    got, touched = row_table.lookup_rows_backward(grad, ids, rows, out=out)
    check_backward(grad, ids, rows, 1.0, got, touched)
    again, _ = row_table.lookup_rows_backward(grad, ids.int() if how == "uniform" else ids, rows)
    assert torch.equal(again, got)


@gpu
@pytest.mark.parametrize("bits", [1, 7, 8, 9, 16, 17, 24, 30])
@pytest.mark.parametrize("n", [700, 3000, 12000, 40000])
def test_sort_over_every_number_of_passes(n, bits):
    """Tables whose row numbers take one to four radix passes; the rows themselves are one column."""
    rows = (1 << bits) - 1
    ids = make_ids(n, rows, "uniform", seed=bits)
    ids[:5] = rows - 1
    grad = rand((n, 1), seed=3)
    got, touched = row_table.lookup_rows_backward(grad, ids, rows)
    uniq, where = ids.unique(return_inverse=True)
    total = torch.zeros(len(uniq), dtype=torch.float64, device=DEV).index_add_(0, where, grad[:, 0].double())
    size = torch.zeros_like(total).index_add_(0, where, grad[:, 0].double().abs())
    count = torch.bincount(where)
    assert ((got[uniq, 0].double() - total).abs() <= ((82 + count / 16) * U * size + 2 * U * total.abs())).all()
    assert int(touched.sum()) == len(uniq) and touched[uniq].all()
    assert int((got != 0).sum()) <= len(uniq)


@gpu
def test_padding_id():
    table = rand((50, 24), seed=1).requires_grad_()
    ids = make_ids(400, 50, "uniform")
    ids[::3] = 7
    out = row_table.lookup_rows(table, ids, padding_id=7)
    assert torch.equal(out.detach(), table.detach()[ids])            # looked up like any other
    g = rand((400, 24), seed=2)
    out.backward(g)
    got, touched = row_table.lookup_rows_backward(g, ids, 50, padding_id=7)
    assert torch.equal(table.grad, got) and not touched[7] and not got[7].any()
    check_backward(g, ids, 50, 1.0, got, touched, padding=7)


@gpu
def test_empty_and_tiny():
    table = rand((4, 6))
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    assert row_table.lookup_rows(table, none).shape == (0, 6)
    got, touched = row_table.lookup_rows_backward(torch.empty((0, 6), device=DEV), none, 4)
    assert got.shape == (4, 6) and not got.any() and not touched.any()
    no_rows = torch.empty((0, 6), device=DEV)
    ids = torch.tensor([0, -1, 3], device=DEV)
    assert not row_table.lookup_rows(no_rows, ids).any()
    got, touched = row_table.lookup_rows_backward(rand((3, 6)), ids, 0)
    assert got.shape == (0, 6) and touched.shape == (0,)
    one = row_table.lookup_rows(table, torch.tensor(2, device=DEV))
    assert torch.equal(one, table[2])
    got, touched = row_table.lookup_rows_backward(one, torch.tensor(2, device=DEV), 4)
    assert torch.equal(got[2], one) and touched.tolist() == [False, False, True, False]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_unaligned_views(dtype):
    wide = rand((90, 41), dtype, seed=5)
    ids = make_ids(700, 90, "uniform").view(7, 100)
    for table in (wide[:, 3:36], wide[:, :1], wide[5:, 1:34]):
        good = ids.clamp(max=table.shape[0] - 1)
        out = row_table.lookup_rows(table, good)
        assert torch.equal(out, table[good])
    cols_first = rand((33, 90), dtype, seed=6).t()                   # [90, 33] with a column stride
    assert torch.equal(row_table.lookup_rows(cols_first, ids), cols_first[ids])
    flat = ids.reshape(-1)
    g_wide = rand((700, 50), dtype, seed=7)
    for g in (g_wide[:, 1:34], g_wide.t().contiguous().t()[:, :20], rand((1, 33), dtype, seed=8).expand(700, 33)):
        got, touched = row_table.lookup_rows_backward(g, flat, 90)
        check_backward(g, flat, 90, 1.0, got, touched)
    got3, _ = row_table.lookup_rows_backward(g_wide.view(7, 100, 50), ids, 90)
    got2, _ = row_table.lookup_rows_backward(g_wide, flat, 90)
    assert torch.equal(got2, got3)
    strided_ids = torch.stack([flat, flat.flip(0)], 1)[:, 0]
    got4, _ = row_table.lookup_rows_backward(g_wide, strided_ids, 90)
    assert torch.equal(got2, got4)
    base = torch.full((90 * 50 + 3,), 5.0, dtype=dtype, device=DEV)
    out, _ = row_table.lookup_rows_backward(g_wide, flat, 90, out=base[1:-2].view(90, 50))
    assert torch.equal(out, got2) and float(base[0]) == 5 and (base[-2:] == 5).all()


@gpu
@pytest.mark.parametrize("rows", [40, 3000, 5000])
@pytest.mark.parametrize("stride", [1 << 20, (1 << 20) + 8])
def test_gradient_rows_far_apart(rows, stride):
    """The largest row distance that is read where it lies, and one that is copied first: byte
    offsets inside a tile of 1024 rows reach 2^32 there."""
    n = 1100
    far = torch.zeros(n * stride, device=DEV)
    grad = far.as_strided((n, 5), (stride, 1))
    grad.copy_(rand((n, 5), seed=2))
    ids = make_ids(n, rows, "uniform")
    got, touched = row_table.lookup_rows_backward(grad, ids, rows)
    check_backward(grad.contiguous(), ids, rows, 1.0, got, touched)


@gpu
def test_what_stands_behind_unused_ids_is_not_read():
    """Gradient rows of ids that name no row may hold anything."""
    grad = rand((500, 16), seed=1)
    ids = make_ids(500, 20, "uniform")
    ids[100:200] = -1
    clean, _ = row_table.lookup_rows_backward(grad, ids, 20)
    grad[100:200] = float("nan")
    got, _ = row_table.lookup_rows_backward(grad, ids, 20)
    assert torch.equal(got, clean)
    grad[0] = float("inf")
    got, _ = row_table.lookup_rows_backward(grad, ids, 20)
    assert torch.isinf(got[ids[0]]).all() and torch.isfinite(got[torch.arange(20, device=DEV) != ids[0]]).all()


@gpu
def test_autograd_matches_the_formula_and_differences():
    table = rand((30, 5), seed=1).requires_grad_()
    ids = make_ids(200, 30, "strays").view(20, 10)
    weight = rand((20, 10, 5), seed=2)
    out = row_table.lookup_rows(table, ids, scale=1.5)
    (out * weight).sum().backward()
    total, size, count = backward64(weight, ids, 30)
    assert ((table.grad.double() - 1.5 * total).abs() <= 1.5 * (84 + 4) * U * size).all()
    # differences: the loss is linear in the table, so a step of one shows the gradient up to the
    # rounding of the two float64 sums over float32 products
    loss = lambda t: float((row_table.lookup_rows(t, ids, scale=1.5).double() * weight.double()).sum())
    for r, c in ((0, 0), (7, 3), (29, 4)):
        moved = table.detach().clone()
        moved[r, c] += 1.0
        scale = float((lookup64(moved, ids, 1.5).abs() * weight.double().abs()).sum())
        assert abs(loss(moved) - loss(table.detach()) - float(table.grad[r, c])) <= 8 * U * scale
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad((row_table.lookup_rows(table, ids) ** 2).sum(), table, create_graph=True)
        g.sum().backward()


@gpu
def test_two_lookups_of_one_table_in_one_step():
    table = rand((40, 12), seed=3).requires_grad_()
    touched = torch.zeros(40, dtype=torch.bool, device=DEV)
    a, b = make_ids(90, 20, "uniform"), make_ids(30, 40, "uniform", seed=9)
    loss = row_table.lookup_rows(table, a, touched=touched).sum() + \
        (2 * row_table.lookup_rows(table, b, scale=0.5, touched=touched)).sum()
    assert not touched.any()
    loss.backward()
    count = torch.bincount(a, minlength=40) + torch.bincount(b, minlength=40)
    assert torch.equal(touched, count > 0)
    assert torch.equal(table.grad, count[:, None].float().expand(40, 12))    # whole numbers: exact


@gpu
def test_more_than_2_to_the_31_elements():
    rows, cols = (1 << 31) // 2048 + 5, 2048
    table = torch.zeros((rows, cols), dtype=torch.bfloat16, device=DEV)
    ids = torch.tensor([rows - 1, 3, rows - 2, rows - 1], device=DEV)
    table[rows - 1], table[rows - 2] = 2.0, 3.0
    out = row_table.lookup_rows(table, ids, scale=2.0)
    assert out[:, 0].tolist() == [4.0, 0.0, 6.0, 4.0] and out[:, -1].tolist() == [4.0, 0.0, 6.0, 4.0]
    got, touched = row_table.lookup_rows_backward(out, ids, rows, out=table)
    assert got[rows - 1, 5] == 8.0 and got[rows - 2, 2047] == 6.0 and int(touched.sum()) == 3
    assert int((got != 0).sum()) == 2 * cols
    # and a gradient of more than 2^31 elements read
    n = rows
    ids = torch.zeros(n, dtype=torch.int64, device=DEV)
    ids[-1] = 1
    table.zero_()
    table[-1], table[-2] = 1.0, 5.0
    got, _ = row_table.lookup_rows_backward(table, ids, 2)
    assert (got[1] == 1).all() and (got[0] == 5).all()


@gpu
def test_refusals_on_the_device():
    t, ids = rand((5, 4)), torch.zeros(3, dtype=torch.int64, device=DEV)
    g = rand((3, 4))
    for call in (lambda: row_table.lookup_rows(t.double(), ids), lambda: row_table.lookup_rows(t, ids.float()),
                 lambda: row_table.lookup_rows(t, ids.short()), lambda: row_table.lookup_rows(t, ids.cpu()),
                 lambda: row_table.lookup_rows(t[0], ids), lambda: row_table.lookup_rows(t[:, :0], ids),
                 lambda: row_table.lookup_rows(t, ids, touched=torch.zeros(4, dtype=torch.bool, device=DEV)),
                 lambda: row_table.lookup_rows(t, ids, touched=torch.zeros(5, device=DEV)),
                 lambda: row_table.lookup_rows_backward(g, ids, -1), lambda: row_table.lookup_rows_backward(g, ids[:2], 5),
                 lambda: row_table.lookup_rows_backward(g, ids, 5, out=torch.empty((5, 3), device=DEV)),
                 lambda: row_table.lookup_rows_backward(g, ids, 5, out=torch.empty((5, 4), dtype=torch.bfloat16, device=DEV)),
                 lambda: row_table.lookup_rows_backward(g, ids, 5, out=torch.empty((4, 5), device=DEV).t()),
                 lambda: row_table.lookup_rows_backward(t[:3], ids, 5, out=t),
                 lambda: row_table.lookup_rows_backward(g, ids, 2 ** 31)):
        with pytest.raises(_lib.VingsError):
            call()


@gpu
@pytest.mark.parametrize("n", [900, 30000])
def test_other_stream_and_replayed_graph(n):
    rows, cols = 500, 40
    table, g = rand((rows, cols), seed=1), rand((n, cols), seed=2)
    ids = make_ids(n, rows, "power")
    want, wt = row_table.lookup_rows_backward(g, ids, rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = row_table.lookup_rows_backward(g, ids, rows)
        out = row_table.lookup_rows(table, ids)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(out, table[ids])
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = row_table.lookup_rows(table, ids, scale=3.0)
        got, touched = row_table.lookup_rows_backward(g, ids, rows)
    with torch.cuda.graph(other, pool=graph.pool()):
        got2, _ = row_table.lookup_rows_backward(g, ids, rows, scale=2.0)
    for k in range(4):
        ids.copy_(make_ids(n, rows, ("uniform", "one", "strays", "sorted")[k]))
        g.copy_(rand((n, cols), seed=10 + k))
        graph.replay(); other.replay()
        torch.cuda.synchronize()
        e, et = row_table.lookup_rows_backward(g, ids, rows)
        e2, _ = row_table.lookup_rows_backward(g, ids, rows, scale=2.0)
        assert torch.equal(got, e) and torch.equal(touched, et) and torch.equal(got2, e2)
        assert torch.equal(out, row_table.lookup_rows(table, ids, scale=3.0))


@gpu
def test_out_counts_as_written():
    """A tensor that autograd saved and the call then overwrote is noticed in the backward pass."""
    ids, g = make_ids(50, 7, "uniform"), rand((50, 3))
    out = torch.ones((7, 3), device=DEV)
    leaf = torch.ones((7, 3), device=DEV, requires_grad=True)
    product = leaf * out
    row_table.lookup_rows_backward(g, ids, 7, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()


@gpu
@pytest.mark.parametrize("padding", [-1, -5, 7, 2 ** 63, 2 ** 64 + 3])
def test_padding_id_that_names_no_row(padding):
    ids, g = make_ids(500, 7, "strays"), rand((500, 3))
    want, wt = row_table.lookup_rows_backward(g, ids, 7)
    got, touched = row_table.lookup_rows_backward(g, ids, 7, padding_id=padding)
    assert torch.equal(got, want) and torch.equal(touched, wt)


@gpu
def test_two_threads_on_two_streams():
    """No state is shared between calls: each thread gets the bits of a solitary call."""
    cases = [(rand((40000, 12), seed=1), make_ids(40000, 80, "power"), 80),
             (rand((9000, 136), torch.bfloat16, seed=2), make_ids(9000, 5000, "power"), 5000)]
    want = [row_table.lookup_rows_backward(*c) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(40):
                got[k].append(row_table.lookup_rows_backward(*cases[k]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert len(got[k]) == 40
        assert all(torch.equal(a, want[k][0]) and torch.equal(b, want[k][1]) for a, b in got[k])


@gpu
@pytest.mark.parametrize("captured", [False, True])
def test_a_run_of_them_together(captured):
    """Per-keyframe colour rows of a map: looked up by every splat's keyframe, differentiated,
    clipped and stepped with the rows that were touched, against the same steps in float64.

    A step's relative error is below 1e-5 (82 u of the gradient's sums over |g| and their norm,
    the moments' 12 u); the first moments and rows of three steps stay within 1e-4 of their size."""
    n, rows, cols, lr, steps = 6000, 80, 12, 0.01, 3
    start = rand((rows, cols), seed=4)
    table = torch.nn.Parameter(start.clone())
    bias = torch.nn.Parameter(rand((rows, 3), seed=5))
    start_bias = bias.detach().clone()
    opt = surfel.SparseGaussianAdam([{"params": [table], "lr": lr}, {"params": [bias], "lr": lr}], lr=0.0, eps=1e-15)
    target = rand((n, cols), seed=6)
    ids = make_ids(n, rows, "strays")
    ids[(ids >= 60) & (ids < 70)] = 3                                  # ten keyframes own nothing
    touched = torch.zeros(rows, dtype=torch.bool, device=DEV)

    def step():
        # gradients by the formula: loss = sum (2 lookup(table) - target)^2 / 2 + sum lookup(bias)
        out = row_table.lookup_rows(table.detach(), ids, scale=2.0)
        g, t = row_table.lookup_rows_backward(out - target, ids, rows, scale=2.0)
        gb, _ = row_table.lookup_rows_backward(torch.ones_like(bias[:1]).expand(n, 3), ids, rows)
        touched.copy_(t)
        table.grad.copy_(g)
        bias.grad.copy_(gb)
        return opt.step(touched, rows, max_norm=5.0)

    if captured:
        table.grad, bias.grad = torch.zeros_like(table), torch.zeros_like(bias)
        for p in (table, bias):
            opt._moments(p)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = step()
    norms = []
    for _ in range(steps):
        if captured:
            graph.replay()
            norms.append(float(norm))
        else:
            opt.zero_grad()
            touched.zero_()
            out = row_table.lookup_rows(table, ids, scale=2.0, touched=touched)
            loss = (out - target).square().sum() / 2 + row_table.lookup_rows(bias, ids, touched=touched).sum()
            loss.backward()
            norms.append(float(opt.step(touched, rows, max_norm=5.0)))

    t, b = start.double(), start_bias.double()
    mom = [[torch.zeros_like(x), torch.zeros_like(x)] for x in (t, b)]
    seen = backward64(target, ids, rows)[2] > 0
    assert torch.equal(touched, seen) and not seen[60:70].any()
    found = ((ids >= 0) & (ids < rows))[:, None]
    for k in range(steps):
        g = backward64(torch.where(found, lookup64(t, ids, 2.0) - target.double(), 0.0), ids, rows)[0] * 2
        gb = backward64(torch.ones((n, 3), device=DEV), ids, rows)[0]
        norm64 = float((g.square().sum() + gb.square().sum()).sqrt())
        assert abs(norms[k] - norm64) <= 1e-5 * norm64
        coef = min(1.0, 5.0 / (norm64 + 1e-6))
        for x, gx, (m, v) in zip((t, b), (g, gb), mom):
            m.mul_(0.9).add_(0.1 * gx * coef)
            v.mul_(0.999).add_(0.001 * (gx * coef) ** 2)
            x -= torch.where(seen[:, None], lr * m / (v.sqrt() + 1e-15), torch.zeros_like(x))
    for p, x, s in ((table, t, start), (bias, b, start_bias)):
        assert float((p.detach().double() - x).norm()) <= 1e-4 * float((x - s.double()).norm())
        assert torch.equal(p.detach()[~seen], s[~seen])
    assert abs(float(gradients.global_norm([table.grad, bias.grad])) - norms[-1]) <= 2 * U * norms[-1]


@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=gpu)])
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_tangents_are_refused(device, leaf):
    """They would be lost: kernels that take addresses see the values alone."""
    fwd = torch.autograd.forward_ad
    ids = torch.zeros(3, dtype=torch.int64, device=device)
    with fwd.dual_level():
        dual = fwd.make_dual(torch.ones((4, 2), device=device, requires_grad=leaf), torch.ones((4, 2), device=device))
        for call in (lambda: row_table.lookup_rows(dual, ids), lambda: row_table.lookup_rows_backward(dual[:3], ids, 5)):
            with pytest.raises(_lib.VingsError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(_lib.VingsError, match="tangent"):
                call()


@gpu
def test_forward_mode_tangent_of_the_incoming_gradient_is_refused():
    """A tangent that first appears in the backward pass; without one an open level changes nothing."""
    fwd = torch.autograd.forward_ad
    ids = make_ids(60, 9, "uniform")
    table = rand((9, 4), seed=1).requires_grad_()
    weight = rand((60, 4), seed=2)
    with fwd.dual_level():
        (row_table.lookup_rows(table, ids) * weight).sum().backward()
        check_backward(weight, ids, 9, 1.0, table.grad, torch.bincount(ids, minlength=9) > 0)
        loss = (row_table.lookup_rows(table, ids) * fwd.make_dual(weight, torch.ones_like(weight))).sum()
        with pytest.raises(_lib.VingsError, match="tangent"):
            loss.backward()


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.VingsError):
        row_table.lookup_rows(torch.ones((3, 2)), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(_lib.VingsError):
        row_table.lookup_rows_backward(torch.ones((1, 2)), torch.zeros(1, dtype=torch.int64), 3)


# ---------------------------------------------------------------------------
# argument checks of the C entry points: they fail before the first HIP call
# ---------------------------------------------------------------------------
host_only = pytest.mark.skipif(torch.cuda.is_available(), reason="host-only argument checks")
FAKE = 0x10000


def _error():
    return _lib.lib().vings_last_error().decode()


@host_only
def test_lookup_arguments():
    def call(n=4, rows=5, cols=3, table=FAKE, ld=3, ty=0, ids=FAKE, idb=8, out=FAKE):
        return _lib.lib().vings_row_lookup(n, rows, cols, table, ld, ty, ids, idb, 1.0, out, None)
    assert call(n=0, table=None, ids=None, out=None) == 0
    for change, text in ((dict(n=-1), "sizes"), (dict(rows=-1), "sizes"), (dict(cols=0), "sizes"), (dict(rows=2 ** 31), "31 bits"),
                         (dict(n=2 ** 31), "31 bits"), (dict(cols=2 ** 20 + 1), "20"), (dict(ty=3), "element type"), (dict(ty=-1), "element type"),
                         (dict(idb=2), "int32 or int64"), (dict(table=None), "null pointer"), (dict(ids=None), "null pointer"),
                         (dict(out=None), "null pointer"), (dict(ld=2), "overlap"), (dict(table=FAKE + 2), "alignment"),
                         (dict(ids=FAKE + 4), "alignment")):
        assert call(**change) != 0 and text in _error(), change


@host_only
def test_backward_arguments():
    L = _lib.lib()
    size = L.vings_row_lookup_backward_workspace_bytes

    def call(n=4, rows=5000, cols=3, grad=FAKE, ld=3, ty=0, ids=FAKE, idb=8, out=FAKE * 2, ot=0, ws=FAKE, ws_bytes=1 << 20):
        return L.vings_row_lookup_backward(n, rows, cols, grad, ld, ty, ids, idb, -1, 1.0, out, ot, None, 0, ws, ws_bytes, None)
    assert call(rows=0, out=None) == 0
    for change, text in ((dict(n=-1), "sizes"), (dict(cols=0), "sizes"), (dict(ot=1), "gradient's type"), (dict(ty=1, ot=2), "gradient's type"),
                         (dict(out=None), "null pointer"), (dict(grad=None), "null pointer"), (dict(ids=None), "null pointer"),
                         (dict(ws=None), "null pointer"), (dict(ld=-1), "2^20"), (dict(ld=2 ** 20 + 1), "2^20"),
                         (dict(grad=FAKE * 2 - 4), "overlaps"), (dict(ids=FAKE * 2), "overlaps"), (dict(cols=2 ** 20 + 1), "20"), (dict(ws=FAKE + 8), "256-byte"),
                         (dict(ws_bytes=16), "too small"), (dict(out=FAKE * 2 + 2), "alignment"), (dict(grad=FAKE + 1), "alignment")):
        assert call(**change) != 0 and text in _error(), change
    assert size(0, 9, 4, 0) == 0 and size(10, 9, 4, 9) == 0 and size(10, 0, 4, 0) == 0
    assert size(10, 5000, 4, 0) >= 80 and size(100000, 5000, 4, 0) >= 4 * 4 * 100000   # both sides of the passes


@host_only
@pytest.mark.parametrize("n,rows,cols,ty", [(1000000, 257, 64, 0), (4000000, 257, 64, 0), (4190000, 260, 90, 1),
                                            (300000, 600, 30, 0), (1000000, 1000, 12, 0), (100000, 4095, 16, 2)])
def test_workspace_of_numbered_runs(n, rows, cols, ty):
    """A tile of 1024 ids leaves min(rows, 1024) partial rows at most; beside those stand two bytes a
    tile and row."""
    size = _lib.lib().vings_row_lookup_backward_workspace_bytes
    tiles = -(-n // 1024)
    assert 0 < size(n, rows, cols, ty) <= tiles * (4 * min(rows, 1024) * cols + 2 * rows) + 4096
