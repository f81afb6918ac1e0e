"""GPU (-m gpu): the embedding lookup with scaling and its gradient by sorted ids, against the formulas in 64 bits.

Tolerances: a row of the output or of the gradient is a sum of n products in fp32, each product rounded at most three times and every addition once:
(n + 4) 2^-24 of the sum of the magnitudes, and half a step of the tensors' type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32) of the result
(fp16 below 2^-14: half of its fixed step there, 2^-25)."""
import pytest
import torch

from nerf_loam_amd import layers, ops

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FLOOR = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _case(V, D, M, bag, dtype, seed, skew=1.0, id_type=torch.int32, invalid=True):
    g = _gen(seed)
    table = _rand(g, V, D, dtype=dtype)
    ids = (torch.rand(M, bag, generator=g, device="cuda", dtype=torch.float64) ** skew * V).long().clamp_(0, V - 1)
    if invalid:
        u = torch.rand(M, bag, generator=g, device="cuda")
        ids = torch.where(u < 0.05, torch.full_like(ids, -1), ids)
        ids = torch.where(u > 0.97, torch.full_like(ids, V), ids)
    return table, ids.to(id_type), torch.rand(M, bag, generator=g, device="cuda") - 0.25, _rand(g, M, D, dtype=dtype)


def _check(table, ids, w, g, scale, y, gt, gw, what):
    V, D = table.shape
    M, bag = ids.shape
    dtype = table.dtype
    ok = (ids >= 0) & (ids < V)
    rows = torch.where(ok, ids, 0).long()
    wd = ok.double() * (1.0 if w is None else w.double())
    t = table.double()[rows] * wd.unsqueeze(2)
    want, S = t.sum(1) * scale, t.abs().sum(1) * abs(scale)
    _close(y, want, (bag + 4) * 2.0 ** -24 * S + EPS[dtype] * want.abs() + FLOOR[dtype], "y " + what)
    if gt is not None:
        per = (g.double() * scale).unsqueeze(1) * wd.unsqueeze(2)
        want = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, rows.view(-1), per.view(-1, D))
        S = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, rows.view(-1), per.view(-1, D).abs())
        n = torch.bincount(rows.view(-1), minlength=V).unsqueeze(1)
        _close(gt, want, (n + 4) * 2.0 ** -24 * S + EPS[dtype] * want.abs() + FLOOR[dtype], "g_table " + what)
    if gw is not None:
        p = (g.double() * scale).unsqueeze(1) * table.double()[rows]
        want, S = p.sum(2) * ok, p.abs().sum(2)
        _close(gw, want, (D + 4) * 2.0 ** -24 * S, "g_weights " + what)


def _close(got, want, tol, what):
    d = (got.double() - want).abs()
    bad = ~(d <= tol + 1e-300)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / (tol + 1e-300)).max()):.3g} times the tolerance, first at {bad.nonzero()[0].tolist()}"


def _grads(table, ids, w, g, scale):
    t = table.detach().requires_grad_(True)
    wl = None if w is None else w.detach().requires_grad_(True)
    y = layers.embedding_lookup(t, ids if w is not None else ids.reshape(-1), scale=scale, weights=wl)
    out = torch.autograd.grad(y, [t] + ([wl] if wl is not None else []), g)
    return y.detach(), out[0], (out[1] if wl is not None else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 3, 4, 8, 16, 24, 245, 256, 1024, 2056])
def test_over_widths(dtype, D):
    for i, (V, M, bag, id_type) in enumerate([(50, 70, 1, torch.int32), (300, 40, 8, torch.int64), (1, 33, 2, torch.int32), (1000, 129, 1, torch.int64)]):
        table, ids, w, g = _case(V, D, M, bag, dtype, 10 * D + i, id_type=id_type)
        w = w if bag > 1 else None
        _check(table, ids, w, g, 0.75, *_grads(table, ids, w, g, 0.75), f"V {V} D {D} M {M} bag {bag}")


@pytest.mark.parametrize("M", [1, 2, 63, 64, 65, 127, 128, 129, 2047, 2048, 2049, 4096, 4097, 8191, 70001])
def test_over_numbers_of_lookups(M):
    """across the borders of the sorting tiles and of the summing chunks; few rows, so that sums cross many chunks, and many"""
    for V, skew in ((3, 1.0), (255, 3.0), (256, 1.0), (70000, 3.0)):
        table, ids, w, g = _case(V, 16, M, 1, torch.float32, M + V, skew=skew)
        _check(table, ids, None, g, 1.5, *_grads(table, ids, None, g, 1.5), f"V {V} M {M}")


def test_one_row_takes_everything():
    """all lookups hit one row, or none hits any"""
    table, ids, w, g = _case(500, 40, 30000, 1, torch.float32, 5, invalid=False)
    ids[:] = 123
    y, gt, _ = _grads(table, ids, None, g, 1.0)
    _check(table, ids, None, g, 1.0, y, gt, None, "one row")
    assert not bool(gt[:123].any()) and not bool(gt[124:].any())
    ids[:] = -1
    y, gt, _ = _grads(table, ids, None, g, 1.0)
    assert not bool(y.any()) and not bool(gt.any())
    ids[:] = 500
    ids[7] = 2 ** 31 - 1
    y, gt, _ = _grads(table, ids, None, g, 1.0)
    assert not bool(y.any()) and not bool(gt.any())
    wide = ids.long()
    wide[3], wide[4], wide[5] = 2 ** 40 + 3, -2 ** 40, 499                  # beyond 32 bits: no row either
    y, gt, _ = _grads(table, wide, None, g, 1.0)
    assert torch.equal(y[5], table[499]) and not bool(y[:5].any()) and torch.equal(gt[499], g[5]) and not bool(gt[:499].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_tables(dtype):
    for V, D, M, bag, skew in ((53847, 16, 60000, 8, 1.0), (20000, 1024, 9000, 1, 4.0), (2000003, 3, 50000, 1, 1.0), (17000000, 2, 3000, 1, 1.0)):
        table, ids, w, g = _case(V, D, M, bag, dtype, V, skew=skew)
        w = w if bag > 1 else None
        _check(table, ids, w, g, 1.0, *_grads(table, ids, w, g, 1.0), f"V {V} D {D}")


def test_same_bits_every_run_and_on_every_stream():
    table, ids, w, g = _case(900, 64, 20000, 2, torch.bfloat16, 77, skew=4.0)
    first = _grads(table, ids, w, g, 2.0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for i in range(4):
        with torch.cuda.stream(s if i % 2 else torch.cuda.current_stream()):
            again = _grads(table, ids, w, g, 2.0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_special_values_stay_in_their_rows():
    table, ids, w, g = _case(40, 8, 100, 2, torch.float32, 88)
    table[7, 2] = float("nan")
    table[9, 1] = float("inf")
    g[3, 5] = float("nan")
    y, gt, gw = _grads(table, ids, w, g, 1.0)
    hit = ((ids == 7) | (ids == 9)).any(1)
    assert bool(torch.isfinite(y[~hit]).all()) and bool(y[(ids == 7).any(1)][:, 2].isnan().all())
    rows = {int(i) for i in ids[3].tolist() if 0 <= i < 40}
    bad = gt.isnan().nonzero()
    assert {int(r) for r, _ in bad} == rows and {int(c) for _, c in bad} <= {5}


def test_no_lookups_and_single_ids():
    for dtype in DTYPES:
        t = torch.randn(5, 7, device="cuda").to(dtype).requires_grad_(True)
        y = layers.embedding_lookup(t, torch.empty(0, dtype=torch.int64, device="cuda"))
        assert y.shape == (0, 7)
        assert not bool(torch.autograd.grad(y, t, torch.empty(0, 7, dtype=dtype, device="cuda"))[0].any())
        one = layers.embedding_lookup(t, torch.tensor(3, device="cuda"), scale=2.0)
        assert one.shape == (7,) and torch.equal(one, (t[3].float() * 2).to(dtype))
        grid = layers.embedding_lookup(t, torch.tensor([[0, 1, 2], [4, 4, 9]], device="cuda"))
        assert grid.shape == (2, 3, 7) and torch.equal(grid[1, 0], t[4]) and not bool(grid[1, 2].any())


def test_strided_tables_and_ids_and_a_table_used_twice():
    table, ids, w, g = _case(60, 12, 50, 3, torch.float32, 99)
    a = _grads(table, ids, w, g, 1.0)
    b = _grads(table.t().contiguous().t(), ids.t().contiguous().t(), w.t().contiguous().t(), g, 1.0)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    t = table.requires_grad_(True)
    y = layers.embedding_lookup(t, ids, weights=w) + layers.embedding_lookup(t, ids, scale=3.0, weights=w)
    twice = torch.autograd.grad(y, t, g)[0]
    want = a[1] + _grads(table.detach(), ids, w, g, 3.0)[1]
    assert torch.equal(twice, want)
    t2 = table.detach().requires_grad_(True)                                  # a gradient that is a broadcast number
    layers.embedding_lookup(t2, ids[:, 0]).sum().backward()
    _check(table.detach(), ids[:, :1].contiguous(), None, torch.ones(50, 12, device="cuda"), 1.0, layers.embedding_lookup(t2.detach(), ids[:, 0]), t2.grad, None, "sum")


def test_graph_replays():
    table, ids, w, g = _case(700, 32, 5000, 2, torch.bfloat16, 111, skew=3.0)
    bufs = [dict(y=torch.empty(5000, 32, dtype=torch.bfloat16, device="cuda"), gt=torch.empty_like(table), gw=torch.empty_like(w)) for _ in range(2)]

    def step(b):
        ops.embedding_forward(table, ids, w, 1.25, out=b["y"])
        ops.embedding_backward(table, ids, g, w, 1.25, g_table=b["gt"], g_weights=b["gw"])
    step(bufs[0])
    torch.cuda.synchronize()
    gph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gph):
        step(bufs[1])
    for it in range(4):
        _, i2, w2, g2 = _case(700, 32, 5000, 2, torch.bfloat16, 120 + it, skew=3.0)
        ids.copy_(i2); w.copy_(w2); g.copy_(g2)
        step(bufs[0])
        gph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bufs[0][k], bufs[1][k]) for k in bufs[0]), it


def test_refusals():
    table, ids, w, g = _case(60, 12, 50, 3, torch.float32, 131)
    for bad in (lambda: layers.embedding_lookup(table, ids.float(), weights=w), lambda: layers.embedding_lookup(table.double(), ids, weights=w),
                lambda: layers.embedding_lookup(table, ids.cpu(), weights=w), lambda: layers.embedding_lookup(table, ids, weights=w.half()),
                lambda: ops.embedding_backward(table, ids, g[:49], w, g_table=torch.empty_like(table)),
                lambda: ops.embedding_backward(table, ids, g, w, g_table=torch.empty(59, 12, device="cuda")),
                lambda: ops.embedding_backward(table, ids, g, w, g_table=torch.empty_like(table), workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("run", [1, 15, 16, 17, 32, 64, 1000, 1024, 1025, 4096])
def test_runs_that_meet_the_borders_of_chunks_and_blocks(run):
    """equal ids in runs of one length: rows that begin and end exactly where chunks (16 entries, 64 for many lookups) and blocks of 64 chunks do, and rows that do not"""
    for L in (9000, 70000):
        ids = (torch.arange(L, device="cuda") // run).to(torch.int32).view(-1, 1)
        V = int(ids.max()) + 1
        g = _rand(_gen(run), L, 4, dtype=torch.float32)
        table = _rand(_gen(1), V, 4, dtype=torch.float32)
        _check(table, ids, None, g, 1.0, *_grads(table, ids, None, g, 1.0), f"run {run} L {L}")


def test_three_levels_of_joins():
    """300000 lookups of two rows: 4688 chunks, 74 blocks, 2 blocks of blocks"""
    g = _rand(_gen(3), 300000, 4, dtype=torch.float32)
    ids = (torch.arange(300000, device="cuda") >= 131072 + 5).to(torch.int64).view(-1, 1)
    table = _rand(_gen(4), 2, 4, dtype=torch.float32)
    _check(table, ids, None, g, 1.0, *_grads(table, ids, None, g, 1.0), "two rows")


def test_tables_beyond_32_bits():
    """a table of more than 2^31 elements: rows at the far end, forward and backward"""
    V, D, M = 700000, 3200, 600
    table = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    ids = (torch.arange(M, device="cuda") * 7 % 13 + V - 13).to(torch.int64).view(-1, 1)
    ids[5] = 671089
    g = _rand(_gen(9), M, D, dtype=torch.bfloat16)
    rows = torch.unique(ids)
    table[rows] = _rand(_gen(8), len(rows), D, dtype=torch.bfloat16)
    y = ops.embedding_forward(table, ids)
    assert torch.equal(y, table[ids.view(-1)])
    gt = torch.full_like(table, 3.0)
    ops.embedding_backward(table, ids, g, g_table=gt)
    want = torch.zeros(V - 671089, D, dtype=torch.float64, device="cuda").index_add_(0, ids.view(-1) - 671089, g.double())
    assert bool(((gt[671089:].double() - want).abs() <= 64 * 2.0 ** -24 * 50 * 5 + 2.0 ** -8 * want.abs()).all())       # at most 50 lookups a row, |g| < 5
    assert not bool(gt[:671089].any())


def test_more_groups_of_threads_than_a_grid_axis_has_threads():
    """2^30 - 64 lookups, the most there may be: forward with four threads a row (2^32 in all) and backward, whose sums are exact whole numbers"""
    V, M = 1 << 24, (1 << 30) - 64
    if torch.cuda.mem_get_info()[0] < 80e9:
        pytest.skip("needs 80 GB of free memory")
    ids = (torch.arange(M, dtype=torch.int32, device="cuda") & (V - 1)).view(M, 1)
    table = (torch.arange(3 * 4096, device="cuda") % 251).to(torch.bfloat16).view(4096, 3)
    small = ids & 4095
    y = ops.embedding_forward(table, small)
    for i in (0, (1 << 22) * 64 - 1, (1 << 22) * 64, (1 << 29) + 5, M - 1):
        assert torch.equal(y[i], table[i & 4095]), i
    assert torch.equal(y[-4096:], table[small[-4096:, 0].long()])
    del y, small
    g = torch.ones(M, 1, dtype=torch.float32, device="cuda")
    gt = torch.empty(V, 1, dtype=torch.float32, device="cuda")
    ops.embedding_backward(torch.empty(V, 1, dtype=torch.float32, device="cuda"), ids, g, g_table=gt)
    want = torch.full((V, 1), 64.0, device="cuda")
    want[-64:] = 63.0
    assert torch.equal(gt, want)


def test_products_of_a_row_with_more_rows_than_a_grid_axis_has_threads():
    M = 1 << 30
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of free memory")
    x = torch.ones(M, 1, dtype=torch.bfloat16, device="cuda")
    at = [0, (1 << 22) * 64 - 1, (1 << 22) * 64, (1 << 29) + 7, M - 1]
    x[at] = 3.0
    w = torch.full((1, 1), 0.5, dtype=torch.bfloat16, device="cuda")
    y = ops.linear_forward(x, w)
    assert bool((y[at] == 1.5).all()) and int((y == 0.5).sum()) == M - len(at)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [4, 8, 12, 16, 20, 24, 72, 1000, 2056])
def test_bags_of_eight(dtype, D):
    """32-bit ids and weights, aligned or not, few and odd numbers of rows, threads of a group without columns; weights of ids without a row may be anything"""
    for M in (1, 3, 257):
        table, ids, w, g = _case(97, D, M, 8, dtype, 1000 * M + D)
        ids[0, 3], ids[0, 4], ids[-1, 7] = -1, 97, 2 ** 31 - 1
        for shift in (0, 1):
            flat = torch.empty(8 * M + shift, dtype=torch.int32, device="cuda")[shift:].view(M, 8).copy_(ids)
            wflat = torch.empty(8 * M + shift, device="cuda")[shift:].view(M, 8).copy_(w)
            _check(table, flat, wflat, g, 0.5, *_grads(table, flat, wflat, g, 0.5), f"D {D} M {M} shift {shift}")
        y = ops.embedding_forward(table, ids, w, 0.5)
        w[(ids < 0) | (ids >= 97)] = float("nan")
        assert torch.equal(ops.embedding_forward(table, ids, w, 0.5), y)


def test_bags_of_eight_over_tables_around_two_gigabytes():
    for V in (67108863, 67108864, 70000001):                                 # 16 bf16: 2^31 - 32 bytes (as far as 32-bit offsets go), 2^31, more
        table = torch.zeros(V, 16, dtype=torch.bfloat16, device="cuda")
        rows = [0, 1, V // 2, V - 2, V - 1]
        table[rows] = (torch.arange(5 * 16, device="cuda").view(5, 16) + 1.0).to(torch.bfloat16)
        ids = torch.tensor([[0, 1, V // 2, V - 2, V - 1, -1, V, 2 ** 31 - 1]], dtype=torch.int32, device="cuda").expand(5, 8).contiguous()
        for k in range(5):
            w = torch.zeros(5, 8, device="cuda")
            w[:, k] = 1.0
            assert torch.equal(ops.embedding_forward(table, ids, w), table[rows[k]].expand(5, 16)), (V, k)
        w = torch.zeros(5, 8, device="cuda")
        w[:, 5:] = 1.0
        assert not bool(ops.embedding_forward(table, ids, w).any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_move_with_their_lookups(dtype):
    """sorts of more than 65536 weighted lookups, one to four passes, whole and partial workgroups; and bags without weights"""
    for V, D, M, bag in ((200, 8, 40000, 2), (40000, 4, 8193, 9), (100000, 3, 22000, 3), (20000003, 2, 33000, 3), (3000, 16, 65537, 8)):
        table, ids, w, g = _case(V, D, M, bag, dtype, V + M)
        _check(table, ids, w, g, 0.75, *_grads(table, ids, w, g, 0.75), f"V {V} D {D} M {M} bag {bag}")
        gt, gt1 = torch.empty_like(table), torch.empty_like(table)
        ops.embedding_backward(table, ids, g, None, 0.75, gt)
        ops.embedding_backward(table, ids, g, torch.ones_like(w), 0.75, gt1)
        assert torch.equal(gt, gt1), (V, M)
