"""GPU (-m gpu): linear layers with their epilogue, their gradients, and the 8-bit checkpoints, against the formulas in 64 bits.

Tolerances, element by element.  u = 2^-24 (fp32, to nearest), eps = half a step of the tensors' type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32).
A product of K terms: 16-bit terms multiply exactly in fp32; fp32 terms are split exactly and lose at most 3 * 2^-26 of |x||w|.  Every fp32 addition
may cost 2u of its running sum (a matrix unit may cut instead of round), at most K + 8 of them in a row (six products per term in fp32):
  e(K) S = (c K + 8) 2u S,  S = sum of the |terms| + |bias|,  c = 1 (16 bits), 6 (fp32)
Activations: |act'| <= 1.13 for all four, and their evaluation costs less than 16 u of (1 + |z|).  Output: eps |y| more.  8-bit codes: half of the step between
neighbouring codes: 2^-4 of the value, or 2^-10 of the block's power of two below the smallest normal code.
A rounding to fp16 below 2^-14 has steps of 2^-24 whatever the value is: half of that, 2^-25, comes on top of eps |v| wherever a value is rounded to the type
(0.0000098 = 2^-16.6 rounds with a relative error of up to 2^-8.4, not 2^-11); the same floor is 2^-126 for the types with fp32's exponents."""
import numpy as np
import pytest
import torch

from nerf_loam_amd import layers, ops

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SIZES = [(1, 1, 1), (1, 300, 64), (3, 5, 7), (16, 16, 32), (17, 33, 65), (64, 64, 64), (65, 129, 257), (300, 200, 100), (130, 256, 16), (257, 512, 256), (1000, 8, 1024), (5, 1, 256),
         (2, 1000, 3), (16, 4096, 512), (700, 31, 40), (333, 777, 129), (512, 512, 512)]


FLOOR = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def _half(v, dtype):
    """the most that rounding v to the type may move it"""
    return EPS[dtype] * v.abs() + FLOOR[dtype]


def _rand(g, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _act64(z, act):
    return {"none": lambda t: t, "relu": torch.relu, "gelu": lambda t: 0.5 * t * (1 + torch.erf(t * 0.5 ** 0.5)), "silu": lambda t: t * torch.sigmoid(t)}[act](z)


def _slope64(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) / (2 * np.pi) ** 0.5
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _e(K, dtype):
    return ((6 if dtype == torch.float32 else 1) * K + 8) * 2.0 ** -23


def _close(got, want, tol, what):
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / tol).max()):.3g} times the tolerance, first at {bad.nonzero()[0].tolist()}"


def mx8_values(x):
    """the 8-bit format by search over all codes, in 64 bits on the host: -> (values, exponents)"""
    mags = np.array([(c % 8) * 2.0 ** -9 if c < 8 else (1 + (c % 8) / 8) * 2.0 ** (c // 8 - 7) for c in range(127)])
    x = np.asarray(x, np.float64)
    M, K = x.shape
    KB = -(-K // 32)
    b = np.zeros((M, KB * 32)); b[:, :K] = x
    b = b.reshape(M, KB, 32)
    fin = np.isfinite(b)
    top = np.where(fin, np.abs(b), 0).max(2)
    e = np.full(top.shape, -126)
    for cand in range(-126, 121):
        e = np.where((top > 448 * 2.0 ** (cand - 1)) & (cand > -126), cand, e)
    e = np.maximum(e, -126)
    a = np.where(fin, np.abs(b), 0) * 2.0 ** -e[..., None].astype(np.float64)
    hi = np.clip(np.searchsorted(mags, a), 0, 126); lo = np.maximum(hi - 1, 0)
    up, dn = mags[hi] - a, a - mags[lo]
    code = np.where(up < dn, hi, np.where(up > dn, lo, np.where(hi % 2 == 0, hi, lo)))
    v = np.copysign(mags[code], np.where(fin, b, 1.0)) * 2.0 ** e[..., None].astype(np.float64)
    v = np.where(fin, v, np.nan)
    return v.reshape(M, KB * 32)[:, :K], e


def _forward_case(M, N, K, dtype, act, seed, bias=True, residual=True):
    g = _gen(seed)
    x, w = _rand(g, M, K, dtype=dtype), _rand(g, N, K, dtype=dtype, std=K ** -0.5)
    b = _rand(g, N, dtype=dtype) if bias else None
    r = _rand(g, M, N, dtype=dtype) if residual else None
    return x, w, b, r


def _z64(x, w, b):
    z = x.double() @ w.double().t()
    S = x.double().abs() @ w.double().abs().t()
    if b is not None:
        z, S = z + b.double(), S + b.double().abs()
    return z, S


def _check_forward(x, w, b, r, act, y, what):
    z, S = _z64(x, w, b)
    ez = _e(x.shape[1], x.dtype) * S
    want = _act64(z, act)
    mag = 1 + z.abs()
    if r is not None:
        want, mag = want + r.double(), mag + r.double().abs()
    _close(y, want, 1.13 * ez + 16 * 2.0 ** -24 * mag + _half(want.abs() + 1.13 * ez, x.dtype), what)
    return z, ez


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_forward_over_sizes(dtype, act):
    for i, (M, N, K) in enumerate(SIZES):
        x, w, b, r = _forward_case(M, N, K, dtype, act, 100 + i, bias=i % 3 != 0, residual=i % 2 == 0)
        y = layers.linear_act(x, w, b, act=act, residual=r)
        assert y.shape == (M, N) and y.dtype == dtype
        _check_forward(x, w, b, r, act, y, f"{M}x{N}x{K}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_the_forward_pass_keeps(dtype):
    for i, (M, N, K) in enumerate(SIZES):
        x, w, b, _ = _forward_case(M, N, K, dtype, "gelu", 200 + i)
        nb = (N + 31) // 32
        z = torch.empty(M, N, dtype=dtype, device="cuda")
        bits = torch.empty(M, nb, dtype=torch.int32, device="cuda")
        z8 = torch.empty(M, 32 * nb, dtype=torch.uint8, device="cuda")
        z8e = torch.empty(M, nb, dtype=torch.uint8, device="cuda")
        ops.linear_forward(x, w, b, "gelu", z=z)
        z64, S = _z64(x, w, b)
        ez = _e(K, dtype) * S + 2.0 ** -24 * S
        _close(z, z64, ez + _half(z64.abs() + ez, dtype), f"z {M}x{N}x{K}")
        ops.linear_forward(x, w, b, "relu", bits=bits)
        on = ((bits.view(M, nb, 1) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool().view(M, -1)
        assert not bool(on[:, N:].any())
        sure = z64.abs() > ez
        assert bool((on[:, :N] == (z64 > 0))[sure].all()), f"bits {M}x{N}x{K}"
        ops.linear_forward(x, w, b, "silu", z8=z8, z8e=z8e)
        assert not bool(z8[:, N:].any())
        e = z8e.double() - 127
        step = torch.exp2(e).repeat_interleave(32, 1)[:, :N] * 2.0 ** -10
        back = ops.mx8_decode(z8, z8e, N, torch.float32).double()
        _close(back, z64, ez + torch.maximum((z64.abs() + ez) * 2.0 ** -4, step), f"z8 {M}x{N}x{K}")
        top = torch.nn.functional.pad(z64.abs(), (0, 32 * nb - N)).view(M, nb, 32).amax(2)
        slack = torch.nn.functional.pad(ez, (0, 32 * nb - N)).view(M, nb, 32).amax(2)
        assert bool((top - slack <= 448 * torch.exp2(e)).all()) and bool(((top + slack > 224 * torch.exp2(e)) | (e == -126)).all())


def _backward_check(gy, x, w, act, saved, dtype, what, x_values=None):
    """gradients of ops.linear_backward against the formula on the tensors it is given"""
    M, N, K = gy.shape[0], gy.shape[1], w.shape[1]
    gx, gw, gb = (torch.full(s, 7.0, dtype=dtype, device="cuda") for s in ((M, K), (N, K), (N,)))
    kw = {k: v for k, v in saved.items() if k in ("z", "bits", "z8", "z8e", "x8", "x8e")}
    ops.linear_backward(gy, x, w, act, gx=gx, gw=gw, gb=gb, **kw)
    g, wd = gy.double(), w.double()
    xd = x.double() if x_values is None else x_values
    slope = saved["on"].double() if act == "relu" else torch.ones_like(g) if act == "none" else _slope64(saved["z_values"], act)
    dz = g * slope
    # the slope to 16 u (1 + |z|) (gelu' holds a product z exp(..)), dz rounded once to the type
    e_dz = (0 if act in ("none", "relu") else 1) * g.abs() * 16 * 2.0 ** -24 * (1 + (saved["z_values"].abs() if "z_values" in saved else 0)) + 2.0 ** -24 * dz.abs()
    e_dz16 = e_dz + (0 if act == "none" else 1) * _half(dz.abs() + e_dz, dtype)
    ad, aw, ax = dz.abs() + e_dz16, wd.abs(), xd.abs()
    for got, want, S, e0, n, name in ((gx, dz @ wd, ad @ aw, e_dz16 @ aw, N, "gx"), (gw, dz.t() @ xd, ad.t() @ ax, e_dz16.t() @ ax, M, "gw"),
                                      (gb, dz.sum(0), (dz.abs() + e_dz).sum(0), e_dz.sum(0), M, "gb")):
        e = e0 + _e(n, dtype) * S
        _close(got, want, e + _half(want.abs() + e, dtype), f"{name} {what}")
    return gx, gw, gb


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("checkpoint", [None, "mx8"])
def test_backward_over_sizes(dtype, act, checkpoint):
    for i, (M, N, K) in enumerate(SIZES):
        x, w, b, _ = _forward_case(M, N, K, dtype, act, 300 + i)
        gy = _rand(_gen(400 + i), M, N, dtype=dtype)
        nb = (N + 31) // 32
        saved, x_values = {}, None
        if act == "relu":
            saved["bits"] = torch.randint(-2 ** 31, 2 ** 31 - 1, (M, nb), dtype=torch.int32, device="cuda", generator=_gen(i))
            saved["on"] = ((saved["bits"].view(M, nb, 1) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool().view(M, -1)[:, :N]
        elif act != "none":
            z = _rand(_gen(500 + i), M, N, dtype=dtype, std=2.0)
            if checkpoint:
                saved["z8"], saved["z8e"] = ops.mx8_encode(z)
                saved["z_values"] = torch.from_numpy(mx8_values(z.double().cpu().numpy())[0]).cuda()
            else:
                saved["z"], saved["z_values"] = z, z.double()
        if checkpoint:
            saved["x8"], saved["x8e"] = ops.mx8_encode(x)
            x_values = torch.from_numpy(mx8_values(x.double().cpu().numpy())[0]).cuda()
        _backward_check(gy, None if checkpoint else x, w, act, saved, dtype, f"{M}x{N}x{K}", x_values)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(70000, 24, 16), (20000, 256, 256), (4096, 1024, 520), (1, 2048, 4096), (9, 4100, 1030), (2100, 3000, 2056)])
def test_long_and_wide_layers(dtype, M, N, K):
    """contractions that are cut, many tiles, few rows"""
    x, w, b, r = _forward_case(M, N, K, dtype, "silu", 7)
    y = layers.linear_act(x, w, b, act="silu", residual=r)
    _check_forward(x, w, b, r, "silu", y, "y")
    gy = _rand(_gen(8), M, N, dtype=dtype)
    z = _rand(_gen(9), M, N, dtype=dtype)
    _backward_check(gy, x, w, "silu", dict(z=z, z_values=z.double()), dtype, "long")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "silu"])
def test_few_rows_of_either_operand(dtype, act):
    """at most eight rows of x, or a weight with at most eight: the kernel without tiles, odd sizes and strides among them"""
    for i, (M, N, K) in enumerate([(m, n, k) for m, n in ((1, 1000), (2, 33), (3, 500), (4, 64), (5, 129), (8, 300), (1000, 1), (999, 2), (77, 3), (513, 8), (9, 7), (8, 8)) for k in (1, 16, 40, 256, 513, 2048)]):
        x, w, b, r = _forward_case(M, N, K, dtype, act, 900 + i, bias=i % 2 == 0, residual=i % 3 == 0)
        _check_forward(x, w, b, r, act, layers.linear_act(x, w, b, act=act, residual=r), f"{M}x{N}x{K}")
        wide = torch.full((M, K + 3), float("nan"), dtype=dtype, device="cuda")
        wide[:, 1:K + 1] = x
        out = torch.full((M, N + 2), 5.0, dtype=dtype, device="cuda")
        ops.linear_forward(wide[:, 1:K + 1], w, b, act, r, out=out[:, 1:N + 1])
        assert bool((out[:, 0] == 5).all()) and bool((out[:, -1] == 5).all())
        _check_forward(x, w, b, r, act, out[:, 1:N + 1], f"strided {M}x{N}x{K}")


@pytest.mark.parametrize("M,N,K", [(300, 256, 512), (4096, 512, 1024), (1, 512, 512)])
def test_fp32_is_fp32(M, N, K):
    """the split products against 64 bits in the 2-norm: independent roundings of 2^-25 on average of a partial sum, not 2^-9"""
    x, w, b, _ = _forward_case(M, N, K, torch.float32, "none", 11)
    y = layers.linear_act(x, w)
    want = x.double() @ w.double().t()
    assert float((y.double() - want).norm() / want.norm()) < 1e-6
    big = x * 1e30                                                            # no 16-bit range in the way
    y2 = layers.linear_act(big, w)
    assert float((y2.double() - want * 1e30).norm() / (want * 1e30).norm()) < 1e-6


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment_do_not_change_a_bit(dtype):
    """the same numbers behind other strides and addresses: rows of a wider tensor, columns from 1, a transposed weight, leading dimensions"""
    M, N, K = 150, 96, 64
    x, w, b, r = _forward_case(M, N, K, dtype, "gelu", 21)
    want = layers.linear_act(x, w, b, act="gelu", residual=r)

    def wide(t, off, extra):
        big = torch.full((t.shape[0], t.shape[1] + extra), float("nan"), dtype=dtype, device="cuda")
        big[:, off:off + t.shape[1]] = t
        return big[:, off:off + t.shape[1]]
    for off, extra in ((0, 8), (1, 1), (3, 5), (8, 16)):
        got = layers.linear_act(wide(x, off, extra), wide(w, off, extra), b, act="gelu", residual=wide(r, off, extra))
        z, ez = _check_forward(x, w, b, r, "gelu", got, f"offset {off} of {extra}")
    assert torch.equal(layers.linear_act(x, w.t().contiguous().t(), b, act="gelu", residual=r), want)
    assert torch.equal(layers.linear_act(x.view(5, 30, K), w, b, act="gelu", residual=r.view(5, 30, N)), want.view(5, 30, N))
    assert torch.equal(layers.linear_act(x[:1].expand(150, K), w, b, act="gelu", residual=r)[0], layers.linear_act(x[:1].repeat(150, 1), w, b, act="gelu", residual=r)[0])
    out = torch.full((M, N + 4), 5.0, dtype=dtype, device="cuda")
    ops.linear_forward(x, w, b, "gelu", r, out=out[:, 1:1 + N])
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 1 + N:] == 5).all())           # nothing beside the rows is written
    _check_forward(x, w, b, r, "gelu", out[:, 1:1 + N], "strided output")
    vec = layers.linear_act(x[0], w, b, act="gelu", residual=r[0])
    assert vec.shape == (N,)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows(dtype):
    x = torch.empty(0, 24, dtype=dtype, device="cuda", requires_grad=True)
    w = torch.randn(8, 24, device="cuda").to(dtype).requires_grad_(True)
    b = torch.randn(8, device="cuda").to(dtype).requires_grad_(True)
    for ck in (None, "mx8"):
        y = layers.linear_act(x, w, b, act="silu", checkpoint=ck)
        assert y.shape == (0, 8)
        gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty(0, 8, dtype=dtype, device="cuda"))
        assert gx.shape == (0, 24) and not bool(gw.any()) and not bool(gb.any())
    assert layers.checkpoint_decode(layers.checkpoint_encode(x.detach())).shape == (0, 24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(5, 40, 48), (300, 300, 300)])
def test_not_a_number_stays_in_its_row(dtype, M, N, K):
    """a NaN or an infinity of x reaches its own row of y and nothing else"""
    x, w, b, _ = _forward_case(M, N, K, dtype, "none", 31)
    clean = layers.linear_act(x, w, b, act="relu")
    x2 = x.clone()
    x2[2, 3] = float("nan")
    x2[4, 1] = float("inf")
    y = layers.linear_act(x2, w, b, act="relu")
    rows = [i for i in range(M) if i not in (2, 4)]
    assert torch.equal(y[rows], clean[rows]) and bool(y[2].isnan().all())
    z4 = x2[4].double() @ w.double().t() + b.double()
    assert bool((y[4].double() == torch.relu(z4)).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("checkpoint", [None, "mx8"])
def test_autograd_runs_the_same_kernels(dtype, act, checkpoint):
    M, N, K = 200, 96, 72
    x, w, b, r = (t.requires_grad_(True) for t in _forward_case(M, N, K, dtype, act, 41))
    gy = _rand(_gen(42), M, N, dtype=dtype)
    y = layers.linear_act(x, w, b, act=act, residual=r, checkpoint=checkpoint)
    got = torch.autograd.grad(y, [x, w, b, r], gy)
    nb = (N + 31) // 32
    saved = {}
    if act == "relu":
        saved["bits"] = torch.empty(M, nb, dtype=torch.int32, device="cuda")
    elif act != "none" and checkpoint:
        saved["z8"], saved["z8e"] = torch.empty(M, 32 * nb, dtype=torch.uint8, device="cuda"), torch.empty(M, nb, dtype=torch.uint8, device="cuda")
    elif act != "none":
        saved["z"] = torch.empty(M, N, dtype=dtype, device="cuda")
    with torch.no_grad():
        y2 = ops.linear_forward(x, w, b, act, r, **saved)
        gx, gw, gb = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
        x8 = dict(zip(("x8", "x8e"), ops.mx8_encode(x))) if checkpoint else {}
        ops.linear_backward(gy, None if checkpoint else x, w, act, gx=gx, gw=gw, gb=gb, **saved, **x8)
    assert torch.equal(y, y2)
    for a, c in zip(got, (gx, gw, gb, gy)):
        assert torch.equal(a, c)
    # any subset of the gradients, a broadcast residual, one tensor used twice
    y = layers.linear_act(x.detach(), w.detach(), b, act=act, checkpoint=checkpoint)
    assert torch.equal(torch.autograd.grad(y, b, gy)[0], gb)
    r1 = torch.randn(N, device="cuda").to(dtype).requires_grad_(True)
    y = layers.linear_act(x.detach(), w.detach(), b.detach(), act=act, residual=r1.expand(M, N), checkpoint=checkpoint)
    assert torch.equal(torch.autograd.grad(y, r1, gy)[0], gy.sum(0))
    with pytest.raises(RuntimeError):                                         # gradients of gradients are not provided
        y = layers.linear_act(x, w, act=act)
        gx1, = torch.autograd.grad(y.float().sum(), x, create_graph=True)
        gx1.float().sum().backward()


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gradient_against_differences(act):
    """central differences of the float32 forward pass along a random direction, h = 2^-6: the third derivative along the direction leaves h^2 / 6 of O(1) terms,
    4e-5; the forward pass is right to about 1e-6 per element and 1 / h = 64 of that remain, averaged over the elements: 1e-3 of the derivative's size is ample"""
    M, N, K = 40, 48, 32
    x, w, b, r = (t.requires_grad_(True) for t in _forward_case(M, N, K, torch.float32, act, 51))
    gy = _rand(_gen(52), M, N, dtype=torch.float32)
    grads = torch.autograd.grad(layers.linear_act(x, w, b, act=act, residual=r), [x, w, b, r], gy)
    h = 2.0 ** -6
    for i, (t, gr) in enumerate(zip((x, w, b, r), grads)):
        v = _rand(_gen(60 + i), *t.shape, dtype=torch.float32)
        v = v / v.norm() * t.numel() ** 0.5 * (K ** -0.5 if i == 1 else 1.0)
        with torch.no_grad():
            f = [(layers.linear_act(*[s + sgn * h * v if s is t else s for s in (x, w, b)], act=act, residual=r + sgn * h * v if t is r else r).double() * gy.double()).sum()
                 for sgn in (1, -1)]
        num, ana = float(f[0] - f[1]) / (2 * h), float((gr.double() * v.double()).sum())
        scale = float(gr.double().norm() * v.double().norm()) / gr.numel() ** 0.5
        assert abs(num - ana) <= 1e-3 * max(scale * gr.numel() ** 0.5, abs(ana)), (i, num, ana)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 31), (5, 32), (7, 33), (64, 100), (129, 256), (33, 1000), (2, 8192)])
def test_checkpoint_values(dtype, M, K):
    """every value is the nearest of the format's: bit for bit"""
    g = _gen(70 + K)
    x = (torch.randn(M, K, generator=g, device="cuda") * torch.exp(4 * torch.randn(M, 1, generator=g, device="cuda"))).to(dtype)
    x[0, 0] = 0
    c = layers.checkpoint_encode(x)
    want, e = mx8_values(x.double().cpu().numpy())
    got = layers.checkpoint_decode(c)
    assert got.dtype == dtype and got.shape == x.shape
    assert np.array_equal(c.exps.cpu().numpy().astype(int) - 127, e)
    want = torch.from_numpy(want).to(dtype).double().numpy().clip(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    same = bool(np.array_equal(got.double().cpu().numpy(), want, equal_nan=True))      # (fp16 inputs may hold infinities: they come back as NaN)
    assert same
    wide = torch.full((M, K + 3), 1e30 if dtype != torch.float16 else 6e4, dtype=dtype, device="cuda")
    wide[:, 1:K + 1] = x
    c2 = layers.checkpoint_encode(wide[:, 1:K + 1])
    assert torch.equal(c2.codes, c.codes) and torch.equal(c2.exps, c.exps)
    assert not bool(c.codes[:, K:].any())


def test_checkpoint_extremes():
    """zeros, the ends of the range, ties, infinities and NaN"""
    x = torch.zeros(8, 32, device="cuda")
    x[1] = torch.finfo(torch.float32).max
    x[2] = torch.finfo(torch.float32).tiny
    x[3, :3] = torch.tensor([448.0, 2.0 ** -9 * 0.5, 2.0 ** -9 * 1.5])         # ties at the small end: to even
    x[4, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0])
    x[5, :3] = torch.tensor([1.0625, 1.1875, 448.0])                            # ties between normal codes
    x[6] = 1e-42
    x[7, :2] = torch.tensor([449.0, 1.0])                                       # one step above 448: the next power of two
    c = layers.checkpoint_encode(x)
    got = layers.checkpoint_decode(c).double().cpu().numpy()
    want, e = mx8_values(x.double().cpu().numpy())
    assert np.array_equal(c.exps.cpu().numpy().astype(int) - 127, e)
    want = want.clip(-torch.finfo(torch.float32).max, torch.finfo(torch.float32).max)
    assert bool(np.array_equal(got, want, equal_nan=True))
    assert got[3, 1] == 0 and got[3, 2] == 2.0 ** -8 and got[5, 0] == 1.0 and got[5, 1] == 1.25
    top = torch.tensor([[65504.0, 63488.0, 61440.0]], device="cuda").half()
    assert layers.checkpoint_decode(layers.checkpoint_encode(top)).tolist() == [[65504.0, 65504.0, 61440.0]]


def test_graphs_replay_forward_and_backward():
    """the functions of ops captured into two graphs of one pool, replayed with eager work between: every replay like the eager result"""
    M, N, K = 260, 130, 520
    for dtype in DTYPES:
        x, w, b, r = _forward_case(M, N, K, dtype, "silu", 81)
        gy = _rand(_gen(82), M, N, dtype=dtype)

        def step(bufs):
            ops.linear_forward(x, w, b, "silu", r, out=bufs["y"], z=bufs["z"])
            ops.linear_backward(gy, x, w, "silu", z=bufs["z"], gx=bufs["gx"], gw=bufs["gw"], gb=bufs["gb"])
        shapes = dict(y=(M, N), z=(M, N), gx=(M, K), gw=(N, K), gb=(N,))
        bufs = [{k: torch.empty(s, dtype=dtype, device="cuda") for k, s in shapes.items()} for _ in range(3)]
        step(bufs[0])
        torch.cuda.synchronize()
        graphs, pool = [], None
        for i in (1, 2):
            gph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gph, pool=pool):
                step(bufs[i])
            pool = gph.pool()
            graphs.append(gph)
        for it in range(4):
            fresh = _rand(_gen(90 + it), M, K, dtype=dtype)
            x.copy_(fresh)
            step(bufs[0])
            for gph in graphs:
                gph.replay()
            torch.cuda.synchronize()
            for i in (1, 2):
                for k in shapes:
                    assert torch.equal(bufs[i][k], bufs[0][k]), (dtype, it, i, k)


def test_autograd_backward_inside_a_capture_is_refused():
    x, w, b, _ = _forward_case(32, 32, 32, torch.bfloat16, "none", 91)
    w.requires_grad_(True)
    gy = torch.ones(32, 32, dtype=torch.bfloat16, device="cuda")
    torch.autograd.grad(layers.linear_act(x, w, b), w, gy)
    torch.cuda.synchronize()
    gph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(gph):
            torch.autograd.grad(layers.linear_act(x, w, b), w, gy)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(layers.linear_act(x, w.detach(), b)).all())


def test_two_streams_at_once():
    """two calls on two streams, each with workspaces of its own: the results of one stream"""
    cases = [_forward_case(300, 140, 900, torch.bfloat16, "gelu", 95 + i) for i in range(2)]
    gy = _rand(_gen(99), 300, 140, dtype=torch.bfloat16)

    def grads(c):
        x, w, b, _ = (t.detach().requires_grad_(True) for t in c)
        y = layers.linear_act(x, w, b, act="gelu", checkpoint="mx8")
        return (y.detach(), *torch.autograd.grad(y, [x, w, b], gy))
    want = [grads(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = grads(cases[i])
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_mixed_types_and_shapes_are_refused():
    x, w, b, r = _forward_case(8, 16, 24, torch.bfloat16, "none", 97)
    for bad in (lambda: layers.linear_act(x, w.float()), lambda: layers.linear_act(x, w, b.float()), lambda: layers.linear_act(x, w, b, residual=r.float()),
                lambda: layers.linear_act(x, w.cpu()), lambda: layers.linear_act(x.double(), w.double()), lambda: layers.linear_act(x.int(), w),
                lambda: ops.linear_forward(x, w, b, out=torch.empty(7, 16, dtype=x.dtype, device="cuda")),
                lambda: ops.linear_backward(r, x, w, "gelu", gx=torch.empty_like(x)),
                lambda: ops.linear_backward(r, x[:7], w, gw=torch.empty_like(w)),
                lambda: ops.linear_backward(r, x, w, gw=torch.empty(15, 24, dtype=x.dtype, device="cuda")),
                lambda: ops.linear_forward(x, w, b, "relu", bits=torch.empty(8, 2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()
    for bad, word in ((lambda: layers.linear_act(x, w[:, :7]), "weight"), (lambda: layers.linear_act(x, w, b[:4]), "bias"), (lambda: layers.linear_act(x, w, residual=r[:, :1]), "residual"),
                      (lambda: layers.linear_act(x[:, :0], w[:, :0]), "elements"), (lambda: layers.checkpoint_encode(x[:, :0]), "checkpoint_encode"),
                      (lambda: layers.embedding_lookup(x[0], torch.zeros(2, dtype=torch.int64, device="cuda")), "table"),
                      (lambda: layers.embedding_lookup(x, torch.zeros(2, 3, dtype=torch.int64, device="cuda"), weights=torch.zeros(2, 2, device="cuda")), "weights")):
        with pytest.raises(ValueError, match=word):
            bad()


def test_offsets_beyond_32_bits():
    """operands and results of more than 2^31 elements: rows at the far end come out as they do in a small call"""
    M, K, N = 270000, 8192, 64
    g = _gen(201)
    w = _rand(g, N, K, dtype=torch.bfloat16, std=K ** -0.5)
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    far = torch.tensor([0, 1, 262143, 262144, 262145, M - 65, M - 2, M - 1], device="cuda")
    x[far] = _rand(g, len(far), K, dtype=torch.bfloat16)
    y = layers.linear_act(x, w, act="none")
    _check_forward(x[far], w, None, None, "none", y[far], "far rows")
    assert int((y != 0).any(1).sum()) == len(far)
    one = layers.linear_act(x, w[:1], act="none")
    _check_forward(x[far], w[:1], None, None, "none", one[far], "far rows, one output")
    gy = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    gy[far] = _rand(g, len(far), N, dtype=torch.bfloat16)
    c8, e8 = ops.mx8_encode(x)
    assert torch.equal(ops.mx8_decode(c8, e8, K, torch.bfloat16)[far], ops.mx8_decode(*ops.mx8_encode(x[far]), K, torch.bfloat16))
    gw, gw8, gx = torch.empty_like(w), torch.empty_like(w), torch.empty_like(x)
    ops.linear_backward(gy, x, w, gw=gw, gx=gx)
    ops.linear_backward(gy, None, w, x8=c8, x8e=e8, gw=gw8)
    want = gy[far].double().t() @ x[far].double()
    S = gy[far].double().abs().t() @ x[far].double().abs()
    _close(gw, want, _e(M, torch.bfloat16) * S + _half(want, torch.bfloat16), "gw")
    x8 = ops.mx8_decode(*ops.mx8_encode(x[far]), K, torch.bfloat16).double()
    want = gy[far].double().t() @ x8
    _close(gw8, want, _e(M, torch.bfloat16) * (gy[far].double().abs().t() @ x8.abs()) + _half(want, torch.bfloat16), "gw from codes")
    want, S = gy[far].double() @ w.double(), gy[far].double().abs() @ w.double().abs()
    _close(gx[far], want, _e(N, torch.bfloat16) * S + _half(want, torch.bfloat16), "gx")


def test_one_tensor_in_several_places():
    """x as its own residual, the weight of one layer in another: the gradients add up"""
    g = _gen(211)
    x = _rand(g, 90, 64, dtype=torch.float32).requires_grad_(True)
    w = _rand(g, 64, 64, dtype=torch.float32, std=0.1).requires_grad_(True)
    gy = _rand(g, 90, 64, dtype=torch.float32)

    def chain(f, x, w):
        return f(f(x, w, x), w, x)
    got = torch.autograd.grad(chain(lambda a, b, r: layers.linear_act(a, b, act="silu", residual=r), x, w), [x, w], gy)
    xd, wd = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    want = torch.autograd.grad(chain(lambda a, b, r: torch.nn.functional.silu(a @ b.t()) + r, xd, wd), [xd, wd], gy.double())
    for a, b in zip(got, want):
        assert float((a.double() - b).norm() / b.norm()) < 1e-5                # two layers of float32, 64 and 90 terms


def test_a_tensor_changed_after_the_forward_pass_is_noticed():
    x, w, b, _ = _forward_case(40, 32, 48, torch.float32, "none", 221)
    for t in (x, w):
        t.requires_grad_(True)
    y = layers.linear_act(x, w, b, act="relu")
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(torch.ones_like(y))


def test_under_no_grad_nothing_is_kept():
    x, w, b, _ = _forward_case(4000, 512, 512, torch.bfloat16, "gelu", 231)
    w.requires_grad_(True)
    layers.linear_act(x, w, b, act="gelu")
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    with torch.no_grad():
        y = layers.linear_act(x, w, b, act="gelu")
    assert not y.requires_grad and torch.cuda.memory_allocated() - base == y.numel() * 2


def test_eight_bit_checkpoints_take_a_quarter_of_float32():
    x, w, b, _ = _forward_case(8192, 1024, 1024, torch.float32, "silu", 241)
    w.requires_grad_(True)
    kept = {}
    for ck in (None, "mx8"):
        x1 = x.clone().requires_grad_(True)
        base = torch.cuda.memory_allocated()
        y = layers.linear_act(x1, w, b, act="silu", checkpoint=ck)
        kept[ck] = torch.cuda.memory_allocated() - base - y.numel() * 4 + (0 if ck else x1.numel() * 4)
        del y, x1
    assert kept["mx8"] * 3.8 < kept[None]                                      # 8.25 bits instead of 32 for the input and for z


CODES_SIZES = [(1, 64, 40), (300, 40, 1), (70, 33, 70), (65, 8, 200), (1003, 1001, 777), (300, 64, 2048), (4096, 96, 512), (129, 8200, 136), (5000, 512, 1024), (4100, 2080, 4096), (20000, 256, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_forward_writes_the_codes_of_its_input(dtype):
    """x8 / x8e of linear_forward are what mx8_encode writes, bit by bit: few rows, every tile, cut contractions, padded and strided rows, values that are not
    finite, blocks of zeros and of denormal numbers; the output does not change"""
    for M, K, N in CODES_SIZES:
        g = torch.Generator(device="cuda").manual_seed(M + K)
        x = torch.randn(M, K + 8, generator=g, device="cuda")
        x = (x * torch.exp(3 * torch.randn(M, K + 8, generator=g, device="cuda"))).to(dtype)
        x[:: 7, : 32] = 0.0
        x[1:: 7, : 32] *= torch.finfo(dtype).smallest_normal
        x = x[:, :K] if M % 2 else x[:, :K].contiguous()
        w = (torch.randn(N, K, generator=g, device="cuda") * K ** -0.5).to(dtype)
        for bad in (False, True):
            if bad:
                x[M // 2, K // 2] = float("nan")
                x[M - 1, K - 1] = -float("inf")
                x[0, : 33] = float("inf")
            want, want_e = ops.mx8_encode(x)
            got, got_e = torch.full_like(want, 77), torch.full_like(want_e, 77)
            y = ops.linear_forward(x, w, x8=got, x8e=got_e)
            assert torch.equal(got, want) and torch.equal(got_e, want_e), (M, K, N, bad)
            z = torch.empty(M, N, dtype=dtype, device="cuda")
            y2 = ops.linear_forward(x, w, act="silu", z=z, x8=got.fill_(77), x8e=got_e.fill_(77))
            assert torch.equal(got, want) and torch.equal(got_e, want_e), (M, K, N, bad)
            if not bad:
                # (fp16: the large values overflow, and the sums of infinities are NaN on both sides)
                for a, b in ((y, ops.linear_forward(x, w)), (y2, ops.linear_forward(x, w, act="silu", z=z))):
                    assert bool(((a == b) | (a.isnan() & b.isnan())).all()), (M, K, N)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_forward_writes_the_codes_of_every_number(dtype):
    """every 16-bit pattern, next to a large, a middling and a small neighbour that sets its block's power of two"""
    every = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16).view(dtype)
    lead = torch.tensor([1.0, 300.0, 2.0 ** -12], device="cuda").to(dtype)
    x = torch.cat([torch.cat([every.view(-1, 16), lead[i].expand(4096, 16)], 1) for i in range(3)] + [every.view(2048, 32).repeat(2, 1)], 0)
    w = torch.ones(96, 32, dtype=dtype, device="cuda")
    want, want_e = ops.mx8_encode(x)
    got, got_e = torch.empty_like(want), torch.empty_like(want_e)
    ops.linear_forward(x, w, x8=got, x8e=got_e)
    assert torch.equal(got, want) and torch.equal(got_e, want_e)
    # in order of magnitude, so that a block holds similar numbers
    order = every[torch.isfinite(every)].view(-1)
    order = order[order.float().abs().argsort()].reshape(-1, 32)
    want, want_e = ops.mx8_encode(order)
    got, got_e = torch.empty_like(want), torch.empty_like(want_e)
    ops.linear_forward(order, w, x8=got, x8e=got_e)
    assert torch.equal(got, want) and torch.equal(got_e, want_e)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("checkpoint", [None, "mx8"])
def test_small_backward_passes_do_not_round_dz(dtype, act, checkpoint):
    """the tolerances of _backward_check without the rounding of dz, with those of an fp32 product"""
    for M, N, K in ((1, 1, 1), (2, 8, 16), (4, 8, 16), (26, 8, 64), (34, 18, 56), (3, 3968, 16), (22, 106, 3119), (1505, 8, 64), (65, 129, 257), (128, 256, 256), (20000, 20, 20)):
        x, w, b, _ = _forward_case(M, N, K, dtype, act, 900 + M)
        gy = _rand(_gen(901 + M), M, N, dtype=dtype)
        z = _rand(_gen(902 + M), M, N, dtype=dtype)
        kw, xd, zd = dict(z=z), x.double(), z.double()
        if checkpoint:
            kw = dict(zip(("z8", "z8e", "x8", "x8e"), (*ops.mx8_encode(z), *ops.mx8_encode(x))))
            xd, zd = (torch.from_numpy(mx8_values(t.double().cpu().numpy())[0]).cuda() for t in (x, z))
        gx, gw = torch.empty(M, K, dtype=dtype, device="cuda"), torch.empty(N, K, dtype=dtype, device="cuda")
        ops.linear_backward(gy, None if checkpoint else x, w, act, gx=gx, gw=gw, **kw)
        dz = gy.double() * _slope64(zd, act)
        e_dz = gy.double().abs() * 16 * 2.0 ** -24 * (1 + zd.abs()) + 2.0 ** -24 * dz.abs()
        S, Sw = dz.abs() + e_dz, w.double().abs()
        for got, want, e, name in ((gx, dz @ w.double(), e_dz @ Sw + _e(N, torch.float32) * (S @ Sw), "gx"),
                                   (gw, dz.t() @ xd, e_dz.t() @ xd.abs() + _e(M, torch.float32) * (S.t() @ xd.abs()), "gw")):
            _close(got, want, e + _half(want.abs() + e, dtype), f"{name} {M}x{N}x{K}")


# many rows (and few), a weight of at most 256 x 256: whole and partial last tiles and widths, rows that are not whole vectors, one output
STREAM_SIZES = [(1, 8, 8), (31, 64, 64), (33, 256, 256), (700, 200, 120), (2000, 256, 256), (4100, 64, 64), (131075, 160, 24), (65536, 136, 256), (32768, 256, 256), (32801, 256, 256), (40007, 136, 72), (33000, 256, 16), (33001, 40, 200), (50000, 8, 256), (32769, 250, 136), (34000, 128, 128), (70001, 72, 8), (32800, 1, 100), (40000, 65, 33)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_many_rows_narrow_layers_forward(dtype, act, monkeypatch):
    monkeypatch.setitem(globals(), "SIZES", STREAM_SIZES)
    test_forward_over_sizes(dtype, act)
    if act == "gelu":
        test_what_the_forward_pass_keeps(dtype)
    if act == "none":
        monkeypatch.setitem(globals(), "CODES_SIZES", [(M, K, N) for M, N, K in STREAM_SIZES])
        test_forward_writes_the_codes_of_its_input(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("checkpoint", [None, "mx8"])
def test_many_rows_narrow_layers_backward(dtype, act, checkpoint):
    for i, (M, N, K) in enumerate(STREAM_SIZES):
        x, w, b, _ = _forward_case(M, N, K, dtype, act, 600 + i)
        gy = _rand(_gen(700 + i), M, N, dtype=dtype)
        nb = (N + 31) // 32
        saved, x_values = {}, None
        if act == "relu":
            saved["bits"] = torch.randint(-2 ** 31, 2 ** 31 - 1, (M, nb), dtype=torch.int32, device="cuda", generator=_gen(i))
            saved["on"] = ((saved["bits"].view(M, nb, 1) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool().view(M, -1)[:, :N]
        elif act != "none":
            z = _rand(_gen(800 + i), M, N, dtype=dtype, std=2.0)
            if checkpoint:
                saved["z8"], saved["z8e"] = ops.mx8_encode(z)
                saved["z_values"] = ops.mx8_decode(saved["z8"], saved["z8e"], N, torch.float32).double()
            else:
                saved["z"], saved["z_values"] = z, z.double()
        if checkpoint:
            saved["x8"], saved["x8e"] = ops.mx8_encode(x)
            x_values = ops.mx8_decode(saved["x8"], saved["x8e"], K, torch.float32).double()
        gx, gw, gb = _backward_check(gy, None if checkpoint else x, w, act, saved, dtype, f"{M}x{N}x{K}", x_values)
        # each gradient alone, gy in rows of another pitch: the same bits where the sums have the same order
        kw = {k: v for k, v in saved.items() if k in ("z", "bits", "z8", "z8e")}
        alone = torch.empty_like(gx)
        ops.linear_backward(gy, None, w, act, gx=alone, **kw)
        assert torch.equal(alone, gx), (M, N, K)
        wide = torch.zeros(M, N + 8, dtype=dtype, device="cuda")
        wide[:, :N] = gy
        ops.linear_backward(wide[:, :N], None, w, act, gx=alone.zero_(), **kw)
        assert torch.equal(alone, gx), (M, N, K)


@pytest.mark.parametrize("M,N,K", [(16384, 512, 512), (8200, 520, 1001), (4100, 1000, 1030), (65536, 136, 520)])
def test_large_fp32_products_with_a_weight_split_beforehand(M, N, K):
    """against the formula with an fp32 product's tolerances; a weight in rows of another pitch gives the same bits; numbers that are not finite stay in their rows and columns"""
    x, w, b, _ = _forward_case(M, N, K, torch.float32, "none", 31, residual=False)
    y = ops.linear_forward(x, w, b)
    _check_forward(x, w, b, None, "none", y, "y")
    gy = _rand(_gen(32), M, N, dtype=torch.float32)
    gx, _, _ = _backward_check(gy, x, w, "none", {}, torch.float32, "gradients")
    wide = torch.zeros(N, K + 3, device="cuda")
    wide[:, 1:K + 1] = w
    assert torch.equal(ops.linear_forward(x, wide[:, 1:K + 1], b), y)
    again = torch.empty_like(gx)
    ops.linear_backward(gy, None, wide[:, 1:K + 1], gx=again)
    assert torch.equal(again, gx)
    w[3, 5], w[7, K - 1], x[11, 2] = float("nan"), float("inf"), float("nan")
    y = ops.linear_forward(x, w, b)
    bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    bad[:, 3] = bad[:, 7] = bad[11] = True
    assert bool((torch.isfinite(y) == ~bad).all())
