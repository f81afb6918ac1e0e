"""GPU (-m gpu): where fp32 products stop being exact, and refusals that must leave their outputs alone.

x = h + m + l, three bf16 numbers.  A number of magnitude 2^e has its last bit at 2^(e - 23); bf16's smallest is 2^-133.  From e = -110 on the three parts hold every bit; below, the
last part is rounded to a multiple of 2^-133, so x is off by at most 2^-134.  With weights of size 2^100 every product is far inside fp32's range, so that is all that is lost beside
the product's own (6 K + 8) 2^-23 of its magnitudes."""
import pytest
import torch

from nerf_loam_amd import _lib as L
from nerf_loam_amd import ops

pytestmark = pytest.mark.gpu


def _off(x):
    return torch.where(x.abs() < 2.0 ** -110, 2.0 ** -134, 0.0).double()


@pytest.mark.parametrize("M,N,K", [(64, 64, 64), (300, 257, 129), (4100, 512, 640), (70, 9, 2000)])      # (the third splits its weight beforehand)
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -110, 1e-36, 2.0 ** -125, 2.0 ** -140])
def test_fp32_products_of_tiny_operands(M, N, K, size):
    g = torch.Generator(device="cuda").manual_seed(M)
    x1, large = torch.randn(M, K, generator=g, device="cuda"), torch.randn(N, K, generator=g, device="cuda") * 2.0 ** 100
    for x, w in ((x1 * size, large), (x1 * 2.0 ** 100, large * 2.0 ** -100 * size)):                     # tiny inputs, and tiny weights
        y = ops.linear_forward(x, w).double()
        X, W = x.double(), w.double()
        tol = (6 * K + 8) * 2.0 ** -23 * (X.abs() @ W.abs().t()) + _off(x) @ W.abs().t() + X.abs() @ _off(w).t() + 2.0 ** -149
        d = (y - X @ W.t()).abs()
        assert bool((d <= tol).all()), float((d / tol).max())
    # and in the gradients
    gx, gw = torch.empty(M, K, device="cuda"), torch.empty(N, K, device="cuda")
    gy = torch.randn(M, N, generator=g, device="cuda") * size
    ops.linear_backward(gy, large[:1].expand(M, K).contiguous(), large, gx=gx, gw=gw)
    G, W, X = gy.double(), large.double(), large[:1].double().expand(M, K)
    for got, want, S, off, n in ((gx, G @ W, G.abs() @ W.abs(), _off(gy) @ W.abs(), N), (gw, G.t() @ X, G.t().abs() @ X.abs(), _off(gy).t() @ X.abs(), M)):
        d = (got.double() - want).abs()
        tol = (6 * n + 8) * 2.0 ** -23 * S + off + 2.0 ** -149
        assert bool((d <= tol).all()), float((d / tol).max())


@pytest.mark.parametrize("exponent", [-100, -109, -110, -111, -118, -126, -130])
def test_fp32_keeps_every_bit_down_to_its_limit(exponent):
    """one product a result: 24-bit numbers of one binade, times a power of two"""
    M = 4096
    m = torch.randint(2 ** 23, 2 ** 24, (M,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).double()
    x = torch.zeros(M, 16, device="cuda")
    x[:, 3] = (m * 2.0 ** (exponent - 23)).float()                       # (below 2^-126 fp32 itself has fewer bits: what is stored counts)
    w = torch.zeros(16, 16, device="cuda")
    w[5, 3] = 2.0 ** 100
    got = ops.linear_forward(x, w)[:, 5].double() * 2.0 ** -100
    d = (got - x[:, 3].double()).abs()
    assert not bool(d.any()) if exponent >= -110 else bool((d <= 2.0 ** -134).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_infinity_by_size(dtype):
    """few rows or few outputs: as IEEE has it; more of both: NaN in fp32 (a part of the split is zero, an infinity times it is not a number), an infinity in 16 bits"""
    for M, N, few in ((8, 40, True), (40, 8, True), (9, 40, False), (40, 9, False)):
        x = torch.full((M, 32), 0.5, device="cuda", dtype=dtype)
        w = torch.full((N, 32), 0.25, device="cuda", dtype=dtype)
        x[1, 3] = float("inf")
        y = ops.linear_forward(x, w)
        assert bool(torch.isfinite(y[0]).all() and torch.isfinite(y[2:]).all())
        assert bool((y[1] == float("inf")).all()) if few or dtype != torch.float32 else bool(y[1].isnan().all()), (M, N)


@pytest.mark.parametrize("V,D,dtype", [(7, 3, torch.bfloat16), (40, 16, torch.float32)])
def test_a_refused_embedding_gradient_writes_nothing(V, D, dtype):
    """a workspace that is missing, too small or misaligned: refused before the first launch"""
    table, g = torch.randn(V, D, device="cuda").to(dtype), torch.randn(20, D, device="cuda").to(dtype)
    ids, wt = torch.zeros(20, 2, dtype=torch.int32, device="cuda"), torch.rand(20, 2, device="cuda")
    gt, gw = torch.full_like(table, 7.0), torch.full_like(wt, 7.0)
    need = L.lib().nl_embedding_workspace(V, D, 20, 2)
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    for p, n in ((None, need), (ws.data_ptr(), need - 1), (ws.data_ptr() + 8, need)):
        assert L.lib().nl_embedding_backward(table.data_ptr(), V, D, L.NL_DTYPES[str(dtype)], ids.data_ptr(), 0, wt.data_ptr(), 20, 2, 1.0, g.data_ptr(), gt.data_ptr(), gw.data_ptr(), p, n,
                                             None) == 1
    torch.cuda.synchronize()
    assert bool((gt == 7).all() and (gw == 7).all())
    ops.embedding_backward(table, ids, g, wt, 1.0, gt, gw, ws)
    assert not bool((gt[0] == 7).all()) and not bool(gt[1:].any()) and not bool((gw == 7).any())
