"""GPU (-m gpu): the streaming product in the forward pass (csrc/nl_narrow.h): many rows, more than 128 outputs, a weight of at most 256 x 256 in 16 bits.  That the sizes here and in
test_gpu_layers.STREAM_SIZES run as it is held on the host (tests/test_layers_streaming_host.py).  Tolerances: test_gpu_layers."""
import pytest
import torch

import test_gpu_layers as T
from nerf_loam_amd import ops

pytestmark = pytest.mark.gpu

# (M, N, K): the decoder's width; outputs and contractions that are no whole vectors, alone and together; the shortest contractions; partial last tiles of rows
FORWARD_SIZES = [(65537, 256, 256), (70001, 250, 136), (66000, 129, 137), (131075, 256, 16), (65536, 160, 5), (65600, 256, 250), (65567, 136, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", FORWARD_SIZES)
@pytest.mark.parametrize("bias,residual", [(True, True), (False, False)])
def test_everything_the_forward_pass_writes(M, N, K, dtype, bias, residual):
    """y with each activation, bias and residual at once or neither; the bits, z, z in 8 bits; the codes of x in the same launch or not; nothing else is written"""
    x, w, b, r = T._forward_case(M, N, K, dtype, "gelu", 1000 + N, bias=bias, residual=residual)
    nb, kb = (N + 31) // 32, (K + 31) // 32
    z64, S = T._z64(x, w, b)
    ez = T._e(K, dtype) * S
    want8, want8e = ops.mx8_encode(x)

    def new(*s, t=torch.uint8):
        return torch.full(s, 77, dtype=t, device="cuda")
    for act, codes in (("none", False), ("none", True), ("relu", False), ("relu", True), ("gelu", False), ("gelu", True), ("silu", False), ("silu", True)):
        kept = {}
        if act == "relu":
            kept["bits"] = new(M, nb, t=torch.int32)
        elif act == "gelu":
            kept["z"] = new(M, N, t=dtype)
        elif act == "silu":
            kept.update(z8=new(M, 32 * nb), z8e=new(M, nb))
        if codes:
            kept.update(x8=new(M, 32 * kb), x8e=new(M, kb))
        out = torch.full((M + 3, N + 6), 5.0, dtype=dtype, device="cuda")
        ops.linear_forward(x, w, b, act, r, out=out[1:M + 1, 2:N + 2], **kept)
        what = f"{act} codes {codes}"
        T._check_forward(x, w, b, r, act, out[1:M + 1, 2:N + 2], "y " + what)
        assert bool((out[0] == 5).all() and (out[M + 1:] == 5).all() and (out[:, :2] == 5).all() and (out[:, N + 2:] == 5).all())
        if codes:
            assert torch.equal(kept["x8"], want8) and torch.equal(kept["x8e"], want8e), what
        if act == "relu":
            on = ((kept["bits"].view(M, nb, 1) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool().view(M, -1)
            assert bool((on[:, :N] == (z64 > 0))[z64.abs() > ez].all()) and not bool(on[:, N:].any()), what
        if act == "gelu":
            T._close(kept["z"], z64, ez + T._half(z64.abs() + ez, dtype), "z " + what)
        if act == "silu":
            e = kept["z8e"].double() - 127
            step = torch.exp2(e).repeat_interleave(32, 1)[:, :N] * 2.0 ** -10
            T._close(ops.mx8_decode(kept["z8"], kept["z8e"], N, torch.float32).double(), z64, ez + torch.maximum((z64.abs() + ez) * 2.0 ** -4, step), "z8 " + what)
            top, slack = (torch.nn.functional.pad(t, (0, 32 * nb - N)).view(M, nb, 32).amax(2) for t in (z64.abs(), ez))
            assert bool((top - slack <= 448 * torch.exp2(e)).all()) and bool(((top + slack > 224 * torch.exp2(e)) | (e == -126)).all()), what
            assert not bool(kept["z8"][:, N:].any()), what


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_numbers_that_are_not_finite_stay_in_their_rows(dtype):
    M, N, K = 65601, 250, 137
    x, w, b, r = T._forward_case(M, N, K, dtype, "relu", 5)
    clean = ops.linear_forward(x, w, b, "relu", r)
    bad = x.clone()
    bad[65600, K - 1], bad[31, 0], bad[40000, 64] = float("nan"), float("inf"), float("nan")
    y = ops.linear_forward(bad, w, b, "relu", r)
    rows = torch.ones(M, dtype=torch.bool, device="cuda")
    rows[[65600, 31, 40000]] = False
    assert torch.equal(y[rows], clean[rows]) and bool(y[65600].isnan().all() and y[40000].isnan().all())
    z = bad[31].double() @ w.double().t() + b.double()
    assert bool((y[31].double() == torch.relu(z) + r[31].double())[~torch.isfinite(z) & (z > 0)].all())
