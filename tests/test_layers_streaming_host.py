"""CPU: enough of the sizes that are meant to test the streaming product run as it, whatever becomes of the rule that chooses it (csrc/nl_linear.hip)"""
import ctypes

import pytest

import test_gpu_layers as T
from nerf_loam_amd import _lib as L
from test_gpu_layers_streaming import FORWARD_SIZES


def _streams(M, N, K, dtype, act, backward=False, **kw):
    p = 1 << 20
    d = L.NlLinear(struct_size=ctypes.sizeof(L.NlLinear), dtype=dtype, act=act, K=K, N=N, M=M, x=p, ldx=K, w=p, ldw=K, y=p, ldy=N)
    if backward:
        d.gy, d.ldgy, d.gx, d.bits, d.z = p, N, p, p, p
    for k, v in kw.items():
        setattr(d, k, v)
    return L.lib().nl_linear_streams(ctypes.byref(d), int(backward))


@pytest.mark.parametrize("dtype", [1, 2])
def test_forward_sizes_stream(dtype):
    p = 1 << 20
    for act in range(4):
        for kept in (dict(), dict(bits=p), dict(z=p), dict(z8=p, z8e=p), dict(x8=p, x8e=p)):
            assert all(_streams(*s, dtype, act, **kept) == 1 for s in FORWARD_SIZES)
    assert any(N == 256 for _, N, _ in FORWARD_SIZES) and any(N % 8 for _, N, _ in FORWARD_SIZES) and any(K % 8 and N % 8 == 0 for _, N, K in FORWARD_SIZES)
    assert any(K <= 128 and N > 128 for _, N, K in FORWARD_SIZES) and any(K > 128 for _, _, K in FORWARD_SIZES) and any(M % 32 for M, _, _ in FORWARD_SIZES)


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("act", [1, 2, 3])
def test_backward_sizes_stream(dtype, act):
    """every pair of whole-vector sizes of the list; both halves of either limit among them"""
    hit = [(M, N, K) for M, N, K in T.STREAM_SIZES if _streams(M, N, K, dtype, act, backward=True) == 1]
    assert len(hit) >= 10 and {(N <= 128, K <= 128) for _, N, K in hit} == {(a, b) for a in (True, False) for b in (True, False)}, hit
    assert any(M % 32 for M, _, _ in hit) and any(M > 65536 for M, _, _ in hit)
    # a residual-free layer without an activation streams for many rows and wide inputs
    assert _streams(65536, 136, 256, dtype, 0, backward=True) == 1


def test_what_does_not_stream():
    p = 1 << 20
    assert _streams(65537, 256, 256, 0, 1) == 0 and _streams(65537, 128, 256, 1, 1) == 0 and _streams(65537, 257, 256, 1, 1) == 0 and _streams(8, 256, 256, 1, 1) == 0
    assert _streams(0, 256, 256, 1, 1) == 0 and _streams(-1, 256, 256, 1, 1) == -1 and _streams(65537, 256, 256, 1, 7) == -1
    assert _streams(65537, 256, 256, 1, 1, backward=True, gy=p + 2) == 0 and _streams(65537, 256, 250, 1, 1, backward=True) == 0
