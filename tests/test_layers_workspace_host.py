"""CPU: the bound that the header gives for the layer operators' workspace, over the sizes that they take"""
import ctypes
import random

import pytest

from nerf_loam_amd import _lib as L


def _up(a, b):
    return -(-a // b) * b


@pytest.mark.parametrize("dtype,es", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("backward", [0, 1])
def test_a_workspace_stays_within_its_bound(dtype, es, backward):
    rng = random.Random(7 + dtype)
    p = 1 << 20
    for i in range(4000):
        M, N, K = (int(2 ** rng.uniform(0, top)) for top in (26, 14, 14))
        act, kept, eight = rng.randrange(4), rng.random() < 0.5, rng.random() < 0.5
        d = L.NlLinear(struct_size=ctypes.sizeof(L.NlLinear), dtype=dtype, act=act, K=K, N=N, M=M, x=p, ldx=K, w=p, ldw=K, b=p, y=p, ldy=N, gy=p, ldgy=N)
        d.bits = p if act == 1 and (kept or backward) else None
        if act > 1 and (kept or backward):
            d.z, d.z8, d.z8e = (None, p, p) if eight else (p, None, None)
        if eight:
            d.x8 = d.x8e = p
        if backward:
            d.gx, d.gw, d.gb = (p if rng.random() < 0.7 else None for _ in range(3))
        need = L.lib().nl_linear_workspace(ctypes.byref(d), backward)
        tiles = -(-M // 64) * -(-max(N, K if backward else 1) // 64)                # the header's limit: fewer than 2^24
        if need < 0 and tiles >= 1 << 24:
            continue
        assert need >= 0, (M, N, K)
        copies = (M * _up(K, 8) + N * _up(K, 8)) * es
        bound = copies + 6 * N * _up(K, 8) + 1500000000 + 4096
        if backward:
            bound += M * _up(N, 8) * 4 + (32 << 20)
        assert need <= bound, (M, N, K, act, need, bound)
        # rows of whole 16 bytes, results of which two pieces would be more than 1.5 GB (8 M N bytes), no gradients: nothing is needed
        if not backward and K % 8 == 0 and M > 8 and N > 8 and dtype and 8 * M * N > 1500000000:
            assert need == 0, (M, N, K)
