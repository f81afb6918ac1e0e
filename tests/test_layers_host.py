"""CPU: the layer operators' descriptor mirror, their argument checks, and their refusal of tensors that do not live on the GPU (tests/test_gpu_layers.py and
tests/test_gpu_embedding.py hold the numerics)."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from nerf_loam_amd import _lib as L
from nerf_loam_amd import layers, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_linear_descriptor_mirror_matches_the_c_struct(tmp_path):
    import shutil
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    names = [n for n, _ in L.NlLinear._fields_]
    src = ['#include "nerfloam_hip.h"', "#include <stddef.h>", "#include <stdio.h>", "int main(void) {", '    printf("%zu", sizeof(NlLinear));']
    src += [f'    printf(" %zu", offsetof(NlLinear, {n}));' for n in names] + ["    return 0;", "}"]
    c = tmp_path / "desc.c"
    c.write_text("\n".join(src))
    exe = tmp_path / "desc"
    r = subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    vals = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(L.NlLinear)
    assert vals[1:] == [getattr(L.NlLinear, n).offset for n in names]
    hdr = open(os.path.join(ROOT, "include", "nerfloam_hip.h")).read()
    consts = dict(re.findall(r"#define\s+(NL_(?:DT|ACT|MX8)_[A-Z0-9]+)\s+(\d+)", hdr))
    assert {k: int(v) for k, v in consts.items()} == {"NL_DT_F32": 0, "NL_DT_BF16": 1, "NL_DT_F16": 2, "NL_ACT_NONE": 0, "NL_ACT_RELU": 1, "NL_ACT_GELU": 2, "NL_ACT_SILU": 3,
                                                      "NL_MX8_BLOCK": L.NL_MX8_BLOCK}
    assert [L.NL_DTYPES[str(t)] for t in (torch.float32, torch.bfloat16, torch.float16)] == [0, 1, 2]
    assert [L.NL_ACTS[a] for a in ("none", "relu", "gelu", "silu")] == [0, 1, 2, 3]


def _desc(**kw):
    d = L.NlLinear(struct_size=ctypes.sizeof(L.NlLinear), dtype=1, act=0, K=64, N=32, M=8)
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 255) & ~255
    d.x = d.w = d.y = d.gy = d.gx = d.gw = p
    d.ldx = d.ldw = 64
    d.ldy = d.ldgy = 32
    d._keep = buf
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("bad", [dict(struct_size=8), dict(dtype=7), dict(dtype=-1), dict(act=4), dict(M=-1), dict(K=0), dict(N=0), dict(K=1 << 23), dict(ldx=63), dict(ldw=63),
                                 dict(ldy=31), dict(x=None), dict(w=None), dict(y=None), dict(x=4097), dict(z8=4096)])
def test_linear_forward_refuses_a_bad_descriptor(bad):
    lib = L.lib()
    assert lib.nl_linear_workspace(ctypes.byref(_desc()), 0) >= 0
    d = _desc(**bad)
    assert lib.nl_linear_workspace(ctypes.byref(d), 0) == -1
    assert lib.nl_linear_forward(ctypes.byref(d), None) == 1


@pytest.mark.parametrize("bad", [dict(gy=None), dict(ldgy=31), dict(w=None), dict(x=None), dict(act=1), dict(act=2), dict(act=3), dict(act=2, z8=4096), dict(x8=4096), dict(act=2, z=4098)])
def test_linear_backward_refuses_a_bad_descriptor(bad):
    lib = L.lib()
    assert lib.nl_linear_workspace(ctypes.byref(_desc()), 1) >= 0
    d = _desc(**bad)
    assert lib.nl_linear_workspace(ctypes.byref(d), 1) == -1
    assert lib.nl_linear_backward(ctypes.byref(d), None) == 1


def test_a_workspace_that_is_too_small_is_refused_before_a_launch():
    """few results, a long contraction: the product is cut and its pieces need a workspace"""
    lib = L.lib()
    d = _desc(M=1 << 16, K=64, N=32, gx=None)
    need = lib.nl_linear_workspace(ctypes.byref(d), 1)
    assert need > 0
    d.ws_bytes = need
    assert lib.nl_linear_backward(ctypes.byref(d), None) == 1                   # no workspace
    d.ws, d.ws_bytes = 1 << 20, need - 1
    assert lib.nl_linear_backward(ctypes.byref(d), None) == 1                   # too small
    d.ws, d.ws_bytes = (1 << 20) + 8, need
    assert lib.nl_linear_backward(ctypes.byref(d), None) == 1                   # misaligned
    assert lib.nl_embedding_backward(None, 10, 16, 1, 1 << 20, 0, None, 100, 1, 1.0, 1 << 20, 1 << 20, None, 1 << 20, 16, None) == 1


def test_checkpoint_and_embedding_entry_points_refuse_bad_arguments():
    lib, p = L.lib(), 1 << 20
    for a in [(p, 31, 4, 32, 1, p, p), (p, 32, -1, 32, 1, p, p), (p, 32, 4, 0, 1, p, p), (p, 32, 4, 32, 5, p, p), (None, 32, 4, 32, 1, p, p), (p, 32, 4, 32, 1, None, p),
              (p, 32, 4, 32, 1, p, None), (p + 1, 32, 4, 32, 1, p, p), (p, 32, 4, 32, 1, p + 4, p)]:
        assert lib.nl_mx8_encode(*a, None) == 1, a
    for a in [(None, p, 4, 32, 1, p), (p, None, 4, 32, 1, p), (p, p, 4, 32, 1, None), (p, p, 4, 32, 9, p), (p, p, 4, 32, 1, p + 2), (p, p, -4, 32, 1, p)]:
        assert lib.nl_mx8_decode(*a, None) == 1, a
    ok = dict(table=p, V=10, D=16, dt=1, ids=p, id64=0, w=None, M=4, bag=1, scale=1.0, out=p)
    for bad in [dict(table=None), dict(V=0), dict(V=1 << 31), dict(D=0), dict(dt=4), dict(ids=None), dict(ids=p + 2), dict(id64=1, ids=p + 4), dict(M=-1), dict(bag=0), dict(out=None),
                dict(M=1 << 31), dict(M=1 << 28, bag=16), dict(w=p + 2), dict(out=p + 1)]:
        assert lib.nl_embedding_forward(*{**ok, **bad}.values(), None) == 1, bad
    assert lib.nl_embedding_workspace(0, 16, 4, 1) == -1 and lib.nl_embedding_workspace(10, 16, 0, 1) == 0 and lib.nl_embedding_workspace(10, 16, 4, 1) > 0


def test_no_cpu_path_and_no_unknown_choice():
    x, w = torch.zeros(4, 8), torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.linear_act(x, w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.linear_act(x.requires_grad_(True), w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.checkpoint_encode(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.checkpoint_decode(layers.Checkpoint8(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), (4, 8), torch.float32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.embedding_lookup(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="act"):
        layers.linear_act(x, w, act="tanh")
    with pytest.raises(ValueError, match="checkpoint"):
        layers.linear_act(x, w, checkpoint="int4")
    assert ops.linear_forward is not None


def test_decoders_of_any_size_refuse_the_cpu_and_unknown_shapes():
    from nerf_loam_amd.decoder import Decoder
    dec = Decoder(depth=3, width=40, in_dim=16, skips=[0])
    assert [tuple(l.weight.shape) for l in dec.pts_linears] == [(40, 16), (40, 56), (40, 40)] and not dec.fused and Decoder().fused
    with pytest.raises(RuntimeError, match="no CPU path"):
        dec(torch.zeros(4, 16))
    with pytest.raises(ValueError):
        Decoder(depth=2, skips=[1])
    with pytest.raises(NotImplementedError):
        Decoder(embedder="gaussian")


def test_sizes_beyond_a_launch_are_refused():
    """what would need more than 2^32 threads along a grid's axis is refused where its workspace is asked for, not where it is launched"""
    lib = L.lib()
    for sizes in [dict(M=(1 << 30) + 1), dict(M=1 << 30, N=2048), dict(K=(1 << 22) + 1, ldx=1 << 23, ldw=1 << 23)]:
        d = _desc(**sizes)
        d.ldy = d.ldgy = d.ldr = max(d.N, d.ldy)
        assert lib.nl_linear_workspace(ctypes.byref(d), 0) == -1 and lib.nl_linear_forward(ctypes.byref(d), None) == 1, sizes
    assert lib.nl_embedding_workspace(10, 4, (1 << 30) - 63, 1) == -1 and lib.nl_embedding_workspace(10, 4, (1 << 30) - 64, 1) > 0


@pytest.mark.parametrize("bad", [dict(x8=4096), dict(x8e=4096), dict(x8=4104, x8e=4096)])
def test_linear_forward_refuses_half_a_checkpoint(bad):
    lib = L.lib()
    assert lib.nl_linear_workspace(ctypes.byref(_desc(x8=4096, x8e=4096)), 0) >= 0
    d = _desc(**bad)
    assert lib.nl_linear_workspace(ctypes.byref(d), 0) == -1
    assert lib.nl_linear_forward(ctypes.byref(d), None) == 1
