"""Differentiable layer operators: what a decoder of any size and its embedding table train with.

The reference composes these from torch.nn.Linear, ReLU (src/variations/lidar.py:105-123) and F.embedding (src/variations/render_helpers.py:85-89) under autograd;
here each is one call into hand-written kernels (csrc/nl_linear.hip, nl_checkpoint.hip, nl_embedding.hip), forward and backward:

* linear_act        act(x weight^T + bias) + residual, optionally with what the backward pass needs kept in 8 bits
* embedding_lookup  scaled (weighted) sums of table rows; the table's gradient is summed over sorted ids - the same bits every run
* checkpoint_encode / checkpoint_decode  the 8-bit format itself

Tensors live on the GPU (there is no CPU path), types are float32, bfloat16 and float16.  Gradients of gradients and forward-mode derivatives are not provided
and refused (a gradient that depends on no trained tensor is a constant).  The backward passes refuse to run through autograd while a stream is being captured: capture ops.linear_forward / linear_backward and ops.embedding_forward / embedding_backward
instead, which are the same kernels on caller-owned tensors (autograd's leaf nodes belong to the stream of an earlier eager pass, and waiting for that stream
inside a capture cannot be undone)."""
import ctypes
import os
from collections import namedtuple

from . import _lib as L

ACTIVATIONS = tuple(L.NL_ACTS)
CHECKPOINTS = (None, "mx8")

Checkpoint8 = namedtuple("Checkpoint8", "codes exps shape dtype")
Checkpoint8.__doc__ = """an activation kept in 8 bits: codes uint8 [rows, up(K, 32)], exps uint8 [rows, ceil(K / 32)], shape and dtype of the tensor it was made from"""

_ext = None


def _load():
    """the compiled host side (torch_ext/layers_torch.cpp), bound to the functions of the library that _lib loaded"""
    global _ext
    if _ext is None:
        lib = L.lib()
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_layers_torch.so")
        if not os.path.exists(path):
            raise L.NerfLoamHipError(f"{path} not found - run `python -m nerf_loam_amd.build`; the layer operators have no PyTorch fallback")
        import torch  # noqa: F401
        from . import _layers_torch
        _layers_torch.bind(L.NerfLoamHipError, {n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in L.EXPORTED_SYMBOLS
                                                if n.startswith(("nl_linear_", "nl_mx8_", "nl_embedding_"))})
        _ext = _layers_torch
    return _ext


def linear_act(x, weight, bias=None, act="none", residual=None, checkpoint=None):
    """act(x weight^T + bias) + residual.

    x [..., K], weight [N, K], bias [N] or None, residual [..., N] or None, all of one type -> [..., N].  act: "none", "relu", "gelu" (exact, with erf), "silu".
    Differentiable with respect to the four tensors.  Kept for the backward pass: x and weight, and of z = x weight^T + bias one bit per element (relu) or z itself
    (gelu, silu); with checkpoint="mx8" x and z are kept in 8 bits with a power of two per 32 features (checkpoint_encode): a quarter of float32's memory, and
    gradients computed from the rounded values.  float32 products are as exact as float32 sums (six bf16 products of splits, exact for magnitudes from 2^-110 on,
    below that off by at most 2^-134); an infinity among float32 operands gives NaN, in calls with more than eight rows and outputs and in backward passes.  In 16 bits the gradient of z is rounded once to the type before it is multiplied (not for short gelu and silu layers, up to 2^23
    multiplications a product: their backward products run like float32's)."""
    code = L.NL_ACTS.get(act)
    if code is None:
        raise ValueError(f"linear_act: act {act!r} must be one of {ACTIVATIONS}")
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"linear_act: checkpoint {checkpoint!r} must be one of {CHECKPOINTS}")
    return (_ext or _load()).linear_act(x, weight, bias, code, residual, checkpoint is not None)


def checkpoint_encode(x):
    """x [..., K] -> Checkpoint8: e4m3 codes, 32 neighbouring features sharing the smallest power of two 2^e (e >= -126) with max |x| <= 448 2^e; to nearest, ties to
    even.  Infinities and NaN come back as NaN."""
    codes, exps = (_ext or _load()).checkpoint_encode(x)
    return Checkpoint8(codes, exps, tuple(x.shape), x.dtype)


def checkpoint_decode(c):
    """the values a Checkpoint8 stands for, in the shape and type of the tensor it was made from (what rounded up beyond the type's largest number is
    that number)"""
    return (_ext or _load()).checkpoint_decode(*c)


def embedding_lookup(table, ids, scale=1.0, weights=None):
    """scale * table[ids], or with weights the weighted sum of a bag of rows: scale * sum_k weights[..., k] table[ids[..., k]].

    table [V, D]; ids [...] (with weights [..., bag]) of int32 or int64, an id outside [0, V) selects no row: zeros, no gradient; weights float32 in the shape of
    ids -> [..., D] of the table's type.  Differentiable with respect to table and weights; the table's gradient is dense and bit-reproducible (sorted ids)."""
    return (_ext or _load()).embedding_lookup(table, ids, scale, weights)
