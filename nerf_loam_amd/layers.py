"""Differentiable layer operators: what a decoder of any size and its embedding table train with.

The reference composes these from torch.nn.Linear, ReLU (src/variations/lidar.py:105-123) and F.embedding (src/variations/render_helpers.py:85-89) under autograd;
here each is one call into hand-written kernels (csrc/nl_linear.hip, nl_checkpoint.hip, nl_embedding.hip), forward and backward:

* linear_act        act(x weight^T + bias) + residual, optionally with what the backward pass needs kept in 8 bits
* embedding_lookup  scaled (weighted) sums of table rows; the table's gradient is summed over sorted ids - the same bits every run
* checkpoint_encode / checkpoint_decode  the 8-bit format itself

Tensors live on the GPU (there is no CPU path), types are float32, bfloat16 and float16.  Gradients of gradients are not provided.  The backward passes
refuse to run through autograd while a stream is being captured: capture ops.linear_forward / linear_backward and ops.embedding_forward / embedding_backward
instead, which are the same kernels on caller-owned tensors (autograd's leaf nodes belong to the stream of an earlier eager pass, and waiting for that stream
inside a capture cannot be undone)."""
from collections import namedtuple

import torch

from . import _lib as L
from . import ops

ACTIVATIONS = tuple(L.NL_ACTS)
CHECKPOINTS = (None, "mx8")

Checkpoint8 = namedtuple("Checkpoint8", "codes exps shape dtype")
Checkpoint8.__doc__ = """an activation kept in 8 bits: codes uint8 [rows, up(K, 32)], exps uint8 [rows, ceil(K / 32)], shape and dtype of the tensor it was made from"""


def _no_capture(what):
    if torch.cuda.is_current_stream_capturing():
        raise L.NerfLoamHipError(f"{what}: the backward pass cannot run through autograd while a stream is being captured; capture the functions of ops instead")


def _rows2d(t, cols):
    """[..., cols] -> [rows, cols] with adjacent elements in a row; a copy only where the strides allow nothing else"""
    t = t.reshape(-1, cols)
    if (cols > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t


def _linear_forward(x, weight, bias, residual, act, checkpoint, keep):
    """-> (y [M,N], what the backward pass needs of z: (z, bits, z8, z8e))"""
    M, N = x.shape[0], weight.shape[0]
    z = bits = z8 = z8e = None
    if keep and act != "none":
        nb = (N + 31) // 32
        if act == "relu":
            bits = torch.empty(M, nb, dtype=torch.int32, device=x.device)
        elif checkpoint == "mx8":
            z8 = torch.empty(M, 32 * nb, dtype=torch.uint8, device=x.device)
            z8e = torch.empty(M, nb, dtype=torch.uint8, device=x.device)
        else:
            z = torch.empty(M, N, dtype=x.dtype, device=x.device)
    y = ops.linear_forward(x, weight, bias, act, residual, z=z, bits=bits, z8=z8, z8e=z8e)
    return y, (z, bits, z8, z8e)


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, checkpoint):
        need = ctx.needs_input_grad
        y, kept = _linear_forward(x, weight, bias, residual, act, checkpoint, need[0] or need[1] or need[2])
        x8 = x8e = None
        if need[1] and checkpoint == "mx8":
            x8, x8e = ops.mx8_encode(x)
        ctx.save_for_backward(x if need[1] and x8 is None else None, weight, x8, x8e, *kept)
        ctx.act = act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        _no_capture("linear_act")
        x, weight, x8, x8e, z, bits, z8, z8e = ctx.saved_tensors
        need = ctx.needs_input_grad
        g2 = _rows2d(gy, weight.shape[0])
        gx = torch.empty(g2.shape[0], weight.shape[1], dtype=gy.dtype, device=gy.device) if need[0] else None
        gw = torch.empty_like(weight, memory_format=torch.contiguous_format) if need[1] else None
        gb = torch.empty(weight.shape[0], dtype=gy.dtype, device=gy.device) if need[2] else None
        if gx is not None or gw is not None or gb is not None:
            ops.linear_backward(g2, x, weight, ctx.act, z, bits, z8, z8e, x8, x8e, gx, gw, gb)
        return gx, gw, gb, (gy if need[3] else None), None, None


def linear_act(x, weight, bias=None, act="none", residual=None, checkpoint=None):
    """act(x weight^T + bias) + residual.

    x [..., K], weight [N, K], bias [N] or None, residual [..., N] or None, all of one type -> [..., N].  act: "none", "relu", "gelu" (exact, with erf), "silu".
    Differentiable with respect to the four tensors.  Kept for the backward pass: x and weight, and of z = x weight^T + bias one bit per element (relu) or z itself
    (gelu, silu); with checkpoint="mx8" x and z are kept in 8 bits with a power of two per 32 features (checkpoint_encode): a quarter of float32's memory, and
    gradients computed from the rounded values.  float32 products are as exact as float32 sums (six bf16 products of exact splits)."""
    if act not in L.NL_ACTS:
        raise ValueError(f"linear_act: act {act!r} must be one of {ACTIVATIONS}")
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"linear_act: checkpoint {checkpoint!r} must be one of {CHECKPOINTS}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_act: x {tuple(x.shape)} must be [..., K] and weight {tuple(weight.shape)} [N, K]")
    N, K = weight.shape
    lead = x.shape[:-1]
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"linear_act: bias {tuple(bias.shape)} must be [{N}]")
    if residual is not None and tuple(residual.shape) != (*lead, N):
        raise ValueError(f"linear_act: residual {tuple(residual.shape)} must be {(*lead, N)}")
    x2 = _rows2d(x, K)
    w2 = _rows2d(weight, K)
    b = None if bias is None else bias.contiguous()
    r2 = None if residual is None else _rows2d(residual, N)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (b is not None and b.requires_grad) or (r2 is not None and r2.requires_grad)):
        y = _LinearAct.apply(x2, w2, b, r2, act, checkpoint)
    else:
        y, _ = _linear_forward(x2, w2, b, r2, act, checkpoint, False)
    return y if len(lead) == 1 else y.view(*lead, N)


def checkpoint_encode(x):
    """x [..., K] -> Checkpoint8: e4m3 codes, 32 neighbouring features sharing the smallest power of two 2^e (e >= -126) with max |x| <= 448 2^e; to nearest, ties to
    even.  Infinities and NaN come back as NaN."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"checkpoint_encode: x {tuple(x.shape)} must be [..., K], K >= 1")
    codes, exps = ops.mx8_encode(_rows2d(x.detach(), x.shape[-1]))
    return Checkpoint8(codes, exps, tuple(x.shape), x.dtype)


def checkpoint_decode(c):
    """the values a Checkpoint8 stands for, in the shape and type of the tensor it was made from (what rounded up beyond the type's largest number is
    that number)"""
    return ops.mx8_decode(c.codes, c.exps, c.shape[-1], c.dtype).view(c.shape)


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, weights, scale):
        ctx.save_for_backward(table, ids, weights)
        ctx.scale = scale
        return ops.embedding_forward(table, ids, weights, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        _no_capture("embedding_lookup")
        table, ids, weights = ctx.saved_tensors
        gt = torch.empty_like(table) if ctx.needs_input_grad[0] else None
        gw = torch.empty_like(weights) if ctx.needs_input_grad[2] else None
        if gt is not None or gw is not None:
            ops.embedding_backward(table, ids, g.contiguous(), weights, ctx.scale, gt, gw)
        return gt, None, gw, None


def embedding_lookup(table, ids, scale=1.0, weights=None):
    """scale * table[ids], or with weights the weighted sum of a bag of rows: scale * sum_k weights[..., k] table[ids[..., k]].

    table [V, D]; ids [...] (with weights [..., bag]) of int32 or int64, an id outside [0, V) selects no row: zeros, no gradient; weights float32 in the shape of
    ids -> [..., D] of the table's type.  Differentiable with respect to table and weights; the table's gradient is dense and bit-reproducible (sorted ids)."""
    if table.dim() != 2:
        raise ValueError(f"embedding_lookup: table {tuple(table.shape)} must be [V, D]")
    if weights is not None and (weights.shape != ids.shape or ids.dim() < 1 or ids.shape[-1] < 1):
        raise ValueError(f"embedding_lookup: weights {tuple(weights.shape)} must have the shape of ids {tuple(ids.shape)}, [..., bag]")
    lead = ids.shape if weights is None else ids.shape[:-1]
    bag = 1 if weights is None else ids.shape[-1]
    i2 = ids.reshape(-1, bag).contiguous()
    w2 = None if weights is None else weights.reshape(-1, bag).contiguous()
    t = table.contiguous()
    if torch.is_grad_enabled() and (table.requires_grad or (weights is not None and weights.requires_grad)):
        y = _EmbeddingLookup.apply(t, i2, w2, float(scale))
    else:
        y = ops.embedding_forward(t, i2, w2, float(scale))
    return y if len(lead) == 1 else y.view(*lead, table.shape[1])
