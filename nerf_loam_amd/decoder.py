"""Decoder: the SDF MLP container.

Mirror of /root/reference/src/variations/lidar.py:80-131; parameter names match (`pts_linears.{i}`, `sdf_out`), so reference checkpoints / state_dicts load.

* The configuration every shipped config uses (depth 2, width 256, in_dim 16, skips [], embedder none => Linear(16,256)-ReLU-Linear(256,256)-ReLU-Linear(256,1)) runs
  the fused matrix-core forward kernel (nl_decoder.hip k_decoder_fwd); the optimisation loops train it inside the engine.  A call of the module is differentiable: it
  keeps its input alone, and its backward pass runs the layers again (with checkpoint="mx8" on activations kept in 8 bits).  get_values gives the values only.
* Every other depth / width / in_dim / skips runs one layers.linear_act call per layer (csrc/nl_linear.hip) and is differentiable with respect to its input and its
  parameters; checkpoint="mx8" keeps the activations of a training step in 8 bits (layers.linear_act).  bundle_adjust_frames / track_frame / render_rays do not take
  such a decoder; get_scores and create_mesh do.

There is no PyTorch GEMM path.  The positional embedders (lidar.py:6-77, used by no config) are not provided and raise."""
import torch
import torch.nn as nn
from torch.autograd.forward_ad import unpack_dual

from . import _lib as L
from . import layers, ops


class _FusedValues(torch.autograd.Function):
    """the fused kernel's values; the backward pass takes its gradients from layer calls on the same input and parameters"""

    @staticmethod
    def forward(ctx, dec, x, *params):
        out = dec._values_fused(x)
        ctx.dec = dec
        ctx.save_for_backward(x, *params)
        return out

    @staticmethod
    def backward(ctx, g):
        again = torch.is_grad_enabled()                                                     # create_graph: the layers say which gradients depend on what
        with torch.enable_grad():
            t = [v.view_as(v) if again else v.detach().requires_grad_(need) for v, need in zip(ctx.saved_tensors, ctx.needs_input_grad[1:])]
            y = ctx.dec._values_layers(t[0].float(), [v.to(g.device, torch.float32) for v in t[1:]])            # the kernel's type, and its device where the module is elsewhere
            wanted = [v for v, need in zip(t, ctx.needs_input_grad[1:]) if need]
            grads = iter(torch.autograd.grad(y, wanted, g, create_graph=again))
        return (None, *(next(grads) if need else None for need in ctx.needs_input_grad[1:]))


class Decoder(nn.Module):
    fused, checkpoint = True, None              # of a module that was pickled whole when there was one configuration

    def __init__(self, depth=2, width=256, in_dim=16, sdf_dim=128, skips=(), multires=0, embedder="none", point_dim=3,
                 local_coord=False, checkpoint=None, **kwargs):
        super().__init__()
        if embedder != "none":
            raise NotImplementedError("the MI355X decoder takes its input as it is: embedder none (the reference's positional embedders are used by no shipped configuration)")
        if depth < 1 or width < 1 or in_dim < 1 or any(s not in range(depth - 1) for s in skips):
            raise ValueError(f"Decoder: depth {depth}, width {width} and in_dim {in_dim} must be positive, skips {list(skips)} name layers below the last one")
        if checkpoint not in layers.CHECKPOINTS:
            raise ValueError(f"Decoder: checkpoint {checkpoint!r} must be one of {layers.CHECKPOINTS}")
        self.D, self.W, self.skips, self.point_dim, self.checkpoint = depth, width, list(skips), point_dim, checkpoint
        self.fused = (depth, width, in_dim, len(skips)) == (2, L.NL_W, L.NL_C, 0)           # the engine's kernels are built for this one
        # lidar.py:96-106: the layer behind a skip takes the input again, in front of the hidden values
        self.pts_linears = nn.ModuleList([nn.Linear(in_dim, width)] + [nn.Linear(width + in_dim if i in self.skips else width, width) for i in range(depth - 1)])
        self.sdf_out = nn.Linear(width, 1)

    def param_list(self):
        return [p for l in (*self.pts_linears, self.sdf_out) for p in (l.weight, l.bias)]

    def flat_params(self, device):
        """decoder parameter block of include/nerfloam_hip.h (W1 b1 W2 b2 W3 b3)"""
        return torch.cat([p.detach().reshape(-1).float() for p in self.param_list()]).to(device).contiguous()

    @torch.no_grad()
    def load_flat(self, flat):
        off = 0
        for p in self.param_list():
            n = p.numel()
            p.copy_(flat[off:off + n].view_as(p))
            off += n

    def get_values(self, x):
        """sdf of points; of the fused configuration the values only, no gradient (forward has one)"""
        if not x.is_cuda:
            raise L.NerfLoamHipError("Decoder.get_values needs a CUDA (HIP) tensor - no CPU path")
        return self._values_fused(x) if self.fused else self._values_layers(x, self.param_list())

    @torch.no_grad()
    def _values_fused(self, x):
        x = x.detach().float().contiguous()
        # the device parameter block + W2 operand planes, kept until somebody writes the parameters (tensor version counters): the same
        # cache bundle_adjust_frames / track_frame use (render_helpers._decoder_device) - no re-flattening, no plane rebuild per call
        from .render_helpers import _decoder_device
        dec = _decoder_device(self, x.device)
        out = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
        ops.decoder_forward(x, dec.params, dec.W2T, x.shape[0], out, L.lib().nl_decoder_grid_hint())
        return out.unsqueeze(-1)

    def _values_layers(self, x, params):
        """lidar.py:109-123, a call per layer; in the parameters' type"""
        x = x.to(params[-2].dtype)
        h = x
        for i in range(self.D):
            h = layers.linear_act(h, params[2 * i], params[2 * i + 1], act="relu", checkpoint=self.checkpoint)
            if i in self.skips:
                h = torch.cat([x, h], -1)
        return layers.linear_act(h, params[-2], params[-1], checkpoint=self.checkpoint)

    def forward(self, inputs):
        if self.fused and inputs.is_cuda:
            params = self.param_list()
            if any(unpack_dual(t).tangent is not None for t in (inputs, *params)):
                raise L.NerfLoamHipError("Decoder: forward-mode derivatives are not provided")
            if torch.is_grad_enabled() and any(t.requires_grad for t in (inputs, *params)):
                return {"sdf": _FusedValues.apply(self, inputs, *params)}
        return {"sdf": self.get_values(inputs)}
