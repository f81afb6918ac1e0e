"""CPU: what the layer operators refuse to derive - forward-mode derivatives, before anything else is asked of the tensors -, and modules of an earlier version"""
import pytest
import torch
import torch.autograd.forward_ad as fw

from nerf_loam_amd import _lib as L
from nerf_loam_amd import layers


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
def test_linear_act_refuses_a_tangent(which, grad_mode):
    t = dict(x=torch.randn(4, 8), weight=torch.randn(3, 8), bias=torch.randn(3), residual=torch.randn(4, 3))
    with fw.dual_level(), torch.set_grad_enabled(grad_mode):
        t[which] = fw.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(L.NerfLoamHipError, match="forward-mode"):
            layers.linear_act(**t)


@pytest.mark.parametrize("which", ["table", "weights"])
def test_embedding_lookup_refuses_a_tangent(which):
    t = dict(table=torch.randn(5, 8), ids=torch.zeros(2, 3, dtype=torch.int64), weights=torch.rand(2, 3))
    with fw.dual_level():
        t[which] = fw.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(L.NerfLoamHipError, match="forward-mode"):
            layers.embedding_lookup(**t)
    with fw.dual_level(), pytest.raises(L.NerfLoamHipError, match="no CPU path"):       # a plain tensor inside a level is as ever
        layers.embedding_lookup(torch.randn(5, 8), t["ids"])


def test_a_module_pickled_before_it_had_a_choice_is_the_one_configuration():
    import io

    from nerf_loam_amd.decoder import Decoder
    old = Decoder()
    for name in ("fused", "checkpoint"):                     # the attributes of a choice that it did not have
        del old.__dict__[name]
    f = io.BytesIO()
    torch.save(old, f)
    f.seek(0)
    new = torch.load(f, weights_only=False)                  # (a file of this test's own)
    assert new.fused and new.checkpoint is None and len(new.param_list()) == 6
    with pytest.raises(L.NerfLoamHipError, match="no CPU path"):
        new(torch.zeros(2, 16))
