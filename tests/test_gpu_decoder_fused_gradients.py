"""GPU (-m gpu): a call of a decoder in the fused configuration is differentiable, against the chain in 64 bits.

The gradients are taken from the layers' fp32 products; a relu mask may differ from the 64-bit chain's where a pre-activation is within its own rounding of zero: they are compared
in the 2-norm, where one flipped unit in a million is 1e-3.  In 8 bits the weight gradients use inputs that are off by up to 2^-4 of their value."""
import pytest
import torch

from nerf_loam_amd import _lib as L
from nerf_loam_amd.decoder import Decoder
from test_gpu_decoder_layers import _chain64, _decoder

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("checkpoint", [None, "mx8"])
@pytest.mark.parametrize("x_trained,trained", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("P", [1, 2000])
def test_a_training_step_of_the_fused_configuration(checkpoint, x_trained, trained, P):
    dec = _decoder(23, checkpoint=checkpoint).requires_grad_(trained)
    x = torch.randn(P, 16, device="cuda", requires_grad=x_trained)
    with torch.no_grad():
        values = dec(x)["sdf"]
    assert not values.requires_grad
    sdf = dec(x)["sdf"]
    assert sdf.requires_grad and torch.equal(sdf, values)
    gy = torch.randn(P, 1, device="cuda")
    (sdf * gy).sum().backward()
    want, leaves = _chain64(dec, x)
    grads = torch.autograd.grad(want, leaves, gy.double())
    for i, (p, g) in enumerate(zip([x] + dec.param_list(), grads)):
        if not (x_trained if i == 0 else trained):
            assert p.grad is None
            continue
        off = float((p.grad.double() - g).norm() / g.norm())
        assert off < (2e-3 if checkpoint is None or i % 2 == 0 else 2.0 ** -4)


def test_values_stay_the_fused_kernels_and_what_is_not_provided_is_refused():
    import torch.autograd.forward_ad as fw
    dec = _decoder(29)
    x = torch.randn(300, 16, device="cuda", requires_grad=True)
    values = dec.get_values(x)
    assert not values.requires_grad and torch.equal(dec(x)["sdf"], values)                     # get_values: the values only
    with torch.no_grad():
        assert not dec(x)["sdf"].requires_grad
    assert not dec.requires_grad_(False)(x.detach())["sdf"].requires_grad
    dec.requires_grad_(True)
    for no_grad in (False, True):
        with torch.set_grad_enabled(not no_grad), fw.dual_level(), pytest.raises(L.NerfLoamHipError, match="forward-mode"):
            dec(fw.make_dual(x.detach(), x.detach()))
    # the gradient of x depends on the weights, so its own derivative is refused; hooks run once; parameters written between the passes are seen
    calls = []
    x.register_hook(lambda g: calls.append(1))
    gx, = torch.autograd.grad(dec(x)["sdf"].sum(), x, create_graph=True)
    assert gx.requires_grad and len(calls) == 1
    with pytest.raises(RuntimeError, match="not provided"):
        gx.pow(2).sum().backward()
    sdf = dec(x)["sdf"]
    with torch.no_grad():
        dec.sdf_out.weight.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace operation"):
        sdf.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_optimiser_step_between_calls_is_seen(dtype):
    """a step of a plain optimiser, then a call: the values of the new parameters, and gradients of the input's type"""
    dec = _decoder(31)
    x = torch.randn(500, 16, device="cuda").to(dtype).requires_grad_(True)
    opt = torch.optim.SGD(dec.parameters(), lr=1e-2)
    for _ in range(3):
        opt.zero_grad()
        x.grad = None
        sdf = dec(x)["sdf"]
        want, leaves = _chain64(dec, x)
        assert float((sdf.detach().double() - want).abs().max()) < 1e-4
        sdf.square().mean().backward()
        grads = torch.autograd.grad(want, leaves, 2 * want.detach() / want.numel())
        assert x.grad.dtype == dtype and float((x.grad.double() - grads[0]).norm() / grads[0].norm()) < (2e-3 if dtype == torch.float32 else 2.0 ** -8)
        opt.step()


def test_a_module_on_the_host_and_a_second_stream():
    """the fused kernel takes a module's parameters from wherever they are: the gradients go back there; passes on another stream than the input's give the same bits"""
    host = Decoder()
    dec = Decoder().cuda()
    dec.load_state_dict(host.state_dict())
    x = torch.randn(700, 16, device="cuda")
    for d in (host, dec):
        d(x)["sdf"].square().sum().backward()
    assert all(a.grad.device.type == "cpu" and torch.equal(a.grad, b.grad.cpu()) for a, b in zip(host.param_list(), dec.param_list()))
    want = [p.grad.clone() for p in dec.param_list()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        dec.zero_grad()
        dec(x)["sdf"].square().sum().backward()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, p.grad) for a, p in zip(want, dec.param_list()))
