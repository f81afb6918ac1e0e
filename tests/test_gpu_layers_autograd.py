"""GPU (-m gpu): what autograd may and may not ask of the layer operators - a gradient that depends on a tensor somebody differentiates by is never handed out as a constant."""
import itertools

import pytest
import torch

from nerf_loam_amd import _lib as L
from nerf_loam_amd import layers

pytestmark = pytest.mark.gpu


def _linear_inputs(dtype, trained, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shapes = dict(x=(40, 24), w=(16, 24), b=(16,), r=(40, 16))
    return {n: torch.randn(*s, generator=g, device="cuda").mul(0.3).to(dtype).requires_grad_(n in trained) for n, s in shapes.items()}


def _depends(name, act, trained, gy):
    """whether the formula of a gradient holds a tensor that is differentiated by: gx = (gy act'(z)) w, gw = (gy act'(z))^T x, gb = sum of gy act'(z), gr = gy, z = x w^T + b;
    act' is constant almost everywhere for none and relu"""
    z = act in ("gelu", "silu") and name != "r" and bool(trained & {"x", "w", "b"})
    return gy or z or (name == "x" and "w" in trained) or (name == "w" and "x" in trained)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("checkpoint", [None, "mx8"])
def test_a_linear_gradient_that_depends_on_a_trained_tensor_is_no_constant(act, checkpoint):
    """every subset of trained tensors, with and without a trained gradient of the output: what depends raises when it is differentiated, what does not stays a constant
    that a loss may contain"""
    names = ("x", "w", "b", "r")
    for dtype in (torch.float32, torch.bfloat16):
        for trained in (set(c) for n in range(1, 5) for c in itertools.combinations(names, n)):
            for gy_trained in (False, True):
                t = _linear_inputs(dtype, trained)
                gy = torch.ones(40, 16, dtype=dtype, device="cuda", requires_grad=gy_trained)
                y = layers.linear_act(t["x"], t["w"], t["b"], act=act, residual=t["r"], checkpoint=checkpoint)
                order = [n for n in names if n in trained]
                for n, g in zip(order, torch.autograd.grad(y, [t[n] for n in order], gy, create_graph=True)):
                    want = _depends(n, act, trained, gy_trained)
                    assert g.requires_grad == want, (act, checkpoint, sorted(trained), gy_trained, n)
                    if want and n != "r":
                        with pytest.raises(RuntimeError, match="not provided"):
                            g.float().pow(2).sum().backward(retain_graph=True)


def test_a_penalty_on_the_gradient_is_not_lost():
    """a frozen layer, a trained input: the penalty's derivative goes through act'(z)"""
    for act in ("gelu", "silu"):
        t = _linear_inputs(torch.float32, {"x"})
        y = layers.linear_act(t["x"], t["w"], t["b"], act=act)
        g, = torch.autograd.grad(y.sum(), t["x"], create_graph=True)
        with pytest.raises(RuntimeError, match="not provided"):
            (y.sum() + g.pow(2).sum()).backward()
    # the same loss where the gradient is a constant trains as ever
    t = _linear_inputs(torch.float32, {"x"})
    y = layers.linear_act(t["x"], t["w"], t["b"], act="none")
    g, = torch.autograd.grad(y.sum(), t["x"], create_graph=True)
    (y.sum() + g.pow(2).sum()).backward()
    assert torch.equal(t["x"].grad, g)


def test_an_embedding_gradient_that_depends_on_a_trained_tensor_is_no_constant():
    """g_table = sums of w g, g_weights = <g, table>"""
    for trained in ({"t"}, {"w"}, {"t", "w"}):
        for g_trained in (False, True):
            table = torch.randn(30, 8, device="cuda").requires_grad_("t" in trained)
            wt = torch.rand(20, 4, device="cuda").requires_grad_("w" in trained)
            ids = torch.randint(-1, 30, (20, 4), device="cuda")
            g = torch.ones(20, 8, device="cuda", requires_grad=g_trained)
            order = [n for n in ("t", "w") if n in trained]
            grads = torch.autograd.grad(layers.embedding_lookup(table, ids, weights=wt), [{"t": table, "w": wt}[n] for n in order], g, create_graph=True)
            for n, v in zip(order, grads):
                want = g_trained or ("w" if n == "t" else "t") in trained
                assert v.requires_grad == want, (sorted(trained), g_trained, n)
                if want:
                    with pytest.raises(RuntimeError, match="not provided"):
                        v.pow(2).sum().backward(retain_graph=True)
    # no weights: the table's gradient depends on the output's alone
    table = torch.randn(30, 8, device="cuda", requires_grad=True)
    y = layers.embedding_lookup(table, torch.randint(0, 30, (20,), device="cuda"))
    assert not torch.autograd.grad(y.sum(), table, create_graph=True)[0].requires_grad


def test_tangents_and_function_transforms_are_refused():
    """on the device as on the host (tests/test_layers_autograd_host.py); a transform's tensors have no memory to read"""
    import torch.autograd.forward_ad as fw
    x, w, table = torch.randn(6, 8, device="cuda"), torch.randn(4, 8, device="cuda"), torch.randn(9, 8, device="cuda")
    ids = torch.zeros(6, dtype=torch.int64, device="cuda")
    for quiet in (False, True):
        with fw.dual_level(), torch.set_grad_enabled(not quiet):
            for a in ((fw.make_dual(x, x), w), (x, fw.make_dual(w, w)), (fw.make_dual(x.requires_grad_(not quiet), x.detach()), w)):
                with pytest.raises(L.NerfLoamHipError, match="forward-mode"):
                    layers.linear_act(*a)
            with pytest.raises(L.NerfLoamHipError, match="forward-mode"):
                layers.embedding_lookup(fw.make_dual(table, table), ids)
    x = x.detach()
    for call in (lambda: torch.func.grad(lambda t: layers.linear_act(t, w).sum())(x), lambda: torch.func.jvp(lambda t: layers.linear_act(t, w), (x,), (x,)),
                 lambda: torch.func.vmap(lambda t: layers.linear_act(t, w))(x[None]), lambda: torch.func.grad(lambda t: layers.embedding_lookup(t, ids).sum())(table)):
        with pytest.raises(RuntimeError):
            call()
    assert torch.equal(layers.linear_act(x, w), layers.linear_act(x, w))


@pytest.mark.parametrize("bag", [1, 4])
def test_a_table_may_change_before_its_gradient_is_taken(bag):
    """the table's gradient does not hold its values: an update in place between the passes changes nothing, unless the weights' gradient needs them"""
    table = torch.randn(50, 12, device="cuda", requires_grad=True)
    ids = torch.randint(-1, 50, (30, bag) if bag > 1 else (30,), device="cuda")
    wt = torch.rand(30, bag, device="cuda") if bag > 1 else None
    g = torch.randn(30, 12, device="cuda")
    want, = torch.autograd.grad(layers.embedding_lookup(table, ids, weights=wt), table, g)
    y = layers.embedding_lookup(table, ids, weights=wt)
    with torch.no_grad():
        table.mul_(2.0)
    assert torch.equal(torch.autograd.grad(y, table, g)[0], want)
    if bag > 1:
        wt.requires_grad_(True)
        y = layers.embedding_lookup(table, ids, weights=wt)
        with torch.no_grad():
            table.mul_(2.0)
        with pytest.raises(RuntimeError, match="inplace operation"):
            torch.autograd.grad(y, [table, wt], g)
        # the weights' own values count in the table's gradient alone
        y = layers.embedding_lookup(table.detach(), ids, weights=wt)
        want, = torch.autograd.grad(y, wt, g, retain_graph=True)
        with torch.no_grad():
            wt.add_(1.0)
        assert torch.equal(torch.autograd.grad(y, wt, g)[0], want)


@pytest.mark.parametrize("checkpoint", [None, "mx8"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
def test_a_weight_may_change_where_the_gradients_do_not_hold_it(act, checkpoint):
    """gw = dz^T x and gb = sum of dz do not hold w; gx = dz w does"""
    x, w, b = torch.randn(33, 20, device="cuda"), torch.randn(9, 20, device="cuda", requires_grad=True), torch.randn(9, device="cuda", requires_grad=True)
    gy = torch.randn(33, 9, device="cuda")
    want = torch.autograd.grad(layers.linear_act(x, w, b, act=act, checkpoint=checkpoint), [w, b], gy)
    y = layers.linear_act(x, w, b, act=act, checkpoint=checkpoint)
    with torch.no_grad():
        w.mul_(3.0)
        b.add_(1.0)
    got = torch.autograd.grad(y, [w, b], gy)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    x.requires_grad_(True)
    y = layers.linear_act(x, w, b, act=act, checkpoint=checkpoint)
    with torch.no_grad():
        w.mul_(3.0)
    with pytest.raises(RuntimeError, match="inplace operation"):
        torch.autograd.grad(y, [x, w, b], gy)
