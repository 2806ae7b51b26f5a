"""The layer operators where something follows torch's operations from outside: traces, forward-mode and second derivatives.  Here with
the launch left out (what is recorded does not depend on it); on the GPU the traced calls are run on other inputs."""
import pytest
import torch
from torch.autograd import forward_ad


def _calls():
    from nerf_amd import ops
    w, b = torch.randn(5, 8), torch.randn(5)
    g = torch.randn(8)
    return [("layer_norm", lambda v: ops.layer_norm(v)), ("layer_norm", lambda v: ops.layer_norm(v, g, g)),
            ("linear_fp8", lambda v: ops.linear_fp8(v, w, b)), ("linear_fp8", lambda v: ops.linear_fp8(v, w, None, True))]


@pytest.fixture
def launches(monkeypatch):
    from nerf_amd import ops
    seen = []
    monkeypatch.setattr(ops, "_launch", lambda dev, name, units, fn, *args: seen.append(name))
    monkeypatch.setattr(ops, "_elem", lambda t, what: ops.ELEM_TYPES[t.dtype])
    return seen


@pytest.mark.parametrize("i", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_a_trace_holds_the_call(launches, i, grad):
    name, f = _calls()[i]
    x = torch.randn(3, 8)
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(f, (x,), check_trace=False)
    kinds = [n.kind() for n in traced.graph.nodes()]
    assert "prim::PythonOp" in kinds and not any(k.startswith("aten::empty") for k in kinds), kinds
    launches.clear()
    assert traced(torch.randn(3, 8)).shape == f(x).shape and launches == [name, name]


@pytest.mark.parametrize("i", range(4))
def test_a_tangent_is_not_dropped(launches, i):
    _, f = _calls()[i]
    x = torch.randn(3, 8)
    with forward_ad.dual_level():
        f(x)                                     # nothing to differentiate
        with pytest.raises(RuntimeError, match="forward mode AD"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode AD"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("i", range(4))
def test_a_second_derivative_is_refused(launches, i):
    _, f = _calls()[i]
    x = torch.randn(3, 8, requires_grad=True)
    dy = torch.randn_like(f(x)).requires_grad_(True)
    for incoming in (dy, dy.detach()):           # (the first gradient depends on x either way)
        (dx,) = torch.autograd.grad(f(x), x, incoming, create_graph=True)
        assert dx.shape == x.shape
        with pytest.raises(RuntimeError, match="differentiable once"):
            (f(x).sum() + (dx ** 2).sum()).backward()
    (dx,) = torch.autograd.grad(f(x), x, dy)
    assert not dx.requires_grad


def test_a_graph_of_torch_operations_is_refused(monkeypatch):
    from torch.fx.experimental.proxy_tensor import make_fx
    from nerf_amd import ops
    monkeypatch.setattr(ops, "_elem", lambda t, what: ops.ELEM_TYPES[t.dtype])
    for _, f in _calls():
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            make_fx(f)(torch.randn(3, 8))


@pytest.mark.gpu
def test_traced_calls_on_other_inputs(device):
    """With weights of either kind, and every step of a product in 8 bits: the trace computes what the call does."""
    from nerf_amd import ops
    w, b, g = torch.randn(24, 200, device=device), torch.randn(24, device=device), torch.randn(200, device=device)
    held = ops.quantize_fp8(w)
    for f in (lambda v: ops.layer_norm(v, g), lambda v: ops.linear_fp8(v, w, b, True), lambda v: ops.linear_fp8(v, held, b),
              lambda v: ops.quantize_fp8(v).codes.float(), lambda v: ops.matmul_fp8(ops.quantize_fp8(v), held, b, True, torch.float32)):
        with torch.no_grad():
            traced = torch.jit.trace(f, (torch.randn(30, 200, device=device),), check_trace=False)
            for rows in (30, 30, 17, 300):
                x = torch.randn(rows, 200, device=device)
                keep = [torch.full((rows, 200), float("nan"), device=device) for _ in range(4)]      # (memory that held no earlier result)
                del keep
                assert torch.equal(traced(x), f(x))


@pytest.mark.gpu
def test_tangents_are_refused_by_every_call(device):
    """(but quantize_fp8, whose codes are no part of x's graph in any mode)"""
    from nerf_amd import ops
    x, b = torch.randn(30, 200, device=device), torch.randn(24, device=device)
    held = ops.quantize_fp8(torch.randn(24, 200, device=device))
    q = ops.quantize_fp8(x)
    with forward_ad.dual_level():
        dx, db = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(b, torch.ones_like(b))
        for f in (lambda: ops.layer_norm(dx), lambda: ops.linear_fp8(dx, held), lambda: ops.linear_fp8(x, held, db),
                  lambda: ops.matmul_fp8(q, held, db)):
            with pytest.raises(RuntimeError, match="forward mode AD"):
                f()
        assert ops.matmul_fp8(q, held, b).shape == (30, 24)
