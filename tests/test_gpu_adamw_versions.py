"""The parameters that optim.AdamW writes count as written: autograd's version counters move with every step, as torch's own optimisers
move them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.bfloat16, 8)])
def test_a_graph_from_before_the_step_is_refused(device, dtype, bits):
    """A backward pass behind the step would mix the old activations with the new weights."""
    from nerf_amd.optim import AdamW
    p, idle = (torch.nn.Parameter(torch.randn(40, device=device).to(dtype)) for _ in range(2))
    opt = AdamW([p, idle], lr=0.1, state_bits=bits)
    x = torch.randn(40, device=device).to(dtype).requires_grad_(True)
    for i in range(3):
        y, z = (p * x).sum(), (idle * x).sum()
        p.grad = torch.ones_like(p)
        v = p._version, idle._version
        opt.step()
        assert p._version > v[0] and idle._version == v[1]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        z.backward()                 # (saved nothing that was written)
        idle.grad = None


def test_the_frameworks_own_layer(device):
    from nerf_amd import ops
    from nerf_amd.optim import AdamW
    w = torch.nn.Parameter(torch.randn(24, 40, device=device))
    x = torch.randn(10, 40, device=device, requires_grad=True)
    y = ops.linear(x, w, None)
    w.grad = torch.ones_like(w)
    AdamW([w], lr=0.1).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    held = ops.linear_fp8(x, w)      # keeps the weight's codes, so its gradients stay those of the weight it used
    want = torch.autograd.grad(ops.linear_fp8(x, w), x, torch.ones_like(y))[0]
    opt = AdamW([w], lr=0.1)
    opt.step()
    assert torch.equal(torch.autograd.grad(held, x, torch.ones_like(y))[0], want)
