"""States of optim.AdamW in 8 bits for gradients so small that a block's scale comes near fp32's smallest values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

B1, B2 = 0.9, 0.99


@pytest.mark.parametrize("size", [1e-12, 1e-15, 1e-16, 1e-17, 1e-18, 1e-20])
def test_the_second_moment_of_small_gradients(device, size):
    """Each step's states are the rule's applied to the states before it, rounded to a neighbour: off by less than a grid step, 2^-3
    (m) and 2^-2 (v) of the value or 2^-9 and 2^-16 of the scale, whichever is larger, and 8 fp32 roundings.  A scale is the
    largest value over 448 and 57344, or 1e-38 where that is less."""
    from nerf_amd.optim import AdamW
    gen = torch.Generator(device=device)
    gen.manual_seed(3)
    p = torch.nn.Parameter(torch.randn(1000, device=device, generator=gen))
    opt = AdamW([p], lr=1e-3, betas=(B1, B2), weight_decay=0.0, state_bits=8)
    m, v = (torch.zeros(1000, device=device, dtype=torch.float64) for _ in range(2))
    for _ in range(4):
        p.grad = size * torch.randn(1000, device=device, generator=gen)
        p.grad[130:200] = 0.0
        g = p.grad.double()
        m, v = m + (1 - B1) * (g - m), v + (1 - B2) * (g * g - v)
        opt.step()
        st = opt.state[p]
        for want, key, col, top, least, bits in ((m, "exp_avg", 0, 448, 2.0 ** -9, 3), (v, "exp_avg_sq", 1, 57344, 2.0 ** -16, 2)):
            scale = st["scale"][:, col].double()
            largest = torch.nn.functional.pad(want.abs(), (0, 24)).view(-1, 128).amax(1)
            assert bool(((scale - (largest / top).clamp_min(1e-38)).abs() <= 2.0 ** -21 * scale).all())
            wide = scale.repeat_interleave(128)[:1000]
            got = st[key].float().double() * wide
            tol = torch.maximum(want.abs() * 2.0 ** -bits, least * wide) + 2.0 ** -21 * want.abs() + 2.0 ** -149
            assert bool(((got - want).abs() <= tol).all()), (key, float(((got - want).abs() / tol).max()))
            # (below 2^-149 fp32 has no value: a square of less, or its hundredth, rounds to 0 before it is a state)
            assert key == "exp_avg" or bool((got[want > 2.0 ** -148] > 0).all())
        m, v = (st[k].float() * st["scale"][:, c].repeat_interleave(128)[:1000] for k, c in (("exp_avg", 0), ("exp_avg_sq", 1)))
        m, v = m.double(), v.double()


def test_blocks_of_zeros_keep_no_scale(device):
    from nerf_amd.optim import AdamW
    p = torch.nn.Parameter(torch.randn(300, device=device))
    p.grad = torch.zeros_like(p)
    p.grad[:128] = 1.0
    opt = AdamW([p], state_bits=8)
    opt.step()
    scale = opt.state[p]["scale"]
    assert bool((scale[0] > 0).all()) and not scale[1:].any()
