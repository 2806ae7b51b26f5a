"""Checkpoints that pass from one optimiser to another: the rule goes with them, or they are refused."""
import copy

import pytest
import torch

LR, BETAS, EPS, WD = 3e-3, (0.9, 0.99), 1e-8, 0.3


def _flat(params, **kw):
    from nerf_amd.optim import FlatAdam
    return FlatAdam(params, lr=1.0, **kw)


def test_eight_bit_states_are_not_taken_for_plain_ones():
    """Their codes without their scales would be moments of another size."""
    p = torch.nn.Parameter(torch.zeros(200))
    ckpt = {"state": {0: {"step": torch.tensor(3.0), "exp_avg": torch.zeros(200, dtype=torch.uint8).view(torch.float8_e4m3fn),
                          "exp_avg_sq": torch.zeros(200, dtype=torch.uint8).view(torch.float8_e5m2), "scale": torch.ones(2, 2)}},
            "param_groups": [dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, capturable=True, params=[0])]}
    opt = _flat([p])
    with pytest.raises(ValueError, match="8 bits"):
        opt.load_state_dict(ckpt)
    assert not opt.state and opt.param_groups[0]["lr"] == 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("decay", [0.0, WD])
@pytest.mark.parametrize("to", ["FlatAdam", "torch.Adam", "torch.AdamW", "AdamW"])
def test_a_run_goes_on_with_its_rule(device, to, decay):
    """AdamW in 32 bits -> the others, and on: each step moves p by -lr wd p - lr mhat / (sqrt(vhat) + eps), the decay outside the
    moments (16 fp32 roundings of the move, 2 of p)."""
    from nerf_amd.optim import AdamW
    gen = torch.Generator(device=device)
    gen.manual_seed(1)
    flat = torch.randn(3000, device=device, generator=gen)
    params = [torch.nn.Parameter(flat[:1000]), torch.nn.Parameter(flat[1000:])]
    grads = torch.empty(3000, device=device)

    def new_grads():
        grads.copy_(torch.randn(3000, device=device, generator=gen) * 0.01)
        params[0].grad, params[1].grad = grads[:1000], grads[1000:]
    opt = AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=decay)
    for _ in range(2):
        new_grads()
        opt.step()
    make = {"FlatAdam": _flat, "torch.Adam": torch.optim.Adam, "torch.AdamW": torch.optim.AdamW, "AdamW": AdamW}[to]
    new = make(params)
    new.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert new.param_groups[0]["lr"] == LR
    m, v = (torch.cat([opt.state[p][k] for p in params]).double() for k in ("exp_avg", "exp_avg_sq"))
    for t in (3, 4):
        new_grads()
        before, g = flat.double(), grads.double()
        m, v = BETAS[0] * m + (1 - BETAS[0]) * g, BETAS[1] * v + (1 - BETAS[1]) * g * g
        move = LR * decay * before + LR * (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)).sqrt() + EPS)
        new.step()
        scale = LR * decay * before.abs() + LR / (1 - BETAS[0] ** t) * (m.abs() + g.abs()) / ((v / (1 - BETAS[1] ** t)).sqrt() + EPS)
        assert bool(((flat.double() - (before - move)).abs() <= 2.0 ** -24 * (16 * t * scale + 2 * before.abs())).all()), t
    if to == "FlatAdam":
        assert new.fast_steps == (0 if decay else 2)
