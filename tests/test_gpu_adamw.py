"""optim.AdamW against the update rule in 64 bits: states in 32 and in 8 bits, parameters of three types, tensors anywhere.

One step is compared with the rule applied to the values the states hold before it (u = 2^-24, half an fp32 step):
  m      two roundings: 4 u (|m| + |g|);  v: 5 u (v + g^2)
  p      the move is off by at most 10 roundings and what m and v carry, the sum by one: 16 u |move| + 2 u |p|, and for 16-bit
         parameters half a step of their type
8-bit states are checked code by code: the rounded value is a neighbour of the exact one, and it is the one the element's random
bits name wherever the exact remainder is not within 2^-15 of the decision.
"""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.99, 1e-8, 0.05


def _opt(params, **kw):
    from nerf_amd.optim import AdamW
    return AdamW(params, **{**dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD), **kw})


def _params(shapes, dtype, device, seed, shift=0):
    """Parameters with gradients; shift: their storage starts that many elements behind an aligned address."""
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    out = []
    for s in shapes:
        n = torch.Size(s).numel()

        def make(scale):
            buf = torch.full((n + shift + 8,), float("nan"), device=device, dtype=dtype)
            buf[shift:shift + n] = (torch.randn(n, device=device, generator=gen) * scale).to(dtype)
            return buf[shift:shift + n].view(s)
        p = torch.nn.Parameter(make(0.1))
        p.grad = make(1e-2)
        out.append(p)
    return out


def _new_grads(params, seed):
    gen = torch.Generator(device=params[0].device)
    gen.manual_seed(seed)
    for p in params:
        p.grad.copy_(torch.randn(p.shape, device=p.device, generator=gen) * 10.0 ** (-1 - seed % 4))


def _noise(n, t):
    i = torch.arange(n, dtype=torch.int64)
    low = 0xFFFFFFFF
    h = (i * 0x9E3779B1 + t * 0x85EBCA77) & low
    h = h ^ (h >> 16)
    h = (h * 0x7FEB352D) & low
    h = h ^ (h >> 15)
    h = (h * 0x846CA68B) & low
    return h ^ (h >> 16)


def _held(opt, p):
    """(m, v, p) as the states hold them, fp64 on the CPU, flat."""
    st = opt.state[p]
    m, v = [st[k].detach().cpu().float().double().reshape(-1) for k in ("exp_avg", "exp_avg_sq")]
    if "scale" in st:
        s = st["scale"].cpu().repeat_interleave(128, 0)[: m.numel()]
        m, v = (m.float() * s[:, 0]).double(), (v.float() * s[:, 1]).double()
    src = st["master"] if "master" in st else p
    return m, v, src.detach().cpu().double().reshape(-1)


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % 128)).view(-1, 128)


def _check_codes(u, err, got, rnd, bits, least, floored=None):
    """got (fp64 codes' values) against stochastic rounding of u (known to +-err) on a grid of `bits` mantissa bits, rnd in [0, 1).
    floored: where what would become 0 becomes the smallest code."""
    step = torch.ldexp(torch.ones_like(u), torch.frexp(u.clamp_min(2.0 ** -30))[1].clamp_min(least + bits + 1) - 1 - bits)
    low = torch.floor(u / step)
    rest, margin = u / step - low, 2.0 ** -15 + err / step
    clear = (rest + rnd - 1).abs() > margin
    clear &= (rest > margin) & (rest < 1 - margin)
    want = (low + (rest + rnd >= 1)) * step
    if floored is not None:
        want = torch.where(floored, want.clamp_min(2.0 ** least), want)
    assert bool((got[clear] == want[clear]).all()), (u[clear][got[clear] != want[clear]][:3], got[clear][got[clear] != want[clear]][:3])
    assert bool(((got >= (u - err) - step * 1.001) & (got <= (u + err) + step * 1.001)).all())
    return float(clear.double().mean())


def _step_and_check(opt, params, t, lr=LR, wd=WD):
    before = [(_held(opt, p) if opt.state.get(p) else (torch.zeros(p.numel(), dtype=torch.float64),) * 2 + (p.detach().cpu().double().reshape(-1),))
              for p in params]
    grads = [p.grad.detach().cpu().double().reshape(-1).clone() for p in params]
    opt.step()
    torch.cuda.synchronize()
    for p, g, (m0, v0, p0) in zip(params, grads, before):
        st = opt.state[p]
        assert float(st["step"]) == t
        m, v = m0 + (1 - B1) * (g - m0), v0 + (1 - B2) * (g * g - v0)
        move = lr * wd * p0 + lr / (1 - B1 ** t) * m / (torch.sqrt(v / (1 - B2 ** t)) + EPS)
        want = p0 - move
        gm, gv, gp = _held(opt, p)
        scale = lr * wd * p0.abs() + lr / (1 - B1 ** t) * (m0.abs() + g.abs()) / (torch.sqrt(v / (1 - B2 ** t)) + EPS)
        tol = 16 * U * scale + 2 * U * p0.abs() + 2.0 ** -149
        assert bool(((gp - want).abs() <= tol).all()), float(((gp - want).abs() / tol).max())
        if p.dtype != torch.float32:
            assert torch.equal(p.detach(), st["master"].to(p.dtype))
        if opt.state_bits == 32:
            assert bool(((gm - m).abs() <= 4 * U * (m0.abs() + g.abs()) + 2.0 ** -149).all())
            assert bool(((gv - v).abs() <= 5 * U * (v0 + g * g) + 2.0 ** -149).all())
            continue
        if not m.numel():
            continue
        # (a largest value is as exact as the values, whose bounds these are, and the division's rounding)
        em, ev = 4 * U * (m0.abs() + g.abs()), 5 * U * (v0 + g * g)
        sm, sv = _blocks(m).abs().amax(1) / 448, _blocks(v).amax(1) / 57344
        got = st["scale"].cpu().double()
        assert bool(((got[:, 0] - sm).abs() <= _blocks(em).amax(1) / 448 + 2 * U * sm + 2.0 ** -148).all())
        assert bool(((got[:, 1] - sv).abs() <= _blocks(ev).amax(1) / 57344 + 2 * U * sv + 2.0 ** -148).all())
        h = _noise(m.numel(), t)
        wide = got.repeat_interleave(128, 0)[: m.numel()].clamp_min(1e-38)
        cm, cv = st["exp_avg"].cpu().float().double().reshape(-1), st["exp_avg_sq"].cpu().float().double().reshape(-1)
        um, uv = (m.abs() / wide[:, 0]).clamp_max(448), (v / wide[:, 1]).clamp_max(57344)
        em, ev = em / wide[:, 0] + 4 * U * um, ev / wide[:, 1] + 4 * U * uv
        a = _check_codes(um, em, cm.abs(), (h & 0xFFFF).double() / 65536, 3, -9)
        b = _check_codes(uv, ev, cv, (h >> 16).double() / 65536, 2, -16, v > 0)
        # in the first step all but the largest of a block lie anywhere between grid points (later ones, when the
        # gradients are far smaller than those before, may leave values on the grid, where the decision is not tested)
        assert t > 1 or min(a, b) > 0.95 or m.numel() < 200, (a, b)
        assert bool(((cm == 0) | (torch.sign(cm) == torch.sign(m)) | (um <= em)).all()) and bool((cv[v > 0] > 0).all()) and bool((cv >= 0).all())


SHAPES = [(1,), (3,), (7, 1), (127,), (128,), (129,), (256, 90), (0,), (64, 64), (2047,), (2048,), (2049,), (33, 77), (5, 0, 3), (100003,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_steps_follow_the_rule(device, dtype, bits, shift):
    params = _params(SHAPES, dtype, device, 1, shift)
    opt = _opt(params, state_bits=bits)
    for t in range(1, 6):
        _new_grads(params, t)
        _step_and_check(opt, params, t)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_launch_takes(device, bits):
    shapes = [((37 * i) % 300 + 1,) for i in range(150)] + [(0,)] * 3 + [(5000,)]
    params = _params(shapes, torch.float32, device, 2)
    opt = _opt(params, state_bits=bits)
    for t in (1, 2):
        _new_grads(params, t)
        _step_and_check(opt, params, t)


def test_states_in_32_bits_follow_torch(device):
    """Twenty steps beside torch.optim.AdamW in 64 bits on the same gradients, parameters that join later included."""
    params = _params([(300, 7), (41,), (1000,)], torch.float32, device, 3)
    other = [torch.nn.Parameter(p.detach().cpu().double()) for p in params]
    opt = _opt(params)
    ref = torch.optim.AdamW(other, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    for t in range(20):
        _new_grads(params, t)
        for p, q in zip(params, other):
            q.grad = p.grad.detach().cpu().double()
        late = params[1].grad
        if t < 5:
            params[1].grad = other[1].grad = None
        opt.step()
        ref.step()
        params[1].grad = late
    assert float(opt.state[params[1]]["step"]) == 15.0 and float(opt.state[params[0]]["step"]) == 20.0
    for p, q in zip(params, other):
        # per step: 16 u of a move of at most lr / (1 - b1) (and the decay), and 2 u of the parameter
        tol = 20 * (16 * U * LR * 10 * 2 + 2 * U * float(q.detach().abs().max()))
        assert float((p.detach().cpu().double() - q.detach()).abs().max()) <= tol


def test_eight_bit_states_keep_their_mean(device):
    """Second moments far from where constant gradients take them move there at the rule's rate, though one step is far below a
    grid step: over 20000 elements the mean of v follows the exact recursion (the standard deviation of one element is below
    half its value, so that of the mean is below 0.4 %; five of them and the 1 % that the top of each block adds)."""
    n = 20096
    for start, end in ((1.0, 0.1), (0.01, 0.1)):
        p = torch.nn.Parameter(torch.zeros(n, device=device))
        opt = _opt([p], state_bits=8, lr=0.0, weight_decay=0.0)
        p.grad = torch.full((n,), start, device=device)
        opt.step()
        st = opt.state[p]
        st["scale"][:, 1] *= 1.0 / (1 - B2)      # v = start^2
        p.grad.fill_(end)
        p.grad[::128] = 2.0                      # one large element per block keeps the scale away from the others
        st["exp_avg_sq"].view(-1, 128)[:, 0] = torch.tensor(57344.0, device=device).to(torch.float8_e5m2)
        st["scale"][:, 1] = 4.0 / 57344
        rest = torch.ones(n, dtype=torch.bool, device=device)
        rest[::128] = False
        held = torch.full((n,), start ** 2, device=device) / (4.0 / 57344)
        st["exp_avg_sq"].copy_(torch.where(rest, held, torch.full_like(held, 57344.0)).to(torch.float8_e5m2))
        v = (st["exp_avg_sq"].float() * (4.0 / 57344))[rest].double().mean()
        for _ in range(150):
            opt.step()
            v = v + (1 - B2) * (end ** 2 - v)
        got = (st["exp_avg_sq"].float().view(-1, 128) * st["scale"][:, 1:]).view(-1)[rest].double().mean()
        assert abs(float(got / v) - 1) < 0.03, (start, end, float(got), float(v))


def test_a_run_repeats_bit_for_bit(device):
    """A few hundred steps of a least-squares problem from one start, twice: the same parameters and states."""
    def run(bits):
        gen = torch.Generator(device=device)
        gen.manual_seed(7)
        a, want = torch.randn(400, 300, device=device, generator=gen), torch.randn(300, device=device, generator=gen)
        p = torch.nn.Parameter(torch.zeros(300, device=device))
        opt = _opt([p], state_bits=bits, lr=2e-2, weight_decay=0.0)
        for _ in range(300):
            p.grad = a.t() @ (a @ (p.detach() - want)) / 400
            opt.step()
        return p.detach(), opt.state[p]
    for bits in (32, 8):
        (p, st), (q, st2) = run(bits), run(bits)
        assert bool(p.isfinite().all()) and torch.equal(p, q)
        assert all(torch.equal(st[k].float(), st2[k].float()) for k in st)


def test_gradients_that_are_not_finite_stay_where_they_are(device):
    for bits in (32, 8):
        params = _params([(1000,)], torch.float32, device, 4)
        opt = _opt(params, state_bits=bits)
        opt.step()
        params[0].grad[300], params[0].grad[700] = float("nan"), float("inf")
        opt.step()
        opt.step()
        bad = ~params[0].detach().isfinite()
        lost = torch.zeros(1000, dtype=torch.bool, device=device)
        if bits == 32:
            lost[300] = lost[700] = True
        else:
            lost[256:384] = lost[640:768] = True
        assert torch.equal(bad | lost, lost) and bool(bad[300]) and bool(bad[700])


def test_zero_gradients_and_tiny_ones(device):
    for bits in (32, 8):
        params = _params([(500,)], torch.float32, device, 5)
        opt = _opt(params, state_bits=bits, weight_decay=0.0)
        params[0].grad.zero_()
        before = params[0].detach().clone()
        opt.step()
        assert torch.equal(before, params[0].detach())
        params[0].grad.fill_(1e-30)
        opt.step()
        # m / (sqrt(v) + eps): v underflows, so the move is lr m / eps, not lr
        assert bool((params[0].detach() - before).abs().max() < 1e-10)


def test_parameters_written_from_outside(device):
    """A 16-bit parameter that was loaded or zeroed between steps is taken as it is; the others keep their master copies."""
    for dtype in (torch.bfloat16, torch.float16):
        params = _params([(1000,)], dtype, device, 6)
        p = params[0]
        opt = _opt(params)
        for t in (1, 2):
            _step_and_check(opt, params, t)
        master = opt.state[p]["master"].clone()
        with torch.no_grad():
            p[:500] = 0.75
        p.grad.zero_()
        opt.step()
        st = opt.state[p]
        want = torch.cat([torch.full((500,), 0.75, device=device), master[500:]]).double()
        m, v = st["exp_avg"].double(), st["exp_avg_sq"].double()
        want = want - (LR * WD * want + LR / (1 - B1 ** 3) * m / (torch.sqrt(v / (1 - B2 ** 3)) + EPS))
        assert float((st["master"].double() - want).abs().max()) <= 20 * U


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_checkpoints(device, dtype, bits, tmp_path):
    """Saved, loaded into another optimiser over copies of the parameters, and continued: the same bits."""
    params = _params([(300, 7), (129,), ()], dtype, device, 8)
    opt = _opt(params, state_bits=bits)
    for t in range(3):
        _new_grads(params, t)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "o.pt")
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    new = _opt(copies, state_bits=bits, lr=1.0)
    new.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
    twin = copy.deepcopy(opt)
    for p, q in zip(params, copies):
        q.grad = p.grad.clone()
    for o in (opt, new):
        o.step()
    assert new.param_groups[0]["lr"] == LR
    for p, q in zip(params, copies):
        assert torch.equal(p, q)
        for k, t in opt.state[p].items():
            s = new.state[q][k]
            assert s.dtype == t.dtype and torch.equal(s.view(torch.uint8) if s.dtype.itemsize == 1 else s, t.view(torch.uint8) if t.dtype.itemsize == 1 else t), k
    assert twin.state_bits == bits
    with pytest.raises(ValueError, match="state_bits"):
        _opt([torch.nn.Parameter(p.detach().clone()) for p in params], state_bits=40 - bits).load_state_dict(opt.state_dict())


def test_checkpoints_of_torch(device):
    params = _params([(50, 6), (13,)], torch.float32, device, 9)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    stock = torch.optim.AdamW(twins, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    for t in range(3):
        _new_grads(params, t)
        for p, q in zip(params, twins):
            q.grad = p.grad.clone()
        stock.step()
    with torch.no_grad():
        for p, q in zip(params, twins):
            p.copy_(q)
    opt = _opt(params, lr=1.0)
    opt.load_state_dict(copy.deepcopy(stock.state_dict()))
    _step_and_check(opt, params, 4)


@pytest.mark.parametrize("bits", [32, 8])
def test_graphs_and_streams(device, bits):
    """Recorded after one eager step and replayed with eager work in between, with a learning rate on the device: the bits of an
    optimiser that takes every step eagerly."""
    shapes = [(300, 70), (129,), (5000,)]
    a, b = _params(shapes, torch.bfloat16, device, 10), _params(shapes, torch.bfloat16, device, 10)
    oa, ob = [_opt(ps, state_bits=bits, lr=torch.tensor(1e-3, device=device)) for ps in (a, b)]
    side = torch.cuda.Stream(device=device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        oa.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            oa.step()
    torch.cuda.current_stream(device).wait_stream(side)
    ob.step()
    for i in range(4):
        for ps, o in ((a, oa), (b, ob)):
            _new_grads(ps, i)
            o.param_groups[0]["lr"].fill_(1e-3 / (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        ob.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), i
    assert float(oa.state[a[0]]["step"]) == 5.0
    fresh = _opt(_params([(4,)], torch.float32, device, 1))
    bad = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), pytest.raises(RuntimeError, match="eager step"):
        with torch.cuda.graph(bad, stream=side):
            fresh.step()


def test_tensors_exchanged_between_steps(device):
    """Whatever is swapped between two steps is seen by the next: gradients that come and go, a parameter's storage, a state's tensor
    or storage, a whole state, the group's list."""
    params = _params([(300,), (40, 30), (700,), (5,)], torch.float32, device, 21)
    opt = _opt(params)
    for t in (1, 2):
        _step_and_check(opt, params, t)
    for p in params:                        # as zero_grad() and a backward pass would
        p.grad = torch.randn_like(p)
    _step_and_check(opt, params, 3)
    params[0].data = params[0].data.clone()
    _step_and_check(opt, params, 4)
    st = opt.state[params[1]]
    st["exp_avg"] = st["exp_avg"].clone()
    st["exp_avg_sq"].data = st["exp_avg_sq"].data.clone()
    _step_and_check(opt, params, 5)
    opt.state[params[2]] = {k: v.clone() for k, v in opt.state[params[2]].items()}
    _step_and_check(opt, params, 6)
    late, params[3].grad = params[3].grad, None
    _step_and_check(opt, params[:3], 7)
    params[3].grad = late
    assert float(opt.state[params[3]]["step"]) == 6.0
    opt.step()
    assert [float(opt.state[p]["step"]) for p in params] == [8.0, 8.0, 8.0, 7.0]
    extra = _params([(64,)], torch.float32, device, 22)
    opt.add_param_group({"params": extra, "lr": 1e-4})
    opt.step()
    assert float(opt.state[extra[0]]["step"]) == 1.0 and float(opt.state[params[0]]["step"]) == 9.0
    opt.state.clear()
    opt.step()
    assert float(opt.state[params[0]]["step"]) == 1.0


def test_a_size_that_no_longer_fits_is_refused(device):
    p = _params([(300,)], torch.float32, device, 23)[0]
    opt = _opt([p])
    opt.step()
    before = p.data.clone()
    p.data = p.data[:10]
    with pytest.raises(ValueError):
        opt.step()
    p.data = before.to("cpu")
    with pytest.raises((TypeError, ValueError)):
        opt.step()


def test_refusals(device):
    from nerf_amd.optim import AdamW
    p = _params([(8, 6)], torch.float32, device, 11)[0]
    opt = _opt([p])
    opt.step()
    keep = p.grad
    p.grad = torch.zeros(8, 6, device=device).to_sparse()
    with pytest.raises(TypeError, match="sparse"):
        opt.step()
    p.grad = keep
    opt.state[p]["exp_avg"] = torch.zeros(7, device=device)
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step()
    opt.state[p]["exp_avg"] = torch.zeros(8, 6, device=device)
    opt.step()
    t = torch.nn.Parameter(torch.zeros(6, 8, device=device).t())
    t.grad = torch.zeros(8, 6, device=device)
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([t]).step()
    # nothing is launched when a later group cannot be: neither its parameters nor an earlier group's move
    a, b = _params([(5,), (6,)], torch.float32, device, 12)
    two = AdamW([{"params": [a]}, {"params": [b], "lr": torch.tensor(1e-3, dtype=torch.float64, device=device)}])
    before = a.detach().clone()
    with pytest.raises(TypeError, match="learning rate"):
        two.step()
    assert torch.equal(a, before) and float(two.state[a]["step"]) == 0.0
    # a gradient of another layout is copied, not refused
    q = torch.nn.Parameter(torch.zeros(8, 6, device=device))
    q.grad = torch.arange(48.0, device=device).view(6, 8).t()
    o = _opt([q], weight_decay=0.0)
    o.step()
    assert torch.equal(o.state[q]["exp_avg"], q.grad * torch.tensor(1 - B1, dtype=torch.float32).item()) or \
        float((o.state[q]["exp_avg"] - (1 - B1) * q.grad).abs().max()) <= 4 * U * 48
    d = torch.nn.Parameter(torch.zeros(4, device=device, dtype=torch.float64))
    d.grad = torch.zeros_like(d)
    with pytest.raises(TypeError, match="float64"):
        AdamW([d]).step()
