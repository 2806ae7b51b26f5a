"""The layer and optimiser operators as a network uses them: a wide NeRF with norms, 8-bit products and AdamW -- its query and
gradients against the same network in 64 bits, its training step eager and replayed, and the training command."""
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _net(device, seed, layer_dtype="fp8", **kw):
    from nerf_amd.run_nerf_helpers import NeRF
    torch.manual_seed(seed)
    m = NeRF(**{**dict(D=6, W=320, input_ch=63, input_ch_views=27, output_ch=5, skips=[4], use_viewdirs=True, layer_norm=True), **kw}).to(device)
    m.layer_dtype = layer_dtype
    with torch.no_grad():
        for norm in m.pts_norms or []:
            norm.weight.copy_(1 + 0.2 * torch.randn_like(norm.weight))
            norm.bias.copy_(0.1 * torch.randn_like(norm.bias))
    return m


def _eight(x):
    """x [r, k] in fp64 as 8 bits hold it (values on the grid of the block's power-of-two scale)."""
    r, k = x.shape
    w = torch.nn.functional.pad(x, (0, -k % 128)).view(r, -1, 128)
    top = w.abs().amax(2, keepdim=True)
    frac, ex = torch.frexp(top)
    unit = torch.ldexp(torch.ones_like(top), (ex - 9 + (frac > 0.875).int()).clamp_min(-126))
    v = w / unit
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp_min(2.0 ** -6))[1] - 4)
    return (torch.round(v / step) * step * unit).view(r, -1)[:, :k]


def _oracle(m, x, eight, inputs=None):
    """The network of _forward_layers in 64 bits on the CPU.  Quantised inputs are steps: an activation that differs in the last bit may
    take another code.  So every quantised layer starts from the activations the network itself fed it (`inputs`)."""
    p = {k: v.detach().double().cpu() for k, v in m.state_dict().items()}
    lin = lambda name, h: h @ p[name + ".weight"].t() + p[name + ".bias"]      # noqa: E731
    wide = (lambda name, h: _eight(h) @ _eight(p[name + ".weight"]).t() + p[name + ".bias"]) if eight else lin
    feed = iter(inputs) if inputs is not None else None
    pts, views = torch.split(x.double().cpu(), [m.input_ch, m.input_ch_views], -1)
    h, errors = pts, []
    for i in range(m.D):
        if i > 0 and feed is not None:
            got = next(feed).double().cpu()
            errors.append(float((got - h).abs().max()))
            h = got
        h = torch.relu((wide if i > 0 else lin)(f"pts_linears.{i}", h))
        if m.pts_norms is not None:
            mu = h.mean(-1, keepdim=True)
            var = ((h - mu) ** 2).mean(-1, keepdim=True)
            h = (h - mu) / torch.sqrt(var + 1e-5) * p[f"pts_norms.{i}.weight"] + p[f"pts_norms.{i}.bias"]
        if i in m.skips:
            h = torch.cat([pts, h], -1)
    alpha = lin("alpha_linear", h)
    if feed is not None:
        got = next(feed).double().cpu()
        errors.append(float((got - h).abs().max()))
        h = got
    h = torch.cat([wide("feature_linear", h), views], -1)
    h = torch.relu(lin("views_linears.0", h))
    return torch.cat([lin("rgb_linear", h), alpha], -1), errors


@pytest.mark.parametrize("eight", [False, True])
def test_network_against_64_bits(device, eight, monkeypatch):
    """Layer by layer: every hidden vector is within 2e-4 of the definition applied to the vector before it (fp32 sums of 400
    values of order 1, a norm that scales by at most 1 / spread), and so is the output."""
    from nerf_amd import ops
    m = _net(device, 1, "fp8" if eight else "f32")
    x = torch.randn(1000, 90, device=device)
    seen = []
    if eight:
        inner = ops.linear_fp8
        monkeypatch.setattr(ops, "linear_fp8", lambda h, *a: (seen.append(h.detach()), inner(h, *a))[1])
    with torch.no_grad():
        got = m(x)
    want, errors = _oracle(m, x, eight, seen if eight else None)
    assert not eight or len(seen) == m.D
    assert float((got.double().cpu() - want).abs().max()) < 2e-4 and all(e < 2e-4 for e in errors), errors


def test_gradients_of_a_stack_with_exact_inputs(device):
    """norm -> product -> product against autograd in 64 bits on the same quantised values (each product's own operands)."""
    from nerf_amd import ops
    gen = torch.Generator(device=device)
    gen.manual_seed(4)
    x = torch.randn(200, 300, device=device, generator=gen, requires_grad=True)
    w, b = torch.randn(300, device=device, generator=gen, requires_grad=True), torch.randn(300, device=device, generator=gen, requires_grad=True)
    v = (torch.randn(130, 300, device=device, generator=gen) * 0.1).requires_grad_(True)
    dy = torch.randn(200, 130, device=device, generator=gen)
    h = ops.layer_norm(x, w, b)
    h.retain_grad()
    ops.linear_fp8(h, v).backward(dy)
    f = lambda t: t.detach().double().cpu()      # noqa: E731
    dh = _eight(f(dy)) @ _eight(f(v).t().contiguous()).t()
    dv = _eight(f(dy).t().contiguous()) @ _eight(f(h).t().contiguous()).t()
    # fp32 sums of at most 200 products of magnitude below 40
    assert float((f(h.grad) - dh).abs().max()) < 1e-4 and float((f(v.grad) - dv).abs().max()) < 4e-4
    xd, wd, bd = (f(t).requires_grad_(True) for t in (x, w, b))
    torch.nn.functional.layer_norm(xd, (300,), wd, bd).backward(f(h.grad))
    for got, want in ((x.grad, xd.grad), (w.grad, wd.grad), (b.grad, bd.grad)):
        assert float((f(got) - want).abs().max()) < 1e-5 * float(want.abs().max()) + 1e-5


@pytest.mark.parametrize("bits", [32, 8])
def test_training_step_eager_and_replayed(device, bits):
    """GraphedTrainStep over two such networks and AdamW walks the weights of the eager loop, with renders between the steps."""
    from nerf_amd.graph_step import GraphedTrainStep
    from nerf_amd.optim import AdamW
    from nerf_amd.run_nerf import render, run_network
    from nerf_amd.run_nerf_helpers import get_embedder, img2mse_pair
    e, _ = get_embedder(10, 0)
    ed, _ = get_embedder(4, 0)
    qf = lambda inputs, viewdirs, fn: run_network(inputs, viewdirs, fn, embed_fn=e, embeddirs_fn=ed, netchunk=1 << 16)      # noqa: E731

    def make():
        ms = [_net(device, s) for s in (5, 6)]
        params = [p for m in ms for p in m.parameters()]
        opt = AdamW(params, lr=torch.tensor(5e-4, device=device), weight_decay=0.01, state_bits=bits)
        kw = dict(network_fn=ms[0], network_query_fn=qf, N_samples=16, N_importance=24, network_fine=ms[1], perturb=0.0,
                  raw_noise_std=0.0, white_bkgd=True, use_viewdirs=True, ndc=False, near=2.0, far=6.0)
        return params, opt, kw
    H = W = 32
    K = np.array([[40.0, 0, 16.0], [0, 40.0, 16.0], [0, 0, 1]])
    gen = torch.Generator(device=device)
    gen.manual_seed(9)
    batches = []
    for _ in range(6):
        o = torch.randn(100, 3, device=device, generator=gen) * 0.1 + torch.tensor([0.0, 0.0, 4.0], device=device)
        d = torch.nn.functional.normalize(torch.randn(100, 3, device=device, generator=gen) * 0.2 - torch.tensor([0.0, 0.0, 1.0], device=device), dim=-1)
        batches.append((torch.stack([o, d]), torch.rand(100, 3, device=device, generator=gen)))
    pa, oa, ka = make()
    losses = []
    for rays, target in batches:
        rgb, _, _, ex = render(H, W, K, chunk=1 << 15, rays=rays, retraw=True, **ka)
        oa.zero_grad()
        img, _, loss = img2mse_pair(rgb, ex["rgb0"], target)
        loss.backward()
        oa.step()
        losses.append(float(loss.detach()))
        assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in pa)
    pb, ob, kb = make()
    stepper = GraphedTrainStep(H, W, K, kb, pb, ob, 100, eager_steps=2)
    got = []
    for rays, target in batches:
        got.append(float(stepper.step(rays, target)))
        with torch.no_grad():
            render(H, W, K, chunk=1 << 15, rays=rays, **kb)
    assert stepper.g_grad is not None
    np.testing.assert_allclose(got, losses, rtol=1e-6)
    assert all(torch.equal(p, q) for p, q in zip(pa, pb))
    assert float(ob.state[pb[0]]["step"]) == 6.0


def test_training_command(device, tmp_path, capsys):
    """--layer_norm --layer_dtype fp8 --optimizer adamw --state_bits 8 on a tiny scene: runs, saves, resumes; another update rule's
    checkpoint is refused."""
    from nerf_amd.run_nerf import train
    from test_datasets import write_blender_scene
    data = os.path.join(tmp_path, "scene")
    write_blender_scene(data, n=(3, 1, 1), size=16)
    common = ["--datadir", data, "--dataset_type", "blender", "--basedir", str(tmp_path), "--expname", "wide", "--N_rand", "64", "--N_samples", "8",
              "--N_importance", "8", "--use_viewdirs", "--white_bkgd", "--no_batching", "--netdepth", "3", "--netwidth", "160", "--netdepth_fine", "3",
              "--netwidth_fine", "160", "--i_print", "1", "--i_weights", "2", "--i_testset", "100000", "--i_video", "100000", "--testskip", "1"]
    wide = ["--layer_norm", "--layer_dtype", "fp8", "--optimizer", "adamw", "--state_bits", "8"]
    os.makedirs(os.path.join(tmp_path, "wide"))
    assert np.isfinite(train(common + wide + ["--N_iters", "4"]))
    assert np.isfinite(train(common + wide + ["--N_iters", "6"]))
    assert "Reloading from" in capsys.readouterr().out
    with pytest.raises(ValueError, match="state_bits"):
        train(common + wide[:-1] + ["32", "--N_iters", "6"])
    saved = torch.load(os.path.join(tmp_path, "wide", "000004.tar"), weights_only=True)
    assert saved["optimizer_state_dict"]["state"][0]["exp_avg"].dtype == torch.float8_e4m3fn
    assert "pts_norms.0.weight" in saved["network_fn_state_dict"]
