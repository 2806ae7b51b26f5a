"""ops.layer_norm, forward and backward, against the definition in 64 bits.

Tolerances (u = 2^-24, half an fp32 step; a sum of N values added by many threads costs at most d(N) u of the sum of magnitudes,
with d(N) = N / 32 + 32 more than the adds any value passes through):
  xh    the mean is exact to d u sigma, a difference to u |x - mu| and r to (d / 2 + 8) u, together e = u (d + 8)(1 + |xh|)
  y     |w| e + 4 u (|xh w| + |b|), and half a step of the output's type
  dx    r u (2 d + 32)(|g| + mean|g| + (1 + |xh|) mean(|g| (1 + |xh|))), and half a step
  dw    u (d(n) + d(c) + 16) sum |dy| (1 + |xh|), db u d(n) sum |dy|, and half a step
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _depth(n):
    return n / 32 + 32


def _step(t, dtype):
    """Half a step of a type at values t (its subnormals have a fixed step)."""
    info = torch.finfo(dtype)
    return torch.maximum(t.abs() * (info.eps / 2), torch.full_like(t, info.smallest_normal * info.eps / 2))


def _oracle(x, w, b, dy, eps):
    x, dy = x.double().cpu(), dy.double().cpu()
    c = x.shape[-1]
    w = torch.ones(c, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(c, dtype=torch.float64) if b is None else b.double().cpu()
    mu = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mu) * r
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    ax, ag = xh.abs(), g.abs()
    n, d = x.shape[0], _depth(c)
    want = {"y": xh * w + b, "dx": dx, "dw": (dy * xh).sum(0), "db": dy.sum(0)}
    tol = {"y": w.abs() * (U * (d + 8) * (1 + ax)) + 4 * U * ((xh * w).abs() + b.abs()),
           "dx": r * U * (2 * d + 32) * (ag + ag.mean(-1, keepdim=True) + (1 + ax) * (ag * (1 + ax)).mean(-1, keepdim=True)),
           "dw": U * (_depth(n) + d + 16) * (dy.abs() * (1 + ax)).sum(0), "db": U * _depth(n) * dy.abs().sum(0)}
    return want, tol


def _check(got, want, tol, what):
    got = got.detach().cpu()
    bound = tol + _step(want, got.dtype) * 1.001 + 1e-300
    err = (got.double() - want).abs()
    assert got.shape == want.shape and bool((err <= bound).all()), (what, float((err / bound).max()))


def _data(n, c, dtype, device, seed, offset=1.0, pad=0):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    normal = lambda *s: torch.randn(*s, device=device, generator=gen)      # noqa: E731
    x = (normal(n, c + pad) * 1.5 + offset * normal(n, 1)).to(dtype)[:, pad:]
    return x, (1 + 0.3 * normal(c)), 0.2 * normal(c), normal(n, c).to(dtype)


SHAPES = [(1, 1), (3, 1), (2, 2), (1, 7), (5, 63), (7, 64), (4, 65), (65, 100), (33, 256), (1, 255), (300, 257), (9, 512), (2, 1000),
          (17, 1024), (5, 1025), (6, 1537), (3, 2048), (2, 2049), (4, 4096), (3, 5000), (2, 8192), (1, 8200), (2, 16384), (1, 20001),
          (2, 33000), (1, 70001), (2000, 8), (5000, 3), (1031, 96), (700, 640), (20011, 128), (17, 129), (9001, 200), (30000, 256)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,c", SHAPES)
def test_forward_and_gradients(device, n, c, dtype):
    from nerf_amd import ops
    x, w, b, dy = _data(n, c, dtype, device, 31 * n + c)
    for wt in {dtype, torch.float32}:
        xl, wl, bl = x.detach().requires_grad_(True), w.to(wt).requires_grad_(True), b.to(wt).requires_grad_(True)
        y = ops.layer_norm(xl, wl, bl)
        assert type(y.grad_fn).__name__ in ("_LayerNormBackward", "ViewBackward0", "UnsafeViewBackward0"), y.grad_fn
        grads = torch.autograd.grad(y, (xl, wl, bl), dy)
        want, tol = _oracle(x, wl.detach(), bl.detach(), dy, 1e-5)
        assert y.dtype == dtype and grads[1].dtype == wt
        for name, got in zip(("y", "dx", "dw", "db"), (y,) + grads):
            _check(got, want[name], tol[name], (name, n, c, dtype, wt))
        again = torch.autograd.grad(ops.layer_norm(xl, wl, bl), (xl, wl, bl), dy)
        assert all(torch.equal(p, q) for p, q in zip(grads, again)), "a second run gave other bits"
        with torch.no_grad():
            assert torch.equal(ops.layer_norm(xl, wl, bl), y)


@pytest.mark.parametrize("n,c,pad", [(50, 257, 3), (33, 256, 64), (70, 127, 1), (300, 131, 2), (20, 1537, 63), (9, 4096, 8), (5, 8192, 1), (3, 20000, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_row_strides_and_missing_parameters(device, n, c, pad, dtype):
    """Rows that are a slice of a wider buffer (starting at any address), a transposed input, a broadcast gradient; weight or bias missing."""
    from nerf_amd import ops
    x, w, b, dy = _data(n, c, dtype, device, n + c, pad=pad)
    assert x.stride(0) == c + pad
    wide = torch.full((n, c + pad), float("nan"), device=device, dtype=dtype)
    wide[:, pad:] = dy
    for xs, dys, ww, bb in ((x, wide[:, pad:], w, b), (x.t().contiguous().t(), dy, None, b), (x, dy[:1].expand(n, c), w, None),
                            (x, dy, None, None)):
        xl = xs.detach().requires_grad_(True)
        leaves = [xl] + [t.to(dtype).requires_grad_(True) for t in (ww, bb) if t is not None]
        params = iter(leaves[1:])
        y = ops.layer_norm(xl, None if ww is None else next(params), None if bb is None else next(params))
        grads = torch.autograd.grad(y, leaves, dys)
        want, tol = _oracle(xs, None if ww is None else ww.to(dtype), None if bb is None else bb.to(dtype), dys, 1e-5)
        names = ["dx"] + (["dw"] if ww is not None else []) + (["db"] if bb is not None else [])
        for name, got in zip(["y"] + names, (y,) + grads):
            _check(got, want[name], tol[name], name)


def test_large_offsets_keep_their_precision(device):
    """Rows whose offset is 1000 times their spread: the values are exact, so the definition's bound holds as anywhere else."""
    from nerf_amd import ops
    for c in (40, 64, 100, 200, 1024, 1500, 5000, 40000):
        x, w, b, dy = _data(6, c, torch.float32, device, c, offset=1500.0)
        xl = x.requires_grad_(True)
        y = ops.layer_norm(xl, w, b)
        (dx,) = torch.autograd.grad(y, (xl,), dy)
        want, tol = _oracle(x.detach(), w, b, dy, 1e-5)
        # (the first mean is off by d u |mu|, which the second pass takes back to d u of ITSELF)
        off = 1500.0 * 4 * _depth(c) * U
        _check(y, want["y"], tol["y"] * (1 + off * 4), ("y", c))
        _check(dx, want["dx"], tol["dx"] * (1 + off * 4), ("dx", c))


def test_constant_rows_and_values_that_are_not_finite(device):
    """A constant row has no spread: xh = 0 and y = b exactly, with gradients scaled by 1 / sqrt(eps).  NaN and inf stay in their row."""
    from nerf_amd import ops
    for c in (1, 64, 300, 2048, 10000, 40000):
        x = torch.full((4, c), 3.25, device=device)
        w, b = torch.rand(c, device=device) + 0.5, torch.randn(c, device=device)
        assert torch.equal(ops.layer_norm(x, w, b), b.expand(4, c))
        x = torch.randn(4, c, device=device)
        clean = ops.layer_norm(x, w, b)
        x[1, c // 2], x[2, 0] = float("nan"), float("inf")
        y = ops.layer_norm(x, w, b)
        assert bool(y[1].isnan().all()) and bool(y[2].isnan().all() if c > 1 else y[2].isnan().all())
        assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])


def test_gradient_against_differences(device):
    """Central differences of a fixed functional in fp64 of the oracle's formula: the gradient is the formula's derivative."""
    from nerf_amd import ops
    x, w, b, dy = _data(3, 37, torch.float32, device, 5)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)

    def f(ts):
        x, w, b = ts
        mu = x.mean(-1, keepdim=True)
        return (((x - mu) / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + 1e-5) * w + b) * dy.double().cpu()).sum()
    base = [t.detach().double().cpu() for t in leaves]
    h = 1e-5
    for i, g in enumerate(grads):
        for k in range(0, base[i].numel(), 5):
            lo, hi = [t.clone() for t in base], [t.clone() for t in base]
            lo[i].view(-1)[k] -= h
            hi[i].view(-1)[k] += h
            slope = float(f(hi) - f(lo)) / (2 * h)
            # differences in fp64: truncation h^2 f''' / 6 and cancellation 2^-53 |f| / h, both below 1e-8; fp32 gradients below 1e-5
            assert abs(float(g.view(-1)[k]) - slope) <= 2e-5 * max(1.0, abs(slope)), (i, k)


def test_empty_and_partial_gradients(device):
    from nerf_amd import ops
    w, b = torch.ones(48, device=device, requires_grad=True), torch.zeros(48, device=device, requires_grad=True)
    x = torch.empty(0, 48, device=device, requires_grad=True)
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 48, device=device))
    assert y.shape == dx.shape == (0, 48) and not dw.any() and not db.any()
    x = torch.randn(5, 2, 48, device=device)
    y = ops.layer_norm(x, w, b)
    (dw,) = torch.autograd.grad(y, (w,), torch.ones_like(y))
    want = torch.nn.functional.layer_norm(x.double().cpu(), (48,)).reshape(-1, 48).sum(0)
    assert y.shape == x.shape and float((dw.double().cpu() - want).abs().max()) <= U * 200 * 20
    assert not ops.layer_norm(x, w.detach(), b.detach()).requires_grad


def test_other_streams_and_captured_graphs(device):
    """Forward and backward on a side stream, and recorded into a graph and replayed on new inputs with eager work in between: the
    bits of the eager call."""
    from nerf_amd import ops
    for n, c in ((700, 256), (40, 5000), (3, 40000)):
        x, w, b, dy = _data(n, c, torch.float32, device, n)
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]

        def both():
            y = ops.layer_norm(*leaves)
            return (y.detach(),) + torch.autograd.grad(y, leaves, dy)
        want = both()
        side = torch.cuda.Stream(device=device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            got = both()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                recorded = both()
        torch.cuda.current_stream(device).wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        for k in range(3):
            with torch.no_grad():
                leaves[0].copy_(torch.randn(n, c, device=device) * (k + 1))
                dy.copy_(torch.randn(n, c, device=device))
            graph.replay()
            torch.cuda.synchronize()
            eager = both()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(recorded, eager)), (n, c, k)
