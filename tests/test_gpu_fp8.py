"""Products in 8 bits (ops.quantize_fp8, matmul_fp8, linear_fp8) against their definition in 64 bits.

Quantisation is exact by definition (a power-of-two scale, one rounding to nearest even): codes and scales are compared for
equality.  Products: the operands' values are known exactly, so with A = sum |a b| over k
  fp32 outputs    products are exact in the bf16 instruction; each of the at most k / 8 + 16 roundings of the running sum (one per group of
                  products it takes in, and the adds that join partial sums) costs at most 2^-23 of A
  16-bit outputs  the fp8 instruction cuts the products of a group of 8 to multiples of 2^(E - 13), E the exponent of the group's
                  largest (which itself, of at most 8 bits, stays whole): the other seven lose less than 2^-13 of it each, together
                  less than 7 * 2^-13 A; the groups are then summed like the fp32 outputs' products; and half a step of the
                  output's type
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def _oracle_quantize(x):
    """x [r, k] (fp64, CPU) -> values after rounding [r, k], scale exponents [r, blocks]."""
    r, k = x.shape
    blocks = -(-k // 128)
    wide = torch.zeros(r, blocks * 128, dtype=torch.float64)
    wide[:, :k] = x
    wide = wide.view(r, blocks, 128)
    mag = torch.where(wide.isfinite(), wide.abs(), torch.zeros_like(wide)).amax(2)
    frac, ex = torch.frexp(mag)
    e = torch.where(mag > 0, ex - 9 + (frac > 0.875).int(), torch.full_like(ex, -126)).clamp_min(-126)
    unit = torch.ldexp(torch.ones_like(mag), e)[:, :, None]
    v = wide / unit
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp_min(2.0 ** -6))[1] - 4)
    q = torch.round(v / step) * step * unit
    q = torch.where(wide.isfinite(), q, torch.full_like(q, float("nan")))
    return q.view(r, -1)[:, :k], e


def _values(q):
    """What an Fp8Rows stands for, in fp64 on the CPU; its padding is checked to be zero."""
    codes, scales = q.codes.cpu().float().double(), q.scales.cpu()
    blocks = codes.shape[1] // 128
    assert not scales[:, blocks:].any() and bool((q.codes.view(torch.uint8).cpu()[:, q.k:] == 0).all())
    unit = torch.ldexp(torch.ones(codes.shape[0], blocks, dtype=torch.float64), scales[:, :blocks].int() - 127)
    return (codes.view(-1, blocks, 128) * unit[:, :, None]).view(codes.shape[0], -1)[:, : q.k], scales[:, :blocks].int() - 127


def _same(a, b):
    return torch.equal(a.nan_to_num(nan=12345.0), b.nan_to_num(nan=12345.0))


def _check(got, want, mag, k, what):
    got = got.detach().cpu()
    info = torch.finfo(got.dtype)
    if got.dtype == torch.float32:
        tol = (k / 8 + 16) * 2.0 ** -23 * mag
    else:
        tol = 7 * 2.0 ** -13 * mag + (k / 8 + 16) * 2.0 ** -23 * mag + torch.maximum(want.abs() * 1.001, torch.full_like(want, info.smallest_normal)) * (info.eps / 2)
    err = (got.double() - want).abs()
    # (the type's largest value and half a step beyond it, 65520 in fp16, is rounded to infinity)
    err[(got == want.sign() * float("inf")) & (want.abs() + tol >= info.max * (1 + info.eps / 4))] = 0
    assert got.shape == want.shape and bool((err <= tol + 1e-300).all()), (what, float((err / (tol + 1e-300)).max()))


def _data(r, k, dtype, device, seed):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    x = torch.randn(r, k, device=device, generator=gen) * torch.exp(2 * torch.randn(r, 1, device=device, generator=gen))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("r,k", [(1, 1), (1, 127), (3, 128), (5, 129), (130, 64), (129, 257), (64, 640), (2, 8200), (1000, 90)])
def test_quantisation_is_the_definition(device, r, k, dtype):
    from nerf_amd import ops
    x = _data(r, k, dtype, device, r + k)
    x[0, 0] = 448.0 * 4                     # a block whose largest value is exactly at the top of its scale's range
    if k > 1:
        x[-1, 1] = 0.0
    got, e = _values(ops.quantize_fp8(x))
    want, we = _oracle_quantize(x.double().cpu())
    assert torch.equal(got, want) and torch.equal(e, we.int())
    # rows of a wider buffer, starting at an odd address; a transposed matrix
    wide = torch.full((r, k + 3), float("nan"), dtype=dtype, device=device)
    wide[:, 3:] = x
    assert torch.equal(_values(ops.quantize_fp8(wide[:, 3:]))[0], want)
    assert torch.equal(_values(ops.quantize_fp8(x.t().contiguous().t()))[0], want)
    for got in ops._quantize(wide[:, 3:], True, True)[:2]:
        assert torch.equal(_values(got)[0], want if got.k == k and got.rows == r else _oracle_quantize(x.double().cpu().t())[0])
    # both directions and the column sums at once, with a mask
    mask = torch.randn(r, k, device=device).to(dtype)
    mask[0, 0] = float("nan")
    q, qt, s = ops._quantize(x, True, True, mask, torch.float32)
    xm = torch.where(mask <= 0, torch.zeros_like(x), x).double().cpu()
    assert torch.equal(_values(q)[0], _oracle_quantize(xm)[0]) and torch.equal(_values(qt)[0], _oracle_quantize(xm.t())[0])
    assert bool(((s.double().cpu() - xm.sum(0)).abs() <= 2.0 ** -24 * 140 * xm.abs().sum(0)).all())


def test_extreme_values(device):
    """Zeros, subnormals, the largest values, and values that are not finite: those become NaN and leave the others alone."""
    from nerf_amd import ops
    x = torch.randn(6, 300, device=device)
    x[0] = 0
    x[1] *= 1e-38
    x[1, 5] = 1e-45
    x[2] *= 3e37
    x[3, 7], x[3, 200], x[4, 0] = float("nan"), float("inf"), float("-inf")
    x[5] = torch.linspace(-448, 448, 300)
    got, e = _values(ops.quantize_fp8(x))
    want, we = _oracle_quantize(x.double().cpu())
    assert _same(got, want) and torch.equal(e, we.int())
    w = torch.randn(20, 300, device=device)
    with torch.no_grad():
        y, clean = ops.linear_fp8(x, w), ops.linear_fp8(x.nan_to_num(0, 0, 0), w)
    assert bool(y[3].isnan().all()) and bool(y[4].isnan().all()) and not y[0].any() and torch.equal(y[5], clean[5])
    relu = ops.linear_fp8(x[3:], w, None, True)
    assert bool(relu[:2].isnan().all()) and bool((relu[2] >= 0).all())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_values_that_are_not_finite_stay_in_their_place(device, dtype):
    """In both directions at once: NaN codes exactly there, everyone else's code and scale as if they were not there."""
    from nerf_amd import ops
    x = _data(300, 290, torch.float32, device, 5).to(dtype)
    for i, j, v in ((0, 0, "inf"), (5, 130, "nan"), (6, 131, "-inf"), (127, 127, "nan"), (128, 128, "inf"), (299, 289, "nan"), (40, 200, "-inf")):
        x[i, j] = float(v)
    x[200:, 250] = float("nan")          # a whole column of a tile
    x[257, :] = float("inf")             # whole blocks of a row
    q, qt, s = ops._quantize(x, True, True, None, torch.float32)
    wide = x.double().cpu()
    for got, w in ((q, wide), (qt, wide.t())):
        want, e = _oracle_quantize(w)
        v, ge = _values(got)
        assert _same(v, want) and torch.equal(ge, e.int())
    bad = ~wide.isfinite().all(0)
    assert bool((~s.isfinite().cpu() == bad).all())
    assert _same(_values(ops.quantize_fp8(x))[0], _oracle_quantize(wide)[0])


PRODUCTS = [(1, 1, 1), (1, 17, 128), (4, 300, 1000), (16, 16, 128), (17, 33, 129), (64, 256, 256), (65, 100, 384), (100, 64, 77), (129, 130, 257),
            (256, 256, 1024), (300, 520, 640), (1, 4096, 2048), (33, 31, 8192), (1000, 4, 256), (513, 700, 90), (260, 1030, 2100), (40, 24, 20000)]


@pytest.mark.parametrize("out", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_products(device, m, n, k, out):
    from nerf_amd import ops
    a, b = ops.quantize_fp8(_data(m, k, torch.float32, device, m)), ops.quantize_fp8(_data(n, k, torch.float32, device, n + 1))
    va, vb = _values(a)[0], _values(b)[0]
    # (scaled so that fp16 can hold the result)
    bias = torch.randn(n, device=device)
    shrink = 1.0
    if out == torch.float16:
        a.scales[:, : -(-k // 128)] -= 12
        shrink = 2.0 ** -12
    want, mag = shrink * (va @ vb.t()), shrink * (va.abs() @ vb.abs().t())
    _check(ops.matmul_fp8(a, b, out_dtype=out), want, mag, k, (m, n, k))
    for bt in {out, torch.float32}:
        wb = want + bias.to(bt).double().cpu()
        extra = mag + bias.abs().double().cpu()
        _check(ops.matmul_fp8(a, b, bias.to(bt), False, out), wb, extra, k, ("bias", bt))
        _check(ops.matmul_fp8(a, b, bias.to(bt), True, out), wb.clamp_min(0), extra, k, ("relu", bt))
    assert torch.equal(ops.matmul_fp8(a, b, out_dtype=out), ops.matmul_fp8(a, b, out_dtype=out))


@pytest.mark.parametrize("m,n,k", [(4353, 4360, 100), (4096, 8192, 768), (4090, 8187, 1000), (6100, 8190, 700)])
@pytest.mark.parametrize("out", TYPES[1:], ids=IDS[1:])
def test_more_large_tiles_than_workgroups(device, m, n, k, out):
    """Large tiles, of which a workgroup takes two or three, asking for the next one's rows while it finishes the last; and small ones."""
    from nerf_amd import ops
    a, b = ops.quantize_fp8(_data(m, k, torch.float32, device, m)), ops.quantize_fp8(_data(n, k, torch.float32, device, n + 1))
    bias = _data(1, n, out, device, 7)[0]
    got = ops.matmul_fp8(a, b, bias, out_dtype=out)
    va, vb, vbias = _values(a)[0].to(device), _values(b)[0].to(device), bias.double()
    want, mag = (va @ vb.t() + vbias).cpu(), (va.abs() @ vb.abs().t() + vbias.abs()).cpu()
    _check(got, want, mag, k, (m, n, k, out))
    assert torch.equal(ops.matmul_fp8(a, b, bias, out_dtype=out), got)


@pytest.mark.parametrize("m,n,k", [(4, 100, 70001), (17, 1024, 16400), (40, 3000, 5000), (64, 515, 9000)])
@pytest.mark.parametrize("out", TYPES, ids=IDS)
def test_few_rows_and_a_long_k(device, m, n, k, out):
    from nerf_amd import ops
    a, b = ops.quantize_fp8(_data(m, k, torch.float32, device, m)), ops.quantize_fp8(_data(n, k, torch.float32, device, n + 1))
    va, vb = _values(a)[0], _values(b)[0]
    _check(ops.matmul_fp8(a, b, out_dtype=out), va @ vb.t(), va.abs() @ vb.abs().t(), k, (m, n, k, out))


@pytest.mark.parametrize("dtype,w_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                           (torch.float16, torch.float16)])
@pytest.mark.parametrize("n,k,m,relu", [(1, 5, 3, False), (130, 90, 256, True), (257, 333, 129, False), (1000, 256, 256, True), (5000, 64, 40, False),
                                        (70, 1030, 515, True), (40000, 130, 20, False)])
def test_linear_and_its_gradients(device, n, k, m, relu, dtype, w_dtype):
    from nerf_amd import ops
    x = _data(n, k, dtype, device, n).requires_grad_(True)
    w = (torch.randn(m, k, device=device) * 0.1).to(w_dtype).requires_grad_(True)
    b = torch.randn(m, device=device).to(w_dtype).requires_grad_(True)
    dy = (torch.randn(n, m, device=device) * 0.01).to(dtype)
    y = ops.linear_fp8(x, w, b, relu)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == db.dtype == w_dtype
    f = lambda t: t.detach().double().cpu()      # noqa: E731
    q = lambda t: _oracle_quantize(t.contiguous())[0]      # noqa: E731
    qx, qw = q(f(x)), q(f(w))
    want, mag = qx @ qw.t() + f(b), qx.abs() @ qw.abs().t() + f(b).abs()
    _check(y, want.clamp_min(0) if relu else want, mag, k, "y")
    g = torch.where(f(y) <= 0, torch.zeros(n, m, dtype=torch.float64), f(dy)) if relu else f(dy)
    for name, got, (p, r) in (("dx", dx, (q(g), q(f(w).t()))), ("dw", dw, (q(g.t()), q(f(x).t())))):
        _check(got, p @ r.t(), p.abs() @ r.abs().t(), p.shape[1], name)
    tol = 2.0 ** -24 * 140 * g.abs().sum(0) + (torch.finfo(w_dtype).eps / 2) * g.sum(0).abs() * 1.001 + 1e-7
    assert bool(((f(db) - g.sum(0)).abs() <= tol).all())
    again = torch.autograd.grad(ops.linear_fp8(x, w, b, relu), (x, w, b), dy)
    assert all(torch.equal(p, r) for p, r in zip((dx, dw, db), again))
    with torch.no_grad():
        held = ops.quantize_fp8(w)
        assert torch.equal(ops.linear_fp8(x, held, b, relu), y)


def test_more_rows_than_a_tile_product_takes_along_k(device):
    """The weight's gradient over 2^22 + 300 rows: its k is more than the tiles' offsets reach."""
    from nerf_amd import ops
    n, k, m = 2 ** 22 + 300, 24, 20
    x, w = torch.randn(n, k, device=device), torch.randn(m, k, device=device, requires_grad=True)
    dy = torch.randn(n, m, device=device)
    y = ops.linear_fp8(x, w)
    (dw,) = torch.autograd.grad(y, w, dy)
    xt, gt = ops._quantize(x, False, True)[1], ops._quantize(dy, False, True)[1]
    vx, vg = _values(xt)[0].to(device), _values(gt)[0].to(device)
    _check(dw, (vg @ vx.t()).cpu(), (vg.abs() @ vx.abs().t()).cpu(), n, "dw")


def test_gradients_against_differences_where_eight_bits_are_exact(device):
    """Small whole numbers are their own e4m3 codes, so the product is the plain one and its differences are the gradient."""
    from nerf_amd import ops
    gen = torch.Generator(device=device)
    gen.manual_seed(3)
    whole = lambda *s: torch.randint(-4, 5, s, device=device, generator=gen).float()      # noqa: E731
    x, w, b, dy = whole(6, 40).requires_grad_(True), whole(9, 40).requires_grad_(True), whole(9).requires_grad_(True), whole(6, 9)
    grads = torch.autograd.grad(ops.linear_fp8(x, w, b), (x, w, b), dy)
    f = lambda: float((ops.linear_fp8(x, w, b) * dy).sum())      # noqa: E731
    with torch.no_grad():
        for t, g in zip((x, w, b), grads):
            for i in range(0, t.numel(), 7):
                flat = t.view(-1)
                keep = float(flat[i])
                flat[i] = keep + 1
                hi = f()
                flat[i] = keep - 1
                lo = f()
                flat[i] = keep
                assert (hi - lo) / 2 == float(g.reshape(-1)[i])


def test_shapes_broadcasts_and_empty_batches(device):
    from nerf_amd import ops
    w, b = torch.randn(24, 50, device=device, requires_grad=True), torch.randn(24, device=device, requires_grad=True)
    x = torch.randn(1, 50, device=device, requires_grad=True)
    y = ops.linear_fp8(x.expand(3, 7, 50), w, b)
    assert y.shape == (3, 7, 24)
    y.sum().backward()
    assert x.grad.shape == (1, 50) and bool((b.grad == 21).all())
    rows = [ops.linear_fp8(x, w, b)[0] for _ in range(2)]
    assert torch.equal(rows[0], y[2, 6].detach()) and torch.equal(rows[0], rows[1])
    w.grad = b.grad = None
    e = torch.empty(0, 50, device=device, requires_grad=True)
    ops.linear_fp8(e, w, b, True).sum().backward()
    assert e.grad.shape == (0, 50) and not w.grad.any() and not b.grad.any()
    v = torch.randn(50, device=device)
    assert torch.equal(ops.linear_fp8(v, w.detach()), ops.linear_fp8(v[None], w.detach())[0])


def test_no_gradient_is_lost_silently(device):
    from nerf_amd import ops
    a, b = ops.quantize_fp8(torch.randn(4, 70, device=device)), ops.quantize_fp8(torch.randn(6, 70, device=device))
    bias = torch.zeros(6, device=device, requires_grad=True)
    with pytest.raises(ValueError, match="no backward pass"):
        ops.matmul_fp8(a, b, bias)
    with pytest.raises(ValueError, match="no backward pass"):
        ops.linear_fp8(torch.randn(4, 70, device=device), b, bias)
    with torch.no_grad():
        assert ops.matmul_fp8(a, b, bias).shape == (4, 6)


def test_streams_and_graphs(device):
    from nerf_amd import ops
    for n, k, m, dtype in ((300, 200, 130, torch.float32), (4, 2048, 640, torch.bfloat16), (3000, 256, 256, torch.bfloat16)):
        x = _data(n, k, dtype, device, 1).requires_grad_(True)
        w = (torch.randn(m, k, device=device) * 0.1).to(dtype).requires_grad_(True)
        b = torch.randn(m, device=device).to(dtype).requires_grad_(True)
        dy = torch.randn(n, m, device=device).to(dtype)

        def both():
            y = ops.linear_fp8(x, w, b, True)
            return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)
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
        for i in range(3):
            with torch.no_grad():
                x.copy_(_data(n, k, dtype, device, 10 + i))
                w.mul_(0.9)
            graph.replay()
            torch.cuda.synchronize()
            eager = both()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(recorded, eager)), (n, i)
