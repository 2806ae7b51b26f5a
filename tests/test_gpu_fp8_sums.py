"""How exactly products in 8 bits are summed (ops.matmul_fp8, linear_fp8).

Where every product and every partial sum, in any order, is a whole multiple of a unit below 2^24 of it, fp32 holds them all: the
result is the definition's, rounded once to the output's type, and compared for equality."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def _whole(rows, k, top, device, seed):
    """Whole numbers of magnitude up to `top` <= 15: their own codes under any scale they get."""
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    return torch.randint(-top, top + 1, (rows, k), device=device, generator=gen).float()


def _product(a, b):
    """a b^T in 64 bits on the GPU."""
    return a.double() @ b.double().t().contiguous()


@pytest.mark.parametrize("m,n,k", [(1, 1, 256), (16, 40, 300), (64, 257, 1024), (65, 100, 700), (200, 300, 256), (129, 257, 5000), (256, 256, 7000)])
@pytest.mark.parametrize("out", TYPES, ids=IDS)
def test_small_products_beside_large_ones_that_cancel(device, m, n, k, out):
    """Products of +-2^8 next to products of 2^-6 in every group of eight: the large ones cancel over the row, the small ones are the
    result.  (sum |a b| <= (k / 8 + 1) 2^8 + 2^-6 k: below 2^24 units of 2^-6 for these k.)  A bf16 output of many rows is the documented
    exception: its products keep 13 bits below the largest of eight."""
    from nerf_amd import ops
    gen = torch.Generator(device=device)
    gen.manual_seed(m + n + k)
    a, b = torch.zeros(m, k, device=device), torch.zeros(n, k, device=device)
    large = torch.arange(0, k - k % 16, 8, device=device)
    sign = torch.ones(large.numel(), device=device)
    sign[1::2] = -1
    a[:, large], b[:, large] = 16.0 * sign, 16.0
    small = torch.arange(k, device=device) % 8 != 0
    a[:, small] = 2.0 ** -3 * torch.randint(0, 2, (m, int(small.sum())), device=device, generator=gen)
    b[:, small] = 2.0 ** -3 * torch.randint(0, 2, (n, int(small.sum())), device=device, generator=gen)
    want = _product(a, b)
    assert float((a.double().abs() @ b.double().abs().t().contiguous()).max()) * 2 ** 6 < 2 ** 24
    got = ops.matmul_fp8(ops.quantize_fp8(a), ops.quantize_fp8(b), out_dtype=out)
    if out == torch.bfloat16 and m > 64:
        mag = a.double().abs() @ b.double().abs().t().contiguous()
        assert bool(((got.double() - want).abs() <= 7 * 2.0 ** -13 * mag + 2.0 ** -8 * want.abs()).all())
    else:
        assert torch.equal(got, want.to(out))


@pytest.mark.parametrize("m,n,k", [(40, 300, 200), (300, 520, 333), (1001, 777, 333), (600, 130, 1001)])
def test_sixteen_bit_floats_of_operands_whose_sizes_vary_along_k(device, m, n, k):
    """fp16 against the definition: half a step, 2^-11 of the value, and what fp32 sums of exact products may lose, at most k / 8 + 16
    roundings of 2^-23 of sum |a b|."""
    from nerf_amd import ops
    gen = torch.Generator(device=device)
    gen.manual_seed(k)
    normal = lambda *s: torch.randn(*s, device=device, generator=gen)      # noqa: E731
    a, b = normal(m, k) * torch.exp(normal(1, k)), normal(n, k) * torch.exp(2 * normal(1, k)) / 64
    qa, qb = ops.quantize_fp8(a), ops.quantize_fp8(b)

    def values(q):
        blocks = q.codes.shape[1] // 128
        unit = torch.ldexp(torch.ones(q.rows, blocks, dtype=torch.float64, device=device), q.scales[:, :blocks].int() - 127)
        return (q.codes.float().double().view(q.rows, blocks, 128) * unit[:, :, None]).view(q.rows, -1)[:, : q.k]
    va, vb = values(qa), values(qb)
    want, mag = _product(va, vb), _product(va.abs(), vb.abs())
    got = ops.matmul_fp8(qa, qb, out_dtype=torch.float16).double()
    assert bool(want.abs().max() < 65504)
    tol = (k / 8 + 16) * 2.0 ** -23 * mag + 2.0 ** -11 * want.abs() * 1.001 + 2.0 ** -25
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


def test_the_layer_in_sixteen_bit_floats(device):
    """linear_fp8 and its three products in fp16: whole numbers, exact up to one rounding."""
    from nerf_amd import ops
    x, w, dy = (_whole(r, c, 4, device, i) for i, (r, c) in enumerate(((200, 300), (130, 300), (200, 130))))
    x, w = x.half().requires_grad_(True), w.half().requires_grad_(True)
    y = ops.linear_fp8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy.half())
    xd, wd = x.detach(), w.detach()
    assert torch.equal(y, _product(xd, wd).half()) and torch.equal(dx, _product(dy, wd.t()).half()) and torch.equal(dw, _product(dy.t(), xd.t()).half())
