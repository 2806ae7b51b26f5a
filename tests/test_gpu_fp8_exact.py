"""Products in 8 bits on whole numbers, where nothing is lost anywhere (ops.matmul_fp8, linear_fp8).

Operands of magnitude at most 4 are their own codes under any scale they get.  With sum |a b| < 2^24 every partial sum, in any
order, is held by fp32 as it is; products in a group differ by less than 2^5, so that the 8-bit instruction cuts none.  So the
result is the definition's, rounded once to the output's type, and a single term left out, taken twice or from another row shows."""
import pytest
import torch

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _whole(rows, k, top, device, seed):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    return torch.randint(-top, top + 1, (rows, k), device=device, generator=gen).float()


def _product(a, b):
    return a.double() @ b.double().t().contiguous()


def _would_show(a, b, want, out):
    """None of these passes for `want`: nothing at all, and one block of 128 left out at either end or in the middle."""
    assert want.any()
    blocks = -(-a.shape[1] // 128)
    for kb in {0, blocks // 2, blocks - 1}:
        part = slice(128 * kb, 128 * (kb + 1))
        assert not torch.equal((want - _product(a[:, part], b[:, part])).to(out), want.to(out)), kb


@pytest.mark.gpu
@pytest.mark.parametrize("out", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (4, 100, 70001), (17, 1024, 16400), (40, 640, 5000), (64, 515, 9000), (65, 129, 1000), (130, 258, 257),
                                   (256, 256, 65536), (257, 300, 20011), (1001, 777, 333), (700, 1030, 2100)])
def test_few_rows_small_tiles_and_slices_of_k(device, m, n, k, out):
    from nerf_amd import ops
    a, b = _whole(m, k, 4, device, m), _whole(n, k, 4, device, n + 1)
    a[0, 0] = b[0, 0] = a[-1, -1] = b[-1, -1] = 3.0
    assert 16 * k < 2 ** 24
    want = _product(a, b)
    _would_show(a, b, want, out)
    assert torch.equal(ops.matmul_fp8(ops.quantize_fp8(a), ops.quantize_fp8(b), out_dtype=out), want.to(out))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2 ** 22 - 1, 2 ** 22 + 300])
def test_the_weights_gradient_over_many_rows(device, rows):
    """On both sides of 2^22 rows, where the product's kernel changes."""
    from nerf_amd import ops
    x, dy = _whole(rows, 24, 1, device, 1), _whole(rows, 20, 1, device, 2)
    w = torch.zeros(20, 24, device=device, requires_grad=True)
    (dw,) = torch.autograd.grad(ops.linear_fp8(x, w), w, dy)
    assert rows < 2 ** 24
    want = _product(dy.t(), x.t())
    _would_show(dy.t(), x.t(), want, torch.float32)
    assert torch.equal(dw.double(), want)
