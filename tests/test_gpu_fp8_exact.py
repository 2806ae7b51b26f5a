"""Products in 8 bits on whole numbers, where nothing is lost anywhere (ops.matmul_fp8, linear_fp8).

Operands of magnitude at most 4 are their own codes under any scale they get.  With sum |a b| < 2^24 every partial sum, in any
order, is held by fp32 as it is; products in a group differ by less than 2^5, so that the 8-bit instruction cuts none.  So the
result is the definition's, rounded once to the output's type, and a single term left out, taken twice or from another row shows."""
import pytest
import torch

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


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


# (m, n, k) -> blocks of k 7, 9, 10, 11, 12, 13 (the image a tile starts in goes by the count's parity, its words of scales by the
# count / 4 rounded up); two and three tiles a workgroup, the last round full and not; fewer tiles than workgroups
LARGE = [(4096, 8192, 896), (4096, 8192, 1100), (4090, 8187, 1280), (6100, 8190, 1400), (5120, 8192, 1536), (4096, 8100, 1601), (4608, 8192, 2100),
         (2560, 3584, 4096), (2500, 3500, 2200), (3840, 4000, 1900)]


def test_the_large_cases_take_large_tiles():
    from nerf_amd._lib import lib
    for m, n, k in LARGE:
        assert lib.nerf_fp8_matmul_tile(m, n, k, 1) == 256, (m, n, k)
        assert lib.nerf_fp8_matmul_tile(m, n, k, 0) == lib.nerf_fp8_matmul_tile(m, n, k, 2) == 128
    tiles = [(-(-m // 256)) * (-(-n // 256)) for m, n, _ in LARGE]
    assert min(tiles) < 256 and max(tiles) > 512 and any(t % 256 for t in tiles if t > 256)
    assert {-(-k // 128) % 4 for _, _, k in LARGE} == {0, 1, 2, 3}
    assert lib.nerf_fp8_matmul_tile(4, 8192, 8192, 1) == 0 and lib.nerf_fp8_matmul_tile(0, 1, 1, 1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", LARGE)
def test_large_tiles(device, m, n, k):
    """bf16, with a bias and without, and the call's repetition."""
    from nerf_amd import ops
    a, b = _whole(m, k, 4, device, m), _whole(n, k, 4, device, n + 1)
    assert 16 * k < 2 ** 24
    want = _product(a, b)
    _would_show(a, b, want, torch.bfloat16)
    qa, qb = ops.quantize_fp8(a), ops.quantize_fp8(b)
    bias = _whole(1, n, 4, device, 5)[0]
    for _ in range(2):
        assert torch.equal(ops.matmul_fp8(qa, qb, out_dtype=torch.bfloat16), want.bfloat16())
        assert torch.equal(ops.matmul_fp8(qa, qb, bias, True, torch.bfloat16), (want + bias.double()).clamp_min(0).bfloat16())


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
