"""Refusals of the layer and optimiser operators, which need no GPU: argument checks of the C ABI and of the Python entry points."""
import ctypes

import pytest
import torch


def _err():
    from nerf_amd._lib import lib
    return lib.nerf_last_error().decode()


def test_layer_norm_argument_errors():
    from nerf_amd import ops
    from nerf_amd._lib import lib
    fwd = lambda n=2, c=8, t=0, ldx=8, wt=0, ldy=8, eps=1e-5, x=16, y=16: lib.nerf_layer_norm_fwd(      # noqa: E731
        n, c, t, x, ldx, wt, None, None, eps, y, ldy, None, None)
    assert fwd(n=0, x=None, y=None) == 0
    for kw, word in ((dict(n=-1), "n=-1"), (dict(c=0), "c=0"), (dict(c=1 << 25), "c="), (dict(t=3), "type=3"), (dict(t=1, wt=2), "w_type=2"),
                     (dict(t=0, wt=1), "w_type=1"), (dict(ldx=7), "ldx=7"), (dict(ldy=7), "ldy=7"), (dict(eps=-1.0), "eps"),
                     (dict(eps=float("nan")), "eps"), (dict(x=None), "null"), (dict(y=None), "null")):
        assert fwd(**kw) == -1 and word in _err(), (kw, _err())
    bwd = lambda n=2, c=8, x=16, dy=16, st=16, dw=16, ws=16, ld=8: lib.nerf_layer_norm_bwd(      # noqa: E731
        n, c, 0, x, ld, dy, ld, 0, None, st, 16, ld, dw, None, ws, None)
    for kw in (dict(x=None), dict(dy=None), dict(st=None), dict(ws=None), dict(c=0), dict(ld=7)):
        assert bwd(**kw) == -1, kw
    assert lib.nerf_layer_norm_workspace_floats(0, 5) >= 10 and lib.nerf_layer_norm_workspace_floats(10 ** 9, 5) < 10 ** 6
    with pytest.raises(TypeError, match="HIP device"):
        ops.layer_norm(torch.zeros(2, 3))
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm(torch.zeros(2, 3), eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm(torch.zeros(2, 3), eps=float("nan"))


def test_fp8_argument_errors():
    from nerf_amd import ops
    from nerf_amd._lib import lib
    assert [lib.nerf_fp8_code_stride(k) for k in (0, 1, 128, 129)] == [0, 128, 128, 256]
    assert [lib.nerf_fp8_scale_stride(k) for k in (0, 1, 512, 513)] == [0, 4, 4, 8]
    q = lambda rows=2, cols=8, t=0, x=16, ldx=8, mask=None, ldm=8, c=16, s=16, ct=None, st=None, sum_t=0, cs=None, ws=None: lib.nerf_fp8_quantize(      # noqa: E731
        rows, cols, t, x, ldx, mask, ldm, c, s, ct, st, sum_t, cs, ws, None)
    assert q(rows=0) == 0
    for kw, word in ((dict(rows=-1), "rows=-1"), (dict(cols=0), "cols=0"), (dict(t=5), "type=5"), (dict(ldx=7), "stride"), (dict(mask=16, ldm=3), "stride"),
                     (dict(x=None), "null"), (dict(s=None), "null"), (dict(ct=16), "null"), (dict(c=None, s=None), "null"), (dict(cs=16), "null"),
                     (dict(t=1, cs=16, ws=16, sum_t=2), "sum_type"), (dict(c=8), "multiple of 16"), (dict(cols=1 << 30, ldx=1 << 30), "more than one launch")):
        assert q(**kw) == -1 and word in _err(), (kw, _err())
    mm = lambda m=2, n=2, k=128, a=16, sa=16, b=16, sb=16, bt=0, bias=None, t=0, c=16, ldc=2: lib.nerf_fp8_matmul(      # noqa: E731
        m, n, k, a, sa, b, sb, bt, bias, 0, t, c, ldc, None, None)
    assert mm(m=0) == 0 and mm(n=0) == 0
    for kw, word in ((dict(m=-1), "m=-1"), (dict(k=0), "k=0"), (dict(t=7), "type=7"), (dict(t=1, bias=16, bt=2), "bias_type"), (dict(ldc=1), "ldc=1"),
                     (dict(a=None), "null"), (dict(c=None), "null"), (dict(a=8), "multiple"), (dict(sb=6), "multiple")):
        assert mm(**kw) == -1 and word in _err(), (kw, _err())
    codes, scales = torch.zeros(3, 128, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(3, 4, dtype=torch.uint8)
    for args, exc, word in (((codes, scales, 0), ValueError, "k=0"), ((codes, scales, 129), ValueError, "expected codes"), ((codes[:2], scales, 100), ValueError, "expected"),
                            ((codes.view(torch.uint8), scales, 100), TypeError, "float8"), ((codes, scales.int(), 100), TypeError, "uint8"),
                            ((codes, scales, 100), TypeError, "HIP device"), ((codes[0], scales, 100), ValueError, "codes")):
        with pytest.raises(exc, match=word):
            ops.Fp8Rows(*args)
    with pytest.raises(ValueError, match="matrix"):
        ops.quantize_fp8(torch.zeros(3))
    with pytest.raises(TypeError, match="HIP device"):
        ops.quantize_fp8(torch.zeros(3, 4))
    with pytest.raises(TypeError, match="HIP device"):
        ops.linear_fp8(torch.zeros(3, 4), torch.zeros(2, 4))
    with pytest.raises(TypeError, match="Fp8Rows"):
        ops.matmul_fp8(torch.zeros(3, 4), torch.zeros(2, 4))


def test_adamw_argument_errors():
    from nerf_amd._lib import lib
    from nerf_amd.optim import AdamW
    ptr = lambda v: (ctypes.c_void_p * 1)(v)      # noqa: E731

    def step(n=1, count=4, t=0, bits=32, p=16, g=16, m=16, v=16, sc=0, ma=0, st=16, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, ws=16):
        return lib.nerf_adamw_step(n, (ctypes.c_int64 * 1)(count), t, bits, ptr(p), ptr(g), ptr(m), ptr(v), ptr(sc), ptr(ma), ptr(st), None, 1e-3, b1, b2, eps,
                                   wd, ws, None)
    assert step(n=0) == 0
    for kw, word in ((dict(n=-1), "n_tensors"), (dict(t=4), "type=4"), (dict(bits=16), "state_bits=16"), (dict(b1=1.0), "beta1"), (dict(b2=-0.1), "beta2"),
                     (dict(eps=-1.0), "eps"), (dict(wd=float("nan")), "weight_decay"), (dict(count=-1), "counts[0]"), (dict(count=1 << 50), "counts[0]"),
                     (dict(p=0), "null"), (dict(g=0), "null"), (dict(m=0), "null"), (dict(bits=8), "null"), (dict(t=1), "null"), (dict(st=0), "step counter"),
                     (dict(ws=None), "null")):
        assert step(**kw) == -1 and word in _err(), (kw, _err())
    p = torch.nn.Parameter(torch.zeros(3))
    for kw, word in ((dict(state_bits=16), "state_bits"), (dict(lr=-1.0), "lr"), (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"),
                     (dict(eps=-1e-8), "eps"), (dict(weight_decay=-0.1), "weight_decay"), (dict(lr=float("nan")), "lr")):
        with pytest.raises(ValueError, match=word):
            AdamW([p], **kw)
    with pytest.raises(ValueError, match="twice"):
        AdamW([p, p])
    opt = AdamW([p])
    opt.step()                     # no gradient: nothing to do
    p.grad = torch.zeros(3)
    with pytest.raises(TypeError, match="HIP device"):
        opt.step()
    assert not opt.state
    assert opt.param_groups[0]["capturable"]
    # rules that are not this one's are refused, whole, before anything is taken over
    for stock in (torch.optim.AdamW([p], amsgrad=True), torch.optim.AdamW([p], maximize=True), torch.optim.Adam([p], weight_decay=0.1)):
        with pytest.raises(ValueError, match="amsgrad, maximize"):
            opt.load_state_dict(stock.state_dict())
    opt.load_state_dict(torch.optim.Adam([p], lr=0.25).state_dict())
    assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[0]["capturable"]


def test_options_of_the_training_command():
    from nerf_amd.run_nerf import config_parser
    a = config_parser().parse_args([])
    assert (a.layer_norm, a.layer_dtype, a.optimizer, a.weight_decay, a.state_bits) == (False, "f32", "adam", 1e-2, 32)
    a = config_parser().parse_args("--layer_norm --layer_dtype fp8 --optimizer adamw --state_bits 8 --weight_decay 0.1".split())
    assert (a.layer_norm, a.layer_dtype, a.optimizer, a.weight_decay, a.state_bits) == (True, "fp8", "adamw", 0.1, 8)
    for bad in ("--layer_dtype fp4", "--optimizer sgd", "--state_bits 16"):
        with pytest.raises(SystemExit):
            config_parser().parse_args(bad.split())


def test_networks_with_norms():
    from nerf_amd.run_nerf_helpers import NeRF
    kw = dict(D=8, W=256, input_ch=63, input_ch_views=27, output_ch=5, skips=[4], use_viewdirs=True)
    plain, normed = NeRF(**kw), NeRF(**kw, layer_norm=True)
    assert plain.fused_arch() and not normed.fused_arch()
    extra = set(normed.state_dict()) - set(plain.state_dict())
    assert extra == {f"pts_norms.{i}.{k}" for i in range(8) for k in ("weight", "bias")}
    plain.layer_dtype = "fp8"
    assert not plain.fused_arch()
    plain.layer_dtype = "int8"
    with pytest.raises(ValueError, match="layer_dtype"):
        plain.fused_arch()
