"""NeRF modules pickled whole (torch.save(model)): with the options of wide networks, and from before there were any."""
import io

import pytest
import torch

KW = dict(D=8, W=256, input_ch=63, input_ch_views=27, output_ch=5, skips=[4], use_viewdirs=True)


def _through_a_file(m):
    buf = io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


def test_a_module_without_the_options():
    from nerf_amd.run_nerf_helpers import NeRF
    m = NeRF(**KW)
    del m.layer_dtype, m.pts_norms
    back = _through_a_file(m)
    assert back.fused_arch() and back.layer_dtype == "f32" and back.pts_norms is None
    assert all(torch.equal(p, q) for p, q in zip(m.parameters(), back.parameters()))


@pytest.mark.parametrize("norm", [False, True])
def test_the_options_come_back(norm):
    from nerf_amd.run_nerf_helpers import NeRF
    m = NeRF(**KW, layer_norm=norm)
    m.layer_dtype = "fp8"
    back = _through_a_file(m)
    assert back.layer_dtype == "fp8" and not back.fused_arch() and (back.pts_norms is not None) == norm
    assert list(back.state_dict()) == list(m.state_dict())
