"""The 8-bit rows of ofi_amd_rms_norm to the bit.  Rows of 32 bits have the norm in d_out as it was before it was divided; what d_q holds is
the quotient of that and the scale in d_scale, each rounded once."""
import pytest
import torch

import _gpu
from _rows import Rows
from test_gpu_rms_norm import gen, norm, values

pytestmark = pytest.mark.gpu


def eight_bits(lib, x, gain, width, group):
    rows = x.n
    groups = 1 if group == 0 else -(-width // group)
    out, q, scale = Rows(rows, width, torch.float32), Rows(rows, width, torch.float8_e4m3fn), Rows(rows, groups, torch.float32)
    assert norm(lib, x, gain, width, "f32", None, None, out, q, scale, group) == 0
    _gpu.sync()
    n, s = out.t.cpu(), scale.t.cpu()
    by = s.repeat_interleave(group or width, dim=1)[:, :width]
    return q.t.cpu(), (n / by).to(torch.float8_e4m3fn), n, s


@pytest.mark.parametrize("group", [0, 32, 128, 256])
@pytest.mark.parametrize("width", [3, 60, 250, 1024, 4099])
@pytest.mark.parametrize("size", [1.0, 1e-30, 1e25])
def test_quotients_are_rounded_once(lib, gpu, group, width, size):
    g = gen(width + group)
    x = Rows(300000 // width, width, torch.float32, values=values(g, 300000 // width, width))
    x.t[:, ::7] = -0.0
    gain = (size * (1 + 0.3 * torch.randn(width, generator=g))).cuda()
    got, want, _, _ = eight_bits(lib, x, gain, width, group)
    off = got.view(torch.uint8) != want.view(torch.uint8)
    assert not bool(off.any()), (int(off.sum()), off.numel())


@pytest.mark.parametrize("group", [0, 64])
def test_values_beside_one_beyond_the_range_are_zero(lib, gpu, group):
    """A gain makes one value infinite, and the scale with it: the others divided by it are 0, and it is no number."""
    x = Rows(4, 256, torch.float32, values=values(gen(2), 4, 256))
    x.t[:, 70] = 20.0 * x.t.abs().amax(dim=1)
    gain = torch.ones(256, device="cuda")
    gain[70] = 3e38
    got, _, n, scale = eight_bits(lib, x, gain, 256, group)
    assert bool(torch.isinf(n[:, 70]).all()) and bool(torch.isfinite(n[:, :70]).all())
    lo, hi = (64, 128) if group else (0, 256)
    assert bool(torch.isinf(scale[:, 1 if group else 0]).all())
    inside = got.float()[:, lo:hi]
    assert bool(torch.isnan(inside[:, 70 - lo]).all())
    inside[:, 70 - lo] = 0.0
    assert bool((inside == 0).all())
