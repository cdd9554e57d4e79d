"""A gated block of so many columns that its workgroups go in two launches."""
import pytest
import torch

import _gpu
import aws_ofi_nccl_amd as m
from _experts import act, act_error, gen
from _rows import U32, within

pytestmark = pytest.mark.gpu


def test_few_rows_into_more_columns_than_one_launch_has(lib, gpu):
    """512 experts with a row each, 2^20 columns in blocks that share a scale: 2^22 workgroups of 1024 lanes."""
    experts, inner = 512, 1 << 20
    g = gen(11)
    w = torch.empty(experts, 2, inner, dtype=torch.float16, device="cuda")  # one value a column: width 1
    for e in range(0, experts, 64):
        w[e:e + 64].copy_(torch.randn(64, 2, inner, generator=g, device="cuda"))
    x = torch.randn(experts, 1, generator=g, device="cuda").to(torch.float16)
    offset = torch.arange(experts + 1, dtype=torch.int32, device="cuda")
    out = torch.full((experts, inner), 0xFF, dtype=torch.uint8, device="cuda")  # NaN
    scale = torch.full((experts, inner // 128), float("nan"), device="cuda")
    assert lib.ofi_amd_expert_gated(x.data_ptr(), 2, None, 0, m.FLOAT16, offset.data_ptr(), experts, experts, w.data_ptr(), 2, 4 * inner, None, 1, inner,
                                    m.SILU, out.data_ptr(), inner, m.E4M3, scale.data_ptr(), inner // 32, None, 0, 0, None, 0, _gpu.stream()) == 0
    _gpu.sync()
    assert not bool((out.bitwise_and(0x7F) == 0x7F).any()) and not bool(torch.isnan(scale).any())
    for e in (0, 1, 63, 255, 256, 257, 510, 511):
        gate, up = (x[e].double() * w[e, p].double() for p in range(2))
        value = act("silu", gate)[0]
        want = (value * up).view(-1, 128)
        off = ((act_error("silu", gate) + 8 * U32 * gate.abs()) * up.abs() + 8 * U32 * (value * up).abs()).view(-1, 128)
        most = want.abs().amax(dim=1)
        within(scale[e], (most / 448).clamp(min=2.0 ** -126), off.amax(dim=1) / 448 + 2 * U32 * most / 448)
        by = scale[e].double()[:, None]
        got = out[e].view(torch.float8_e4m3fn).float().double().view(-1, 128) * by
        within(got, want, off + 2.0 ** -4 * (want.abs() + off) + 2.0 ** -10 * by + 4 * U32 * want.abs())
