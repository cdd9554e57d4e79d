"""Workspaces of the norm's gradient and of the sort: nothing beyond the bytes asked for is written, and what they held does not matter; and
the norm under the bounds of what a lane holds.

Bounds, U = 2^-24.  A lane adds at most 32 squares (chunks times elements), then there are six additions of lanes and four of wavefronts; a
term has the rounding of the residual's addition twice: 44 U of a sum of squares.  Mean and eps a rounding each, half of all that for the
root, root and inverse one each: 25 U, and what is beyond first order: 26 U of rstd.  n has three more roundings, a scale one more than
that, and a quotient both errors and a rounding of its own: 29, 30 and 60 U.  The mean of the gradient: 32 + 10 additions and three roundings
a term, 48 U of the mean of sizes.  A gain's gradient: a workgroup's rows (of 512 workgroups, and of up to 8 rows at once), 8 more to join those,
16 parts a lane and 32 lanes, two roundings a term; up to 256 rows 16 a wavefront and 16 wavefronts: (rows / 512 + 66) U of the sum of sizes."""
import numpy as np
import pytest
import torch

import _gpu
from _rows import TYPES, U32, Rows, within
from test_gpu_rms_norm import EPS, gen, grad, norm, values
from test_gpu_token_dispatch import Call, byte_rows, make_ids

pytestmark = pytest.mark.gpu
GUARD = 4096


def guarded(need, fill):
    work = torch.full((need + GUARD,), fill, dtype=torch.uint8, device="cuda")
    work[need:] = 0xC3
    return work


@pytest.mark.parametrize("rows", [1, 100, 257, 511, 512, 513, 2000])
@pytest.mark.parametrize("width", [1, 7, 100, 1999, 4100, 9001, 32767])
def test_workspace_of_the_gradient(lib, gpu, rows, width):
    rows = min(rows, 600) if width > 5000 else rows
    dtype = TYPES["bf16"][0]
    s, dout = (Rows(rows, width, dtype, values=torch.randn(rows, width, generator=gen(k))) for k in (1, 2))
    gain, rstd = torch.ones(width, dtype=dtype, device="cuda"), torch.ones(rows, device="cuda")
    need = lib.ofi_amd_rms_norm_grad_work_bytes(rows, width)
    got = []
    for fill in (0x00, 0xFF):
        work, dx, dgain = guarded(need, fill), Rows(rows, width, dtype), torch.full((width,), 3.0, device="cuda")
        assert grad(lib, dout, s, rstd, gain, width, "bf16", None, dx, dgain, work, work_bytes=need) == 0
        _gpu.sync()
        assert bool((work[need:] == 0xC3).all())
        got.append((dx.t.clone(), dgain))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("tokens,top_k", [(4096, 2), (4097, 2), (9000, 8), (33000, 8), (140000, 8)])
@pytest.mark.parametrize("experts", [1, 60, 1024])
def test_workspace_of_the_sort(lib, gpu, tokens, top_k, experts):
    rng = np.random.default_rng(tokens)
    ids = make_ids(rng, tokens, top_k, experts, 0.1, True)
    need = lib.ofi_amd_token_dispatch_work_bytes(tokens, top_k, experts)
    x = byte_rows(rng, tokens, 16)
    for fill in (0x00, 0xFF):
        call = Call(lib, ids, experts, tokens * top_k, x, 16)
        work = guarded(need, fill)
        call.work = work[:need] if need else None
        assert call.run() == 0
        _gpu.sync()
        call.check(ids)
        assert bool((work[need:] == 0xC3).all())


@pytest.mark.parametrize("width", [5, 33, 300, 1999, 4096, 8192, 8200, 20000, 32768])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [4, 700])
def test_norms_within_what_a_lane_adds(lib, gpu, width, kind, rows):
    dtype, _, u = TYPES[kind]
    g = gen(width)
    x, r = (Rows(rows, width, dtype, values=values(g, rows, width)) for _ in range(2))
    gain = (1 + 0.3 * torch.randn(width, generator=g)).cuda()
    out, rstd = Rows(rows, width, dtype), torch.zeros(rows, device="cuda")
    q, scale = Rows(rows, width, torch.float8_e4m3fn), Rows(rows, 1, torch.float32)
    assert norm(lib, x, gain, width, kind, r, None, out, q, scale, 0, rstd, gain_kind="f32") == 0
    _gpu.sync()
    s64 = x.t.double() + r.t.double()
    r64 = 1.0 / torch.sqrt((s64 * s64).mean(dim=1, keepdim=True) + EPS)
    n64 = s64 * r64 * gain.double()
    within(rstd, r64[:, 0], 26 * U32 * r64[:, 0])
    within(out.t, n64, ((u if kind != "f32" else 0.0) + 29 * U32) * n64.abs())
    sc64 = n64.abs().amax(dim=1, keepdim=True) / 448.0
    within(scale.t, sc64, 30 * U32 * sc64)
    v64 = n64 / sc64
    within(q.t.float(), v64, torch.clamp(v64.abs() * 2.0 ** -4, min=2.0 ** -10) + 60 * U32 * v64.abs())
    dout = Rows(rows, width, dtype, values=values(g, rows, width, 0.1))
    s = Rows(rows, width, dtype, values=s64)
    dx, dgain = Rows(rows, width, dtype), torch.zeros(width, device="cuda")
    work = torch.empty(lib.ofi_amd_rms_norm_grad_work_bytes(rows, width), dtype=torch.uint8, device="cuda")
    assert grad(lib, dout, s, rstd, gain, width, kind, None, dx, dgain, work, gain_kind="f32") == 0
    _gpu.sync()
    rr, d64 = rstd.double()[:, None], dout.t.double()
    h, gd = s.t.double() * rr, d64 * gain.double()
    mean, sizes = (gd * h).mean(dim=1, keepdim=True), (gd * h).abs().mean(dim=1, keepdim=True)
    dx64 = rr * (gd - h * mean)
    within(dx.t, dx64, u * dx64.abs() + U32 * rr * (4 * gd.abs() + h.abs() * (48 * sizes + 4 * mean.abs())) + 2.0 ** -149)
    within(dgain, (d64 * h).sum(dim=0), U32 * (rows / 512 + 66) * (d64 * h).abs().sum(dim=0))
