"""ofi_amd_rms_norm and its gradient against the formulas in 64 bits.

Bounds.  u is the unit roundoff of the rows' type, U = 2^-24.  A row's sum of squares adds at most 128 values a lane, then
64 lanes, then 16 wavefronts (128 + 6 + 16 additions of positive terms, each term with two roundings), so its relative
error is below 160 U, rstd's below 90 U, and n's below 100 U; a scale's below 110 U.  An output in the rows' type adds
u of itself.  e4m3 has four significant bits (half a unit: 2^-4 of the value) and steps of 2^-9 below 2^-6."""
import errno

import pytest
import torch

import _gpu
import aws_ofi_nccl_amd as m
from _rows import TYPES, U32, Rows, ptr, within

pytestmark = pytest.mark.gpu

EPS = 1e-6


def gen(seed):
    return torch.Generator().manual_seed(seed)


def values(g, n, width, scale=1.0):
    v = torch.randn(n, width, generator=g, dtype=torch.float64) * scale
    return v * torch.exp(torch.randn(n, 1, generator=g, dtype=torch.float64))


def norm(lib, x, gain, width, kind, residual=None, total=None, out=None, q=None, scale=None, group=0, rstd=None, eps=EPS,
         n=None, gain_kind=None, stream=None):
    r = lambda t: (t.ptr(), t.pitch) if t is not None else (None, 0)
    return lib.ofi_amd_rms_norm(*r(x), *r(residual), ptr(gain), TYPES[gain_kind or kind][1], x.n if n is None else n, width,
                                TYPES[kind][1], eps, *r(total), *r(out), *r(q), *r(scale), group, ptr(rstd),
                                _gpu.stream() if stream is None else stream)


def check_norm(lib, rows, width, kind, group, residual=True, train=True, pad=0, shift=0, gain_kind=None, seed=1, x64=None, in_place=None):
    g = gen(seed)
    dtype, _, u = TYPES[kind]
    x = Rows(rows, width, dtype, pad, shift, x64 if x64 is not None else values(g, rows, width))
    r = Rows(rows, width, dtype, pad, shift, values(g, rows, width)) if residual else None
    gain = (1 + 0.3 * torch.randn(width, generator=g, dtype=torch.float64)).to(TYPES[gain_kind or kind][0]).cuda()
    s64 = x.t.double().cpu() + (r.t.double().cpu() if r else 0.0)
    groups = 1 if group == 0 else -(-width // group)
    total = {None: Rows(rows, width, dtype, pad, shift), "x": x, "residual": r}[in_place]
    out, rstd = Rows(rows, width, dtype, 0, shift), torch.full((rows,), 7.0, device="cuda")
    q, scale = Rows(rows, width, torch.float8_e4m3fn, pad, shift), Rows(rows, groups, torch.float32, pad)
    assert norm(lib, x, gain, width, kind, r, total, out if train else None, q, scale, group, rstd if train else None,
                gain_kind=gain_kind) == 0
    _gpu.sync()
    rstd64 = 1.0 / torch.sqrt((s64 * s64).mean(dim=1, keepdim=True) + EPS)
    n64 = s64 * rstd64 * gain.double().cpu()
    within(total.t, s64, (u + U32) * s64.abs() + 2.0 ** -25)
    if train:
        within(rstd, rstd64[:, 0], 90 * U32 * rstd64[:, 0])
        within(out.t, n64, (u + 100 * U32) * n64.abs() + 2.0 ** -25)
    wide = torch.nn.functional.pad(n64, (0, groups * (group or width) - width)).view(rows, groups, -1)
    amax = wide.abs().amax(dim=2)
    scale64 = torch.where(amax / 448.0 < 2.0 ** -126, torch.full_like(amax, 2.0 ** -126), amax / 448.0)
    within(scale.t, scale64, 110 * U32 * scale64)
    v64 = (wide / scale64[:, :, None]).view(rows, -1)[:, :width]
    within(q.t.float(), v64, torch.clamp(v64.abs() * 2.0 ** -4, min=2.0 ** -10) + 256 * U32 * v64.abs())
    for b in (x, total, out, q, scale) + ((r,) if r else ()):
        assert b.untouched()
    return dict(x=x, r=r, gain=gain, total=total, rstd=rstd, q=q, scale=scale, n64=n64)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("width", [1, 3, 4, 7, 8, 9, 31, 64, 127, 129, 255, 256, 257, 500, 511, 512, 513, 1000, 1999, 2048, 2049,
                                   4096, 4100, 8192, 8193, 12345, 16384, 16385, 20000, 32767, 32768])
def test_widths(lib, gpu, kind, width):
    check_norm(lib, 3, width, kind, group=128 if width % 2 else 0, seed=width)
    check_norm(lib, 2, width, kind, group=0 if width % 2 else 128, seed=width + 1, pad=3, shift=1)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("group", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("width", [32, 250, 1024, 4000])
def test_groups(lib, gpu, kind, group, width):
    check_norm(lib, 5, width, kind, group, residual=group != 64, seed=group + width)


@pytest.mark.parametrize("rows", [1, 2, 63, 1000, 4097])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (1, 0), (5, 3)])
def test_rows_pitches_and_alignments(lib, gpu, rows, pad, shift):
    check_norm(lib, rows, 520, "bf16", 128, pad=pad, shift=shift, seed=rows)


@pytest.mark.parametrize("in_place", ["x", "residual"])
@pytest.mark.parametrize("width", [77, 4096, 9000])
def test_the_sum_may_replace_an_input(lib, gpu, in_place, width):
    check_norm(lib, 40, width, "bf16", 128, in_place=in_place, seed=3)


def test_a_gain_in_32_bits_beside_rows_of_16(lib, gpu):
    check_norm(lib, 9, 1001, "bf16", 128, gain_kind="f32")
    check_norm(lib, 9, 1024, "f16", 0, gain_kind="f32")


def test_rows_of_zeros_and_groups_of_zeros(lib, gpu):
    x = values(gen(5), 6, 640)
    x[0] = 0
    x[1, 128:256] = 0
    x[2, 639:] = 1e-30
    x[3] *= 1e-4
    got = check_norm(lib, 6, 640, "f32", 128, residual=False, x64=x)
    assert bool((got["scale"].t[0] == 2.0 ** -126).all()) and bool((got["q"].t[0].float() == 0).all())
    assert float(got["scale"].t[1, 1]) == 2.0 ** -126


@pytest.mark.parametrize("group", [0, 64])
def test_nan_and_infinity_show_in_their_row_and_in_no_other(lib, gpu, group):
    g, width = gen(8), 300
    x = values(g, 5, width)
    x[1, 17], x[3, 100], x[4, 299] = float("nan"), float("inf"), float("-inf")
    dtype = TYPES["bf16"][0]
    xr = Rows(5, width, dtype, values=x)
    gain = torch.ones(width, dtype=dtype, device="cuda")
    groups = 1 if group == 0 else -(-width // group)
    out, q, scale = Rows(5, width, dtype), Rows(5, width, torch.float8_e4m3fn), Rows(5, groups, torch.float32)
    rstd = torch.zeros(5, device="cuda")
    assert norm(lib, xr, gain, width, "bf16", None, None, out, q, scale, group, rstd) == 0
    _gpu.sync()
    assert bool(torch.isnan(out.t[1]).all()) and bool(torch.isnan(scale.t[1]).all()) and bool(torch.isnan(q.t[1].float()).all())
    for row, at in ((3, 100), (4, 299)):                       # rstd is 0: 0 * inf at the infinity, 0 elsewhere
        assert float(rstd[row]) == 0.0
        nan = torch.isnan(out.t[row])
        assert bool(nan[at]) and int(nan.sum()) == 1
        bad = torch.isnan(scale.t[row])
        assert int(bad.sum()) == 1 and bool(bad[at // group if group else 0])
    for row in (0, 2):
        assert bool(torch.isfinite(out.t[row]).all()) and bool(torch.isfinite(scale.t[row]).all())


def test_rows_far_apart_pass_32_bits_of_offset(lib, gpu):
    width, pitch = 1000, 1 << 30
    dtype = TYPES["bf16"][0]
    big = torch.zeros((5 * pitch + 4096,), dtype=torch.uint8, device="cuda")
    v = values(gen(4), 6, width).to(dtype)
    rows = [big[k * pitch:k * pitch + 2 * width].view(dtype) for k in range(6)]
    for k, row in enumerate(rows):
        row.copy_(v[k])
    gain = torch.ones(width, dtype=dtype, device="cuda")
    out = Rows(6, width, dtype)
    assert lib.ofi_amd_rms_norm(big.data_ptr(), pitch, None, 0, ptr(gain), m.BFLOAT16, 6, width, m.BFLOAT16, EPS, None, 0,
                                out.ptr(), out.pitch, None, 0, None, 0, 0, None, _gpu.stream()) == 0
    _gpu.sync()
    n64 = v.double() / torch.sqrt((v.double() ** 2).mean(dim=1, keepdim=True) + EPS)
    within(out.t, n64, (TYPES["bf16"][2] + 100 * U32) * n64.abs())


def grad(lib, dout, s, rstd, gain, width, kind, dsum, dx, dgain, work, n=None, gain_kind=None, work_bytes=None):
    r = lambda t: (t.ptr(), t.pitch) if t is not None else (None, 0)
    return lib.ofi_amd_rms_norm_grad(*r(dout), *r(s), ptr(rstd), ptr(gain), TYPES[gain_kind or kind][1], s.n if n is None else n,
                                     width, TYPES[kind][1], *r(dsum), *r(dx), ptr(dgain), ptr(work),
                                     (0 if work is None else work.numel()) if work_bytes is None else work_bytes, _gpu.stream())


def check_grad(lib, rows, width, kind, through=True, pad=0, shift=0, seed=2, in_place=None, gain_kind=None, want_gain=True):
    g = gen(seed)
    dtype, _, u = TYPES[kind]
    s = Rows(rows, width, dtype, pad, shift, values(g, rows, width))
    dout = Rows(rows, width, dtype, pad, shift, values(g, rows, width, 0.1))
    dsum = Rows(rows, width, dtype, pad, shift, values(g, rows, width, 0.1)) if through else None
    gain = (1 + 0.3 * torch.randn(width, generator=g, dtype=torch.float64)).to(TYPES[gain_kind or kind][0]).cuda()
    s64, d64, g64 = s.t.double().cpu(), dout.t.double().cpu(), gain.double().cpu()
    p64 = dsum.t.double().cpu() if through else torch.zeros_like(s64)
    rstd = (1.0 / torch.sqrt((s64 * s64).mean(dim=1) + EPS)).float().cuda()
    dx = {None: Rows(rows, width, dtype, pad, shift), "dout": dout, "dsum": dsum}[in_place]
    dgain = torch.full((width + 2,), 3.0, device="cuda")
    work = torch.full((max(16, lib.ofi_amd_rms_norm_grad_work_bytes(rows, width)),), 0x7F, dtype=torch.uint8, device="cuda")
    guard = torch.full((64,), 0x5A, dtype=torch.uint8, device="cuda")
    assert grad(lib, dout, s, rstd, gain, width, kind, dsum, dx, dgain if want_gain else None, work if want_gain else None,
                gain_kind=gain_kind) == 0
    _gpu.sync()
    r64 = rstd.double().cpu()[:, None]
    h = s64 * r64
    gd = d64 * g64
    mean = (gd * h).mean(dim=1, keepdim=True)
    dx64 = p64 + r64 * (gd - h * mean)
    absmean = (gd * h).abs().mean(dim=1, keepdim=True)
    # the mean: 128 + 6 + 16 additions and three roundings a term; the rest a handful of roundings of each term
    bound = u * dx64.abs() + U32 * (r64 * (4 * gd.abs() + h.abs() * (170 * absmean + 4 * mean.abs())) + 2 * p64.abs()) + 2.0 ** -25
    within(dx.t, dx64, bound)
    for b in (s, dout, dx) + ((dsum,) if through else ()):
        assert b.untouched()
    if want_gain:
        terms = (d64 * h)
        # a workgroup adds its rows one after the other, then the parts are added: never more additions than rows + 6 + 16
        within(dgain[:width], terms.sum(dim=0), U32 * (rows + 24) * terms.abs().sum(dim=0))
        assert bool((dgain[width:] == 3.0).all())
    assert bool((guard == 0x5A).all())
    return dict(s64=s64, d64=d64, g64=g64, p64=p64, dx=dx.t.double().cpu(), dgain=dgain[:width].double().cpu())


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("width", [1, 3, 8, 9, 64, 255, 257, 512, 513, 1999, 2048, 4096, 4097, 8192, 10000, 16384, 16385, 32767,
                                   32768])
def test_gradient_widths(lib, gpu, kind, width):
    check_grad(lib, 5, width, kind, seed=width)


@pytest.mark.parametrize("rows", [1, 2, 3, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025, 2049, 5000])
def test_gradient_rows(lib, gpu, rows):
    check_grad(lib, rows, 200, "bf16", through=rows % 2 == 0, seed=rows)


@pytest.mark.parametrize("rows,width", [(300, 4096), (1500, 1000), (3001, 64)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 0), (8, 0), (3, 5)])
def test_gradient_pitches(lib, gpu, rows, width, pad, shift):
    check_grad(lib, rows, width, "f16", pad=pad, shift=shift, seed=rows + pad)


@pytest.mark.parametrize("in_place", ["dout", "dsum"])
@pytest.mark.parametrize("rows,width", [(1100, 1030), (40, 1030), (256, 4099), (3, 10000), (2, 30000)])
def test_the_gradient_may_replace_an_input(lib, gpu, in_place, rows, width):
    check_grad(lib, rows, width, "bf16", in_place=in_place)


@pytest.mark.parametrize("rows", [1, 17, 255, 256, 257])
@pytest.mark.parametrize("width", [1, 7, 64, 65, 1999, 8192, 8193])
def test_gradient_of_few_rows(lib, gpu, rows, width):
    check_grad(lib, rows, width, "f16", pad=rows % 3, seed=rows + width)


def test_gradient_without_the_gains_and_with_a_gain_in_32_bits(lib, gpu):
    check_grad(lib, 70, 900, "bf16", want_gain=False)
    check_grad(lib, 70, 900, "bf16", gain_kind="f32")


def test_gradient_against_differences(lib, gpu):
    """d/de of sum(dout * n(x + e d, gain + e c)) + sum(dsum * s) by central differences of the formula in 64 bits."""
    got = check_grad(lib, 6, 333, "f32", seed=12)
    g = gen(77)
    dx, dg = torch.randn(6, 333, generator=g, dtype=torch.float64), torch.randn(333, generator=g, dtype=torch.float64)

    def loss(e_x, e_g):
        s = got["s64"] + e_x * dx
        n = s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + EPS) * (got["g64"] + e_g * dg)
        return ((got["d64"] * n).sum() + (got["p64"] * s).sum()).item()

    e = 1e-5
    by_x, by_g = (loss(e, 0) - loss(-e, 0)) / (2 * e), (loss(0, e) - loss(0, -e)) / (2 * e)
    assert abs(by_x - (got["dx"] * dx).sum().item()) <= 1e-5 * (got["dx"] * dx).abs().sum().item()
    assert abs(by_g - (got["dgain"] * dg).sum().item()) <= 1e-5 * (got["dgain"] * dg).abs().sum().item()


@pytest.mark.parametrize("width", [5, 8, 100, 129, 255, 520, 1001, 2047, 4099, 9001])
@pytest.mark.parametrize("pad,shift", [(3, 1), (2, 1), (9, 0)])
def test_what_lies_beside_the_rows_does_not_reach_them(lib, gpu, monkeypatch, width, pad, shift):
    """Bytes of 0xff are NaN in every type."""
    monkeypatch.setattr(Rows, "guard", 0xFF)
    for kind in ("bf16", "f16", "f32"):
        check_norm(lib, 7, width, kind, 32, pad=pad, shift=shift, seed=width)
        check_grad(lib, 7, width, kind, pad=pad, shift=shift, seed=width)


def test_no_rows(lib, gpu):
    x, gain, dgain = Rows(0, 8, torch.float32), torch.ones(8, device="cuda"), torch.full((8,), 5.0, device="cuda")
    assert norm(lib, x, gain, 8, "f32", total=x) == 0
    work = torch.zeros(64, dtype=torch.uint8, device="cuda")
    assert grad(lib, x, x, gain, gain, 8, "f32", None, x, dgain, work) == 0
    _gpu.sync()
    assert bool((dgain == 0).all())


def test_the_same_call_gives_the_same_bits_and_another_streams_call_too(lib, gpu):
    rows, width = 2500, 1024
    dtype = TYPES["bf16"][0]
    s = Rows(rows, width, dtype, values=values(gen(1), rows, width))
    d = Rows(rows, width, dtype, values=values(gen(2), rows, width))
    gain, rstd = torch.ones(width, dtype=dtype, device="cuda"), torch.ones(rows, device="cuda")
    work = torch.empty(lib.ofi_amd_rms_norm_grad_work_bytes(rows, width), dtype=torch.uint8, device="cuda")
    got = []
    _gpu.sync()
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.current_stream()):
        dx, dgain = Rows(rows, width, dtype), torch.zeros(width, device="cuda")
        _gpu.sync()
        with torch.cuda.stream(stream):
            assert grad(lib, d, s, rstd, gain, width, "bf16", None, dx, dgain, work) == 0
        _gpu.sync()
        got.append((dx.t.clone(), dgain))
    for a, b in got[1:]:
        assert torch.equal(a, got[0][0]) and torch.equal(b, got[0][1])


def test_refusals(lib, gpu):
    x, t = Rows(4, 64, torch.bfloat16, values=torch.ones(4, 64)), Rows(4, 64, torch.bfloat16)
    q, scale = Rows(4, 64, torch.float8_e4m3fn), Rows(4, 1, torch.float32)
    gain = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    inval, toobig = -errno.EINVAL, -errno.E2BIG
    call = lambda **k: norm(lib, k.pop("x", x), k.pop("gain", gain), k.pop("width", 64), "bf16", total=k.pop("total", t), **k)
    assert call() == 0
    assert call(width=0) == inval and call(width=32769) == toobig and call(n=1 << 31) == toobig
    assert call(gain=None) == inval and call(total=None) == inval
    assert call(eps=-1.0) == inval and call(eps=float("nan")) == inval
    assert call(q=q) == inval and call(scale=scale) == inval
    assert call(q=q, scale=scale, group=16) == inval and call(q=q, scale=scale, group=512) == inval
    assert call(q=q, scale=scale, group=128) == 0
    assert call(width=65) == inval                                     # the pitch is below a row
    assert lib.ofi_amd_rms_norm(None, 128, None, 0, ptr(gain), m.BFLOAT16, 4, 64, m.BFLOAT16, EPS, t.ptr(), 128, None, 0, None, 0, None, 0,
                                0, None, _gpu.stream()) == inval
    assert lib.ofi_amd_rms_norm(x.ptr() + 1, 128, None, 0, ptr(gain), m.BFLOAT16, 4, 64, m.BFLOAT16, EPS, t.ptr(), 128, None, 0, None, 0,
                                None, 0, 0, None, _gpu.stream()) == inval
    assert lib.ofi_amd_rms_norm(x.ptr(), 129, None, 0, ptr(gain), m.BFLOAT16, 4, 64, m.BFLOAT16, EPS, t.ptr(), 128, None, 0, None, 0,
                                None, 0, 0, None, _gpu.stream()) == inval
    for gain_type, kind in ((m.FLOAT16, m.BFLOAT16), (m.BFLOAT16, m.FLOAT16), (m.INT32, m.INT32), (m.BFLOAT16, 8)):
        assert lib.ofi_amd_rms_norm(x.ptr(), 128, None, 0, ptr(gain), gain_type, 4, 64, kind, EPS, t.ptr(), 128, None, 0, None, 0, None, 0,
                                    0, None, _gpu.stream()) == inval
    rstd, dgain = torch.ones(4, device="cuda"), torch.ones(64, device="cuda")
    need = lib.ofi_amd_rms_norm_grad_work_bytes(4, 64)
    work = torch.zeros(need, dtype=torch.uint8, device="cuda")
    back = lambda **k: grad(lib, k.pop("dout", x), x, k.pop("rstd", rstd), gain, k.pop("width", 64), "bf16", None, k.pop("dx", t),
                            k.pop("dgain", dgain), k.pop("work", work), **k)
    assert back() == 0
    assert back(work=None) == inval and back(work_bytes=need - 1) == inval and back(rstd=None) == inval and back(dout=None) == inval
    assert back(dx=None) == inval and back(width=0) == inval and back(width=32769) == toobig and back(n=1 << 31) == toobig
    _gpu.sync()
    assert _gpu.fetch_async_errors(lib) == 0
