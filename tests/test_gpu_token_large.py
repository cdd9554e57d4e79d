"""Norms and token exchanges at sizes whose kernels read and write past the caches (beyond 100 MB and beyond 256 MB a call) and that
take several launches, against the formulas in 64 bits, computed on the GPU in parts.  The bounds are those of
test_gpu_rms_norm.py and test_gpu_token_combine.py."""
import pytest
import torch

import _gpu
import aws_ofi_nccl_amd as m
from _rows import TYPES, U32, ptr

pytestmark = pytest.mark.gpu

EPS = 1e-6


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows(g, n, width, dtype, pitch=None):
    """n rows in a buffer `pitch` elements apart; what lies between them is 7."""
    full = torch.full((n, pitch or width), 7.0, device="cuda", dtype=dtype)
    full[:, :width] = torch.randn(n, width, generator=g, device="cuda")
    return full, full[:, :width]


def where(t):
    return t.data_ptr(), t.stride(0) * t.element_size()


def close(got, want, bound):
    far = (got.double() - want).abs() > bound
    assert not bool(far.any()), (int(far.sum()), torch.nonzero(far)[0].tolist())
    assert bool(torch.isfinite(got).all())


def parts(n, width):
    step = max(1, (1 << 24) // width)
    return [(lo, min(n, lo + step)) for lo in range(0, n, step)]


@pytest.mark.parametrize("n,width,pitch,kind,group", [(4000, 8190, 8192, "bf16", 128), (9000, 8192, 8192, "bf16", 128),
                                                      (3000, 16384, 16384, "bf16", 0), (20000, 2044, 2048, "f32", 64),
                                                      (60000, 1024, 1024, "f16", 256), ((1 << 21) + 5, 16, 16, "f16", 0),
                                                      (9000, 4001, 4003, "bf16", 0), (50000, 250, 251, "f16", 64),
                                                      (100000, 97, 101, "bf16", 32), (7000, 8191, 8191, "f16", 128)])
def test_norms(lib, gpu, n, width, pitch, kind, group):
    dtype, code, u = TYPES[kind]
    g = gen(n)
    _, x = rows(g, n, width, dtype, pitch)
    _, r = rows(g, n, width, dtype, pitch)
    total_full, total = rows(g, n, width, dtype, pitch)
    out_full, out = rows(g, n, width, dtype, pitch)
    gain = (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).to(dtype)
    groups = 1 if group == 0 else -(-width // group)
    q = torch.full((n, pitch), 0.5, device="cuda").to(torch.float8_e4m3fn)
    scale, rstd = torch.zeros(n, groups, device="cuda"), torch.zeros(n, device="cuda")
    assert lib.ofi_amd_rms_norm(*where(x), *where(r), ptr(gain), code, n, width, code, EPS, *where(total), *where(out), ptr(q), pitch,
                                *where(scale), group, ptr(rstd), _gpu.stream()) == 0
    _gpu.sync()
    if pitch > width:
        assert bool((total_full[:, width:] == 7).all()) and bool((out_full[:, width:] == 7).all())
        assert bool((q.view(torch.uint8)[:, width:] == q.new_full((1,), 0.5, dtype=torch.float32).to(torch.float8_e4m3fn)
                     .view(torch.uint8)).all())
    for lo, hi in parts(n, width):
        s64 = x[lo:hi].double() + r[lo:hi].double()
        r64 = 1.0 / torch.sqrt((s64 * s64).mean(dim=1, keepdim=True) + EPS)
        n64 = s64 * r64 * gain.double()
        close(total[lo:hi], s64, (u + U32) * s64.abs() + 2.0 ** -25)
        close(rstd[lo:hi], r64[:, 0], 90 * U32 * r64[:, 0])
        close(out[lo:hi], n64, (u + 100 * U32) * n64.abs() + 2.0 ** -25)
        wide = torch.nn.functional.pad(n64, (0, groups * (group or width) - width)).view(hi - lo, groups, -1)
        sc64 = (wide.abs().amax(dim=2) / 448.0).clamp(min=2.0 ** -126)   # x and residual may cancel in a whole group
        close(scale[lo:hi], sc64, 110 * U32 * sc64)
        v64 = (wide / sc64[:, :, None]).view(hi - lo, -1)[:, :width]
        close(q[lo:hi, :width].float(), v64, torch.clamp(v64.abs() * 2.0 ** -4, min=2.0 ** -10) + 256 * U32 * v64.abs())


@pytest.mark.parametrize("n,width,pitch,kind,in_place", [(5000, 4096, 4096, "bf16", None), (12000, 4092, 4096, "bf16", "dsum"),
                                                         (9000, 8192, 8192, "bf16", "dout"), (70000, 512, 512, "f32", None),
                                                         (200000, 250, 256, "f16", None), (3000, 16380, 16384, "bf16", "dout"),
                                                         (2000, 12288, 12288, "f32", "dsum"), (600, 32768, 32768, "f32", None),
                                                         (1500, 32000, 32000, "bf16", "dsum"), (9000, 4001, 4003, "bf16", "dsum"),
                                                         (50000, 1021, 1023, "f16", None)])
def test_gradients_of_norms(lib, gpu, n, width, pitch, kind, in_place):
    dtype, code, u = TYPES[kind]
    g = gen(n)
    _, s = rows(g, n, width, dtype, pitch)
    _, dout = rows(g, n, width, dtype, pitch)
    _, dsum = rows(g, n, width, dtype, pitch)
    keep_d, keep_p = dout.clone(), dsum.clone()
    dx = {None: rows(g, n, width, dtype, pitch)[1], "dout": dout, "dsum": dsum}[in_place]
    gain = (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).to(dtype)
    rstd = torch.rsqrt(s.float().square().mean(dim=1) + EPS)
    dgain = torch.zeros(width, device="cuda")
    work = torch.empty(lib.ofi_amd_rms_norm_grad_work_bytes(n, width), dtype=torch.uint8, device="cuda")
    assert lib.ofi_amd_rms_norm_grad(*where(dout), *where(s), ptr(rstd), ptr(gain), code, n, width, code, *where(dsum), *where(dx),
                                     ptr(dgain), ptr(work), work.numel(), _gpu.stream()) == 0
    _gpu.sync()
    want, sizes = torch.zeros(width, dtype=torch.float64, device="cuda"), torch.zeros(width, dtype=torch.float64, device="cuda")
    for lo, hi in parts(n, width):
        d, r = keep_d[lo:hi].double(), rstd[lo:hi].double()[:, None]
        h, gd, p = s[lo:hi].double() * r, d * gain.double(), keep_p[lo:hi].double()
        mean, absmean = (gd * h).mean(dim=1, keepdim=True), (gd * h).abs().mean(dim=1, keepdim=True)
        dx64 = p + r * (gd - h * mean)
        close(dx[lo:hi], dx64, u * dx64.abs() + U32 * (r * (4 * gd.abs() + h.abs() * (170 * absmean + 4 * mean.abs())) + 2 * p.abs()) +
              2.0 ** -25)
        want += (d * h).sum(dim=0)
        sizes += (d * h).abs().sum(dim=0)
    close(dgain, want, U32 * (n / 512 + 200) * sizes)      # 512 workgroups add their rows, then their 512 parts are added


def table(g, tokens, top_k, missing):
    pairs = tokens * top_k
    row_of = torch.randperm(pairs, generator=g, device="cuda").to(torch.int32)
    row_of[torch.rand(pairs, generator=g, device="cuda") < missing] = -1
    return row_of.view(tokens, top_k)


@pytest.mark.parametrize("tokens,top_k,width,pitch,kind", [(2000, 8, 4096, 4096, "bf16"), (5000, 8, 4090, 4096, "bf16"), (9000, 3, 3001, 3004, "f32"),
                                                           (30000, 10, 512, 512, "f16"), ((1 << 22) + 9, 2, 8, 8, "bf16")])
@pytest.mark.parametrize("weighted", [False, True])
def test_sums_and_their_gradients(lib, gpu, tokens, top_k, width, pitch, kind, weighted):
    dtype, code, u = TYPES[kind]
    g = gen(tokens)
    n = tokens * top_k
    row_of = table(g, tokens, top_k, 0.1)
    _, y = rows(g, n, width, dtype, pitch)
    _, add = rows(g, tokens, width, dtype, pitch)
    out_full, out = rows(g, tokens, width, dtype, pitch)
    drows_full, drows = rows(g, n, width, dtype, pitch)
    before = drows.clone()
    weight = torch.rand(tokens, top_k, generator=g, device="cuda") if weighted else None
    dweight = torch.zeros(tokens, top_k, device="cuda")
    assert lib.ofi_amd_token_combine(*where(y), n, ptr(row_of), ptr(weight), tokens, top_k, width, code, *where(add), *where(out),
                                     _gpu.stream()) == 0
    assert lib.ofi_amd_token_combine_grad(*where(add), *where(y), n, ptr(row_of), ptr(weight), tokens, top_k, width, code, *where(drows),
                                          ptr(dweight), _gpu.stream()) == 0
    _gpu.sync()
    if pitch > width:
        assert bool((out_full[:, width:] == 7).all()) and bool((drows_full[:, width:] == 7).all())
    named = torch.zeros(n, dtype=torch.bool, device="cuda")
    for lo, hi in parts(tokens, width * top_k):
        a64 = add[lo:hi].double()
        want, sizes = a64.clone(), a64.abs()
        for k in range(top_k):
            at = row_of[lo:hi, k].long()
            v = at >= 0
            w = weight[lo:hi, k].double() if weighted else torch.ones(hi - lo, dtype=torch.float64, device="cuda")
            term = torch.where(v[:, None], w[:, None] * y[at.clamp(min=0)].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
            want += term
            sizes += term.abs()
            d64 = (w[:, None] * a64)[v]
            close(drows[at[v]], d64, (u + 2 * U32) * d64.abs() + 2.0 ** -25)
            named[at[v]] = True
            dots = a64 * y[at.clamp(min=0)].double()
            zero = torch.zeros((), dtype=torch.float64, device="cuda")
            close(dweight[lo:hi, k], torch.where(v, dots.sum(dim=1), zero), (width / 64 + 30) * U32 * torch.where(v, dots.abs().sum(dim=1), zero))
        close(out[lo:hi], want, u * want.abs() + (top_k + 1) * U32 * sizes + 2.0 ** -25)
    assert torch.equal(drows[~named], before[~named])


@pytest.mark.parametrize("tokens,top_k,experts,row_bytes,scale_bytes", [(33000, 8, 256, 2048, 64), (70000, 8, 100, 512, 0), ((1 << 22) + 9, 2, 17, 16, 4),
                                                                        (1 << 20, 8, 1024, 16, 0)])
def test_sorts(lib, gpu, tokens, top_k, experts, row_bytes, scale_bytes):
    g = gen(tokens)
    pairs = tokens * top_k
    ids = torch.randint(-1, experts, (tokens, top_k), generator=g, device="cuda")
    x = torch.randint(0, 256, (tokens, row_bytes), generator=g, device="cuda", dtype=torch.uint8)
    sc = torch.randint(0, 256, (tokens, scale_bytes), generator=g, device="cuda", dtype=torch.uint8) if scale_bytes else None
    out = torch.full((pairs, row_bytes), 9, device="cuda", dtype=torch.uint8)
    sco = torch.full((pairs, scale_bytes), 9, device="cuda", dtype=torch.uint8) if scale_bytes else None
    offset = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    row_of, pair_of = torch.zeros(pairs, dtype=torch.int32, device="cuda"), torch.zeros(pairs, dtype=torch.int32, device="cuda")
    work = torch.empty(lib.ofi_amd_token_dispatch_work_bytes(tokens, top_k, experts), dtype=torch.uint8, device="cuda")
    two = lambda t: where(t) if t is not None else (None, 0)
    assert lib.ofi_amd_token_dispatch(ptr(ids), m.INT64, tokens, top_k, experts, pairs, ptr(offset), ptr(row_of), ptr(pair_of), *where(x),
                                      *where(out), row_bytes, *two(sc), *two(sco), scale_bytes, ptr(work), work.numel(), _gpu.stream()) == 0
    _gpu.sync()
    flat = ids.reshape(-1)
    valid = torch.nonzero(flat >= 0)[:, 0]
    order = valid[torch.sort(flat[valid], stable=True).indices]
    kept = order.numel()
    assert torch.equal(pair_of[:kept].long(), order) and bool((pair_of[kept:] == -1).all())
    assert torch.equal(row_of[order].long(), torch.arange(kept, device="cuda")) and bool((row_of[flat < 0] == -1).all())
    assert torch.equal(offset.long(), torch.searchsorted(flat[order], torch.arange(experts + 1, device="cuda")))
    assert torch.equal(out[:kept], x[order // top_k]) and bool((out[kept:] == 9).all())
    if sc is not None:
        assert torch.equal(sco[:kept], sc[order // top_k]) and bool((sco[kept:] == 9).all())
    assert _gpu.fetch_async_errors(lib) == 0
