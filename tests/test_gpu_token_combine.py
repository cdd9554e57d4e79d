"""ofi_amd_token_combine and its gradient against the formulas in 64 bits.

Bounds.  u is the unit roundoff of the rows' type, U = 2^-24.  A sum of K products and one addend takes K fused operations, each
with a rounding of at most U of the sum of sizes so far; the output adds u of itself.  A weight's gradient adds W products: at most
W / 64 a lane one after the other, then 6 + 16 more."""
import ctypes
import errno

import pytest
import torch

import _gpu
import aws_ofi_nccl_amd as m
from _rows import TYPES, U32, Rows, ptr, within

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def plan(g, tokens, top_k, max_rows, missing):
    """row_of with distinct rows; a `missing` share of the pairs has none, in several spellings."""
    pairs = tokens * top_k
    row_of = torch.full((pairs,), -1, dtype=torch.int64)
    order = torch.randperm(pairs, generator=g)
    n = min(max_rows, int(round(pairs * (1 - missing))))
    row_of[order[:n]] = torch.randperm(max_rows, generator=g)[:n] if max_rows else torch.zeros(0, dtype=torch.int64)
    odd = torch.tensor([-1, max_rows, max_rows + 5, 2 ** 31 - 1, -2 ** 31])
    none = row_of < 0
    row_of[none] = odd[torch.randint(0, 5, (int(none.sum()),), generator=g)]
    return row_of.view(tokens, top_k).to(torch.int32)


def combine(lib, rows, row_of, weight, width, kind, add, out, tokens=None, top_k=None, max_rows=None, stream=None):
    r = lambda t: (t.ptr(), t.pitch) if t is not None else (None, 0)
    return lib.ofi_amd_token_combine(*r(rows), rows.n if max_rows is None else max_rows, ptr(row_of), ptr(weight),
                                     row_of.shape[0] if tokens is None else tokens, row_of.shape[1] if top_k is None else top_k, width,
                                     TYPES[kind][1], *r(add), *r(out), _gpu.stream() if stream is None else stream)


def check_combine(lib, tokens, top_k, width, kind="bf16", missing=0.2, weighted=True, added=True, pad=0, shift=0, seed=1, max_rows=None,
                  in_place=False):
    g = gen(seed)
    dtype, _, u = TYPES[kind]
    max_rows = tokens * top_k if max_rows is None else max_rows
    row_of = plan(g, tokens, top_k, max_rows, missing)
    rows = Rows(max_rows, width, dtype, pad, shift, torch.randn(max_rows, width, generator=g, dtype=torch.float64))
    weight = torch.rand(tokens, top_k, generator=g) if weighted else None
    valid = (row_of >= 0) & (row_of < max_rows)
    if weighted:
        weight[~valid] = float("nan")                         # a pair without a row is not multiplied
    add = Rows(tokens, width, dtype, pad, shift, torch.randn(tokens, width, generator=g, dtype=torch.float64)) if added else None
    out = add if in_place else Rows(tokens, width, dtype, pad, shift)
    y = torch.cat([rows.t.double().cpu(), torch.zeros(1, width, dtype=torch.float64)])
    at = torch.where(valid, row_of.long(), torch.full_like(row_of, max_rows).long())
    w = torch.where(valid, weight.double() if weighted else torch.ones(tokens, top_k, dtype=torch.float64),
                    torch.zeros(tokens, top_k, dtype=torch.float64))
    a64 = add.t.double().cpu() if added else torch.zeros(tokens, width, dtype=torch.float64)
    want, sizes = a64.clone(), a64.abs()
    for k in range(top_k):
        term = w[:, k, None] * y[at[:, k]]
        want += term
        sizes += term.abs()
    d_row, d_weight = row_of.cuda(), weight.cuda() if weighted else None
    assert combine(lib, rows, d_row, d_weight, width, kind, add, out) == 0
    _gpu.sync()
    within(out.t, want, u * want.abs() + (top_k + 1) * U32 * sizes + 2.0 ** -25)
    assert out.untouched() and rows.untouched() and (add is None or add.untouched())


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("width", [1, 3, 7, 8, 9, 63, 64, 255, 256, 257, 511, 513, 1023, 1999, 2048, 4096, 4097, 9000, 40000])
def test_widths(lib, gpu, kind, width):
    check_combine(lib, 5, 8, width, kind, seed=width)
    check_combine(lib, 4, 3, width, kind, seed=width, pad=1, shift=3, weighted=False, added=False)


@pytest.mark.parametrize("top_k", [1, 2, 3, 4, 5, 6, 7, 8, 9, 15, 16, 17, 33, 64])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("added", [False, True])
def test_choices(lib, gpu, top_k, weighted, added):
    check_combine(lib, 21, top_k, 700, "bf16", weighted=weighted, added=added, seed=top_k)


@pytest.mark.parametrize("tokens", [1, 2, 255, 256, 257, 3001])
@pytest.mark.parametrize("missing", [0.0, 0.5, 0.9, 1.0])
def test_tokens_and_pairs_without_rows(lib, gpu, tokens, missing):
    check_combine(lib, tokens, 4, 264, "f16", missing=missing, seed=tokens, added=tokens % 2 == 0)


@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (4, 0), (1, 1), (5, 0)])
def test_pitches_and_alignments(lib, gpu, pad, shift):
    for kind in TYPES:
        check_combine(lib, 60, 6, 1160, kind, pad=pad, shift=shift)


@pytest.mark.parametrize("width", [5, 8, 100, 513, 1001, 2047, 4099])
@pytest.mark.parametrize("pad,shift", [(3, 1), (9, 0)])
def test_what_lies_beside_the_rows_does_not_reach_them(lib, gpu, monkeypatch, width, pad, shift):
    """Bytes of 0xff are NaN in every type."""
    monkeypatch.setattr(Rows, "guard", 0xFF)
    for kind in TYPES:
        check_combine(lib, 9, 5, width, kind, pad=pad, shift=shift, seed=width)
        check_grad(lib, 9, 5, width, kind, pad=pad, shift=shift, seed=width)
        check_grad(lib, 9, 5, width, kind, pad=pad, shift=shift, seed=width, in_place=True, missing=0.0)


@pytest.mark.parametrize("top_k", [1, 2])
@pytest.mark.parametrize("width", [1, 7, 8, 9, 255, 257, 1024, 2049, 4224, 8191, 16385, 20000, 40000])
def test_one_and_two_rows_of_a_token(lib, gpu, monkeypatch, width, top_k):
    monkeypatch.setattr(Rows, "guard", 0xFF)
    for kind in TYPES:
        check_combine(lib, 13, top_k, width, kind, seed=width)
        check_combine(lib, 6, top_k, width, kind, seed=width, pad=3, shift=1, weighted=False, added=False)
        check_combine(lib, 6, top_k, width, kind, seed=width, pad=3, shift=1, in_place=True, missing=0.5)


def test_the_output_may_replace_the_addend(lib, gpu):
    check_combine(lib, 33, 8, 1025, "bf16", in_place=True)


def test_no_rows_and_no_tokens(lib, gpu):
    check_combine(lib, 7, 3, 100, max_rows=0)
    row_of = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    rows = Rows(4, 8, torch.bfloat16)
    assert combine(lib, rows, row_of, None, 8, "bf16", None, rows) == 0


def test_rows_far_apart_pass_32_bits_of_offset(lib, gpu):
    pitch, n, width = 1 << 28, 20, 600
    g = gen(6)
    v = torch.randn(n, width, generator=g).to(torch.bfloat16)
    far = torch.zeros(n * pitch, dtype=torch.uint8, device="cuda")
    for k in range(n):
        far[k * pitch:k * pitch + 2 * width].view(torch.bfloat16).copy_(v[k])
    row_of = torch.randperm(n, generator=g).to(torch.int32).view(10, 2).cuda()
    out = Rows(10, width, torch.bfloat16)
    assert lib.ofi_amd_token_combine(ptr(far), pitch, n, ptr(row_of), None, 10, 2, width, m.BFLOAT16, None, 0, out.ptr(), out.pitch,
                                     _gpu.stream()) == 0
    _gpu.sync()
    want = v.double()[row_of.cpu().long()].sum(dim=1)
    within(out.t, want, 2.0 ** -8 * want.abs() + 4 * U32 * v.double().abs()[row_of.cpu().long()].sum(dim=1))


def grad(lib, dout, rows, row_of, weight, width, kind, drows, dweight, max_rows=None, tokens=None, top_k=None):
    r = lambda t: (t.ptr(), t.pitch) if t is not None else (None, 0)
    return lib.ofi_amd_token_combine_grad(*r(dout), *r(rows), (rows or drows).n if max_rows is None else max_rows, ptr(row_of), ptr(weight),
                                          row_of.shape[0] if tokens is None else tokens, row_of.shape[1] if top_k is None else top_k, width,
                                          TYPES[kind][1], *r(drows), ptr(dweight), _gpu.stream())


def check_grad(lib, tokens, top_k, width, kind="bf16", missing=0.2, weighted=True, pad=0, shift=0, seed=1, max_rows=None, want_rows=True,
               want_weight=True, in_place=False):
    g = gen(seed)
    dtype, _, u = TYPES[kind]
    max_rows = tokens * top_k if max_rows is None else max_rows
    row_of = plan(g, tokens, top_k, max_rows, missing)
    valid = (row_of >= 0) & (row_of < max_rows)
    rows = Rows(max_rows, width, dtype, pad, shift, torch.randn(max_rows, width, generator=g, dtype=torch.float64))
    dout = Rows(tokens, width, dtype, pad, shift, torch.randn(tokens, width, generator=g, dtype=torch.float64))
    weight = torch.rand(tokens, top_k, generator=g) if weighted else None
    if weighted:
        weight[~valid] = float("nan")
    y64, d64 = rows.t.double().cpu(), dout.t.double().cpu()
    w64 = weight.double() if weighted else torch.ones(tokens, top_k, dtype=torch.float64)
    drows = rows if in_place else Rows(max_rows, width, dtype, pad, shift)
    before = drows.t.clone()
    dweight = torch.full((tokens * top_k + 1,), 9.0, device="cuda")
    assert grad(lib, dout, rows, row_of.cuda(), weight.cuda() if weighted else None, width, kind, drows if want_rows else None,
                dweight if want_weight else None) == 0
    _gpu.sync()
    at = row_of.long()
    if want_rows:
        named = torch.zeros(max_rows, dtype=torch.bool)
        want = torch.zeros(max_rows, width, dtype=torch.float64)
        t, k = torch.nonzero(valid, as_tuple=True)
        want[at[t, k]] = w64[t, k, None] * d64[t]
        named[at[t, k]] = True
        within(drows.t[named.cuda()], want[named], (u + 2 * U32) * want[named].abs() + 2.0 ** -25)
        assert torch.equal(drows.t[~named.cuda()].view(torch.uint8), before[~named.cuda()].view(torch.uint8)) and drows.untouched()
    if want_weight:
        want, sizes = torch.zeros(tokens, top_k, dtype=torch.float64), torch.zeros(tokens, top_k, dtype=torch.float64)
        for k in range(top_k):
            v = valid[:, k]
            term = d64[v] * y64[at[v, k]]
            want[v, k], sizes[v, k] = term.sum(dim=1), term.abs().sum(dim=1)
        within(dweight[:-1].view(tokens, top_k), want, (width / 64 + 30) * U32 * sizes)
        assert float(dweight[-1]) == 9.0
    assert dout.untouched() and rows.untouched()
    return dict(d64=d64, y64=y64, w64=w64, at=at, valid=valid, drows=drows.t.double().cpu(), dweight=dweight[:-1].double().cpu())


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("width", [1, 3, 8, 9, 64, 255, 256, 257, 512, 513, 1999, 2048, 2049, 4096, 5000, 9001, 40000])
def test_gradient_widths(lib, gpu, kind, width):
    check_grad(lib, 6, 8, width, kind, seed=width)
    check_grad(lib, 3, 5, width, kind, seed=width, pad=1, shift=1, weighted=False)


@pytest.mark.parametrize("width", [1, 7, 8, 9, 257, 1024, 2049, 4224, 8191, 16385, 40000])
def test_gradient_of_one_row_of_a_token(lib, gpu, monkeypatch, width):
    monkeypatch.setattr(Rows, "guard", 0xFF)
    for kind in TYPES:
        check_grad(lib, 13, 1, width, kind, seed=width)
        check_grad(lib, 6, 1, width, kind, seed=width, pad=3, shift=1, weighted=False)
        check_grad(lib, 6, 1, width, kind, seed=width, pad=3, shift=1, in_place=True, missing=0.0)


@pytest.mark.parametrize("top_k", [1, 2, 3, 4, 5, 6, 7, 8, 9, 16, 17, 31, 64])
@pytest.mark.parametrize("tokens", [1, 19, 2600])
def test_gradient_choices(lib, gpu, top_k, tokens):
    check_grad(lib, tokens, top_k, 200 if tokens > 100 else 2100, "bf16", seed=top_k, weighted=top_k % 2 == 0)


@pytest.mark.parametrize("missing", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (3, 0), (0, 1)])
def test_gradient_missing_rows_pitches_and_alignments(lib, gpu, missing, pad, shift):
    check_grad(lib, 300, 6, 520, "f16", missing=missing, pad=pad, shift=shift)


def test_gradient_parts_and_in_place(lib, gpu):
    check_grad(lib, 50, 8, 1030, want_rows=False)
    check_grad(lib, 50, 8, 1030, want_weight=False)
    check_grad(lib, 50, 8, 1030, in_place=True)
    check_grad(lib, 50, 17, 1030, in_place=True)
    check_grad(lib, 7, 3, 100, max_rows=0)


def test_gradient_against_differences(lib, gpu):
    """d/de of sum(dout * out(rows + e a, weight + e b)) by central differences of the formula in 64 bits."""
    got = check_grad(lib, 9, 5, 333, "f32", seed=4)
    g = gen(70)
    valid, at = got["valid"], got["at"]
    a = torch.randn(got["y64"].shape, generator=g, dtype=torch.float64)
    b = torch.randn(9, 5, generator=g, dtype=torch.float64)

    def loss(e_a, e_b):
        y, w = got["y64"] + e_a * a, got["w64"] + e_b * b
        out = torch.zeros_like(got["d64"])
        for k in range(5):
            v = valid[:, k]
            out[v] += w[v, k, None] * y[at[v, k]]
        return (got["d64"] * out).sum().item()

    e = 1e-4
    named = torch.zeros(got["y64"].shape[0], dtype=torch.bool)
    named[at[valid]] = True
    by_rows, by_weight = (loss(e, 0) - loss(-e, 0)) / (2 * e), (loss(0, e) - loss(0, -e)) / (2 * e)
    terms = (got["drows"] * a)[named]
    assert abs(by_rows - terms.sum().item()) <= 1e-6 * terms.abs().sum().item()
    terms = got["dweight"] * b.reshape(-1)
    assert abs(by_weight - terms.sum().item()) <= 1e-6 * terms.abs().sum().item()


def test_the_gradient_of_dispatch_is_the_sum_without_weights(lib, gpu):
    """Rows copied by ofi_amd_token_dispatch; the gradient of the tokens adds up the gradients of their rows."""
    g = gen(9)
    tokens, top_k, experts, width = 50, 4, 12, 96
    ids = torch.randint(-1, experts, (tokens, top_k), generator=g).cuda()
    x = torch.randn(tokens, width, generator=g).cuda()
    offset = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    row_of = torch.zeros(tokens, top_k, dtype=torch.int32, device="cuda")
    rows = torch.zeros(tokens * top_k, width, device="cuda")
    need = lib.ofi_amd_token_dispatch_work_bytes(tokens, top_k, experts)
    work = torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")
    assert lib.ofi_amd_token_dispatch(ptr(ids), m.INT64, tokens, top_k, experts, tokens * top_k, ptr(offset), ptr(row_of), None, ptr(x),
                                      4 * width, ptr(rows), 4 * width, 4 * width, None, 0, None, 0, 0, ptr(work), work.numel(),
                                      _gpu.stream()) == 0
    drows = torch.randn(tokens * top_k, width, generator=g).cuda()
    dx = torch.zeros(tokens, width, device="cuda")
    assert lib.ofi_amd_token_combine(ptr(drows), 4 * width, tokens * top_k, ptr(row_of), None, tokens, top_k, width, m.FLOAT32, None, 0,
                                     ptr(dx), 4 * width, _gpu.stream()) == 0
    _gpu.sync()
    # <drows, dispatch(x)> = <dx, x>: the two maps are each other's transpose
    n = int(offset[experts])
    left = (drows[:n].double() * rows[:n].double()).sum().item()
    right = (dx.double() * x.double()).sum().item()
    assert abs(left - right) <= 8 * U32 * (drows[:n].double() * rows[:n].double()).abs().sum().item()


def test_the_same_call_gives_the_same_bits_on_any_stream_and_in_a_replayed_graph(lib, gpu):
    g = gen(3)
    tokens, top_k, width = 700, 8, 1000
    row_of = plan(g, tokens, top_k, tokens * top_k, 0.1).cuda()
    weight = torch.rand(tokens, top_k, generator=g).cuda()
    rows = Rows(tokens * top_k, width, torch.bfloat16, values=torch.randn(tokens * top_k, width, generator=g))
    dout = Rows(tokens, width, torch.bfloat16, values=torch.randn(tokens, width, generator=g))
    out, drows = Rows(tokens, width, torch.bfloat16), Rows(tokens * top_k, width, torch.bfloat16)
    dweight = torch.zeros(tokens, top_k, device="cuda")

    def both():
        assert combine(lib, rows, row_of, weight, width, "bf16", None, out) == 0
        assert grad(lib, dout, rows, row_of, weight, width, "bf16", drows, dweight) == 0

    def seen():
        _gpu.sync()
        got = [out.t.clone(), drows.t.clone(), dweight.clone()]
        for t in (out.t, drows.t, dweight):
            t.zero_()
        _gpu.sync()
        return got

    drows.t.zero_()
    both()
    first = seen()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both()
    assert all(torch.equal(a, b) for a, b in zip(first, seen()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(first, seen()))
        both()
        assert all(torch.equal(a, b) for a, b in zip(first, seen()))


def test_refusals(lib, gpu):
    inval, toobig = -errno.EINVAL, -errno.E2BIG
    rows, out = Rows(32, 64, torch.bfloat16, values=torch.ones(32, 64)), Rows(4, 64, torch.bfloat16)
    row_of = torch.arange(32, dtype=torch.int32, device="cuda").view(4, 8)
    weight = torch.ones(4, 8, device="cuda")
    call = lambda **k: combine(lib, k.pop("rows", rows), k.pop("row_of", row_of), k.pop("weight", weight), k.pop("width", 64),
                               k.pop("kind", "bf16"), k.pop("add", None), k.pop("out", out), **k)
    assert call() == 0
    assert call(width=0) == inval and call(top_k=0) == inval and call(width=65) == inval and call(out=None) == inval
    assert call(width=(1 << 20) + 1) == toobig and call(top_k=65) == toobig and call(max_rows=1 << 31) == toobig
    assert call(tokens=1 << 29) == toobig
    vp = ctypes.c_void_p
    raw = lambda rp, row_p, w_p, kind=m.BFLOAT16, pitch=128: lib.ofi_amd_token_combine(
        vp(rp), pitch, 32, vp(row_p), vp(w_p), 4, 8, 64, kind, None, 0, out.ptr(), out.pitch, _gpu.stream())
    good = (rows.ptr(), row_of.data_ptr(), weight.data_ptr())
    assert raw(*good) == 0 and raw(*good, kind=m.INT32) == inval and raw(*good, pitch=126) == inval and raw(*good, pitch=129) == inval
    assert raw(None, *good[1:]) == inval and raw(good[0], None, good[2]) == inval and raw(good[0] + 1, *good[1:]) == inval
    assert raw(good[0], good[1] + 2, good[2]) == inval and raw(good[0], good[1], good[2] + 1) == inval
    dweight, drows = torch.zeros(4, 8, device="cuda"), Rows(32, 64, torch.bfloat16)
    back = lambda **k: grad(lib, k.pop("dout", out), k.pop("rows", rows), row_of, weight, k.pop("width", 64), "bf16", k.pop("drows", drows),
                            k.pop("dweight", dweight), max_rows=k.pop("max_rows", 32), **k)
    assert back() == 0
    assert back(drows=None, dweight=None) == inval and back(dout=None) == inval and back(rows=None) == inval
    assert back(rows=None, dweight=None) == 0 and back(width=0) == inval and back(top_k=65) == toobig and back(max_rows=1 << 31) == toobig
    _gpu.sync()
    assert _gpu.fetch_async_errors(lib) == 0
