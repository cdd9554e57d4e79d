"""The experts' products for tests: calls of the library, the formulas in 64 bits, and how far a result may be from them.

Bounds.  u is the unit roundoff of an output's type, U = 2^-24.  A sum of K products in 32 bits, in whatever order and with steps that may cut
off instead of round, is off by at most 2 (K + 4) U times the sum of the products' sizes (`sizes`).  The activations are off by at most
(24 + 4 |v| + v^2) U of the larger of 1 and |v| (an exponential's argument is rounded, a fit is 5e-7 = 8.4 U off, two dozen operations),
and carry what their argument is off by with a slope below 1.2.  8-bit values are off by half a step: 2^-4 of the value, or
2^-10 of the scale where they are subnormal."""
import ctypes
import math

import torch

import _gpu
import aws_ofi_nccl_amd as m
from _rows import U32, Rows, within

KIND = {"bf16": (torch.bfloat16, m.BFLOAT16, 2.0 ** -8), "f16": (torch.float16, m.FLOAT16, 2.0 ** -11),
        "f32": (torch.float32, m.FLOAT32, 2.0 ** -24), "e4m3": (torch.float8_e4m3fn, m.E4M3, 2.0 ** -4)}
ACT = {"none": m.NO_ACTIVATION, "relu": m.RELU, "silu": m.SILU, "gelu": m.GELU}
TINY = 2.0 ** -24  # subnormal float16 results, half a step


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def blocks(n):
    return -(-n // 128)


def rnd(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float64)


def to_type(v, kind):
    return v.clamp(-448, 448).to(torch.float32).to(KIND[kind][0]) if kind == "e4m3" else v.to(KIND[kind][0])


class Matrix:
    """Rows (with guards around) of values in 64 bits as a type holds them, with scales for e4m3 in `parts` equal runs of columns."""

    def __init__(self, n, width, kind, pad=0, shift=0, values=None, parts=1, scale=None):
        self.kind, self.parts, self.width = kind, parts, width
        self.rows = Rows(n, width, KIND[kind][0], pad, shift)
        self.scales = Rows(n, parts * blocks(width // parts), torch.float32, 1 if pad else 0) if kind == "e4m3" else None
        if values is not None and n:
            self.rows.t.view(torch.uint8).copy_(to_type(values, kind).view(torch.uint8)) if kind == "e4m3" else self.rows.t.copy_(to_type(values, kind))
            if scale is not None:
                self.scales.t.copy_(scale)

    def args(self):
        return self.rows.ptr(), self.rows.pitch

    def scale_args(self):
        return (self.scales.ptr(), self.scales.pitch) if self.scales else (None, 0)

    def spread(self):
        n = self.width // self.parts
        s = self.scales.t.double()
        b = blocks(n)
        return torch.cat([s[:, p * b:(p + 1) * b].repeat_interleave(128, dim=1)[:, :n] for p in range(self.parts)], dim=1)

    def values(self):
        v = self.rows.t.float().double()
        return v * self.spread() if self.scales else v

    def untouched(self):
        return self.rows.untouched() and (self.scales is None or self.scales.untouched())


class Weights:
    """[experts, parts * n, width] with `pad` elements from row to row and `apart` more rows' worth from expert to expert."""

    def __init__(self, g, experts, parts, n, width, kind, pad=0, apart=0):
        self.kind, self.shape = kind, (experts, parts, n, width)
        total = parts * n
        v = rnd(g, experts * (total + apart), width) * (130.0 if kind == "e4m3" else width ** -0.5)
        self.m = Rows(experts * (total + apart), width, KIND[kind][0], pad)
        self.m.t.view(torch.uint8).copy_(to_type(v, kind).view(torch.uint8)) if kind == "e4m3" else self.m.t.copy_(to_type(v, kind))
        self.expert_pitch = (total + apart) * self.m.pitch
        self.scale = ((torch.rand(experts, parts, blocks(n), blocks(width), generator=g, device="cuda") + 0.5) * width ** -0.5 / 130.0
                      if kind == "e4m3" else None)
        self.total, self.apart = total, apart

    def args(self):
        return self.m.ptr(), self.m.pitch, self.expert_pitch

    def scale_ptr(self):
        return self.scale.data_ptr() if self.scale is not None else None

    def values(self, e):
        experts, parts, n, width = self.shape
        at = e * (self.total + self.apart)
        v = self.m.t[at:at + self.total].float().double()
        if self.scale is not None:
            s = self.scale[e].double().repeat_interleave(128, dim=1)[:, :n].reshape(self.total, -1)
            v = v * s.repeat_interleave(128, dim=1)[:, :width]
        return v


def offsets(first, counts):
    at = [first]
    for c in counts:
        at.append(at[-1] + c)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def runs(offset, max_rows, experts):
    at = [0, max_rows] if offset is None else [min(max(int(v), 0), max_rows) for v in offset.cpu()]
    return [(e, at[e], at[e + 1]) for e in range(experts) if at[e + 1] > at[e]]


def act(kind, v):
    if kind == "none":
        return v, torch.ones_like(v)
    if kind == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v), torch.where(v > 0, 1.0, 0.0).double()
    if kind == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    share = 0.5 * torch.special.erfc(-v * math.sqrt(0.5))
    return v * share, share + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)


def act_error(kind, v):
    if kind in ("none", "relu"):
        return torch.zeros_like(v)
    return (24 + 4 * v.abs() + v * v) * U32 * v.abs().clamp(min=1)


def sum_error(k, sizes):
    return 2 * (k + 4) * U32 * sizes


def check_output(out, lo, hi, want, error, parts=1):
    """Rows [lo, hi) of an output against values in 64 bits that 32 bits may miss by `error`."""
    kind = out.kind
    u = KIND[kind][2]
    if kind != "e4m3":
        within(out.rows.t[lo:hi], want, error + u * (want.abs() + error) + TINY)
        return
    n, b = want.shape[1] // parts, blocks(want.shape[1] // parts)
    for p in range(parts):
        for j in range(b):
            at = slice(p * n + 128 * j, p * n + min(128 * (j + 1), n))
            big, off = want[:, at].abs().amax(dim=1), error[:, at].amax(dim=1)
            scale = out.scales.t[lo:hi, p * b + j].double()
            nan = torch.isnan(want[:, at]).any(dim=1)
            target = torch.where(nan, torch.full_like(big, float("nan")), (big / 448).clamp(min=2.0 ** -126))
            within(scale, target, off / 448 + 2 * U32 * target)
            got = out.rows.t[lo:hi, at].float().double() * scale[:, None]
            within(got[~nan], want[:, at][~nan], (error[:, at] + u * (want[:, at].abs() + error[:, at]) + 2.0 ** -10 * scale[:, None] +
                                                  4 * U32 * want[:, at].abs())[~nan])


def scaled_values(g, n, width, kind, parts=1):
    """(values, scales) of an input."""
    if kind != "e4m3":
        return rnd(g, n, width), None
    return rnd(g, n, width) * 130.0, (torch.rand(n, parts * blocks(width // parts), generator=g, device="cuda") + 0.5) / 130.0


def stream_of(stream):
    return _gpu.stream() if stream is None else stream


def gated(lib, x, w, offset, experts, max_rows, width, inner, a, out, saved=None, stream=None):
    return lib.ofi_amd_expert_gated(*x.args(), *x.scale_args(), KIND[x.kind][1], offset.data_ptr() if offset is not None else None, experts,
                                    max_rows, *w.args(), w.scale_ptr(), width, inner, ACT[a], *out.args(), KIND[out.kind][1],
                                    *out.scale_args(), *(saved.args() if saved else (None, 0)), KIND[saved.kind][1] if saved else 0,
                                    *(saved.scale_args() if saved else (None, 0)), stream_of(stream))


def product(lib, x, w, offset, experts, max_rows, width, n, a, out, bias=None, residual=None, saved=None, stream=None):
    types = {torch.float32: m.FLOAT32, torch.float16: m.FLOAT16, torch.bfloat16: m.BFLOAT16}
    return lib.ofi_amd_expert_product(*x.args(), *x.scale_args(), KIND[x.kind][1], offset.data_ptr() if offset is not None else None, experts,
                                      max_rows, *w.args(), w.scale_ptr(), width, n, bias.data_ptr() if bias is not None else None,
                                      types[bias.dtype] if bias is not None else 0, ACT[a], *(residual.args() if residual else (None, 0)),
                                      *out.args(), KIND[out.kind][1], *out.scale_args(), *(saved.args() if saved else (None, 0)),
                                      KIND[saved.kind][1] if saved else 0, *(saved.scale_args() if saved else (None, 0)), stream_of(stream))


def hidden_grad(lib, dout, w, offset, experts, max_rows, width, inner, is_gated, a, saved, dsaved, hidden=None, stream=None):
    return lib.ofi_amd_expert_hidden_grad(*dout.args(), KIND[dout.kind][1], offset.data_ptr() if offset is not None else None, experts, max_rows,
                                          *w.args(), width, inner, int(is_gated), ACT[a], *saved.args(), KIND[saved.kind][1],
                                          *saved.scale_args(), *dsaved.args(), *(hidden.args() if hidden else (None, 0)), stream_of(stream))


def rows_grad(lib, dout, w, offset, experts, max_rows, width, n, drows, add=None, stream=None):
    return lib.ofi_amd_expert_rows_grad(*dout.args(), KIND[dout.kind][1], offset.data_ptr() if offset is not None else None, experts, max_rows,
                                        *w.args(), width, n, *(add.args() if add else (None, 0)), *drows.args(), stream_of(stream))


def weight_grad(lib, dout, x, offset, experts, max_rows, width, n, dw, expert_pitch, add=None, dbias=None, bias_add=None, stream=None):
    return lib.ofi_amd_expert_weight_grad(*dout.args(), *x.args(), KIND[x.kind][1], offset.data_ptr() if offset is not None else None, experts,
                                          max_rows, width, n, add.rows.ptr() if add else None, *dw.args(), expert_pitch, KIND[dw.kind][1],
                                          bias_add.data_ptr() if bias_add is not None else None,
                                          dbias.data_ptr() if dbias is not None else None, stream_of(stream))


def left_alone(out, offset, max_rows, experts):
    """Rows that no expert has are as they were: guard bytes."""
    at = [0, max_rows] if offset is None else [min(max(int(v), 0), max_rows) for v in offset.cpu()]
    for r in (out.rows, out.scales):
        if r is None or r.n == 0:
            continue
        t = r.t.view(torch.uint8) if r.size == 1 else r.t.view(torch.uint8).view(r.t.shape[0], -1)
        if not bool((t[:at[0]] == r.guard).all()) or not bool((t[at[-1]:] == r.guard).all()):
            return False
    return True


def check_gated(lib, counts, width, inner, kind="bf16", out_kind=None, saved_kind=None, a="silu", first=0, spare=0, pad=0, shift=0, apart=0, seed=1,
                dense=False, bad=None):
    g = gen(seed)
    out_kind = out_kind or kind
    experts, max_rows = len(counts), first + sum(counts) + spare
    offset = None if dense else offsets(first, counts)
    values, scale = scaled_values(g, max_rows, width, kind)
    if bad:
        bad(values, offset)
    x = Matrix(max_rows, width, kind, pad, shift, values, scale=scale)
    w = Weights(g, experts, 2, inner, width, kind, pad, apart)
    out = Matrix(max_rows, inner, out_kind, pad, shift)
    saved = Matrix(max_rows, 2 * inner, saved_kind, pad, shift, parts=2) if saved_kind else None
    assert gated(lib, x, w, offset, experts, max_rows, width, inner, a, out, saved) == 0
    _gpu.sync()
    for e, lo, hi in runs(offset, max_rows, experts):
        v, wv = x.values()[lo:hi], w.values(e)
        both, off = v @ wv.t().contiguous(), sum_error(width, v.abs() @ wv.abs().t().contiguous())
        gate, up, dg, du = both[:, :inner], both[:, inner:], off[:, :inner], off[:, inner:]
        value = act(a, gate)[0]
        da = act_error(a, gate) + 1.2 * dg
        want = value * up
        check_output(out, lo, hi, want, da * (up.abs() + du) + value.abs() * du + 2 * U32 * want.abs())
        if saved:
            check_output(saved, lo, hi, both, off, 2)
    assert out.untouched() and x.untouched() and w.m.untouched() and (not saved or saved.untouched())
    assert left_alone(out, offset, max_rows, experts) and (not saved or left_alone(saved, offset, max_rows, experts))
    return out


def check_product(lib, counts, width, n, kind="bf16", out_kind=None, saved_kind=None, a="none", bias_type=None, residual=False, first=0, spare=0, pad=0,
                  shift=0, apart=0, seed=1, dense=False, in_place=False):
    g = gen(seed)
    out_kind = out_kind or (kind if kind != "e4m3" else "bf16")
    experts, max_rows = len(counts), first + sum(counts) + spare
    offset = None if dense else offsets(first, counts)
    values, scale = scaled_values(g, max_rows, width, kind)
    x = Matrix(max_rows, width, kind, pad, shift, values, scale=scale)
    w = Weights(g, experts, 1, n, width, kind, pad, apart)
    res = Matrix(max_rows, n, out_kind, pad, shift, rnd(g, max_rows, n)) if residual else None
    res_was = res.values().clone() if res else None
    out = res if in_place else Matrix(max_rows, n, out_kind, pad, shift)
    saved = Matrix(max_rows, n, saved_kind, pad, shift) if saved_kind else None
    bias = rnd(g, experts, n).to(bias_type) if bias_type else None
    assert product(lib, x, w, offset, experts, max_rows, width, n, a, out, bias, res, saved) == 0
    _gpu.sync()
    for e, lo, hi in runs(offset, max_rows, experts):
        v, wv = x.values()[lo:hi], w.values(e)
        pre, off = v @ wv.t().contiguous(), sum_error(width, v.abs() @ wv.abs().t().contiguous())
        if bias is not None:
            pre = pre + bias[e].double()
            off = off + U32 * (pre.abs() + off)
        value = act(a, pre)[0]
        da = act_error(a, pre) + (1.2 if a != "none" else 1.0) * off
        want = value if res is None else value + res_was[lo:hi]
        check_output(out, lo, hi, want, da + U32 * (want.abs() + da))
        if saved:
            check_output(saved, lo, hi, pre, off)
    assert out.untouched() and x.untouched() and w.m.untouched() and (not saved or saved.untouched())
    assert in_place or left_alone(out, offset, max_rows, experts)
    return out


def check_hidden(lib, counts, width, inner, kind="bf16", saved_kind=None, is_gated=True, a="silu", first=0, spare=0, pad=0, shift=0, apart=0, seed=1,
                 dense=False, with_hidden=True):
    g = gen(seed)
    saved_kind = saved_kind or kind
    parts = 2 if is_gated else 1
    experts, max_rows = len(counts), first + sum(counts) + spare
    offset = None if dense else offsets(first, counts)
    dout = Matrix(max_rows, width, kind, pad, shift, rnd(g, max_rows, width))
    w = Weights(g, experts, 1, width, inner, kind, pad, apart)
    values, scale = scaled_values(g, max_rows, parts * inner, saved_kind, parts)
    saved = Matrix(max_rows, parts * inner, saved_kind, pad, shift, values, parts, scale)
    dsaved = Matrix(max_rows, parts * inner, kind, pad, shift)
    hidden = Matrix(max_rows, inner, kind, pad, shift) if with_hidden else None
    assert hidden_grad(lib, dout, w, offset, experts, max_rows, width, inner, is_gated, a, saved, dsaved, hidden) == 0
    _gpu.sync()
    for e, lo, hi in runs(offset, max_rows, experts):
        d, wv, kept = dout.values()[lo:hi], w.values(e), saved.values()[lo:hi]
        dh, off = d @ wv, sum_error(width, d.abs() @ wv.abs())
        gate = kept[:, :inner]
        value, slope = act(a, gate)
        ea = act_error(a, gate) + 2 * U32 * gate.abs()
        es = ea * (1 + gate.abs())
        up = kept[:, inner:] if is_gated else torch.ones_like(gate)
        want = dh * up * slope
        error = off * (up * slope).abs() + (dh.abs() + off) * up.abs() * es + 6 * U32 * want.abs()
        if is_gated:
            du = dh * value
            want, error = torch.cat([want, du], dim=1), torch.cat([error, off * value.abs() + (dh.abs() + off) * ea + 4 * U32 * du.abs()], dim=1)
        check_output(dsaved, lo, hi, want, error)
        if hidden:
            h = value * up
            check_output(hidden, lo, hi, h, ea * up.abs() + 4 * U32 * h.abs())
    assert dsaved.untouched() and saved.untouched() and dout.untouched() and (not hidden or hidden.untouched())
    assert left_alone(dsaved, offset, max_rows, experts) and (not hidden or left_alone(hidden, offset, max_rows, experts))


def check_rows(lib, counts, width, n, kind="bf16", added=False, in_place=False, first=0, spare=0, pad=0, shift=0, apart=0, seed=1, dense=False):
    g = gen(seed)
    experts, max_rows = len(counts), first + sum(counts) + spare
    offset = None if dense else offsets(first, counts)
    dout = Matrix(max_rows, n, kind, pad, shift, rnd(g, max_rows, n))
    w = Weights(g, experts, 1, n, width, kind, pad, apart)
    add = Matrix(max_rows, width, kind, pad, shift, rnd(g, max_rows, width)) if added else None
    was = add.values().clone() if add else None
    drows = add if in_place else Matrix(max_rows, width, kind, pad, shift)
    assert rows_grad(lib, dout, w, offset, experts, max_rows, width, n, drows, add) == 0
    _gpu.sync()
    for e, lo, hi in runs(offset, max_rows, experts):
        d, wv = dout.values()[lo:hi], w.values(e)
        want, off = d @ wv, sum_error(n, d.abs() @ wv.abs())
        if add:
            want = want + was[lo:hi]
        check_output(drows, lo, hi, want, off + U32 * (want.abs() + off))
    assert drows.untouched() and dout.untouched() and (in_place or left_alone(drows, offset, max_rows, experts))


def check_weights(lib, counts, width, n, kind="bf16", out_kind="f32", added=False, in_place=False, bias=False, first=0, spare=0, pad=0, shift=0, apart=0,
                  seed=1, dense=False):
    g = gen(seed)
    experts, max_rows = len(counts), first + sum(counts) + spare
    offset = None if dense else offsets(first, counts)
    dout = Matrix(max_rows, n, kind, pad, shift, rnd(g, max_rows, n))
    x = Matrix(max_rows, width, kind, pad, shift, rnd(g, max_rows, width))
    each = n + apart
    add = Matrix(experts * each, width, out_kind, pad, shift, rnd(g, experts * each, width)) if added else None
    was = add.values().clone() if add else None
    dw = add if in_place else Matrix(experts * each, width, out_kind, pad, shift)
    dbias = torch.full((experts, n), 7.0, device="cuda") if bias else None
    bias_add = rnd(g, experts, n).float() if bias and added else None
    assert weight_grad(lib, dout, x, offset, experts, max_rows, width, n, dw, each * dw.rows.pitch, add, dbias, bias_add) == 0
    _gpu.sync()
    at = [0, max_rows] if offset is None else [int(v) for v in offset.cpu()]
    for e in range(experts):
        d, v = dout.values()[at[e]:at[e + 1]], x.values()[at[e]:at[e + 1]]
        rows = d.shape[0]
        want, off = d.t().contiguous() @ v, sum_error(rows, d.abs().t().contiguous() @ v.abs())
        if add:
            want = want + was[e * each:e * each + n]
        check_output(dw, e * each, e * each + n, want, off + U32 * (want.abs() + off))
        if bias:
            b, boff = d.sum(dim=0), sum_error(rows, d.abs().sum(dim=0))
            if bias_add is not None:
                b = b + bias_add[e].double()
            within(dbias[e], b, boff + U32 * (b.abs() + boff))
    assert dw.untouched() and dout.untouched() and x.untouched()
