"""The activations where they are small: errors relative to the value, far out where it is a tiny part of its argument.

An 8-bit output's scale is the largest of its block of 128 columns, divided by 448, in 32 bits: a block with a single value shows that value with
all of its bits, whichever way a product of rows goes.  The product's sums are zeros, the values come as its bias.

Bounds, in units of U = 2^-24, for v * share, share = e^(-v^2/2) t P(t) below 0, t = 1 / (1 + 0.45 |v| / sqrt 2): t 4 (its constant, an fma, a
reciprocal off by 2) times t P's sensitivity to it, 2.51 at most; P's coefficients 1.73 and its roundings 2.94, sums of sizes over the value, at
t = 1; the fit 0.5; the power 2; three products and the scale's division 4: 21.2, so 24.  Besides, v^2/2 is rounded, and its product with
log2(e), whose constant is 0.2 off: 2.2 times v^2/2.  Above 0 the share is 1 minus that, off by no more.  For v / (1 + e^-v): the exponent's
rounding and its constant's 1.2 |v|, the power 2, the sum 1, the reciprocal 2, the product and the division 2: 8 + 2 |v|."""
import pytest
import torch

import _gpu
from _experts import Matrix, Weights, act, gen, hidden_grad, product
from _rows import U32, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("a,low,high", [("gelu", -12.0, 9.0), ("silu", -75.0, 75.0)])
@pytest.mark.parametrize("kind", ["f16", "e4m3"])
@pytest.mark.parametrize("rows", [1, 70])
def test_values_relative_to_themselves(lib, gpu, a, low, high, kind, rows):
    """One row: streams of weights; 70: tiles.  1024 arguments, even over the range and around 0."""
    parts, width = 1024, 16
    n = 128 * parts
    g = gen(parts + rows)
    v = torch.cat([torch.linspace(low, high, parts - 128, device="cuda"), torch.linspace(-1, 1, 128, device="cuda")]).float()
    bias = torch.zeros(n, device="cuda")
    bias[::128] = v
    x = Matrix(rows, width, kind, values=torch.zeros(rows, width, device="cuda"), 
               scale=torch.ones(rows, 1, device="cuda") if kind == "e4m3" else None)
    out = Matrix(rows, n, "e4m3")
    assert product(lib, x, Weights(g, 1, 1, n, width, kind), None, 1, rows, width, n, a, out, bias=bias) == 0
    _gpu.sync()
    want = act(a, v.double())[0].abs()
    assert want.max() > 1 and want[want > 0].min() < 1e-20
    units = 24 + 1.1 * v.double() ** 2 if a == "gelu" else 8 + 2 * v.abs().double()
    assert (units * U32 < 2e-5).all()         # what is nearly 0 has its value, not just something near 0
    for scale in (out.scales.t[0], out.scales.t[-1]):
        within(scale, (want / 448).clamp(min=2.0 ** -126), units * U32 * want / 448 + U32 * 2.0 ** -126)


@pytest.mark.parametrize("a,low", [("gelu", -12.0), ("silu", -75.0)])
@pytest.mark.parametrize("is_gated", [False, True])
def test_gradients_relative_to_themselves(lib, gpu, a, low, is_gated):
    """dh is 1: the slope, rounded once to bfloat16 (2^-8), relative to the larger of its two terms, which cancel near its zero; the activation's
    value comes back as `hidden`."""
    n, rows = 256, 96
    dout = Matrix(rows, 8, "bf16", values=torch.eye(8, device="cuda")[:1].expand(rows, 8))
    w = Weights(gen(1), 1, 1, 8, n, "bf16")
    w.m.t.zero_()
    w.m.t[0] = 1
    gate = torch.linspace(low, -low, rows * n, device="cuda", dtype=torch.float64).view(rows, n)
    kept = torch.cat([gate, torch.ones_like(gate)], dim=1) if is_gated else gate
    saved = Matrix(rows, kept.shape[1], "bf16", values=kept)
    dsaved, hidden = Matrix(rows, kept.shape[1], "bf16"), Matrix(rows, n, "bf16")
    assert hidden_grad(lib, dout, w, None, 1, rows, 8, n, is_gated, a, saved, dsaved, hidden) == 0
    _gpu.sync()
    v = saved.values()[:, :n]
    value, slope = act(a, v)
    share = 0.5 * torch.special.erfc(-v * 0.5 ** 0.5) if a == "gelu" else torch.sigmoid(v)
    units = 32 + 4 * v.abs() + (1.1 * v * v if a == "gelu" else 0)
    within(hidden.rows.t, value, (2.0 ** -8 + units * U32) * value.abs())
    terms = share + (slope - share).abs()
    within(dsaved.rows.t[:, :n], slope, 2.0 ** -8 * slope.abs() + (1 + 2.0 ** -8) * units * U32 * terms)
    if is_gated:
        within(dsaved.rows.t[:, n:], value, (2.0 ** -8 + units * U32) * value.abs())
