"""Gated blocks, products and their gradients over rows sorted by expert, against the formulas in 64 bits (tests/_experts.py has the bounds)."""
import pytest
import torch

import _gpu
import aws_ofi_nccl_amd as m
from _experts import check_gated, check_hidden, check_product, check_rows, check_weights, gen, rnd
from _rows import Rows

pytestmark = pytest.mark.gpu

# rows of each expert: one row; few; experts without rows; tiles of 64, 128 and 256 rows with ragged ends
FEW = [[1], [0, 1, 0], [3, 0, 5, 1], [17, 0, 2, 33, 16], [64], [8] * 9]
MANY = [[65, 0, 1, 200], [129] * 3, [300, 5, 256, 0, 257]]
WIDTHS = [(64, 128), (128, 128), (200, 136), (264, 392), (1000, 72)]  # whole chunks
ODD = [(1, 1), (7, 3), (63, 130), (129, 127), (1001, 257)]


@pytest.mark.parametrize("counts", FEW + MANY)
@pytest.mark.parametrize("kind,out,saved", [("bf16", "bf16", "e4m3"), ("f16", "e4m3", None), ("e4m3", "e4m3", "e4m3"), ("e4m3", "bf16", "f16"),
                                            ("f16", "f16", "f16"), ("e4m3", "f16", None)])
def test_gated_rows_of_experts(lib, gpu, counts, kind, out, saved):
    check_gated(lib, counts, 264, 200, kind, out, saved)


@pytest.mark.parametrize("width,inner", WIDTHS + ODD)
@pytest.mark.parametrize("kind,out,saved", [("bf16", "bf16", "bf16"), ("e4m3", "e4m3", "e4m3"), ("f16", "e4m3", "f16")])
def test_gated_widths(lib, gpu, width, inner, kind, out, saved):
    for counts in ([2, 0, 9], [70, 140]):
        check_gated(lib, counts, width, inner, kind, out, saved, seed=width)


@pytest.mark.parametrize("a", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("kind", ["bf16", "f16", "e4m3"])
def test_activations(lib, gpu, a, kind):
    check_gated(lib, [40, 90], 256, 128, kind, "f16" if kind != "bf16" else "bf16", a=a)
    check_product(lib, [40, 90], 256, 264, kind, a=a, bias_type=torch.float32, saved_kind="e4m3")
    if kind != "e4m3":
        for is_gated in (False, True):
            check_hidden(lib, [40, 90], 128, 136, kind, "e4m3", is_gated, a)


@pytest.mark.parametrize("counts", FEW + MANY)
@pytest.mark.parametrize("kind,out", [("bf16", None), ("f16", None), ("e4m3", "bf16"), ("e4m3", "e4m3"), ("bf16", "e4m3")])
def test_products_of_experts(lib, gpu, counts, kind, out):
    check_product(lib, counts, 264, 392, kind, out)


@pytest.mark.parametrize("width,n", WIDTHS + ODD)
@pytest.mark.parametrize("kind", ["bf16", "f16", "e4m3"])
def test_product_widths(lib, gpu, width, n, kind):
    for counts in ([2, 0, 9], [70, 140]):
        check_product(lib, counts, width, n, kind, a="gelu", bias_type=torch.float16, residual=True, saved_kind="e4m3", seed=width)


@pytest.mark.parametrize("rows", [1, 16, 17, 33, 64, 65, 500, 4500])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("bias_type", [None, torch.float32, torch.float16, torch.bfloat16])
def test_a_layer_of_one_expert(lib, gpu, rows, kind, bias_type):
    """No offsets; 4500 rows by 4100 columns are tiles of 256 rows."""
    check_product(lib, [rows], 200, 4100 if rows == 4500 else 264, kind, a="silu", bias_type=bias_type, residual=True, dense=True)
    check_product(lib, [rows], 200, 264, kind, bias_type=bias_type, residual=True, dense=True, in_place=True)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_large_tiles(lib, gpu, kind):
    """The forward products' tiles of 256 rows; gradients over nearly as many."""
    counts = [700, 0, 513, 256, 1, 2000]
    check_gated(lib, counts, 264, 2176, kind, kind, "e4m3")
    check_product(lib, counts, 200, 4104, kind, a="gelu", bias_type=torch.float32, residual=True, saved_kind=kind)
    check_hidden(lib, counts, 264, 4104, kind, "e4m3")
    check_hidden(lib, counts, 136, 4104, kind, kind, False, "gelu")
    check_rows(lib, counts, 4104, 264, kind, added=True)
    check_weights(lib, counts, 1032, 2056, kind, "f32", added=True, bias=True)
    check_weights(lib, counts, 1032, 2056, kind, kind, bias=True)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("summed", [8, 40, 72, 136, 264])
def test_tiles_in_pairs(lib, gpu, kind, summed):
    """Gradients over 512 tiles of 128 rows and more, of which a compute unit has two: sums of half a step, an odd number of halves, several steps."""
    counts = [700, 0, 513, 256, 1, 2000]  # 30 row tiles if they were alike, 18 column tiles
    check_hidden(lib, counts, summed, 4480, kind, "e4m3")
    check_hidden(lib, counts, summed, 4480, kind, kind, False, "gelu", with_hidden=False)
    check_rows(lib, counts, 4480, summed, kind, added=True)


@pytest.mark.parametrize("kind,out", [("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_weight_tiles_in_pairs(lib, gpu, kind, out):
    """The same where the rows of an expert are summed: none, one, half a step and one more, several steps; the bias is of the first column tile."""
    counts = [700, 0, 33, 64, 1, 65, 32, 129]  # 8 x 13 x 5 tiles
    check_weights(lib, counts, 1032, 1560, kind, out, bias=True)
    check_weights(lib, counts, 1280, 1664, kind, out, added=True, bias=True, in_place=True)


@pytest.mark.parametrize("width,n", [(64, 64), (256, 264), (2048, 8192), (33, 65)])
@pytest.mark.parametrize("pitch", [0, 16])
def test_one_row_with_any_pitch(lib, gpu, width, n, pitch):
    """A single row is summed once, whatever its pitch says of a next one."""
    g = gen(width)
    dout, x = (rnd(g, 1, k).to(torch.bfloat16) for k in (n, width))
    dw, dbias = torch.full((n, width), 7.0, device="cuda"), torch.full((n,), 7.0, device="cuda")
    assert lib.ofi_amd_expert_weight_grad(dout.data_ptr(), pitch, x.data_ptr(), pitch, m.BFLOAT16, None, 1, 1, width, n, None, dw.data_ptr(),
                                          4 * width, 0, m.FLOAT32, None, dbias.data_ptr(), None) == 0
    _gpu.sync()
    assert torch.equal(dw, dout.float().t() * x.float())  # a product of two bfloat16 values is a float32 value
    assert torch.equal(dbias, dout[0].float())


def test_large_tiles_of_8_bits(lib, gpu):
    counts = [700, 0, 513, 256, 1, 2000]
    check_gated(lib, counts, 400, 2176, "e4m3", "e4m3", "e4m3")
    check_product(lib, counts, 272, 4104, "e4m3", "bf16", a="gelu", bias_type=torch.float32, residual=True, saved_kind="f16")


@pytest.mark.parametrize("counts", FEW + MANY)
@pytest.mark.parametrize("kind,saved,is_gated", [("bf16", "e4m3", True), ("f16", "f16", True), ("f16", "e4m3", False), ("bf16", "bf16", False)])
def test_hidden_gradients_of_experts(lib, gpu, counts, kind, saved, is_gated):
    check_hidden(lib, counts, 264, 200, kind, saved, is_gated)


@pytest.mark.parametrize("width,inner", WIDTHS + ODD)
def test_hidden_gradient_widths(lib, gpu, width, inner):
    for counts in ([2, 0, 9], [70, 140]):
        check_hidden(lib, counts, width, inner, "bf16", "e4m3", True, seed=width)
        check_hidden(lib, counts, width, inner, "f16", "f16", False, "gelu", seed=width, with_hidden=False)


@pytest.mark.parametrize("counts", FEW + MANY)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_row_and_weight_gradients_of_experts(lib, gpu, counts, kind):
    check_rows(lib, counts, 264, 200, kind)
    check_weights(lib, counts, 264, 200, kind, "f32", bias=True)
    check_weights(lib, counts, 264, 200, kind, kind, added=True, bias=True)


@pytest.mark.parametrize("width,n", WIDTHS + ODD)
def test_row_and_weight_gradient_widths(lib, gpu, width, n):
    for counts in ([2, 0, 9], [70, 140]):
        check_rows(lib, counts, width, n, "f16", added=True, seed=width)
        check_rows(lib, counts, width, n, "bf16", added=True, in_place=True, seed=width)
        check_weights(lib, counts, width, n, "bf16", "f32", added=True, in_place=True, bias=True, seed=width)
        check_weights(lib, counts, width, n, "f16", "f16", bias=True, seed=width)


@pytest.mark.parametrize("pad,shift,apart", [(8, 0, 0), (16, 8, 3), (1, 0, 1), (5, 3, 0), (64, 0, 1)])
@pytest.mark.parametrize("guard", [0xA5, 0xFF])
def test_pitches_and_alignments(lib, gpu, monkeypatch, pad, shift, apart, guard):
    """What lies beside the rows, NaN among it (0xff in every type), does not reach them."""
    monkeypatch.setattr(Rows, "guard", guard)
    for counts in ([3, 0, 8], [80, 3, 200]):
        opts = dict(pad=pad, shift=shift, apart=apart, first=2, spare=5)
        for width, n in ((136, 200), (130, 77)):
            check_gated(lib, counts, width, n, "bf16", "e4m3", "bf16", **opts)
            check_gated(lib, counts, width, n, "e4m3", "f16", "e4m3", **opts)
            check_product(lib, counts, width, n, "f16", a="silu", residual=True, bias_type=torch.bfloat16, **opts)
            check_hidden(lib, counts, width, n, "bf16", "e4m3", **opts)
            check_rows(lib, counts, width, n, "f16", added=True, **opts)
            check_weights(lib, counts, width, n, "bf16", "f32", added=True, bias=True, **opts)


def test_no_rows_at_all(lib, gpu):
    for spare in (0, 9):
        opts = dict(spare=spare)
        check_gated(lib, [0, 0], 64, 32, **opts)
        check_product(lib, [0, 0], 64, 32, **opts)
        check_hidden(lib, [0, 0], 64, 32, **opts)
        check_rows(lib, [0, 0], 64, 32, **opts)
        check_weights(lib, [0, 0], 64, 32, bias=True, **opts)
        check_weights(lib, [0, 0], 64, 32, added=True, bias=True, **opts)


@pytest.mark.parametrize("experts", [64, 65, 200, 1024])
def test_many_experts(lib, gpu, experts):
    counts = [(7 * e * e + e) % 23 if e % 3 else 0 for e in range(experts)]
    check_gated(lib, counts, 72, 40, "e4m3", "e4m3")
    check_product(lib, counts, 40, 72, "bf16")
    check_hidden(lib, counts, 72, 40)
    check_rows(lib, counts, 72, 40)
    check_weights(lib, counts, 72, 40, bias=True)
    check_product(lib, [c * 20 for c in counts[:130]], 40, 72, "bf16")


@pytest.mark.parametrize("counts", [[5, 3], [200, 130]])
@pytest.mark.parametrize("kind,out", [("bf16", "bf16"), ("f16", "e4m3"), ("e4m3", "e4m3")])
def test_a_row_with_nan_or_infinity_is_alone_with_it(lib, gpu, counts, kind, out):
    def bad(values, offset):
        values[1, 7] = float("nan")
        if kind != "e4m3":                    # 8-bit rows have no infinities
            values[4, 3] = float("inf")

    result = check_gated_rows(lib, counts, kind, out, bad)
    assert bool(torch.isnan(result.values()[1]).all())


def check_gated_rows(lib, counts, kind, out, bad):
    """Rows with a NaN or an infinity: every other row is as it was without."""
    import _gpu
    from _experts import Matrix, Weights, gated, gen, offsets, scaled_values
    results = []
    for put in (None, bad):
        g = gen(3)
        n = sum(counts)
        values, scale = scaled_values(g, n, 136, kind)
        if put:
            put(values, None)
        x = Matrix(n, 136, kind, values=values, scale=scale)
        if put and kind == "e4m3":
            x.rows.t.view(torch.uint8)[1, 7] = 0x7F
        w = Weights(g, len(counts), 2, 72, 136, kind)
        y = Matrix(n, 72, out)
        assert gated(lib, x, w, offsets(0, counts), len(counts), n, 136, 72, "silu", y) == 0
        _gpu.sync()
        results.append(y)
    a, b = (r.rows.t.view(torch.uint8).clone() for r in results)
    same = (a == b).all(dim=1)
    same[1] = True
    if kind != "e4m3":
        same[4] = True
    assert bool(same.all())
    return results[1]


def test_offsets_that_point_outside_the_rows_are_cut(lib, gpu):
    """Within [0, max_rows]: an expert whose rows would begin or end elsewhere has those that are there."""
    import _gpu
    from _experts import Matrix, Weights, gen, product, rnd, sum_error, check_output, left_alone
    g = gen(5)
    x, w, out = Matrix(40, 64, "bf16", values=rnd(g, 40, 64)), Weights(g, 3, 1, 48, 64, "bf16"), Matrix(40, 48, "bf16")
    offset = torch.tensor([-7, 10, 25, 90], dtype=torch.int32, device="cuda")
    assert product(lib, x, w, offset, 3, 40, 64, 48, "none", out) == 0
    _gpu.sync()
    for e, (lo, hi) in enumerate([(0, 10), (10, 25), (25, 40)]):
        v, wv = x.values()[lo:hi], w.values(e)
        check_output(out, lo, hi, v @ wv.t().contiguous(), sum_error(64, v.abs() @ wv.abs().t().contiguous()))
    assert out.untouched() and left_alone(out, offset, 40, 3)
