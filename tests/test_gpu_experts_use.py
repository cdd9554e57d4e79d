"""The experts' products as a layer uses them: one after the other from the dispatch's offsets, captured into graphs, on other streams, over rows
whose offsets pass 32 bits, and their gradients against differences of the formula."""
import ctypes

import pytest
import torch

import _gpu
import aws_ofi_nccl_amd as m
from _experts import (KIND, Matrix, Weights, act, check_output, gated, gen, hidden_grad, left_alone, offsets, product, rnd, rows_grad, runs,
                      sum_error, weight_grad)
from _rows import Rows, within

pytestmark = pytest.mark.gpu


class Layer:
    """An expert's block and the product behind it, forward and back, with all buffers."""

    def __init__(self, rows, width, inner, experts, kind="bf16", saved_kind="e4m3", seed=1):
        g = gen(seed)
        self.sizes = rows, width, inner, experts
        self.kind = kind
        self.x = Matrix(rows, width, kind, values=rnd(g, rows, width))
        self.w1, self.w2 = Weights(g, experts, 2, inner, width, kind), Weights(g, experts, 1, width, inner, kind)
        self.dout = Matrix(rows, width, kind, values=rnd(g, rows, width) * 0.1)
        self.offset = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
        self.fresh(saved_kind)

    def fresh(self, saved_kind="e4m3"):
        rows, width, inner, experts = self.sizes
        self.h, self.h2, self.y, self.dx = (Matrix(rows, n, self.kind) for n in (inner, inner, width, width))
        self.saved, self.dsaved = Matrix(rows, 2 * inner, saved_kind, parts=2), Matrix(rows, 2 * inner, self.kind)
        self.dw1, self.dw2 = Matrix(experts * 2 * inner, width, "f32"), Matrix(experts * width, inner, "f32")

    def outputs(self):
        return [t.rows.bytes for t in (self.h, self.h2, self.y, self.dx, self.saved, self.dsaved, self.dw1, self.dw2)] + (
            [self.saved.scales.bytes] if self.saved.scales else [])

    def run(self, lib, stream=None):
        rows, width, inner, experts = self.sizes
        args = self.offset, experts, rows
        assert gated(lib, self.x, self.w1, *args, width, inner, "silu", self.h, self.saved, stream) == 0
        assert product(lib, self.h, self.w2, *args, inner, width, "none", self.y, stream=stream) == 0
        assert hidden_grad(lib, self.dout, self.w2, *args, width, inner, True, "silu", self.saved, self.dsaved, self.h2, stream) == 0
        assert weight_grad(lib, self.dout, self.h2, *args, inner, width, self.dw2, width * self.dw2.rows.pitch, stream=stream) == 0
        assert rows_grad(lib, self.dsaved, self.w1, *args, width, 2 * inner, self.dx, stream=stream) == 0
        assert weight_grad(lib, self.dsaved, self.x, *args, width, 2 * inner, self.dw1, 2 * inner * self.dw1.rows.pitch, stream=stream) == 0


def formula(x, w1, w2):
    inner = w1.shape[0] // 2
    both = x @ w1.t()
    return (act("silu", both[:, :inner])[0] * both[:, inner:]) @ w2.t()


@pytest.mark.parametrize("counts,width,inner", [([3, 0, 2], 72, 40), ([130, 7, 0, 65], 136, 200), ([33, 1], 77, 33)])
@pytest.mark.parametrize("saved_kind", ["e4m3", "f16"])
def test_a_layer_forward_and_back(lib, gpu, counts, width, inner, saved_kind):
    """Against gradients of the formula in 64 bits.  Each of the few tensors on the way is rounded to 2^-11 of a value (2^-4 where it is kept in
    8 bits, as errors that are independent from value to value): the whole of a gradient is off by at most 8 times that."""
    layer = Layer(sum(counts), width, inner, len(counts), "f16", saved_kind)
    layer.offset.copy_(offsets(0, counts))
    layer.run(lib)
    _gpu.sync()
    rough = 8 * 2.0 ** -11 if saved_kind == "f16" else 2.0 ** -4
    for e, lo, hi in runs(layer.offset, sum(counts), len(counts)):
        x, w1, w2 = (v.clone().requires_grad_(True) for v in (layer.x.values()[lo:hi], layer.w1.values(e), layer.w2.values(e)))
        y = formula(x, w1, w2)
        dx, dw1, dw2 = torch.autograd.grad(y, (x, w1, w2), layer.dout.values()[lo:hi])
        off = lambda got, want: ((got - want).norm() / want.norm()).item()
        assert off(layer.y.values()[lo:hi], y.detach()) < 8 * 2.0 ** -11
        assert off(layer.dx.values()[lo:hi], dx) < rough
        assert off(layer.dw1.values()[e * 2 * inner:(e + 1) * 2 * inner], dw1) < rough
        assert off(layer.dw2.values()[e * width:(e + 1) * width], dw2) < rough


def test_gradients_against_differences(lib, gpu):
    """The loss sum(y * dout) along random directions, by central differences in 64 bits.  h = 1e-4 leaves (h^2 / 6) of a third derivative,
    far below the 2^-11 of what is rounded on the way."""
    counts, width, inner = [40, 25], 72, 40
    layer = Layer(sum(counts), width, inner, 2, "f16", "f16")
    layer.offset.copy_(offsets(0, counts))
    layer.run(lib)
    _gpu.sync()
    g, h = gen(9), 1e-4
    for e, lo, hi in runs(layer.offset, sum(counts), 2):
        at = [layer.x.values()[lo:hi], layer.w1.values(e), layer.w2.values(e)]
        got = [layer.dx.values()[lo:hi], layer.dw1.values()[e * 2 * inner:(e + 1) * 2 * inner], layer.dw2.values()[e * width:(e + 1) * width]]
        d = layer.dout.values()[lo:hi]
        for k in range(3):
            way = rnd(g, *at[k].shape)
            loss = lambda s: (formula(*[v + s * way if i == k else v for i, v in enumerate(at)]) * d).sum()
            slope = ((loss(h) - loss(-h)) / (2 * h)).item()
            along = (got[k] * way).sum().item()
            assert abs(along - slope) < 8 * 2.0 ** -11 * (got[k].norm() * way.norm()).item()


@pytest.mark.parametrize("rows,width,inner,experts", [(6, 264, 136, 5), (300, 136, 200, 3), (5000, 72, 2056, 2)])
def test_graphs(lib, gpu, rows, width, inner, experts):
    """Two captured layers, replayed in turn on inputs and offsets that change, with eager runs between: every replay has an eager run's bits."""
    layers = [Layer(rows, width, inner, experts, seed=s) for s in (1, 2)]
    eager = Layer(rows, width, inner, experts, seed=3)

    def change(layer, seed):
        g = gen(seed)
        layer.x.rows.t.copy_(rnd(g, rows, width))
        cut = torch.sort(torch.randint(0, rows + 1, (experts - 1,), generator=g, device="cuda"))[0]
        layer.offset.copy_(torch.cat([cut.new_zeros(1), cut, cut.new_full((1,), rows)]).to(torch.int32))

    graphs = []
    for k, layer in enumerate(layers):
        change(layer, k)
        layer.run(lib)
        _gpu.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer.run(lib)
        graphs.append(graph)
    for seed in range(10, 14):
        for layer, graph in zip(layers, graphs):
            change(layer, seed)
            for t in layer.outputs():
                t.fill_(Rows.guard)
            graph.replay()
            _gpu.sync()
            eager.x, eager.w1, eager.w2, eager.dout, eager.offset = layer.x, layer.w1, layer.w2, layer.dout, layer.offset
            eager.fresh()
            eager.run(lib)
            _gpu.sync()
            for a, b in zip(layer.outputs(), eager.outputs()):
                assert torch.equal(a, b)


def test_other_streams_at_once(lib, gpu):
    layers = [Layer(700, 136, 264, 3, seed=4) for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in layers]
    for layer in layers:
        layer.offset.copy_(offsets(0, [300, 0, 400]))
    _gpu.sync()
    for _ in range(3):
        for layer, s in zip(layers, streams):
            layer.run(lib, ctypes.c_void_p(s.cuda_stream))
    _gpu.sync()
    for layer in layers[1:]:
        for a, b in zip(layers[0].outputs(), layer.outputs()):
            assert torch.equal(a, b)


def test_the_same_call_gives_the_same_bits(lib, gpu):
    layer = Layer(900, 264, 520, 4)
    layer.offset.copy_(offsets(0, [500, 1, 0, 399]))
    layer.run(lib)
    _gpu.sync()
    first = [t.clone() for t in layer.outputs()]
    for _ in range(5):
        layer.run(lib)
        _gpu.sync()
        for a, b in zip(first, layer.outputs()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("counts", [[3, 6], [12, 8]])
def test_rows_far_apart_pass_32_bits_of_offset(lib, gpu, counts):
    pitch, n, width = 1 << 28, sum(counts), 72
    g = gen(6)
    far = torch.zeros(n * pitch, dtype=torch.uint8, device="cuda")
    v = rnd(g, n, width).to(torch.bfloat16)
    for k in range(n):
        far[k * pitch:k * pitch + 2 * width].view(torch.bfloat16).copy_(v[k])
    w, out, offset = Weights(g, len(counts), 1, 48, width, "bf16"), Matrix(n, 48, "bf16"), offsets(0, counts)
    dw = Matrix(len(counts) * width, width, "f32")
    p = ctypes.c_void_p(far.data_ptr())
    assert lib.ofi_amd_expert_product(p, pitch, None, 0, m.BFLOAT16, offset.data_ptr(), len(counts), n, *w.args(), None, width, 48, None, 0, 0, None, 0,
                                      *out.args(), m.BFLOAT16, None, 0, None, 0, 0, None, 0, _gpu.stream()) == 0
    assert lib.ofi_amd_expert_weight_grad(p, pitch, p, pitch, m.BFLOAT16, offset.data_ptr(), len(counts), n, width, width, None, *dw.args(),
                                          width * dw.rows.pitch, m.FLOAT32, None, None, _gpu.stream()) == 0
    _gpu.sync()
    for e, lo, hi in runs(offset, n, len(counts)):
        d, wv = v[lo:hi].double(), w.values(e)
        check_output(out, lo, hi, d @ wv.t().contiguous(), sum_error(width, d.abs() @ wv.abs().t().contiguous()))
        check_output(dw, e * width, (e + 1) * width, d.t().contiguous() @ d, sum_error(hi - lo, d.abs().t().contiguous() @ d.abs()))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_weights_behind_32_bits_of_offset(lib, gpu, kind):
    """Experts 3 GiB apart: the third's weights begin beyond 2^32 bytes."""
    width, n, apart, counts = 64, 40, 3 << 30, [2, 3, 70]
    g = gen(7)
    far = torch.zeros(2 * apart + n * width * 2, dtype=torch.uint8, device="cuda")
    w = rnd(g, 3, n, width).to(KIND[kind][0])
    for e in range(3):
        far[e * apart:e * apart + n * width * 2].view(KIND[kind][0]).copy_(w[e].reshape(-1))
    x, out, dx, offset = Matrix(75, width, kind, values=rnd(g, 75, width)), Matrix(75, n, kind), Matrix(75, width, kind), offsets(0, counts)
    p = ctypes.c_void_p(far.data_ptr())
    assert lib.ofi_amd_expert_product(*x.args(), None, 0, KIND[kind][1], offset.data_ptr(), 3, 75, p, 2 * width, apart, None, width, n, None, 0, 0, None, 0,
                                      *out.args(), KIND[kind][1], None, 0, None, 0, 0, None, 0, _gpu.stream()) == 0
    assert lib.ofi_amd_expert_rows_grad(*out.args(), KIND[kind][1], offset.data_ptr(), 3, 75, p, 2 * width, apart, width, n, None, 0, *dx.args(),
                                        _gpu.stream()) == 0
    _gpu.sync()
    for e, lo, hi in runs(offset, 75, 3):
        v, wv = x.values()[lo:hi], w[e].double()
        check_output(out, lo, hi, v @ wv.t().contiguous(), sum_error(width, v.abs() @ wv.abs().t().contiguous()))
        d = out.values()[lo:hi]
        check_output(dx, lo, hi, d @ wv, sum_error(n, d.abs() @ wv.abs()))


def test_the_dispatch_leaves_what_the_products_take(lib, gpu):
    """Rows of e4m3 sorted by the library, some pairs elsewhere, room for more rows than there are: gated block on what the dispatch left."""
    tokens, top_k, experts, width, inner = 37, 3, 6, 256, 136
    g = gen(8)
    pairs, room = tokens * top_k, tokens * top_k + 20
    ids = torch.randint(-1, experts, (tokens, top_k), generator=g, device="cuda", dtype=torch.int32)
    q = (rnd(g, tokens, width) * 100).clamp(-448, 448).float().to(torch.float8_e4m3fn)
    scale = torch.rand(tokens, 2, generator=g, device="cuda") / 100
    x = Matrix(room, width, "e4m3")
    offset, row_of, pair_of = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (experts + 1, pairs, room))
    work = torch.empty(max(16, lib.ofi_amd_token_dispatch_work_bytes(tokens, top_k, experts)), dtype=torch.uint8, device="cuda")
    assert lib.ofi_amd_token_dispatch(ids.data_ptr(), m.INT32, tokens, top_k, experts, room, offset.data_ptr(), row_of.data_ptr(), pair_of.data_ptr(),
                                      q.data_ptr(), width, *x.args(), width, scale.data_ptr(), 8, *x.scale_args(), 8, work.data_ptr(), work.numel(),
                                      _gpu.stream()) == 0
    w, out = Weights(g, experts, 2, inner, width, "e4m3"), Matrix(room, inner, "bf16")
    assert gated(lib, x, w, offset, experts, room, width, inner, "silu", out) == 0
    _gpu.sync()
    values = (q.double() * scale.double().repeat_interleave(128, dim=1))
    for pair, row in enumerate(row_of.tolist()):
        if row >= 0:
            both = w.values(int(ids.view(-1)[pair])) @ values[pair // top_k]
            want = act("silu", both[:inner])[0] * both[inner:]
            within(out.rows.t[row], want, 2.0 ** -8 * want.abs() + 2.0 ** -14 * want.abs().max())
    assert out.untouched() and left_alone(out, offset, room, experts)
