"""Norms, sums of tokens and their gradients captured into a graph, replayed on inputs that change between the replays, with eager calls and
synchronizations between them: each replay has the bits of an eager call on the same inputs."""
import pytest
import torch

import _gpu
from _rows import TYPES, Rows
from test_gpu_rms_norm import gen, grad as norm_grad, norm, values
from test_gpu_token_combine import combine, grad as combine_grad, plan

pytestmark = pytest.mark.gpu


def replayed(call, change, outputs):
    """call(k): the call, into the k-th set of outputs; change(seed): other inputs; outputs: two sets of tensors."""
    def cleared(k):
        for t in outputs[k]:
            t.view(torch.uint8).fill_(0x3C)

    change(0)
    call(0)
    _gpu.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0)
    for seed in range(1, 5):
        change(seed)
        cleared(0)
        graph.replay()
        _gpu.sync()
        cleared(1)
        call(1)
        _gpu.sync()
        for a, b in zip(*outputs):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            assert not bool((a.view(torch.uint8) == 0x3C).all())


@pytest.mark.parametrize("rows,width", [(1, 4096), (300, 100), (3000, 1999), (9000, 1024)])
def test_norms(lib, gpu, rows, width):
    dtype = TYPES["bf16"][0]
    x, r = Rows(rows, width, dtype), Rows(rows, width, dtype)
    gain = torch.zeros(width, dtype=dtype, device="cuda")
    out = [(Rows(rows, width, dtype), Rows(rows, width, dtype), Rows(rows, width, torch.float8_e4m3fn), Rows(rows, -(-width // 128), torch.float32),
            torch.zeros(rows, device="cuda")) for _ in range(2)]

    def change(seed):
        for t in (x, r):
            t.t.copy_(values(gen(seed), rows, width))
        gain.copy_(1 + 0.3 * torch.randn(width, generator=gen(seed)))

    def call(k):
        total, normed, q, scale, rstd = out[k]
        assert norm(lib, x, gain, width, "bf16", r, total, normed, q, scale, 128, rstd) == 0

    replayed(call, change, [[t.bytes[:t.n * t.pitch] for t in o[:4]] + [o[4]] for o in out])


@pytest.mark.parametrize("rows,width", [(1, 4096), (256, 1000), (257, 1000), (700, 16385), (3000, 513)])
def test_gradients_of_norms(lib, gpu, rows, width):
    """In one launch up to 256 rows, in two and with a workspace beyond."""
    dtype = TYPES["f16"][0]
    s, dout, dsum = (Rows(rows, width, dtype) for _ in range(3))
    gain, rstd = torch.ones(width, dtype=dtype, device="cuda"), torch.zeros(rows, device="cuda")
    out = [(Rows(rows, width, dtype), torch.zeros(width, device="cuda")) for _ in range(2)]
    work = torch.full((lib.ofi_amd_rms_norm_grad_work_bytes(rows, width),), 0x7F, dtype=torch.uint8, device="cuda")

    def change(seed):
        for k, t in enumerate((s, dout, dsum)):
            t.t.copy_(values(gen(10 * seed + k), rows, width, 0.1))
        rstd.copy_(torch.rand(rows, generator=gen(seed)) + 0.5)

    def call(k):
        assert norm_grad(lib, dout, s, rstd, gain, width, "f16", dsum, out[k][0], out[k][1], work) == 0

    replayed(call, change, [[o[0].bytes[:rows * o[0].pitch], o[1]] for o in out])


@pytest.mark.parametrize("tokens,top_k,width", [(1, 8, 4096), (700, 8, 1000), (900, 1, 520), (2000, 2, 300), (300, 17, 100)])
def test_sums_and_their_gradients(lib, gpu, tokens, top_k, width):
    dtype, n = TYPES["bf16"][0], tokens * top_k
    rows, add, dout = Rows(n, width, dtype), Rows(tokens, width, dtype), Rows(tokens, width, dtype)
    row_of = torch.zeros(tokens, top_k, dtype=torch.int32, device="cuda")
    weight = torch.zeros(tokens, top_k, device="cuda")
    out = [(Rows(tokens, width, dtype), Rows(n, width, dtype), torch.zeros(tokens, top_k, device="cuda")) for _ in range(2)]

    def change(seed):
        for k, t in enumerate((rows, add, dout)):
            t.t.copy_(torch.randn(t.n, width, generator=gen(10 * seed + k)))
        row_of.copy_(plan(gen(seed), tokens, top_k, n, 0.2 if n > 8 else 0.0))
        weight.copy_(torch.rand(tokens, top_k, generator=gen(seed)))

    def call(k):
        assert combine(lib, rows, row_of, weight, width, "bf16", add, out[k][0]) == 0
        assert combine_grad(lib, dout, rows, row_of, weight, width, "bf16", out[k][1], out[k][2]) == 0

    replayed(call, change, [[o[0].bytes[:tokens * o[0].pitch], o[1].bytes[:n * o[1].pitch], o[2]] for o in out])
