"""Gradients of an expert's block against differences of its loss, along directions in which a gradient that is a percent off shows."""
import pytest
import torch

import _gpu
from _experts import gen, offsets, runs
from test_gpu_experts_use import Layer, formula

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts,width,inner", [([40, 25], 72, 40), ([1, 0, 130], 136, 72), ([33], 77, 33)])
def test_gradients_along_themselves(lib, gpu, counts, width, inner):
    """The loss sum(y * dout), by central differences in 64 bits with h = 1e-5 of a step whose size is 1, along the gradient's own direction
    (the formula's) and along its halves and quarters by rows and columns, and random halves of it.  What is rounded to 2^-11 on the way leaves a
    gradient off by at most 8 times that of its size, in any direction: of a slope along a part with a share s of the gradient's square,
    0.4 % / sqrt(s)."""
    layer = Layer(sum(counts), width, inner, len(counts), "f16", "f16")
    layer.offset.copy_(offsets(0, counts))
    layer.run(lib)
    _gpu.sync()
    g, h, seen = gen(9), 1e-5, 0
    for e, lo, hi in runs(layer.offset, sum(counts), len(counts)):
        at = [layer.x.values()[lo:hi], layer.w1.values(e), layer.w2.values(e)]
        got = [layer.dx.values()[lo:hi], layer.dw1.values()[e * 2 * inner:(e + 1) * 2 * inner], layer.dw2.values()[e * width:(e + 1) * width]]
        d = layer.dout.values()[lo:hi]
        leaves = [v.clone().requires_grad_(True) for v in at]
        want = torch.autograd.grad((formula(*leaves) * d).sum(), leaves)
        for k in range(3):
            rows, columns = want[k].shape
            low = torch.arange(rows, device="cuda")[:, None] < (rows + 1) // 2, torch.arange(columns, device="cuda")[None, :] < columns // 2
            parts = [torch.ones_like(want[k], dtype=torch.bool)]
            parts += [(low[0] == a) & (low[1] == b) for a in (True, False) for b in (True, False)]
            parts += [torch.rand(rows, columns, generator=g, device="cuda") < 0.5 for _ in range(3)]
            for part in parts:
                size = (want[k] * part).norm().item()
                if size == 0:                 # a single row has no second half
                    continue
                way = want[k] * part / size
                loss = lambda s: (formula(*[v + s * way if i == k else v for i, v in enumerate(at)]) * d).sum()
                slope, along = ((loss(h) - loss(-h)) / (2 * h)).item(), (got[k] * way).sum().item()
                room = 8 * 2.0 ** -11 * want[k].norm().item()
                assert abs(slope - size) < 1e-4 * size   # the direction is the gradient's: its slope is its size
                assert abs(along - slope) < room
                assert room < 0.02 * slope               # two percent off would show
                seen += 1
    assert seen >= 20
