"""The way back of aws_ofi_nccl_amd.expert_exchange: the rows' gradients are put to their ranks and the experts' are fetched."""
import pytest
import torch

from aws_ofi_nccl_amd import expert_exchange as ex

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,width,experts,top_k,ranks", [(40, 256, 8, 2, 4), (7, 130, 5, 5, 5)])
def test_gradients_cross_the_link(lib, gpu, tokens, width, experts, top_k, ranks):
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    x, residual, dout = (normal(tokens, width).to(torch.bfloat16) for _ in range(3))
    gain = torch.ones(width, dtype=torch.bfloat16, device="cuda")
    top, ids = torch.topk(normal(tokens, experts), top_k, dim=1)
    weight = torch.softmax(top, dim=1).contiguous()
    up, down = normal(experts, width, 32) / width ** 0.5, normal(experts, 32, width) / 32 ** 0.5
    link = ex.Link(lib, ranks, tokens * top_k, width)
    moved = []
    put_signal, get = link.put_signal, link.get
    link.put_signal = lambda rank, at, size: (moved.append(("put", rank, size)), put_signal(rank, at, size))
    link.get = lambda rank, at, size: (moved.append(("get", rank, size)), get(rank, at, size))
    try:
        got = ex.layer(lib, link, x, residual, gain, ids, weight, up, down)
        forward = list(moved)
        torch.cuda.synchronize()
        assert link.counters.cpu().tolist() == [1 if hi > lo else 0 for lo, hi in got["runs"]]
        moved.clear()
        got = ex.layer(lib, link, x, residual, gain, ids, weight, up, down, dout)
        torch.cuda.synchronize()
        assert link.counters.cpu().tolist() == [3 if hi > lo else 0 for lo, hi in got["runs"]]
    finally:
        link.close()
    sizes = {r: (hi - lo) * width for r, (lo, hi) in enumerate(got["runs"]) if hi > lo}
    assert forward == [("put", r, n) for r, n in sizes.items()] + [("get", r, 2 * n) for r, n in sizes.items()]
    assert moved == forward + [("put", r, 2 * n) for r, n in sizes.items()] + [("get", r, 2 * n) for r, n in sizes.items()]
    want = ex.plain(got, x, residual, gain, ids, weight, up, down, dout)
    for key in ("out", "dx", "dgain", "dweight"):
        # a rounding to bfloat16 (2^-8 of a value at most) of each of the few tensors on the way
        assert ((got[key].double() - want[key]).norm() / want[key].norm()).item() < 0.015, key
