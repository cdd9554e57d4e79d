"""ofi_amd_token_dispatch against its definition: pairs in the order (expert, pair), rows copied byte for byte."""
import ctypes
import errno

import numpy as np
import pytest
import torch

import _gpu
import aws_ofi_nccl_amd as m
from _rows import Rows, ptr

pytestmark = pytest.mark.gpu

TOKEN_ROWS_BIT = 1 << 4


def table(ids, experts, max_rows):
    """(offsets, row of each pair, pair of each row, rows in all) from the definition."""
    flat = ids.reshape(-1).astype(np.int64)
    where = np.flatnonzero((flat >= 0) & (flat < experts))
    where = where[np.argsort(flat[where], kind="stable")]
    offset = np.minimum(np.concatenate([[0], np.cumsum(np.bincount(flat[where], minlength=experts))]), max_rows)
    row_of, pair_of = np.full(flat.size, -1), np.full(max_rows, -1)
    kept = where[:max_rows]
    row_of[kept] = np.arange(kept.size)
    pair_of[:kept.size] = kept
    return offset, row_of, pair_of, where.size


def make_ids(rng, tokens, top_k, experts, invalid, wide, skew=True):
    if skew:
        p = np.exp(rng.standard_normal(experts))
        ids = rng.choice(experts, size=(tokens, top_k), p=p / p.sum())
    else:
        ids = np.full((tokens, top_k), rng.integers(experts))
    ids = ids.astype(np.int64)
    if invalid:
        bad = [-1, experts, experts + 1, 2 ** 31 - 1, -2 ** 31] + ([2 ** 32, 2 ** 32 + experts - 1, -2 ** 32, 2 ** 63 - 1, -2 ** 63] if wide
                                                                    else [])
        hit = rng.random((tokens, top_k)) < invalid
        ids[hit] = np.array(bad, dtype=np.int64)[rng.integers(0, len(bad), int(hit.sum()))]
    return ids if wide else ids.astype(np.int32)


class Call:
    """Everything one call needs, with guards around what it may write."""

    def __init__(self, lib, ids, experts, max_rows, x=None, row_bytes=0, scale=None, scale_bytes=0, pad=0, shift=0, pairs=True):
        self.lib, self.experts, self.max_rows = lib, experts, max_rows
        self.tokens, self.top_k = ids.shape
        self.type = m.INT64 if ids.dtype == np.int64 else m.INT32
        self.ids = torch.from_numpy(ids).cuda()
        self.offset = torch.full((experts + 2,), 77, dtype=torch.int32, device="cuda")
        self.row_of = torch.full((ids.size + 1,), 77, dtype=torch.int32, device="cuda")
        self.pair_of = torch.full((max_rows + 1,), 77, dtype=torch.int32, device="cuda") if pairs else None
        self.x, self.scale, self.row_bytes, self.scale_bytes = x, scale, row_bytes, scale_bytes
        self.rows = Rows(max_rows, row_bytes, torch.uint8, pad, shift) if x is not None else None
        self.scale_rows = Rows(max_rows, scale_bytes, torch.uint8, pad, shift) if scale is not None else None
        need = lib.ofi_amd_token_dispatch_work_bytes(self.tokens, self.top_k, experts)
        self.work = torch.full((need,), 0xEE, dtype=torch.uint8, device="cuda") if need else None

    def run(self, stream=None):
        r = lambda t: (t.ptr(), t.pitch) if t is not None else (None, 0)
        return self.lib.ofi_amd_token_dispatch(
            ptr(self.ids), self.type, self.tokens, self.top_k, self.experts, self.max_rows, ptr(self.offset), ptr(self.row_of),
            ptr(self.pair_of), *r(self.x), *r(self.rows), self.row_bytes, *r(self.scale), *r(self.scale_rows), self.scale_bytes,
            ptr(self.work), 0 if self.work is None else self.work.numel(), _gpu.stream() if stream is None else stream)

    def check(self, ids):
        offset, row_of, pair_of, total = table(ids, self.experts, self.max_rows)
        n = ids.size
        got = self.offset.cpu().numpy()
        assert np.array_equal(got[:-1], offset) and got[-1] == 77
        got = self.row_of.cpu().numpy()
        assert np.array_equal(got[:n], row_of) and got[n] == 77
        if self.pair_of is not None:
            got = self.pair_of.cpu().numpy()
            assert np.array_equal(got[:-1], pair_of) and got[-1] == 77
        kept = pair_of[pair_of >= 0]
        for src, dst in ((self.x, self.rows), (self.scale, self.scale_rows)):
            if src is None:
                continue
            want = torch.full((self.max_rows, dst.width), 0xA5, dtype=torch.uint8, device="cuda")
            if kept.size:
                want[:kept.size] = src.t[torch.from_numpy(kept // self.top_k).cuda()]
            assert torch.equal(dst.t, want) and dst.untouched() and src.untouched()
        assert _gpu.fetch_async_errors(self.lib) == (TOKEN_ROWS_BIT if total > self.max_rows else 0)


def byte_rows(rng, n, width, pad=0, shift=0):
    return Rows(n, width, torch.uint8, pad, shift, torch.from_numpy(rng.integers(0, 256, (n, width), dtype=np.uint8)))


def check(lib, tokens, top_k, experts, seed=1, invalid=0.1, wide=False, row_bytes=64, scale_bytes=0, max_rows=None, pad=0, shift=0, **k):
    rng = np.random.default_rng(seed)
    ids = make_ids(rng, tokens, top_k, experts, invalid, wide, k.pop("skew", True))
    x = byte_rows(rng, tokens, row_bytes, pad, shift) if row_bytes else None
    scale = byte_rows(rng, tokens, scale_bytes, pad, shift) if scale_bytes else None
    call = Call(lib, ids, experts, tokens * top_k if max_rows is None else max_rows, x, row_bytes, scale, scale_bytes, pad, shift, **k)
    assert call.run() == 0
    _gpu.sync()
    call.check(ids)


@pytest.mark.parametrize("experts", [1, 2, 3, 31, 63, 64, 65, 255, 256, 257, 511, 1000, 1023, 1024])
@pytest.mark.parametrize("tokens", [1, 13, 700])
def test_experts(lib, gpu, experts, tokens):
    check(lib, tokens, 4, experts, seed=experts + tokens, wide=experts % 2 == 0)


@pytest.mark.parametrize("tokens,top_k", [(1, 1), (1, 64), (2, 33), (7, 9), (31, 2), (63, 1), (64, 1), (65, 1), (127, 2), (128, 8), (129, 8),
                                          (255, 8), (256, 8), (257, 8), (341, 6), (511, 8), (512, 8), (513, 8), (1000, 3), (2047, 1),
                                          (2048, 2), (2049, 2), (4095, 8), (4096, 8), (4097, 8), (16385, 2), (33000, 8)])
def test_pairs(lib, gpu, tokens, top_k):
    check(lib, tokens, top_k, 40, seed=tokens * top_k, wide=tokens % 2 == 0, scale_bytes=12 if top_k % 2 else 0)


@pytest.mark.parametrize("row_bytes", [1, 2, 3, 15, 16, 17, 31, 33, 100, 1023, 1024, 1040, 4095, 4096, 4097, 5120, 8191, 8192, 16384, 70000])
@pytest.mark.parametrize("pad,shift", [(0, 0), (16, 0), (3, 5)])
def test_row_lengths_pitches_and_alignments(lib, gpu, row_bytes, pad, shift):
    check(lib, 37, 6, 16, seed=row_bytes, row_bytes=row_bytes, scale_bytes=row_bytes // 32 + 1, pad=pad, shift=shift)
    check(lib, 1100, 2, 16, seed=row_bytes, row_bytes=row_bytes, pad=pad, shift=shift)


@pytest.mark.parametrize("scale_bytes", [1, 4, 6, 8, 12, 20, 32, 60, 64, 100, 128, 132, 224, 252, 255, 256, 260, 1000])
@pytest.mark.parametrize("pad,shift,pairs", [(0, 0, True), (4, 4, True), (1, 0, True), (0, 0, False)])
def test_scales_beside_rows(lib, gpu, scale_bytes, pad, shift, pairs):
    """Short rows in whole words are copied by their place where the table of pairs is asked for; others by token."""
    check(lib, 700, 8, 24, seed=scale_bytes, row_bytes=300, scale_bytes=scale_bytes, pad=pad, shift=shift, pairs=pairs, invalid=0.4)
    check(lib, 1500, 3, 24, seed=scale_bytes, row_bytes=5000, scale_bytes=scale_bytes, pad=pad, shift=shift, pairs=pairs, max_rows=2001)
    check(lib, 40, 3, 24, seed=scale_bytes, row_bytes=48, scale_bytes=scale_bytes, pad=pad, shift=shift, pairs=pairs, max_rows=200)


@pytest.mark.parametrize("tokens", [5, 300, 5000])
def test_nothing_but_one_expert_and_nothing_at_all(lib, gpu, tokens):
    check(lib, tokens, 8, 256, skew=False, invalid=0.0)
    check(lib, tokens, 8, 256, invalid=1.0, scale_bytes=8)


@pytest.mark.parametrize("tokens,most", [(1, 3), (16, 50), (16, 0), (300, 1000), (3000, 7), (3000, 9999), (3000, 0), (5000, 50000)])
def test_more_pairs_than_rows_and_more_rows_than_pairs(lib, gpu, tokens, most):
    check(lib, tokens, 8, 60, invalid=0.0, max_rows=most, seed=most, scale_bytes=4)


def test_the_table_alone(lib, gpu):
    for tokens in (3, 500, 9000):
        check(lib, tokens, 5, 100, row_bytes=0, pairs=tokens != 500)


def test_no_tokens(lib, gpu):
    ids = np.zeros((0, 8), dtype=np.int32)
    call = Call(lib, ids, 20, 10, Rows(0, 16, torch.uint8), 16)
    assert call.run() == 0
    _gpu.sync()
    call.check(ids)


def test_rows_far_apart_pass_32_bits_of_offset(lib, gpu):
    rng = np.random.default_rng(3)
    pitch, tokens = 1 << 28, 24
    ids = make_ids(rng, tokens, 1, 7, 0.0, False)
    x = byte_rows(rng, tokens, 5000)
    far = torch.zeros((tokens * pitch,), dtype=torch.uint8, device="cuda")
    call = Call(lib, ids, 7, tokens)
    assert lib.ofi_amd_token_dispatch(ptr(call.ids), m.INT32, tokens, 1, 7, tokens, ptr(call.offset), ptr(call.row_of), None, x.ptr(),
                                      x.pitch, ptr(far), pitch, 5000, None, 0, None, 0, 0, ptr(call.work),
                                      0 if call.work is None else call.work.numel(), _gpu.stream()) == 0
    back = torch.zeros(tokens * pitch, dtype=torch.uint8, device="cuda")  # and read from rows as far apart
    _gpu.sync()
    _, row_of, pair_of, _ = table(ids, 7, tokens)
    for row in range(tokens):
        assert torch.equal(far[row * pitch:row * pitch + 5000], x.t[int(pair_of[row])])
    assert lib.ofi_amd_token_dispatch(ptr(call.ids), m.INT32, tokens, 1, 7, tokens, ptr(call.offset), ptr(call.row_of), None, ptr(far),
                                      pitch, ptr(back), pitch, 5000, None, 0, None, 0, 0, ptr(call.work),
                                      0 if call.work is None else call.work.numel(), _gpu.stream()) == 0
    _gpu.sync()
    for row in range(tokens):
        assert torch.equal(back[row * pitch:row * pitch + 5000], far[int(pair_of[row]) * pitch:int(pair_of[row]) * pitch + 5000])


@pytest.mark.parametrize("tokens", [9, 900, 9000])
def test_another_stream_and_a_replayed_graph(lib, gpu, tokens):
    """Captured once, replayed on ids that change between the replays, with eager calls and synchronizations between them."""
    rng = np.random.default_rng(tokens)
    x = byte_rows(rng, tokens, 256)
    ids = make_ids(rng, tokens, 8, 128, 0.2, True)
    call = Call(lib, ids, 128, tokens * 8, x, 256)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert call.run() == 0
    side.synchronize()
    call.check(ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call.run() == 0
    for k in range(4):
        ids = make_ids(rng, tokens, 8, 128, 0.1 * k, True)
        call.ids.copy_(torch.from_numpy(ids))
        call.rows.t.fill_(0xA5)
        call.offset[:-1] = 5
        graph.replay()
        _gpu.sync()
        call.check(ids)
        other = make_ids(rng, tokens, 8, 128, 0.3, True)
        eager = Call(lib, other, 128, tokens * 8, x, 256)
        assert eager.run() == 0
        _gpu.sync()
        eager.check(other)


def test_refusals(lib, gpu):
    inval, toobig = -errno.EINVAL, -errno.E2BIG
    ids = torch.zeros(40000, dtype=torch.int64, device="cuda")
    t = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    p = t.data_ptr()
    good = dict(ids=ids.data_ptr(), type=m.INT64, tokens=4096, k=8, experts=64, most=32768, offset=p, row_of=p + 4096, pair_of=None, x=None,
                xp=0, rows=None, rp=0, rb=0, s=None, sp=0, sr=None, srp=0, sb=0, work=p + 300000, wb=500000)

    def call(**changed):
        a = dict(good, **changed)
        vp = ctypes.c_void_p
        return lib.ofi_amd_token_dispatch(vp(a["ids"]), a["type"], a["tokens"], a["k"], a["experts"], a["most"], vp(a["offset"]),
                                          vp(a["row_of"]), vp(a["pair_of"]), vp(a["x"]), a["xp"], vp(a["rows"]), a["rp"], a["rb"], vp(a["s"]),
                                          a["sp"], vp(a["sr"]), a["srp"], a["sb"], vp(a["work"]), a["wb"], _gpu.stream())

    assert call() == 0
    assert call(type=m.FLOAT32) == inval and call(k=0) == inval and call(experts=0) == inval
    assert call(experts=1025) == toobig and call(k=65) == toobig and call(tokens=1 << 30) == toobig and call(most=1 << 31) == toobig
    assert call(ids=None) == inval and call(ids=ids.data_ptr() + 4) == inval and call(offset=None) == inval and call(offset=p + 2) == inval
    assert call(row_of=None) == inval and call(row_of=p + 1) == inval and call(pair_of=p + 3) == inval
    need = lib.ofi_amd_token_dispatch_work_bytes(4096, 8, 64)
    assert need > 0 and call(work=None) == inval and call(wb=need - 1) == inval and call(work=p + 300002) == inval and call(wb=need) == 0
    rows = dict(x=p, xp=16, rows=p, rp=16, rb=16)
    assert call(x=p, xp=16, rb=16) == inval and call(rows=p, rp=16, rb=16) == inval
    assert call(**dict(rows, xp=15)) == inval and call(**dict(rows, rp=15)) == inval and call(**dict(rows, rb=0)) == inval
    assert call(**dict(rows, rb=(1 << 24) + 1, xp=1 << 25, rp=1 << 25)) == toobig
    assert call(s=p, sp=16, sr=p, srp=16, sb=16) == inval            # scales without rows
    assert call(**dict(rows, s=p, sp=16, sb=16)) == inval
    _gpu.sync()
    assert _gpu.fetch_async_errors(lib) == 0
