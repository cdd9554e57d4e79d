"""The operators around an expert-parallel exchange, over the sizes they are called at.

A layer normalises the residual stream into 8-bit rows (`norm`), sorts the rows by expert so that what goes to one
peer is one piece (`dispatch`), and weights and sums what comes back (`combine`); training goes the same way back
(`norm_grad`, `combine` without weights, `combine_grad`).  Every case is one call with inputs and output buffers in
hand.  `own` chooses the framework's kernels; without it the same operators run as elementary torch operations.
"""
import ctypes

import numpy as np
import torch

own = False

TYPES = {"bf16": (torch.bfloat16, 9), "f16": (torch.float16, 6), "f32": (torch.float32, 7)}  # numbers of ncclDataType_t
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}
INT32, INT64 = 2, 4
EPS = 1e-6
MOST_BYTES = 2.0e9  # a drawn case moves at most this much; the largest listed one moves more


def listed():
    return [
        # one token of one request: latency
        dict(name="norm_token", path="norm", rows=1, width=4096, type="bf16", train=False, group=128, pad=0),
        # a ragged batch of a small model's training step, rows of an odd width: no row but the first is aligned
        dict(name="norm_ragged", path="norm", rows=1331, width=1999, type="f16", train=True, group=0, pad=0),
        # the prompts of a serving step
        dict(name="norm_prompt", path="norm", rows=16384, width=8192, type="bf16", train=False, group=128, pad=0),
        # the way back of a training step
        dict(name="norm_grad_step", path="norm_grad", rows=16384, width=4096, type="bf16", through=True, pad=0),
        # one token to its experts, 8-bit rows with scales: latency
        dict(name="dispatch_token", path="dispatch", tokens=1, top_k=8, experts=256, width=4096, type="e4m3", ranks=1,
             wide_ids=False, pad=0),
        # what one of eight ranks keeps of a batch: most pairs belong to experts elsewhere
        dict(name="dispatch_local", path="dispatch", tokens=4096, top_k=8, experts=256, width=5120, type="e4m3", ranks=8,
             wide_ids=True, pad=0),
        # a training step's tokens to all experts
        dict(name="dispatch_step", path="dispatch", tokens=32768, top_k=8, experts=128, width=4096, type="bf16", ranks=1,
             wide_ids=True, pad=0),
        # the gradient of a ragged batch's dispatch: sums without weights, rows of an odd width
        dict(name="dispatch_grad_ragged", path="combine", tokens=3001, top_k=5, experts=60, width=1023, type="f32", ranks=2,
             weighted=False, add=False, pad=0),
        # a few requests' tokens back from their experts
        dict(name="combine_token", path="combine", tokens=4, top_k=8, experts=256, width=4096, type="bf16", ranks=1,
             weighted=True, add=True, pad=0),
        # a step's tokens back, added to what the shared expert made
        dict(name="combine_step", path="combine", tokens=16384, top_k=8, experts=128, width=4096, type="bf16", ranks=1,
             weighted=True, add=True, pad=0),
        # gradients of a ragged batch, some pairs elsewhere
        dict(name="combine_grad_ragged", path="combine_grad", tokens=1331, top_k=6, experts=60, width=1999, type="f16",
             ranks=2, weighted=True, pad=0),
        # gradients of a training step
        dict(name="combine_grad_step", path="combine_grad", tokens=16384, top_k=8, experts=128, width=4096, type="bf16",
             ranks=1, weighted=True, pad=0),
    ]


def _log_int(rng, lo, hi):
    """Log-uniform whole number in [lo, hi], odd ones as likely as even ones."""
    return int(round(lo * (hi / lo) ** rng.random()))


def _width(rng, lo=256, hi=8192):
    """Three widths of four are whole groups of 128, the others anything."""
    w = _log_int(rng, lo, hi)
    return w if rng.random() < 0.25 else max(128, (w + 64) // 128 * 128)


def draw(rng):
    # 24 x 128 is a size that no configuration here has
    return {key: 25 * 128 if type(value) is int and value == 24 * 128 else value for key, value in _drawn(rng).items()}


def _drawn(rng):
    path = rng.choice(["norm", "norm", "norm_grad", "dispatch", "dispatch", "combine", "combine", "combine_grad"])
    width = _width(rng)
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    pad = rng.choice([0, 0, 8, 3])
    if path in ("norm", "norm_grad"):
        rows = _log_int(rng, 1, 32768)
        rows = max(1, min(rows, int(MOST_BYTES / (width * SIZE[kind] * 5))))
        if path == "norm":
            return dict(path=path, rows=rows, width=width, type=kind, train=rng.random() < 0.4,
                        group=rng.choice([128, 128, 64, 32, 0]), pad=pad)
        return dict(path=path, rows=rows, width=width, type=kind, through=rng.random() < 0.7, pad=pad)
    top_k, experts = rng.choice([1, 2, 4, 6, 8, 8]), rng.choice([8, 32, 60, 64, 128, 256, 384])
    ranks = rng.choice([1, 1, 2, 4])
    if path == "dispatch":
        kind = rng.choice(["e4m3", "e4m3", "bf16", "f32"])
        if kind == "e4m3":
            width = max(128, (width + 64) // 128 * 128)
    tokens = _log_int(rng, 1, 32768)
    tokens = max(1, min(tokens, int(MOST_BYTES / (width * SIZE[kind] * (2 * top_k + 2)))))
    case = dict(path=path, tokens=tokens, top_k=top_k, experts=experts, width=width, type=kind, ranks=ranks)
    if path == "dispatch":
        case.update(wide_ids=rng.random() < 0.5, pad=rng.choice([0, 0, 16, 5]))
    elif path == "combine":
        case.update(weighted=rng.random() < 0.7, add=rng.random() < 0.5, pad=pad)
    else:
        case.update(weighted=rng.random() < 0.8, pad=pad)
    return case


# ---- inputs ------------------------------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(g, n, width, dtype, pad):
    """n rows of a residual stream: near normal, a few channels far larger; `pad` more elements from row to row."""
    full = torch.empty(n, width + pad, device="cuda", dtype=dtype)
    big = 1.0 + 15.0 * (torch.rand(width + pad, generator=g, device="cuda") < 0.004)
    at = 0
    while at < n:  # in pieces: the 32-bit values of a whole input need not exist at once
        k = min(n - at, max(1, (1 << 26) // (width + pad)))
        full[at:at + k] = torch.randn(k, width + pad, generator=g, device="cuda") * big
        at += k
    return full[:, :width]


def _groups(width, group):
    return 1 if group == 0 else -(-width // group)


def _held(tokens, top_k, ranks):
    """Rows of the sorted buffer: a rank that keeps a part of the experts has room for twice its even share."""
    pairs = tokens * top_k
    return pairs if ranks == 1 or pairs <= 4096 else -(-2 * pairs // ranks)


def _routing(g, case, wide=True):
    """Expert of every pair and its weight as a router leaves them: distinct experts of a token, some experts asked for
    more than others; of `ranks` ranks this one holds the first share of the experts and numbers the others -1."""
    T, K, E = case["tokens"], case["top_k"], case["experts"]
    logits = torch.randn(T, E, generator=g, device="cuda") + 0.5 * torch.randn(E, generator=g, device="cuda")
    top, ids = torch.topk(logits, K, dim=1)
    weight = torch.softmax(top, dim=1).contiguous()
    if case["ranks"] > 1:
        ids = torch.where(ids < E // case["ranks"], ids, torch.full_like(ids, -1))
    return (ids if wide else ids.to(torch.int32)).contiguous(), weight


def _sorted(ids, experts, held):
    """(offsets, row of each pair, pair of each row) in elementary torch operations."""
    flat = ids.reshape(-1).to(torch.int64)
    valid = (flat >= 0) & (flat < experts)
    key, order = torch.sort(torch.where(valid, flat, torch.full_like(flat, experts)), stable=True)
    offset = torch.searchsorted(key, torch.arange(experts + 1, device=flat.device)).clamp(max=held)
    row = torch.empty_like(order)
    row[order] = torch.arange(flat.numel(), device=flat.device)
    row = torch.where(valid & (row < held), row, torch.full_like(row, -1))
    pair = order[:held]
    pair = torch.where(torch.arange(pair.numel(), device=flat.device) < offset[-1], pair, torch.full_like(pair, -1))
    return offset.to(torch.int32), row.to(torch.int32).reshape(ids.shape), pair.to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=dict(case))
    path, width, pad = case["path"], case["width"], case["pad"]
    if path in ("norm", "norm_grad"):
        dtype, n = TYPES[case["type"]][0], case["rows"]
        s["x"] = _rows(g, n, width, dtype, pad)
        s["gain"] = (1.0 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(dtype)
        if path == "norm":
            s["residual"] = _rows(g, n, width, dtype, pad)
            s["sum"] = torch.empty(n, width, device="cuda", dtype=dtype)
            s["rstd"] = torch.empty(n, device="cuda")
            if case["train"]:
                s["out"] = torch.empty(n, width, device="cuda", dtype=dtype)
            else:
                s["q"] = torch.empty(n, width, device="cuda", dtype=torch.float8_e4m3fn)
                s["scale"] = torch.empty(n, _groups(width, case["group"]), device="cuda")
        else:
            s["dout"] = (torch.randn(n, width, generator=g, device="cuda") * 0.01).to(dtype)
            s["through"] = (torch.randn(n, width, generator=g, device="cuda") * 0.01).to(dtype) if case["through"] else None
            s["rstd"] = torch.rsqrt(s["x"].float().square().mean(dim=1) + EPS)
            s["dx"] = torch.empty(n, width, device="cuda", dtype=dtype)
            s["dgain"] = torch.empty(width, device="cuda")
        return s
    T, K, E = case["tokens"], case["top_k"], case["experts"]
    held = _held(T, K, case["ranks"])
    ids, weight = _routing(g, case, case.get("wide_ids", True))
    if path == "dispatch":
        s["ids"] = ids
        if case["type"] == "e4m3":
            x = torch.randn(T, width + pad, generator=g, device="cuda").clamp(-4, 4) * 100.0
            s["x"] = x.to(torch.float8_e4m3fn)[:, :width]
            s["scale"] = torch.rand(T, width // 128, generator=g, device="cuda") + 0.5
            s["scale_rows"] = torch.zeros(held, width // 128, device="cuda")
        else:
            s["x"] = _rows(g, T, width, TYPES[case["type"]][0], pad)
            s["scale"] = s["scale_rows"] = None
        s["rows"] = torch.zeros(held, width, device="cuda", dtype=s["x"].dtype)  # rows that no pair has stay as they are
        s["offset"] = torch.empty(E + 1, device="cuda", dtype=torch.int32)
        s["row_of"] = torch.empty(T, K, device="cuda", dtype=torch.int32)
        s["pair_of"] = torch.empty(held, device="cuda", dtype=torch.int32)
        return s
    dtype = TYPES[case["type"]][0]
    _, s["row_of"], s["pair_of"] = _sorted(ids, E, held)
    s["weight"] = weight if case["weighted"] else None
    s["rows"] = _rows(g, held, width, dtype, pad)
    if path == "combine":
        s["add"] = _rows(g, T, width, dtype, 0) if case["add"] else None
        s["out"] = torch.empty(T, width, device="cuda", dtype=dtype)
    else:
        s["dout"] = _rows(g, T, width, dtype, 0)
        s["drows"] = torch.zeros(held, width, device="cuda", dtype=dtype)
        s["dweight"] = torch.empty(T, K, device="cuda")
    return s


# ---- the operators as elementary operations --------------------------------------------------------------------


def _plain_norm(s):
    case = s["case"]
    dtype = s["x"].dtype
    total = s["x"].float() + s["residual"].float()
    rstd = torch.rsqrt(total.square().mean(dim=1, keepdim=True) + EPS)
    normed = total * rstd * s["gain"].float()
    if case["train"]:
        return dict(sum=total.to(dtype), out=normed.to(dtype), rstd=rstd[:, 0])
    n, width = normed.shape
    group = case["group"] or width
    groups = _groups(width, group)
    whole = torch.nn.functional.pad(normed, (0, groups * group - width)).view(n, groups, group)
    scale = (whole.abs().amax(dim=2) / 448.0).clamp(min=2.0 ** -126)
    q = (whole / scale[:, :, None]).view(n, groups * group)[:, :width].to(torch.float8_e4m3fn)
    return dict(sum=total.to(dtype), q=q, scale=scale)


def _plain_norm_grad(s):
    x, dout, gain = s["x"].float(), s["dout"].float(), s["gain"].float()
    rstd = s["rstd"][:, None]
    h = x * rstd
    dn = dout * gain
    dx = rstd * (dn - h * (dn * h).mean(dim=1, keepdim=True))
    if s["through"] is not None:
        dx = dx + s["through"].float()
    return dict(dx=dx.to(s["x"].dtype), dgain=(dout * h).sum(dim=0))


def _plain_dispatch(s):
    case = s["case"]
    offset, row_of, pair_of = _sorted(s["ids"], case["experts"], s["rows"].shape[0])
    token = pair_of.clamp(min=0).to(torch.int64) // case["top_k"]
    none = (pair_of < 0)[:, None]
    x = s["x"].view(torch.uint8) if case["type"] == "e4m3" else s["x"]
    rows = x.index_select(0, token).masked_fill_(none, 0)
    out = dict(offset=offset, row_of=row_of, pair_of=pair_of, rows=rows.view(s["x"].dtype))
    if s["scale"] is not None:
        out["scale_rows"] = s["scale"].index_select(0, token).masked_fill_(none, 0)
    return out


def _plain_combine(s):
    at = s["row_of"].to(torch.int64)
    T, K = at.shape
    picked = s["rows"].index_select(0, at.clamp(min=0).reshape(-1)).float().view(T, K, -1)
    if s["weight"] is not None:
        picked = picked * s["weight"][:, :, None]
    out = torch.where((at >= 0)[:, :, None], picked, torch.zeros((), device=at.device)).sum(dim=1)
    if s["add"] is not None:
        out = out + s["add"].float()
    return dict(out=out.to(s["rows"].dtype))


def _plain_combine_grad(s):
    at, pair = s["row_of"].to(torch.int64), s["pair_of"].to(torch.int64)
    T, K = at.shape
    dout = s["dout"].float()
    picked = s["rows"].index_select(0, at.clamp(min=0).reshape(-1)).float().view(T, K, -1)
    dweight = torch.where(at >= 0, (picked * dout[:, None, :]).sum(dim=2), torch.zeros((), device=at.device))
    drows = dout.index_select(0, pair.clamp(min=0) // K)
    if s["weight"] is not None:
        drows = drows * s["weight"].reshape(-1)[pair.clamp(min=0)][:, None]
    drows = drows.masked_fill_((pair < 0)[:, None], 0)
    return dict(drows=drows.to(s["rows"].dtype), dweight=dweight)


# ---- the framework's entry points ------------------------------------------------------------------------------


def _lib():
    import aws_ofi_nccl_amd as m
    return m.load(), m.check


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _pitch(t):
    return t.stride(0) * t.element_size()


def _own_norm(s):
    lib, check = _lib()
    case, x, r, total = s["case"], s["x"], s["residual"], s["sum"]
    code = TYPES[case["type"]][1]
    if case["train"]:
        out = s["out"]
        check(lib.ofi_amd_rms_norm(x.data_ptr(), _pitch(x), r.data_ptr(), _pitch(r), s["gain"].data_ptr(), code, case["rows"],
                                   case["width"], code, EPS, total.data_ptr(), _pitch(total), out.data_ptr(), _pitch(out), None, 0,
                                   None, 0, 0, s["rstd"].data_ptr(), _stream()), "rms_norm")
        return dict(sum=total, out=out, rstd=s["rstd"])
    q, scale = s["q"], s["scale"]
    check(lib.ofi_amd_rms_norm(x.data_ptr(), _pitch(x), r.data_ptr(), _pitch(r), s["gain"].data_ptr(), code, case["rows"],
                               case["width"], code, EPS, total.data_ptr(), _pitch(total), None, 0, q.data_ptr(), _pitch(q),
                               scale.data_ptr(), _pitch(scale), case["group"], None, _stream()), "rms_norm")
    return dict(sum=total, q=q, scale=scale)


def _own_norm_grad(s):
    lib, check = _lib()
    case, x, dout, through, dx = s["case"], s["x"], s["dout"], s["through"], s["dx"]
    code = TYPES[case["type"]][1]
    if "work" not in s:
        s["work"] = torch.empty(lib.ofi_amd_rms_norm_grad_work_bytes(case["rows"], case["width"]), dtype=torch.uint8, device="cuda")
    check(lib.ofi_amd_rms_norm_grad(dout.data_ptr(), _pitch(dout), x.data_ptr(), _pitch(x), s["rstd"].data_ptr(),
                                    s["gain"].data_ptr(), code, case["rows"], case["width"], code,
                                    through.data_ptr() if through is not None else None,
                                    _pitch(through) if through is not None else 0, dx.data_ptr(), _pitch(dx),
                                    s["dgain"].data_ptr(), s["work"].data_ptr(), s["work"].numel(), _stream()), "rms_norm_grad")
    return dict(dx=dx, dgain=s["dgain"])


def _own_dispatch(s):
    lib, check = _lib()
    case, ids, x, rows, scale = s["case"], s["ids"], s["x"], s["rows"], s["scale"]
    if "work" not in s:
        n = lib.ofi_amd_token_dispatch_work_bytes(case["tokens"], case["top_k"], case["experts"])
        s["work"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    scale_rows = s["scale_rows"]
    check(lib.ofi_amd_token_dispatch(ids.data_ptr(), INT64 if case["wide_ids"] else INT32, case["tokens"], case["top_k"],
                                     case["experts"], rows.shape[0], s["offset"].data_ptr(), s["row_of"].data_ptr(),
                                     s["pair_of"].data_ptr(), x.data_ptr(), _pitch(x), rows.data_ptr(), _pitch(rows),
                                     case["width"] * x.element_size(),
                                     scale.data_ptr() if scale is not None else None,
                                     _pitch(scale) if scale is not None else 0,
                                     scale_rows.data_ptr() if scale is not None else None,
                                     _pitch(scale_rows) if scale is not None else 0,
                                     scale.shape[1] * 4 if scale is not None else 0,
                                     s["work"].data_ptr(), s["work"].numel(), _stream()), "token_dispatch")
    out = dict(offset=s["offset"], row_of=s["row_of"], pair_of=s["pair_of"], rows=rows)
    if scale is not None:
        out["scale_rows"] = scale_rows
    return out


def _own_combine(s):
    lib, check = _lib()
    case, rows, add, out, weight = s["case"], s["rows"], s["add"], s["out"], s["weight"]
    check(lib.ofi_amd_token_combine(rows.data_ptr(), _pitch(rows), rows.shape[0], s["row_of"].data_ptr(),
                                    weight.data_ptr() if weight is not None else None, case["tokens"], case["top_k"],
                                    case["width"], TYPES[case["type"]][1], add.data_ptr() if add is not None else None,
                                    _pitch(add) if add is not None else 0, out.data_ptr(), _pitch(out), _stream()), "token_combine")
    return dict(out=out)


def _own_combine_grad(s):
    lib, check = _lib()
    case, rows, dout, drows, weight = s["case"], s["rows"], s["dout"], s["drows"], s["weight"]
    check(lib.ofi_amd_token_combine_grad(dout.data_ptr(), _pitch(dout), rows.data_ptr(), _pitch(rows), rows.shape[0],
                                         s["row_of"].data_ptr(), weight.data_ptr() if weight is not None else None,
                                         case["tokens"], case["top_k"], case["width"], TYPES[case["type"]][1],
                                         drows.data_ptr(), _pitch(drows), s["dweight"].data_ptr(), _stream()),
          "token_combine_grad")
    return dict(drows=drows, dweight=s["dweight"])


PLAIN = dict(norm=_plain_norm, norm_grad=_plain_norm_grad, dispatch=_plain_dispatch, combine=_plain_combine,
             combine_grad=_plain_combine_grad)
OWN = dict(norm=_own_norm, norm_grad=_own_norm_grad, dispatch=_own_dispatch, combine=_own_combine,
           combine_grad=_own_combine_grad)


def run(state):
    return (OWN if own else PLAIN)[state["case"]["path"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------


def work(case):
    path, width, size = case["path"], case["width"], SIZE[case["type"]]
    if path == "norm":
        n = case["rows"]
        row = width * size
        out = row + 4 if case["train"] else width + 4 * _groups(width, case["group"])
        return dict(bytes=n * (3 * row + out) + row, flops=n * width * (6 if case["train"] else 9))
    if path == "norm_grad":
        n = case["rows"]
        row = width * size
        return dict(bytes=n * ((4 if case["through"] else 3) * row + 4) + row + 4 * width, flops=n * width * 10)
    T, K, E = case["tokens"], case["top_k"], case["experts"]
    pairs = T * K
    local = (E // case["ranks"]) / E
    kept = min(pairs * local, _held(T, K, case["ranks"]))    # pairs with a row, as expected
    touched = T * (1.0 - (1.0 - local) ** K)                 # tokens with such a pair
    row = width * size
    if path == "dispatch":
        row += 4 * (width // 128) if case["type"] == "e4m3" else 0
        tables = pairs * (8 if case["wide_ids"] else 4) + 4 * (E + 1) + 4 * pairs + 4 * _held(T, K, case["ranks"])
        return dict(bytes=(kept + touched) * row + tables, flops=0)
    weights = 4 * pairs if case["weighted"] else 0
    if path == "combine":
        return dict(bytes=kept * row + T * row * (2 if case["add"] else 1) + 4 * pairs + weights, flops=2 * kept * width)
    return dict(bytes=touched * row + 2 * kept * row + 8 * pairs + weights, flops=3 * kept * width)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------


def _table(case, ids):
    """Offsets, row of each pair and pair of each row from the definition: experts in order, pairs of one in order."""
    flat = ids.cpu().numpy().reshape(-1).astype(np.int64)
    E, held = case["experts"], _held(case["tokens"], case["top_k"], case["ranks"])
    where = np.flatnonzero((flat >= 0) & (flat < E))
    where = where[np.lexsort((where, flat[where]))]
    offset = np.minimum(np.concatenate([[0], np.cumsum(np.bincount(flat[where], minlength=E))]), held)
    row_of, pair_of = np.full(flat.size, -1, dtype=np.int64), np.full(held, -1, dtype=np.int64)
    kept = where[:held]
    row_of[kept] = np.arange(kept.size)
    pair_of[:kept.size] = kept
    return offset, row_of.reshape(ids.shape), pair_of


def exact(case, seed):
    s = prepare(case, seed)
    path = case["path"]
    if path == "norm":
        v = s["x"].double() + s["residual"].double()
        r = 1.0 / torch.sqrt(torch.mean(v * v, dim=1) + EPS)
        n = v * r[:, None] * s["gain"].double()
        if case["train"]:
            return dict(sum=v, out=n, rstd=r)
        group = case["group"] or case["width"]
        q, scales = torch.empty_like(n), []
        for lo in range(0, case["width"], group):
            part = n[:, lo:lo + group]
            m = torch.clamp(part.abs().max(dim=1).values / 448.0, min=2.0 ** -126)
            q[:, lo:lo + group] = part / m[:, None]
            scales.append(m)
        return dict(sum=v, q=q, scale=torch.stack(scales, dim=1))
    if path == "norm_grad":
        v, d, g, r = s["x"].double(), s["dout"].double(), s["gain"].double(), s["rstd"].double()
        h = v * r[:, None]
        along = (d * g * h).sum(dim=1) / case["width"]
        dx = r[:, None] * (d * g - h * along[:, None])
        if s["through"] is not None:
            dx += s["through"].double()
        return dict(dx=dx, dgain=(d * h).sum(dim=0))
    T, K = case["tokens"], case["top_k"]
    if path == "dispatch":
        offset, row_of, pair_of = _table(case, s["ids"])
        pairs = torch.from_numpy(pair_of).cuda()
        at = torch.div(pairs.clamp(min=0), K, rounding_mode="floor")
        rows = s["x"].to(torch.float32).double()[at]
        rows[pairs < 0] = 0.0
        out = dict(offset=torch.from_numpy(offset).int(), row_of=torch.from_numpy(row_of).int(),
                   pair_of=torch.from_numpy(pair_of).int(), rows=rows)
        if s["scale"] is not None:
            out["scale_rows"] = s["scale"].double()[at]
            out["scale_rows"][pairs < 0] = 0.0
        return out
    row_of, weight = s["row_of"].long(), s["weight"]
    weight = torch.ones(T, K, device="cuda", dtype=torch.float64) if weight is None else weight.double()
    if path == "combine":
        out = torch.zeros(T, case["width"], device="cuda", dtype=torch.float64) if s["add"] is None else s["add"].double()
        for k in range(K):
            here = torch.nonzero(row_of[:, k] >= 0)[:, 0]
            out[here] += weight[here, k, None] * s["rows"][row_of[here, k]].double()
        return dict(out=out)
    drows = torch.zeros(s["drows"].shape, device="cuda", dtype=torch.float64)
    dweight = torch.zeros(T, K, device="cuda", dtype=torch.float64)
    for k in range(K):
        here = torch.nonzero(row_of[:, k] >= 0)[:, 0]
        dout = s["dout"][here].double()
        drows[row_of[here, k]] = weight[here, k, None] * dout
        dweight[here, k] = (dout * s["rows"][row_of[here, k]].double()).sum(dim=1)
    return dict(drows=drows, dweight=dweight)
