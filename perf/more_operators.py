"""The experts of an expert-parallel layer, over the sizes they are called at.

Rows sorted by expert, as the dispatch leaves them, go through each expert's gated block (`gated`) and the product behind
it (`product`, with one expert an ordinary layer's product with bias, activation and residual).  Training keeps what the
activation was taken of, in 8 bits or 16, and goes back through it (`hidden_grad`), to the rows (`rows_grad`) and to the
weights (`weight_grad`).  Every case is one call with inputs and output buffers in hand.  `own` chooses the framework's
kernels; without it the same operators run as elementary torch operations.
"""
import ctypes
import math

import torch

own = False

TYPES = {"bf16": (torch.bfloat16, 9), "f16": (torch.float16, 6), "f32": (torch.float32, 7),
         "e4m3": (torch.float8_e4m3fn, 10)}  # numbers of ncclDataType_t
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
BLOCK = 128          # columns of a row that share a scale; rows and columns of a weight that do
MOST_FLOPS = 1.0e12  # a drawn case computes at most this much and has at most MOST_WEIGHTS weights; a listed one has more of both
MOST_WEIGHTS = 4.0e8


def listed():
    return [
        # one token to its experts in 8 bits, on a rank that holds 32 of them: latency, weights read once
        dict(name="gated_token", path="gated", rows=8, experts=32, width=4096, inner=2048, type="e4m3", act="silu",
             out="e4m3", saved=None, spare=0, pad=0),
        # the prompts of a serving step: 8-bit rows and weights, 8-bit rows for the product behind
        dict(name="gated_prompt", path="gated", rows=16384, experts=32, width=4096, inner=2048, type="e4m3", act="silu",
             out="e4m3", saved=None, spare=16384, pad=0),
        # a training step's rows, 8-bit checkpoints for the way back
        dict(name="gated_step", path="gated", rows=32768, experts=32, width=4096, inner=2048, type="bf16", act="silu",
             out="bf16", saved="e4m3", spare=0, pad=0),
        # the product behind the gated block, for the same token
        dict(name="product_token", path="product", rows=8, experts=32, width=2048, out_width=4096, type="e4m3",
             act="none", out="bf16", bias=False, residual=False, saved=None, spare=0, pad=0),
        # an ordinary layer's product: one expert that has all rows, bias, activation and residual
        dict(name="product_dense", path="product", rows=8192, experts=0, width=4096, out_width=4096, type="bf16",
             act="gelu", out="bf16", bias=True, residual=True, saved=None, spare=0, pad=0),
        # the product behind the gated block of a training step
        dict(name="product_step", path="product", rows=32768, experts=32, width=2048, out_width=4096, type="bf16",
             act="none", out="bf16", bias=False, residual=False, saved=None, spare=0, pad=0),
        # back through the product and the gated block, from 8-bit checkpoints
        dict(name="hidden_grad_step", path="hidden_grad", rows=32768, experts=32, width=4096, inner=2048, type="bf16",
             gated=True, act="silu", saved="e4m3", spare=0, pad=0),
        # a small model's ragged batch through one activation, odd widths: no row but the first is aligned
        dict(name="hidden_grad_ragged", path="hidden_grad", rows=1331, experts=5, width=999, inner=1023, type="f16",
             gated=False, act="gelu", saved="f16", spare=100, pad=0),
        # the gradient of a training step's rows
        dict(name="rows_grad_step", path="rows_grad", rows=32768, experts=32, width=4096, out_width=4096, type="bf16",
             add=False, spare=0, pad=0),
        # the gradient of a fine-tuning batch's rows, some experts without any, added to what another branch left
        dict(name="rows_grad_ragged", path="rows_grad", rows=700, experts=60, width=1408, out_width=1000, type="f16",
             add=True, spare=0, pad=8),
        # the weights' gradients of a training step, added in float32 to the sum of those before
        dict(name="weight_grad_step", path="weight_grad", rows=32768, experts=32, width=4096, out_width=4096,
             type="bf16", out="f32", accumulate=True, bias=False, spare=0, pad=0),
        # the weights' and biases' gradients of a ragged batch, odd widths, some experts without rows
        dict(name="weight_grad_ragged", path="weight_grad", rows=1331, experts=60, width=1023, out_width=777,
             type="bf16", out="bf16", accumulate=False, bias=True, spare=0, pad=3),
    ]


def _log_int(rng, lo, hi):
    """Log-uniform whole number in [lo, hi], odd ones as likely as even ones."""
    return int(round(lo * (hi / lo) ** rng.random()))


def _width(rng, lo=128, hi=8192):
    """Three widths of four are whole blocks, the others anything."""
    w = _log_int(rng, lo, hi)
    return w if rng.random() < 0.25 else max(BLOCK, (w + BLOCK // 2) // BLOCK * BLOCK)


def draw(rng):
    path = rng.choice(["gated", "gated", "product", "product", "hidden_grad", "rows_grad", "weight_grad"])
    serving = path in ("gated", "product")
    case = dict(path=path, rows=_log_int(rng, 1, 32768), experts=rng.choice([0, 1, 4, 8, 16, 32, 60, 64]), width=_width(rng))
    other = "inner" if path in ("gated", "hidden_grad") else "out_width"
    case[other] = _width(rng, hi=4096)
    case["type"] = rng.choice(["bf16", "f16", "e4m3", "e4m3"] if serving else ["bf16", "bf16", "f16"])
    sixteen = case["type"] if case["type"] != "e4m3" else "bf16"
    if path == "gated":
        case.update(act=rng.choice(["silu", "silu", "gelu"]), out=rng.choice(["e4m3", sixteen]),
                    saved=rng.choice([None, None, "e4m3", sixteen]))
    elif path == "product":
        case.update(act=rng.choice(["none", "none", "silu", "gelu", "relu"]), out=sixteen, bias=rng.random() < 0.4,
                    residual=rng.random() < 0.4, saved=rng.choice([None, None, None, "e4m3"]))
    elif path == "hidden_grad":
        case.update(gated=rng.random() < 0.7, act=rng.choice(["silu", "silu", "gelu", "relu"]), saved=rng.choice(["e4m3", sixteen]))
    elif path == "rows_grad":
        case.update(add=rng.random() < 0.4)
    else:
        case.update(out=rng.choice(["f32", case["type"]]), accumulate=rng.random() < 0.4, bias=rng.random() < 0.3)
    parts = 2 if path == "gated" else 1
    E = max(1, case["experts"])
    while E * parts * case["width"] * case[other] > MOST_WEIGHTS:
        case["width"] = max(BLOCK, case["width"] // 2)
    case["rows"] = max(1, min(case["rows"], int(MOST_FLOPS / (2 * parts * case["width"] * case[other]))))
    case.update(spare=rng.choice([0, 0, case["rows"]]) if case["experts"] else 0, pad=rng.choice([0, 0, 8, 3]))
    if case["type"] == "e4m3":
        case["pad"] = rng.choice([0, 0, 16, 5])
    return case


# ---- inputs ------------------------------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _blocks(n):
    return -(-n // BLOCK)


def _matrix(g, n, width, dtype, pad, size):
    """n rows near normal of the given size; `pad` more elements from row to row."""
    full = torch.empty(n, width + pad, device="cuda", dtype=dtype)
    at = 0
    while at < n:  # in pieces: the 32-bit values of a whole input need not exist at once
        k = min(n - at, max(1, (1 << 26) // (width + pad)))
        full[at:at + k] = (torch.randn(k, width + pad, generator=g, device="cuda") * size).clamp_(-448.0, 448.0)  # e4m3's largest
        at += k
    return full[:, :width]


def _rows(g, n, width, kind, pad, size=1.0):
    """(rows, scales): 8-bit rows are values up to their type's largest, one scale to each block of columns."""
    if kind != "e4m3":
        return _matrix(g, n, width, TYPES[kind][0], pad, size), None
    q = _matrix(g, n, width, TYPES[kind][0], pad, 130.0)
    scale = (torch.rand(n, _blocks(width), generator=g, device="cuda") + 0.5) * (size / 130.0)
    return q, scale


def _weights(g, experts, parts, n, width, kind):
    """(weights, scales): [experts, parts * n, width], of a size that keeps a product's variance; 8-bit ones have a scale to each
    block of 128 x 128 of a part."""
    size = width ** -0.5
    if kind != "e4m3":
        return _matrix(g, experts * parts * n, width, TYPES[kind][0], 0, size).view(experts, parts * n, width), None
    q = _matrix(g, experts * parts * n, width, TYPES[kind][0], 0, 130.0).view(experts, parts * n, width)
    scale = (torch.rand(experts, parts, _blocks(n), _blocks(width), generator=g, device="cuda") + 0.5) * (size / 130.0)
    return q, scale


def _offsets(g, case):
    """First row of each expert and the rows in all, as a router leaves them: some experts are asked for more than others."""
    if not case["experts"]:
        return None
    E, R = case["experts"], case["rows"]
    popular = torch.softmax(0.5 * torch.randn(E, generator=g, device="cuda"), dim=0)
    if R <= E // 2:  # a token's choices are distinct experts
        chosen = torch.multinomial(popular, R, replacement=False, generator=g)
    else:
        chosen = torch.multinomial(popular, R, replacement=True, generator=g)
    count = torch.bincount(chosen, minlength=E)
    return torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), torch.cumsum(count, 0)]).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=dict(case))
    path, width, pad, kind = case["path"], case["width"], case["pad"], case["type"]
    R = case["rows"] + case["spare"]  # rows behind the last expert's are left as they are
    E = max(1, case["experts"])
    s["max_rows"] = R
    s["offset"] = _offsets(g, case)
    empty = lambda n, w, k: torch.zeros(n, w, device="cuda", dtype=TYPES[k][0])
    if path in ("gated", "product"):
        parts, n = (2, case["inner"]) if path == "gated" else (1, case["out_width"])
        s["x"], s["scale"] = _rows(g, R, width, kind, pad)
        s["w"], s["w_scale"] = _weights(g, E, parts, n, width, kind)
        s["out"] = empty(R, n, case["out"])
        s["out_scale"] = torch.zeros(R, _blocks(n), device="cuda") if case["out"] == "e4m3" else None
        if case["saved"]:
            s["saved"] = empty(R, parts * n, case["saved"])
            s["saved_scale"] = torch.zeros(R, parts * _blocks(n), device="cuda") if case["saved"] == "e4m3" else None
        else:
            s["saved"] = s["saved_scale"] = None
        if path == "product":
            dtype = TYPES[case["out"]][0]
            s["bias"] = (0.1 * torch.randn(E, n, generator=g, device="cuda")).to(dtype) if case["bias"] else None
            s["residual"] = _matrix(g, R, n, dtype, 0, 1.0) if case["residual"] else None
        return s
    if path == "hidden_grad":
        parts, n = (2 if case["gated"] else 1), case["inner"]
        s["dout"], _ = _rows(g, R, width, kind, pad, 0.01)
        s["w"], _ = _weights(g, E, 1, width, n, kind)  # the product's behind: [experts, width, inner]
        s["saved"], scale = _rows(g, R, parts * n, case["saved"], 0)
        if scale is not None:  # the blocks of each part begin with it
            scale = (torch.rand(R, parts * _blocks(n), generator=g, device="cuda") + 0.5) / 130.0
        s["saved_scale"] = scale
        s["dsaved"], s["hidden"] = empty(R, parts * n, kind), empty(R, n, kind)
        return s
    n = case["out_width"]
    s["dout"], _ = _rows(g, R, n, kind, pad, 0.01)
    if path == "rows_grad":
        s["w"], _ = _weights(g, E, 1, n, width, kind)
        s["add"] = _matrix(g, R, width, TYPES[kind][0], 0, 0.01) if case["add"] else None
        s["drows"] = empty(R, width, kind)
        return s
    s["x"], _ = _rows(g, R, width, kind, pad)
    s["dw"] = torch.empty(E, n, width, device="cuda", dtype=TYPES[case["out"]][0])
    s["before"] = (0.1 * torch.randn(E, n, width, generator=g, device="cuda")).to(s["dw"].dtype) if case["accumulate"] else None
    s["dbias"] = torch.zeros(E, n, device="cuda") if case["bias"] else None
    return s


# ---- the operators as elementary operations --------------------------------------------------------------------


def _runs(s):
    """(expert, first row, row behind the last) of every expert that has rows."""
    if s["offset"] is None:
        return [(0, 0, s["max_rows"])]
    at = s["offset"].tolist()
    return [(e, at[e], at[e + 1]) for e in range(len(at) - 1) if at[e + 1] > at[e]]


def _act(kind, v):
    if kind == "none":
        return v
    if kind == "relu":
        return v.clamp(min=0)
    if kind == "silu":
        return v / (1 + torch.exp(-v))
    return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))


def _slope(kind, v):
    if kind == "none":
        return torch.ones_like(v)
    if kind == "relu":
        return (v > 0).to(v.dtype)
    if kind == "silu":
        sig = 1 / (1 + torch.exp(-v))
        return sig * (1 + v * (1 - sig))
    return 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) * (0.5 / math.pi) ** 0.5


def _spread(scale, width):
    """A scale for every column."""
    return scale.repeat_interleave(BLOCK, dim=-1)[..., :width]


def _values(q, scale):
    return q.float() if scale is None else q.float() * _spread(scale, q.shape[-1])


def _weight_values(s, e, parts, n):
    w = s["w"][e].float()
    if s["w_scale"] is not None:
        blocks = s["w_scale"][e].repeat_interleave(BLOCK, dim=1)[:, :n].reshape(parts * n, -1)
        w = w * _spread(blocks, w.shape[1])
    return w


def _to_blocks(v):
    """(8-bit values, scales) of float32 rows."""
    n, width = v.shape
    blocks = _blocks(width)
    whole = torch.nn.functional.pad(v, (0, blocks * BLOCK - width)).view(n, blocks, BLOCK)
    scale = (whole.abs().amax(dim=2) / 448.0).clamp(min=2.0 ** -126)
    q = (whole / scale[:, :, None]).view(n, blocks * BLOCK)[:, :width].to(torch.float8_e4m3fn)
    return q, scale


def _keep(out, name, lo, hi, values, parts=1):
    """Rounds rows into out[name], and their scales into out[name + "_scale"] where it is there."""
    if out.get(name + "_scale") is None:
        out[name][lo:hi] = values.to(out[name].dtype)
        return
    n = values.shape[1] // parts
    for p in range(parts):
        q, scale = _to_blocks(values[:, p * n:(p + 1) * n])
        out[name].view(torch.uint8)[lo:hi, p * n:(p + 1) * n] = q.view(torch.uint8)
        out[name + "_scale"][lo:hi, p * _blocks(n):(p + 1) * _blocks(n)] = scale


def _fresh(s, *names):
    out = {}
    for name in names:
        for key in (name, name + "_scale"):
            if s.get(key) is not None:
                out[key] = torch.zeros_like(s[key])
    return out


def _plain_gated(s):
    case = s["case"]
    n = case["inner"]
    out = _fresh(s, "out", "saved")
    for e, lo, hi in _runs(s):
        x = _values(s["x"][lo:hi], None if s["scale"] is None else s["scale"][lo:hi])
        both = x @ _weight_values(s, e, 2, n).t()
        _keep(out, "out", lo, hi, _act(case["act"], both[:, :n]) * both[:, n:])
        if s["saved"] is not None:
            _keep(out, "saved", lo, hi, both, parts=2)
    return out


def _plain_product(s):
    case = s["case"]
    out = _fresh(s, "out", "saved")
    for e, lo, hi in _runs(s):
        x = _values(s["x"][lo:hi], None if s["scale"] is None else s["scale"][lo:hi])
        y = x @ _weight_values(s, e, 1, case["out_width"]).t()
        if s["bias"] is not None:
            y = y + s["bias"][e].float()
        if s["saved"] is not None:
            _keep(out, "saved", lo, hi, y)
        y = _act(case["act"], y)
        if s["residual"] is not None:
            y = y + s["residual"][lo:hi].float()
        _keep(out, "out", lo, hi, y)
    return out


def _plain_hidden_grad(s):
    case = s["case"]
    n, act = case["inner"], case["act"]
    out = _fresh(s, "dsaved", "hidden")
    for e, lo, hi in _runs(s):
        dh = s["dout"][lo:hi].float() @ s["w"][e].float()
        kept = s["saved"][lo:hi].float()
        if s["saved_scale"] is not None:
            scale, b = s["saved_scale"][lo:hi], _blocks(n)
            kept = kept * torch.cat([_spread(scale[:, at:at + b], n) for at in range(0, scale.shape[1], b)], dim=1)
        gate = kept[:, :n]
        if case["gated"]:
            up = kept[:, n:]
            out["dsaved"][lo:hi] = torch.cat([dh * up * _slope(act, gate), dh * _act(act, gate)], dim=1).to(out["dsaved"].dtype)
            out["hidden"][lo:hi] = (_act(act, gate) * up).to(out["hidden"].dtype)
        else:
            out["dsaved"][lo:hi] = (dh * _slope(act, gate)).to(out["dsaved"].dtype)
            out["hidden"][lo:hi] = _act(act, gate).to(out["hidden"].dtype)
    return out


def _plain_rows_grad(s):
    out = _fresh(s, "drows")
    for e, lo, hi in _runs(s):
        d = s["dout"][lo:hi].float() @ s["w"][e].float()
        if s["add"] is not None:
            d = d + s["add"][lo:hi].float()
        out["drows"][lo:hi] = d.to(out["drows"].dtype)
    return out


def _plain_weight_grad(s):
    dw = torch.zeros_like(s["dw"]) if s["before"] is None else s["before"].clone()
    out = dict(dw=dw)
    if s["dbias"] is not None:
        out["dbias"] = torch.zeros_like(s["dbias"])
    for e, lo, hi in _runs(s):
        d = s["dout"][lo:hi].float()
        dw[e] = (dw[e].float() + d.t() @ s["x"][lo:hi].float()).to(dw.dtype)
        if s["dbias"] is not None:
            out["dbias"][e] = d.sum(dim=0)
    return out


# ---- the framework's entry points ------------------------------------------------------------------------------


def _lib():
    import aws_ofi_nccl_amd as m
    return m.load(), m.check


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _pitched(t):
    """A matrix's address and the bytes from row to row."""
    return (None, 0) if t is None else (t.data_ptr(), t.stride(0) * t.element_size())


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stacked(t):
    """Address of the experts' matrices, bytes from row to row and from expert to expert."""
    return t.data_ptr(), t.stride(1) * t.element_size(), t.stride(0) * t.element_size()


def _groups(s):
    """Where each expert's rows begin, the experts, and the rows there is room for."""
    return _ptr(s["offset"]), max(1, s["case"]["experts"]), s["max_rows"]


def _code(kind):
    return TYPES[kind][1] if kind else 0


def _outputs(s, *names):
    return {key: s[key] for name in names for key in (name, name + "_scale") if s.get(key) is not None}


def _own_gated(s):
    lib, check = _lib()
    case = s["case"]
    check(lib.ofi_amd_expert_gated(*_pitched(s["x"]), *_pitched(s["scale"]), _code(case["type"]), *_groups(s), *_stacked(s["w"]),
                                   _ptr(s["w_scale"]), case["width"], case["inner"], ACTIVATIONS[case["act"]], *_pitched(s["out"]),
                                   _code(case["out"]), *_pitched(s["out_scale"]), *_pitched(s["saved"]), _code(case["saved"]),
                                   *_pitched(s["saved_scale"]), _stream()), "expert_gated")
    return _outputs(s, "out", "saved")


def _own_product(s):
    lib, check = _lib()
    case = s["case"]
    check(lib.ofi_amd_expert_product(*_pitched(s["x"]), *_pitched(s["scale"]), _code(case["type"]), *_groups(s), *_stacked(s["w"]),
                                     _ptr(s["w_scale"]), case["width"], case["out_width"], _ptr(s["bias"]), _code(case["out"]),
                                     ACTIVATIONS[case["act"]], *_pitched(s["residual"]), *_pitched(s["out"]), _code(case["out"]),
                                     *_pitched(s["out_scale"]), *_pitched(s["saved"]), _code(case["saved"]),
                                     *_pitched(s["saved_scale"]), _stream()), "expert_product")
    return _outputs(s, "out", "saved")


def _own_hidden_grad(s):
    lib, check = _lib()
    case = s["case"]
    check(lib.ofi_amd_expert_hidden_grad(*_pitched(s["dout"]), _code(case["type"]), *_groups(s), *_stacked(s["w"]), case["width"],
                                         case["inner"], int(case["gated"]), ACTIVATIONS[case["act"]], *_pitched(s["saved"]),
                                         _code(case["saved"]), *_pitched(s["saved_scale"]), *_pitched(s["dsaved"]),
                                         *_pitched(s["hidden"]), _stream()), "expert_hidden_grad")
    return _outputs(s, "dsaved", "hidden")


def _own_rows_grad(s):
    lib, check = _lib()
    case = s["case"]
    check(lib.ofi_amd_expert_rows_grad(*_pitched(s["dout"]), _code(case["type"]), *_groups(s), *_stacked(s["w"]), case["width"],
                                       case["out_width"], *_pitched(s["add"]), *_pitched(s["drows"]), _stream()), "expert_rows_grad")
    return _outputs(s, "drows")


def _own_weight_grad(s):
    lib, check = _lib()
    case = s["case"]
    check(lib.ofi_amd_expert_weight_grad(*_pitched(s["dout"]), *_pitched(s["x"]), _code(case["type"]), *_groups(s), case["width"],
                                         case["out_width"], _ptr(s["before"]), *_stacked(s["dw"]), _code(case["out"]), None,
                                         _ptr(s["dbias"]), _stream()), "expert_weight_grad")
    return _outputs(s, "dw", "dbias")


PLAIN = dict(gated=_plain_gated, product=_plain_product, hidden_grad=_plain_hidden_grad, rows_grad=_plain_rows_grad,
             weight_grad=_plain_weight_grad)
OWN = dict(gated=_own_gated, product=_own_product, hidden_grad=_own_hidden_grad, rows_grad=_own_rows_grad,
           weight_grad=_own_weight_grad)


def run(state):
    return (OWN if own else PLAIN)[state["case"]["path"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------


def work(case):
    path, R, width = case["path"], case["rows"], case["width"]
    E = max(1, case["experts"])
    used = E if case["experts"] == 0 else min(E, R) if R <= E // 2 else E * (1.0 - (1.0 - 1.0 / E) ** R)  # experts with rows, about
    n = case["inner"] if path in ("gated", "hidden_grad") else case["out_width"]

    def rows(w, kind, blocks=None):
        return R * (w * SIZE[kind] + (4 * (blocks or _blocks(w)) if kind == "e4m3" else 0))

    kind = case["type"]
    table = 4 * (E + 1) if case["experts"] else 0
    if path in ("gated", "product"):
        parts = 2 if path == "gated" else 1
        weights = used * parts * (n * width * SIZE[kind] + (4 * _blocks(n) * _blocks(width) if kind == "e4m3" else 0))
        moved = rows(width, kind) + weights + rows(n, case["out"]) + table
        if case["saved"]:
            moved += rows(parts * n, case["saved"], parts * _blocks(n))
        if path == "product":
            moved += (used * n * SIZE[case["out"]] if case["bias"] else 0) + (rows(n, case["out"]) if case["residual"] else 0)
        return dict(bytes=moved, flops=2 * parts * R * width * n)
    if path == "hidden_grad":
        parts = 2 if case["gated"] else 1
        moved = rows(width, kind) + used * n * width * SIZE[kind] + rows(parts * n, case["saved"], parts * _blocks(n))
        return dict(bytes=moved + rows((parts + 1) * n, kind) + table, flops=2 * R * width * n)
    if path == "rows_grad":
        moved = rows(n, kind) + used * n * width * SIZE[kind] + rows(width, kind) * (2 if case["add"] else 1)
        return dict(bytes=moved + table, flops=2 * R * width * n)
    times = 2 if case["accumulate"] else 1
    moved = rows(n, kind) + rows(width, kind) + times * E * n * width * SIZE[case["out"]] + (4 * E * n if case["bias"] else 0)
    return dict(bytes=moved + table, flops=2 * R * width * n)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------


def _wide(q, scale, first=0):
    """8-bit values times their scales, in 64 bits; scale column `first` belongs to the first block."""
    v = q.double()
    if scale is not None:
        for lo in range(0, v.shape[1], BLOCK):
            v[:, lo:lo + BLOCK] *= scale[:, first + lo // BLOCK, None].double()
    return v


def _sigma(kind, v):
    """The activation and its derivative in 64 bits."""
    if kind == "none":
        return v, torch.ones_like(v)
    if kind == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v)), torch.where(v > 0, 1.0, 0.0).double()
    if kind == "silu":
        sig = torch.sigmoid(v)
        return v * sig, sig + v * sig * (1.0 - sig)
    cdf = 0.5 * torch.special.erfc(-v / 2.0 ** 0.5)
    return v * cdf, cdf + v * torch.exp(-v * v / 2.0) / (2.0 * math.pi) ** 0.5


def _eight(v, parts=1):
    """Rows divided by the scale of their block, not rounded, and the scales."""
    n = v.shape[1] // parts
    q, scales = torch.empty_like(v), []
    for p in range(parts):
        for lo in range(p * n, (p + 1) * n, BLOCK):
            hi = min(lo + BLOCK, (p + 1) * n)
            m = torch.clamp(v[:, lo:hi].abs().max(dim=1).values / 448.0, min=2.0 ** -126)
            q[:, lo:hi] = v[:, lo:hi] / m[:, None]
            scales.append(m)
    return q, torch.stack(scales, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    path, R, E = case["path"], s["max_rows"], max(1, case["experts"])
    first = [0, R] if s["offset"] is None else s["offset"].cpu().tolist()
    n = case["inner"] if path in ("gated", "hidden_grad") else case["out_width"]
    out = {}

    def put(name, lo, hi, value):
        if name not in out:
            out[name] = torch.zeros(R, value.shape[1], device="cuda", dtype=torch.float64)
        out[name][lo:hi] = value

    def put_kept(name, kind, lo, hi, value, parts=1):
        if kind == "e4m3":
            q, scale = _eight(value, parts)
            put(name, lo, hi, q)
            put(name + "_scale", lo, hi, scale)
        else:
            put(name, lo, hi, value)

    if path == "weight_grad":
        dw = torch.zeros(E, n, case["width"], device="cuda", dtype=torch.float64) if s["before"] is None else s["before"].double()
        out["dw"] = dw
        if case["bias"]:
            out["dbias"] = torch.zeros(E, n, device="cuda", dtype=torch.float64)
    for e in range(E):
        lo, hi = first[e], first[e + 1]
        if hi <= lo:
            continue
        if path in ("gated", "product"):
            x = _wide(s["x"][lo:hi], None if s["scale"] is None else s["scale"][lo:hi])
            made = []
            for p in range(2 if path == "gated" else 1):
                w = s["w"][e, p * n:(p + 1) * n].double()
                if s["w_scale"] is not None:
                    for at in range(0, n, BLOCK):
                        w[at:at + BLOCK] = _wide(w[at:at + BLOCK], s["w_scale"][e, p, at // BLOCK].expand(min(BLOCK, n - at), -1))
                made.append(torch.mm(x, w.t().contiguous()))
            if path == "gated":
                y = _sigma(case["act"], made[0])[0] * made[1]
                kept = torch.cat(made, dim=1)
            else:
                kept = made[0] if s["bias"] is None else made[0] + s["bias"][e].double()
                y = _sigma(case["act"], kept)[0]
                if s["residual"] is not None:
                    y = y + s["residual"][lo:hi].double()
            put_kept("out", case["out"], lo, hi, y)
            if case["saved"]:
                put_kept("saved", case["saved"], lo, hi, kept, len(made))
        elif path == "hidden_grad":
            dh = torch.mm(s["dout"][lo:hi].double(), s["w"][e].double())
            scale = None if s["saved_scale"] is None else s["saved_scale"][lo:hi]
            gate = _wide(s["saved"][lo:hi, :n], scale)
            value, slope = _sigma(case["act"], gate)
            if case["gated"]:
                up = _wide(s["saved"][lo:hi, n:], scale, _blocks(n))
                put("dsaved", lo, hi, torch.cat([dh * up * slope, dh * value], dim=1))
                put("hidden", lo, hi, value * up)
            else:
                put("dsaved", lo, hi, dh * slope)
                put("hidden", lo, hi, value)
        elif path == "rows_grad":
            d = torch.mm(s["dout"][lo:hi].double(), s["w"][e].double())
            put("drows", lo, hi, d if s["add"] is None else d + s["add"][lo:hi].double())
        else:
            d = s["dout"][lo:hi].double()
            dw[e] += torch.mm(d.t().contiguous(), s["x"][lo:hi].double())
            if case["bias"]:
                out["dbias"][e] = d.sum(dim=0)
    return out
