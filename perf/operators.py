"""The 8-bit layer operators whose speed this repository answers for.

A linear layer that answers in 8 bits takes three operators: the RMS norm that
adds the residual and rounds its rows to 8-bit integers, the product of 8-bit
integers with a scale for each token and each channel, and the activation that
rounds its rows to 8 bits for the next product.  `listed()` names twelve calls,
`draw(rng)` gives more of the same kinds and ranges.

A case's "kind" says which operator it takes:
  product   einsum_ir_amd.ContractionI8Plan
  norm      einsum_ir_amd.NormQuantPlan
  act       einsum_ir_amd.ActQuantPlan
Sizes of products are written "t=24,k=4096,o=10240": tokens t (of a batch b),
channels o, contracted k, and z for products that share nothing (one weight
each).  8-bit rows are returned as the values that they stand for, in the type
of the operator's input.
"""
import math

import torch

own = False

EPS = 1e-6


def listed():
    return [
        # one token through a square layer of the width of the 4-layer MLP:
        # latency and the weights' bytes
        dict(name="product_1_token", kind="product", expr="tk,ok->to", sizes="k=2048,o=2048,t=1", out="bf16",
             bias=False, relu=False),
        # a batch of sequences, one token each, into a wide layer: the
        # weights' bytes
        dict(name="product_24_tokens", kind="product", expr="tk,ok->to", sizes="k=4096,o=10240,t=24", out="bf16",
             bias=True, relu=True),
        # the first layer of the bias/ReLU MLP on its batch of 1152: few
        # output tiles
        dict(name="product_mlp", kind="product", expr="tk,ok->to", sizes="k=784,o=512,t=1152", out="fp32",
             bias=True, relu=True),
        # an ordinary linear layer over a ragged number of tokens
        dict(name="product_ragged", kind="product", expr="btk,ok->bto", sizes="b=8,k=2048,o=2048,t=509", out="bf16",
             bias=False, relu=False),
        # products that share nothing, every size odd, rows at any byte
        dict(name="product_odd", kind="product", expr="ztk,zok->zto", sizes="k=1001,o=333,t=77,z=5", out="fp32",
             bias=True, relu=False),
        # a long prompt through a wide layer: the matrix rate
        dict(name="product_large", kind="product", expr="tk,ok->to", sizes="k=8192,o=8192,t=8192", out="bf16",
             bias=False, relu=False),
        # the norm in front of a layer, one token: latency
        dict(name="norm_1_token", kind="norm", rows=1, cols=2048, dtype="bf16", residual=True),
        # the same over the ragged batch of tokens above
        dict(name="norm_ragged", kind="norm", rows=4072, cols=2048, dtype="bf16", residual=True),
        # a first norm in single precision, with no residual yet, odd rows
        dict(name="norm_odd", kind="norm", rows=509, cols=5001, dtype="fp32", residual=False),
        # a long prompt of a wide model: bytes
        dict(name="norm_large", kind="norm", rows=16384, cols=8192, dtype="bf16", residual=True),
        # gated activation between two products, a few tokens: latency
        dict(name="act_6_tokens", kind="act", rows=6, cols=8192, dtype="bf16", act="silu", gated=True),
        # the same for a long prompt: bytes
        dict(name="act_large", kind="act", rows=8192, cols=8192, dtype="bf16", act="silu", gated=True),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm, odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A layer's width: mostly a multiple of 16, as layers have, now and then any."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.25 else max(16, n // 16 * 16)


def draw(rng):
    what = rng.choice(["tokens", "product", "product", "shared", "norm", "norm", "act"])
    if what in ("norm", "act"):
        while True:
            rows, cols = _log(rng, 1, 16384), _width(rng, 64, 16384)
            if rows * cols <= (16384 if what == "norm" else 8192) * 8192:
                break
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        if dtype == "fp32":
            rows = max(1, rows // 2)
        if what == "norm":
            return dict(kind="norm", rows=rows, cols=cols, dtype=dtype, residual=rng.random() < 0.7)
        # in fp32 two exponentials that are both right in all but the last bit
        # may round to different 8-bit integers, so SiLU comes with bf16
        return dict(kind="act", rows=rows, cols=cols, dtype=dtype,
                    act=rng.choice(["silu", "relu", "none"] if dtype == "bf16" else ["relu", "none"]),
                    gated=rng.random() < 0.6)
    case = dict(kind="product", out=rng.choice(["bf16", "bf16", "fp32"]), bias=rng.random() < 0.5,
                relu=rng.random() < 0.3)
    while True:
        s = dict(k=_width(rng, 64, 12288), o=_width(rng, 10, 16384))
        if what == "tokens":
            case["expr"], s["t"] = "tk,ok->to", _log(rng, 1, 64)
        elif what == "shared":
            case["expr"], s["z"], s["t"] = "ztk,zok->zto", _log(rng, 2, 16), _log(rng, 1, 1024)
        else:
            case["expr"], s["t"] = rng.choice(["tk,ok->to", "btk,ok->bto"]), _log(rng, 65, 8192)
            if "b" in case["expr"]:
                s["b"], s["t"] = 4, max(1, s["t"] // 4)
        if math.prod(s.values()) <= 8192 ** 3 and s.get("z", 1) * s["k"] * s["o"] <= 1 << 28:
            return dict(case, sizes=",".join("%s=%d" % (d, s[d]) for d in sorted(s)))


_TORCH = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _sizes(case):
    return {k: int(v) for k, v in (p.split("=") for p in case["sizes"].split(","))}


def _shape(dims, sizes):
    return [sizes[d] for d in dims]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows_i8(shape, g):
    """8-bit rows of normal values and their scales, as the two quantising operators leave them."""
    x = torch.randn(shape, device="cuda", generator=g)
    a = x.abs().amax(-1, keepdim=True)
    return torch.round(x * (127 / a)).to(torch.int8), (a / 127).squeeze(-1)


def _product_inputs(case, seed):
    g, s = _generator(seed), _sizes(case)
    ins = case["expr"].split("->")[0].split(",")
    left, scale_left = _rows_i8(_shape(ins[0], s), g)
    right, scale_right = _rows_i8(_shape(ins[1], s), g)
    scale_right = scale_right / s["k"] ** 0.5
    bias = torch.randn(scale_right.shape, device="cuda", generator=g) if case["bias"] else None
    return left, scale_left, right, scale_right, bias


def _norm_inputs(case, seed):
    """Hidden states with a few wide channels, as deep layers have them, and a weight around one."""
    g, rows, cols, dtype = _generator(seed), case["rows"], case["cols"], _TORCH[case["dtype"]]
    wide = 1 + 7 * (torch.rand(cols, device="cuda", generator=g) < 0.01)
    x = (torch.randn((rows, cols), device="cuda", generator=g) * wide).to(dtype)
    r = None
    if case["residual"]:
        r = (3 * torch.randn((rows, cols), device="cuda", generator=g) * wide).to(dtype)
    w = (1 + 0.2 * torch.randn(cols, device="cuda", generator=g)).to(dtype)
    return x, r, w


def _act_inputs(case, seed):
    """The product in front of the activation; a gated one holds the gates in the first half of its columns."""
    g = _generator(seed)
    h = torch.randn((case["rows"], case["cols"] * (2 if case["gated"] else 1)), device="cuda", generator=g)
    return h.to(_TORCH[case["dtype"]])


def _own_product(case, state):
    import einsum_ir_amd as eir
    s = _sizes(case)
    ins, out = case["expr"].split("->")
    lp = eir.contraction_i8_loops(case["expr"], s, scale_left=ins.split(",")[0].replace("k", ""),
                                  scale_right=ins.split(",")[1].replace("k", ""),
                                  bias=ins.split(",")[1].replace("k", "") if case["bias"] else None)
    state["plan"] = eir.ContractionI8Plan(**lp, dtype_out=eir.BF16 if case["out"] == "bf16" else eir.FP32,
                                          ktype_last_touch=eir.RELU if case["relu"] else eir.UNDEFINED_KTYPE)
    state["result"] = torch.empty(_shape(out, s), device="cuda", dtype=_TORCH[case["out"]])


def _own_rows(case, state):
    import einsum_ir_amd as eir
    rows, cols, dtype = case["rows"], case["cols"], _TORCH[case["dtype"]]
    kind = eir.BF16 if case["dtype"] == "bf16" else eir.FP32
    state["q"] = torch.empty((rows, cols), device="cuda", dtype=torch.int8)
    state["scale"] = torch.empty(rows, device="cuda")
    state["values"] = torch.empty((rows, cols), device="cuda", dtype=dtype)
    if case["kind"] == "norm":
        state["plan"] = eir.NormQuantPlan(rows, cols, dtype=kind, eps=EPS)
        state["total"] = torch.empty((rows, cols), device="cuda", dtype=dtype) if case["residual"] else None
    else:
        h, ktype = state["h"], {"none": eir.UNDEFINED_KTYPE, "relu": eir.RELU, "silu": eir.SILU}[case["act"]]
        state["plan"] = eir.ActQuantPlan(rows, cols, dtype=kind, ktype=ktype, ld_in=h.shape[1], ld_gate=h.shape[1])
        state["x"], state["gate"] = (h[:, cols:], h[:, :cols]) if case["gated"] else (h, None)


def prepare(case, seed):
    state = dict(case=case, stream=torch.cuda.current_stream())
    if case["kind"] == "product":
        state["in"] = _product_inputs(case, seed)
    elif case["kind"] == "norm":
        state["in"] = _norm_inputs(case, seed)
    else:
        state["h"] = _act_inputs(case, seed)
    if own:  # the plan and the buffers that a program of the framework keeps
        (_own_product if case["kind"] == "product" else _own_rows)(case, state)
    return state


def _run_own(state):
    kind, plan, stream = state["case"]["kind"], state["plan"], state["stream"]
    if kind == "product":
        left, scale_left, right, scale_right, bias = state["in"]
        plan.execute(left, right, state["result"], scale_left=scale_left, scale_right=scale_right, bias=bias,
                     stream=stream)
        return state["result"]
    if kind == "norm":
        x, r, w = state["in"]
        plan.execute(x, state["q"], state["scale"], residual=r, weight=w, total=state["total"],
                     values=state["values"], stream=stream)
        return dict(values=state["values"], scale=state["scale"], total=state["total"])
    plan.execute(state["x"], state["q"], state["scale"], gate=state["gate"], values=state["values"], stream=stream)
    return dict(values=state["values"], scale=state["scale"])


def _round_rows(t):
    """8-bit integers of the rows of t (as fp32 numbers), and the rows' largest magnitudes."""
    a = t.abs().amax(-1, keepdim=True)
    inv = torch.where(a > 0, torch.div(torch.full_like(a, 127.0), a), torch.zeros_like(a))
    return torch.round(t * inv), a


def _plain_product(case, left, scale_left, right, scale_right, bias):
    left, right = left.float(), right.float().transpose(-1, -2).contiguous()
    y = left @ right * scale_left.unsqueeze(-1) * scale_right.unsqueeze(-2 if scale_right.dim() > 1 else 0)
    if bias is not None:
        y = y + bias.unsqueeze(-2)
    if case["relu"]:
        y = y.clamp_min(0)
    return y.to(_TORCH[case["out"]])


def _plain_norm(case, x, r, w):
    s = x.float() if r is None else x.float() + r.float()
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + EPS)
    q, a = _round_rows(s * w.float())
    scale = a * rstd / 127
    return dict(values=(q * scale).to(x.dtype), scale=scale.squeeze(-1), total=s.to(x.dtype) if r is not None else None)


def _plain_act(case, h):
    n = case["cols"]
    f = h[:, :n].float()
    if case["act"] == "relu":
        f = f.clamp_min(0)
    elif case["act"] == "silu":
        f = f / (1 + torch.exp(-f))
    q, a = _round_rows(f * h[:, n:].float() if case["gated"] else f)
    scale = a / 127
    return dict(values=(q * scale).to(h.dtype), scale=scale.squeeze(-1))


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["kind"] == "product":
        return _plain_product(case, *state["in"])
    if case["kind"] == "norm":
        return _plain_norm(case, *state["in"])
    return _plain_act(case, state["h"])


def work(case):
    if case["kind"] == "product":
        s = _sizes(case)
        (left, right), out = case["expr"].split("->")[0].split(","), case["expr"].split("->")[1]
        numel = lambda t: math.prod(s[d] for d in t)  # noqa: E731
        per_row = numel(left.replace("k", "")) + numel(right.replace("k", "")) * (2 if case["bias"] else 1)
        return dict(bytes=numel(left) + numel(right) + 4 * per_row + _TORCH[case["out"]].itemsize * numel(out),
                    flops=2 * math.prod(s.values()))
    item, rows, cols = _TORCH[case["dtype"]].itemsize, case["rows"], case["cols"]
    # read: the input, the residual or the gate, the weight; written: the sum
    # with the residual, the 8-bit rows, the values that they stand for
    if case["kind"] == "norm":
        return dict(bytes=rows * cols * (item * (4 if case["residual"] else 2) + 1) + item * cols + 4 * rows,
                    flops=7 * rows * cols)
    return dict(bytes=rows * cols * (item * (3 if case["gated"] else 2) + 1) + 4 * rows, flops=6 * rows * cols)


def _exact_rows(y, factor):
    """values and scales of 64-bit rows y, the scales times factor."""
    top = y.abs().max(dim=-1).values
    step = torch.where(top > 0, top, torch.ones_like(top))[:, None] / 127
    scale = top / 127 * factor
    return dict(values=(y / step).round() * scale[:, None], scale=scale)


def exact(case, seed):
    if case["kind"] == "product":
        left, scale_left, right, scale_right, bias = _product_inputs(case, seed)
        # the scales multiplied into the 64-bit operands
        left = left.double() * scale_left.double()[..., None]
        right = right.double() * scale_right.double()[..., None]
        if left.dim() == right.dim():
            y = torch.matmul(left, right.mT.contiguous())
        else:
            y = torch.matmul(left.flatten(0, -2), right.T.contiguous()).unflatten(0, left.shape[:-1])
        if bias is not None:
            y += bias.double()[..., None, :]
        return torch.relu(y) if case["relu"] else y
    if case["kind"] == "norm":
        x, r, w = _norm_inputs(case, seed)
        s = x.double()
        if r is not None:
            s = s + r.double()
        length = torch.linalg.vector_norm(s, dim=-1)
        found = _exact_rows(s * w.double(), (length.square() / case["cols"] + EPS).rsqrt())
        return dict(found, total=s if r is not None else None)
    h = _act_inputs(case, seed).double()
    x, gate = (h[:, case["cols"]:], h[:, :case["cols"]]) if case["gated"] else (1.0, h)
    f = {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v)}[case["act"]](gate)
    return _exact_rows(f * x, 1.0)
