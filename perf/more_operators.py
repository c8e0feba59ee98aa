"""The operators of 8-bit floating point and of experts whose speed this
repository answers for.

An expert layer in 8 bits takes three operators: the rounding of rows (or of an
activation of them, or of weights) to 8-bit floating point with a scale for each
block of 128, the product of such blocks, and the product whose rows are grouped
by expert, each group with weights of its own.  Their gradients are products of
the same kinds in other layouts.  `listed()` names twelve calls, `draw(rng)` gives
more of the same kinds and ranges.

A case's "kind" says which operator it takes:
  quant     einsum_ir_amd.QuantF8Plan
  product   einsum_ir_amd.ContractionF8Plan
  grouped   einsum_ir_amd.ContractionGroupedPlan
Products are written as einsum strings over tokens t (of a batch b), channels o,
width k and experts e, with sizes as "t=24,k=4096,o=10240".  "scale" says whether
the scales are fp32, any value, or e8m0, powers of two in one byte.  The rows of
a grouped product are sorted by expert, group g from offsets[g] to
offsets[g + 1]; groups are of very unequal sizes, some empty, and with "spare" the
last rows belong to none.  Quantised blocks are returned as the values that they
stand for, in the type of the operator's input.
"""
import math
import random

import torch

own = False

BLOCK = 128


def listed():
    return [
        # gated activation between two products of a long prompt: bytes
        dict(name="quant_gated", kind="quant", batch=1, rows=8192, cols=8192, dtype="bf16", block="1x128", act="relu",
             gated=True, q="e4m3"),
        # the weights of four experts laid out once
        dict(name="quant_weights", kind="quant", batch=4, rows=2048, cols=2048, dtype="fp32", block="128x128",
             act="none", gated=False, q="e4m3"),
        # one token through a square layer with a checkpoint's scales: latency
        # and the weights' bytes
        dict(name="f8_1_token", kind="product", expr="tk,ok->to", sizes="k=2048,o=2048,t=1", left="e4m3", scale="fp32",
             out="bf16", bias=False),
        # an ordinary linear layer over a ragged number of tokens
        dict(name="f8_ragged", kind="product", expr="btk,ok->bto", sizes="b=8,k=2048,o=2048,t=509", left="e4m3",
             scale="fp32", out="bf16", bias=True),
        # a long prompt through a wide layer: the matrix rate
        dict(name="f8_large", kind="product", expr="tk,ok->to", sizes="k=8192,o=8192,t=8192", left="e4m3",
             scale="e8m0", out="bf16", bias=False),
        # the gradient of a layer's input, read against the weights as they lie
        dict(name="f8_grad_input", kind="product", expr="to,ok->tk", sizes="k=2048,o=4096,t=4072", left="e5m2",
             scale="fp32", out="bf16", bias=False),
        # the gradient of its weights, blocks of 128 tokens
        dict(name="f8_grad_weight", kind="product", expr="to,tk->ok", sizes="k=2048,o=4096,t=8192", left="e5m2",
             scale="fp32", out="fp32", bias=False),
        # a few tokens, each to a few of 16 experts: the weights' bytes
        dict(name="grouped_decode", kind="grouped", expr="tk,eok->to", sizes="e=16,k=2048,o=2048,t=24", left="bf16",
             scale="none", out="bf16", spare=False),
        # a prompt through 16 experts in 8 bits
        dict(name="grouped_prompt_f8", kind="grouped", expr="tk,eok->to", sizes="e=16,k=4096,o=2048,t=8192",
             left="e4m3", scale="fp32", out="bf16", spare=False),
        # a training batch through 8 wide experts: the matrix rate
        dict(name="grouped_large", kind="grouped", expr="tk,eok->to", sizes="e=8,k=4096,o=4096,t=16384", left="bf16",
             scale="none", out="bf16", spare=False),
        # the gradient of the experts' weights, one sum over each group's rows
        dict(name="grouped_grad_weight", kind="grouped", expr="to,tk->eok", sizes="e=16,k=2048,o=2048,t=8192",
             left="bf16", scale="none", out="fp32", spare=True),
        # every size odd, rows at any byte
        dict(name="grouped_odd", kind="grouped", expr="tk,eok->to", sizes="e=5,k=1001,o=333,t=509", left="bf16",
             scale="none", out="fp32", spare=True),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm, odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A layer's width: mostly a multiple of 16, as layers have, now and then any."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.2 else max(16, n // 16 * 16)


def _text(s):
    return ",".join("%s=%d" % (d, s[d]) for d in sorted(s))


def draw(rng):
    what = rng.choice(["quant", "quant", "tokens", "product", "grad", "grouped_tokens", "grouped", "grouped_grad"])
    if what == "quant":
        while True:
            batch, rows, cols = rng.choice([1, 1, _log(rng, 2, 16)]), _log(rng, 1, 16384), _width(rng, 64, 16384)
            if batch * rows * cols <= 8192 * 8192:
                break
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        # the product with a gate is exact in fp32 where both are bf16, so both
        # forms round the same number to 8 bits
        return dict(kind="quant", batch=batch, rows=rows, cols=cols, dtype=dtype,
                    block=rng.choice(["1x128", "1x128", "128x128", "128x1"]), act=rng.choice(["none", "none", "relu"]),
                    gated=dtype == "bf16" and rng.random() < 0.4, q=rng.choice(["e4m3", "e4m3", "e5m2"]))
    while True:
        s = dict(k=_width(rng, 64, 12288), o=_width(rng, 64, 12288))
        if what in ("tokens", "product", "grad"):
            case = dict(kind="product", left=rng.choice(["e4m3", "e4m3", "e5m2"]), scale=rng.choice(["fp32", "e8m0"]),
                        out=rng.choice(["bf16", "bf16", "fp32"]), bias=what != "grad" and rng.random() < 0.3)
            s["t"] = _log(rng, 1, 64) if what == "tokens" else _log(rng, 65, 16384)
            case["expr"] = rng.choice(["to,ok->tk", "to,tk->ok"] if what == "grad" else ["tk,ok->to", "btk,ok->bto"])
            if "b" in case["expr"]:
                s["b"], s["t"] = 4, max(1, s["t"] // 4)
            weights = s["k"] * s["o"]
        else:
            s["e"] = _log(rng, 2, 64)
            few = what == "grouped_tokens"
            s["t"] = _log(rng, 1, 128) if few else _log(rng, 129, 32768)
            f8 = what != "grouped_grad" and rng.random() < 0.5
            case = dict(kind="grouped", left="e4m3" if f8 else "bf16",
                        scale=rng.choice(["fp32", "e8m0"]) if f8 else "none", out=rng.choice(["bf16", "bf16", "fp32"]),
                        spare=rng.random() < 0.5)
            case["expr"] = rng.choice(["to,eok->tk", "to,tk->eok"]) if what == "grouped_grad" else "tk,eok->to"
            weights = s["e"] * s["k"] * s["o"]
        ops = math.prod(v for d, v in s.items() if d != "e")
        if weights <= 1 << 28 and ops <= (8192 ** 3 if case["left"] != "bf16" else 8192 ** 3 // 2):
            return dict(case, sizes=_text(s))


_TORCH = {"fp32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}


def _sizes(case):
    return {k: int(v) for k, v in (p.split("=") for p in case["sizes"].split(","))}


def _split(case):
    ins, out = case["expr"].split("->")
    left, right = ins.split(",")
    return left, right, out


def _block_of(case, dims):
    """Rows and columns that share a scale, for an operand's last two dimensions: 128 along the contracted one, and
    128 of the weights' other one."""
    left, right, out = _split(case)
    contracted = [d for d in left if d in right and d not in out][0]
    other = BLOCK if "o" in dims and "k" in dims else 1
    return (other, BLOCK) if dims[-1] == contracted else (BLOCK, other)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _power(e):
    """2^e as fp32, by way of 64 bits, whose exponential is exact there (32 bits' and ldexp are not)."""
    return torch.exp2(e.double()).float()


def _spread(s, block, shape):
    """A scale for each element."""
    s = s.repeat_interleave(block[0], -2)[..., :shape[-2], :]
    return s.repeat_interleave(block[1], -1)[..., :shape[-1]]


def _blocks_f8(shape, block, q, scale, g):
    """8-bit blocks of normal values and their scales: any fp32 number, or the byte of a power of two."""
    x = torch.randn(shape, device="cuda", generator=g)
    pad = torch.nn.functional.pad(x, (0, -shape[-1] % block[1], 0, -shape[-2] % block[0]))
    a = pad.unflatten(-1, (-1, block[1])).unflatten(-3, (-1, block[0])).abs().amax((-3, -1))
    s = a / _LARGEST[q]
    if scale == "e8m0":
        m, e = torch.frexp(s)
        e = e - (m == 0.5).to(e.dtype)
        s, bytes_ = _power(e), (e + 127).to(torch.uint8)
    values = (x / _spread(s, block, shape)).clamp(-_LARGEST[q], _LARGEST[q]).to(_TORCH[q])
    return values, bytes_ if scale == "e8m0" else s


def _group_sizes(case, seed):
    """Rows of each expert: very unequal, some without any."""
    s, rng = _sizes(case), random.Random(int(seed))
    share = [rng.expovariate(1.0) if rng.random() < 0.9 else 0.0 for _ in range(s["e"])]
    share[rng.randrange(s["e"])] += 0.5
    rows = s["t"] - (s["t"] // 8 if case["spare"] else 0)
    ends, run_ = [], 0.0
    for v in share:
        run_ += v
        ends.append(int(round(rows * run_ / sum(share))))
    return [b - a for a, b in zip([0] + ends, ends)]


def _inputs(case, seed):
    """Operands, their scales (None in bf16) and the bias of a product, plain or grouped."""
    g, s = _generator(seed), _sizes(case)
    left, right, out = _split(case)
    shape_l, shape_r = [s[d] for d in left], [s[d] for d in right]
    contracted = [d for d in left if d in right and d not in out][0]
    wide = s[contracted] ** -0.5
    if case["left"] == "bf16":
        a = torch.randn(shape_l, device="cuda", generator=g).to(torch.bfloat16)
        b = (torch.randn(shape_r, device="cuda", generator=g) * wide).to(torch.bfloat16)
        sa = sb = None
    else:
        a, sa = _blocks_f8(shape_l, _block_of(case, left), case["left"], case["scale"], g)
        b, sb = _blocks_f8(shape_r, _block_of(case, right), "e4m3", case["scale"], g)
        if case["scale"] == "fp32":
            sb = sb * wide
    bias = torch.randn(s["o"], device="cuda", generator=g) if case.get("bias") else None
    return a, sa, b, sb, bias


def _quant_inputs(case, seed):
    """Hidden states with a few wide channels, as deep layers have them; a gated one holds the gates in the first
    half of its columns."""
    g, cols = _generator(seed), case["cols"] * (2 if case["gated"] else 1)
    wide = 1 + 7 * (torch.rand(cols, device="cuda", generator=g) < 0.01)
    x = torch.randn((case["batch"], case["rows"], cols), device="cuda", generator=g) * wide
    return x.to(_TORCH[case["dtype"]])


def _quant_block(case):
    return tuple(int(v) for v in case["block"].split("x"))


def _own_quant(case, state):
    import einsum_ir_amd as eir
    batch, rows, cols, dtype = case["batch"], case["rows"], case["cols"], _TORCH[case["dtype"]]
    h, block = state["in"], _quant_block(case)
    state["plan"] = eir.QuantF8Plan(
        rows, cols, batch=batch, dtype=eir.BF16 if case["dtype"] == "bf16" else eir.FP32,
        dtype_q=eir.F8E4M3 if case["q"] == "e4m3" else eir.F8E5M2, block=block,
        ktype=eir.RELU if case["act"] == "relu" else eir.UNDEFINED_KTYPE, ld_in=h.shape[-1], ld_gate=h.shape[-1])
    state["q"] = torch.empty((batch, rows, cols), device="cuda", dtype=_TORCH[case["q"]])
    state["scale"] = torch.empty((batch, -(-rows // block[0]), -(-cols // block[1])), device="cuda")
    state["values"] = torch.empty((batch, rows, cols), device="cuda", dtype=dtype)
    state["x"], state["gate"] = (h[..., cols:], h) if case["gated"] else (h, None)


def _own_product(case, state):
    import einsum_ir_amd as eir
    left, right, out = _split(case)
    types = {"bf16": eir.BF16, "e4m3": eir.F8E4M3, "e5m2": eir.F8E5M2, "fp32": eir.FP32}
    kinds = dict(dtype_left=types[case["left"]], dtype_out=types[case["out"]])
    s = _sizes(case)
    if case["left"] != "bf16":
        kinds.update(dtype_right=eir.F8E4M3, dtype_scale=eir.E8M0 if case["scale"] == "e8m0" else eir.FP32)
        free = lambda dims: min(_block_of(case, dims))  # noqa: E731
        blocks = dict(block_left=free(left), block_right=free(right))
    if case["kind"] == "product":
        lp = eir.contraction_f8_loops(case["expr"], s, bias="o" if case["bias"] else None, **blocks)
        state["plan"] = eir.ContractionF8Plan(**lp, **kinds)
    else:
        if case["left"] == "bf16":
            lp = eir.grouped_loops(case["expr"], s, group="e", ragged="t")
        else:
            lp = eir.grouped_loops(case["expr"], s, group="e", ragged="t", scales=True, **blocks)
        state["plan"] = eir.ContractionGroupedPlan(**lp, **kinds)
    # zeros, for the rows that belong to no group
    state["result"] = torch.zeros([s[d] for d in out], device="cuda", dtype=_TORCH[case["out"]])


def prepare(case, seed):
    state = dict(case=case, stream=torch.cuda.current_stream())
    if case["kind"] == "quant":
        state["in"] = _quant_inputs(case, seed)
    else:
        state["in"] = _inputs(case, seed)
    if case["kind"] == "grouped":
        n = state["groups"] = _group_sizes(case, seed)
        state["offsets"] = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device="cuda")
    if own:  # the plan and the buffers that a program of the framework keeps
        (_own_quant if case["kind"] == "quant" else _own_product)(case, state)
    return state


def _run_own(state):
    case, plan, stream = state["case"], state["plan"], state["stream"]
    if case["kind"] == "quant":
        plan.execute(state["x"], state["q"], state["scale"], gate=state["gate"], values=state["values"], stream=stream)
        return dict(values=state["values"], scale=state["scale"])
    a, sa, b, sb, bias = state["in"]
    if case["kind"] == "product":
        plan.execute(a, b, state["result"], scale_left=sa, scale_right=sb, bias=bias, stream=stream)
    else:
        plan.execute(a, b, state["result"], state["offsets"], scale_left=sa, scale_right=sb, stream=stream)
    return state["result"]


def _plain_quant(case, h):
    cols, block = case["cols"], _quant_block(case)
    y = h[..., :cols].float()
    if case["act"] == "relu":
        y = y.clamp_min(0)
    if case["gated"]:
        y = y * h[..., cols:].float()
    shape, fmax = y.shape, _LARGEST[case["q"]]
    y = torch.nn.functional.pad(y, (0, -cols % block[1], 0, -shape[1] % block[0]))
    y = y.unflatten(-1, (-1, block[1])).unflatten(-3, (-1, block[0]))        # batch, rows, of block, cols, of block
    a = y.abs().amax((-3, -1), keepdim=True)
    m, e = torch.frexp(a)                     # a = m 2^e, 0.5 <= m < 1; fmax is 0.875 times a power of two
    e = e - int(math.log2(fmax / 0.875)) + (m > 0.875).to(e.dtype)
    s = torch.where(a > 0, _power(e), torch.ones_like(a))
    q = (y / s).to(_TORCH[case["q"]]).float()
    values = (q * s).flatten(-2).flatten(1, 2)[:, :shape[1], :cols]
    return dict(values=values.to(h.dtype), scale=s.squeeze(-1).squeeze(-2))


def _dequantised(t, s, block):
    """An operand in fp32."""
    if s is None:
        return t.float()
    if s.dtype == torch.uint8:
        s = _power(s.int() - 127)
    return t.float() * _spread(s, block, t.shape)


def _plain_product(case, a, sa, b, sb, bias):
    left, right, out = _split(case)
    a, b = _dequantised(a, sa, _block_of(case, left)), _dequantised(b, sb, _block_of(case, right))
    if case["expr"] == "to,tk->ok":
        y = a.t() @ b
    else:
        y = a @ (b if right[-1] == out[-1] else b.t())
    if bias is not None:
        y = y + bias
    return y.to(_TORCH[case["out"]])


def _plain_grouped(case, groups, a, sa, b, sb):
    left, right, out = _split(case)
    a, b = _dequantised(a, sa, _block_of(case, left)), _dequantised(b, sb, _block_of(case, right))
    s, at = _sizes(case), 0
    y = torch.zeros([s[d] for d in out], device=a.device)
    for g, n in enumerate(groups):
        rows = slice(at, at + n)
        if case["expr"] == "to,tk->eok":
            y[g] = a[rows].t() @ b[rows]
        else:
            y[rows] = a[rows] @ (b[g] if right[-1] == out[-1] else b[g].t())
        at += n
    return y.to(_TORCH[case["out"]])


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["kind"] == "quant":
        return _plain_quant(case, state["in"])
    if case["kind"] == "product":
        return _plain_product(case, *state["in"])
    return _plain_grouped(case, state["groups"], *state["in"][:4])


def work(case):
    if case["kind"] == "quant":
        n, item, block = case["batch"] * case["rows"] * case["cols"], _TORCH[case["dtype"]].itemsize, _quant_block(case)
        blocks = case["batch"] * -(-case["rows"] // block[0]) * -(-case["cols"] // block[1])
        # read: the input and the gate; written: the 8-bit blocks, the values that they stand for, the scales
        return dict(bytes=n * (item * (3 if case["gated"] else 2) + 1) + 4 * blocks, flops=4 * n)
    s = _sizes(case)
    left, right, out = _split(case)
    numel = lambda t: math.prod(s[d] for d in t)  # noqa: E731
    read = dict.fromkeys((left, right))
    for t in (left, right):
        # experts without rows are not read
        n = numel(t) if "e" not in t else numel(t) // s["e"] * min(s["e"], s["t"])
        read[t] = n * _TORCH[case["left"]].itemsize
        if case["left"] != "bf16":
            b = _block_of(case, t)
            read[t] += (1 if case["scale"] == "e8m0" else 4) * n // (b[0] * b[1])
    total = sum(read.values()) + _TORCH[case["out"]].itemsize * numel(out)
    return dict(bytes=total + (4 * s["o"] if case.get("bias") else 0) + (4 * (s["e"] + 1) if "e" in s else 0),
                flops=2 * math.prod(v for d, v in s.items() if d != "e"))


def _exact_quant(case, h):
    h, cols, (br, bc), batch, rows = h.double(), case["cols"], _quant_block(case), case["batch"], case["rows"]
    y = torch.relu(h[..., :cols]) if case["act"] == "relu" else h[..., :cols]
    if case["gated"]:
        y = y * h[..., cols:]
    low, bits = (-6, 3) if case["q"] == "e4m3" else (-14, 2)
    top = {"e4m3": 8, "e5m2": 15}[case["q"]]
    full = torch.zeros((batch, -(-rows // br) * br, -(-cols // bc) * bc), dtype=torch.float64, device=y.device)
    full[:, :rows, :cols] = y
    full = full.view(batch, full.shape[1] // br, br, full.shape[2] // bc, bc).transpose(2, 3)
    a = full.abs().flatten(3).max(-1).values
    e = torch.floor(torch.log2(a)) - top
    e = torch.where(a > _LARGEST[case["q"]] * torch.exp2(e), e + 1, e)
    scale = torch.where(a > 0, torch.exp2(e), torch.ones_like(a))
    v = full / scale[..., None, None]
    step = torch.exp2(torch.floor(torch.log2(v.abs())).clamp_min(low) - bits)
    v = torch.round(v / step) * step * scale[..., None, None]
    v = v.transpose(2, 3).reshape(batch, -(-rows // br) * br, -1)[:, :rows, :cols]
    return dict(values=v.contiguous(), scale=scale)


def _exact_operand(t, s, block):
    """An operand in 64 bits: every element's scale looked up by its block."""
    t = t.double()
    if s is None:
        return t
    s = torch.exp2(s.double() - 127) if s.dtype == torch.uint8 else s.double()
    row = torch.arange(t.shape[-2], device=t.device) // block[0]
    col = torch.arange(t.shape[-1], device=t.device) // block[1]
    return t * s[..., row, :][..., col]


def exact(case, seed):
    if case["kind"] == "quant":
        return _exact_quant(case, _quant_inputs(case, seed))
    a, sa, b, sb, bias = _inputs(case, seed)
    left, right, out = _split(case)
    a = _exact_operand(a, sa, _block_of(case, left))
    b = _exact_operand(b, sb, _block_of(case, right))
    # both as [rows, contracted] and [contracted, columns]
    if left[-1] in out:
        a = a.mT.contiguous()
    if right[-1] not in out:
        b = b.mT.contiguous()
    if case["kind"] == "product":
        y = torch.matmul(a.flatten(0, -2), b).unflatten(0, a.shape[:-1])
        return y if bias is None else y + bias.double()
    n = _group_sizes(case, seed)
    if "e" in out:
        return torch.stack([torch.mm(p, q) for p, q in
                            zip(a[:, :sum(n)].split(n, 1), b[:sum(n)].split(n, 0))])
    y = [torch.mm(p, q) for p, q in zip(a[:sum(n)].split(n), b)]
    return torch.cat(y + [torch.zeros((a.shape[0] - sum(n), b.shape[-1]), dtype=a.dtype, device=a.device)])
