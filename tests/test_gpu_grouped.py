"""GPU parity of the products grouped by expert (etir_hip_contraction_grouped_*)
against 64 bits.  No counterpart in the reference."""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu

FORWARD, GRAD_ROWS, GRAD_WEIGHTS = "tk,eok->to", "to,eok->tk", "to,tk->eok"


def run(torch, expr, groups, k, o, spare=0, first=0, left=eir.BF16, scale=eir.FP32, out=eir.BF16, pad=0, shift=(0, 0, 0),
        block_right=128, seed=0, offsets=None):
    """One product; NaN around the operands and in the rows of no group, 7 in the output before."""
    import block_products as bp
    g = torch.Generator(device="cuda").manual_seed(seed)
    at = [first]
    for n in groups:
        at.append(at[-1] + n)
    sizes = dict(t=at[-1] + spare, k=k, o=o, e=len(groups))
    outer = {d: v + (pad if d != "e" else 0) for d, v in sizes.items()} if pad else None
    ins, res = expr.split("->")
    l, r = ins.split(",")
    f8 = left != eir.BF16

    def operand(dims, dtype, contracted_last, block, shift):
        shape = [sizes[d] for d in dims]
        if f8:
            q, s, v = bp.blocks_f8(shape, (block, 128) if contracted_last else (128, block), dtype, scale, g)
        else:
            q, s = torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16), None
            v = q.double()
        if dims[0] == "t":
            for a, b in ((0, first), (at[-1], sizes["t"])):
                q.view(torch.uint8 if f8 else torch.int16)[a:b] = 0x7f if f8 else 0x7fc0
        return bp.strided(q, None if outer is None else [outer[d] for d in dims], float("nan"), shift) + (s, v)

    contracted = [d for d in l if d in r and d not in res][0]
    # the buffers have to live as long as their addresses are used
    lbuf, _, pl, sl, vl = operand(l, left, l[-1] == contracted, 1, shift[0])
    rbuf, _, pr, sr, vr = operand(r, eir.F8E4M3 if f8 else left, r[-1] == contracted, block_right, shift[1])
    kinds = dict(scales=True, block_right=block_right) if f8 and scale is not None else {}
    lp = eir.grouped_loops(expr, sizes, group="e", ragged="t", sizes_outer_left=outer, sizes_outer_right=outer,
                           sizes_outer_out=outer, **kinds)
    plan = eir.ContractionGroupedPlan(**lp, dtype_left=left, dtype_scale=eir.FP32 if scale is None else scale, dtype_out=out)
    shape = [sizes[d] for d in res]
    flat, view, po = bp.strided(torch.full(shape, 7.0, device="cuda", dtype=bp.TORCH[out]),
                                None if outer is None else [outer[d] for d in res], 7.0, shift[2])
    off = torch.tensor(at if offsets is None else offsets, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    plan.execute(pl, pr, po, off, scale_left=sl, scale_right=sr)
    torch.cuda.synchronize()
    desc = plan.describe()
    got = view.clone()
    view.fill_(7.0)
    assert bool((flat == 7.0).all()), f"{desc}: wrote outside the output"

    want = torch.full(shape, 7.0, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(want)
    longest = k if expr == FORWARD else o if expr == GRAD_ROWS else max(groups, default=0)
    for e in range(len(groups)):
        rows = slice(at[e], at[e + 1])
        for to, f in ((want, lambda v: v), (mag, torch.abs)):
            a, b = f(vl[rows]), f(vr[rows]) if expr == GRAD_WEIGHTS else f(vr[e])
            if expr == FORWARD:
                to[rows] = a @ b.t().contiguous()
            elif expr == GRAD_ROWS:
                to[rows] = a @ b
            else:
                to[e] = a.t().contiguous() @ b
    tol = bp.tolerance(mag, want, longest, f8 and out == eir.BF16, out, f8)
    if expr != GRAD_WEIGHTS:
        for a, b in ((0, first), (at[-1], sizes["t"])):
            tol[a:b] = 0.0
    bp.within(got, want, tol, desc)
    plan.close()
    del lbuf, rbuf
    return desc


GROUPS = [[1], [0], [0, 0, 5], [1, 0, 2, 0], [3, 64, 65, 0, 17], [128, 129, 1, 0, 255], [300, 0, 13], [1] * 70, [0] * 65 + [9],
          [2, 0, 1, 1, 0, 0, 4, 7] * 3, [511, 1, 640]]


@pytest.mark.parametrize("expr", [FORWARD, GRAD_ROWS, GRAD_WEIGHTS])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("groups", GROUPS, ids=lambda g: "-".join(map(str, g[:6])))
def test_groups(torch_cuda, expr, groups, out):
    run(torch_cuda, expr, groups, 272, 144, spare=3, out=out, seed=sum(groups))


@pytest.mark.parametrize("expr", [FORWARD, GRAD_ROWS])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("scale", [None, eir.FP32, eir.E8M0])
@pytest.mark.parametrize("groups", GROUPS, ids=lambda g: "-".join(map(str, g[:6])))
def test_groups_in_8_bits(torch_cuda, expr, groups, out, scale):
    run(torch_cuda, expr, groups, 272, 304, spare=3, left=eir.F8E5M2 if len(groups) == 3 else eir.F8E4M3, scale=scale, out=out,
        seed=sum(groups))


@pytest.mark.parametrize("expr", [FORWARD, GRAD_ROWS, GRAD_WEIGHTS])
@pytest.mark.parametrize("k,o", [(1, 1), (8, 8), (1, 64), (64, 1), (17, 33), (96, 40), (129, 127), (128, 256), (257, 640), (1001, 333),
                                 (1040, 16), (2048, 520)])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
def test_sizes(torch_cuda, expr, k, o, out):
    run(torch_cuda, expr, [5, 0, 150, 33], k, o, spare=2, first=3, out=out, seed=k + o)


@pytest.mark.parametrize("expr", [FORWARD, GRAD_ROWS])
@pytest.mark.parametrize("k,o", [(16, 16), (17, 33), (96, 48), (129, 127), (128, 256), (256, 640), (1001, 333), (1040, 16)])
@pytest.mark.parametrize("block_right", [1, 128])
def test_sizes_in_8_bits(torch_cuda, expr, k, o, block_right):
    run(torch_cuda, expr, [5, 0, 150, 33], k, o, spare=2, first=3, left=eir.F8E4M3, block_right=block_right, seed=k + o)


@pytest.mark.parametrize("expr", [FORWARD, GRAD_ROWS, GRAD_WEIGHTS])
@pytest.mark.parametrize("shift", [(1, 0, 0), (0, 3, 0), (8, 8, 1), (5, 2, 3)])
@pytest.mark.parametrize("pad", [0, 1, 8, 24])
@pytest.mark.parametrize("left", [eir.BF16, eir.F8E4M3])
def test_views_and_alignment(torch_cuda, expr, shift, pad, left):
    if left != eir.BF16 and expr == GRAD_WEIGHTS:
        pytest.skip("a ragged K takes bf16")
    run(torch_cuda, expr, [9, 0, 140, 33], 144, 272, spare=2, left=left, pad=pad, shift=shift, seed=pad + 3)
    run(torch_cuda, expr, [2, 1, 0, 1], 272, 144, left=left, pad=pad, shift=shift, seed=pad + 4)


@pytest.mark.parametrize("expr", [FORWARD, GRAD_WEIGHTS])
def test_one_large_and_many_small_groups(torch_cuda, expr):
    run(torch_cuda, expr, [1500] + [3] * 40 + [0] * 60 + [700], 512, 384, spare=100, seed=1)


def test_more_groups_than_a_wave(torch_cuda):
    run(torch_cuda, FORWARD, [(7 * i) % 5 for i in range(300)], 64, 48, out=eir.FP32, seed=1)
    run(torch_cuda, FORWARD, [0] * 200 + [1] + [0] * 99, 64, 48, out=eir.FP32, seed=1)


def test_gradient_against_differences(torch_cuda):
    """The three products are one function and its gradient: along random directions of rows and weights the change of
    sum(out * c) is what the gradients say (fp32 outputs of bf16 operands; the function is linear in each)."""
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(4)
    groups, k, o = [17, 0, 130, 64], 96, 80
    t, e = sum(groups), len(groups)
    off = torch.tensor([sum(groups[:i]) for i in range(e + 1)], dtype=torch.int32, device="cuda")
    sizes = dict(t=t, k=k, o=o, e=e)
    plans = {x: eir.ContractionGroupedPlan(**eir.grouped_loops(x, sizes, group="e", ragged="t"), dtype_out=eir.FP32)
             for x in (FORWARD, GRAD_ROWS, GRAD_WEIGHTS)}
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    x, w, c, dx, dw = rand(t, k), rand(e, o, k), rand(t, o), rand(t, k), rand(e, o, k)

    def call(expr, a, b, *shape):
        y = torch.zeros(*shape, device="cuda")
        torch.cuda.synchronize()
        plans[expr].execute(a, b, y, off)
        torch.cuda.synchronize()
        return y.double()
    value = lambda a, b: (call(FORWARD, a, b, t, o) * c.double()).sum()  # noqa: E731
    grad_x, grad_w = call(GRAD_ROWS, c, w, t, k), call(GRAD_WEIGHTS, c, x, e, o, k)
    # sums of t o k products of three normal numbers, each off by (K + 1) 2^-23 of its magnitude
    allowed = 8 * (t * o * k) * 200 * 2.0 ** -23 * 0.01
    assert abs(value(dx, w) - (grad_x * dx.double()).sum()) <= allowed
    assert abs(value(x, dw) - (grad_w * dw.double()).sum()) <= allowed


@pytest.mark.parametrize("expr", [FORWARD, GRAD_WEIGHTS])
@pytest.mark.parametrize("bad", [[-5, 3, 1000, 40, 41], [60, 50, 40, 30, 20], [0, 0, 0, 0, 2 ** 31 - 1], [-2 ** 31] * 5])
def test_offsets_outside_the_rows_are_cut(torch_cuda, expr, bad):
    """Nothing outside the tensors is read or written, whatever the offsets are."""
    torch = torch_cuda
    t, k, o, e = 48, 64, 32, 4
    x = torch.ones(t, k if expr == FORWARD else o, device="cuda", dtype=torch.bfloat16)
    w = torch.ones((e, o, k) if expr == FORWARD else (t, k), device="cuda", dtype=torch.bfloat16)
    shape = (t, o) if expr == FORWARD else (e, o, k)
    flat = torch.full((64 + torch.Size(shape).numel() + 64,), 7.0, device="cuda")
    y = flat[64:-64].view(shape)
    plan = eir.ContractionGroupedPlan(**eir.grouped_loops(expr, dict(t=t, k=k, o=o, e=e), group="e", ragged="t"),
                                      dtype_out=eir.FP32)
    off = torch.tensor(bad, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    plan.execute(x, w, y, off)
    torch.cuda.synchronize()
    assert bool((flat[:64] == 7.0).all()) and bool((flat[-64:] == 7.0).all())
    cut = [min(max(v, 0), t) for v in bad]
    spans = [(cut[i], max(cut[i + 1], cut[i])) for i in range(e)]
    if expr == GRAD_WEIGHTS:
        for i, (a, b) in enumerate(spans):
            assert bool((y[i] == float(b - a)).all())
    else:
        member = torch.zeros(t, dtype=torch.bool, device="cuda")
        for a, b in spans:
            member[a:b] = True
        assert bool((y[member] == float(k)).all()) and bool((y[~member] == 7.0).all())


def test_graph_replays_with_other_groups(torch_cuda):
    """The groups are read on the device: a captured product follows its offsets."""
    torch = torch_cuda
    t, k, o, e = 200, 128, 96, 6
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(t, k, device="cuda", generator=g).to(torch.bfloat16)
    w = torch.randn(e, o, k, device="cuda", generator=g).to(torch.bfloat16)
    plan = eir.ContractionGroupedPlan(**eir.grouped_loops(FORWARD, dict(t=t, k=k, o=o, e=e), group="e", ragged="t"))
    y, off = torch.zeros(t, o, device="cuda", dtype=torch.bfloat16), torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.execute(x, w, y, off, stream=torch.cuda.current_stream())
    for at in ([0, 10, 10, 100, 150, 199, 200], [0, 0, 0, 0, 0, 0, 0], [0, 200, 200, 200, 200, 200, 200], [0, 1, 2, 3, 4, 5, 6]):
        off.copy_(torch.tensor(at, dtype=torch.int32))
        y.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        again = torch.full_like(y, 7.0)
        plan.execute(x, w, again, off, stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert torch.equal(y, again)
        assert bool((y[at[-1]:] == 7.0).all())
