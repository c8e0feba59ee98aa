"""GPU parity of grouped products whose operands' modes lie in other orders than
rows of k, against 64 bits, with groups that start and end at any element.  No
counterpart in the reference."""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu


def run(torch, expr, groups, k, o, spare=0, first=0, left=eir.BF16, scale=eir.FP32, out=eir.BF16, pad=0, shift=(0, 0, 0),
        block_left=1, block_right=128, nan_group=None, seed=0):
    """One product.  NaN lies around the operands, in the rows of no group and in those of nan_group (of both operands,
    where both have rows); 7 in the output before."""
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
    contracted = [d for d in l if d in r and d not in res][0]
    unknown = [(0, first), (at[-1], sizes["t"])]
    if nan_group is not None:
        unknown.append((at[nan_group], at[nan_group + 1]))

    def operand(dims, dtype, block, shift):
        """Its buffer, address and scales, and the values that it stands for, 0 in place of NaN."""
        # blocks are along the contracted dimension and the operand's other one, wherever they lie
        order = sorted(dims, key=lambda d: (d != "e", d == contracted))
        shape = [sizes[d] for d in order]
        if f8:
            q, s, v = bp.blocks_f8(shape, (block, 128), dtype, scale, g)
        else:
            q, s = torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16), None
            v = q.double()
        q, s, v = (None if x is None else x.permute([order.index(d) for d in dims]).contiguous() for x in (q, s, v))
        if "t" in dims:
            for a, b in unknown:
                q.view(torch.uint8 if f8 else torch.int16).movedim(dims.index("t"), 0)[a:b] = 0x7f if f8 else 0x7fc0
                v.movedim(dims.index("t"), 0)[a:b] = 0.0
        buf, _, ptr = bp.strided(q, None if outer is None else [outer[d] for d in dims], float("nan"), shift)
        return buf, ptr, s, v

    # the buffers have to live as long as their addresses are used
    lbuf, pl, sl, vl = operand(l, left, block_left, shift[0])
    rbuf, pr, sr, vr = operand(r, eir.F8E4M3 if f8 else left, block_right, shift[1])
    kinds = dict(scales=True, block_left=block_left, block_right=block_right) if f8 and scale is not None else {}
    lp = eir.grouped_loops(expr, sizes, group="e", ragged="t", sizes_outer_left=outer, sizes_outer_right=outer,
                           sizes_outer_out=outer, **kinds)
    plan = eir.ContractionGroupedPlan(**lp, dtype_left=left, dtype_scale=eir.FP32 if scale is None else scale, dtype_out=out)
    shape = [sizes[d] for d in res]
    flat, view, po = bp.strided(torch.full(shape, 7.0, device="cuda", dtype=bp.TORCH[out]),
                                None if outer is None else [outer[d] for d in res], 7.0, shift[2])
    off = torch.tensor(at, dtype=torch.int32, device="cuda")
    desc = plan.describe()
    print(desc, flush=True)
    torch.cuda.synchronize()
    plan.execute(pl, pr, po, off, scale_left=sl, scale_right=sr)
    torch.cuda.synchronize()
    got = view.clone()
    view.fill_(7.0)
    assert bool((flat == 7.0).all()), f"{desc}: wrote outside the output"

    def laid(v, dims, order):
        return v.permute([dims.index(d) for d in order]).contiguous()
    m = [d for d in l if d != contracted][0]
    n = [d for d in r if d not in (contracted, "e")][0]
    canonical = ("e" if "e" not in r else "") + m + n          # of the output
    want = torch.full([sizes[d] for d in canonical], 7.0, dtype=torch.float64, device="cuda")
    mag, free = torch.zeros_like(want), torch.zeros(want.shape, dtype=torch.bool, device="cuda")
    nan = torch.zeros_like(free)
    for to, f in ((want, lambda v: v), (mag, torch.abs)):
        a = laid(f(vl), l, m + contracted)
        b = laid(f(vr), r, ("e" if "e" in r else "") + contracted + n)
        for e in range(len(groups)):
            rows = slice(at[e], at[e + 1])
            if "e" in r:
                to[rows] = a[rows] @ b[e]
                nan[rows] |= e == nan_group
            else:
                to[e] = a[:, rows].contiguous() @ b[rows]
                nan[e] |= e == nan_group and groups[e] > 0
    if "e" in r:
        for a, b in unknown[:2]:
            free[a:b] = True
    want, mag, nan, free = (v.permute([canonical.index(d) for d in res]) for v in (want, mag, nan, free))
    longest = sizes[contracted] if contracted != "t" else max(groups, default=0)
    tol = bp.tolerance(mag, want, longest, f8 and out == eir.BF16, out, f8)
    tol = torch.where(free, 0.0, tol)
    assert torch.equal(torch.isnan(got), nan), f"{desc}: NaN of another group, or none of its own"
    bp.within(torch.where(nan, 0.0, got.double()), torch.where(nan, 0.0, want), tol, desc)
    plan.close()
    del lbuf, rbuf
    return desc


GROUPS = [[1], [0], [0, 0, 5], [1, 0, 2, 0], [3, 64, 65, 0, 17], [128, 129, 1, 0, 255], [300, 0, 13], [1] * 70, [0] * 65 + [9],
          [2, 0, 1, 1, 0, 0, 4, 7] * 3, [511, 1, 640], [3, 65, 150]]
RAGGED_K = ["ot,kt->eok", "ot,tk->eok", "to,kt->eok"]


@pytest.mark.parametrize("expr", RAGGED_K)
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("groups", GROUPS, ids=lambda g: "-".join(map(str, g[:6])))
def test_ragged_k(torch_cuda, expr, groups, out):
    """272 and 144 are multiples of 16, and the number of k is made one of 8: only the groups lie anywhere."""
    spare = -sum(groups) % 8
    run(torch_cuda, expr, groups, 272, 144, spare=spare, out=out, seed=sum(groups))
    longest = max(range(len(groups)), key=lambda e: groups[e])
    run(torch_cuda, expr, groups, 272, 144, spare=spare, out=out, nan_group=longest, seed=sum(groups))


@pytest.mark.parametrize("expr", RAGGED_K + ["ot,kt->eko", "ot,tk->oek"])
@pytest.mark.parametrize("k,o", [(1, 1), (8, 8), (1, 64), (64, 1), (17, 33), (129, 127), (512, 512), (257, 640)])
def test_sizes_of_a_ragged_k(torch_cuda, expr, k, o):
    run(torch_cuda, expr, [5, 0, 150, 33], k, o, spare=1, first=3, out=eir.FP32, nan_group=3, seed=k + o)


@pytest.mark.parametrize("expr", RAGGED_K)
@pytest.mark.parametrize("shift", [(1, 0, 0), (0, 3, 0), (8, 8, 1), (5, 2, 3)])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_views_of_a_ragged_k(torch_cuda, expr, shift, pad):
    run(torch_cuda, expr, [9, 0, 140, 33], 144, 272, spare=2, pad=pad, shift=shift, nan_group=0, seed=pad)


@pytest.mark.parametrize("kernel", range(15))
@pytest.mark.parametrize("expr", RAGGED_K)
@pytest.mark.parametrize("k,o", [(272, 400), (131, 77)])
def test_every_kernel_on_a_ragged_k(torch_cuda, monkeypatch, kernel, expr, k, o):
    """A kernel that does not take the operands is not taken although it is asked for."""
    monkeypatch.setenv("ETIR_BLOCK_KERNEL", str(kernel))
    for groups in ([5, 0, 150, 33, 1], [300, 2, 0, 257]):
        for out in (eir.FP32, eir.BF16):
            run(torch_cuda, expr, groups, k, o, spare=-(2 + sum(groups)) % 8, first=2, out=out, nan_group=0, seed=k)


RAGGED_ROWS = ["kt,eko->to", "kt,eok->to", "tk,eko->to", "ot,eok->tk"]
LEFTS = [(eir.BF16, None), (eir.F8E4M3, eir.FP32), (eir.F8E5M2, eir.E8M0), (eir.F8E4M3, None)]


@pytest.mark.parametrize("expr", RAGGED_ROWS)
@pytest.mark.parametrize("left,scale", LEFTS)
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("groups", GROUPS, ids=lambda g: "-".join(map(str, g[:6])))
def test_ragged_rows(torch_cuda, expr, left, scale, groups, out):
    """The rows' number is made a multiple of 16: only the groups lie anywhere."""
    longest = max(range(len(groups)), key=lambda e: groups[e])
    run(torch_cuda, expr, groups, 272, 400, spare=-(3 + sum(groups)) % 16, first=3, left=left, scale=scale, out=out,
        nan_group=longest, seed=sum(groups))


@pytest.mark.parametrize("expr", RAGGED_ROWS + ["kt,oek->to", "kt,eko->ot", "tk,eok->ot"])
@pytest.mark.parametrize("left,scale", LEFTS)
@pytest.mark.parametrize("k,o", [(1, 1), (8, 8), (1, 64), (64, 1), (17, 33), (129, 127), (512, 512), (257, 640)])
def test_sizes_of_ragged_rows(torch_cuda, expr, left, scale, k, o):
    run(torch_cuda, expr, [5, 0, 150, 33], k, o, spare=1, first=3, left=left, scale=scale, block_left=128 if k == 17 else 1,
        block_right=1 if k == 129 else 128, nan_group=3, seed=k + o)


@pytest.mark.parametrize("expr", RAGGED_ROWS)
@pytest.mark.parametrize("left,scale", LEFTS[:2])
@pytest.mark.parametrize("shift", [(1, 0, 0), (0, 3, 0), (8, 8, 1), (5, 2, 3)])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_views_of_ragged_rows(torch_cuda, expr, left, scale, shift, pad):
    run(torch_cuda, expr, [9, 0, 140, 33], 144, 272, spare=2, left=left, scale=scale, pad=pad, shift=shift, nan_group=0, seed=pad)


@pytest.mark.parametrize("kernel", range(15))
@pytest.mark.parametrize("expr", RAGGED_ROWS)
@pytest.mark.parametrize("left,scale", LEFTS[:3])
@pytest.mark.parametrize("k,o", [(272, 400), (131, 77)])
def test_every_kernel_on_ragged_rows(torch_cuda, monkeypatch, kernel, expr, left, scale, k, o):
    monkeypatch.setenv("ETIR_BLOCK_KERNEL", str(kernel))
    for groups in ([5, 0, 150, 33, 1], [300, 2, 0, 257]):
        run(torch_cuda, expr, groups, k, o, spare=-(2 + sum(groups)) % 16, first=2, left=left, scale=scale,
            out=eir.FP32 if kernel % 2 else eir.BF16, nan_group=0, seed=k)
