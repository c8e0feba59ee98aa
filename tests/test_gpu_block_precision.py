"""How exact the products of 8-bit floating point blocks are, on the GPU: whole
numbers, of which no kernel may lose any, and the error of a sum that a bias takes
away.  No counterpart in the reference."""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu

KERNELS = range(15)          # places of the kernels (ETIR_BLOCK_KERNEL); those that do not take the operands are not taken
DENSE = ["tk,ok->to", "to,ok->tk", "to,tk->ok", "kt,ok->to"]
GROUPED = ["tk,eok->to", "to,eok->tk", "kt,eko->to"]


def _operand(torch, g, dims, sizes, contracted, block, top, dtype, scale):
    """Whole numbers up to `top` and scales of 1 to 8 for blocks of 128 along `contracted` and `block` along the other
    dimension: in 8 bits, the scales, and what they stand for with the contracted dimension last."""
    order = sorted(dims, key=lambda d: (d != "e", d == contracted))
    shape = [sizes[d] for d in order]
    q = torch.randint(-top, top + 1, shape, device="cuda", generator=g).float()
    n = shape[:-2] + [-(-shape[-2] // block), -(-shape[-1] // 128)]
    e = torch.randint(0, 4, n, device="cuda", generator=g)
    v = q * (2.0 ** e.float()).repeat_interleave(block, -2)[..., :shape[-2], :].repeat_interleave(128, -1)[..., :shape[-1]]
    s = (127 + e).to(torch.uint8) if scale == eir.E8M0 else 2.0 ** e.float()
    back = [order.index(d) for d in dims]
    return q.permute(back).contiguous().to(dtype), s.permute(back).contiguous(), v.double()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("left", [eir.F8E4M3, eir.F8E5M2])
@pytest.mark.parametrize("scale", [eir.FP32, eir.E8M0])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("expr", DENSE + GROUPED)
def test_whole_numbers(torch_cuda, monkeypatch, kernel, left, scale, out, expr):
    """A block's products are whole numbers of up to 64, 6 binary places apart (the matrix cores cut 13 below the largest),
    scales multiply them by powers of two up to 64, and sums of 1168 stay below 2^24: all is exact but the output's one
    rounding.  A lost or doubled element, or a neighbour's scale, shows.  (e5m2 holds the whole numbers up to 4.)"""
    torch = torch_cuda
    import block_products as bp
    monkeypatch.setenv("ETIR_BLOCK_KERNEL", str(kernel))
    g = torch.Generator(device="cuda").manual_seed(kernel + 1)
    ins, res = expr.split("->")
    l, r = ins.split(",")
    contracted = [d for d in l if d in r and d not in res][0]
    groups = [101, 0, 203]
    sizes = dict(t=304, k=272, o=400, e=3)
    sizes[contracted] = 1168
    bl, br = (1, 128) if kernel % 2 else (128, 1)
    a, sa, va = _operand(torch, g, l, sizes, contracted, bl, 4 if left == eir.F8E5M2 else 8, bp.TORCH[left], scale)
    b, sb, vb = _operand(torch, g, r, sizes, contracted, br, 8, bp.TORCH[eir.F8E4M3], scale)
    y = torch.zeros([sizes[d] for d in res], device="cuda", dtype=bp.TORCH[out])
    vb = vb.mT.contiguous()
    if expr in DENSE:
        plan = eir.ContractionF8Plan(**eir.contraction_f8_loops(expr, sizes, block_left=bl, block_right=br), dtype_left=left,
                                     dtype_scale=scale, dtype_out=out)
        want, rest = va @ vb, {}
    else:
        plan = eir.ContractionGroupedPlan(**eir.grouped_loops(expr, sizes, "e", "t", scales=True, block_left=bl, block_right=br),
                                          dtype_left=left, dtype_scale=scale, dtype_out=out)
        at = [sum(groups[:i]) for i in range(4)]
        rest = dict(offsets=torch.tensor(at, dtype=torch.int32, device="cuda"))
        want = torch.cat([va[at[i]:at[i + 1]] @ vb[i] for i in range(3)])
    torch.cuda.synchronize()
    plan.execute(a, b, y, scale_left=sa, scale_right=sb, **rest)
    torch.cuda.synchronize()
    assert float(want.abs().max()) < 2 ** 24
    wrong = y != want.float().to(y.dtype)
    assert not bool(wrong.any()), f"{plan.describe()}: {int(wrong.sum())} of {wrong.numel()}, first {wrong.nonzero()[0].tolist()}"


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("left", [eir.F8E4M3, eir.F8E5M2])
@pytest.mark.parametrize("scale", [eir.FP32, eir.E8M0])
@pytest.mark.parametrize("k", [128, 2048, 8192])
def test_error_of_a_sum(torch_cuda, monkeypatch, kernel, left, scale, k):
    """Normal numbers, the bias minus their exact sum: what is left is the sum's error.  A product is cut by less than 2^-13 of
    the largest of its 8, whose square is at most the 8 squares' sum; errors of random signs then have a root mean square of
    less than 8^0.5 2^-13 that of the products' squares summed, beside (K + 4) 2^-24 of magnitudes for the additions in fp32.
    Measured: 2^-16.1 (e4m3), 2^-16.5 (e5m2) of the sums'."""
    torch = torch_cuda
    import block_products as bp
    monkeypatch.setenv("ETIR_BLOCK_KERNEL", str(kernel))
    g = torch.Generator(device="cuda").manual_seed(k)
    n = 4096
    x = bp.blocks_f8([1, k], (1, 128), left, None, g)[0]
    w = bp.blocks_f8([n, k], (1, 128), eir.F8E4M3, None, g)[0]
    p = w.double() * x.double()
    want = p.sum(1)
    bias = (-want).float()
    plan = eir.ContractionF8Plan(**eir.contraction_f8_loops("tk,ok->to", dict(t=1, k=k, o=n), bias="o", block_right=1),
                                 dtype_left=left, dtype_scale=scale, dtype_out=eir.BF16)
    y = torch.zeros(1, n, device="cuda", dtype=torch.bfloat16)
    one = lambda rows: (torch.full((rows, k // 128), 127, dtype=torch.uint8, device="cuda") if scale == eir.E8M0 else  # noqa: E731
                        torch.ones(rows, k // 128, device="cuda"))
    sx, sw = one(1), one(n)
    torch.cuda.synchronize()
    plan.execute(x, w, y, scale_left=sx, scale_right=sw, bias=bias)
    torch.cuda.synchronize()
    rms = lambda v: float(v.pow(2).mean().sqrt())  # noqa: E731
    left_over = y[0].double() - (want + bias.double())
    allowed = 8 ** 0.5 * 2.0 ** -13 * float(p.pow(2).sum(1).mean().sqrt()) + (k + 4) * 2.0 ** -24 * rms(p.abs().sum(1))
    assert rms(left_over) <= allowed, f"{plan.describe()}: {rms(left_over)} of {allowed}"
