"""GPU parity of the product of 8-bit floating point blocks
(etir_hip_contraction_f8_*) against 64 bits.  No counterpart in the reference."""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu


def run(torch, expr, sizes, left=eir.F8E4M3, scale=eir.FP32, out=eir.BF16, block_left=1, block_right=128, bias=False,
        relu=False, outer=(None, None, None), shift=(0, 0, 0), seed=0, stream=None):
    """One product; what lies around the operands is NaN, what lies around the output has to stay."""
    import block_products as bp
    g = torch.Generator(device="cuda").manual_seed(seed)
    ins, res = expr.split("->")
    l, r = ins.split(",")
    contracted = [d for d in l if d in r and d not in res][0]

    def operand(dims, dtype, block, outer, shift):
        b = (block, 128) if dims[-1] == contracted else (128, block)
        # a tensor of one dimension beside the contracted one, or a batch of such
        q, s, v = bp.blocks_f8([sizes[d] for d in dims], b, dtype, scale, g)
        return bp.strided(q, None if outer is None else [outer[d] for d in dims], float("nan"), shift) + (s, v)

    # the buffers have to live as long as their addresses are used
    lbuf, _, pl, sl, vl = operand(l, left, block_left, outer[0], shift[0])
    rbuf, _, pr, sr, vr = operand(r, eir.F8E4M3, block_right, outer[1], shift[1])
    free = [d for d in r if d in res and d not in l][0]
    c = torch.randn(sizes[free], device="cuda", generator=g) if bias else None
    lp = eir.contraction_f8_loops(expr, sizes, block_left=block_left, block_right=block_right, scales=scale is not None,
                                  bias=free if bias else None, sizes_outer_left=outer[0], sizes_outer_right=outer[1],
                                  sizes_outer_out=outer[2])
    plan = eir.ContractionF8Plan(**lp, dtype_left=left, dtype_scale=eir.FP32 if scale is None else scale, dtype_out=out,
                                 ktype_last_touch=eir.RELU if relu else eir.UNDEFINED_KTYPE)
    shape = [sizes[d] for d in res]
    flat, view, po = bp.strided(torch.full(shape, 7.0, device="cuda", dtype=bp.TORCH[out]),
                                None if outer[2] is None else [outer[2][d] for d in res], 7.0, shift[2])
    torch.cuda.synchronize()
    plan.execute(pl, pr, po, scale_left=sl, scale_right=sr, bias=c, stream=stream)
    torch.cuda.synchronize()
    desc = plan.describe()
    got = view.clone()
    view.fill_(7.0)
    assert bool((flat == 7.0).all()), f"{desc}: wrote outside the output"
    # in float64 on the CPU's side of einsum: only matrix products of contiguous operands
    want, mag = torch.einsum(expr, vl.cpu(), vr.cpu()).cuda(), torch.einsum(expr, vl.abs().cpu(), vr.abs().cpu()).cuda()
    if c is not None:
        at = [sizes[d] if d == free else 1 for d in res]
        want, mag = want + c.double().view(at), mag + c.abs().double().view(at)
    if relu:
        want = want.clamp_min(0)
    tol = bp.tolerance(mag, want, sizes[contracted], out == eir.BF16, out, scale is not None)
    bp.within(got, want, tol, desc)
    plan.close()
    del lbuf, rbuf
    return desc


# one to many of every size, odd ones, and sizes next to the tiles' and blocks' edges
MKN = [(1, 1, 1), (1, 2048, 2048), (1, 16, 33), (2, 17, 1), (3, 15, 5), (5, 64, 31), (7, 65, 64), (16, 128, 16),
       (17, 127, 15), (24, 4096, 640), (31, 96, 257), (33, 1001, 77), (64, 129, 65), (65, 256, 63), (100, 784, 10),
       (127, 1040, 130), (128, 512, 128), (129, 1024, 256), (200, 48, 300), (256, 384, 256), (257, 640, 528),
       (700, 784, 512), (300, 2048, 1), (512, 16, 512), (511, 80, 1040), (1025, 208, 304)]


@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("m,k,n", MKN)
def test_tokens_times_channels(torch_cuda, m, k, n, out):
    run(torch_cuda, "tk,ok->to", dict(t=m, k=k, o=n), out=out, seed=m + k + n, relu=(m + n) % 2 == 0, bias=n % 3 == 0)


@pytest.mark.parametrize("scale", [None, eir.FP32, eir.E8M0])
@pytest.mark.parametrize("left", [eir.F8E4M3, eir.F8E5M2])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("m,k,n", [(1, 400, 70), (9, 1024, 256), (150, 272, 144), (290, 1152, 400)])
def test_types(torch_cuda, m, k, n, left, scale, out):
    run(torch_cuda, "tk,ok->to", dict(t=m, k=k, o=n), left=left, scale=scale, out=out, seed=m)


@pytest.mark.parametrize("blocks", [(1, 1), (1, 128), (128, 1), (128, 128)])
@pytest.mark.parametrize("expr", ["tk,ok->to", "to,ok->tk", "to,tk->ok", "kt,ok->to", "tk,ok->ot", "kt,ko->ot"])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
def test_layouts_and_blocks(torch_cuda, expr, blocks, out):
    run(torch_cuda, expr, dict(t=272, k=400, o=304), block_left=blocks[0], block_right=blocks[1], out=out, seed=5,
        scale=eir.E8M0 if blocks[0] == 1 else eir.FP32)


@pytest.mark.parametrize("expr", ["to,ok->tk", "to,tk->ok", "kt,ko->to"])
@pytest.mark.parametrize("m,k,n", [(1, 40, 96), (70, 100, 33), (130, 64, 208), (96, 1, 17), (300, 1040, 272), (33, 257, 31)])
@pytest.mark.parametrize("left", [eir.F8E4M3, eir.F8E5M2])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
def test_orders_of_modes(torch_cuda, expr, m, k, n, left, out):
    run(torch_cuda, expr, dict(t=m, k=k, o=n), left=left, out=out, block_right=1 if expr == "to,tk->ok" else 128, seed=m * k)


@pytest.mark.parametrize("expr,sizes", [
    ("btk,ok->bto", dict(b=3, t=37, k=144, o=70)),
    ("btk,ok->bto", dict(b=4, t=129, k=256, o=272)),
    ("ztk,zok->zto", dict(z=5, t=77, k=1001, o=33)),
    ("ztk,zok->zto", dict(z=3, t=140, k=256, o=272)),
    ("ztk,zok->zto", dict(z=9, t=1, k=256, o=300)),
    ("tk,ok->to", dict(t=6, k=0, o=5)),
    ("tk,ok->to", dict(t=0, k=32, o=5)),
    ("ztk,zok->zto", dict(z=0, t=4, k=32, o=5)),
])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
def test_modes_and_batches(torch_cuda, expr, sizes, out):
    run(torch_cuda, expr, sizes, out=out, seed=3)


@pytest.mark.parametrize("shift", [(1, 0, 0), (0, 3, 0), (16, 16, 1), (4, 8, 2), (7, 9, 3), (0, 0, 1)])
@pytest.mark.parametrize("m,k,n", [(1, 1040, 96), (12, 272, 100), (300, 256, 272)])
@pytest.mark.parametrize("expr", ["tk,ok->to", "to,ok->tk"])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
def test_any_alignment(torch_cuda, m, k, n, shift, expr, out):
    run(torch_cuda, expr, dict(t=m, k=k, o=n), out=out, shift=shift, seed=11)


@pytest.mark.parametrize("pad", [1, 16, 48])
@pytest.mark.parametrize("m,k,n", [(1, 256, 96), (20, 272, 112), (300, 384, 272)])
@pytest.mark.parametrize("expr", ["tk,ok->to", "to,ok->tk", "to,tk->ok"])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
def test_views_into_larger_tensors(torch_cuda, m, k, n, pad, expr, out):
    sizes = dict(t=m, k=k, o=n)
    outer = {d: v + pad for d, v in sizes.items()}
    run(torch_cuda, expr, sizes, out=out, outer=(outer, outer, outer), block_right=1 if expr == "to,tk->ok" else 128, seed=7)


def test_two_streams_and_a_graph(torch_cuda):
    """Executions of one plan overlap; a captured one replays like the eager one."""
    torch = torch_cuda
    import block_products as bp
    g = torch.Generator(device="cuda").manual_seed(1)
    t, k, o = 300, 640, 272
    plan = eir.ContractionF8Plan(**eir.contraction_f8_loops("tk,ok->to", dict(t=t, k=k, o=o)), dtype_out=eir.BF16)
    w, sw, _ = bp.blocks_f8([o, k], (128, 128), eir.F8E4M3, eir.FP32, g)
    xs = [bp.blocks_f8([t, k], (1, 128), eir.F8E4M3, eir.FP32, g) for _ in range(3)]
    outs = [torch.empty(t, o, device="cuda", dtype=torch.bfloat16) for _ in xs]
    for (x, sx, _), y in zip(xs, outs):
        plan.execute(x, w, y, scale_left=sx, scale_right=sw, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    want = [y.clone() for y in outs]
    streams = [torch.cuda.Stream() for _ in xs]
    for y in outs:
        y.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (x, sx, _), y in zip(streams, xs, outs):
            plan.execute(x, w, y, scale_left=sx, scale_right=sw, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    x, sx = xs[0][0].clone(), xs[0][1].clone()
    y = torch.zeros_like(outs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.execute(x, w, y, scale_left=sx, scale_right=sw, stream=torch.cuda.current_stream())
    for i in (1, 2, 0, 1):
        x.copy_(xs[i][0])
        sx.copy_(xs[i][1])
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])


@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("scale", [eir.FP32, eir.E8M0])
@pytest.mark.parametrize("m,k,n", [(3, 300, 40), (140, 272, 144), (300, 1024, 272)])
def test_nan_stays_in_its_row(torch_cuda, m, k, n, scale, out):
    """A NaN scale or operand makes its own row (column) NaN and nothing else."""
    torch = torch_cuda
    import block_products as bp
    g = torch.Generator(device="cuda").manual_seed(2)
    x, sx, _ = bp.blocks_f8([m, k], (1, 128), eir.F8E4M3, scale, g)
    w, sw, _ = bp.blocks_f8([n, k], (1, 128), eir.F8E4M3, scale, g)
    sx[1, 0] = 255 if scale == eir.E8M0 else float("nan")
    w.view(torch.uint8)[7, k - 1] = 0x7f
    plan = eir.ContractionF8Plan(**eir.contraction_f8_loops("tk,ok->to", dict(t=m, k=k, o=n), block_right=1), dtype_out=out,
                                 dtype_scale=scale)
    y = torch.zeros(m, n, device="cuda", dtype=bp.TORCH[out])
    torch.cuda.synchronize()
    plan.execute(x, w, y, scale_left=sx, scale_right=sw)
    torch.cuda.synchronize()
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[1] = True
    bad[:, 7] = True
    assert torch.equal(torch.isnan(y), bad)
