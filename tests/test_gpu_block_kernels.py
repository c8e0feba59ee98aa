"""Every kernel of the products of 8-bit floating point and of the grouped
products, forced where it takes the operands (ETIR_BLOCK_KERNEL), and operands far
apart.  The products themselves: test_gpu_contract_f8.py, test_gpu_grouped.py."""
import pytest

import einsum_ir_amd as eir
import test_gpu_contract_f8 as dense
import test_gpu_grouped as grouped

pytestmark = pytest.mark.gpu

KERNELS = ["general", "few 4", "few 8 parts", "few 16", "few 32", "tile 32x32", "tile 64x64 K", "tile 64x64", "tile 128x128",
           "tile 256x128", "tile 256x256", "staged 32x32", "staged 64x64 K", "staged 64x64", "staged 128x128"]


@pytest.fixture(params=range(len(KERNELS)), ids=lambda i: KERNELS[i].replace(" ", "_"))
def forced(request, monkeypatch):
    monkeypatch.setenv("ETIR_BLOCK_KERNEL", str(request.param))
    return KERNELS[request.param]


def _ran(desc, name, fits):
    assert (f" {name} C=" in desc or f" {name} groups=" in desc) == fits, desc


@pytest.mark.parametrize("expr", ["tk,ok->to", "to,ok->tk", "to,tk->ok"])
@pytest.mark.parametrize("left,scale", [(eir.F8E4M3, eir.FP32), (eir.F8E4M3, eir.E8M0), (eir.F8E5M2, eir.FP32), (eir.F8E5M2, None)])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("t,k,o", [(300, 640, 400), (77, 273, 131)])
def test_dense(torch_cuda, forced, expr, left, scale, out, t, k, o):
    desc = dense.run(torch_cuda, expr, dict(t=t, k=k, o=o), left=left, scale=scale, out=out, bias=expr == "tk,ok->to",
                     block_right=1 if expr == "to,tk->ok" else 128, seed=t)
    direct = t == 300 and scale is not None and not (out == eir.FP32 and forced == "tile 256x256")
    if forced.startswith("tile"):
        # the rows' stride has to be a multiple of 16 bytes
        _ran(desc, forced, direct)
    elif forced.startswith("few"):
        _ran(desc, forced, expr == "tk,ok->to")
    else:
        _ran(desc, forced, True)


@pytest.mark.parametrize("expr", [grouped.FORWARD, grouped.GRAD_ROWS, grouped.GRAD_WEIGHTS])
@pytest.mark.parametrize("left", [eir.BF16, eir.F8E4M3])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("k,o", [(272, 400), (131, 77)])
def test_groups(torch_cuda, forced, expr, left, out, k, o):
    if left != eir.BF16 and expr == grouped.GRAD_WEIGHTS:
        pytest.skip("a ragged K takes bf16")
    for groups in ([5, 0, 150, 33, 1], [300, 2, 0, 257]):
        desc = grouped.run(torch_cuda, expr, groups, k, o, spare=3, first=2, left=left, out=out, seed=k)
        if forced.startswith("tile"):
            _ran(desc, forced, k == 272 and not (out == eir.FP32 and left != eir.BF16 and forced == "tile 256x256"))
        elif forced.startswith("few"):
            _ran(desc, forced, expr == grouped.FORWARD)
        else:
            _ran(desc, forced, True)


@pytest.mark.parametrize("expr", [grouped.FORWARD, grouped.GRAD_WEIGHTS])
def test_a_nan_stays_in_its_group(torch_cuda, forced, expr):
    """A row of NaN makes its own row, or its own group's weights, NaN."""
    torch = torch_cuda
    groups, k, o = [70, 1, 130], 144, 80
    t, e = sum(groups), len(groups)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(t, k if expr == grouped.FORWARD else o, device="cuda", generator=g).to(torch.bfloat16)
    w = torch.randn((e, o, k) if expr == grouped.FORWARD else (t, k), device="cuda", generator=g).to(torch.bfloat16)
    x[70] = float("nan")          # group 1, between the others
    off = torch.tensor([0, 70, 71, 201], dtype=torch.int32, device="cuda")
    y = torch.zeros((t, o) if expr == grouped.FORWARD else (e, o, k), device="cuda")
    plan = eir.ContractionGroupedPlan(**eir.grouped_loops(expr, dict(t=t, k=k, o=o, e=e), group="e", ragged="t"), dtype_out=eir.FP32)
    torch.cuda.synchronize()
    plan.execute(x, w, y, off)
    torch.cuda.synchronize()
    bad = torch.isnan(y)
    if expr == grouped.FORWARD:
        assert bool(bad[70].all()) and not bool(bad[:70].any()) and not bool(bad[71:].any())
    else:
        assert bool(bad[1].all()) and not bool(bad[0].any()) and not bool(bad[2].any())


# ---- operands far apart: offsets beyond 32 bits -----------------------------

FAR = 6 << 30        # bytes of a buffer


def _far_view(torch, shape, strides, dtype):
    """A strided view into a large buffer of its own."""
    item = torch.empty(0, dtype=dtype).element_size()
    assert sum((n - 1) * s for n, s in zip(shape, strides)) * item < FAR
    return torch.empty(FAR // item, dtype=dtype, device="cuda").as_strided(shape, strides)


@pytest.mark.parametrize("kernel", [None, 0, 1, 3, 7, 13])
@pytest.mark.parametrize("what,m,n,k", [
    ("left rows", 5, 48, 144), ("left rows", 40, 80, 272), ("right rows", 33, 5, 144), ("right rows", 3, 40, 256),
    ("left k", 32, 48, 600), ("right k", 33, 48, 600), ("out rows", 5, 48, 144)])
def test_far_operands(torch_cuda, monkeypatch, kernel, what, m, n, k):
    torch = torch_cuda
    import block_products as bp
    if kernel is not None:
        monkeypatch.setenv("ETIR_BLOCK_KERNEL", str(kernel))
    g = torch.Generator(device="cuda").manual_seed(1)
    f8 = torch.float8_e4m3fn
    a, sa, va = bp.blocks_f8([m, k], (1, 128), eir.F8E4M3, eir.FP32, g)
    b, sb, vb = bp.blocks_f8([n, k], (1, 128), eir.F8E4M3, eir.FP32, g)
    step = lambda count: (FAR - (1 << 20)) // count // 16 * 16  # noqa: E731
    s_a, s_b, s_o = [k, 1], [k, 1], [n, 1]
    if what == "left rows":
        s_a = [step(m), 1]
    elif what == "right rows":
        s_b = [step(n), 1]
    elif what == "left k":
        s_a = [1, step(k)]
    elif what == "right k":
        s_b = [1, step(k)]
    else:
        s_o = [step(m) // 4, 1]
    left = _far_view(torch, [m, k], s_a, f8) if what.startswith("left") else torch.empty([m, k], dtype=f8, device="cuda")
    right = _far_view(torch, [n, k], s_b, f8) if what.startswith("right") else torch.empty([n, k], dtype=f8, device="cuda")
    out = _far_view(torch, [m, n], s_o, torch.float32) if what == "out rows" else torch.empty([m, n], device="cuda")
    left.copy_(a)
    right.copy_(b)
    kb = -(-k // 128)
    plan = eir.ContractionF8Plan([eir.DIM_M, eir.DIM_N, eir.DIM_K], [m, n, k], [s_a[0], 0, s_a[1]], [0, s_b[0], s_b[1]], [s_o[0], s_o[1], 0],
                                 [kb, 0, 1], [0, kb, 1], block_right=1, dtype_out=eir.FP32)
    torch.cuda.synchronize()
    plan.execute(left, right, out, scale_left=sa, scale_right=sb)
    torch.cuda.synchronize()
    want, mag = va @ vb.t().contiguous(), va.abs() @ vb.abs().t().contiguous()
    bp.within(out, want, bp.tolerance(mag, want, k, False, eir.FP32, True), plan.describe())


@pytest.mark.parametrize("kernel", [None, 0, 3, 7, 13])
@pytest.mark.parametrize("groups", [[2, 0, 3], [70, 5, 0]])
def test_far_experts(torch_cuda, monkeypatch, kernel, groups):
    torch = torch_cuda
    import block_products as bp
    if kernel is not None:
        monkeypatch.setenv("ETIR_BLOCK_KERNEL", str(kernel))
    g = torch.Generator(device="cuda").manual_seed(2)
    t, e, k, o = sum(groups), 3, 96, 40
    far = (FAR // 2 - (1 << 20)) // 2 // 8 * 8
    at = [0, groups[0], groups[0] + groups[1], t]
    x = torch.randn(t, k, device="cuda", generator=g).to(torch.bfloat16)
    w = _far_view(torch, [e, o, k], [far, k, 1], torch.bfloat16)
    w.copy_(torch.randn(e, o, k, device="cuda", generator=g))
    off = torch.tensor(at, dtype=torch.int32, device="cuda")
    y = torch.zeros(t, o, device="cuda")
    plan = eir.ContractionGroupedPlan([eir.DIM_G, eir.DIM_M, eir.DIM_N, eir.DIM_K], [e, t, o, k], [0, k, 0, 1], [far, 0, k, 1],
                                      [0, o, 1, 0], 1, dtype_out=eir.FP32)
    torch.cuda.synchronize()
    plan.execute(x, w, y, off)
    torch.cuda.synchronize()
    for i in range(e):
        a, b = x[at[i]:at[i + 1]].double(), w[i].double().t().contiguous()
        want, mag = a @ b, a.abs() @ b.abs()
        bp.within(y[at[i]:at[i + 1]], want, bp.tolerance(mag, want, k, False, eir.FP32, False), plan.describe())


def test_far_rows_are_rounded(torch_cuda):
    torch = torch_cuda
    rows, cols = 5, 300
    far = (FAR // 2 - (1 << 20)) // rows
    x = _far_view(torch, [rows, cols], [far, 1], torch.bfloat16)
    x.copy_(torch.randn(rows, cols, device="cuda"))
    for block in ((1, 128), (128, 128), (128, 1)):
        q = _far_view(torch, [rows, cols], [far, 1], torch.float8_e4m3fn)
        near_q = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
        n = (-(-rows // block[0])) * (-(-cols // block[1]))
        s, near_s = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        near = x.contiguous()
        torch.cuda.synchronize()
        eir.QuantF8Plan(rows, cols, block=block, ld_in=far, ld_q=far).execute(x, q, s)
        eir.QuantF8Plan(rows, cols, block=block).execute(near, near_q, near_s)
        torch.cuda.synchronize()
        assert torch.equal(q.contiguous().view(torch.uint8), near_q.view(torch.uint8)) and torch.equal(s, near_s)


@pytest.mark.parametrize("left", [eir.F8E4M3, eir.F8E5M2])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("expr", ["tk,ok->to", "to,ok->tk", "to,tk->ok"])
def test_ends_of_byte_scales(torch_cuda, forced, left, out, expr):
    """Bytes 0 (2^-127) and 254 (2^127), one of each in every block's pair, so that each pair's product is 1."""
    torch = torch_cuda
    import block_products as bp
    g = torch.Generator(device="cuda").manual_seed(11)
    sizes = dict(t=272, k=400, o=304)
    ins, res = expr.split("->")
    l, r = ins.split(",")
    contracted = [d for d in l if d in r and d not in res][0]
    block = [(1, 128) if d[-1] == contracted else (128, 1) for d in (l, r)]
    x, sx, _ = bp.blocks_f8([sizes[d] for d in l], block[0], left, eir.E8M0, g)
    w, sw, _ = bp.blocks_f8([sizes[d] for d in r], block[1], eir.F8E4M3, eir.E8M0, g)
    ends = torch.tensor([0, 254, 1, 253], dtype=torch.uint8, device="cuda")
    for s, dims, turn in ((sx, l, ends), (sw, r, 254 - ends)):
        n = s.shape[-1] if dims[-1] == contracted else s.shape[-2]
        s.copy_(turn[:n] if dims[-1] == contracted else turn[:n, None])
    plan = eir.ContractionF8Plan(**eir.contraction_f8_loops(expr, sizes, block_right=1), dtype_left=left,
                                 dtype_scale=eir.E8M0, dtype_out=out)
    y = torch.zeros([sizes[d] for d in res], device="cuda", dtype=bp.TORCH[out])
    torch.cuda.synchronize()
    plan.execute(x, w, y, scale_left=sx, scale_right=sw)
    torch.cuda.synchronize()
    vx, vw = x.cpu().float().double(), w.cpu().float().double()
    want, mag = torch.einsum(expr, vx, vw).cuda(), torch.einsum(expr, vx.abs(), vw.abs()).cuda()
    bp.within(y, want, bp.tolerance(mag, want, sizes[contracted], out == eir.BF16, out, True), plan.describe())
