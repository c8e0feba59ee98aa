"""GPU parity of the rounding to 8-bit floating point blocks
(etir_hip_quant_f8_*).  No counterpart in the reference.

Oracle: the definition in float64.  Without an activation, with ReLU, and with a
gate where the input is bf16 (a product of two bf16 numbers is exact in fp32),
every number before rounding is exact and the division by a power of two too:
scales, q and values are compared bit for bit.  SiLU carries at most 8 roundings
of 2^-24, a gate in fp32 one more: q is then within half a step and 2^-20 of y.
"""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu

GUARD = 32
LARGEST = {eir.F8E4M3: 448.0, eir.F8E5M2: 57344.0}
LOWEST = {eir.F8E4M3: (-6, 3), eir.F8E5M2: (-14, 2)}
ROWS_COLS = [(1, 1), (1, 2048), (3, 5), (2, 8), (7, 63), (5, 127), (4, 128), (9, 129), (6, 512), (3, 1000), (130, 2048), (127, 96),
             (128, 24), (129, 300), (300, 136), (1000, 24), (3, 8200), (2, 16385), (1, 40000), (257, 640)]


def _f8(torch, dtype):
    return torch.float8_e4m3fn if dtype == eir.F8E4M3 else torch.float8_e5m2


def _spread(s, block, shape):
    return s.repeat_interleave(block[0], -2)[..., :shape[-2], :].repeat_interleave(block[1], -1)[..., :shape[-1]]


def _step(torch, v, dtype):
    """The distance of 8-bit numbers around v."""
    low, bits = LOWEST[dtype]
    return torch.exp2(torch.floor(torch.log2(v.abs())).clamp_min(low) - bits)


def run(torch, rows, cols, batch=1, dtype=None, dtype_q=eir.F8E4M3, block=(1, 128), act=None, gated=False, scale=eir.FP32,
        pad=0, shift=0, values=True, seed=0, prepare=None, stream=None):
    dtype = eir.BF16 if dtype is None else dtype
    act = eir.UNDEFINED_KTYPE if act is None else act
    td = torch.bfloat16 if dtype == eir.BF16 else torch.float32
    tq = _f8(torch, dtype_q)
    g = torch.Generator(device="cuda").manual_seed(seed + rows + cols)
    ld, n = cols + pad, batch * rows

    def view(buf):
        return buf[GUARD + shift:].as_strided((batch, rows, cols), (rows * ld, ld, 1))

    def tensor(t, fill):
        buf = torch.full((n * ld + 2 * GUARD + shift,), fill, device="cuda").to(t)
        return buf, view(buf)
    ins = []
    for _ in range(2 if gated else 1):
        _, v = tensor(td, float("nan"))
        v.copy_(torch.randn((batch, rows, cols), device="cuda", generator=g))
        ins.append(v)
    x, gate = ins[0], ins[1] if gated else None
    if prepare is not None:
        prepare(x, gate)
    q_buf, q = tensor(tq, 3.0)
    v_buf, v = tensor(td, 3.0)
    blocks = (batch, -(-rows // block[0]), -(-cols // block[1]))
    s_buf = torch.full((GUARD + blocks[0] * blocks[1] * blocks[2] + GUARD,), 77.0, device="cuda")
    if scale == eir.E8M0:
        s_buf = s_buf.to(torch.uint8)
    s = s_buf[GUARD:-GUARD].view(blocks)
    plan = eir.QuantF8Plan(rows, cols, batch=batch, dtype=dtype, dtype_q=dtype_q, block=block, ktype=act, dtype_scale=scale,
                           ld_in=ld, ld_gate=ld, ld_q=ld, ld_values=ld)
    torch.cuda.synchronize()
    plan.execute(x, q, s, gate=gate, values=v if values else None, stream=stream)
    torch.cuda.synchronize()
    desc = plan.describe()
    plan.close()

    got_q, got_v, got_s = q.clone(), v.clone(), s.clone()
    q.copy_(torch.full((batch, rows, cols), 3.0, device="cuda"))
    v.fill_(3.0)
    s.fill_(77)
    assert all(bool((b.float() == k).all()) for b, k in ((q_buf, 3.0), (v_buf, 3.0), (s_buf, 77.0))), f"{desc}: wrote outside"

    y = (gate if gated else x).double()
    if act == eir.RELU:
        y = torch.where(y < 0, torch.zeros_like(y), y)
    elif act == eir.SILU:
        y = torch.where(y < -88.6, torch.zeros_like(y), y * torch.sigmoid(y))
    if gated:
        y = y * x.double()
    full = torch.zeros((batch, blocks[1] * block[0], blocks[2] * block[1]), dtype=torch.float64, device="cuda")
    full[:, :rows, :cols] = y
    a = full.view(batch, blocks[1], block[0], blocks[2], block[1]).abs().amax((2, 4))
    finite = torch.isfinite(a)
    s64 = torch.exp2(got_s.double() - 127) if scale == eir.E8M0 else got_s.double()
    if scale == eir.E8M0:
        s64 = torch.where(got_s == 255, torch.full_like(s64, float("nan")), s64)
    assert torch.equal(torch.isfinite(s64), finite), f"{desc}: scales that are not finite"
    exact = act != eir.SILU and (not gated or dtype == eir.BF16)
    fmax = LARGEST[dtype_q]
    m, e = torch.frexp(torch.where(finite, a, torch.ones_like(a)))       # fmax: 0.875 times a power of two
    want = torch.exp2((e - (9 if fmax == 448.0 else 16) + (m > 0.875)).clamp_min(-126).double())
    want = torch.where(a > 0, want, torch.ones_like(a))
    if exact:
        assert torch.equal(s64[finite], want[finite]), f"{desc}: scales"
    else:
        slack = 1 + 2.0 ** -20
        assert bool(((a <= fmax * s64 * slack) & ((a * 2 * slack >= fmax * s64) | (a == 0) | (s64 == 2.0 ** -126)))[finite].all())
    se = _spread(torch.where(finite, s64, torch.ones_like(s64)), block, (rows, cols))
    z = torch.where(_spread(finite.double(), block, (rows, cols)) > 0, y, torch.zeros_like(y)) / se
    q64 = got_q.double()
    if exact:
        step = _step(torch, z, dtype_q)
        assert torch.equal(q64, torch.round(z / step) * step), f"{desc}: q"
    else:
        assert bool(((q64 - z).abs() <= 0.5 * _step(torch, z * (1 + 2.0 ** -20), dtype_q) + z.abs() * 2.0 ** -20).all()), f"{desc}: q"
    if values:
        se = _spread(s64, block, (rows, cols))
        assert torch.equal(torch.nan_to_num(got_v, 5.0), torch.nan_to_num((q64 * se).to(td), 5.0)), f"{desc}: values"
    else:
        assert bool((got_v == 3.0).all())


BLOCKS = [(1, 128), (128, 128), (128, 1)]


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("dtype", [eir.BF16, eir.FP32])
@pytest.mark.parametrize("rows,cols", ROWS_COLS)
def test_sizes(torch_cuda, rows, cols, dtype, block):
    run(torch_cuda, rows, cols, dtype=dtype, block=block, dtype_q=eir.F8E5M2 if cols % 2 else eir.F8E4M3)


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("dtype", [eir.BF16, eir.FP32])
@pytest.mark.parametrize("dtype_q", [eir.F8E4M3, eir.F8E5M2])
@pytest.mark.parametrize("act", [eir.UNDEFINED_KTYPE, eir.RELU, eir.SILU])
@pytest.mark.parametrize("gated", [False, True])
def test_activations(torch_cuda, block, dtype, dtype_q, act, gated):
    run(torch_cuda, 140, 272, dtype=dtype, block=block, dtype_q=dtype_q, act=act, gated=gated)
    run(torch_cuda, 5, 77, dtype=dtype, block=block, dtype_q=dtype_q, act=act, gated=gated, scale=eir.E8M0, values=False)


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("pad,shift", [(1, 0), (0, 1), (3, 5), (8, 8), (16, 0)])
@pytest.mark.parametrize("dtype", [eir.BF16, eir.FP32])
@pytest.mark.parametrize("batch", [1, 3])
def test_views_and_batches(torch_cuda, block, pad, shift, dtype, batch):
    run(torch_cuda, 130, 200, batch=batch, dtype=dtype, block=block, pad=pad, shift=shift, scale=eir.E8M0)
    run(torch_cuda, 3, 17, batch=batch, dtype=dtype, block=block, pad=pad, shift=shift)


def _extremes(x, gate):
    flat = x.view(-1) if x.is_contiguous() else x[0, 0]
    n = flat.numel()
    for i, v in enumerate([0.0, -0.0, 1e-30, -1e-38, 3e38, 448.0, 449.0, 1e-45, 57344.0]):
        if i * 3 < n:
            flat[i * 3] = v


def _zeros(x, gate):
    x.zero_()


def _tiny(x, gate):
    x.mul_(1e-38)


def _tops(x, gate):
    """Blocks whose largest value is fmax times a power of two, and just above it."""
    x.clamp_(-0.5, 0.5)
    for r in range(x.shape[1]):
        x[:, r, 0] = 0.875 * 2.0 ** (r % 40 - 20) * (1 if r % 2 else 1 + 2.0 ** -7)


def _not_finite(x, gate):
    x[0, 0, 0] = float("inf")
    if x.shape[1] > 2:
        x[0, 2, x.shape[2] - 1] = float("nan")
        x[0, 1, 0] = float("-inf")


@pytest.mark.parametrize("prepare", [_extremes, _zeros, _tiny, _tops, _not_finite])
@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("dtype", [eir.BF16, eir.FP32])
@pytest.mark.parametrize("scale", [eir.FP32, eir.E8M0])
def test_borders(torch_cuda, prepare, block, dtype, scale):
    for dtype_q in (eir.F8E4M3, eir.F8E5M2):
        run(torch_cuda, 200, 257, dtype=dtype, block=block, prepare=prepare, scale=scale, dtype_q=dtype_q)


def test_nothing_to_do(torch_cuda):
    for rows, cols, batch in ((0, 5, 1), (5, 0, 1), (5, 5, 0)):
        eir.QuantF8Plan(rows, cols, batch=batch).execute(None, None, None)


def test_blocks_feed_the_products(torch_cuda):
    """A gated expert layer in 8 bits, forward: rows and weights rounded, grouped product, gated activation rounded,
    grouped product; against the same numbers in 64 bits."""
    torch = torch_cuda
    import block_products as bp
    g = torch.Generator(device="cuda").manual_seed(3)
    groups, k, f = [9, 0, 150, 41], 272, 400
    t, e = sum(groups), len(groups)
    at = [sum(groups[:i]) for i in range(e + 1)]
    s = torch.cuda.current_stream()
    rand = lambda *n: torch.randn(*n, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    x, up, down = rand(t, k), rand(e, 2 * f, k) / k ** 0.5, rand(e, k, f) / f ** 0.5
    off = torch.tensor(at, dtype=torch.int32, device="cuda")

    def quant(v, block, gate=None, act=eir.UNDEFINED_KTYPE, cols=None, ld=None):
        b, rows, cols = v.shape[0] if v.dim() == 3 else 1, v.shape[-2], cols or v.shape[-1]
        q = torch.empty([b, rows, cols], device="cuda", dtype=torch.float8_e4m3fn)
        sc = torch.empty([b, -(-rows // block[0]), -(-cols // 128)], device="cuda", dtype=torch.uint8)
        eir.QuantF8Plan(rows, cols, batch=b, block=block, ktype=act, dtype_scale=eir.E8M0, ld_in=ld, ld_gate=ld).execute(
            v, q, sc, gate=gate, stream=s)
        return q, sc, q.double() * bp.spread(torch.exp2(sc.double() - 127), block, (rows, cols))

    def product(q, sc, w, sw, n):
        y = torch.zeros(t, n, device="cuda", dtype=torch.bfloat16)
        lp = eir.grouped_loops("tk,eok->to", dict(t=t, k=q.shape[-1], o=n, e=e), group="e", ragged="t", scales=True)
        eir.ContractionGroupedPlan(**lp, dtype_left=eir.F8E4M3, dtype_scale=eir.E8M0).execute(
            q, w, y, off, scale_left=sc, scale_right=sw, stream=s)
        return y
    qx, sx, vx = quant(x, (1, 128))
    qu, su, vu = quant(up, (128, 128))
    qd, sd, vd = quant(down, (128, 128))
    h = product(qx, sx, qu, su, 2 * f)
    qa, sa, va = quant(h[:, f:], (1, 128), gate=h, act=eir.SILU, cols=f, ld=2 * f)
    y = product(qa, sa, qd, sd, k)
    torch.cuda.synchronize()
    for i in range(e):
        rows = slice(at[i], at[i + 1])
        for got, a, b in ((h, vx[0], vu[i]), (y, va[0], vd[i])):
            want, mag = a[rows] @ b.t().contiguous(), a[rows].abs() @ b.abs().t().contiguous()
            bp.within(got[rows], want, bp.tolerance(mag, want, a.shape[1], True, eir.BF16, True), f"group {i}")
