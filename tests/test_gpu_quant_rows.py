"""GPU parity of the operators that round rows to 8 bits (etir_hip_norm_quant_*,
etir_hip_act_quant_*).  No counterpart in the reference.

Oracle: the formulas in float64.  With y the row before rounding and a its
largest magnitude, the kernel's y carries at most 2 roundings (norm: sum and
product) or 8 (SiLU: exponential, sum, quotient, product), its 127 / a two more
and the product with it one, each 2^-24 relative: q is within 0.5 + 127 * 12 *
2^-24 < 0.5 + 1e-4 of y * 127 / a, and a scale within 12 * 2^-24 < 2^-20.
total and values are roundings of what they are defined by and compared bit for
bit.
"""
import numpy as np
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu

GUARD = 32
ROWS_COLS = [(1, 1), (1, 2048), (3, 5), (2, 8), (7, 63), (5, 64), (4, 65), (9, 511), (6, 512), (3, 1000), (2, 1025),
             (130, 2048), (3, 2049), (5, 4096), (3, 5001), (2, 8192), (3, 8200), (2, 16384), (2, 16385), (1, 40000),
             (300, 96), (1000, 24)]


def _buffer(torch, rows, ld, dtype, fill):
    return torch.full((rows * ld + 2 * GUARD,), fill, dtype=dtype, device="cuda")


def _view(buf, rows, cols, ld, shift=0):
    return buf[GUARD + shift:].as_strided((rows, cols), (ld, 1))


def _check(torch, y, q, scale, values, factor, desc):
    """y: rows before rounding and factor: of the scale, both float64."""
    y, q64, s64 = y.double(), q.double(), scale.double()
    a = y.abs().amax(-1, keepdim=True) if y.shape[1] else torch.zeros((y.shape[0], 1), device="cuda")
    exact = torch.where(a > 0, y * 127 / a, torch.zeros_like(y))
    off = float((q64 - exact).abs().max()) if q.numel() else 0.0
    assert off <= 0.5 + 1e-4, f"{desc}: q off by {off}"
    want = (a.squeeze(-1) / 127) * factor
    want = torch.where(a.squeeze(-1) > 0, want, torch.zeros_like(want))
    err = float(((s64 - want).abs() - want.abs() * 2.0 ** -20).max())
    assert err <= 0, f"{desc}: scale off by {err}"
    if values is not None:
        assert torch.equal(values, (q.float() * scale[:, None]).to(values.dtype)), f"{desc}: values"


def _rows(torch, g, rows, cols, dtype, ld, shift=0):
    buf = torch.full((rows * ld + 2 * GUARD,), float("nan"), device="cuda").to(dtype)
    v = _view(buf, rows, cols, ld, shift)
    v.copy_(torch.randn((rows, cols), device="cuda", generator=g))
    return v


def run_norm(torch, rows, cols, dtype, residual=True, weight="same", total="own", values=True, pad=0, shift=0, seed=0,
             eps=1e-6, prepare=None):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + cols)
    td = torch.bfloat16 if dtype == eir.BF16 else torch.float32
    ld = cols + pad
    x = _rows(torch, g, rows, cols, td, ld, shift)
    r = _rows(torch, g, rows, cols, td, ld, shift) if residual else None
    w = None
    if weight is not None:
        w = 1 + 0.3 * torch.randn(cols, device="cuda", generator=g)
        w = w.to(td if weight == "same" else torch.float32)
    if prepare:
        prepare(x, r)
    s32 = x.float() + (r.float() if residual else 0.0)
    x64, r64 = x.double(), r.double() if residual else None
    want_total = s32.to(td)
    bufs = dict(q=_buffer(torch, rows, ld, torch.int8, 99), v=_buffer(torch, rows, ld, td, 7.0),
                t=_buffer(torch, rows, ld, td, 7.0))
    q, v, t = (_view(bufs[n], rows, cols, ld, shift) for n in "qvt")
    if total == "residual":
        t = r
    elif total == "in":
        t = x
    scale = torch.full((rows + 2,), 5.0, device="cuda")
    plan = eir.NormQuantPlan(rows, cols, dtype=dtype, dtype_weight=eir.FP32 if weight == "fp32" else None, eps=eps,
                             ld_in=ld, ld_residual=ld, ld_total=ld, ld_q=ld, ld_values=ld)
    desc = plan.describe()
    plan.execute(x, q, scale[1:], residual=r, weight=w, total=t if total else None, values=v if values else None,
                 stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    s = x64 + r64 if residual else x64
    y = s * w.double() if w is not None else s
    rstd = 1 / torch.sqrt(s.square().mean(-1) + eps) if cols else torch.ones(rows, device="cuda").double()
    sc = scale[1:rows + 1]
    assert float(scale[0]) == 5.0 and float(scale[-1]) == 5.0
    if total:
        same = (t == want_total) | (torch.isnan(t) & torch.isnan(want_total))
        assert bool(same.all()), f"{desc}: total"
    return plan, s, y, rstd, q, sc, (v if values else None), t, bufs


def _guards(torch, bufs, rows, cols, ld, shift, written):
    """What lies between and around the rows is as it was."""
    for name, buf in bufs.items():
        fill = 99 if name == "q" else 7
        if name in written:
            _view(buf, rows, cols, ld, shift).fill_(fill)
        assert bool((buf == fill).all()), f"wrote outside of {name}"


@pytest.mark.parametrize("dtype", [eir.BF16, eir.FP32])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,cols", ROWS_COLS)
def test_norm(torch_cuda, rows, cols, residual, dtype):
    torch = torch_cuda
    plan, s, y, rstd, q, sc, v, t, bufs = run_norm(torch, rows, cols, dtype, residual=residual)
    _check(torch, y, q, sc, v, rstd, plan.describe())
    _guards(torch, bufs, rows, cols, cols, 0, "qvt")


@pytest.mark.parametrize("dtype", [eir.BF16, eir.FP32])
@pytest.mark.parametrize("cols", [40, 700, 2048, 9000])
@pytest.mark.parametrize("weight,total,values,pad,shift", [
    (None, "own", True, 0, 0), ("fp32", "own", True, 8, 0), ("same", "residual", True, 0, 0), ("same", "in", False, 3, 1),
    ("same", None, False, 16, 8), ("fp32", None, True, 1, 3), (None, "residual", True, 24, 4)])
def test_norm_options(torch_cuda, cols, weight, total, values, pad, shift, dtype):
    torch = torch_cuda
    plan, s, y, rstd, q, sc, v, t, bufs = run_norm(torch, 5, cols, dtype, weight=weight, total=total, values=values,
                                                   pad=pad, shift=shift)
    _check(torch, y, q, sc, v, rstd, plan.describe())
    _guards(torch, bufs, 5, cols, cols + pad, shift,
            "q" + ("v" if values else "") + ("t" if total == "own" else ""))


@pytest.mark.parametrize("cols", [64, 2048, 20000])
def test_norm_in_range_and_out_of_it(torch_cuda, cols):
    """Rows of zeros, of values whose squares leave fp32, of the smallest numbers, with infinities and NaN."""
    torch = torch_cuda

    def prepare(x, r):
        r.zero_()
        x[0] = 0
        x[1] *= 1e30
        x[2] *= 1e-30
        x[3] *= 1e-38
        x[4, 7] = float("inf")
        x[5, cols - 1] = float("nan")
        x[6, 0], r[6, 0] = 3e38, 3e38
        x[7] = 0
        x[7, 3] = 1e-42

    plan, s, y, rstd, q, sc, v, t, bufs = run_norm(torch, 9, cols, eir.FP32, weight=None, prepare=prepare, eps=0.0)
    good = [0, 1, 2, 8]
    _check(torch, y[good], q[good], sc[good], v[good], rstd[good].nan_to_num(posinf=0.0), plan.describe())
    # values below 2^-126 carry fewer bits: their largest is 127 and nothing is lost to zero
    assert int(q[3].abs().max()) == 127 and int(q[7, 3]) == 127 and bool(torch.isfinite(sc[[3, 7]]).all())
    assert bool(torch.isnan(sc[4:7]).all()) and int(q[4:7].abs().max()) == 0
    assert float(sc[0]) == 0.0 and int(q[0].abs().max()) == 0


def test_norm_broadcast_input(torch_cuda):
    """One row for all rows (a row stride of 0)."""
    torch = torch_cuda
    x = torch.randn(96, device="cuda").bfloat16()
    r = torch.randn((6, 96), device="cuda").bfloat16()
    q, sc = torch.empty((6, 96), dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
    plan = eir.NormQuantPlan(6, 96, ld_in=0)
    plan.execute(x, q, sc, residual=r, stream=torch.cuda.current_stream())
    s = x.double() + r.double()
    _check(torch, s, q, sc, None, 1 / torch.sqrt(s.square().mean(-1) + 1e-6), plan.describe())


F = {eir.UNDEFINED_KTYPE: lambda v: v, eir.RELU: lambda v: v.clamp_min(0), eir.SILU: lambda v: v * v.sigmoid()}


@pytest.mark.parametrize("dtype", [eir.BF16, eir.FP32])
@pytest.mark.parametrize("ktype", sorted(F))
@pytest.mark.parametrize("gated,pad,shift", [(True, 0, 0), (False, 0, 0), (True, 5, 3), (False, 8, 8)])
@pytest.mark.parametrize("rows,cols", ROWS_COLS)
def test_act(torch_cuda, rows, cols, gated, pad, shift, ktype, dtype):
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    td = torch.bfloat16 if dtype == eir.BF16 else torch.float32
    ld = (2 if gated else 1) * cols + pad
    h = _rows(torch, g, rows, (2 if gated else 1) * cols, td, ld, shift)
    x, gate = (h[:, cols:], h[:, :cols]) if gated else (h, None)
    lo = cols + pad
    bufs = dict(q=_buffer(torch, rows, lo, torch.int8, 99), v=_buffer(torch, rows, lo, td, 7.0))
    q, v = (_view(bufs[n], rows, cols, lo, shift) for n in "qv")
    sc = torch.empty(rows, device="cuda")
    plan = eir.ActQuantPlan(rows, cols, dtype=dtype, ktype=ktype, ld_in=ld, ld_gate=ld, ld_q=lo, ld_values=lo)
    plan.execute(x, q, sc, gate=gate, values=v, stream=torch.cuda.current_stream())
    y = F[ktype](gate.double()) * x.double() if gated else F[ktype](x.double())
    _check(torch, y, q, sc, v, 1.0, plan.describe())
    _guards(torch, bufs, rows, cols, lo, shift, "qv")


def test_act_edges(torch_cuda):
    """Rows of zeros (ReLU of negatives), of infinities and NaN; SiLU far out."""
    torch = torch_cuda
    x = torch.randn((6, 300), device="cuda")
    x[0] = -x[0].abs() - 0.1
    x[1, 5] = float("inf")
    x[2, 6] = float("nan")
    x[3] = torch.linspace(-200, 200, 300, device="cuda")
    q, sc = torch.empty((6, 300), dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
    for ktype in (eir.RELU, eir.SILU):
        plan = eir.ActQuantPlan(6, 300, dtype=eir.FP32, ktype=ktype)
        plan.execute(x, q, sc, stream=torch.cuda.current_stream())
        good = [0, 3, 4, 5]
        _check(torch, F[ktype](x[good].double()), q[good], sc[good], None, 1.0, plan.describe())
        assert bool(torch.isnan(sc[1:3]).all()) and int(q[1:3].abs().max()) == 0
        if ktype == eir.RELU:
            assert float(sc[0]) == 0.0 and int(q[0].abs().max()) == 0


@pytest.mark.parametrize("rows,cols", [(0, 8), (3, 0), (0, 0)])
def test_lengths_of_zero(torch_cuda, rows, cols):
    torch = torch_cuda
    x = torch.zeros(64, device="cuda").bfloat16()
    q = torch.full((64,), 9, dtype=torch.int8, device="cuda")
    sc = torch.full((8,), 5.0, device="cuda")
    for plan in (eir.NormQuantPlan(rows, cols), eir.ActQuantPlan(rows, cols)):
        sc.fill_(5.0)
        plan.execute(x, q, sc, stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert bool((q == 9).all()) and bool((sc[rows:] == 5.0).all()) and bool((sc[:rows] == 0.0).all())


def test_many_rows(torch_cuda):
    """More rows than workgroups of one launch."""
    torch = torch_cuda
    rows, cols = (1 << 20) * 4 + 777, 4
    x = torch.randn((rows, cols), device="cuda")
    q, sc = torch.empty((rows, cols), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    eir.ActQuantPlan(rows, cols, dtype=eir.FP32).execute(x, q, sc, stream=torch.cuda.current_stream())
    _check(torch, x, q, sc, None, 1.0, "many rows")


def test_row_offsets_past_32_bits(torch_cuda):
    torch = torch_cuda
    step, cols = (1 << 31) + 8, 64
    buf = torch.zeros(step + cols, device="cuda", dtype=torch.bfloat16)
    x = buf.as_strided((2, cols), (step, 1))
    x.copy_(torch.randn((2, cols), device="cuda"))
    q, sc = torch.empty((2, cols), dtype=torch.int8, device="cuda"), torch.empty(2, device="cuda")
    eir.ActQuantPlan(2, cols, ld_in=step).execute(x, q, sc, stream=torch.cuda.current_stream())
    _check(torch, x, q, sc, None, 1.0, "far rows")


def test_refuses_missing_tensors(torch_cuda):
    torch = torch_cuda
    t = torch.zeros(64, device="cuda")
    for plan in (eir.NormQuantPlan(2, 8), eir.ActQuantPlan(2, 8)):
        for missing in ("x", "q", "scale"):
            with pytest.raises(eir.EinsumIrError) as e:
                plan.execute(**dict(dict(x=t, q=t, scale=t), **{missing: None}))
            assert e.value.code == eir.NO_DATA_PTR_PROVIDED
    lib = eir.hip_lib()
    norm, act = eir.NormQuantPlan(2, 8), eir.ActQuantPlan(2, 8)
    p = t.data_ptr()
    assert lib.etir_hip_norm_quant_execute(act.handle, *[p] * 7, None) == eir.CALLED_BEFORE_COMPILATION
    assert lib.etir_hip_act_quant_execute(norm.handle, *[p] * 5, None) == eir.CALLED_BEFORE_COMPILATION
    assert lib.etir_hip_act_quant_execute(None, *[p] * 5, None) == eir.CALLED_BEFORE_COMPILATION
    assert norm.bytes == 2 * (8 * 9 + 4) + 16 and act.bytes == 2 * (8 * 7 + 4) and act.flops == 0
