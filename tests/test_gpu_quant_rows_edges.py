"""Paths of the operators that round rows to 8 bits (etir_hip_norm_quant_*) at
the ends of their arguments.  No counterpart in the reference.
"""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dtype_weight", [(eir.BF16, eir.FP32), (eir.FP32, eir.BF16), (eir.BF16, eir.BF16)])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_rows_of_nothing(torch_cuda, off, dtype, dtype_weight):
    """No columns, q off a multiple of 4 bytes and rows of it apart: scales of 0, nothing else is touched."""
    torch = torch_cuda
    td = {eir.BF16: torch.bfloat16, eir.FP32: torch.float32}
    x = torch.zeros(64, device="cuda", dtype=td[dtype])
    w = torch.ones(64, device="cuda", dtype=td[dtype_weight])
    q = torch.full((64,), 9, dtype=torch.int8, device="cuda")
    sc = torch.full((8,), 5.0, device="cuda")
    plan = eir.NormQuantPlan(5, 0, dtype=dtype, dtype_weight=dtype_weight, ld_q=1, ld_in=1, ld_total=1, ld_values=1)
    plan.execute(x, q[off:], sc, residual=x, weight=w, total=x, values=x, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert bool((q == 9).all()) and bool((x == 0).all())
    assert bool((sc[:5] == 0.0).all()) and bool((sc[5:] == 5.0).all())


@pytest.mark.parametrize("dtype,dtype_weight", [(eir.BF16, eir.FP32), (eir.FP32, eir.BF16)])
@pytest.mark.parametrize("cols", [1, 3, 5, 7, 64, 301, 2048, 9001, 20003])
@pytest.mark.parametrize("off", [0, 1])
def test_weight_of_the_other_type(torch_cuda, off, cols, dtype, dtype_weight):
    """q within 0.5 + 1e-4 of t * 127 / a and the scale within 2^-20 (2 roundings of t, two of 127 / a, one of their
    product, each 2^-24); total is a rounding of the sum, bit for bit."""
    torch = torch_cuda
    td = {eir.BF16: torch.bfloat16, eir.FP32: torch.float32}
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn((3, cols), device="cuda", generator=g).to(td[dtype])
    r = torch.randn((3, cols), device="cuda", generator=g).to(td[dtype])
    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(td[dtype_weight])
    q = torch.full((3 * cols + 8,), 99, dtype=torch.int8, device="cuda")
    sc, total = torch.empty(3, device="cuda"), torch.empty_like(x)
    plan = eir.NormQuantPlan(3, cols, dtype=dtype, dtype_weight=dtype_weight)
    plan.execute(x, q[off:], sc, residual=r, weight=w, total=total, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    s = x.double() + r.double()
    t = s * w.double()
    a = t.abs().amax(-1, keepdim=True)
    got = q[off:off + 3 * cols].reshape(3, cols).double()
    assert float((got - t * 127 / a).abs().max()) <= 0.5 + 1e-4
    want = a.squeeze(-1) / (127 * torch.sqrt(s.square().mean(-1) + 1e-6))
    assert bool(((sc.double() - want).abs() <= want * 2.0 ** -20).all())
    assert torch.equal(total, (x.float() + r.float()).to(td[dtype]))
    assert bool((q[:off] == 99).all()) and bool((q[off + 3 * cols:] == 99).all())
