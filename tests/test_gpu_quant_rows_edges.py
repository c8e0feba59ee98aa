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
