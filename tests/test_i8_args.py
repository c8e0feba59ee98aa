"""Refusals of the 8-bit layer operators' plans: arguments are checked before
anything touches the GPU."""
import pytest

import einsum_ir_amd as eir

C, M, N, K = eir.DIM_C, eir.DIM_M, eir.DIM_N, eir.DIM_K


def _good():
    return dict(dim_types=[M, N, K], sizes=[4, 6, 8], strides_left=[8, 0, 1], strides_right=[0, 8, 1],
                strides_out=[6, 1, 0], strides_scale_left=[1, 0, 0], strides_scale_right=[0, 1, 0],
                strides_bias=[0, 1, 0])


@pytest.mark.parametrize("change,code", [
    (dict(dtype_out=eir.FP64), eir.INVALID_DTYPE),
    (dict(dtype_out=eir.INT8), eir.INVALID_DTYPE),
    (dict(ktype_last_touch=eir.ADD), eir.INVALID_KTYPE),
    (dict(ktype_last_touch=eir.SILU), eir.INVALID_KTYPE),
    (dict(dim_types=[M, N, eir.DIM_CPX]), eir.COMPILATION_FAILED),
    (dict(dim_types=[M, N, 77]), eir.COMPILATION_FAILED),
    (dict(sizes=[4, -1, 8]), eir.COMPILATION_FAILED),
    (dict(sizes=[4, 6, 131072]), eir.COMPILATION_FAILED),
    (dict(sizes=[1 << 40, 6, 8]), eir.COMPILATION_FAILED),
    (dict(sizes=[1 << 30, 1 << 30, 8], strides_out=[1 << 30, 1, 0]), eir.COMPILATION_FAILED),
    (dict(strides_left=[-8, 0, 1]), eir.COMPILATION_FAILED),
    (dict(strides_out=[6, 0, 0]), eir.COMPILATION_FAILED),
    (dict(strides_scale_left=[1, 1, 0]), eir.COMPILATION_FAILED),
    (dict(strides_scale_left=[1, 0, 1]), eir.COMPILATION_FAILED),
    (dict(strides_scale_right=[1, 1, 0]), eir.COMPILATION_FAILED),
    (dict(strides_bias=[0, 1, 1]), eir.COMPILATION_FAILED),
])
def test_contraction_i8(change, code):
    with pytest.raises(eir.EinsumIrError) as e:
        eir.ContractionI8Plan(**dict(_good(), **change))
    assert e.value.code == code


def test_contraction_i8_too_many_loops():
    n = 7
    sizes = [2] * n + [3, 8]
    far = [5 ** (n - i) for i in range(n)]
    with pytest.raises(eir.EinsumIrError) as e:
        eir.ContractionI8Plan([M] * n + [N, K], sizes, [f * 8 for f in far] + [0, 1], [0] * n + [8, 1],
                              [f * 3 for f in far] + [1, 0])
    assert e.value.code == eir.COMPILATION_FAILED


def test_null_plan_pointers():
    lib = eir.hip_lib()
    assert lib.etir_hip_contraction_i8_create(0, None, None, None, None, None, None, None, None, 0, 99, None) != 0
    assert lib.etir_hip_norm_quant_create(1, 1, 1, 1, 1, 1, 1, 0, 0, 0.0, None) != 0
    assert lib.etir_hip_act_quant_create(1, 1, 1, 1, 1, 1, 0, 99, None) != 0
    for f, n in ((lib.etir_hip_contraction_i8_execute, 7), (lib.etir_hip_norm_quant_execute, 8),
                 (lib.etir_hip_act_quant_execute, 6)):
        assert f(None, *[None] * n) == eir.CALLED_BEFORE_COMPILATION


@pytest.mark.parametrize("make,code", [
    (lambda: eir.NormQuantPlan(2, 8, dtype=eir.FP64), eir.INVALID_DTYPE),
    (lambda: eir.NormQuantPlan(2, 8, dtype_weight=eir.INT8), eir.INVALID_DTYPE),
    (lambda: eir.NormQuantPlan(-1, 8), eir.COMPILATION_FAILED),
    (lambda: eir.NormQuantPlan(2, -8), eir.COMPILATION_FAILED),
    (lambda: eir.NormQuantPlan(1 << 31, 8), eir.COMPILATION_FAILED),
    (lambda: eir.NormQuantPlan(2, 8, ld_q=7), eir.COMPILATION_FAILED),
    (lambda: eir.NormQuantPlan(2, 8, ld_values=0), eir.COMPILATION_FAILED),
    (lambda: eir.NormQuantPlan(2, 8, ld_total=4), eir.COMPILATION_FAILED),
    (lambda: eir.NormQuantPlan(2, 8, ld_in=-8), eir.COMPILATION_FAILED),
    (lambda: eir.NormQuantPlan(2, 8, eps=-1.0), eir.COMPILATION_FAILED),
    (lambda: eir.NormQuantPlan(2, 8, eps=float("nan")), eir.COMPILATION_FAILED),
    (lambda: eir.NormQuantPlan(2, 8, eps=float("inf")), eir.COMPILATION_FAILED),
    (lambda: eir.ActQuantPlan(2, 8, dtype=eir.INT8), eir.INVALID_DTYPE),
    (lambda: eir.ActQuantPlan(2, 8, ktype=eir.MADD), eir.INVALID_KTYPE),
    (lambda: eir.ActQuantPlan(2, 8, ld_gate=-1), eir.COMPILATION_FAILED),
    (lambda: eir.ActQuantPlan(2, 8, ld_q=4), eir.COMPILATION_FAILED),
    (lambda: eir.ActQuantPlan(2, -1), eir.COMPILATION_FAILED),
])
def test_rows(make, code):
    with pytest.raises(eir.EinsumIrError) as e:
        make()
    assert e.value.code == code


def test_loops_refuse_foreign_dimensions():
    sizes = dict(t=4, k=8, o=6)
    with pytest.raises(ValueError):
        eir.contraction_i8_loops("tk,ok->to", sizes, scale_left="o")
    with pytest.raises(ValueError):
        eir.contraction_i8_loops("tk,ok->to", sizes, bias="t")
    lp = eir.contraction_i8_loops("tk,ok->to", sizes, scale_left="t", scale_right="o")
    assert lp["strides_scale_left"] == [1, 0, 0] and lp["strides_scale_right"] == [0, 1, 0]
    assert lp["strides_bias"] is None and lp["strides_out"] == [6, 1, 0]


def test_other_plans_refuse_int8():
    with pytest.raises(eir.EinsumIrError) as e:
        eir.ContractionPlan([M, N, K], [4, 6, 8], [8, 0, 1], [0, 8, 1], [6, 1, 0], dtype_left=eir.INT8,
                            dtype_right=eir.INT8)
    assert e.value.code in (eir.INVALID_DTYPE, eir.UNDEFINED_ERROR)
