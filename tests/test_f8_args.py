"""Refusals of the plans of 8-bit floating point and of grouped products:
arguments are checked before anything touches the GPU."""
import pytest

import einsum_ir_amd as eir

C, M, N, K, G = eir.DIM_C, eir.DIM_M, eir.DIM_N, eir.DIM_K, eir.DIM_G


def _good():
    return dict(dim_types=[M, N, K], sizes=[4, 6, 300], strides_left=[300, 0, 1], strides_right=[0, 300, 1],
                strides_out=[6, 1, 0], strides_scale_left=[3, 0, 1], strides_scale_right=[0, 3, 1], strides_bias=[0, 1, 0],
                block_left=1, block_right=1)


@pytest.mark.parametrize("change,code", [
    (dict(dtype_out=eir.FP64), eir.INVALID_DTYPE),
    (dict(dtype_out=eir.F8E4M3), eir.INVALID_DTYPE),
    (dict(dtype_left=eir.BF16), eir.INVALID_DTYPE),
    (dict(dtype_left=eir.INT8), eir.INVALID_DTYPE),
    (dict(dtype_right=eir.F8E5M2), eir.INVALID_DTYPE),
    (dict(dtype_scale=eir.BF16), eir.INVALID_DTYPE),
    (dict(ktype_last_touch=eir.SILU), eir.INVALID_KTYPE),
    (dict(block_left=2), eir.COMPILATION_FAILED),
    (dict(block_right=0), eir.COMPILATION_FAILED),
    (dict(dim_types=[M, N, eir.DIM_CPX]), eir.COMPILATION_FAILED),
    (dict(dim_types=[M, N, 77]), eir.COMPILATION_FAILED),
    (dict(dim_types=[M, G, K]), eir.COMPILATION_FAILED),
    (dict(sizes=[4, -1, 300]), eir.COMPILATION_FAILED),
    (dict(sizes=[1 << 40, 6, 300]), eir.COMPILATION_FAILED),
    (dict(sizes=[1 << 30, 1 << 30, 8], strides_out=[1 << 30, 1, 0]), eir.COMPILATION_FAILED),
    (dict(strides_left=[-8, 0, 1]), eir.COMPILATION_FAILED),
    (dict(strides_left=[1 << 60, 0, 1]), eir.COMPILATION_FAILED),
    (dict(strides_out=[6, 0, 0]), eir.COMPILATION_FAILED),
    (dict(strides_scale_left=[3, 1, 1]), eir.COMPILATION_FAILED),
    (dict(strides_scale_right=[1, 3, 1]), eir.COMPILATION_FAILED),
    (dict(strides_bias=[0, 1, 1]), eir.COMPILATION_FAILED),
])
def test_contraction_f8(change, code):
    with pytest.raises(eir.EinsumIrError) as e:
        eir.ContractionF8Plan(**dict(_good(), **change))
    assert e.value.code == code


def test_loops_that_do_not_fuse():
    """Rows of a view whose two loops do not fuse, blocks of 128 over two loops, two K loops."""
    with pytest.raises(eir.EinsumIrError):
        eir.ContractionF8Plan(**eir.contraction_f8_loops("btk,ok->bto", dict(b=3, t=4, k=128, o=8),
                                                         sizes_outer_left=dict(b=3, t=9, k=128)))
    with pytest.raises(eir.EinsumIrError):
        eir.ContractionF8Plan(**eir.contraction_f8_loops("btk,ok->bto", dict(b=3, t=4, k=128, o=8), block_left=128))
    with pytest.raises(ValueError):
        eir.contraction_f8_loops("tkl,okl->to", dict(t=3, k=4, l=5, o=8))
    with pytest.raises(eir.EinsumIrError):
        eir.ContractionF8Plan(**eir.contraction_f8_loops("tkl,okl->to", dict(t=3, k=4, l=5, o=8), scales=False))
    with pytest.raises(ValueError):
        eir.contraction_f8_loops("tk,ok->to", dict(t=3, k=4, o=8), bias="t")


def test_lists_that_do_not_fit():
    with pytest.raises(ValueError):
        eir.ContractionF8Plan(**dict(_good(), strides_left=[300, 0]))
    with pytest.raises(ValueError):
        eir.ContractionF8Plan(**dict(_good(), strides_scale_right=[0, 3, 1, 0]))
    with pytest.raises(ValueError):
        eir.ContractionGroupedPlan([G, M, N, K], [2, 4, 6, 8], [0, 8, 0, 1], [48, 0, 8, 1], [0, 6, 1], 1)


def _grouped():
    return dict(dim_types=[G, M, N, K], sizes=[3, 40, 6, 8], strides_left=[0, 8, 0, 1], strides_right=[48, 0, 8, 1],
                strides_out=[0, 6, 1, 0], ragged=1)


@pytest.mark.parametrize("change,code", [
    (dict(dtype_left=eir.FP32), eir.INVALID_DTYPE),
    (dict(dtype_right=eir.F8E4M3), eir.INVALID_DTYPE),
    (dict(dtype_left=eir.F8E4M3, dtype_right=eir.BF16), eir.INVALID_DTYPE),
    (dict(dtype_out=eir.INT8), eir.INVALID_DTYPE),
    (dict(strides_scale_left=[0, 1, 0, 1]), eir.INVALID_DTYPE),
    (dict(ragged=-1), eir.COMPILATION_FAILED),
    (dict(ragged=4), eir.COMPILATION_FAILED),
    (dict(ragged=2), eir.COMPILATION_FAILED),
    (dict(ragged=0), eir.COMPILATION_FAILED),
    (dict(dim_types=[C, M, N, K]), eir.COMPILATION_FAILED),
    (dict(dim_types=[M, M, N, K], strides_left=[999, 8, 0, 1], strides_out=[999, 6, 1, 0]), eir.COMPILATION_FAILED),
    (dict(dim_types=[G, M, G, K]), eir.COMPILATION_FAILED),
    (dict(sizes=[3, -4, 6, 8]), eir.COMPILATION_FAILED),
    (dict(strides_out=[0, 0, 1, 0]), eir.COMPILATION_FAILED),
])
def test_contraction_grouped(change, code):
    with pytest.raises(eir.EinsumIrError) as e:
        eir.ContractionGroupedPlan(**dict(_grouped(), **change))
    assert e.value.code == code


def test_grouped_k_takes_bf16():
    lp = eir.grouped_loops("to,tk->eok", dict(t=40, k=8, o=6, e=3), group="e", ragged="t")
    with pytest.raises(eir.EinsumIrError) as e:
        eir.ContractionGroupedPlan(**lp, dtype_left=eir.F8E4M3)
    assert e.value.code == eir.INVALID_DTYPE
    # groups whose output matrices lie on each other
    with pytest.raises(eir.EinsumIrError):
        eir.ContractionGroupedPlan(**dict(lp, strides_out=[0] + lp["strides_out"][1:]))


def test_grouped_loops():
    sizes = dict(t=40, k=8, o=6, e=3)
    lp = eir.grouped_loops("tk,eok->to", sizes, group="e", ragged="t")
    assert lp == dict(dim_types=[G, M, N, K], sizes=[3, 40, 6, 8], strides_left=[0, 8, 0, 1], strides_right=[48, 0, 8, 1],
                      strides_out=[0, 6, 1, 0], ragged=1)
    lp = eir.grouped_loops("to,tk->eok", sizes, group="e", ragged="t")
    assert lp == dict(dim_types=[G, M, N, K], sizes=[3, 6, 8, 40], strides_left=[0, 1, 0, 6], strides_right=[0, 0, 1, 8],
                      strides_out=[48, 8, 1, 0], ragged=3)
    for expr, group, ragged in (("tk,eok->to", "e", "k"), ("tk,eok->to", "t", "t"), ("etk,eok->eto", "e", "t"),
                                ("tk,ok->to", "e", "t"), ("tk,eok->to", "o", "t"), ("to,tk->eok", "e", "o")):
        with pytest.raises(ValueError):
            eir.grouped_loops(expr, dict(sizes), group=group, ragged=ragged)
    lp = eir.grouped_loops("tk,eok->to", dict(t=40, k=300, o=200, e=3), group="e", ragged="t", scales=True)
    assert lp["strides_scale_left"] == [0, 3, 0, 1] and lp["strides_scale_right"] == [6, 0, 3, 1]


def test_f8_loops():
    lp = eir.contraction_f8_loops("to,ok->tk", dict(t=40, o=300, k=200))
    assert lp["strides_scale_left"] == [3, 0, 1] and lp["strides_scale_right"] == [0, 1, 2]
    lp = eir.contraction_f8_loops("to,tk->ok", dict(t=300, o=40, k=50), block_right=1)
    assert lp["strides_scale_left"] == [1, 0, 40] and lp["strides_scale_right"] == [0, 1, 50]
    lp = eir.contraction_f8_loops("btk,ok->bto", dict(b=2, t=5, o=40, k=50), bias="o")
    assert lp["strides_scale_left"] == [5, 1, 0, 0] and lp["strides_bias"] == [0, 0, 1, 0]


@pytest.mark.parametrize("make,code", [
    (lambda: eir.QuantF8Plan(2, 8, dtype=eir.FP64), eir.INVALID_DTYPE),
    (lambda: eir.QuantF8Plan(2, 8, dtype_q=eir.INT8), eir.INVALID_DTYPE),
    (lambda: eir.QuantF8Plan(2, 8, dtype_scale=eir.BF16), eir.INVALID_DTYPE),
    (lambda: eir.QuantF8Plan(2, 8, ktype=eir.MADD), eir.INVALID_KTYPE),
    (lambda: eir.QuantF8Plan(2, 8, block=(1, 1)), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(2, 8, block=(1, 64)), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(2, 8, block=(64, 128)), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(-1, 8), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(2, -8), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(2, 8, batch=-1), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(1 << 31, 8), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(1 << 30, 1 << 20), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(1 << 20, 8, batch=1 << 20), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(2, 8, ld_q=7), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(2, 8, ld_values=0), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(1, 8, batch=2, ld_q=7), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(2, 8, ld_in=-8), eir.COMPILATION_FAILED),
    (lambda: eir.QuantF8Plan(2, 8, ld_gate=1 << 50), eir.COMPILATION_FAILED),
])
def test_quant_f8(make, code):
    with pytest.raises(eir.EinsumIrError) as e:
        make()
    assert e.value.code == code


def test_null_pointers():
    lib = eir.hip_lib()
    assert lib.etir_hip_contraction_f8_create(0, None, None, None, None, None, None, None, None, 1, 128, 4, 4, 0, 0, 99, None) != 0
    assert lib.etir_hip_contraction_grouped_create(0, None, None, None, None, None, None, None, 0, 1, 128, 2, 2, 0, 2, None) != 0
    assert lib.etir_hip_contraction_grouped_create(0, None, None, None, None, None, None, None, -1, 1, 128, 2, 2, 0, 2, None) != 0
    assert lib.etir_hip_quant_f8_create(1, 1, 1, 1, 1, 1, 1, 1, 128, 0, 4, 0, 99, None) != 0
    for f, n in ((lib.etir_hip_contraction_f8_execute, 7), (lib.etir_hip_contraction_grouped_execute, 7),
                 (lib.etir_hip_quant_f8_execute, 6)):
        assert f(None, *[None] * n) == eir.CALLED_BEFORE_COMPILATION


@pytest.mark.gpu
def test_plans_that_fit(torch_cuda):
    """The arguments that the refusals change one by one are good ones; null tensors are refused at execution."""
    eir.ContractionF8Plan(**{k: iter(v) if isinstance(v, list) and k != "sizes" else v for k, v in _good().items()})
    for plan, call in ((eir.ContractionF8Plan(**_good()), lambda p: p.execute(None, None, None)),
                       (eir.ContractionF8Plan(**_good()), lambda p: p.execute(64, 64, 64, scale_left=64, bias=64)),
                       (eir.ContractionGroupedPlan(**_grouped()), lambda p: p.execute(64, 64, 64, None)),
                       (eir.QuantF8Plan(2, 8), lambda p: p.execute(64, 64, None))):
        with pytest.raises(eir.EinsumIrError) as e:
            call(plan)
        assert e.value.code == eir.NO_DATA_PTR_PROVIDED


def test_other_plans_refuse_the_types():
    for t in (eir.F8E4M3, eir.F8E5M2, eir.E8M0):
        with pytest.raises(eir.EinsumIrError):
            eir.ContractionPlan([M, N, K], [4, 6, 8], [8, 0, 1], [0, 8, 1], [6, 1, 0], dtype_left=t, dtype_right=t)
        with pytest.raises(eir.EinsumIrError):
            eir.ActQuantPlan(2, 8, dtype=t)
    with pytest.raises(eir.EinsumIrError):
        eir.ContractionPlan([G, M, K], [4, 6, 8], [8, 0, 1], [0, 8, 1], [6, 1, 0])
