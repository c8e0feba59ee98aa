"""GPU parity of block and grouped products at pointers that are less aligned than
their plans' strides, in sizes that take each of the kernels through registers.  No
counterpart in the reference."""
import pytest

import einsum_ir_amd as eir
import test_gpu_contract_f8 as dense
import test_gpu_grouped as grouped

pytestmark = pytest.mark.gpu

SHIFTS = [(1, 0, 0), (0, 7, 0), (3, 2, 1), (8, 8, 0)]


@pytest.mark.parametrize("shift", SHIFTS)
@pytest.mark.parametrize("expr", ["tk,ok->to", "to,ok->tk", "to,tk->ok"])
@pytest.mark.parametrize("out", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("t,k,o", [(32, 2048, 64), (96, 1024, 96), (256, 512, 512), (1024, 2048, 1024), (2048, 1024, 2048)])
def test_dense(torch_cuda, monkeypatch, t, k, o, expr, out, shift):
    monkeypatch.setenv("ETIR_BLOCK_KERNEL", "7")
    desc = dense.run(torch_cuda, expr, dict(t=t, k=k, o=o), out=out, shift=shift, scale=eir.E8M0 if t == 96 else eir.FP32,
                     block_right=1 if expr == "to,tk->ok" else 128, seed=t)
    assert " tile 64x64 " in desc and " off 16 bytes=staged " in desc


@pytest.mark.parametrize("shift", SHIFTS)
@pytest.mark.parametrize("expr", [grouped.FORWARD, grouped.GRAD_ROWS, grouped.GRAD_WEIGHTS])
@pytest.mark.parametrize("left", [eir.BF16, eir.F8E4M3])
@pytest.mark.parametrize("groups,k,o", [([5, 0, 3, 8], 1024, 64), ([150, 0, 33, 73], 512, 512), ([700, 1, 0, 1347], 1024, 1024)])
def test_groups(torch_cuda, monkeypatch, groups, k, o, expr, left, shift):
    if left != eir.BF16 and expr == grouped.GRAD_WEIGHTS:
        pytest.skip("a ragged K takes bf16")
    monkeypatch.setenv("ETIR_BLOCK_KERNEL", "7")
    desc = grouped.run(torch_cuda, expr, groups, k, o, left=left, shift=shift, seed=sum(groups))
    assert " tile 64x64 " in desc and " off 16 bytes=staged " in desc
