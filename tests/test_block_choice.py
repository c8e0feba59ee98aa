"""Which kernels block and grouped products get, and what planning refuses,
without a GPU (tests/cpp/block_plan.cpp)."""
import pytest

import block_plans
import einsum_ir_amd as eir

SIZES = [dict(t=8192, k=2048, o=2048, e=16), dict(t=256, k=512, o=512, e=5), dict(t=256, k=64, o=64, e=5),
         dict(t=64, k=128, o=128, e=1), dict(t=4096, k=256, o=4096, e=64)]
TILES = range(5, 11)          # places of the tiles that are loaded into LDS directly (ETIR_BLOCK_KERNEL)


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    return block_plans.build(tmp_path_factory.mktemp("block_plan"))


def _all(program, lines):
    """What every line is described as, unforced and with each of the direct tiles forced."""
    found = block_plans.describe(program, lines)
    for k in TILES:
        found += block_plans.describe(program, lines, env=dict(ETIR_BLOCK_KERNEL=str(k)))
    return found


@pytest.mark.parametrize("expr", ["ot,kt->eok", "ot,tk->eok", "to,kt->eok", "ot,kt->eko"])
def test_a_ragged_k_along_an_operand_is_not_loaded_in_pieces(program, expr):
    """A group's k start at any element and end at any: no kernel that loads 16 bytes of k at a time takes them."""
    lines = [block_plans.grouped_line(eir.grouped_loops(expr, s, "e", "t"), out=out) for s in SIZES for out in (eir.BF16, eir.FP32)]
    for desc in _all(program, lines):
        assert desc.startswith("contraction_grouped ") and " tile " not in desc, desc


def test_a_ragged_k_along_no_operand_is(program):
    lines = [block_plans.grouped_line(eir.grouped_loops("to,tk->eok", s, "e", "t")) for s in SIZES]
    for desc in block_plans.describe(program, lines):
        assert " tile " in desc, desc


@pytest.mark.parametrize("expr", ["kt,eko->to", "ot,eok->tk"])
def test_ragged_rows_along_the_left_operand_are_not_loaded_in_pieces(program, expr):
    """A group's rows start at any row: neither a tile's address nor its extent is a multiple of 4 bytes."""
    lines = [block_plans.grouped_line(eir.grouped_loops(expr, s, "e", "t"), out=out) for s in SIZES for out in (eir.BF16, eir.FP32)]
    for s in SIZES:
        loops = eir.grouped_loops(expr, s, "e", "t", scales=True)
        lines += [block_plans.grouped_line(loops, left=left, scale=scale, out=out) for left in (eir.F8E4M3, eir.F8E5M2)
                  for scale in (eir.FP32, eir.E8M0) for out in (eir.BF16, eir.FP32)]
    for desc in _all(program, lines):
        assert desc.startswith("contraction_grouped ") and " tile " not in desc, desc


def test_ragged_rows_of_k_are(program):
    for expr in ("tk,eok->to", "to,eok->tk"):
        lines = [block_plans.grouped_line(eir.grouped_loops(expr, s, "e", "t")) for s in SIZES]
        for desc in block_plans.describe(program, lines, env=dict(ETIR_BLOCK_KERNEL="7")):
            assert " tile 64x64 " in desc, desc
