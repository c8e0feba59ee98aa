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


def _batches(c, m, n, k, expr="cmk,cnk->cmn", **kinds):
    return block_plans.f8_line(eir.contraction_f8_loops(expr, dict(c=c, m=m, n=n, k=k), **kinds))


@pytest.mark.parametrize("c", [(1 << 22) - 1, 1 << 22, 5000000, 1 << 23, (1 << 24) - 1])
def test_many_batches_have_a_kernel(program, c):
    """More tiles than workgroups of 1024 threads can be launched, none larger that would do with fewer."""
    lines = [_batches(c, 2, 2, 16), _batches(c, 2, 2, 16, scales=False), _batches(c, 1, 1, 8), _batches(c, 33, 64, 40, "ckm,cnk->cnm")]
    for desc in block_plans.describe(program, lines):
        assert desc.startswith("contraction_f8 ") and f" C={c} " in desc, desc


def test_large_outputs_have_a_kernel(program):
    for n in ((1 << 17) - 64, 1 << 17, 1 << 18):
        sizes = dict(m=(1 << 18) - 64, n=n, k=32)
        lines = [block_plans.f8_line(eir.contraction_f8_loops(e, sizes)) for e in ("mk,nk->mn", "km,nk->mn", "mk,nk->nm")]
        # a group more than there are blocks of rows
        lines.append(block_plans.grouped_line(eir.grouped_loops("mk,enk->mn", dict(sizes, e=1, m=sizes["m"] - 64), "e", "m")))
        for desc in block_plans.describe(program, lines):
            assert desc.startswith("contraction_"), desc


def test_many_groups_have_a_kernel(program):
    for e in (1 << 22, 5000000, (1 << 23) - 1):
        line = block_plans.grouped_line(eir.grouped_loops("to,tk->eok", dict(t=1 << 23, e=e, o=3, k=5), "e", "t"))
        desc, = block_plans.describe(program, [line])
        assert desc.startswith("contraction_grouped ") and f" groups={e} " in desc, desc


def test_grids_that_are_too_large_are_refused(program):
    lines = [_batches(1 << 24, 2, 2, 16), _batches((1 << 30) - 1, 1, 1, 1),
             block_plans.f8_line(eir.contraction_f8_loops("mk,nk->mn", dict(m=1 << 18, n=1 << 18, k=32))),
             block_plans.grouped_line(eir.grouped_loops("to,tk->eok", dict(t=1 << 24, e=1 << 24, o=3, k=5), "e", "t")),
             block_plans.grouped_line(eir.grouped_loops("tk,eok->to", dict(t=1 << 18, e=4, o=1 << 18, k=5), "e", "t"))]
    for desc in block_plans.describe(program, lines):
        assert desc.startswith(f"{eir.COMPILATION_FAILED} ") and desc.endswith(": grid too large"), desc


def _groups(e, t, o):
    return block_plans.grouped_line(eir.grouped_loops("tk,eok->to", dict(t=t, e=e, o=o, k=64), "e", "t"))


def test_groups_of_rows_that_take_seconds_to_find_are_refused(program):
    """Every workgroup looks through the offsets: groups times workgroups are bounded, for every kernel."""
    many = [_groups(1 << 22, 1 << 22, 64), _groups(4500000, 4500000, 3), _groups(1 << 18, 1 << 18, 64), _groups(1 << 16, 1 << 27, 1)]
    for desc in _all(program, many) + block_plans.describe(program, many, env=dict(ETIR_BLOCK_KERNEL="1")):
        assert desc.startswith(f"{eir.COMPILATION_FAILED} ") and desc.endswith(": too many groups for as many blocks"), desc
    some = [_groups(1 << 17, 1 << 17, 64), _groups(1 << 16, 1 << 24, 1), _groups(4096, 1 << 29, 1)]
    for desc in block_plans.describe(program, some):
        assert desc.startswith("contraction_grouped "), desc
    # 32 times as many workgroups
    desc, = block_plans.describe(program, some[:1], env=dict(ETIR_BLOCK_KERNEL="1"))
    assert " few 4 " not in desc, desc


def test_a_side_without_scales_may_have_several_loops(program):
    """Blocks of 128 rows are said of a side whose scales are not given; its loops fuse."""
    s = dict(t=40, a=3, b=50, k=144, e=4)
    lines = [block_plans.f8_line(eir.contraction_f8_loops("tk,abk->tab", s, scales=False)),
             block_plans.f8_line(eir.contraction_f8_loops("abk,tk->abt", s, block_left=128, scales=False)),
             block_plans.grouped_line(eir.grouped_loops("tk,eabk->tab", s, "e", "t"))]
    for desc, mn in zip(block_plans.describe(program, lines), ("M=40 N=150", "M=150 N=40", "M=40 N=150")):
        assert desc.startswith("contraction_") and f" {mn} K=144" in desc, desc
    one = eir.contraction_f8_loops("tk,abk->tab", s)
    refused = [block_plans.f8_line(one), block_plans.f8_line(dict(one, strides_scale_left=None)),
               block_plans.f8_line(eir.contraction_f8_loops("abk,tk->abt", s, block_left=128)),
               block_plans.grouped_line(eir.grouped_loops("tk,eabk->tab", s, "e", "t", scales=True), left=eir.F8E4M3)]
    for desc in block_plans.describe(program, refused):
        assert desc.endswith(": blocks of 128 run along one loop"), desc


def test_pointers_off_16_bytes_have_a_kernel_chosen_by_size(program):
    """A plan of direct tiles names the kernel of calls whose pointers are less aligned than its strides: the one through
    registers with the least estimated time, as for strides that are."""
    seen = set()
    for t, k, o in ((32, 4096, 256), (256, 1024, 512), (300, 4096, 1024), (1024, 1024, 1024), (4096, 4096, 4096), (8192, 8192, 8192)):
        s = dict(t=t, k=k, o=o)
        for f, kinds in ((eir.contraction_f8_loops, {}), (eir.grouped_loops, dict(group="e", ragged="t"))):
            expr = "tk,ok->to" if f is eir.contraction_f8_loops else "tk,eok->to"
            line = block_plans.f8_line if f is eir.contraction_f8_loops else block_plans.grouped_line
            loops = f(expr, dict(s, e=4), **kinds)
            # rows one element apart from that: no direct kernel, and hardly any other size
            off = f(expr, dict(s, e=4), sizes_outer_left=dict(t=t, k=k + 1), **kinds)
            forced, = block_plans.describe(program, [line(loops)], env=dict(ETIR_BLOCK_KERNEL="7"))
            assert " tile 64x64 " in forced and " off 16 bytes=staged " in forced, forced
            chosen, other = block_plans.describe(program, [line(loops), line(off)])
            assert (" off 16 bytes=" in chosen) == (" tile " in chosen), chosen
            assert " tile " not in other and " off 16 bytes=" not in other, other
            name = forced.split(" off 16 bytes=")[1]
            if " staged " in other:
                assert f" {name} " in other, (forced, other)
            seen.add(name)
    assert len(seen) > 1, seen
