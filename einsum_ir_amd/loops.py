"""Lowering of einsum strings to the loop IR accepted by the C ABI.

Python restatement (for Python callers of the C ABI) of what the reference's
operator classes do before handing loops to a backend:

* dimension typing -- BinaryContraction::dim_types / dim_types_ids
  (reference src/backend/BinaryContraction.cpp:7-221): C = left & right & out,
  M = left & out, N = right & out, K = left & right, I = left only,
  J = right only;
* row-major strides keyed by dimension, 0 for dims of size < 2 --
  BinaryContraction::strides (BinaryContraction.cpp:223-248);
* loop order C, M, N (output order) then K (left order), one loop per
  dimension with the strides of every tensor -- BinaryContractionTpp::compile
  (reference src/backend/BinaryContractionTpp.cpp:46-66);
* the unary path's sizes and input strides in output order --
  Unary::compile_base (reference src/backend/Unary.cpp:82-113).

The C++ classes in libeinsum_ir.so do the same for C++ callers.
"""
from ._lib import DIM_C, DIM_M, DIM_N, DIM_K, DIM_I, DIM_J, DIM_G


def _split(expr):
    expr = expr.replace(" ", "")
    lhs, out = expr.split("->")
    ins = lhs.split(",")
    return ins, out


def dim_types(left, right, out):
    """Dimension types of the output, left and right tensors (lists of names)."""
    def typ(d, in_l, in_r, in_o):
        if in_l and in_r and in_o:
            return DIM_C
        if in_l and in_o:
            return DIM_M
        if in_r and in_o:
            return DIM_N
        if in_l and in_r:
            return DIM_K
        if in_l:
            return DIM_I
        if in_r:
            return DIM_J
        return None
    sl, sr, so = set(left), set(right), set(out)
    return {d: typ(d, d in sl, d in sr, d in so) for d in list(left) + list(right) + list(out)}


def row_major_strides(dims, sizes):
    """Row-major element strides of a tensor; dims of size < 2 get stride 0."""
    strides = {}
    acc = 1
    for d in reversed(list(dims)):
        strides[d] = acc if sizes[d] >= 2 else 0
        acc *= sizes[d]
    return strides


def binary_loops(expr, sizes, sizes_outer_left=None, sizes_outer_right=None,
                 sizes_outer_out=None, sizes_outer_aux=None):
    """Loop IR of a binary contraction ``"ab,bc->ac"``.

    sizes maps dimension names to (inner) sizes; the optional outer-size maps
    describe tensors that are views into larger buffers (the reference's
    outer sizes).  Returns a dict with dim_types, sizes and the four stride
    lists, in the reference's loop order (C, M, N, K)."""
    (left, right), out = _split(expr)
    types = dim_types(left, right, out)
    sl = row_major_strides(left, sizes_outer_left or sizes)
    sr = row_major_strides(right, sizes_outer_right or sizes)
    so = row_major_strides(out, sizes_outer_out or sizes)
    sa = row_major_strides(out, sizes_outer_aux) if sizes_outer_aux else so
    order = ([d for d in out if types[d] == DIM_C] + [d for d in out if types[d] == DIM_M]
             + [d for d in out if types[d] == DIM_N] + [d for d in left if types[d] == DIM_K])
    return {
        "dims": order,
        "dim_types": [types[d] for d in order],
        "sizes": [sizes[d] for d in order],
        "strides_left": [sl.get(d, 0) for d in order],
        "strides_right": [sr.get(d, 0) for d in order],
        "strides_out": [so.get(d, 0) for d in order],
        "strides_out_aux": [sa.get(d, 0) for d in order],
    }


def contraction_i8_loops(expr, sizes, scale_left=None, scale_right=None, bias=None, sizes_outer_left=None,
                         sizes_outer_right=None, sizes_outer_out=None):
    """Arguments of ContractionI8Plan for an einsum string: the loops of
    binary_loops with the row-major strides of the scales and the bias, whose
    dimensions are given as strings (``scale_left="bt"``; None: not there)."""
    lp = binary_loops(expr, sizes, sizes_outer_left, sizes_outer_right, sizes_outer_out)
    (left, right), _ = _split(expr)
    for name, dims, of in (("scale_left", scale_left, left), ("scale_right", scale_right, right), ("bias", bias, right)):
        if dims is not None and not set(dims) <= set(of):
            raise ValueError(f"{name} has dimensions that its operand lacks: {dims!r} of {of!r}")

    def strides(dims):
        if dims is None:
            return None
        s = row_major_strides(dims, sizes)
        return [s.get(d, 0) for d in lp["dims"]]
    return {k: lp[k] for k in ("dim_types", "sizes", "strides_left", "strides_right", "strides_out")} | {
        "strides_scale_left": strides(scale_left), "strides_scale_right": strides(scale_right),
        "strides_bias": strides(bias)}


SCALE_BLOCK = 128     # contracted indices that share a scale


def _scale_strides(dims, lp, contracted, rows, block, sizes):
    """Strides, from block to block, of a row-major scale tensor with an operand's dimensions: blocks of 128 along the
    contracted one and of `block` along those of `rows`."""
    of = {d: SCALE_BLOCK if d == contracted else block if d in rows else 1 for d in dims}
    s = row_major_strides(dims, {d: -(-sizes[d] // of[d]) for d in dims})
    return [s.get(d, 0) for d in lp["dims"]]


def _f8_scales(left, right, out, lp, sizes, block_left, block_right):
    """Scale arguments; only dimensions that an operand shares with the output have blocks of rows."""
    contracted = [d for d in left if d in right and d not in out]
    if len(contracted) != 1:
        raise ValueError("blocks of 128 run along one contracted dimension")
    return {"strides_scale_left": _scale_strides(left, lp, contracted[0], [d for d in left if d in out and d not in right],
                                                 block_left, sizes),
            "strides_scale_right": _scale_strides(right, lp, contracted[0], [d for d in right if d in out and d not in left],
                                                  block_right, sizes),
            "block_left": block_left, "block_right": block_right}


def contraction_f8_loops(expr, sizes, block_left=1, block_right=128, scales=True, bias=None, sizes_outer_left=None,
                         sizes_outer_right=None, sizes_outer_out=None):
    """Arguments of ContractionF8Plan for an einsum string: the loops of
    binary_loops with the strides of row-major scale tensors, whose dimensions are
    their operand's, one entry for 128 contracted indices and for block_left
    (block_right) others, and of the bias, whose dimensions are given as a string.
    scales=False: none."""
    lp = binary_loops(expr, sizes, sizes_outer_left, sizes_outer_right, sizes_outer_out)
    (left, right), out = _split(expr)
    if bias is not None and not set(bias) <= set(right):
        raise ValueError(f"bias has dimensions that its operand lacks: {bias!r} of {right!r}")
    found = {k: lp[k] for k in ("dim_types", "sizes", "strides_left", "strides_right", "strides_out")}
    if scales:
        found.update(_f8_scales(left, right, out, lp, sizes, block_left, block_right))
    strides = None if bias is None else row_major_strides(bias, sizes)
    return found | {"strides_bias": None if bias is None else [strides.get(d, 0) for d in lp["dims"]]}


def grouped_loops(expr, sizes, group, ragged, scales=False, block_left=1, block_right=128, sizes_outer_left=None,
                  sizes_outer_right=None, sizes_outer_out=None):
    """Arguments of ContractionGroupedPlan for an einsum string with a group and a
    ragged dimension: ``"tk,eok->to"`` (experts' products), ``"to,eok->tk"`` (the
    gradient of their rows) or ``"to,tk->eok"`` (of their weights) with
    group="e", ragged="t".  scales: with the strides of the scale tensors, as in
    contraction_f8_loops."""
    (left, right), out = _split(expr)
    if ragged not in left or (ragged in right) == (ragged in out):
        raise ValueError("the ragged dimension is left's, and either right's or the output's")
    if group in left or (group in right) == (group in out) or (group in out) != (ragged in right):
        raise ValueError("groups are of the right operand where the ragged dimension is the output's, else of the output")
    types = dim_types(left.replace(group, ""), right.replace(group, ""), out.replace(group, ""))
    inner = ([d for d in out if types.get(d) == DIM_M] + [d for d in out if types.get(d) == DIM_N]
             + [d for d in left if types.get(d) == DIM_K])
    if set(inner) | {group} != set(left + right + out):
        raise ValueError("beside the groups, dimensions are shared by two of the three tensors")
    sl = row_major_strides(left, sizes_outer_left or sizes)
    sr = row_major_strides(right, sizes_outer_right or sizes)
    so = row_major_strides(out, sizes_outer_out or sizes)
    dims = [group] + inner
    lp = {"dims": dims}
    found = {"dim_types": [DIM_G] + [types[d] for d in inner], "sizes": [sizes[d] for d in dims],
             "strides_left": [sl.get(d, 0) for d in dims], "strides_right": [sr.get(d, 0) for d in dims],
             "strides_out": [so.get(d, 0) for d in dims], "ragged": dims.index(ragged)}
    if scales:
        found.update(_f8_scales(left, right, out, lp, sizes, block_left, block_right))
    return found


def unary_dims(expr, sizes):
    """Sizes, input strides (reordered to output order) and output strides of a
    permutation ``"abcd->dbca"`` with row-major tensors."""
    (inp,), out = _split(expr)
    # Unary::strides uses the plain row-major product (no zero for size 1)
    si, acc = {}, 1
    for d in reversed(inp):
        si[d] = acc
        acc *= sizes[d]
    so, acc = {}, 1
    for d in reversed(out):
        so[d] = acc
        acc *= sizes[d]
    return {
        "dims": list(out),
        "sizes": [sizes[d] for d in out],
        "strides_in": [si[d] for d in out],
        "strides_out": [so[d] for d in out],
    }
