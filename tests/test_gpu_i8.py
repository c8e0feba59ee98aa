"""GPU parity of the product of 8-bit integers with scales
(etir_hip_contraction_i8_*).  No counterpart in the reference.

Oracle: the same contraction in float64.  The integer sum is exact, so an
output is off by the roundings of the fp32 epilogue alone: the sum to fp32, two
products and one addition, each within 2^-24 of a value no larger than
|scaled sum| + |bias|, and half a unit of the output's last place.
"""
import numpy as np
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu

GUARD = 64        # elements in front of and behind the output that have to stay


def _out_tolerance(scaled, bias, dtype):
    mag = np.abs(scaled) + np.abs(bias)
    return mag * 5 * 2.0 ** -24 + (mag * 2.0 ** -8 if dtype == eir.BF16 else 0.0) + 1e-37


def _einsum(expr, a, b):
    """np.einsum in float64, as a matrix product where it can be one."""
    return np.einsum(expr, a.astype(np.float64), b.astype(np.float64), optimize=True)


def run(torch, expr, sizes, dtype_out=None, relu=False, scales=True, bias=True, seed=0, outer_left=None,
        outer_right=None, outer_out=None, shift=(0, 0, 0), extreme=False, stream=None, scale_dims=None):
    """One product against float64.  shift: bytes (elements of the output) that
    the operands and the output start after an aligned address."""
    dtype_out = eir.FP32 if dtype_out is None else dtype_out
    rng = np.random.default_rng(seed)
    ins, out = expr.split("->")
    left, right = ins.split(",")
    kdims = [d for d in left if d in right and d not in out]
    sl, sr = (scale_dims or ("".join(d for d in t if d not in kdims) for t in (left, right)))

    def operand(dims, outer, off):
        shape = [(outer or sizes)[d] for d in dims]
        n = int(np.prod(shape))
        full = rng.integers(-128, 128, n).astype(np.int8)
        if extreme:
            full[:] = -128
        # the last element of the tensor ends the allocation: what is read past it is out of bounds
        buf = torch.from_numpy(np.concatenate([np.zeros(off, np.int8), full])).cuda()
        view = full.reshape(shape)[tuple(slice(0, sizes[d]) for d in dims)]
        return buf, buf.data_ptr() + off, view

    l_buf, l_ptr, l_np = operand(left, outer_left, shift[0])
    r_buf, r_ptr, r_np = operand(right, outer_right, shift[1])
    a_np = rng.uniform(0.01, 2.0, [sizes[d] for d in sl]).astype(np.float32)
    b_np = rng.uniform(0.01, 2.0, [sizes[d] for d in sr]).astype(np.float32)
    c_np = rng.standard_normal([sizes[d] for d in sr]).astype(np.float32)
    lp = eir.contraction_i8_loops(expr, sizes, scale_left=sl if scales else None, scale_right=sr if scales else None,
                                  bias=sr if bias else None, sizes_outer_left=outer_left,
                                  sizes_outer_right=outer_right, sizes_outer_out=outer_out)
    plan = eir.ContractionI8Plan(**lp, dtype_out=dtype_out, ktype_last_touch=eir.RELU if relu else eir.UNDEFINED_KTYPE)
    shape_out = [(outer_out or sizes)[d] for d in out]
    n_out = int(np.prod(shape_out))
    item = 2 if dtype_out == eir.BF16 else 4
    t_out = torch.bfloat16 if dtype_out == eir.BF16 else torch.float32
    buf = torch.full((n_out + 2 * GUARD + shift[2],), 7.0, dtype=t_out, device="cuda")
    dev = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    a, b, c = dev(a_np), dev(b_np), dev(c_np)
    torch.cuda.synchronize()
    plan.execute(l_ptr, r_ptr, buf.data_ptr() + (GUARD + shift[2]) * item, scale_left=a if scales else None,
                 scale_right=b if scales else None, bias=c if bias else None, stream=stream)
    torch.cuda.synchronize()
    desc = plan.describe()
    got_all = buf.float().cpu().numpy()
    first = GUARD + shift[2]
    got_full = got_all[first:first + n_out].reshape(shape_out)
    inside = tuple(slice(0, sizes[d]) for d in out)
    got = got_full[inside].astype(np.float64)
    mask = np.ones(shape_out, bool)
    mask[inside] = False
    assert np.all(got_all[:first] == 7.0) and np.all(got_all[first + n_out:] == 7.0), f"{desc}: wrote outside"
    assert np.all(got_full[mask] == 7.0), f"{desc}: wrote between the view's rows"

    ref = _einsum(expr, l_np, r_np)
    spread = lambda x, dims: np.einsum(f"{dims}->{''.join(d for d in out if d in dims)}", x.astype(np.float64)).reshape(  # noqa: E731
        [sizes[d] if d in dims else 1 for d in out])
    if scales:
        ref = ref * spread(a_np, sl) * spread(b_np, sr)
    add = spread(c_np, sr) if bias else np.zeros(())
    full = ref + add
    if relu:
        full = np.maximum(full, 0.0)
    err = np.abs(got - full) - _out_tolerance(ref, add, dtype_out)
    worst = np.unravel_index(np.argmax(err), err.shape) if err.size else ()
    assert err.size == 0 or err.max() <= 0.0, f"{desc}: {worst}: {got[worst]} for {full[worst]}"
    plan.close()
    return desc, got


# one to many of every size, odd ones, and sizes next to the tiles' edges
MKN = [(1, 1, 1), (1, 2048, 2048), (1, 16, 33), (2, 17, 1), (3, 15, 5), (5, 64, 31), (7, 65, 64), (16, 128, 16),
       (17, 127, 15), (24, 4096, 640), (31, 96, 257), (33, 1001, 77), (64, 63, 65), (65, 256, 63), (100, 784, 10),
       (127, 129, 130), (128, 512, 128), (129, 1024, 255), (200, 48, 300), (256, 384, 256), (257, 640, 513),
       (1152, 784, 512), (300, 2048, 1), (1, 2048, 1), (512, 16, 512), (511, 80, 1025), (1025, 208, 300)]


@pytest.mark.parametrize("dtype", [eir.FP32, eir.BF16])
@pytest.mark.parametrize("m,k,n", MKN)
def test_tokens_times_channels(torch_cuda, m, k, n, dtype):
    run(torch_cuda, "tk,ok->to", dict(t=m, k=k, o=n), dtype, seed=m + k + n, relu=(m + n) % 2 == 0)


@pytest.mark.parametrize("expr", ["tk,ok->ot", "tk,ko->to", "kt,ko->to", "kt,ok->ot", "kt,ko->ot", "tk,ko->ot"])
@pytest.mark.parametrize("m,k,n", [(1, 40, 96), (70, 100, 33), (130, 64, 200), (96, 1, 17)])
@pytest.mark.parametrize("dtype", [eir.FP32, eir.BF16])
def test_orders_of_modes(torch_cuda, expr, m, k, n, dtype):
    run(torch_cuda, expr, dict(t=m, k=k, o=n), dtype, seed=m * k)


@pytest.mark.parametrize("expr,sizes", [
    ("btk,ok->bto", dict(b=3, t=37, k=144, o=70)),
    ("abkl,cdkl->abcd", dict(a=4, b=9, c=7, d=5, k=6, l=16)),
    ("abkl,cdlk->acbd", dict(a=4, b=9, c=7, d=5, k=6, l=11)),
    ("zakm,zbkn->zabmn", dict(z=3, a=4, m=5, b=6, n=7, k=33)),
    ("ztk,zok->zto", dict(z=5, t=77, k=1001, o=33)),
    ("tzk,zok->tzo", dict(z=5, t=20, k=128, o=64)),
    ("ztk,zok->toz", dict(z=4, t=20, k=64, o=30)),
    ("ztk,zok->zto", dict(z=9, t=1, k=256, o=300)),
    ("tk,ok->to", dict(t=6, k=0, o=5)),
    ("tk,ok->to", dict(t=0, k=32, o=5)),
    ("ztk,zok->zto", dict(z=0, t=4, k=32, o=5)),
])
@pytest.mark.parametrize("dtype", [eir.FP32, eir.BF16])
def test_modes_and_batches(torch_cuda, expr, sizes, dtype):
    run(torch_cuda, expr, sizes, dtype, seed=3)


@pytest.mark.parametrize("scales,bias,relu", [(False, False, False), (False, True, True), (True, False, True),
                                              (True, True, False)])
@pytest.mark.parametrize("m,k,n", [(1, 2048, 130), (20, 512, 300), (260, 256, 270)])
@pytest.mark.parametrize("expr", ["tk,ok->to", "tk,ok->ot"])
def test_optional_tensors(torch_cuda, expr, m, k, n, scales, bias, relu):
    run(torch_cuda, expr, dict(t=m, k=k, o=n), eir.BF16, scales=scales, bias=bias, relu=relu, seed=5)


@pytest.mark.parametrize("shift", [(1, 0, 0), (0, 3, 0), (16, 16, 1), (4, 8, 2), (7, 9, 3), (0, 0, 1)])
@pytest.mark.parametrize("m,k,n", [(1, 1040, 96), (12, 272, 100), (300, 256, 260)])
@pytest.mark.parametrize("dtype", [eir.FP32, eir.BF16])
def test_any_alignment(torch_cuda, m, k, n, shift, dtype):
    run(torch_cuda, "tk,ok->to", dict(t=m, k=k, o=n), dtype, shift=shift, seed=11)


@pytest.mark.parametrize("m,k,n,pad", [(5, 256, 64, 16), (5, 256, 64, 3), (150, 384, 140, 64), (150, 384, 140, 1),
                                       (40, 100, 36, 4)])
@pytest.mark.parametrize("dtype", [eir.FP32, eir.BF16])
def test_views_of_larger_tensors(torch_cuda, m, k, n, pad, dtype):
    run(torch_cuda, "tk,ok->to", dict(t=m, k=k, o=n), dtype, outer_left=dict(t=m, k=k + pad),
        outer_right=dict(o=n, k=k + 2 * pad), outer_out=dict(t=m, o=n + pad), seed=13)


@pytest.mark.parametrize("m,n", [(1, 20), (40, 70), (256, 256)])
def test_largest_sums(torch_cuda, m, n):
    """Every product 16384: sums up to the end of 32 bits stay exact."""
    run(torch_cuda, "tk,ok->to", dict(t=m, k=131071, o=n), eir.FP32, extreme=True, scales=False, bias=False)


@pytest.mark.parametrize("scale_dims", [("t", ""), ("", "o"), ("", "")])
def test_shared_scales(torch_cuda, scale_dims):
    """One scale for all tokens, or for all channels."""
    torch = torch_cuda
    rng = np.random.default_rng(1)
    m, k, n = 70, 160, 90
    x, w = (rng.integers(-127, 128, s).astype(np.int8) for s in ((m, k), (n, k)))
    sl, sr = scale_dims
    a = rng.uniform(0.5, 1, m if sl else 1).astype(np.float32)
    b = rng.uniform(0.5, 1, n if sr else 1).astype(np.float32)
    lp = eir.contraction_i8_loops("tk,ok->to", dict(t=m, k=k, o=n), scale_left=sl, scale_right=sr)
    plan = eir.ContractionI8Plan(**lp, dtype_out=eir.FP32)
    dev = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    out = torch.empty((m, n), device="cuda")
    t = [dev(v) for v in (x, w, a, b)]
    plan.execute(t[0], t[1], out, scale_left=t[2], scale_right=t[3], stream=torch.cuda.current_stream())
    ref = x.astype(np.float64) @ w.astype(np.float64).T * (a.astype(np.float64)[:, None] * b.astype(np.float64))
    assert np.all(np.abs(out.cpu().numpy() - ref) <= _out_tolerance(ref, 0.0, eir.FP32))


@pytest.mark.parametrize("m,k,n", [(1, 512, 64), (48, 512, 64), (300, 512, 300)])
@pytest.mark.parametrize("relu", [False, True])
def test_nan_scale_marks_its_token(torch_cuda, m, k, n, relu):
    """A row that could not be rounded to 8 bits has a NaN scale: all of its outputs are NaN, no other's."""
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(-127, 128, (m, k), device="cuda", generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), device="cuda", generator=g, dtype=torch.int8)
    a, b = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    x[m // 2] = 0
    a[m // 2] = float("nan")
    lp = eir.contraction_i8_loops("tk,ok->to", dict(t=m, k=k, o=n), scale_left="t", scale_right="o")
    plan = eir.ContractionI8Plan(**lp, dtype_out=eir.BF16, ktype_last_touch=eir.RELU if relu else eir.UNDEFINED_KTYPE)
    out = torch.empty((m, n), device="cuda", dtype=torch.bfloat16)
    plan.execute(x, w, out, scale_left=a, scale_right=b, stream=torch.cuda.current_stream())
    nan = torch.isnan(out)
    assert bool(nan[m // 2].all()) and int(nan.sum()) == n


def test_offsets_past_32_bits(torch_cuda):
    """Rows that lie 2^31 bytes and more apart."""
    torch = torch_cuda
    n, k, step = 3, 64, (1 << 31) + 16
    w = torch.zeros(2 * step + k, dtype=torch.int8, device="cuda")
    x = torch.randint(-127, 128, (5, k), dtype=torch.int8, device="cuda")
    for i in range(n):
        w[i * step:i * step + k] = torch.arange(k, device="cuda", dtype=torch.int8) - 30 * i
    plan = eir.ContractionI8Plan([eir.DIM_M, eir.DIM_N, eir.DIM_K], [5, n, k], [k, 0, 1], [0, step, 1], [n, 1, 0])
    out = torch.empty((5, n), device="cuda")
    plan.execute(x, w, out, stream=torch.cuda.current_stream())
    rows = torch.stack([w[i * step:i * step + k] for i in range(n)]).double()
    assert torch.equal(out.double(), x.double() @ rows.T.contiguous())


def test_runs_on_the_given_stream_and_in_a_graph(torch_cuda):
    torch = torch_cuda
    lib = eir.hip_lib()
    m, k, n = 20, 512, 256
    x = torch.randint(-127, 128, (m, k), dtype=torch.int8, device="cuda")
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda")
    plan = eir.ContractionI8Plan([eir.DIM_M, eir.DIM_N, eir.DIM_K], [m, n, k], [k, 0, 1], [0, k, 1], [n, 1, 0])
    s = torch.cuda.Stream()
    out = torch.zeros((m, n), device="cuda")
    torch.cuda.synchronize()
    ref = lambda: (x.double() @ w.double().T.contiguous()).float()  # noqa: E731
    plan.execute(x, w, out, stream=s)
    s.synchronize()
    assert torch.equal(out, ref())
    import ctypes
    eir.check(lib.etir_hip_graph_begin(s.cuda_stream))
    plan.execute(x, w, out, stream=s)
    graph = ctypes.c_void_p()
    eir.check(lib.etir_hip_graph_end(s.cuda_stream, ctypes.byref(graph)))
    for i in range(3):
        x.copy_(torch.randint(-127, 128, (m, k), dtype=torch.int8, device="cuda"))
        out.zero_()
        torch.cuda.synchronize()
        eir.check(lib.etir_hip_graph_launch(graph, s.cuda_stream))
        s.synchronize()
        assert torch.equal(out, ref()), i
    eir.check(lib.etir_hip_graph_destroy(graph))


def test_refuses_missing_tensors(torch_cuda):
    torch = torch_cuda
    lp = eir.contraction_i8_loops("tk,ok->to", dict(t=4, k=8, o=4), scale_left="t", scale_right="o", bias="o")
    plan = eir.ContractionI8Plan(**lp)
    x = torch.zeros(64, dtype=torch.int8, device="cuda")
    f = torch.zeros(64, device="cuda")
    full = dict(left=x, right=x, out=f, scale_left=f, scale_right=f, bias=f)
    for name in full:
        with pytest.raises(eir.EinsumIrError) as e:
            plan.execute(**dict(full, **{name: None}))
        assert e.value.code == eir.NO_DATA_PTR_PROVIDED
    assert plan.flops == 2 * 4 * 4 * 8
    assert plan.bytes == 4 * 8 + 4 * 8 + 3 * 4 * 4 + 4 * 4 * 4
    other = eir.ActQuantPlan(4, 4)
    with pytest.raises(eir.EinsumIrError) as e:
        eir.check(eir.hip_lib().etir_hip_contraction_i8_execute(other.handle, *[f.data_ptr()] * 6, None))
    assert e.value.code == eir.CALLED_BEFORE_COMPILATION


# a size for each kernel that a product may take, with tiles cut off on both
# sides, one K block and several, K ending inside a block
KERNELS = [("few 4", 1, 4096, 500), ("few 4", 4, 5012, 130), ("few 4", 3, 4607, 301),
           ("few 8 parts", 8, 4096, 500), ("few 8 parts", 5, 5012, 130), ("few 8 parts", 7, 4607, 301),
           ("few 16 parts", 16, 8192, 500), ("few 16 parts", 9, 5012, 130), ("few 16 parts", 13, 4607, 301), ("few 16", 5, 1040, 140), ("few 16", 5, 997, 140), ("few 16", 5, 1044, 140), ("few 32", 29, 2064, 140),
           ("few 32", 29, 515, 140), ("few 32", 29, 1044, 140), ("tile 32x32", 70, 1040, 200),
           ("tile 64x32", 130, 1040, 2050), ("tile 64x64", 70, 96, 200), ("tile 64x64", 600, 2064, 1300), ("tile 128x64", 1400, 2064, 1300),
           ("tile 128x128", 1500, 4112, 2050), ("tile 128x128", 3000, 96, 700), ("tile 256x128", 4072, 2048, 2048),
           ("tile 256x256", 2100, 1040, 4300), ("shift 32x32", 70, 1044, 200), ("shift 32x32", 70, 1041, 140),
           ("shift 64x64", 70, 515, 140), ("shift 64x64", 600, 1044, 1300), ("shift 256x128", 2100, 2061, 4300),
           ("shift 128x128", 1000, 515, 4050), ("shift 256x128", 2000, 1044, 2050), ("shift 128x128", 1000, 1044, 4050)]


@pytest.mark.parametrize("name,m,k,n", KERNELS)
@pytest.mark.parametrize("swap", [False, True])
def test_every_kernel(torch_cuda, name, m, k, n, swap):
    """The size takes the kernel that it is here for, bias along both sides of the tile."""
    desc, _ = run(torch_cuda, "tk,ok->ot" if swap else "tk,ok->to", dict(t=m, k=k, o=n),
                  eir.BF16 if n % 4 else eir.FP32, relu=True, seed=m)
    assert desc.startswith(f"contraction_i8 {name} C="), desc


@pytest.mark.parametrize("k", [1008, 1024, 1040, 2064, 4096, 4111, 6147, 8192, 9001])
@pytest.mark.parametrize("m,n", [(1, 37), (2, 203), (3, 1030), (4, 64), (64, 4), (6, 90), (8, 513), (9, 70), (16, 200)])
def test_parts_of_k(torch_cuda, m, n, k):
    """K in 4 parts of whole and cut pieces, parts with nothing in them."""
    run(torch_cuda, "tk,ok->to", dict(t=m, k=k, o=n), eir.BF16, seed=k)
    run(torch_cuda, "ztk,zok->zto", dict(z=3, t=m, k=k, o=n), eir.FP32, seed=k + 1)


@pytest.mark.parametrize("k", [16, 112, 128, 129, 256, 260, 383, 384, 500, 512, 640, 1024, 1025, 1100])
@pytest.mark.parametrize("m,n", [(200, 70), (900, 1000), (3000, 600), (4000, 2400)])
def test_ends_of_k(torch_cuda, m, n, k):
    """K of fewer blocks than buffers, of as many, and ending at any place of a block."""
    run(torch_cuda, "tk,ok->to", dict(t=m, k=k, o=n), eir.BF16, seed=k)
