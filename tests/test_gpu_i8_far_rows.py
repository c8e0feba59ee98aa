"""The product of 8-bit integers over operands whose rows lie up to 2^31 bytes
from a tile's first one.  No counterpart in the reference.

Without scales the sums are exact below 2^24: equal to those in float64.
"""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu

K, FAR_ROWS = 80, 40


@pytest.mark.parametrize("far_left", [True, False])
@pytest.mark.parametrize("other,step,name", [
    (8, 1 << 26, "few 16"), (40, 1 << 24, "tile 64x64"), (40, (1 << 24) + 1, "shift 64x64"),
    # 32 rows of these strides reach past 2^31 bytes: no tile
    (40, 1 << 26, "general"), (40, (1 << 26) + 4, "general"), (40, (1 << 26) + 1, "general"),
    # the last strides that tiles of 32 rows take
    (40, (1 << 26) - 16, ("tile 32x32", "tile 64x32")), (40, (1 << 26) - 3, "shift 32x32")])
def test_far_rows(torch_cuda, other, step, name, far_left):
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(step % 1000)
    far = torch.zeros((FAR_ROWS - 1) * step + K, dtype=torch.int8, device="cuda")
    rows = far.as_strided((FAR_ROWS, K), (step, 1))
    rows.copy_(torch.randint(-128, 128, (FAR_ROWS, K), device="cuda", generator=g))
    near = torch.randint(-128, 128, (other, K), device="cuda", generator=g, dtype=torch.int8)
    left, right = (rows, near) if far_left else (near, rows)
    m, n = left.shape[0], right.shape[0]
    plan = eir.ContractionI8Plan([eir.DIM_M, eir.DIM_N, eir.DIM_K], [m, n, K], [left.stride(0), 0, 1],
                                 [0, right.stride(0), 1], [n, 1, 0])
    out = torch.full((m + 2, n), 7.0, device="cuda")
    plan.execute(left, right, out[1:], stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    if isinstance(name, tuple):     # far rows on the tile's side of 64, or of 32
        name = name[0 if far_left else 1]
    assert plan.describe().startswith(f"contraction_i8 {name} C="), plan.describe()
    want = left.double() @ right.double().T.contiguous()
    assert torch.equal(out[1:-1].double(), want)
    assert bool((out[0] == 7.0).all()) and bool((out[-1] == 7.0).all())
