"""SiLU of etir_hip_act_quant_* over the whole range of its type.  No counterpart
in the reference.

Oracle: v / (1 + exp(-v)) in float64, as for the other rows rounded to 8 bits: the
kernel's y carries at most 8 roundings (exponential, sum, quotient, product), its
127 / a two more and the product with it one, each 2^-24 relative, so q is within
0.5 + 127 * 12 * 2^-24 < 0.5 + 1e-4 of y * 127 / a, and a scale within 12 * 2^-24 <
2^-20.
"""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu


def _silu(v):
    return v * v.sigmoid()


def _run(torch, gate, x, dtype):
    """q and scale of silu(gate), or of silu(gate) * x, and the rows before rounding in float64."""
    rows, cols = gate.shape
    q, sc = torch.empty((rows, cols), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    plan = eir.ActQuantPlan(rows, cols, dtype=dtype, ktype=eir.SILU)
    plan.execute(gate if x is None else x, q, sc, gate=None if x is None else gate, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    y = _silu(gate.double())
    return q.double(), sc.double(), y if x is None else y * x.double()


def _check(q, sc, y, slack, rel):
    a = y.abs().amax(-1, keepdim=True)
    off = float((q - y * 127 / a).abs().max())
    assert off <= 0.5 + slack, f"q off by {off}"
    want = a.squeeze(-1) / 127
    assert bool(((sc - want).abs() <= want * rel).all()), f"scales {sc.tolist()} for {want.tolist()}"


@pytest.mark.parametrize("dtype", [eir.BF16, eir.FP32])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("cols", [8, 300, 17000])
@pytest.mark.parametrize("far", [100.0, 130.0, 3e4, 2.3e38, 2.4e38, 3e38, 3.38e38])
def test_large_gates(torch_cuda, far, cols, gated, dtype):
    """A finite gate of any size is itself (or nothing, below zero), and its row is finite; gated, a small partner
    brings the product back into range."""
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(cols)
    td = torch.bfloat16 if dtype == eir.BF16 else torch.float32
    gate = torch.randn((3, cols), device="cuda", generator=g)
    gate[0, 3], gate[1, cols - 1], gate[2, 0], gate[2, 5] = far, -far, far, -far
    x = None
    if gated:
        x = torch.randn((3, cols), device="cuda", generator=g)
        x[gate.abs() > 10] = 2.0 / far
        x = x.to(td)
    q, sc, y = _run(torch, gate.to(td), x, dtype)
    _check(q, sc, y, 1e-4, 2.0 ** -20)


@pytest.mark.parametrize("dtype", [eir.BF16, eir.FP32])
@pytest.mark.parametrize("gated", [False, True])
def test_gates_at_the_end_of_exp(torch_cuda, gated, dtype):
    """Down to -88.7, where exp(-v) ends in fp32, no quotient is lost.  From -87.3 on it is below 2^-126 and has down to
    22 bits: 4 units of 2^-24 more than elsewhere, and the scale, as small, as many: q within 0.5 + 127 * 16 * 2^-24 <
    0.5 + 2e-4, a scale within 20 * 2^-24 < 2^-19.  Below, the formula in fp32 gives 0."""
    torch = torch_cuda
    td = torch.bfloat16 if dtype == eir.BF16 else torch.float32
    gate = torch.stack([torch.linspace(-88.5, -85.0, 300), torch.linspace(-88.5, -87.5, 300),
                        torch.full((300,), -88.0), torch.linspace(-95.0, -89.0, 300)]).cuda().to(td)
    x = torch.linspace(1e30, 2e30, 1200, device="cuda").reshape(4, 300).to(td) if gated else None
    q, sc, y = _run(torch, gate, x, dtype)
    _check(q[:3], sc[:3], y[:3], 2e-4, 2.0 ** -19)
    assert bool((q[3] == 0).all()) and float(sc[3]) == 0.0
