"""The 8-bit layer operators together: a residual MLP answered in 8 bits
(einsum_ir_amd.mlp_i8).  No counterpart in the reference.

Two checks against float64.  The same network with the same roundings (rows and
weights to 8 bits, hidden states to their type): what differs is fp32 against
float64 between the roundings, which moves a value across a rounding now and
then, so a bar of two half units of bf16 (2^-8) or, for fp32 hidden states, of a
few 8-bit steps in many (2e-3).  And the network with nothing rounded to 8 bits:
a row of n normal values is rounded with steps of max / 127, about 0.03 of its
root mean square, an error of 0.9 % for rows and for weights, 1.3 % a product; a
gated activation's row has a longer tail, about 3 %.  Two blocks and a head are
five products: a bar of 0.1.
"""
import ctypes

import pytest

import einsum_ir_amd as eir
from einsum_ir_amd import harness

pytestmark = pytest.mark.gpu


def _net(torch, width, hidden, classes, num, gated, td, seed=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda o, i: (torch.randn(o, i, device="cuda", generator=g) / i ** 0.5).to(td)  # noqa: E731
    vec = lambda n, s: s * torch.randn(n, device="cuda", generator=g)  # noqa: E731
    blocks = []
    for _ in range(num):
        b = dict(norm=1 + vec(width, 0.1), up=rand(hidden * (2 if gated else 1), width), down=rand(width, hidden))
        if bias:
            b.update(up_bias=vec(b["up"].shape[0], 0.1), down_bias=vec(width, 0.1))
        blocks.append(b)
    return blocks, 1 + vec(width, 0.1), rand(classes, width)


def _rounded(torch, v):
    """8-bit rows of float64 values, as the values that they stand for: rint(v * (127 / a)) is defined in fp32, which
    decides ties (bf16 rows have many: every value that is half the largest)."""
    t = v.float()
    a = t.abs().amax(-1, keepdim=True)
    inv = torch.where(a > 0, torch.div(torch.full_like(a, 127.0), a), torch.zeros_like(a))
    return torch.round(t * inv).double() * (a.double() / 127)


def _same_roundings(torch, blocks, norm, head, x, f, gated, td, eps=1e-6):
    to = lambda v: v.to(td).double()  # noqa: E731
    mul = lambda a, w: a @ _rounded(torch, w.double()).T.contiguous()  # noqa: E731
    rms = lambda v, w: _rounded(torch, v * to(w)) / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)  # noqa: E731
    state, delta = x.double(), 0.0
    for b in blocks:
        s = state + delta
        n, state = rms(s, b["norm"]), to(s)
        h = to(mul(n, b["up"]) + (b["up_bias"].double() if "up_bias" in b else 0.0))
        if gated:
            gate, h = h.chunk(2, dim=1)
            a = f(gate) * h
        else:
            a = f(h)
        delta = to(mul(_rounded(torch, a), b["down"]) + (b["down_bias"].double() if "down_bias" in b else 0.0))
    return to(mul(rms(state + delta, norm), head))


@pytest.mark.parametrize("dtype", [eir.BF16, eir.FP32])
@pytest.mark.parametrize("act,gated", [("RELU", False), ("SILU", True)])
@pytest.mark.parametrize("tokens", [1, 5, 33, 300])
@pytest.mark.parametrize("width,hidden,classes", [(256, 512, 10), (500, 777, 33)])
def test_mlp(torch_cuda, tokens, width, hidden, classes, act, gated, dtype):
    torch = torch_cuda
    from einsum_ir_amd.mlp_i8 import MlpI8
    td = torch.bfloat16 if dtype == eir.BF16 else torch.float32
    blocks, norm, head = _net(torch, width, hidden, classes, 2, gated, td, bias=not gated)
    x = torch.randn(tokens, width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(tokens)).to(td)
    net = MlpI8(blocks, norm, head, dtype=dtype, ktype={"RELU": eir.RELU, "SILU": eir.SILU}[act], gated=gated)
    got = net(x).double()
    f = {"RELU": torch.relu, "SILU": torch.nn.functional.silu}[act]
    ref = _same_roundings(torch, blocks, norm, head, x, f, gated, td)
    err = float((got - ref).norm() / ref.norm())
    assert err <= (2.0 ** -8 if dtype == eir.BF16 else 2e-3), err
    if not gated:
        for b in blocks:
            b.pop("up_bias"), b.pop("down_bias")
        net = MlpI8(blocks, norm, head, dtype=dtype, ktype=eir.RELU)
        got = net(x).double()
    full = harness.mlp_float64(torch, blocks, norm.to(td), head, x, act, gated)
    err = float((got - full).norm() / full.norm())
    assert err <= 0.1, err


def test_repeats_bit_for_bit(torch_cuda):
    """Integer sums and maxima have no order: the same call gives the same bits."""
    torch = torch_cuda
    from einsum_ir_amd.mlp_i8 import MlpI8
    blocks, norm, head = _net(torch, 500, 777, 33, 2, True, torch.float32, bias=False)
    net = MlpI8(blocks, norm, head, dtype=eir.FP32, ktype=eir.SILU, gated=True)
    for tokens in (1, 5, 200):
        x = torch.randn(tokens, 500, device="cuda")
        first = net(x).clone()
        for _ in range(10):
            assert torch.equal(net(x), first)


def test_numbers_of_tokens_and_graph(torch_cuda):
    """Calls with other numbers of tokens do not disturb each other, and a captured call replays."""
    torch = torch_cuda
    from einsum_ir_amd.mlp_i8 import MlpI8
    blocks, norm, head = _net(torch, 128, 256, 16, 2, False, torch.bfloat16, seed=3)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    net = MlpI8(blocks, norm, head, stream=s)
    x = {n: torch.randn(n, 128, device="cuda").bfloat16() for n in (1, 7, 64)}
    torch.cuda.synchronize()
    first = {}
    for n in x:
        y = net(x[n])
        s.synchronize()
        first[n] = y.clone()
    for n in reversed(sorted(x)):
        y = net(x[n])
        s.synchronize()
        assert torch.equal(y, first[n])
    lib, graph = eir.hip_lib(), ctypes.c_void_p()
    eir.check(lib.etir_hip_graph_begin(s.cuda_stream))
    y = net(x[7])
    eir.check(lib.etir_hip_graph_end(s.cuda_stream, ctypes.byref(graph)))
    for i in range(3):
        x[7].copy_(torch.randn(7, 128, device="cuda"))
        torch.cuda.synchronize()
        eir.check(lib.etir_hip_graph_launch(graph, s.cuda_stream))
        s.synchronize()
        replayed = y.clone()
        torch.cuda.synchronize()
        again = net(x[7])
        s.synchronize()
        assert torch.equal(replayed, again), i
    eir.check(lib.etir_hip_graph_destroy(graph))


def test_refusals(torch_cuda):
    torch = torch_cuda
    from einsum_ir_amd.mlp_i8 import LinearI8, MlpI8
    blocks, norm, head = _net(torch, 64, 96, 8, 1, False, torch.float32)
    net = MlpI8(blocks, norm, head, dtype=eir.FP32)
    for bad in (torch.zeros(3, 65, device="cuda"), torch.zeros(3, 64, device="cuda").bfloat16(), torch.zeros(3, 64),
                torch.zeros(64, device="cuda"), torch.zeros(64, 3, device="cuda").T):
        with pytest.raises(ValueError):
            net(bad)
    with pytest.raises(ValueError):
        MlpI8(blocks, norm[:10], head)
    with pytest.raises(ValueError):
        MlpI8(blocks, norm, head, gated=True)
    with pytest.raises(ValueError):
        MlpI8(blocks, norm, head, dtype=eir.FP64)
    with pytest.raises(ValueError):
        LinearI8(torch, torch.zeros(4, 4, device="cuda"), bias=torch.zeros(3, device="cuda"))


def test_harness_mlp_i8(torch_cuda, capsys):
    assert harness.main(["mlp_i8", "40,256,512,2,10", "GATED_SILU"]) == 0
    assert "CSV_DATA: einsum_ir,\"mlp_i8\"" in capsys.readouterr().out
    assert harness.main(["mlp_i8", "40,256"]) == 1
