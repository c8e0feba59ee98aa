"""Weights of einsum_ir_amd.mlp_i8.LinearI8 laid out on streams.  No counterpart
in the reference.

Oracle: the definition q = rint(w * (127 / a)), scale = a / 127 in fp32, bit for
bit.
"""
import pytest

pytestmark = pytest.mark.gpu


def _rows(torch, w):
    a = w.float().abs().amax(-1, keepdim=True)
    return torch.round(w.float() * torch.div(torch.full_like(a, 127.0), a)).to(torch.int8), torch.div(a, torch.full_like(a, 127.0)).squeeze(-1)


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("stream", ["none", "side", "handle"])
@pytest.mark.parametrize("under", ["default", "other"])
def test_weights_made_just_before(torch_cuda, under, stream, transposed):
    """Weights that the current stream is still making, laid out on it or on another stream, then dropped and their
    memory used again: neither stream is waited for in between."""
    torch = torch_cuda
    from einsum_ir_amd.mlp_i8 import LinearI8
    first = torch.randn((1500, 900), device="cuda").bfloat16()
    busy = torch.randn((4096, 4096), device="cuda")
    want = _rows(torch, first + 1)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.default_stream() if under == "default" else other):
        for _ in range(3):
            for _ in range(5):
                busy = busy @ busy * 1e-4
            w = (first + 1).T.contiguous().T if transposed else first + 1
            layer = LinearI8(torch, w, torch.ones(1500, device="cuda"),
                             stream={"none": None, "side": side, "handle": side.cuda_stream}[stream])
            del w
            again = [torch.full((1500, 900), float(i), device="cuda", dtype=torch.bfloat16) for i in range(4)]
            got = layer.q.clone(), layer.scale.clone()
            del again
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            del layer
