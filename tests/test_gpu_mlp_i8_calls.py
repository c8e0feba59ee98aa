"""Arguments, streams and memory of einsum_ir_amd.mlp_i8.MlpI8.  No counterpart in
the reference."""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu


def _net(torch, width=64, hidden=96, classes=8, num=2, seed=0, **kw):
    from einsum_ir_amd.mlp_i8 import MlpI8
    return MlpI8(*_tensors(torch, width, hidden, classes, num, seed), **kw)


def _tensors(torch, width=64, hidden=96, classes=8, num=2, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda o, i: (torch.randn(o, i, device="cuda", generator=g) / i ** 0.5).bfloat16()  # noqa: E731
    ones = lambda: 1 + 0.1 * torch.randn(width, device="cuda", generator=g)  # noqa: E731
    blocks = [dict(norm=ones(), up=rand(hidden, width), down=rand(width, hidden),
                   up_bias=torch.ones(hidden, device="cuda"), down_bias=None) for _ in range(num)]
    return blocks, ones(), rand(classes, width)


@pytest.mark.parametrize("where", ["norm", "block", "head", "up", "bias"])
def test_refuses_tensors_off_the_gpu(torch_cuda, where):
    """Refused when the network is made: its kernels would read them at their host addresses."""
    torch = torch_cuda
    from einsum_ir_amd.mlp_i8 import MlpI8
    blocks, norm, head = _tensors(torch)
    if where == "norm":
        norm = norm.cpu()
    elif where == "head":
        head = head.cpu()
    else:
        name = {"block": "norm", "up": "up", "bias": "up_bias"}[where]
        blocks[1][name] = blocks[1][name].cpu()
    with pytest.raises(ValueError):
        MlpI8(blocks, norm, head)
