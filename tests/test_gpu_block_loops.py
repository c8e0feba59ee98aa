"""GPU parity of block and grouped products without scales whose sides have
several loops that fuse.  No counterpart in the reference."""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu


def _whole(torch, g, *shape):
    """Whole numbers up to 8: every product and sum is exact."""
    return torch.randint(-8, 9, shape, device="cuda", generator=g).float()


@pytest.mark.parametrize("t,a,b,k", [(1, 3, 5, 16), (40, 3, 50, 144), (300, 2, 130, 131)])
@pytest.mark.parametrize("expr", ["tk,abk->tab", "abk,tk->abt"])
def test_without_scales(torch_cuda, expr, t, a, b, k):
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = _whole(torch, g, t, k), _whole(torch, g, a, b, k)
    want = x @ w.view(a * b, k).t().contiguous()
    loops = eir.contraction_f8_loops(expr, dict(t=t, a=a, b=b, k=k), block_left=128, scales=False)
    plan = eir.ContractionF8Plan(**loops, dtype_out=eir.FP32)
    x8, w8 = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    y = torch.empty(t, a * b, device="cuda") if expr == "tk,abk->tab" else torch.empty(a * b, t, device="cuda")
    torch.cuda.synchronize()
    plan.execute(*((x8, w8) if expr == "tk,abk->tab" else (w8, x8)), y)
    torch.cuda.synchronize()
    assert torch.equal(y, want if expr == "tk,abk->tab" else want.t())


@pytest.mark.parametrize("a,b,k", [(3, 5, 16), (3, 50, 144), (2, 130, 131)])
def test_groups(torch_cuda, a, b, k):
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(2)
    groups = [7, 0, 129, 1]
    t, e = sum(groups), len(groups)
    x, w = _whole(torch, g, t, k), _whole(torch, g, e, a, b, k)
    off = torch.tensor([sum(groups[:i]) for i in range(e + 1)], dtype=torch.int32, device="cuda")
    of = torch.repeat_interleave(torch.arange(e, device="cuda"), torch.tensor(groups, device="cuda"))
    want = torch.stack([x[i] @ w[int(of[i])].view(a * b, k).t().contiguous() for i in range(t)]).view(t, a, b)
    plan = eir.ContractionGroupedPlan(**eir.grouped_loops("tk,eabk->tab", dict(t=t, a=a, b=b, k=k, e=e), "e", "t"), dtype_out=eir.FP32)
    y = torch.empty(t, a, b, device="cuda")
    xb, wb = x.to(torch.bfloat16), w.to(torch.bfloat16)
    torch.cuda.synchronize()
    plan.execute(xb, wb, y, off)
    torch.cuda.synchronize()
    assert torch.equal(y, want)
