"""GPU parity of block and grouped products with more batches or groups than
workgroups of 1024 threads can be launched.  No counterpart in the reference."""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu

KERNELS = [None, 0, 1, 3, 7, 13]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("scale", [None, eir.FP32])
def test_batches(torch_cuda, monkeypatch, kernel, scale):
    """Whole numbers: every product and sum is exact."""
    torch = torch_cuda
    if kernel is not None:
        monkeypatch.setenv("ETIR_BLOCK_KERNEL", str(kernel))
    c, m, n, k = 5000000, 2, 2, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    a, b = (torch.randint(-8, 9, (c, 2, k), device="cuda", generator=g).float() for _ in range(2))
    s = 2.0 ** torch.randint(-3, 4, (c, 2, 1), device="cuda", generator=g).float()
    want = torch.stack([torch.stack([(a[:, i] * b[:, j]).sum(-1) for j in range(n)], -1) for i in range(m)], -2)
    if scale is not None:
        want *= s
    f8 = [v.to(torch.float8_e4m3fn) for v in (a, b)]
    del a, b
    plan = eir.ContractionF8Plan(**eir.contraction_f8_loops("cmk,cnk->cmn", dict(c=c, m=m, n=n, k=k), scales=scale is not None),
                                 dtype_out=eir.FP32)
    print(plan.describe(), flush=True)
    y = torch.empty(c, m, n, device="cuda")
    one = torch.ones(c, 1, 1, device="cuda")
    torch.cuda.synchronize()
    plan.execute(*f8, y, scale_left=None if scale is None else s, scale_right=None if scale is None else one)
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("kernel", KERNELS)
def test_groups_of_k(torch_cuda, monkeypatch, kernel):
    """4.5 million groups of 0 to 2 indices of K, whole numbers."""
    torch = torch_cuda
    if kernel is not None:
        monkeypatch.setenv("ETIR_BLOCK_KERNEL", str(kernel))
    e, k, o = 4500000, 8, 3
    g = torch.Generator(device="cuda").manual_seed(2)
    rows = torch.arange(e, device="cuda") % 3
    off = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), rows.cumsum(0)])
    t = int(off[-1])
    x, w = (torch.randint(-8, 9, (t, n), device="cuda", generator=g).float() for n in (o, k))
    # sums of whole numbers from the first row on are exact in 64 bits
    sums = torch.zeros(t + 1, o, k, device="cuda", dtype=torch.float64)
    torch.cumsum((x[:, :, None] * w[:, None, :]).double(), 0, out=sums[1:])
    want = (sums[off[1:]] - sums[off[:-1]]).float()
    plan = eir.ContractionGroupedPlan(**eir.grouped_loops("to,tk->eok", dict(t=t, e=e, o=o, k=k), "e", "t"), dtype_out=eir.FP32)
    print(plan.describe(), flush=True)
    y = torch.empty(e, o, k, device="cuda")
    a, b, at = x.to(torch.bfloat16), w.to(torch.bfloat16), off.int()
    torch.cuda.synchronize()
    plan.execute(a, b, y, at)
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("kernel", KERNELS)
def test_groups_of_rows(torch_cuda, monkeypatch, kernel):
    """20000 groups of 0 to 2 rows, whole numbers."""
    torch = torch_cuda
    if kernel is not None:
        monkeypatch.setenv("ETIR_BLOCK_KERNEL", str(kernel))
    e, k, o = 20000, 16, 5
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = torch.arange(e, device="cuda") % 3
    off = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), rows.cumsum(0)]).int()
    t = int(off[-1])
    of = torch.repeat_interleave(torch.arange(e, device="cuda"), rows)
    x, w = (torch.randint(-8, 9, s, device="cuda", generator=g).to(torch.bfloat16) for s in ((t, k), (e, o, k)))
    want = torch.stack([(x.float() * w[:, j].float()[of]).sum(-1) for j in range(o)], -1)
    plan = eir.ContractionGroupedPlan(**eir.grouped_loops("tk,eok->to", dict(t=t, e=e, o=o, k=k), "e", "t"), dtype_out=eir.FP32)
    print(plan.describe(), flush=True)
    y = torch.empty(t, o, device="cuda")
    torch.cuda.synchronize()
    plan.execute(x, w, y, off)
    torch.cuda.synchronize()
    assert torch.equal(y, want)
