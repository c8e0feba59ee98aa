"""Arguments, streams and memory of einsum_ir_amd.mlp_i8.MlpI8.  No counterpart in
the reference."""
import pytest

import einsum_ir_amd as eir

pytestmark = pytest.mark.gpu

KEPT = 64       # numbers of tokens whose logits a network keeps


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


def _work(torch, n=3):
    """Keeps the current stream busy for some ms."""
    a = torch.full((4096, 4096), 1e-3, device="cuda")
    for _ in range(n):
        a = a @ a
    return a


@pytest.mark.parametrize("made_on", ["default", "side"])
def test_calls_on_two_streams_at_once(torch_cuda, made_on):
    """Calls with as many tokens on two streams, neither waiting for the other: each has buffers of its own."""
    torch = torch_cuda
    x = [torch.randn(40, 256, device="cuda").bfloat16() for _ in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0] if made_on == "side" else torch.cuda.default_stream()):
        net = _net(torch, 256, 4096, 300, 3)
    want = []
    for v in x:
        want.append(net(v).clone())
        torch.cuda.synchronize()
    got, ptrs = [[], []], set()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                y = net(x[i])
                ptrs.add((i, y.data_ptr()))
                got[i].append(y.clone())
    torch.cuda.synchronize()
    assert len(ptrs) == 2 and len({p for _, p in ptrs}) == 2
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i]), i


def test_first_call_beside_work_of_the_current_stream(torch_cuda):
    """A network with a stream of its own takes no memory that work still pending on the current stream writes."""
    torch = torch_cuda
    s = torch.cuda.Stream()
    net = _net(torch, 256, 4096, 300, 2, stream=s)
    x = torch.randn(300, 256, device="cuda").bfloat16()
    torch.cuda.synchronize()
    _work(torch)
    for _ in range(4):      # freed at once, written when the work is done
        for size in (300 * 256, 300 * 4096, 300 * 4096 * 2, 300 * 300 * 2):
            torch.empty(size, dtype=torch.int8, device="cuda").fill_(77)
    y = net(x)
    s.synchronize()
    first = y.clone()
    torch.cuda.synchronize()
    again = net(x)
    s.synchronize()
    assert torch.equal(first, y) and torch.equal(again, first)


@pytest.mark.parametrize("own_stream", [False, True])
def test_network_made_from_tensors_in_the_making(torch_cuda, own_stream):
    """Weights that the current stream is still making, and calls on another stream right after."""
    torch = torch_cuda
    from einsum_ir_amd.mlp_i8 import MlpI8
    blocks, norm, head = _tensors(torch, 256, 1024, 33)
    x = torch.randn(9, 256, device="cuda").bfloat16()
    want = MlpI8(blocks, norm, head)(x).clone()
    torch.cuda.synchronize()
    _work(torch)
    late = [{k: None if v is None else v.clone() for k, v in b.items()} for b in blocks]
    s = torch.cuda.Stream()
    net = MlpI8(late, norm.clone(), head.clone(), stream=s if own_stream else None)
    del late
    with torch.cuda.stream(s):
        y = net(x)
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_memory_of_many_numbers_of_tokens(torch_cuda):
    """Every number of tokens up to 300: the work buffers of the most, and the logits of the last 64 numbers, each block
    of memory rounded up to 512 bytes."""
    torch = torch_cuda
    width, hidden, classes, most = 256, 1024, 33, 300
    net = _net(torch, width, hidden, classes)
    x = torch.randn(most, width, device="cuda").bfloat16()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for tokens in list(range(1, most + 1)) + list(range(most, 0, -1)):
        net(x[:tokens])
    torch.cuda.synchronize()
    per_token = width + 4 + hidden + 4 + 2 * hidden + 2 * 2 * width
    bound = most * per_token + 7 * 512 + KEPT * (most * classes * 2 + 512)
    assert torch.cuda.memory_allocated() - before <= bound


def test_logits_of_other_calls_stay(torch_cuda):
    """Calls with other numbers of tokens, larger ones and more of them than are kept, leave a call's logits alone."""
    torch = torch_cuda
    net = _net(torch, 256, 512, 33)
    x = torch.randn(200, 256, device="cuda").bfloat16()
    y = net(x[:7])
    first = y.clone()
    for tokens in list(range(8, 8 + 2 * KEPT)) + [200, 1]:
        net(x[-tokens:])
    torch.cuda.synchronize()
    assert torch.equal(y, first)
    assert torch.equal(net(x[:7]), first)


def test_graph_outlives_larger_calls(torch_cuda):
    """A captured call replays after calls that need larger buffers and after its numbers of tokens is forgotten."""
    import ctypes
    torch = torch_cuda
    s = torch.cuda.Stream()
    net = _net(torch, 256, 512, 33, stream=s)
    x = torch.randn(7, 256, device="cuda").bfloat16()
    big = torch.randn(300, 256, device="cuda").bfloat16()
    torch.cuda.synchronize()
    net(x)
    s.synchronize()
    lib, graph = eir.hip_lib(), ctypes.c_void_p()
    eir.check(lib.etir_hip_graph_begin(s.cuda_stream))
    y = net(x)
    eir.check(lib.etir_hip_graph_end(s.cuda_stream, ctypes.byref(graph)))
    for i in range(3):
        for tokens in [300] + list(range(100, 101 + KEPT)):
            net(big[:tokens])
        s.synchronize()
        with torch.cuda.stream(s):      # takes what memory is free
            junk = [torch.full((n,), 55, dtype=torch.int8, device="cuda") for n in (7 * 256, 7 * 512, 7 * 1024, 512) * 20]
        x.copy_(torch.randn(7, 256, device="cuda"))
        torch.cuda.synchronize()
        eir.check(lib.etir_hip_graph_launch(graph, s.cuda_stream))
        s.synchronize()
        replayed = y.clone()
        assert all(bool((j == 55).all()) for j in junk), i
        torch.cuda.synchronize()
        again = net(x)
        s.synchronize()
        assert torch.equal(replayed, again), i
        del junk
    eir.check(lib.etir_hip_graph_destroy(graph))
