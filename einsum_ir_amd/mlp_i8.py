"""A residual multi-layer perceptron answered in 8 bits, from the 8-bit layer
operators (NormQuantPlan, ContractionI8Plan, ActQuantPlan).  No counterpart in
the reference, whose bench_mlp (reference src/bench_mlp.cpp:85-307) runs its
layers in fp32.

    x += delta                      norm_quant: the residual's addition,
    n  = rms_norm(x) * norm                     the norm and its 8-bit rows
    h  = n up^T + up_bias           contraction_i8
    a  = f(h), or f(gate) * h       act_quant, 8-bit rows
    delta = a down^T + down_bias    contraction_i8

for each block, then a last norm and the product with the head's weights.  Every
product reads 8-bit rows with a scale for each token and 8-bit weights with a
scale for each channel; the hidden states between are bf16 or fp32.
"""
from collections import OrderedDict

from . import ActQuantPlan, BF16, ContractionI8Plan, FP32, NormQuantPlan, RELU, contraction_i8_loops


def _torch_stream(torch, stream):
    """A torch stream of a stream, a handle, or None (the current one)."""
    if stream is None:
        return torch.cuda.current_stream()
    if isinstance(stream, int):
        return torch.cuda.ExternalStream(stream) if stream else torch.cuda.default_stream()
    return stream


class LinearI8:
    """Weights [channels, width] laid out once as 8-bit rows with a scale a channel.

    They are laid out on the given stream (None: torch's current one), which waits for the current stream's work
    before, and the current stream for it after: on both the weight may come straight from its making, be dropped
    and the rows be used."""

    def __init__(self, torch, weight, bias=None, stream=None):
        if weight.dim() != 2 or weight.dtype not in (torch.bfloat16, torch.float32) or not weight.is_cuda:
            raise ValueError("weights are [channels, width] tensors of bf16 or fp32 on the GPU")
        if bias is not None and (tuple(bias.shape) != (weight.shape[0],) or bias.dtype != torch.float32
                                 or not bias.is_cuda):
            raise ValueError("a bias holds one fp32 value a channel, on the GPU")
        self.channels, self.width = weight.shape
        plan = ActQuantPlan(self.channels, self.width, dtype=BF16 if weight.dtype == torch.bfloat16 else FP32)
        s, current = _torch_stream(torch, stream), torch.cuda.current_stream()
        # the copies and buffers come from the stream's own pool, as they are used on it
        s.wait_stream(current)
        with torch.cuda.stream(s):
            weight = weight.contiguous()
            self.q = torch.empty(weight.shape, dtype=torch.int8, device=weight.device)
            self.scale = torch.empty(self.channels, device=weight.device)
            self.bias = None if bias is None else bias.contiguous()
            plan.execute(weight, self.q, self.scale, stream=s)
        current.wait_stream(s)

    def plan(self, tokens, dtype):
        """The product of this layer with 8-bit rows of so many tokens."""
        return ContractionI8Plan(**contraction_i8_loops(
            "tk,ok->to", dict(t=tokens, k=self.width, o=self.channels), scale_left="t", scale_right="o",
            bias=None if self.bias is None else "o"), dtype_out=dtype)


class MlpI8:
    """blocks: dicts of the tensors ``norm`` [width], ``up`` [hidden, width] (gated: [2 hidden, width], the gates'
    rows first), ``down`` [width, hidden] and, where there are such, ``up_bias`` and ``down_bias``; ``norm`` [width] and
    ``head`` [classes, width] end the network.  Weights are bf16 or fp32 and rounded to 8 bits here; norms have the
    type of the hidden states (dtype), biases fp32.  ktype: UNDEFINED_KTYPE, RELU or SILU.

    The weights are laid out when the network is made, which waits for it: calls may follow on any stream.  They
    enqueue on the given stream (None: torch's current one when they are made), where x has to be ready.  Each stream
    has buffers of its own, so calls on different streams may overlap: work buffers for the most tokens that it has
    seen, and the logits of a number of tokens, which the next call on the stream with as many writes again.  Plans and
    logits are kept for the last KEPT streams and numbers of tokens.  A call with one of these and no more tokens than
    before allocates nothing and can be captured; what a captured call uses stays as long as this object."""

    KEPT = 64

    def __init__(self, blocks, norm, head, dtype=BF16, ktype=RELU, gated=False, eps=1e-6, stream=None):
        import torch
        if dtype not in (BF16, FP32):
            raise ValueError("hidden states are BF16 or FP32")
        # kernels read the norms through their addresses: all tensors on the head's GPU
        names = ("norm", "up", "down", "up_bias", "down_bias")
        for t in [norm, head] + [b.get(n) for b in blocks for n in names]:
            if t is not None and (not t.is_cuda or t.device != head.device):
                raise ValueError("the network's tensors are on one GPU")
        self._torch, self.dtype, self.ktype, self.gated, self.eps = torch, dtype, ktype, gated, eps
        self.stream = None if stream is None else _torch_stream(torch, stream)
        s, td = self._stream(), self._torch_dtype()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            self.blocks = [dict(norm=b["norm"].to(td).contiguous(),
                                up=LinearI8(torch, b["up"], b.get("up_bias"), s),
                                down=LinearI8(torch, b["down"], b.get("down_bias"), s)) for b in blocks]
            self.norm = norm.to(td).contiguous()
            self.head = LinearI8(torch, head, None, s)
        self.width, self._td, self._device = self.head.width, td, self.head.q.device
        for b in self.blocks:
            hidden = b["up"].channels // (2 if gated else 1)
            if (b["up"].width != self.width or b["down"].channels != self.width or b["down"].width != hidden
                    or b["norm"].numel() != self.width or (gated and b["up"].channels % 2)):
                raise ValueError("the blocks' tensors do not fit each other")
        if self.norm.numel() != self.width:
            raise ValueError("the last norm does not fit the head")
        self._calls = OrderedDict()      # plans and logits by stream and tokens, the last used at the end
        self._work = {}                  # work buffers by stream
        self._captured = {}              # what graphs may write
        s.synchronize()

    def _stream(self):
        return self.stream if self.stream is not None else self._torch.cuda.current_stream()

    def _torch_dtype(self):
        return self._torch.bfloat16 if self.dtype == BF16 else self._torch.float32

    def _work_buffers(self, tokens):
        """What no caller sees, for up to so many tokens."""
        torch, td, dev = self._torch, self._td, self._device
        empty = lambda *shape, **kw: torch.empty(shape, device=dev, **kw)  # noqa: E731
        wide = max([b["down"].width for b in self.blocks], default=0)
        return dict(tokens=tokens, q=empty(tokens, self.width, dtype=torch.int8), q_scale=empty(tokens),
                    a=empty(tokens * wide, dtype=torch.int8), a_scale=empty(tokens),
                    h=empty(tokens * wide * (2 if self.gated else 1), dtype=td),
                    total=empty(tokens, self.width, dtype=td), delta=empty(tokens, self.width, dtype=td))

    def _prepare(self, tokens):
        """Plans and logits of a number of tokens."""
        p = dict(norm=NormQuantPlan(tokens, self.width, dtype=self.dtype, eps=self.eps),
                 logits=self._torch.empty((tokens, self.head.channels), device=self._device, dtype=self._td),
                 head=self.head.plan(tokens, self.dtype), blocks=[])
        for b in self.blocks:
            f, n = b["down"].width, b["up"].channels
            p["blocks"].append((b["up"].plan(tokens, self.dtype),
                                ActQuantPlan(tokens, f, dtype=self.dtype, ktype=self.ktype, ld_in=n, ld_gate=n),
                                b["down"].plan(tokens, self.dtype)))
        return p

    def _of_call(self, s, tokens):
        """Plans and logits, and work buffers of a call on s, the current stream."""
        key = s.cuda_stream, tokens
        p, w = self._calls.get(key), self._work.get(s.cuda_stream)
        if p is None:
            p = self._calls[key] = self._prepare(tokens)
            if len(self._calls) > self.KEPT:
                (gone, _), _ = self._calls.popitem(last=False)
                if all(stream != gone for stream, _ in self._calls):
                    self._work.pop(gone, None)
        else:
            self._calls.move_to_end(key)
        if w is None or w["tokens"] < tokens:
            # the smaller ones go back to the stream's pool, in order with its work
            w = self._work[s.cuda_stream] = self._work_buffers(tokens)
        if self._torch.cuda.is_current_stream_capturing():
            self._captured.update({id(p): p, id(w): w})
        return p, w

    def __call__(self, x):
        """Logits [tokens, classes] of hidden states x [tokens, width]."""
        if (x.dim() != 2 or x.shape[1] != self.width or x.dtype != self._td or x.device != self._device
                or not x.is_contiguous()):
            raise ValueError(f"x is a contiguous [tokens, {self.width}] tensor of {self._td} on the weights' GPU")
        s = self._stream()
        if self.stream is None:
            p, w = self._of_call(s, x.shape[0])
        else:
            with self._torch.cuda.stream(s):      # the buffers come from the pool of the stream that uses them
                p, w = self._of_call(s, x.shape[0])
        state, delta = x, None
        for b, (up, act, down) in zip(self.blocks, p["blocks"]):
            p["norm"].execute(state, w["q"], w["q_scale"], residual=delta, weight=b["norm"],
                              total=None if delta is None else w["total"], stream=s)
            up.execute(w["q"], b["up"].q, w["h"], scale_left=w["q_scale"], scale_right=b["up"].scale,
                       bias=b["up"].bias, stream=s)
            f = b["down"].width
            act.execute(w["h"][f:] if self.gated else w["h"], w["a"], w["a_scale"],
                        gate=w["h"] if self.gated else None, stream=s)
            if delta is not None:
                state = w["total"]
            down.execute(w["a"], b["down"].q, w["delta"], scale_left=w["a_scale"], scale_right=b["down"].scale,
                         bias=b["down"].bias, stream=s)
            delta = w["delta"]
        p["norm"].execute(state, w["q"], w["q_scale"], residual=delta, weight=self.norm, stream=s)
        p["head"].execute(w["q"], self.head.q, p["logits"], scale_left=w["q_scale"], scale_right=self.head.scale, stream=s)
        return p["logits"]

    def num_ops(self, tokens):
        """Operations of the products of one call."""
        per = sum(b[k].channels * b[k].width for b in self.blocks for k in ("up", "down"))
        return 2 * tokens * (per + self.head.channels * self.head.width)
