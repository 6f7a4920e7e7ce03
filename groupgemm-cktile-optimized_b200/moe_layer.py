"""A mixture-of-experts layer on the B200 backend: the router, token movement and the grouped GEMM
of one layer together, in training and in serving.

    y_t = sum_j weights_tj * (W[ids_tj] @ x_t)        W [experts, n, k], x [tokens, k], y [tokens, n]

TrainingLayer: route -> dispatch -> grouped GEMM -> combine, and back: combine's gradient -> dgrad
and wgrad -> dispatch's gradient, router's gradient. The grouped GEMM takes its group sizes on the host
(they size its tile schedule), so a step reads the router's counts back once.

ServingLayer: route -> 4-bit products (which gather the tokens themselves) -> combine. Nothing comes
back to the host and nothing is allocated, so a step can be captured in a CUDA graph.

quantize_w4() makes the 4-bit weights that gg_prepare_w4 reads from 16- or 32-bit ones.

    python moe_layer.py        one training step and one serving step on the GPU, checked against plain torch
"""
from __future__ import annotations

import importlib.util
import os
import sys
import weakref

import torch

HERE = os.path.dirname(os.path.abspath(__file__))


def load_package():
    """The binding (the directory's name is not a Python identifier)."""
    if "gg_b200" not in sys.modules:
        spec = importlib.util.spec_from_file_location("gg_b200", os.path.join(HERE, "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["gg_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["gg_b200"]


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ready(why: str) -> None:
    if why:
        raise ValueError(why)


def _ptr(t) -> int:
    """Address of a tensor as the kernels read it: row by row without gaps, on the current device."""
    if t is None:
        return 0
    if not t.is_contiguous():
        raise ValueError(f"a tensor of shape {tuple(t.shape)} and strides {t.stride()} is not contiguous")
    if not t.is_cuda or t.device.index != torch.cuda.current_device():
        raise ValueError(f"a tensor of shape {tuple(t.shape)} is on {t.device}, not on the current CUDA device")
    return t.data_ptr()


def _check(name: str, t, shape: tuple, *dtypes: torch.dtype):
    """t, if it has this shape and one of these types: the kernels see an address only."""
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != shape or t.dtype not in dtypes:
        what = f"{t.dtype} {list(t.shape)}" if isinstance(t, torch.Tensor) else repr(t)
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)} {list(shape)}, not {what}")
    return t


HALF = (torch.bfloat16, torch.float16)
LOGITS = (torch.float32,) + HALF
BYTES = (torch.uint8, torch.int8)
MASK = BYTES + (torch.bool,)  # a byte a token


def _dtype(gg, dtype: torch.dtype) -> int:
    return {torch.bfloat16: gg.BF16, torch.float16: gg.FP16, torch.float32: gg.F32}[dtype]


def quantize_w4(w: torch.Tensor, group: int, symmetric: bool = True):
    """w [experts, n, k] -> (qweight [experts, n, k / 2] uint8, scales [experts, n, ceil(k / group)] in w's type
    (bf16 for fp32), zeros uint8 of the same shape, or None when symmetric). Rounds to the nearest of the 16 values
    that a group's scale gives: (q - 8) scale, or (q - zero) scale with the zero point of the group's range."""
    e, n, k = w.shape
    groups = -(-k // group)
    x = torch.nn.functional.pad(w.float(), (0, groups * group - k)).view(e, n, groups, group)
    dtype = w.dtype if w.dtype in HALF else torch.bfloat16
    if symmetric:
        scales = (x.abs().amax(3) / 7).to(dtype)
    else:
        low, high = x.amin(3).clamp(max=0), x.amax(3).clamp(min=0)
        scales = ((high - low) / 15).to(dtype)
    scales = torch.where(scales == 0, 1, scales)  # a group of zeros, or one below the type's range
    zero = torch.full_like(scales, 8, dtype=torch.float32) if symmetric else (-low / scales.float()).round().clamp(0, 15)
    q = ((x / scales.float()[..., None]).round() + zero[..., None]).clamp(0, 15).to(torch.uint8)
    q = q.view(e, n, groups * group)[:, :, :k]
    packed = (q[:, :, 0::2] | (q[:, :, 1::2] << 4)).contiguous()
    return packed, scales.contiguous(), None if symmetric else zero.to(torch.uint8).contiguous()


class Router:
    """The router's handle and outputs (gg_prepare_route) for a buffer of logits [tokens, experts] and one of mask bytes [tokens], which
    run() reads anew each time and which have to be contiguous for that. `backends`: the handles of the run and of the gradient."""

    def __init__(self, logits: torch.Tensor, top_k: int, mask: torch.Tensor | None = None, normalize: bool = True, losses: bool = True,
                 backends=None):
        gg = load_package()
        t, e = logits.shape
        _check("logits", logits, (t, e), *LOGITS)
        if mask is not None:
            _check("mask", mask, (t,), *MASK)
        new = lambda *shape, dtype=torch.int32: torch.empty(*shape, dtype=dtype, device=logits.device)  # noqa: E731
        f32 = torch.float32
        self.logits, self.mask, self.top_k, self.normalize = logits, mask, top_k, normalize
        self.ids, self.dest, self.src = new(t, top_k), new(t, top_k), new(t * top_k)
        self.counts, self.offsets, self.live = new(e), new(e + 1), new(1)
        self.weights, self.lse = new(t, top_k, dtype=f32), new(t, dtype=f32)
        self.prob, self.losses = (new(e, dtype=f32), new(2, dtype=f32)) if losses else (None, None)
        self.backend, self.grad_backend = backends or (gg.make_b200_backend(), gg.make_b200_backend())
        self._prepare()

    def _prepare(self) -> None:
        logits = self.logits
        _ready(self.backend.prepare_route(
            _dtype(load_package(), logits.dtype), *logits.shape, self.top_k, _ptr(logits), _ptr(self.ids), _ptr(self.weights), _ptr(self.counts),
            _ptr(self.offsets), _ptr(self.live), _ptr(self.dest), _ptr(self.src), lse_ptr=_ptr(self.lse), prob_ptr=_ptr(self.prob),
            losses_ptr=_ptr(self.losses), mask_ptr=_ptr(self.mask), normalize=self.normalize, stream=_stream()))
        self.backend.router = weakref.ref(self)

    def run(self) -> None:
        if self.backend.router() is not self:  # a handle that a later router was given too
            self._prepare()
        self.backend.run(_stream())

    def grad(self, dweights: torch.Tensor | None, dlosses: torch.Tensor | None) -> torch.Tensor:
        """d logits of the last run, for gradients of the weights [tokens, top_k] and of the two losses [2]."""
        gg = load_package()
        t, e = self.logits.shape
        if dweights is not None:
            dweights = _check("dweights", dweights, (t, self.top_k), torch.float32).contiguous()
        if dlosses is not None:
            dlosses = _check("dlosses", dlosses, (2,), torch.float32).contiguous()
        dlogits = torch.empty_like(self.logits)
        b = self.grad_backend
        _ready(b.prepare_route_grad(
            _dtype(gg, self.logits.dtype), t, e, self.top_k, _ptr(self.logits), _ptr(dlogits), _ptr(self.ids), _ptr(self.lse),
            _ptr(self.counts), _ptr(self.live), dweights_ptr=_ptr(dweights), dlosses_ptr=_ptr(dlosses), mask_ptr=_ptr(self.mask),
            normalize=self.normalize, stream=_stream()))
        b.run(_stream())
        return dlogits


class TrainingLayer:
    """One layer's forward and backward pass over 16-bit experts `w` [experts, n, k], which have to be contiguous. The tensors of a step
    may have any strides (an expanded gradient, a transposed view): what is not contiguous is copied first.

    Each operator has a handle of its own, so that what its kernels report (an index out of range, a wait that gave up) stays there for
    check(), until the same operator is prepared again: the forward's until the next forward, the backward's until the next backward. check()
    waits for the GPU and takes about 130 us, a third of a small step, so it is the caller's to call."""

    OPERATORS = ("route", "dispatch", "products", "combine", "combine_grad", "dgrad", "wgrad", "dispatch_grad", "route_grad")

    def __init__(self, w: torch.Tensor, top_k: int, normalize: bool = True):
        self.gg = load_package()
        e, n, k = w.shape
        if not _check("w", w, (e, n, k), *HALF).is_contiguous():
            raise ValueError("w must be contiguous")
        self.w, self.top_k, self.normalize = w, top_k, normalize
        self.backends = {name: self.gg.make_b200_backend() for name in self.OPERATORS}

    def check(self) -> None:
        """Waits for the current stream and raises if a kernel of the last forward or backward reported an error."""
        s = _stream()
        bad = [f"{name}: {b.last_error()}" for name, b in self.backends.items() if b.device_status(s)]
        if bad:
            raise RuntimeError("; ".join(bad))

    def _run(self, name: str, prepare: str, *args, **kw) -> None:
        b, s = self.backends[name], _stream()
        _ready(getattr(b, prepare)(*args, stream=s, **kw))
        b.run(s)

    def forward(self, x: torch.Tensor, logits: torch.Tensor, mask: torch.Tensor | None = None):
        """x [tokens, k] in w's type, logits [tokens, experts] -> (y [tokens, n], losses [2]: balance and z)."""
        (e, n, k), t = self.w.shape, x.shape[0]
        x = _check("x", x, (t, k), self.w.dtype).contiguous()
        logits = _check("logits", logits, (t, e), *LOGITS).contiguous()
        if mask is not None:
            mask = _check("mask", mask, (t,), *MASK).contiguous()
        self.router = r = Router(logits, self.top_k, mask, self.normalize, backends=(self.backends["route"], self.backends["route_grad"]))
        r.run()
        dt = _dtype(self.gg, x.dtype)
        self.x_rows = torch.empty(t * self.top_k, k, dtype=x.dtype, device=x.device)
        self.rows = torch.empty(t * self.top_k, n, dtype=x.dtype, device=x.device)
        y = torch.empty(t, n, dtype=x.dtype, device=x.device)
        self._run("dispatch", "prepare_dispatch", dt, t, self.top_k, e, k, _ptr(x), _ptr(r.dest), _ptr(r.offsets), _ptr(self.x_rows))
        self.group_m = r.counts.tolist()
        self._run("products", "prepare", dt, self.group_m, n, k, _ptr(self.x_rows), _ptr(self.w), _ptr(self.rows))
        self._run("combine", "prepare_combine", dt, t, self.top_k, e, n, _ptr(self.rows), _ptr(r.dest), _ptr(y), weights_ptr=_ptr(r.weights))
        return y, r.losses

    def backward(self, dy: torch.Tensor, dlosses: torch.Tensor | None = None):
        """(dx, dw, dlogits) of the last forward, for dy [tokens, n] in w's type and the losses' gradients [2] in fp32."""
        (e, n, k), (t, _) = self.w.shape, self.router.logits.shape
        dy = _check("dy", dy, (t, n), self.w.dtype).contiguous()
        if dlosses is not None:
            dlosses = _check("dlosses", dlosses, (2,), torch.float32).contiguous()
        r, dt = self.router, _dtype(self.gg, dy.dtype)
        drows = torch.empty_like(self.rows)
        dweights = torch.empty_like(r.weights)
        dx_rows, dx, dw = torch.empty_like(self.x_rows), torch.empty(t, k, dtype=dy.dtype, device=dy.device), torch.empty_like(self.w)
        self._run("combine_grad", "prepare_combine_grad", dt, t, self.top_k, e, n, _ptr(dy), _ptr(self.rows), _ptr(r.dest), _ptr(r.offsets),
                  _ptr(drows), weights_ptr=_ptr(r.weights), dweights_ptr=_ptr(dweights))
        self._run("dgrad", "prepare_grad", self.gg.OP_DGRAD, dt, self.group_m, n, k, dy_ptr=_ptr(drows), w_ptr=_ptr(self.w), dx_ptr=_ptr(dx_rows))
        self._run("wgrad", "prepare_grad", self.gg.OP_WGRAD, dt, self.group_m, n, k, dy_ptr=_ptr(drows), x_ptr=_ptr(self.x_rows), dw_ptr=_ptr(dw))
        self._run("dispatch_grad", "prepare_combine", dt, t, self.top_k, e, k, _ptr(dx_rows), _ptr(r.dest), _ptr(dx))
        return dx, dw, r.grad(dweights, dlosses)


class ServingLayer:
    """One layer for up to a fixed number of tokens a step, over 4-bit experts; all buffers and handles are made here."""

    def __init__(self, qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, group: int, tokens: int, top_k: int,
                 logits_dtype: torch.dtype = torch.float32, normalize: bool = True):
        gg = load_package()
        e, n, half = qweight.shape
        k, dev, dtype = 2 * half, qweight.device, scales.dtype
        _check("qweight", qweight, (e, n, half), *BYTES)
        _check("scales", scales, (e, n, -(-k // group)), *HALF)
        if zeros is not None:
            _check("zeros", zeros, (e, n, -(-k // group)), *BYTES)
        self.keep = (qweight, scales, zeros)
        self.x = torch.zeros(tokens, k, dtype=dtype, device=dev)
        self.mask = torch.zeros(tokens, dtype=torch.uint8, device=dev)  # places without a token
        self.logits = torch.zeros(tokens, e, dtype=logits_dtype, device=dev)
        self.rows = torch.empty(tokens * top_k, n, dtype=dtype, device=dev)
        self.y = torch.empty(tokens, n, dtype=dtype, device=dev)
        self.router = r = Router(self.logits, top_k, self.mask, normalize, losses=False)
        dt, s = _dtype(gg, dtype), _stream()
        self.products, self.combine = gg.make_b200_backend(), gg.make_b200_backend()
        _ready(self.products.prepare_w4(dt, e, n, k, group, tokens * top_k, _ptr(self.x), _ptr(qweight), _ptr(scales), _ptr(r.offsets),
                                        _ptr(self.rows), zeros_ptr=_ptr(zeros), src_ptr=_ptr(r.src), tokens=tokens, top_k=top_k, stream=s))
        _ready(self.combine.prepare_combine(dt, tokens, top_k, e, n, _ptr(self.rows), _ptr(r.dest), _ptr(self.y),
                                            weights_ptr=_ptr(r.weights), stream=s))

    def run(self) -> torch.Tensor:
        """One step on what x, mask and logits hold; y [tokens, n], zero where mask is."""
        s = _stream()
        self.router.backend.run(s)
        self.products.run(s)
        self.combine.run(s)
        return self.y


def plain_layer(x, w, logits, top_k, mask=None):
    """The layer in elementary operations with autograd: (y, losses) in x's type and fp32, for normalised weights."""
    t, e = logits.shape
    live = torch.ones(t, dtype=torch.bool, device=x.device) if mask is None else mask != 0
    l = logits.float()
    top, ids = torch.topk(l, top_k, dim=1)
    weights = torch.softmax(top, dim=1) * live[:, None]
    every = torch.einsum("tk,enk->ten", x, w)
    y = (every.gather(1, ids[..., None].expand(-1, -1, w.shape[1])) * weights[..., None]).sum(1)
    p = torch.softmax(l, dim=1)[live]
    counts = torch.bincount(ids[live].flatten(), minlength=e).float()
    n = live.sum()
    losses = torch.stack([e * (counts / (top_k * n) * p.mean(0)).sum(), torch.logsumexp(l[live], 1).square().mean()])
    return y, losses


def main() -> None:
    torch.manual_seed(0)
    tokens, e, n, k, top_k, group = 200, 8, 512, 384, 2, 128
    x = torch.randn(tokens, k, device="cuda").bfloat16()
    w = (torch.randn(e, n, k, device="cuda") / k ** 0.5).bfloat16()
    logits = torch.randn(tokens, e, device="cuda")
    mask = (torch.rand(tokens, device="cuda") > 0.1).to(torch.uint8)
    dy = torch.randn(tokens, n, device="cuda").bfloat16()
    dlosses = torch.tensor([0.01, 0.001], device="cuda")

    layer = TrainingLayer(w, top_k)
    y, losses = layer.forward(x, logits, mask)
    dx, dw, dlogits = layer.backward(dy, dlosses)
    layer.check()
    leaves = [v.double().requires_grad_() for v in (x, w)] + [logits.double().requires_grad_()]
    py, pl = plain_layer(leaves[0], leaves[1], leaves[2], top_k, mask)
    (torch.sum(py * dy.double()) + torch.sum(pl * dlosses.double())).backward()
    def far(a, b):
        d = ((a.double() - b.double()).norm() / b.double().norm()).item()
        assert d < 2e-2, d  # five roundings to bf16
        return d

    print("training: y %.2g losses %.2g dx %.2g dw %.2g dlogits %.2g (relative to 64 bits)" % (
        far(y, py), far(losses, pl), far(dx, leaves[0].grad), far(dw, leaves[1].grad), far(dlogits, leaves[2].grad)))

    q, scales, zeros = quantize_w4(w, group)
    serve = ServingLayer(q, scales, zeros, group, 16, top_k)
    serve.x.copy_(x[:16])
    serve.logits.copy_(logits[:16])
    serve.mask.fill_(1)
    nibbles = torch.stack([q & 15, q >> 4], 3).view(e, n, k).double() - 8
    py, _ = plain_layer(x[:16].double(), nibbles * scales.double().repeat_interleave(group, 2), logits[:16].double(), top_k)
    print("serving: y %.2g (relative to 64 bits on the same 4-bit weights)" % far(serve.run(), py))


if __name__ == "__main__":
    main()
