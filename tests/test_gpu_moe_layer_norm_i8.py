"""The layer norm and the 8-bit products together with the other operators, as a training block and as a serving layer (moe_layer.py),
against 64 bits.

Tolerances as in test_gpu_moe_layer.py: a tensor that passed n roundings to 16 bits of unit u on its way is within n u (2-norms). Of the
training block, beside the layer's own: normed 1, so y 3; dx of the layer is dnormed (3, and 1 by normed), dx of the norm 5; dgamma and dbeta
take dnormed, 4, dw 3, dlogits 2. The serving layer against its own 8-bit rows and weights: rows and y, 2.
"""
import importlib.util
import os
import sys

import numpy as np
import pytest

from conftest import PKG_DIR
from test_gpu_norm_i8 import quant_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer(gg):
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    spec = importlib.util.spec_from_file_location("moe_layer", os.path.join(PKG_DIR, "moe_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    sys.modules["moe_layer"] = mod
    spec.loader.exec_module(mod)
    return mod


def far(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30)).item()


@pytest.mark.parametrize("tokens,e,n,k,top_k,kind,params,strided", [
    (200, 8, 512, 384, 2, "bf16", "f32", False), (33, 4, 136, 72, 4, "fp16", "fp16", True), (1000, 16, 264, 520, 3, "bf16", "bf16", False)])
def test_training_block(layer, tokens, e, n, k, top_k, kind, params, strided):
    import torch

    types = dict(bf16=torch.bfloat16, fp16=torch.float16, f32=torch.float32)
    dt, u = types[kind], 2.0 ** -8 if kind == "bf16" else 2.0 ** -11
    g = torch.Generator(device="cuda").manual_seed(tokens)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, res, w, dy = rand(tokens, k).to(dt), rand(tokens, k).to(dt), (rand(e, n, k) / k ** 0.5).to(dt), rand(tokens, n).to(dt)
    if strided:
        x = x.t().contiguous().t()
    gamma, beta = (1 + 0.2 * rand(k)).to(types[params]), (0.1 * rand(k)).to(types[params])
    logits, dpast = rand(tokens, e), rand(tokens, k).to(dt)
    norm, step = layer.Norm(gamma, beta), layer.TrainingLayer(w, top_k)
    normed, past = norm.forward(x, res)
    y, losses = step.forward(normed, logits)
    dnormed, dw, dlogits = step.backward(dy)
    dx, dgamma, dbeta = norm.backward(dnormed, dpast)
    step.check()
    norm.check()
    assert torch.equal(past, (x.float() + res.float()).to(dt))
    leaves = [v.double().requires_grad_() for v in (past, w, logits, gamma, beta)]
    c = leaves[0] - leaves[0].mean(1, keepdim=True)
    py, _ = layer.plain_layer(c * torch.rsqrt(c.square().mean(1, keepdim=True) + 1e-5) * leaves[3] + leaves[4], leaves[1], leaves[2], top_k)
    (torch.sum(py * dy.double()) + torch.sum(leaves[0] * dpast.double())).backward()
    for got, want, roundings in ((y, py, 3), (dx, leaves[0].grad, 5), (dw, leaves[1].grad, 3), (dlogits, leaves[2].grad, 2),
                                 (dgamma, leaves[3].grad, 4), (dbeta, leaves[4].grad, 4)):
        assert far(got, want) <= roundings * u + 1e-5
    again, same = norm.forward(past)  # without a residual what goes past is the input
    assert same is past and torch.equal(again, normed)


@pytest.mark.parametrize("tokens,e,n,k,top_k,norm,residual", [
    (1, 8, 512, 384, 2, True, True), (16, 4, 136, 96, 2, False, False), (300, 8, 264, 528, 4, True, False), (64, 33, 264, 1024, 8, True, True)])
def test_serving_layer_in_a_graph(layer, tokens, e, n, k, top_k, norm, residual):
    import torch

    g = torch.Generator(device="cuda").manual_seed(tokens)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    weight, scales = layer.quantize_i8((rand(e, n, k) / k ** 0.5).bfloat16())
    gamma, beta = ((1 + 0.2 * rand(k)).bfloat16(), (0.1 * rand(k)).bfloat16()) if norm else (None, None)
    s = layer.ServingLayerI8(weight, scales, tokens, top_k, gamma=gamma, beta=beta, residual=residual)
    wr = rand(k, e)

    def step():
        s.logits.copy_((s.norm() if norm else s.x).float() @ wr)
        s.run()

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for live in (tokens, (tokens + 1) // 2):
        s.x.copy_(rand(tokens, k).bfloat16())
        if residual:
            s.residual.copy_(rand(tokens, k).bfloat16())
        s.mask.zero_()
        s.mask[:live] = 1
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        rows = s.x
        if norm:
            total = (s.x.float() + s.residual.float()).bfloat16() if residual else s.x
            assert torch.equal(s.sum, total)
            c = total.double() - total.double().mean(1, keepdim=True)
            assert far(s.normed, c * torch.rsqrt(c.square().mean(1, keepdim=True) + 1e-5) * gamma.double() + beta.double()) <= 2.0 ** -8
            rows = s.normed
        q, qs = quant_ref(rows.float().cpu().numpy())
        if norm:
            assert np.array_equal(s.rounded[0].cpu().numpy(), q) and np.array_equal(s.rounded[1].cpu().numpy(), qs)
        x8 = torch.from_numpy(q).cuda().double() * torch.from_numpy(qs).cuda().double()[:, None]
        py, _ = layer.plain_layer(x8[:live], weight.double() * scales.double()[..., None], s.logits[:live].double(), top_k)
        assert far(s.y[:live], py) <= 2 * 2.0 ** -8
        assert (s.y[live:] == 0).all()
    for b in [s.router.backend, s.products, s.combine] + ([s.norms] if norm else []):
        assert b.device_status() == 0


def test_quantized_weights(layer):
    """Each weight within half a step of its row's scale, rows of zeros included."""
    import torch

    for dt in (torch.bfloat16, torch.float16, torch.float32):
        w = torch.randn(3, 40, 136, device="cuda").to(dt)
        w[1, 2] = 0
        weight, scales = layer.quantize_i8(w.transpose(0, 1).contiguous().transpose(0, 1))
        q, s = quant_ref(w.float().cpu().numpy().reshape(120, 136))
        assert np.array_equal(weight.cpu().numpy().reshape(120, 136), q) and np.array_equal(scales.cpu().numpy().reshape(120), s)


def test_two_layers_on_two_streams(layer):
    """Two serving layers at a time, each with handles and buffers of its own, give what they give alone."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(9)
    layers, want = [], []
    for i, (t, e, n, k) in enumerate(((40, 6, 520, 512), (700, 3, 1032, 256))):
        weight, scales = layer.quantize_i8(torch.randn(e, n, k, generator=g, device="cuda"))
        s = layer.ServingLayerI8(weight, scales, t, 2, torch.float16 if i else torch.bfloat16)
        s.x.normal_(generator=g)
        s.logits.normal_(generator=g)
        s.mask.fill_(1)
        layers.append(s)
        want.append(s.run().clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(20):
        for s, stream in zip(layers, streams):
            with torch.cuda.stream(stream):
                s.run()
    torch.cuda.synchronize()
    for s, w in zip(layers, want):
        assert torch.equal(s.y, w)
        assert s.products.device_status() == 0
