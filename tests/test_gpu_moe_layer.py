"""The layer operators together with the grouped GEMM, as a training step and as a serving step
(moe_layer.py), against the layer in 64 bits with autograd.

Tolerances (2-norm of the difference over the 2-norm of the result): a tensor that passed `n` roundings to 16 bits of unit
u (2^-8 bf16, 2^-11 fp16) on its way is within n u: y 2 (rows, y), dx 3 (drows, dx rows, dx), dw 2 (drows, dw); dlogits
take the rows' rounding through <dy, rows> (1) and are fp32 beside it.
"""
import importlib.util
import os
import sys

import pytest

from conftest import PKG_DIR

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


@pytest.mark.parametrize("tokens,e,n,k,top_k,kind", [(200, 8, 512, 384, 2, "bf16"), (33, 4, 136, 72, 4, "fp16"), (1000, 16, 264, 520, 3, "bf16")])
def test_training_step(layer, tokens, e, n, k, top_k, kind):
    import torch

    dt, u = (torch.bfloat16, 2.0 ** -8) if kind == "bf16" else (torch.float16, 2.0 ** -11)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w, dy = rand(tokens, k).to(dt), (rand(e, n, k) / k ** 0.5).to(dt), rand(tokens, n).to(dt)
    logits = rand(tokens, e)
    mask = (torch.rand(tokens, generator=g, device="cuda") > 0.1).to(torch.uint8)
    dlosses = torch.tensor([0.3, 0.02], device="cuda")
    step = layer.TrainingLayer(w, top_k)
    y, losses = step.forward(x, logits, mask)
    dx, dw, dlogits = step.backward(dy, dlosses)
    leaves = [v.double().requires_grad_() for v in (x, w, logits)]
    py, pl = layer.plain_layer(*leaves, top_k, mask)
    (torch.sum(py * dy.double()) + torch.sum(pl * dlosses.double())).backward()
    assert far(y, py) <= 2 * u
    assert far(losses, pl) <= 1e-5
    assert far(dx, leaves[0].grad) <= 3 * u
    assert far(dw, leaves[1].grad) <= 2 * u
    assert far(dlogits, leaves[2].grad) <= u + 1e-5
    assert (y[mask == 0] == 0).all() and (dx[mask == 0] == 0).all() and (dlogits[mask == 0] == 0).all()


@pytest.mark.parametrize("tokens,e,n,k,top_k,group,symmetric", [(1, 8, 512, 384, 2, 128, True), (16, 4, 136, 96, 2, 32, False), (64, 8, 264, 512, 8, 64, True)])
def test_serving_step_in_a_graph(layer, tokens, e, n, k, top_k, group, symmetric):
    import torch

    g = torch.Generator(device="cuda").manual_seed(tokens)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = (rand(e, n, k) / k ** 0.5).bfloat16()
    q, scales, zeros = layer.quantize_w4(w, group, symmetric)
    # the quantised weights are within half a scale of the given ones, plus the scale's own rounding at the range's end
    z = 8 if zeros is None else zeros.double().repeat_interleave(group, 2)[:, :, :k]
    grown = scales.double().repeat_interleave(group, 2)[:, :, :k]
    wq = (torch.stack([q & 15, q >> 4], 3).view(e, n, k).double() - z) * grown
    assert ((wq - w.double()).abs() <= grown * (0.5 + 16 * 2.0 ** -8 + (0 if symmetric else 0.5))).all()
    s = layer.ServingLayer(q, scales, zeros, group, tokens, top_k)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        s.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        s.run()
    for live in (tokens, (tokens + 1) // 2):
        s.x.copy_(rand(tokens, k).bfloat16())
        s.logits.copy_(rand(tokens, e))
        s.mask.zero_()
        s.mask[:live] = 1
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        py, _ = layer.plain_layer(s.x[:live].double(), wq, s.logits[:live].double(), top_k)
        assert far(s.y[:live], py) <= 2 * 2.0 ** -8
        assert (s.y[live:] == 0).all()
    for b in (s.router.backend, s.products, s.combine):
        assert b.device_status() == 0
