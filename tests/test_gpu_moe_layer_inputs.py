"""A training step of the layer (moe_layer.py) on tensors as autograd and slicing hand them on: the same bits as on dense copies."""
import importlib.util
import os

import pytest

from conftest import PKG_DIR

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer(gg):
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    spec = importlib.util.spec_from_file_location("moe_layer_inputs", os.path.join(PKG_DIR, "moe_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def a_step(layer, w, top_k, x, logits, mask, dy, dlosses):
    step = layer.TrainingLayer(w, top_k)
    return step.forward(x, logits, mask) + step.backward(dy, dlosses)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_strides(layer, kind):
    import torch

    t, e, n, k, top_k = 150, 8, 136, 72, 3
    dt = torch.bfloat16 if kind == "bf16" else torch.float16
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = (rand(e, n, k) / k ** 0.5).to(dt)
    views = dict(
        x=[rand(k, t).to(dt).t(), rand(t, k + 8).to(dt)[:, :k], rand(2 * t, k).to(dt)[::2]],
        logits=[rand(e, t).t(), rand(t, 2 * e)[:, ::2].bfloat16(), rand(1, e).expand(t, e)],
        mask=[(rand(t, 2) > -1).to(torch.uint8)[:, 0], rand(t) > -1, None],
        dy=[rand(()).to(dt).expand(t, n), rand(1, n).to(dt).expand(t, n), rand(n, t).to(dt).t()],  # the first: the gradient of y.sum()
        dlosses=[rand(()).expand(2), rand(4)[::2], None])
    for i in range(3):
        at = [views[name][i] for name in ("x", "logits", "mask", "dy", "dlosses")]
        dense = [v if v is None else v.clone(memory_format=torch.contiguous_format) for v in at]
        for a, b in zip(a_step(layer, w, top_k, *at), a_step(layer, w, top_k, *dense)):
            assert a.is_contiguous() and torch.equal(a, b)


def test_refused_on_the_device(layer):
    import torch

    w = torch.zeros(4, 16, 32, dtype=torch.bfloat16, device="cuda")
    step = layer.TrainingLayer(w, 2)
    x, logits = torch.zeros(6, 32, dtype=torch.bfloat16, device="cuda"), torch.zeros(6, 4, device="cuda")
    for bad in (dict(x=x.half()), dict(x=x.cpu()), dict(logits=logits.cpu()), dict(mask=torch.ones(6, dtype=torch.int64, device="cuda")),
                dict(mask=torch.ones(6, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            step.forward(**dict(dict(x=x, logits=logits), **bad))
    step.forward(x, logits)
    with pytest.raises(ValueError):
        step.backward(torch.zeros(6, 16, device="cuda"))
    with pytest.raises(ValueError):
        step.backward(torch.zeros(6, 16, dtype=torch.bfloat16))
    dx, dw, dlogits = step.backward(torch.zeros(6, 16, dtype=torch.bfloat16, device="cuda"))
    assert (dx == 0).all() and (dw == 0).all() and (dlogits == 0).all()


def test_no_live_token(layer):
    """Nothing to route: outputs and gradients are zero, the experts' too."""
    import torch

    w = torch.randn(4, 16, 32, device="cuda").bfloat16()
    step = layer.TrainingLayer(w, 2)
    x, logits = torch.randn(6, 32, device="cuda").bfloat16(), torch.randn(6, 4, device="cuda")
    y, losses = step.forward(x, logits, torch.zeros(6, dtype=torch.bool, device="cuda"))
    for v in (y, losses) + step.backward(torch.randn(6, 16, device="cuda").bfloat16(), torch.ones(2, device="cuda")):
        assert (v == 0).all()


def test_what_kernels_report_is_kept_for_check(layer):
    """An index that a kernel finds out of range is reported though other operators ran after it."""
    import torch

    t, e, n, k = 50, 8, 64, 64
    step = layer.TrainingLayer(torch.randn(e, n, k, device="cuda").bfloat16(), 2)
    x, logits, dy = torch.randn(t, k, device="cuda").bfloat16(), torch.randn(t, e, device="cuda"), torch.randn(t, n, device="cuda").bfloat16()
    step.forward(x, logits)
    step.backward(dy)
    step.check()
    step.forward(x, logits)
    step.router.offsets[e] = 1 << 30  # read by combine's gradient alone
    step.backward(dy)
    step.forward(x, logits)  # the forward's own handles are prepared again
    with pytest.raises(RuntimeError, match="^combine_grad: index out of range: status 0x2012$"):
        step.check()
    step.check()  # read and cleared
    step.router.ids[7, 1] = e  # read by the router's gradient alone
    step.backward(dy)
    with pytest.raises(RuntimeError, match="^route_grad: index out of range: status 0x2013$"):
        step.check()
    step.forward(x, logits)
    step.backward(dy)
    step.check()


def test_one_layer_steps_of_many_sizes(layer):
    """The handles are kept from step to step: other numbers of tokens, and no tokens, between two equal steps."""
    import torch

    e, n, k = 8, 136, 72
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = (rand(e, n, k) / k ** 0.5).bfloat16()
    kept = layer.TrainingLayer(w, 3)
    for t in (40, 700, 0, 1, 40, 3000, 40):
        x, logits, dy, dlosses = rand(t, k).bfloat16(), rand(t, e), rand(t, n).bfloat16(), rand(2)
        got = kept.forward(x, logits) + kept.backward(dy, dlosses)
        kept.check()
        for a, b in zip(got, a_step(layer, w, 3, x, logits, None, dy, dlosses)):
            assert torch.equal(a, b)


def test_router_of_an_earlier_step(layer):
    """The router of a step, kept by its user, stays that step's: it can be run again and differentiated after later steps."""
    import torch

    e, n, k = 8, 64, 64
    step = layer.TrainingLayer(torch.randn(e, n, k, device="cuda").bfloat16(), 2)
    a = torch.randn(50, e, device="cuda")
    step.forward(torch.randn(50, k, device="cuda").bfloat16(), a)
    first, dw = step.router, torch.randn(50, 2, device="cuda")
    ids, d = first.ids.clone(), first.grad(dw, None)
    step.forward(torch.randn(70, k, device="cuda").bfloat16(), torch.randn(70, e, device="cuda"))
    later = step.router.ids.clone()
    first.ids.zero_()
    first.run()
    assert torch.equal(first.ids, ids) and torch.equal(step.router.ids, later) and torch.equal(first.grad(dw, None), d)
    step.router.ids.zero_()
    step.router.run()
    assert torch.equal(step.router.ids, later) and torch.equal(first.ids, ids)


def test_bytes_of_any_type(layer):
    """Masks and packed weights are bytes: int8 and bool are read as uint8 is."""
    import torch

    t, e, n, k, top_k = 40, 4, 64, 64, 2
    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w, x, logits = rand(e, n, k).bfloat16(), rand(t, k).bfloat16(), rand(t, e)
    mask = (rand(t) > 0).to(torch.uint8)
    want = layer.TrainingLayer(w, top_k).forward(x, logits, mask)
    for as_type in (torch.int8, torch.bool):
        for a, b in zip(layer.TrainingLayer(w, top_k).forward(x, logits, mask.to(as_type)), want):
            assert torch.equal(a, b)
    q, scales, zeros = layer.quantize_w4(w, 32, symmetric=False)
    out = []
    for as_type in (torch.uint8, torch.int8):
        s = layer.ServingLayer(q.view(as_type), scales, zeros.view(as_type), 32, t, top_k)
        s.x.copy_(x), s.logits.copy_(logits), s.mask.copy_(mask)
        out.append(s.run().clone())
    assert torch.equal(*out) and (out[0][mask == 0] == 0).all()
