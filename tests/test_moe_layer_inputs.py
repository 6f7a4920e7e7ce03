"""What the layer (moe_layer.py) refuses before it hands an address to a kernel: types, shapes, strides, devices. On the CPU."""
import importlib.util
import os
import types

import pytest

from conftest import PKG_DIR

T, E, N, K, TOP = 6, 4, 16, 32, 2


@pytest.fixture(scope="module")
def layer(gg):
    spec = importlib.util.spec_from_file_location("moe_layer_inputs", os.path.join(PKG_DIR, "moe_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def good():
    import torch

    return dict(x=torch.zeros(T, K, dtype=torch.bfloat16), logits=torch.zeros(T, E), mask=torch.ones(T, dtype=torch.uint8))


FORWARD = [
    ("x", lambda torch: torch.zeros(T, K, dtype=torch.float16), "x must be torch.bfloat16"),
    ("x", lambda torch: torch.zeros(T, K), "x must be torch.bfloat16"),
    ("x", lambda torch: torch.zeros(T, K + 8, dtype=torch.bfloat16), "x must be"),
    ("x", lambda torch: torch.zeros(T, 1, K, dtype=torch.bfloat16), "x must be"),
    ("logits", lambda torch: torch.zeros(T, E, dtype=torch.float64), "logits must be"),
    ("logits", lambda torch: torch.zeros(T - 1, E), "logits must be"),
    ("logits", lambda torch: torch.zeros(E, T), "logits must be"),
    ("mask", lambda torch: torch.ones(T), "mask must be torch.uint8"),
    ("mask", lambda torch: torch.ones(T, dtype=torch.int32), "mask must be"),
    ("mask", lambda torch: torch.ones(T, dtype=torch.int64), "mask must be"),
    ("mask", lambda torch: torch.ones(T - 1, dtype=torch.bool), "mask must be"),
    ("mask", lambda torch: torch.ones(T, 1, dtype=torch.bool), "mask must be"),
    ("mask", lambda torch: torch.ones(T, dtype=torch.bool), "not on the current CUDA device"),  # all as it should be, but on the host
]


@pytest.mark.parametrize("which,make,reason", FORWARD)
def test_forward_refuses(layer, which, make, reason):
    import torch

    step = layer.TrainingLayer(torch.zeros(E, N, K, dtype=torch.bfloat16), TOP)
    with pytest.raises(ValueError, match=reason):
        step.forward(**dict(good(), **{which: make(torch)}))


@pytest.mark.parametrize("dy,dlosses,reason", [
    (lambda torch: torch.zeros(T, N), None, "dy must be"),
    (lambda torch: torch.zeros(T, N, dtype=torch.float16), None, "dy must be"),
    (lambda torch: torch.zeros(T, K, dtype=torch.bfloat16), None, "dy must be"),
    (lambda torch: torch.zeros(T + 1, N, dtype=torch.bfloat16), None, "dy must be"),
    (lambda torch: torch.zeros(T, N, dtype=torch.bfloat16), lambda torch: torch.zeros(2, dtype=torch.bfloat16), "dlosses must be"),
    (lambda torch: torch.zeros(T, N, dtype=torch.bfloat16), lambda torch: torch.zeros(2, dtype=torch.float64), "dlosses must be"),
    (lambda torch: torch.zeros(T, N, dtype=torch.bfloat16), lambda torch: torch.zeros(1), "dlosses must be"),
    (lambda torch: torch.zeros(T, N, dtype=torch.bfloat16), lambda torch: torch.zeros(()), "dlosses must be"),
])
def test_backward_refuses(layer, dy, dlosses, reason):
    import torch

    step = layer.TrainingLayer(torch.zeros(E, N, K, dtype=torch.bfloat16), TOP)
    step.router = types.SimpleNamespace(logits=torch.zeros(T, E))
    with pytest.raises(ValueError, match=reason):
        step.backward(dy(torch), dlosses(torch) if dlosses else None)


@pytest.mark.parametrize("make", [
    lambda torch: torch.zeros(E, N, K),
    lambda torch: torch.zeros(E, K, N, dtype=torch.bfloat16).transpose(1, 2),
    lambda torch: torch.zeros(E, N, 2 * K, dtype=torch.bfloat16)[:, :, ::2],
])
def test_experts_refused(layer, make):
    import torch

    with pytest.raises(ValueError, match="w must be"):
        layer.TrainingLayer(make(torch), TOP)


@pytest.mark.parametrize("logits,mask,reason", [
    (lambda torch: torch.zeros(E, T).t(), None, "not contiguous"),
    (lambda torch: torch.zeros(T, 2 * E)[:, ::2], None, "not contiguous"),
    (lambda torch: torch.zeros(1, E).expand(T, E), None, "not contiguous"),
    (lambda torch: torch.zeros(T, E, dtype=torch.int32), None, "logits must be"),
    (lambda torch: torch.zeros(T, E), lambda torch: torch.ones(T, dtype=torch.int64), "mask must be"),
    (lambda torch: torch.zeros(T, E), None, "not on the current CUDA device"),
])
def test_router_refuses(layer, logits, mask, reason):
    """A router reads the buffers it was given again in each run, so it takes no copies."""
    import torch

    with pytest.raises(ValueError, match=reason):
        layer.Router(logits(torch), TOP, mask(torch) if mask else None)


@pytest.mark.parametrize("dweights,dlosses,reason", [
    (lambda torch: torch.zeros(T, TOP, dtype=torch.bfloat16), None, "dweights must be"),
    (lambda torch: torch.zeros(T, TOP + 1), None, "dweights must be"),
    (None, lambda torch: torch.zeros(2, dtype=torch.float16), "dlosses must be"),
])
def test_router_gradient_refuses(layer, dweights, dlosses, reason):
    import torch

    r = object.__new__(layer.Router)
    r.logits, r.top_k = torch.zeros(T, E), TOP
    with pytest.raises(ValueError, match=reason):
        r.grad(dweights(torch) if dweights else None, dlosses(torch) if dlosses else None)


@pytest.mark.parametrize("which,make,reason", [
    ("qweight", lambda torch: torch.zeros(E, N, K // 2, dtype=torch.int32), "qweight must be"),
    ("scales", lambda torch: torch.zeros(E, N, 1), "scales must be"),
    ("scales", lambda torch: torch.zeros(E, N, 2, dtype=torch.bfloat16), "scales must be"),
    ("zeros", lambda torch: torch.zeros(E, N, 1, dtype=torch.int32), "zeros must be"),
    ("zeros", lambda torch: torch.zeros(E, 1, 1, dtype=torch.uint8), "zeros must be"),
    ("zeros", lambda torch: None, "not on the current CUDA device"),
])
def test_serving_layer_refuses(layer, which, make, reason):
    import torch

    a = dict(qweight=torch.zeros(E, N, K // 2, dtype=torch.uint8), scales=torch.zeros(E, N, 1, dtype=torch.bfloat16), zeros=None)
    a[which] = make(torch)
    with pytest.raises(ValueError, match=reason):
        layer.ServingLayer(a["qweight"], a["scales"], a["zeros"], 128, T, TOP)
