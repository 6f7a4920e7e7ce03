"""What the layer norm and the 8-bit serving layer (moe_layer.py) refuse before they hand an address to a kernel: types, shapes, strides,
devices. On the CPU."""
import importlib.util
import os

import pytest

from conftest import PKG_DIR

T, E, N, K, TOP = 6, 4, 16, 32, 2


@pytest.fixture(scope="module")
def layer(gg):
    spec = importlib.util.spec_from_file_location("moe_layer_norm_i8", os.path.join(PKG_DIR, "moe_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("gamma,beta,reason", [
    (lambda t: t.ones(K, dtype=t.float64), lambda t: None, "gamma must be"),
    (lambda t: t.ones(1, K), lambda t: None, "gamma must be"),
    (lambda t: [1.0] * K, lambda t: None, "gamma must be"),
    (lambda t: None, lambda t: t.ones(2 * K)[::2], "beta must be contiguous"),
    (lambda t: t.ones(K), lambda t: t.ones(K, dtype=t.bfloat16), "one type"),
])
def test_norm_parameters(layer, gamma, beta, reason):
    import torch

    with pytest.raises(ValueError, match=reason):
        layer.Norm(gamma(torch), beta(torch))


@pytest.mark.parametrize("x,residual,reason", [
    (lambda t: t.zeros(T, K, dtype=t.float64), lambda t: None, "x must be"),
    (lambda t: t.zeros(T, K + 8, dtype=t.bfloat16), lambda t: None, "gamma must be"),
    (lambda t: t.zeros(T, K, dtype=t.float16), lambda t: None, "gamma and beta must be torch.float16 or torch.float32"),
    (lambda t: t.zeros(T, K, dtype=t.bfloat16), lambda t: t.zeros(T, K), "residual must be"),
    (lambda t: t.zeros(T, K, dtype=t.bfloat16), lambda t: t.zeros(T - 1, K, dtype=t.bfloat16), "residual must be"),
    (lambda t: t.zeros(T, K, dtype=t.bfloat16), lambda t: None, "not on the current CUDA device"),
])
def test_norm_forward(layer, x, residual, reason):
    import torch

    norm = layer.Norm(torch.ones(K, dtype=torch.bfloat16), torch.zeros(K, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match=reason):
        norm.forward(x(torch), residual(torch))


def test_norm_backward(layer):
    import torch

    norm = layer.Norm(None, None)
    with pytest.raises(ValueError, match="forward"):
        norm.backward(torch.zeros(T, K))
    norm.sum, norm.mean, norm.rstd = torch.zeros(T, K), torch.zeros(T), torch.zeros(T)
    for dy, dsum, reason in ((torch.zeros(T, K + 1), None, "dy must be"), (torch.zeros(T, K).half(), None, "dy must be"),
                             (torch.zeros(T, K), torch.zeros(K, T), "dsum must be"), (torch.zeros(T, K), None, "not on the current CUDA device")):
        with pytest.raises(ValueError, match=reason):
            norm.backward(dy, dsum)


def test_norm_backward_after_a_refused_forward(layer):
    """It would pair the tokens of one forward with the statistics of another."""
    import torch

    norm = layer.Norm(None, None)
    norm.sum, norm.mean, norm.rstd = torch.zeros(T, K), torch.zeros(T), torch.zeros(T)
    with pytest.raises(ValueError, match="not on the current CUDA device"):
        norm.forward(torch.zeros(1, K))
    with pytest.raises(ValueError, match="forward before it"):
        norm.backward(torch.zeros(T, K))


@pytest.mark.parametrize("change,reason", [
    (dict(weight=lambda t: t.zeros(E, N, K)), "weight must be torch.int8"),
    (dict(scales=lambda t: t.zeros(E, N, dtype=t.bfloat16)), "scales must be torch.float32"),
    (dict(scales=lambda t: t.zeros(N, E)), "scales must be"),
    (dict(dtype=lambda t: t.float32), "dtype must be"),
    (dict(gamma=lambda t: t.ones(K)), "go together"),
    (dict(residual=lambda t: True), "needs gamma"),
    (dict(), "not on the current CUDA device"),
])
def test_serving(layer, change, reason):
    import torch

    args = dict(weight=lambda t: t.zeros(E, N, K, dtype=t.int8), scales=lambda t: t.zeros(E, N), tokens=lambda t: T, top_k=lambda t: TOP)
    with pytest.raises(ValueError, match=reason):
        layer.ServingLayerI8(**{n: v(torch) for n, v in dict(args, **change).items()})


def test_quantize(layer):
    import torch

    for w, reason in ((torch.zeros(E, N, K, dtype=torch.float64), "w must be"), (torch.zeros(E, N, K), "not on the current CUDA device")):
        with pytest.raises(ValueError, match=reason):
            layer.quantize_i8(w)
