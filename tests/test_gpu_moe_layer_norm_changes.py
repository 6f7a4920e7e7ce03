"""What Norm.backward (moe_layer.py) reads again is what its forward saw, or the call is refused."""
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


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("what", ["sum", "gamma"])
def test_a_change_between_forward_and_backward_is_refused(layer, residual, what):
    import torch

    x, res, dy = (torch.randn(40, 64, device="cuda").bfloat16() for _ in range(3))
    gamma, beta = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    norm = layer.Norm(gamma, beta)
    _, past = norm.forward(x, res if residual else None)
    want = norm.backward(dy)
    keep = past.clone(), gamma.clone()
    {"sum": past, "gamma": gamma}[what].mul_(2)
    with pytest.raises(ValueError, match="changed in place"):
        norm.backward(dy)
    past.copy_(keep[0])
    gamma.copy_(keep[1])
    norm.forward(past)
    assert all(torch.equal(a, b) for a, b in zip(norm.backward(dy), want))


def test_changes_of_what_backward_does_not_read(layer):
    """The terms of a sum, a copy of a strided input, the bias and the result; and tensors of inference mode, which count no changes."""
    import torch

    x, res, dy = (torch.randn(40, 64, device="cuda").bfloat16() for _ in range(3))
    gamma, beta = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    norm = layer.Norm(gamma, beta)
    y, _ = norm.forward(x, res)
    want = norm.backward(dy)
    for v in (x, res, beta, y):
        v.zero_()
    assert all(torch.equal(a, b) for a, b in zip(norm.backward(dy), want))
    strided = torch.randn(64, 40, device="cuda").bfloat16().t()
    norm.forward(strided)
    want = norm.backward(dy)
    strided.zero_()
    assert all(torch.equal(a, b) for a, b in zip(norm.backward(dy), want))
    with torch.inference_mode():
        x = torch.randn(40, 64, device="cuda").bfloat16()
        y, past = norm.forward(x)
        norm.backward(dy)
    norm.check()


def test_changes_beside_a_part_of_a_larger_tensor(layer):
    """One buffer for the activations of many layers, whose changes torch counts together, and a parameter of a flat one."""
    import torch

    acts, params = torch.randn(3, 40, 64, device="cuda").bfloat16(), torch.randn(4, 64, device="cuda")
    dy = torch.randn(40, 64, device="cuda").bfloat16()
    for x, gamma in ((acts[0], params[1]), (acts[0].detach(), params[1].detach())):
        norm = layer.Norm(gamma, None)
        norm.forward(x)
        want = norm.backward(dy)
        acts[1].mul_(2)
        params[2].mul_(2)
        assert all(torch.equal(a, b) for a, b in zip(norm.backward(dy), want))
