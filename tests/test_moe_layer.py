"""quantize_w4 of the layer (moe_layer.py) on the CPU: shapes, order of the nibbles, error of a weight.

Bound: a weight is half a step of its scale off, and an end of its range as much more as the scale's own rounding moves it
(8 or 15 steps x 2^-8 in bf16, 2^-11 in fp16) and, with a zero point, as the zero point's rounding does (half a step).
"""
import importlib.util
import os

import pytest

from conftest import PKG_DIR


@pytest.fixture(scope="module")
def layer(gg):
    spec = importlib.util.spec_from_file_location("moe_layer", os.path.join(PKG_DIR, "moe_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("kind,k,group", [("bfloat16", 128, 32), ("float16", 96, 64), ("float32", 264, 128)])
def test_error_of_a_weight(layer, kind, k, group, symmetric):
    import torch

    torch.manual_seed(k)
    w = torch.randn(3, 5, k).to(getattr(torch, kind))
    w[1, 2] = 0
    w[2, 3] = w[2, 3].abs()
    q, scales, zeros = layer.quantize_w4(w, group, symmetric)
    groups = -(-k // group)
    assert q.shape == (3, 5, k // 2) and q.dtype == torch.uint8 and scales.shape == (3, 5, groups)
    assert (zeros is None) == symmetric and scales.dtype == (torch.float16 if kind == "float16" else torch.bfloat16)
    step = scales.double().repeat_interleave(group, 2)[:, :, :k]
    zero = 8 if zeros is None else zeros.double().repeat_interleave(group, 2)[:, :, :k]
    got = (torch.stack([q & 15, q >> 4], 3).view(3, 5, k).double() - zero) * step
    assert torch.isfinite(step).all() and (step > 0).all()
    unit = 2.0 ** -11 if kind == "float16" else 2.0 ** -8
    slack = 8 * unit if symmetric else 15 * unit + 0.5
    assert ((got - w.double()).abs() <= step * (0.5 + slack)).all()
    assert (got[1, 2] == 0).all()
