"""The layer norm and its gradients over many more rows than a group's ring holds: each slot is loaded again several times, and its barrier's
phase turns. What the rows are compared with is as in test_gpu_norm_i8.py."""
import re

import pytest

import test_gpu_norm_i8 as base
from test_gpu_moe_ops import _torch, _type

pytestmark = pytest.mark.gpu


def turns_and_slots(b, tokens):
    """The rows that a group takes at least, and those that its ring holds, of a prepared handle."""
    n = {k: int(v) for k, v in re.findall(r"(blocks|groups|slots|warps)=(\d+)", b.detail())}
    return tokens // (n["blocks"] * n["groups"]), n["slots"], n["warps"]


@pytest.mark.parametrize("tokens,hidden,kind,params,dsum,slots,warps", [
    # slots, warps: at least so many of a ring, and of a group (1: exactly, whose barrier is another)
    (2048, 4096, "f32", "f32", True, 2, 2),
    (2400, 7168, "bf16", "bf16", True, 2, 2),
    (2400, 8200, "fp16", "f32", True, 2, 2),
    (40000, 72, "bf16", "bf16", True, 4, 1),
    (40000, 256, "f32", "f32", False, 4, 1),
    (18000, 1024, "fp16", "fp16", False, 2, 2),
    (700, 16384, "f32", "f32", True, 1, 2),
])
def test_norm_grad_rings(gg, tokens, hidden, kind, params, dsum, slots, warps):
    torch = _torch()
    x = torch.zeros(16, dtype=torch.float32, device="cuda").data_ptr()
    b = gg.make_b200_backend()
    assert b.prepare_norm_grad(_type(gg, kind), tokens, hidden, x, x, x, x, x, dsum_ptr=x if dsum else 0, gamma_ptr=x, param_type=_type(gg, params)) == ""
    turns, ring, group = turns_and_slots(b, tokens)
    assert turns > 2 * ring and ring >= slots and (group == 1 if warps == 1 else group >= warps), b.detail()
    base.test_norm_grad(gg, tokens, hidden, kind, params, dsum)


@pytest.mark.parametrize("tokens,hidden,kind,params,residual,q,slots,warps", [
    (40000, 72, "bf16", "bf16", True, True, 4, 1),
    (40000, 248, "f32", "f32", False, False, 2, 1),
    (9000, 1024, "fp16", "f32", True, False, 2, 2),
    (4000, 7168, "bf16", "bf16", True, True, 2, 2),
    (3000, 8200, "fp16", "f32", False, True, 2, 2),
    (3000, 4096, "f32", "f32", True, False, 2, 2),
])
def test_norm_rings(gg, tokens, hidden, kind, params, residual, q, slots, warps):
    torch = _torch()
    x = torch.zeros(16, dtype=torch.float32, device="cuda").data_ptr()
    b = gg.make_b200_backend()
    assert b.prepare_norm(_type(gg, kind), tokens, hidden, x, x, residual_ptr=x if residual else 0, q_ptr=x if q else 0, q_scales_ptr=x if q else 0,
                          gamma_ptr=x, param_type=_type(gg, params)) == ""
    turns, ring, group = turns_and_slots(b, tokens)
    assert turns > 2 * ring and ring >= slots and (group == 1 if warps == 1 else group >= warps), b.detail()
    base.test_norm(gg, tokens, hidden, kind, params, residual, q)
