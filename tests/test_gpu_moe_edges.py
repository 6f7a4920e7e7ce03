"""The layer operators (router, dispatch / combine, 4-bit products) where sizes, handles and values meet the limits of a kernel's
variant. Plain implementations, tolerances and helpers are those of test_gpu_moe_ops.py.
"""
import math

import numpy as np
import pytest

from test_gpu_moe_ops import HALF_ULP, TINY, U, Route, _torch, check_route, close, make_logits, run_w4, w4_case, w4_ref

pytestmark = pytest.mark.gpu


# ---- router -----------------------------------------------------------------------------------


@pytest.mark.parametrize("e,k,kind,normalize", [(512, 8, "bf16", True), (513, 8, "f32", True), (1000, 32, "fp16", False), (1024, 1, "f32", False)])
@pytest.mark.parametrize("t", [0, 1, 7, 8, 9, 16, 17, 32, 33])
def test_route_few_tokens_of_many_experts(gg, t, e, k, kind, normalize):
    """One block with and without a thread an expert, and two blocks: the whole order, counts and losses."""
    torch = _torch()
    logits, mask = make_logits(torch, kind, t, e, 5 * t + e, pad=0.1 if t > 1 else 0.0, closed=0.1)
    for optional in (True, False):
        r = Route(gg, torch, kind, logits, mask, k, normalize, optional=optional)
        got = r.run()
        check_route(got, logits, mask, k, normalize)
        again = r.run()
        for n in got:
            assert got[n].tobytes() == again[n].tobytes(), n


@pytest.mark.parametrize("kind", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("large,small", [(256, 129), (256, 160), (128, 65), (512, 300), (1024, 600)])
def test_routers_of_one_kernel_beside_one_another(gg, kind, large, small):
    """Two handles prepared before either runs, the second with fewer experts of the same kernel."""
    torch = _torch()
    made = []
    for e in (large, small):
        logits, mask = make_logits(torch, kind, 300, e, e, pad=0.1)
        made.append((Route(gg, torch, kind, logits, mask, 4, True), logits, mask))
    for _ in range(2):
        for r, logits, mask in made:
            check_route(r.run(), logits, mask, 4, True)


def test_route_lse_near_zero(gg):
    """Rows of two open experts with logits 0 and x: lse = log(1 + e^x), whose sum rounds once (u) where its exponential is within (|x| + 4) u
    and the logarithm within one unit in its last place (2 u). An approximate logarithm misses this by up to 2 u more."""
    torch = _torch()
    t, e = 4000, 8
    x = torch.linspace(-10, -0.01, t, device="cuda")
    logits = torch.full((t, e), -math.inf, device="cuda")
    logits[:, 3], logits[:, 5] = 0.0, x
    got = Route(gg, torch, "f32", logits, None, 2, True).run()["lse"]
    x = x.double().cpu().numpy()
    want = np.log1p(np.exp(x))
    close(got, want, U * (1 + (4 - x) * np.exp(x) / (1 + np.exp(x)) + 2 * want))


# ---- 4-bit products -----------------------------------------------------------------------------------


@pytest.mark.parametrize("counts", [[2, 3], [40, 33]])  # one form and the other
@pytest.mark.parametrize("k,group", [(96, 64), (160, 32), (2880, 64), (1056, 32), (480, 64), (992, 32)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_w4_scales_stay_in_their_row(gg, counts, k, group, bad, kind):
    """A scale that is not finite makes its own weight row so, and no other: k ends inside a step, so the step has groups past the row."""
    torch = _torch()
    n = 24
    for zeros in (False, True):
        c = w4_case(torch, counts, n, k, group, zeros, kind, 0, 0)
        clean, _ = run_w4(gg, torch, c, counts, n, k, group, kind, 0)
        c["scales"][0, 5, 0] = bad
        c["scales"][1, 0, 0] = bad
        got, _ = run_w4(gg, torch, c, counts, n, k, group, kind, 0)
        m = counts[0]
        assert not torch.isfinite(got.t[:m, 5]).any() and not torch.isfinite(got.t[m:, 0]).any()
        keep = [i for i in range(n) if i != 5]
        assert torch.equal(got.t[:m][:, keep], clean.t[:m][:, keep])
        assert torch.equal(got.t[m:, 1:], clean.t[m:, 1:])


@pytest.mark.parametrize("counts", [[2, 3, 0, 1], [40, 33, 0, 20]])
@pytest.mark.parametrize("top_k", [0, 2])
def test_w4_falling_offsets(gg, counts, top_k):
    """Offsets that fall are reported and leave no expert any rows; those that only reach past the rows are cut there."""
    torch = _torch()
    n, k, group, rows = 600, 256, 128, sum(counts)
    c = w4_case(torch, counts, n, k, group, False, "bf16", top_k, 0)
    good, _ = run_w4(gg, torch, c, counts, n, k, group, "bf16", top_k)
    for bad in ([0, rows, 0, rows, 0], [0, rows, 0, rows, rows], [-5, 0, 1, 2, rows], [0, 2, 1, 5, rows], [0, 1, 2, 2, -(1 << 31)], [0, 1 << 30, 0, 1 << 30, rows]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        got, _ = run_w4(gg, torch, dict(c, offsets=offsets), counts, n, k, group, "bf16", top_k, status=0x2012)
        assert (got.t == 0).all()
    offsets = c["offsets"].clone()
    offsets[-1] = (1 << 31) - 1
    got, _ = run_w4(gg, torch, dict(c, offsets=offsets), counts, n, k, group, "bf16", top_k, status=0x2012)
    assert torch.equal(got.t, good.t)


@pytest.mark.parametrize("counts", [[2, 3], [40, 33]])
@pytest.mark.parametrize("k,group", [(256, 128), (160, 32), (4096, 64)])
@pytest.mark.parametrize("power", [127, -100])
def test_w4_scales_of_any_size(gg, counts, k, group, power):
    """Scales up to the type's largest times a small x, and scales near its smallest times a large x."""
    torch = _torch()
    n = 24
    c = w4_case(torch, counts, n, k, group, True, "bf16", 0, 0)
    c["scales"] = c["scales"] * 2.0 ** power
    c["x"] = c["x"] * 2.0 ** (-100 if power > 0 else 90)
    assert torch.isfinite(c["scales"]).all()
    out, _ = run_w4(gg, torch, c, counts, n, k, group, "bf16", 0)
    at = 0
    for e, m in enumerate(counts):
        ref, mag = w4_ref(torch, c["q"][e], c["scales"][e], c["zeros"][e], group, c["x"][at:at + m])
        tol = (k / 8 + 64) * 2 * U * mag
        tol = tol + HALF_ULP["bf16"] * (ref.abs() + tol) + TINY["bf16"]
        close(out.t[at:at + m].double().cpu().numpy(), ref.cpu().numpy(), tol.cpu().numpy())
        at += m
