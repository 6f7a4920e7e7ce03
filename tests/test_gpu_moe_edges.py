"""The layer operators (router, dispatch / combine, 4-bit products) where sizes, handles and values meet the limits of a kernel's
variant. Plain implementations, tolerances and helpers are those of test_gpu_moe_ops.py.
"""
import pytest

from test_gpu_moe_ops import Route, _torch, check_route, make_logits

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
