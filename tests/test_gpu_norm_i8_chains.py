"""Kernels one behind the other without the host between them, where each starts before the one in front of it has ended: the same bits as with
plain launches ("pdl" 0), for contents that change from run to run."""
import importlib.util
import os
import sys

import pytest

from conftest import PKG_DIR
from test_gpu_moe_ops import _torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer(gg):
    _torch()
    spec = importlib.util.spec_from_file_location("moe_layer", os.path.join(PKG_DIR, "moe_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    sys.modules["moe_layer"] = mod
    spec.loader.exec_module(mod)
    return mod


def captured(torch, step, times):
    """A graph of `times` steps, which have run once before."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for _ in range(times):
            step()
    return graph


@pytest.mark.parametrize("tokens,top_k,k,norm", [(1, 8, 1024, False), (1, 8, 1024, True), (5, 2, 7168, False), (300, 4, 512, True)])
def test_serving_steps_whose_routing_changes(layer, tokens, top_k, k, norm):
    """Router, products and combine in a graph, replayed with other logits and tokens each time."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(tokens + k)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    e, n = 64, 520
    weight, scales = layer.quantize_i8((rand(e, n, k) / k ** 0.5).bfloat16())
    gamma, beta = ((1 + 0.2 * rand(k)).bfloat16(), (0.1 * rand(k)).bfloat16()) if norm else (None, None)
    fast, plain = (layer.ServingLayerI8(weight, scales, tokens, top_k, gamma=gamma, beta=beta) for _ in range(2))
    for b in [plain.router.backend, plain.products, plain.combine] + ([plain.norms] if norm else []):
        b.set_option("pdl", 0)

    def step(s):
        if norm:
            s.norm()
        s.run()

    graph = captured(torch, lambda: step(fast), 3)
    for i in range(40):
        for to, v in ((fast.x, rand(tokens, k).bfloat16()), (fast.logits, rand(tokens, e)), (fast.mask, (torch.rand(tokens, generator=g, device="cuda") > 0.1) | (tokens == 1))):
            to.copy_(v)
        for a, b in ((plain.x, fast.x), (plain.logits, fast.logits), (plain.mask, fast.mask)):
            a.copy_(b)
        graph.replay()
        step(plain)
        assert torch.equal(fast.router.offsets, plain.router.offsets)
        assert torch.equal(fast.y.view(torch.int16), plain.y.view(torch.int16)), i
    assert fast.products.device_status() == 0 and plain.products.device_status() == 0
