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


@pytest.mark.parametrize("tokens,top_k,k", [(1, 8, 1024), (40, 4, 512), (300, 4, 512)])
def test_4_bit_serving_steps_whose_routing_changes(layer, tokens, top_k, k):
    """The same over 4-bit experts, for few rows an expert and for many."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(tokens + k)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    e, n = 64, 520
    q, scales, zeros = layer.quantize_w4((rand(e, n, k) / k ** 0.5).bfloat16(), 64)
    fast, plain = (layer.ServingLayer(q, scales, zeros, 64, tokens, top_k) for _ in range(2))
    for b in (plain.router.backend, plain.products, plain.combine):
        b.set_option("pdl", 0)
    fast.mask.fill_(1)
    plain.mask.fill_(1)
    graph = captured(torch, fast.run, 3)
    for i in range(40):
        for a, b, v in ((fast.x, plain.x, rand(tokens, k).bfloat16()), (fast.logits, plain.logits, rand(tokens, e))):
            a.copy_(v)
            b.copy_(v)
        graph.replay()
        plain.run()
        assert torch.equal(fast.router.offsets, plain.router.offsets)
        assert torch.equal(fast.y.view(torch.int16), plain.y.view(torch.int16)), i
    assert fast.products.device_status() == 0 and plain.products.device_status() == 0


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_each_operator_behind_the_one_that_writes_its_input(gg, kind):
    """Norm -> its gradients -> rounding -> 8-bit products, and norm -> 4-bit products, in one graph, with contents that change."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t, h, n, group = 37, 1024, 264, 64
    dt, half = dict(bf16=torch.bfloat16, f32=torch.float32)[kind], torch.bfloat16
    kt = dict(bf16=gg.BF16, f32=gg.F32)[kind]
    x, dy, w = rand(t, h).to(dt), rand(t, h).to(dt), rand(n, h).to(dt)
    offsets = torch.tensor([0, t], dtype=torch.int32, device="cuda")
    qweight = torch.randint(0, 256, (1, n, h // 2), dtype=torch.uint8, generator=g, device="cuda")
    w4_scales = (0.01 * torch.rand(1, n, h // group, generator=g, device="cuda")).to(half)

    def chain(pdl):
        f32 = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        o = dict(y=torch.zeros_like(x), mean=f32(t), rstd=f32(t), dx=torch.zeros_like(x), dgamma=f32(h), dbeta=f32(h), q=torch.zeros(t, h, dtype=torch.int8, device="cuda"),
                 qs=f32(t), wq=torch.zeros(1, n, h, dtype=torch.int8, device="cuda"), ws=f32(1, n), out=torch.zeros(t, n, dtype=half, device="cuda"),
                 out4=torch.zeros(t, n, dtype=half, device="cuda"))
        p = {k: v.data_ptr() for k, v in o.items()}
        b = [gg.make_b200_backend() for _ in range(6)]
        whys = [b[0].prepare_norm(kt, t, h, x.data_ptr(), p["y"], mean_ptr=p["mean"], rstd_ptr=p["rstd"]),
                b[1].prepare_norm_grad(kt, t, h, x.data_ptr(), p["mean"], p["rstd"], dy.data_ptr(), p["dx"], dgamma_ptr=p["dgamma"], dbeta_ptr=p["dbeta"]),
                b[2].prepare_quant(kt, t, h, p["dx"], p["q"], p["qs"]),
                b[3].prepare_quant(kt, n, h, w.data_ptr(), p["wq"], p["ws"]),
                b[4].prepare_i8(gg.BF16, 1, n, h, t, p["q"], p["wq"], p["ws"], offsets.data_ptr(), p["out"], x_scales_ptr=p["qs"])]
        if kind == "bf16":
            whys.append(b[5].prepare_w4(gg.BF16, 1, n, h, group, t, p["y"], qweight.data_ptr(), w4_scales.data_ptr(), offsets.data_ptr(), p["out4"]))
        assert not any(whys), whys
        for v in b:
            v.set_option("pdl", pdl)
        order = [0, 1, 2, 3, 4] + ([0, 5] if kind == "bf16" else [])

        def step():
            s = torch.cuda.current_stream().cuda_stream
            for i in order:
                b[i].run(s)

        return o, step, b

    fast, run_fast, backends = chain(1)
    plain, run_plain, _ = chain(0)
    graph = captured(torch, run_fast, 2)
    for i in range(30):
        for v in (x, dy, w):
            v.copy_(rand(*v.shape).mul_(1 + i).to(dt))
        graph.replay()
        run_plain()
        for k in fast:
            assert torch.equal(fast[k].view(torch.uint8), plain[k].view(torch.uint8)), (k, i)
    assert not any(v.device_status() for v in backends[:5])
