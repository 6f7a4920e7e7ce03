"""The layer operators (router, dispatch / combine, 4-bit products) where sizes, handles and values meet the limits of a kernel's
variant. Plain implementations, tolerances and helpers are those of test_gpu_moe_ops.py.
"""
import math

import numpy as np
import pytest

from test_gpu_moe_ops import (HALF_ULP, TINY, U, Guarded, Route, _torch, _type, check_route, close, grad_ref, make_logits, run_w4, w4_case,
                              w4_ref)

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


@pytest.mark.parametrize("t,e,k,kind,normalize", [
    (14000, 256, 8, "f32", True),
    (14000, 256, 8, "bf16", False),
    (30011, 33, 3, "fp16", True),
    (30011, 32, 4, "f32", False),
    (9001, 1000, 32, "bf16", True),
])
def test_route_grad_of_more_rows_than_warps(gg, t, e, k, kind, normalize):
    """Each warp takes several rows: the next row on its way, the slots' own part cleared between rows, dead rows among live ones."""
    torch = _torch()
    logits, mask = make_logits(torch, kind, t, e, t + e, pad=0.2, closed=0.1)
    logits[mask == 0] = math.nan
    r = Route(gg, torch, kind, logits, mask, k, normalize)
    o = r.run()
    rng = np.random.RandomState(t)
    dw = rng.randn(t, k).astype(np.float32)
    dw[o["ids"] < 0] = np.nan
    dl = np.array([0.3, 0.02], np.float32)
    dwt, dlt = torch.from_numpy(dw).cuda(), torch.from_numpy(dl).cuda()
    out = Guarded(torch, (t, e), logits.dtype)
    b, s = gg.make_b200_backend(), torch.cuda.current_stream().cuda_stream
    assert b.prepare_route_grad(_type(gg, kind), t, e, k, logits.data_ptr(), out.ptr(), r.out["ids"].ptr(), r.out["lse"].ptr(),
                                r.out["counts"].ptr(), r.out["live"].ptr(), dweights_ptr=dwt.data_ptr(), dlosses_ptr=dlt.data_ptr(),
                                mask_ptr=mask.data_ptr(), normalize=normalize) == ""
    blocks = int(b.detail().split("blocks=")[1])
    assert t > 2 * 8 * blocks, "a warp has to get more than two rows"
    b.run(s)
    assert b.device_status(s) == 0
    out.check(torch)
    got = out.t.float().cpu().numpy().astype(np.float64)
    l = logits.float().cpu().numpy().astype(np.float64)
    m = mask.cpu().numpy()
    l[m == 0] = 0.0
    dw64 = np.where(o["ids"] >= 0, dw, 0.0).astype(np.float64)
    ref = grad_ref(l, m, o["ids"], o["counts"], int(o["live"][0]), dw64, dl.astype(np.float64), k, normalize, 1.0)
    n = max(int(o["live"][0]), 1)
    size = np.abs(dw64).sum(1) + dl[0] * e * o["counts"].max(initial=0) / (k * n * n) + 2 * dl[1] * np.abs(
        np.where(np.isfinite(o["lse"]), o["lse"], 0)) / n
    close(got, ref, 512 * U * size[:, None] + HALF_ULP[kind] * np.abs(ref) + TINY[kind])
    assert (got[m == 0] == 0).all()
    first = out.t.clone()
    b.run(s)
    assert torch.equal(first.view(torch.uint8), out.t.view(torch.uint8))


def test_handles_on_two_streams(gg):
    """Routers and products of different sizes on two streams at a time, over and over: each handle's own results, bit for bit."""
    torch = _torch()
    streams, jobs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i, (t, e, k, counts) in enumerate([(3000, 256, 8, [3] * 20), (2000, 200, 4, [40, 9, 33])]):
        logits, mask = make_logits(torch, "f32", t, e, i, pad=0.1)
        r = Route(gg, torch, "f32", logits, mask, k, True)
        want = r.run()
        c = w4_case(torch, counts, 1032, 2048, 64, True, "bf16", 0, 0, seed=i)
        out, b = run_w4(gg, torch, c, counts, 1032, 2048, 64, "bf16", 0)
        jobs.append((r, want, c, out, b, out.t.clone()))
        for v in r.out.values():
            v.t.zero_()
        out.t.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (r, _, _, _, b, _) in zip(streams, jobs):
            r.b.run(s.cuda_stream)
            b.run(s.cuda_stream)
    for s, (r, want, _, out, b, product) in zip(streams, jobs):
        assert r.b.device_status(s.cuda_stream) == 0 and b.device_status(s.cuda_stream) == 0
        torch.cuda.synchronize()
        for n, v in r.out.items():
            assert v.t.cpu().numpy().tobytes() == want[n].tobytes(), n
        assert torch.equal(out.t.view(torch.int16), product.view(torch.int16))


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


@pytest.mark.parametrize("counts", [[70000], [1, 40000, 0, 29997], [5] * 1024])
@pytest.mark.parametrize("top_k", [0, 3])
def test_w4_many_rows(gg, counts, top_k):
    """More rows than the gather has blocks (65536), and an expert of many chunks."""
    torch = _torch()
    n, k, group, extra = 8, 32, 32, 5
    c = w4_case(torch, counts, n, k, group, True, "bf16", top_k, extra)
    out, _ = run_w4(gg, torch, c, counts, n, k, group, "bf16", top_k)
    at = 0
    for e, m in enumerate(counts):
        r = torch.arange(at, at + m, device="cuda")
        x = c["x"][c["src"][r].long() // top_k] if top_k else c["x"][r]
        ref, mag = w4_ref(torch, c["q"][e], c["scales"][e], c["zeros"][e], group, x)
        tol = (k / 8 + 64) * 2 * U * mag
        tol = tol + HALF_ULP["bf16"] * (ref.abs() + tol) + TINY["bf16"]
        assert ((out.t[r].double() - ref).abs() <= tol).all(), e
        at += m
    assert (out.t[at:] == 0).all()


@pytest.mark.parametrize("counts", [[3, 12], [40, 33]])
def test_w4_bad_source_rows(gg, counts):
    """A source that is not a slot: reported, and no row but its own differs, in either form."""
    torch = _torch()
    n, k, group = 48, 256, 128
    c = w4_case(torch, counts, n, k, group, False, "bf16", 2, 0)
    good, _ = run_w4(gg, torch, c, counts, n, k, group, "bf16", 2)
    for bad in (-1, c["tokens"] * 2, (1 << 31) - 1, -(1 << 31)):
        src = c["src"].clone()
        src[4] = bad
        got, _ = run_w4(gg, torch, dict(c, src=src), counts, n, k, group, "bf16", 2, status=0x2011)
        keep = [r for r in range(sum(counts)) if r != 4]
        assert torch.equal(got.t[keep], good.t[keep]) and (got.t[4] == 0).all()


def test_w4_forms_meet(gg):
    """Numbers of rows on both sides of the change from one form to the other: each has the results of the definition."""
    torch = _torch()
    n, k, group = 264, 1152, 128
    seen = set()
    for counts in ([8] * 4, [8, 8, 8, 9], [0, 31, 1, 0], [0, 32, 1, 0], [33, 0, 0, 0]):
        c = w4_case(torch, counts, n, k, group, True, "fp16", 0, 0)
        out, b = run_w4(gg, torch, c, counts, n, k, group, "fp16", 0)
        seen.add(b.detail().split("<")[1].split(">")[0])
        at = 0
        for e, m in enumerate(counts):
            ref, mag = w4_ref(torch, c["q"][e], c["scales"][e], c["zeros"][e], group, c["x"][at:at + m])
            tol = (k / 8 + 64) * 2 * U * mag
            tol = tol + HALF_ULP["fp16"] * (ref.abs() + tol) + TINY["fp16"]
            close(out.t[at:at + m].double().cpu().numpy(), ref.cpu().numpy(), tol.cpu().numpy())
            at += m
    assert seen == {"fp16,few", "fp16,many"}
