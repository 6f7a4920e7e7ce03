"""The layer operators around the grouped GEMM (router, dispatch / combine, 4-bit products) against
plain implementations of their definitions in 64 bits, through the C ABI.

Whole numbers have to be equal. Tolerances for computed values, u = 2^-24 (one fp32 rounding):
  softmax terms   |l - max| u from the difference, 4 u from exp and the division, 40 u from a sum of up to
                  1024 terms (32 a lane, 5 levels): (|l - max| + 64) u relative; differences here stay below 192,
                  so 256 u (2^-16)
  lse             its own rounding and the sum's relative error: (|lse| + 64) u
  sums over t     tokens one after the other in a warp, then warps, then blocks: (tokens + 256) u of the sum of magnitudes
  k-term sums     (k + 1) u of the sum of magnitudes
  dot products    8 terms a vector, vectors one after the other in a thread, then the tree: (8 ceil(h / 2048) + 24) u of the sum of magnitudes
  4-bit products  16 products a step, one rounding (or truncation, 2 u) a step: (k / 8 + 64) 2 u of the sum of magnitudes
and half a unit in the last place where the output has 16 bits.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "f32": U}  # 8, 11 and 24 significant bits
TINY = {"bf16": 1e-38, "fp16": 2.0 ** -25, "f32": 1e-37}
GUARD = 64


def _torch():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


def _type(gg, name):
    return {"bf16": gg.BF16, "fp16": gg.FP16, "f32": gg.F32}[name]


def _dtype(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}[name]


class Guarded:
    """An output with a canary behind it: a store past the end is seen."""

    def __init__(self, torch, shape, dtype):
        self.n = int(np.prod(shape))
        self.all = torch.empty(self.n + GUARD, dtype=dtype, device="cuda")
        self.all.view(torch.uint8).fill_(0x5A)
        self.shape = shape
        self.want = self.all[self.n:].view(torch.uint8).clone()

    @property
    def t(self):
        return self.all[: self.n].view(self.shape)

    def ptr(self):
        return self.all.data_ptr()

    def check(self, torch):
        assert torch.equal(self.all[self.n:].view(torch.uint8), self.want), "store past the end of an output"


def close(got, want, tol):
    """|got - want| <= tol elementwise in 64 bits, with equal infinities and NaN."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    tol = np.broadcast_to(tol, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    off = np.abs(got[fine] - want[fine]) - tol[fine]
    assert off.size == 0 or off.max() <= 0, f"off by {off.max():.3g} over the tolerance, {np.count_nonzero(off > 0)} of {off.size}"


# ---- router -----------------------------------------------------------------------------------


def route_ref(logits, mask, k, normalize, scale=1.0):
    l = logits.astype(np.float64)
    t, e = l.shape
    l = np.where(mask[:, None] != 0, l, -np.inf)
    alive = ~(l == -np.inf).all(1)
    with np.errstate(all="ignore"):
        mx = np.where(alive, l.max(1, initial=-np.inf), 0.0)
        ex = np.exp(l - mx[:, None])
        lse = np.where(alive, mx + np.log(ex.sum(1)), -np.inf)
        p = np.where(alive[:, None], ex / ex.sum(1, keepdims=True), 0.0)
    order = np.where(np.isnan(l), np.inf, l)
    # NaN first, then falling values, ties to the lower index
    pick = np.stack([np.lexsort((np.arange(e), -order[i], ~np.isnan(l[i]))) for i in range(t)]) if t else np.zeros((0, e), int)
    pick = pick[:, :k]
    there = ~(np.take_along_axis(l, pick, 1) == -np.inf)
    ids = np.where(there, pick, -1)
    q = np.where(there, np.take_along_axis(p, pick, 1), 0.0)
    if normalize:
        with np.errstate(all="ignore"):
            q = np.where(there, q / q.sum(1, keepdims=True), 0.0)
    w = q * scale
    flat = ids.ravel()
    counts = np.bincount(flat[flat >= 0], minlength=e)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    order = np.argsort(np.where(flat < 0, e, flat), kind="stable")
    total = int(counts.sum())
    src = np.where(np.arange(flat.size) < total, order, -1)
    dest = np.full(flat.size, -1)
    dest[order[:total]] = np.arange(total)
    live = int(alive.sum())
    n = max(live, 1)
    prob = p.sum(0) / n
    losses = np.array([e * (counts / (k * n) * prob).sum(), (lse[alive] ** 2).sum() / n])
    return dict(ids=ids, weights=w, lse=lse, counts=counts, offsets=offsets, live=np.array([live]), dest=dest.reshape(t, k), src=src,
                prob=prob, losses=losses)


class Route:
    def __init__(self, gg, torch, kind, logits, mask, k, normalize, scale=1.0, optional=True):
        t, e = logits.shape
        i32, f32 = torch.int32, torch.float32
        self.torch = torch
        self.logits = logits.contiguous()
        self.mask = mask
        o = dict(ids=((t, k), i32), weights=((t, k), f32), counts=((e,), i32), offsets=((e + 1,), i32), live=((1,), i32), dest=((t, k), i32),
                 src=((t * k,), i32))
        if optional:
            o.update(lse=((t,), f32), prob=((e,), f32), losses=((2,), f32))
        self.out = {n: Guarded(torch, *v) for n, v in o.items()}
        self.b = gg.make_b200_backend()
        why = self.b.prepare_route(_type(gg, kind), t, e, k, self.logits.data_ptr(), mask_ptr=0 if mask is None else mask.data_ptr(),
                                   normalize=normalize, scale=scale, **{n + "_ptr": v.ptr() for n, v in self.out.items()})
        assert why == "", why

    def run(self, stream=None):
        s = stream or self.torch.cuda.current_stream()
        self.b.run(s.cuda_stream)
        assert self.b.device_status(s.cuda_stream) == 0
        for v in self.out.values():
            v.check(self.torch)
        return {n: v.t.cpu().numpy() for n, v in self.out.items()}


def make_logits(torch, kind, t, e, seed, pad=0.0, closed=0.0, coarse=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(t, e, generator=g, device="cuda") * 2 + torch.randn(e, generator=g, device="cuda")
    if coarse:
        x = (x * 2).round() / 2  # many ties
    x = x.to(_dtype(torch, kind))
    if closed:
        x[torch.rand(t, e, generator=g, device="cuda") < closed] = -math.inf
    mask = (torch.rand(t, generator=g, device="cuda") >= pad).to(torch.uint8)
    return x, mask


def check_route(got, logits, mask, k, normalize, scale=1.0):
    l = logits.float().cpu().numpy()
    m = np.ones(l.shape[0]) if mask is None else mask.cpu().numpy()
    ref = route_ref(l, m, k, normalize, scale)
    for n in ("ids", "counts", "offsets", "live", "dest", "src"):
        assert np.array_equal(got[n], ref[n]), n
    close(got["weights"], ref["weights"], 256 * U * np.abs(ref["weights"]) + 1e-37)
    if "lse" in got:
        close(got["lse"], ref["lse"], (np.abs(np.where(np.isfinite(ref["lse"]), ref["lse"], 0)) + 64) * U)
        many = (l.shape[0] + 512) * U
        close(got["prob"], ref["prob"], many * np.abs(ref["prob"]) + 1e-37)
        with np.errstate(over="ignore"):
            losses = ref["losses"].astype(np.float32).astype(np.float64)  # a square past fp32's range is infinite there
        close(got["losses"], losses, 2 * many * np.abs(losses) + 1e-37)
    return ref


ROUTES = [
    # tokens, experts, top_k, type, normalize, pad, closed, coarse
    (1, 256, 8, "f32", True, 0.0, 0.0, False),
    (1, 1, 1, "bf16", False, 0.0, 0.0, False),
    (0, 16, 2, "f32", True, 0.0, 0.0, False),
    (2, 3, 3, "fp16", True, 0.0, 0.3, False),
    (7, 33, 5, "bf16", True, 0.0, 0.0, True),
    (64, 64, 6, "f32", False, 0.1, 0.2, True),
    (65, 32, 32, "f32", True, 0.0, 0.5, False),
    (129, 100, 8, "fp16", False, 0.3, 0.0, True),
    (300, 1024, 32, "f32", True, 0.0, 0.1, False),
    (1000, 1023, 3, "bf16", True, 0.1, 0.0, False),
    (1187, 7, 2, "f32", False, 0.5, 0.6, True),
    (2500, 128, 4, "bf16", True, 0.05, 0.05, True),
    (20011, 256, 8, "f32", True, 0.02, 0.0, False),
    (20011, 8, 2, "fp16", True, 0.02, 0.1, True),
    (1031, 512, 7, "f32", False, 0.1, 0.1, False),
    (2000, 1000, 8, "bf16", True, 0.0, 0.3, False),
    (8192, 256, 8, "f32", True, 0.0, 0.0, False),
    (9000, 130, 4, "fp16", False, 0.9, 0.2, True),
]


@pytest.mark.parametrize("t,e,k,kind,normalize,pad,closed,coarse", ROUTES)
def test_route(gg, t, e, k, kind, normalize, pad, closed, coarse):
    torch = _torch()
    logits, mask = make_logits(torch, kind, t, e, 11 + t + e, pad, closed, coarse)
    r = Route(gg, torch, kind, logits, mask, k, normalize, 1.0 if normalize else 2.5)
    got = r.run()
    check_route(got, logits, mask, k, normalize, 1.0 if normalize else 2.5)
    again = r.run()
    for n in got:
        assert got[n].tobytes() == again[n].tobytes(), f"{n}: the same inputs gave other bits"


@pytest.mark.parametrize("kind", ["f32", "bf16", "fp16"])
def test_route_special_rows(gg, kind):
    """Rows that leave nothing, the type's lowest value, signed zeros, infinities and NaN."""
    torch = _torch()
    dt = _dtype(torch, kind)
    low = torch.finfo(dt).min
    inf, nan = math.inf, math.nan
    rows = [
        [-inf] * 6,                        # nothing open
        [low] * 6,                         # lowest finite value everywhere: open, uniform
        [low, 1.0, low, low, low, low],    # masked by the lowest value: open still, probability 0
        [-inf, -inf, 2.0, -inf, -inf, -inf],
        [0.0, -0.0, 0.0, -0.0, 0.0, -0.0],  # one value
        [nan, nan, inf, -inf, 1.0, 2.0],   # masked row
        [1.0, inf, 0.0, inf, 2.0, 3.0],    # +inf in a live row
        [1.0, nan, inf, 4.0, nan, -inf],   # NaN in a live row
        [-inf, 3.0, -inf, 5.0, 5.0, -inf],
    ]
    mask = [1, 1, 1, 1, 1, 0, 0, 0, 1]
    logits = torch.tensor(rows, device="cuda").to(dt)
    m = torch.tensor(mask, dtype=torch.uint8, device="cuda")
    for k in (1, 2, 4, 6):
        for normalize in (True, False):
            check_route(Route(gg, torch, kind, logits, m, k, normalize).run(), logits, m, k, normalize)
    # the same rows live: their own values are NaN, and the sums over all tokens too
    m[5:8] = 1
    for k in (1, 4):
        got = Route(gg, torch, kind, logits, m, k, True).run()
        ref = route_ref(logits.float().cpu().numpy(), m.cpu().numpy(), k, True)
        for n in ("ids", "counts", "offsets", "live", "dest", "src"):
            assert np.array_equal(got[n], ref[n]), n
        good = [0, 1, 2, 3, 4, 8]
        close(got["weights"][good], ref["weights"][good], 256 * U)
        assert np.isnan(got["weights"][5:8][ref["ids"][5:8] >= 0]).all()
        assert np.isnan(got["lse"][5:8]).all()
        assert np.isnan(got["losses"]).all()


def test_route_without_optional_outputs_or_mask(gg):
    torch = _torch()
    logits, _ = make_logits(torch, "f32", 77, 40, 5)
    check_route(Route(gg, torch, "f32", logits, None, 4, True, optional=False).run(), logits, None, 4, True)


def test_route_all_tokens_masked(gg):
    torch = _torch()
    logits, mask = make_logits(torch, "bf16", 50, 16, 6)
    logits[3] = math.nan
    mask.zero_()
    got = Route(gg, torch, "bf16", logits, mask, 2, True).run()
    check_route(got, logits, mask, 2, True)
    assert got["live"][0] == 0 and (got["losses"] == 0).all() and (got["prob"] == 0).all()


def test_route_new_contents_other_stream_and_graph(gg):
    """One handle: other contents in the same buffers, a stream of its own, a captured graph."""
    torch = _torch()
    logits, mask = make_logits(torch, "f32", 500, 64, 7, pad=0.1)
    r = Route(gg, torch, "f32", logits, mask, 6, True)
    check_route(r.run(), r.logits, mask, 6, True)
    other, m2 = make_logits(torch, "f32", 500, 64, 8, pad=0.3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        r.logits.copy_(other)
        mask.copy_(m2)
        got = r.run(s)
    check_route(got, other, m2, 6, True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        r.b.run(s.cuda_stream)
    third, m3 = make_logits(torch, "f32", 500, 64, 9, pad=0.2)
    torch.cuda.synchronize()
    r.logits.copy_(third)
    mask.copy_(m3)
    g.replay()
    torch.cuda.synchronize()
    check_route({n: v.t.cpu().numpy() for n, v in r.out.items()}, third, m3, 6, True)


# ---- router's gradient ---------------------------------------------------------------------------


def objective(l, mask, ids, counts, live, dw, dl, k, normalize, scale):
    """Sum of dw * weights and dl * losses for fixed choices and counts, in 64 bits."""
    t, e = l.shape
    l = np.where(mask[:, None] != 0, l, -np.inf)
    alive = np.isfinite(l).any(1)
    n = max(live, 1)
    with np.errstate(all="ignore"):
        mx = np.where(alive, l.max(1), 0.0)
        ex = np.exp(l - mx[:, None])
        lse = np.where(alive, mx + np.log(ex.sum(1)), 0.0)
        p = np.where(alive[:, None], ex / ex.sum(1, keepdims=True), 0.0)
    there = ids >= 0
    q = np.where(there, np.take_along_axis(p, np.maximum(ids, 0), 1), 0.0)
    if normalize:
        s = q.sum(1, keepdims=True)
        q = np.where(s > 0, q / np.where(s > 0, s, 1.0), 0.0)
    w = scale * np.where(there, q * np.where(there, dw, 0.0), 0.0).sum()
    balance = e * (counts / (k * n) * (p.sum(0) / n)).sum()
    return w + dl[0] * balance + dl[1] * (lse[alive] ** 2).sum() / n


def grad_ref(l, mask, ids, counts, live, dw, dl, k, normalize, scale):
    t, e = l.shape
    l = np.where(mask[:, None] != 0, l.astype(np.float64), -np.inf)
    alive = np.isfinite(l).any(1)
    n = max(live, 1)
    with np.errstate(all="ignore"):
        mx = np.where(alive, l.max(1), 0.0)
        ex = np.exp(l - mx[:, None])
        lse = np.where(alive, mx + np.log(ex.sum(1)), 0.0)
        p = np.where(alive[:, None], ex / ex.sum(1, keepdims=True), 0.0)
    g = np.tile(dl[0] * e * counts / (k * n * n), (t, 1))
    add = np.zeros((t, e))
    for i in range(t):
        at = ids[i][ids[i] >= 0]
        d = scale * dw[i][ids[i] >= 0]
        if not len(at):
            continue
        if normalize:
            q = p[i, at] / p[i, at].sum()
            add[i, at] += q * (d - (q * d).sum())
        else:
            g[i, at] += d
    return add + p * (g - (p * g).sum(1, keepdims=True)) + p * (2 * dl[1] * lse / n)[:, None]


GRADS = [
    (1, 256, 8, "f32", True, 0.0, 0.0),
    (5, 1, 1, "f32", False, 0.0, 0.0),
    (33, 33, 3, "bf16", False, 0.2, 0.2),
    (64, 7, 7, "fp16", True, 0.0, 0.5),
    (257, 100, 8, "f32", False, 0.1, 0.0),
    (40, 1024, 32, "f32", True, 0.1, 0.1),
    (1500, 64, 2, "bf16", True, 0.1, 0.0),
]


@pytest.mark.parametrize("with_dw,with_dl", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("t,e,k,kind,normalize,pad,closed", GRADS)
def test_route_grad(gg, t, e, k, kind, normalize, pad, closed, with_dw, with_dl):
    torch = _torch()
    logits, mask = make_logits(torch, kind, t, e, 3 * t + e, pad, closed)
    logits[mask == 0] = math.nan  # nothing of a padding token is used
    scale = 1.0 if normalize else 1.5
    r = Route(gg, torch, kind, logits, mask, k, normalize, scale)
    o = r.run()
    rng = np.random.RandomState(t)
    dw = rng.randn(t, k).astype(np.float32)
    dw[o["ids"] < 0] = np.nan  # not read
    dl = np.array([0.3, 0.02], np.float32)
    dwt, dlt = torch.from_numpy(dw).cuda(), torch.from_numpy(dl).cuda()
    out = Guarded(torch, (t, e), logits.dtype)
    b = gg.make_b200_backend()
    why = b.prepare_route_grad(_type(gg, kind), t, e, k, logits.data_ptr(), out.ptr(), ids_ptr=r.out["ids"].ptr(), lse_ptr=r.out["lse"].ptr(),
                               counts_ptr=r.out["counts"].ptr(), live_ptr=r.out["live"].ptr(), mask_ptr=mask.data_ptr(),
                               dweights_ptr=dwt.data_ptr() if with_dw else 0, dlosses_ptr=dlt.data_ptr() if with_dl else 0,
                               normalize=normalize, scale=scale)
    assert why == "", why
    s = torch.cuda.current_stream().cuda_stream
    b.run(s)
    assert b.device_status(s) == 0
    out.check(torch)
    got = out.t.float().cpu().numpy().astype(np.float64)
    l = logits.float().cpu().numpy().astype(np.float64)
    m = mask.cpu().numpy()
    l[m == 0] = 0.0
    dw64 = np.where(o["ids"] >= 0, dw, 0.0).astype(np.float64) * with_dw
    dl64 = dl.astype(np.float64) * with_dl
    args = (m, o["ids"], o["counts"], int(o["live"][0]), dw64, dl64, k, normalize, scale)
    ref = grad_ref(l, *args)
    n = max(int(o["live"][0]), 1)
    # every addend is a probability times at most this; each product and sum of them rounds, exp as in the header
    size = scale * np.abs(dw64).sum(1) + dl64[0] * e * o["counts"].max(initial=0) / (k * n * n) + 2 * dl64[1] * np.abs(
        np.where(np.isfinite(o["lse"]), o["lse"], 0)) / n
    close(got, ref, 512 * U * size[:, None] + HALF_ULP[kind] * np.abs(ref) + TINY[kind])
    if not (with_dw or with_dl):
        assert (got == 0).all()
    # against central differences of the objective, in some places (choices and counts fixed)
    eps = 1e-5
    for _ in range(12):
        i, j = rng.randint(t), rng.randint(e)
        if not np.isfinite(l[i, j]) or m[i] == 0:
            assert got[i, j] == 0
            continue
        up, down = l.copy(), l.copy()
        up[i, j] += eps
        down[i, j] -= eps
        d = (objective(up, *args) - objective(down, *args)) / (2 * eps)
        # second-order error of the difference: eps^2 times a third derivative of the same size, rounding 2^-52 |f| / eps
        f = abs(objective(l, *args)) + np.abs(dw64).sum() + 1
        assert abs(got[i, j] - d) <= 512 * U * size[i] + HALF_ULP[kind] * abs(d) + TINY[kind] + eps * eps * size[i] * 8 + 2.0 ** -50 * f / eps


def test_route_grad_reports_bad_ids(gg):
    torch = _torch()
    t, e, k = 20, 8, 2
    logits, mask = make_logits(torch, "f32", t, e, 1)
    r = Route(gg, torch, "f32", logits, mask, k, True)
    r.run()
    ids = r.out["ids"].t
    ids[4, 1] = 9
    out, dw = Guarded(torch, (t, e), torch.float32), torch.ones(t, k, device="cuda")
    b = gg.make_b200_backend()
    assert b.prepare_route_grad(gg.F32, t, e, k, logits.data_ptr(), out.ptr(), r.out["ids"].ptr(), r.out["lse"].ptr(),
                                r.out["counts"].ptr(), r.out["live"].ptr(), dweights_ptr=dw.data_ptr()) == ""
    s = torch.cuda.current_stream().cuda_stream
    b.run(s)
    assert b.device_status(s) == 0x2013
    assert b.device_status(s) == 0  # read and cleared
    out.check(torch)


# ---- dispatch / combine ------------------------------------------------------------------------------


def make_slots(torch, t, k, e, seed, dead=0.0, none=0.0):
    """dest, src, offsets of random distinct choices; `dead` tokens have none, `none` of the other slots are -1."""
    rng = np.random.RandomState(seed)
    ids = np.argsort(rng.rand(t, e), axis=1)[:, :k] if t else np.zeros((0, k), int)
    ids[rng.rand(t, k) < none] = -1
    ids[rng.rand(t) < dead] = -1
    flat = ids.ravel()
    counts = np.bincount(flat[flat >= 0], minlength=e)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    order = np.argsort(np.where(flat < 0, e, flat), kind="stable")
    total = int(counts.sum())
    dest = np.full(flat.size, -1)
    dest[order[:total]] = np.arange(total)
    src = np.where(np.arange(flat.size) < total, order, -1)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    return dict(dest=i32(dest.reshape(t, k)), src=i32(src), offsets=i32(offsets), total=total, dest_np=dest.reshape(t, k), src_np=src,
                offsets_np=offsets)


MOVES = [
    # tokens, top_k, experts, hidden, type, dead, none
    (1, 1, 1, 8, "bf16", 0.0, 0.0),
    (1, 8, 256, 7168, "bf16", 0.0, 0.0),
    (3, 2, 5, 136, "fp16", 0.0, 0.4),
    (64, 4, 32, 7168, "fp16", 0.0, 0.0),
    (333, 32, 40, 40, "bf16", 0.2, 0.1),
    (999, 2, 16, 2880, "bf16", 0.1, 0.0),
    (40, 3, 8, 4104, "fp16", 1.0, 0.0),
    (5000, 6, 64, 264, "bf16", 0.05, 0.05),
    (70, 7, 9, 20000, "fp16", 0.0, 0.1),
]


@pytest.mark.parametrize("t,k,e,h,kind,dead,none", MOVES)
def test_dispatch_combine(gg, t, k, e, h, kind, dead, none):
    torch = _torch()
    dt, ty = _dtype(torch, kind), _type(gg, kind)
    s = make_slots(torch, t, k, e, t + h, dead, none)
    stream = torch.cuda.current_stream().cuda_stream
    g = torch.Generator(device="cuda").manual_seed(t)
    x = torch.randn(t, h, generator=g, device="cuda").to(dt)
    x[(s["dest"] < 0).all(1)] = math.nan  # a token without experts goes nowhere
    total, d = s["total"], s["dest"].long()
    used = d >= 0

    rows = Guarded(torch, (t * k, h), dt)
    b = gg.make_b200_backend()
    assert b.prepare_dispatch(ty, t, k, e, h, x.data_ptr(), s["dest"].data_ptr(), s["offsets"].data_ptr(), rows.ptr()) == ""
    b.run(stream)
    assert b.device_status(stream) == 0
    rows.check(torch)
    want = torch.zeros(t * k, h, dtype=dt, device="cuda")
    for j in range(k):
        want[d[used[:, j], j]] = x[used[:, j]]
    assert torch.equal(rows.t, want)

    ye = torch.randn(t * k, h, generator=g, device="cuda").to(dt)
    ye[total:] = math.nan  # rows without a slot are not read
    w = torch.randn(t, k, generator=g, device="cuda")
    w[~used] = math.nan  # nor weights without a row
    for weights in (w, None):
        y = Guarded(torch, (t, h), dt)
        assert b.prepare_combine(ty, t, k, e, h, ye.data_ptr(), s["dest"].data_ptr(), y.ptr(),
                                 weights_ptr=0 if weights is None else weights.data_ptr()) == ""
        b.run(stream)
        assert b.device_status(stream) == 0
        y.check(torch)
        ref = torch.zeros(t, h, dtype=torch.float64, device="cuda")
        mag = torch.zeros_like(ref)
        for j in range(k):
            at = used[:, j]
            term = ye[d[at, j]].double() * (weights[at, j, None].double() if weights is not None else 1.0)
            ref[at] += term
            mag[at] += term.abs()
        tol = (k + 1) * U * mag + HALF_ULP[kind] * (ref.abs() + (k + 1) * U * mag) + TINY[kind]
        close(y.t.double().cpu().numpy(), ref.cpu().numpy(), tol.cpu().numpy())

    dy = torch.randn(t, h, generator=g, device="cuda").to(dt)
    dy[~used.any(1)] = math.nan
    for weights, want_dw in ((w, True), (None, True), (w, False)):
        drows, dw = Guarded(torch, (t * k, h), dt), Guarded(torch, (t, k), torch.float32)
        assert b.prepare_combine_grad(ty, t, k, e, h, dy.data_ptr(), ye.data_ptr() if want_dw else 0, s["dest"].data_ptr(),
                                      s["offsets"].data_ptr(), drows.ptr(), weights_ptr=0 if weights is None else weights.data_ptr(),
                                      dweights_ptr=dw.ptr() if want_dw else 0) == ""
        b.run(stream)
        assert b.device_status(stream) == 0
        drows.check(torch)
        dw.check(torch)
        ref = torch.zeros(t * k, h, dtype=torch.float64, device="cuda")
        dref = torch.zeros(t, k, dtype=torch.float64, device="cuda")
        dmag = torch.zeros(t, k, dtype=torch.float64, device="cuda")
        for j in range(k):
            at = used[:, j]
            ref[d[at, j]] = dy[at].double() * (weights[at, j, None].double() if weights is not None else 1.0)
            prod = dy[at].double() * ye[d[at, j]].double()
            dref[at, j] = prod.sum(1)
            dmag[at, j] = prod.abs().sum(1)
        close(drows.t.double().cpu().numpy(), ref.cpu().numpy(), ((HALF_ULP[kind] + 2 * U) * ref.abs() + TINY[kind]).cpu().numpy())
        if want_dw:
            close(dw.t.cpu().numpy(), dref.cpu().numpy(), (8 * -(-h // 2048) + 24) * U * dmag.cpu().numpy() + 1e-37)
    # differences: y is linear in the rows and in the weights, so a step of 1 gives the gradient itself
    if total:
        rng = np.random.RandomState(0)
        drows64, dy64 = drows.t.double().cpu().numpy(), dy.double().cpu().numpy()
        for _ in range(5):
            r, c = rng.randint(total), rng.randint(h)
            token, j = divmod(int(s["src_np"][r]), k)
            step = dy64[token, c] * float(w[token, j])  # (loss with rows[r, c] + 1) - (loss with rows[r, c])
            assert abs(drows64[r, c] - step) <= (HALF_ULP[kind] + 2 * U) * abs(step) + TINY[kind]


def test_permute_reports_bad_indices(gg):
    """dest and offsets out of range: reported, skipped, nothing written out of bounds."""
    torch = _torch()
    t, k, e, h = 30, 2, 4, 64
    stream = torch.cuda.current_stream().cuda_stream
    s = make_slots(torch, t, k, e, 3)
    x = torch.randn(t, h, device="cuda").bfloat16()
    ye = torch.randn(t * k, h, device="cuda").bfloat16()
    for bad in (t * k, 1 << 30, -2):
        dest = s["dest"].clone()
        dest[5, 1] = bad
        rows, y, dr, dw = (Guarded(torch, (t * k, h), torch.bfloat16), Guarded(torch, (t, h), torch.bfloat16),
                           Guarded(torch, (t * k, h), torch.bfloat16), Guarded(torch, (t, k), torch.float32))
        b = gg.make_b200_backend()
        for prepare in (lambda: b.prepare_dispatch(gg.BF16, t, k, e, h, x.data_ptr(), dest.data_ptr(), s["offsets"].data_ptr(), rows.ptr()),
                        lambda: b.prepare_combine(gg.BF16, t, k, e, h, ye.data_ptr(), dest.data_ptr(), y.ptr()),
                        lambda: b.prepare_combine_grad(gg.BF16, t, k, e, h, x.data_ptr(), ye.data_ptr(), dest.data_ptr(),
                                                       s["offsets"].data_ptr(), dr.ptr(), dweights_ptr=dw.ptr())):
            assert prepare() == ""
            b.run(stream)
            assert b.device_status(stream) == 0x2010
            assert "index out of range" in b.last_error()
        for v in (rows, y, dr, dw):
            v.check(torch)
    offsets = s["offsets"].clone()
    offsets[e] = t * k + 1
    assert b.prepare_dispatch(gg.BF16, t, k, e, h, x.data_ptr(), s["dest"].data_ptr(), offsets.data_ptr(), rows.ptr()) == ""
    b.run(stream)
    assert b.device_status(stream) == 0x2012
    rows.check(torch)


def test_rows_beyond_32_bit_offsets(gg):
    """More than 2^32 bytes and 2^31 elements of rows: the last rows arrive and come back."""
    torch = _torch()
    t, k, h = 38000, 8, 7168
    assert t * k * h > 1 << 31
    dest = torch.arange(t * k, dtype=torch.int32, device="cuda").view(t, k).flip(0).contiguous()
    offsets = torch.tensor([0, t * k], dtype=torch.int32, device="cuda")
    x = torch.randn(t, h, device="cuda").bfloat16()
    rows = torch.empty(t * k, h, dtype=torch.bfloat16, device="cuda")
    y = torch.empty_like(x)
    b, stream = gg.make_b200_backend(), torch.cuda.current_stream().cuda_stream
    assert b.prepare_dispatch(gg.BF16, t, k, 1, h, x.data_ptr(), dest.data_ptr(), offsets.data_ptr(), rows.data_ptr()) == ""
    b.run(stream)
    assert b.device_status(stream) == 0
    assert torch.equal(rows.view(t, k, h)[:, 3], x.flip(0))
    w = torch.full((t, k), 0.125, device="cuda")
    assert b.prepare_combine(gg.BF16, t, k, 1, h, rows.data_ptr(), dest.data_ptr(), y.data_ptr(), weights_ptr=w.data_ptr()) == ""
    b.run(stream)
    assert b.device_status(stream) == 0
    assert torch.equal(y, x)


# ---- 4-bit products -----------------------------------------------------------------------------------


def w4_ref(torch, q, scales, zeros, group, x):
    """x [r, k] in 64 bits times one expert's weights; the product and the sum of magnitudes."""
    n, half = q.shape
    w = torch.empty(n, 2 * half, dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = (q & 15).double(), (q >> 4).double()
    grow = lambda v: v.double().repeat_interleave(group, 1)[:, : 2 * half]  # noqa: E731
    w = (w - (grow(zeros & 15) if zeros is not None else 8.0)) * grow(scales)
    return x.double() @ w.t(), x.double().abs() @ w.abs().t()


W4 = [
    # rows of each expert, n, k, group, zeros, type, gather (top_k or 0), rows of no expert at the end
    ([1], 8, 32, 128, False, "bf16", 0, 0),
    ([0, 1, 0], 16, 64, 32, True, "fp16", 0, 0),
    ([1, 0, 2, 8], 40, 128, 128, False, "bf16", 2, 0),
    ([9, 16, 17, 0, 33, 1], 264, 384, 64, True, "bf16", 3, 2),
    ([5, 100], 72, 2880, 128, True, "fp16", 1, 3),
    ([7, 3], 2880, 2880, 64, False, "bf16", 0, 0),
    ([0, 0, 0], 64, 64, 32, False, "bf16", 0, 4),
    ([4, 31, 32, 64], 512, 384, 32, False, "fp16", 0, 1),
    ([1] * 8, 4096, 7168, 128, False, "bf16", 8, 0),
    ([2, 0, 11], 1000, 1056, 128, True, "bf16", 1, 0),
    ([3, 6], 136, 96, 64, True, "fp16", 0, 0),
    ([1 if i % 7 == 0 else 0 for i in range(1024)], 24, 160, 32, True, "bf16", 0, 0),
]


def w4_case(torch, counts, n, k, group, zeros, kind, top_k, extra, seed=1):
    e, rows = len(counts), sum(counts) + extra
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _dtype(torch, kind)
    c = dict(rows=rows, offsets=torch.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), device="cuda"))
    tokens = -(-rows // top_k) if top_k else rows
    c["tokens"], c["src"] = tokens, None
    c["x"] = torch.randn(max(tokens, 1), k, generator=g, device="cuda").to(dt)
    if top_k:
        src = torch.randperm(tokens * top_k, generator=g, device="cuda")[:rows].int()
        src[sum(counts):] = -1
        c["src"] = src
    c["q"] = torch.randint(0, 256, (e, n, k // 2), dtype=torch.uint8, generator=g, device="cuda")
    groups = -(-k // group)
    c["scales"] = (torch.rand(e, n, groups, generator=g, device="cuda") * 0.02 - 0.01).to(dt)
    c["zeros"] = torch.randint(0, 256, (e, n, groups), dtype=torch.uint8, generator=g, device="cuda") if zeros else None
    return c


def run_w4(gg, torch, c, counts, n, k, group, kind, top_k, status=0):
    out = Guarded(torch, (c["rows"], n), _dtype(torch, kind))
    b, stream = gg.make_b200_backend(), torch.cuda.current_stream().cuda_stream
    ptr = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
    why = b.prepare_w4(_type(gg, kind), len(counts), n, k, group, c["rows"], ptr(c["x"]), ptr(c["q"]), ptr(c["scales"]), ptr(c["offsets"]),
                       out.ptr(), zeros_ptr=ptr(c["zeros"]), src_ptr=ptr(c["src"]), tokens=c["tokens"], top_k=top_k or 1)
    assert why == "", why
    b.run(stream)
    assert b.device_status(stream) == status
    out.check(torch)
    return out, b


@pytest.mark.parametrize("counts,n,k,group,zeros,kind,top_k,extra", W4)
def test_w4(gg, counts, n, k, group, zeros, kind, top_k, extra):
    torch = _torch()
    c = w4_case(torch, counts, n, k, group, zeros, kind, top_k, extra)
    out, b = run_w4(gg, torch, c, counts, n, k, group, kind, top_k)
    at = 0
    for e, m in enumerate(counts):
        if not m:
            continue
        r = torch.arange(at, at + m, device="cuda")
        x = c["x"][c["src"][r].long() // top_k] if top_k else c["x"][r]
        ref, mag = w4_ref(torch, c["q"][e], c["scales"][e], c["zeros"][e] if zeros else None, group, x)
        tol = (k / 8 + 64) * 2 * U * mag
        tol = tol + HALF_ULP[kind] * (ref.abs() + tol) + TINY[kind]
        close(out.t[r].double().cpu().numpy(), ref.cpu().numpy(), tol.cpu().numpy())
        at += m
    assert (out.t[at:] == 0).all()
    first = out.t.clone()
    b.run(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(first.view(torch.int16), out.t.view(torch.int16))


@pytest.mark.parametrize("counts,n,k,group,zeros,kind", [
    ([1, 2, 0, 5, 1, 1, 1, 1], 8192, 7168, 128, False, "bf16"),  # units of 12 steps
    ([3] * 8, 4608, 4096, 64, True, "fp16"),
    ([17, 9, 30, 8], 1032, 4096, 128, True, "bf16"),  # work cut at any step
    ([33, 9, 30, 20], 776, 2048, 32, True, "fp16"),
    ([33, 9, 30, 20], 776, 2016, 32, True, "bf16"),
])
def test_w4_rows_of_groups_in_eights(gg, counts, n, k, group, zeros, kind):
    """Rows of scales in multiples of eight, and one that is not, with work that begins inside an eight."""
    test_w4(gg, counts, n, k, group, zeros, kind, 0, 0)


@pytest.mark.parametrize("group,zeros,kind", [(32, True, "bf16"), (64, False, "fp16"), (128, True, "bf16"), (128, False, "fp16")])
def test_w4_chunks_of_every_length(gg, group, zeros, kind):
    """Chunks of tokens that need one accumulator and chunks that need both, after one another and in either order; the last tile of
    256 weight rows is there in part of its first half only."""
    test_w4(gg, [40, 3, 70, 0, 33, 64, 16, 17, 130, 32, 1, 65, 48], 600, 1152, group, zeros, kind, 0, 2)


def test_w4_special_values(gg):
    """Infinities and NaN stay in their own row of x, and in their own weight row."""
    torch = _torch()
    counts, n, k, group = [3, 12], 48, 256, 128
    c = w4_case(torch, counts, n, k, group, False, "bf16", 0, 0)
    clean, _ = run_w4(gg, torch, c, counts, n, k, group, "bf16", 0)
    c["x"][4, 7] = math.nan
    c["x"][6, 100] = math.inf
    c["scales"][1, 5, 1] = math.nan
    got, _ = run_w4(gg, torch, c, counts, n, k, group, "bf16", 0)
    assert torch.isnan(got.t[4]).all()
    assert not torch.isfinite(got.t[6]).any()
    assert torch.isnan(got.t[3:, 5]).all()
    keep_r = [r for r in range(15) if r not in (4, 6)]
    keep_n = [i for i in range(n) if i != 5]
    assert torch.equal(got.t[keep_r][:, keep_n], clean.t[keep_r][:, keep_n])
    assert torch.equal(got.t[:3], clean.t[:3])


def test_w4_reports_bad_indices(gg):
    torch = _torch()
    counts, n, k, group = [3, 12], 48, 256, 128
    c = w4_case(torch, counts, n, k, group, False, "bf16", 2, 0)
    good, _ = run_w4(gg, torch, c, counts, n, k, group, "bf16", 2)
    for bad in (-1, c["tokens"] * 2, 1 << 30):
        src = c["src"].clone()
        src[4] = bad
        got, _ = run_w4(gg, torch, dict(c, src=src), counts, n, k, group, "bf16", 2, status=0x2011)
        keep = [r for r in range(15) if r != 4]
        assert torch.equal(got.t[keep], good.t[keep])
    for bad in ([0, 3, 16], [0, 16, 15], [-1, 3, 15], [0, 7, 3], [0, 3, 1 << 30]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        run_w4(gg, torch, dict(c, offsets=offsets), counts, n, k, group, "bf16", 2, status=0x2012)


def test_w4_weights_beyond_32_bit_offsets(gg):
    """More than 2^32 bytes of weights: an expert at their end."""
    torch = _torch()
    e, n, k, group = 300, 4096, 7168, 128
    assert e * n * k // 2 > 1 << 32
    counts = [0] * e
    counts[0], counts[e - 1] = 1, 2
    c = w4_case(torch, [1, 2], n, k, group, False, "bf16", 0, 0)
    q = torch.zeros(e, n, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(e, n, k // group, dtype=torch.bfloat16, device="cuda")
    q[0], q[e - 1], scales[0], scales[e - 1] = c["q"][0], c["q"][1], c["scales"][0], c["scales"][1]
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), device="cuda")
    small, _ = run_w4(gg, torch, c, [1, 2], n, k, group, "bf16", 0)
    large, _ = run_w4(gg, torch, dict(c, q=q, scales=scales, offsets=offsets), counts, n, k, group, "bf16", 0)
    assert torch.equal(small.t, large.t)


# ---- together --------------------------------------------------------------------------------------


def test_handle_changes_between_operators(gg, orc):
    """One handle: a grouped GEMM, then a layer operator, then the GEMM again."""
    torch = _torch()
    group_m, n, k = [256] * 4, 512, 384
    x, w = orc.make_inputs(group_m, n, k, gg.BF16)
    xd, wd = (torch.from_numpy(v.view(np.int16)).cuda() for v in (x, w))
    ref = orc.grouped_gemm_f32(x, w, group_m, gg.BF16)
    b, s = gg.make_b200_backend(), torch.cuda.current_stream().cuda_stream
    for _ in range(2):
        out = torch.zeros(sum(group_m), n, dtype=torch.int16, device="cuda")
        assert b.prepare(gg.BF16, group_m, n, k, xd.data_ptr(), wd.data_ptr(), out.data_ptr(), s) == ""
        b.run(s)
        assert b.device_status(s) == 0
        assert orc.check16(out.cpu().numpy().view(np.uint16), ref, gg.BF16)[0] == 0
        rows = torch.randn(16, 64, device="cuda").bfloat16()
        dest = torch.arange(16, dtype=torch.int32, device="cuda").view(8, 2)
        y = torch.empty(8, 64, dtype=torch.bfloat16, device="cuda")
        assert b.prepare_combine(gg.BF16, 8, 2, 4, 64, rows.data_ptr(), dest.data_ptr(), y.data_ptr(), stream=s) == ""
        assert "gg_combine" in b.detail()
        b.run(s)
        assert b.device_status(s) == 0
        want = rows.view(8, 2, 64).float().sum(1).bfloat16()
        assert torch.equal(y, want)
    b.release()
    with pytest.raises(gg.GGError):
        b.run(s)
