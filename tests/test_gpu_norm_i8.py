"""The layer norm and its gradients, the rounding of rows to 8-bit integers and the 8-bit products against plain implementations of their
definitions in 64 bits, through the C ABI.

Whole numbers have to be equal. Tolerances for computed values, u = 2^-24 (one fp32 rounding), A = the row's mean magnitude:
  sums along a row   16 terms in a thread, 5 levels in a warp, 5 over the warps, the terms' own roundings: 48 u of the sum of magnitudes
  mean               48 u A
  rstd               half of var's relative error: 48 u of the sum of squares, and 2 * 48 u A / sigma from the means' errors
  y                  |gamma| rstd (mean's error + u |s - mean|) + |y - beta| (rstd's error + 4 u) + 2 u |y|
  dx                 rstd (48 u mean|d| + |c| 48 u mean|d c| + 6 u (|d| + |level| + |c along|)) + 2 u |dx|
  sums over tokens   a group's rows one after the other, up to 14 groups, 19 of a block's eighth, 8 warps, 4 of a term:
                     (tokens / 148 + 48) u of the sum of magnitudes
  8-bit products     the whole sum exact, then its rounding and two products: 3 u
and half a unit in the last place where the output has 16 bits (u where it has 32).
"""
import math

import numpy as np
import pytest

from test_gpu_moe_ops import HALF_ULP, TINY, U, Guarded, _dtype, _torch, _type, close

pytestmark = pytest.mark.gpu

f64 = np.float64


def _np(t):
    return t.double().cpu().numpy()


# ---- layer norm -----------------------------------------------------------------------------------


def rows_of(torch, g, tokens, hidden, kind, shift=0.3):
    """Rows of uneven size with a mean and a few large channels."""
    x = torch.randn(tokens, hidden, generator=g, device="cuda")
    x = x * torch.exp(0.5 * torch.randn(tokens, 1, generator=g, device="cuda")) + shift
    x[:, ::37] *= 6
    return x.to(_dtype(torch, kind))


def norm_ref(s, gamma, beta, eps):
    """y, mean, rstd in 64 bits and their tolerances before the output's rounding."""
    mean = s.mean(1, keepdims=True)
    var = ((s - mean) ** 2).mean(1, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    level = np.abs(s).mean(1, keepdims=True)
    t_mean = 48 * U * level
    r_rstd = 24 * U + 48 * U * level * rstd + 2 * U
    scaled = (s - mean) * rstd * gamma
    y = scaled + beta
    t_y = np.abs(gamma) * rstd * (t_mean + U * np.abs(s - mean)) + np.abs(scaled) * (r_rstd + 4 * U) + 2 * U * np.abs(y)
    return y, mean[:, 0], rstd[:, 0], t_y, t_mean[:, 0], (rstd * r_rstd)[:, 0]


def run(gg, torch, op, *args, status=0, **kw):
    b, stream = gg.make_b200_backend(), torch.cuda.current_stream().cuda_stream
    why = getattr(b, "prepare_" + op)(*args, stream=stream, **kw)
    assert why == "", why
    b.run(stream)
    assert b.device_status(stream) == status
    return b


NORM = [
    # tokens, hidden, type, parameters' type, residual, 8-bit rows
    (1, 8, "bf16", "bf16", False, False),
    (1, 7168, "bf16", "bf16", True, True),
    (3, 64, "fp16", "f32", False, True),
    (7, 256, "f32", "f32", True, False),
    (33, 264, "bf16", "f32", True, True),
    (1000, 2880, "fp16", "f32", False, False),
    (149, 4096, "f32", "f32", True, True),
    (300, 4104, "bf16", "bf16", False, True),
    (2000, 1032, "fp16", "fp16", True, False),
    (5000, 72, "bf16", "bf16", True, True),
    (700, 8192, "bf16", "bf16", True, False),
    (310, 8200, "fp16", "f32", True, True),
    (160, 16384, "bf16", "bf16", False, False),
    (160, 16384, "f32", "f32", True, True),
    (1100, 7168, "bf16", "bf16", True, True),
    (900, 5120, "fp16", "f32", False, True),
    (400, 9216, "bf16", "f32", False, True),
    (3000, 1024, "f32", "f32", False, True),
]


@pytest.mark.parametrize("tokens,hidden,kind,params,residual,q", NORM)
def test_norm(gg, tokens, hidden, kind, params, residual, q):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(tokens + hidden)
    dt, pt = _dtype(torch, kind), _dtype(torch, params)
    x = rows_of(torch, g, tokens, hidden, kind)
    res = rows_of(torch, g, tokens, hidden, kind, -0.1) if residual else None
    gamma = (1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")).to(pt)
    beta = (0.2 * torch.randn(hidden, generator=g, device="cuda")).to(pt)
    y, total = Guarded(torch, (tokens, hidden), dt), Guarded(torch, (tokens, hidden), dt)
    mean, rstd, scales = (Guarded(torch, (tokens,), torch.float32) for _ in range(3))
    rows = Guarded(torch, (tokens, hidden), torch.int8)
    b = run(gg, torch, "norm", _type(gg, kind), tokens, hidden, x.data_ptr(), y.ptr(), gamma_ptr=gamma.data_ptr(), beta_ptr=beta.data_ptr(),
            param_type=_type(gg, params), residual_ptr=res.data_ptr() if residual else 0, sum_ptr=total.ptr() if residual else 0,
            mean_ptr=mean.ptr(), rstd_ptr=rstd.ptr(), q_ptr=rows.ptr() if q else 0, q_scales_ptr=scales.ptr() if q else 0, eps=1e-5)
    s = x
    if residual:
        s = (x.float() + res.float()).to(dt)
        assert torch.equal(total.t, s)
    ref, m, r, t_y, t_m, t_r = norm_ref(_np(s), _np(gamma), _np(beta), 1e-5)
    close(_np(mean.t), m, t_m)
    close(_np(rstd.t), r, t_r)
    close(_np(y.t), ref, t_y + HALF_ULP[kind] * (np.abs(ref) + t_y) + TINY[kind])
    if q:
        want, want_scales = quant_ref(y.t.float().cpu().numpy())
        assert np.array_equal(scales.t.cpu().numpy(), want_scales)
        assert np.array_equal(rows.t.cpu().numpy(), want)
    for o in (y, total, mean, rstd, scales, rows):
        o.check(torch)
    first = y.t.clone()
    b.run(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(first.view(torch.uint8), y.t.view(torch.uint8))


def test_norm_without_parameters_and_only_8_bit_rows(gg):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(5)
    x = rows_of(torch, g, 37, 512, "fp16")
    y = torch.empty_like(x)
    run(gg, torch, "norm", gg.FP16, 37, 512, x.data_ptr(), y.data_ptr())
    ref, _, _, t_y, _, _ = norm_ref(_np(x), f64(1.0), f64(0.0), 1e-5)
    close(_np(y), ref, t_y + HALF_ULP["fp16"] * (np.abs(ref) + t_y) + TINY["fp16"])
    q, scales = torch.empty(37, 512, dtype=torch.int8, device="cuda"), torch.empty(37, device="cuda")
    run(gg, torch, "norm", gg.FP16, 37, 512, x.data_ptr(), q_ptr=q.data_ptr(), q_scales_ptr=scales.data_ptr())
    want, want_scales = quant_ref(y.float().cpu().numpy())
    assert np.array_equal(q.cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), want_scales)


@pytest.mark.parametrize("hidden,kind", [(1024, "bf16"), (7168, "f32"), (16384, "bf16"), (2880, "f32")])
def test_norm_of_rows_whose_squares_pass_fp32(gg, hidden, kind):
    """Squares around the mean beyond fp32's largest value count as infinite wherever in the row they are: rstd is 0 and y the bias."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(hidden)
    dt = _dtype(torch, kind)
    x = rows_of(torch, g, 6, hidden, kind)
    x[1, hidden // 2:] = 1e25
    x[2, : hidden // 2] = -1e25
    x[3, hidden // 3] = 1e30
    x[4, 256:512] = torch.tensor([1e25, -1e25], device="cuda").repeat(128).to(dt)
    beta = torch.randn(hidden, generator=g, device="cuda").to(dt)
    y, rstd = torch.empty_like(x), torch.empty(6, device="cuda")
    run(gg, torch, "norm", _type(gg, kind), 6, hidden, x.data_ptr(), y.data_ptr(), beta_ptr=beta.data_ptr(), param_type=_type(gg, kind),
        rstd_ptr=rstd.data_ptr())
    assert (rstd[1:5] == 0).all() and (rstd[[0, 5]] > 0).all()
    assert torch.equal(y[1:5], beta.expand(4, hidden))


@pytest.mark.parametrize("hidden,kind,params,q", [(64, "bf16", "bf16", False), (4096, "fp16", "f32", True), (16384, "bf16", "bf16", False),
                                                  (16384, "f32", "f32", True), (8200, "bf16", "f32", False)])
@pytest.mark.parametrize("which", ["gamma", "beta"])
def test_norm_with_one_parameter(gg, hidden, kind, params, q, which):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(hidden)
    x = rows_of(torch, g, 150, hidden, kind)
    v = (1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")).to(_dtype(torch, params))
    y, rows, scales = torch.empty_like(x), torch.empty(150, hidden, dtype=torch.int8, device="cuda"), torch.empty(150, device="cuda")
    run(gg, torch, "norm", _type(gg, kind), 150, hidden, x.data_ptr(), y.data_ptr(), param_type=_type(gg, params), q_ptr=rows.data_ptr() if q else 0,
        q_scales_ptr=scales.data_ptr() if q else 0, **{which + "_ptr": v.data_ptr()})
    ref, _, _, t_y, _, _ = norm_ref(_np(x), _np(v) if which == "gamma" else f64(1.0), _np(v) if which == "beta" else f64(0.0), 1e-5)
    close(_np(y), ref, t_y + HALF_ULP[kind] * (np.abs(ref) + t_y) + TINY[kind])
    if q:
        want, want_scales = quant_ref(y.float().cpu().numpy())
        assert np.array_equal(rows.cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), want_scales)


def test_norm_far_mean_equal_rows_and_special_values(gg):
    """A mean far above the spread costs no more than its own rounding; rows of one value give beta; NaN and infinities stay in their row."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(6)
    h = 3000
    x = 1000 + torch.randn(40, h, generator=g, device="cuda")
    beta = torch.randn(h, generator=g, device="cuda")
    x[3], x[4], x[5] = 2.5, 0.0, -7.0
    y = torch.empty_like(x)
    args = dict(beta_ptr=beta.data_ptr(), eps=1e-5)
    run(gg, torch, "norm", gg.F32, 40, h, x.data_ptr(), y.data_ptr(), **args)
    ref, _, _, t_y, _, _ = norm_ref(_np(x), f64(1.0), _np(beta), 1e-5)
    close(_np(y), ref, t_y)
    clean = y.clone()
    x[7, 11], x[9, 2999], x[12, 0] = math.nan, math.inf, -math.inf
    run(gg, torch, "norm", gg.F32, 40, h, x.data_ptr(), y.data_ptr(), **args)
    for r in range(40):
        if r in (7, 9, 12):
            assert torch.isnan(y[r]).any()
        else:
            assert torch.equal(y[r], clean[r])


@pytest.mark.parametrize("into", ["x", "residual"])
def test_norm_in_place(gg, into):
    """The sum over one of its terms, or the result over the input, as the header allows."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(8)
    x, res = rows_of(torch, g, 1500, 1024, "bf16"), rows_of(torch, g, 1500, 1024, "bf16")
    want, y0 = (x.float() + res.float()).bfloat16(), torch.empty_like(x)
    run(gg, torch, "norm", gg.BF16, 1500, 1024, want.data_ptr(), y0.data_ptr())
    a, b, y = x.clone(), res.clone(), torch.empty_like(x)
    target = a if into == "x" else b
    run(gg, torch, "norm", gg.BF16, 1500, 1024, a.data_ptr(), y.data_ptr(), residual_ptr=b.data_ptr(), sum_ptr=target.data_ptr())
    assert torch.equal(target, want) and torch.equal(y, y0)
    run(gg, torch, "norm", gg.BF16, 1500, 1024, want.data_ptr(), want.data_ptr())
    assert torch.equal(want, y0)


@pytest.mark.parametrize("hidden", [64, 520, 7168])
def test_norm_of_rows_of_one_value_is_beta(gg, hidden):
    """Whatever the value (small whole numbers: their sums are exact), to the last bit."""
    torch = _torch()
    x = torch.arange(-40, 40, device="cuda").float()[:, None].expand(80, hidden).bfloat16().contiguous()
    beta = torch.randn(hidden, device="cuda").bfloat16()
    y, mean = torch.empty_like(x), torch.empty(80, device="cuda")
    run(gg, torch, "norm", gg.BF16, 80, hidden, x.data_ptr(), y.data_ptr(), beta_ptr=beta.data_ptr(), mean_ptr=mean.data_ptr())
    assert torch.equal(mean, x[:, 0].float()) and torch.equal(y, beta.expand(80, hidden))


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_norm_residual_sums_of_any_values(gg, kind):
    """The sum is the terms' sum in 32 bits, rounded, for every pair of exponents, subnormal, infinite and NaN values among them."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(17)
    dt = _dtype(torch, kind)
    bits = lambda: torch.randint(-2 ** 15, 2 ** 15, (700, 2880), generator=g, device="cuda").to(torch.int16).view(dt)  # noqa: E731
    x, res = bits(), bits()
    res[350:] = (-x[350:].float() * (1 + 2.0 ** -9 * torch.randn(350, 2880, generator=g, device="cuda"))).to(dt)  # near cancellation
    total, y = torch.empty_like(x), torch.empty_like(x)
    run(gg, torch, "norm", _type(gg, kind), 700, 2880, x.data_ptr(), y.data_ptr(), residual_ptr=res.data_ptr(), sum_ptr=total.data_ptr())
    want = (x.float() + res.float()).to(dt)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(total), nan)
    assert torch.equal(total[~nan].view(torch.int16), want[~nan].view(torch.int16))


def test_no_tokens(gg):
    torch = _torch()
    run(gg, torch, "norm", gg.BF16, 0, 64, 0, 0)
    dg, db = (torch.full((64,), 3.0, device="cuda") for _ in range(2))
    run(gg, torch, "norm_grad", gg.BF16, 0, 64, 0, 0, 0, 0, 0, dgamma_ptr=dg.data_ptr(), dbeta_ptr=db.data_ptr())
    assert not dg.any() and not db.any()
    run(gg, torch, "quant", gg.BF16, 0, 64, 0, 0, 0)


NORM_GRAD = [
    # tokens, hidden, type, parameters' type, dsum
    (1, 8, "bf16", "bf16", False),
    (1, 7168, "fp16", "f32", True),
    (5, 64, "f32", "f32", True),
    (1000, 2880, "fp16", "f32", False),
    (449, 4096, "f32", "f32", True),
    (3001, 72, "bf16", "bf16", True),
    (2222, 520, "fp16", "fp16", False),
    (700, 4104, "bf16", "bf16", True),
    (400, 8192, "bf16", "f32", True),
    (333, 8200, "fp16", "fp16", False),
    (160, 16384, "bf16", "bf16", True),
    (151, 16384, "f32", "f32", True),
]


def grad_ref(x, dy, mean, rstd, gamma, dsum):
    mean, rstd = mean[:, None], rstd[:, None]
    c, d = (x - mean) * rstd, dy * gamma
    level, along = d.mean(1, keepdims=True), (d * c).mean(1, keepdims=True)
    dx = rstd * (d - level - c * along) + dsum
    m_d, m_dc = np.abs(d).mean(1, keepdims=True), np.abs(d * c).mean(1, keepdims=True)
    t = rstd * (48 * U * m_d + np.abs(c) * 48 * U * m_dc + 6 * U * (np.abs(d) + np.abs(level) + np.abs(c * along))) + 2 * U * (np.abs(dx) + np.abs(dsum))
    return dx, t, (dy * c).sum(0), np.abs(dy * c).sum(0), dy.sum(0), np.abs(dy).sum(0)


@pytest.mark.parametrize("tokens,hidden,kind,params,dsum", NORM_GRAD)
def test_norm_grad(gg, tokens, hidden, kind, params, dsum):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(tokens * 3 + hidden)
    dt = _dtype(torch, kind)
    x = rows_of(torch, g, tokens, hidden, kind)
    dy = torch.randn(tokens, hidden, generator=g, device="cuda").to(dt)
    more = torch.randn(tokens, hidden, generator=g, device="cuda").to(dt) if dsum else None
    gamma = (1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")).to(_dtype(torch, params))
    mean = x.float().mean(1)
    rstd = (x.float().var(1, unbiased=False) + 1e-5).rsqrt()
    dx = Guarded(torch, (tokens, hidden), dt)
    dgamma, dbeta = (Guarded(torch, (hidden,), torch.float32) for _ in range(2))
    args = (_type(gg, kind), tokens, hidden, x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dy.data_ptr())
    kw = dict(gamma_ptr=gamma.data_ptr(), param_type=_type(gg, params), dsum_ptr=more.data_ptr() if dsum else 0)
    b = run(gg, torch, "norm_grad", *args, dx.ptr(), dgamma_ptr=dgamma.ptr(), dbeta_ptr=dbeta.ptr(), **kw)
    ref, t, dg, a_dg, db, a_db = grad_ref(_np(x), _np(dy), _np(mean), _np(rstd), _np(gamma), _np(more) if dsum else f64(0.0))
    close(_np(dx.t), ref, t + HALF_ULP[kind] * (np.abs(ref) + t) + TINY[kind])
    many = (tokens // 148 + 48) * U
    close(_np(dgamma.t), dg, many * a_dg + 1e-37)
    close(_np(dbeta.t), db, many * a_db + 1e-37)
    for o in (dx, dgamma, dbeta):
        o.check(torch)
    first = [o.t.clone() for o in (dx, dgamma, dbeta)]
    b.run(torch.cuda.current_stream().cuda_stream)
    for o, w in zip((dx, dgamma, dbeta), first):
        assert torch.equal(o.t.view(torch.uint8), w.view(torch.uint8))
    # one of the sums, none of them, and the result over each of the inputs that it may take the place of
    again = torch.full((hidden,), 9.0, device="cuda")
    run(gg, torch, "norm_grad", *args, dx.ptr(), dbeta_ptr=again.data_ptr(), **kw)
    assert torch.equal(again, first[2])
    for over in [dy] + ([more] if dsum else []):
        keep = over.clone()
        run(gg, torch, "norm_grad", *args, over.data_ptr(), **kw)
        assert torch.equal(over.view(torch.uint8), first[0].view(torch.uint8))
        over.copy_(keep)


def test_norm_grad_against_differences(gg):
    """The kernel's gradients of sum(w y) against central differences of the norm's definition in 64 bits: differences are off by
    step^2 times a third derivative (below 1e-8 here) and by 64-bit cancellation (1e-16 / step), far below 1e-5 of the largest."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(11)
    t, h, eps, step = 4, 24, 1e-5, 1e-5
    x, w = (torch.randn(t, h, generator=g, device="cuda") for _ in range(2))
    gamma, beta = 1 + 0.3 * torch.randn(h, generator=g, device="cuda"), torch.randn(h, generator=g, device="cuda")
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd, dgamma, dbeta = (torch.empty(n, device="cuda") for n in (t, t, h, h))
    run(gg, torch, "norm", gg.F32, t, h, x.data_ptr(), y.data_ptr(), gamma_ptr=gamma.data_ptr(), beta_ptr=beta.data_ptr(), mean_ptr=mean.data_ptr(),
        rstd_ptr=rstd.data_ptr(), eps=eps)
    run(gg, torch, "norm_grad", gg.F32, t, h, x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), dx.data_ptr(), gamma_ptr=gamma.data_ptr(),
        dgamma_ptr=dgamma.data_ptr(), dbeta_ptr=dbeta.data_ptr())

    def loss(x, gamma, beta):
        return (norm_ref(x, gamma, beta, eps)[0] * _np(w)).sum()

    leaves = [_np(x), _np(gamma), _np(beta)]
    for i, got in enumerate((dx, dgamma, dbeta)):
        want = np.zeros_like(leaves[i])
        for at in np.ndindex(want.shape):
            both = []
            for sign in (1, -1):
                moved = [v.copy() for v in leaves]
                moved[i][at] += sign * step
                both.append(loss(*moved))
            want[at] = (both[0] - both[1]) / (2 * step)
        close(_np(got), want, 1e-5 * np.abs(want).max())


# ---- rounding to 8-bit integers -----------------------------------------------------------------------------------


def quant_ref(x):
    """By the definition; in 64 bits 127 x is exact and the quotient's error far below its distance from a half, unless it is one."""
    bad = ~np.isfinite(x).all(1)
    v = np.where(bad[:, None], 0, x)
    top = np.abs(v).max(1)
    with np.errstate(all="ignore"):
        scales = np.where(bad, np.float32(np.nan), (top.astype(np.float32) / np.float32(127)).astype(np.float32)).astype(np.float32)
    q = np.rint(v.astype(f64) * 127 / np.where(top > 0, top, 1).astype(f64)[:, None])
    return q.astype(np.int8), scales


@pytest.mark.parametrize("kind", ["bf16", "fp16", "f32"])
@pytest.mark.parametrize("rows,k", [(1, 8), (5, 64), (3, 4096), (700, 2880), (1300, 264), (2, 17000), (1, 131056)])
def test_quant(gg, kind, rows, k):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(rows + k)
    x = rows_of(torch, g, rows, k, kind, 0.0)
    q, scales = Guarded(torch, (rows, k), torch.int8), Guarded(torch, (rows,), torch.float32)
    run(gg, torch, "quant", _type(gg, kind), rows, k, x.data_ptr(), q.ptr(), scales.ptr())
    want, want_scales = quant_ref(x.float().cpu().numpy())
    assert np.array_equal(scales.t.cpu().numpy(), want_scales)
    assert np.array_equal(q.t.cpu().numpy(), want)
    q.check(torch)
    scales.check(torch)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "f32"])
def test_quant_halves_and_their_neighbours(gg, kind):
    """Rows whose largest value has an odd or even mantissa, and in them the values at each half, next below and next above, in the type."""
    torch = _torch()
    dt = _dtype(torch, kind)
    tops = torch.tensor([1.0, 2.0, 127.0, 254.0, 3.0, 1.2890625, 0.0078125, 100.0], device="cuda").to(dt)
    halves = (torch.arange(-127, 127, device="cuda").double() + 0.5) / 127
    near = (halves[None, :] * tops.double()[:, None]).to(dt)
    bits = near.view(torch.int32 if kind == "f32" else torch.int16)
    x = torch.cat([tops[:, None].expand(-1, 6), near, (bits + 1).view(dt), (bits - 1).view(dt)], 1)
    x = torch.minimum(torch.maximum(x, -tops[:, None]), tops[:, None]).contiguous()
    k = x.shape[1]
    assert k % 8 == 0
    q, scales = torch.empty(8, k, dtype=torch.int8, device="cuda"), torch.empty(8, device="cuda")
    run(gg, torch, "quant", _type(gg, kind), 8, k, x.data_ptr(), q.data_ptr(), scales.data_ptr())
    want, want_scales = quant_ref(x.float().cpu().numpy())
    assert np.array_equal(q.cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), want_scales)


@pytest.mark.parametrize("kind,bits,below", [("bf16", 7, 10), ("fp16", 10, 9)])
def test_quant_every_pair_of_mantissas(gg, kind, bits, below):
    """A row for each mantissa of its largest value, with every mantissa of smaller ones, from its own exponent down to what rounds to zero."""
    torch = _torch()
    m = torch.arange(1 << bits, 2 << bits, device="cuda").double()
    v = torch.cat([m * 2.0 ** -(bits + e) for e in range(below)])
    v = torch.where(torch.arange(v.numel(), device="cuda") % 2 == 0, v, -v)
    for scale in (1.0, 0.25):
        x = torch.where(v[None, :].abs() <= m[:, None] * 2.0 ** -bits, v[None, :], 0.0)
        x[:, 0] = m * 2.0 ** -bits
        x = (x * scale).to(_dtype(torch, kind))
        rows, k = x.shape
        q, scales = torch.empty(rows, k, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
        run(gg, torch, "quant", _type(gg, kind), rows, k, x.data_ptr(), q.data_ptr(), scales.data_ptr())
        want, want_scales = quant_ref(x.float().cpu().numpy())
        assert np.array_equal(q.cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), want_scales)


@pytest.mark.parametrize("kind,small", [("bf16", 2.0 ** -133), ("fp16", 2.0 ** -24), ("f32", 2.0 ** -149)])
def test_quant_extreme_rows(gg, kind, small):
    """Zeros, the type's smallest and largest values, NaN and infinities (in any place of a long row)."""
    torch = _torch()
    dt, k = _dtype(torch, kind), 17000
    torch.manual_seed(14)
    x = torch.zeros(7, k, device="cuda").to(dt)
    x[1, 3], x[1, 16999] = small * 5, -small * 2
    x[2] = torch.randn(k, device="cuda").clamp(-1, 1).double().mul(float(torch.finfo(dt).max) * 0.999).to(dt)
    x[3, 16998] = math.nan
    x[4, 0] = math.inf
    x[5, 9000] = -math.inf
    x[6] = torch.randn(k, device="cuda").double().mul(1e-37 if kind != "fp16" else 1e-5).to(dt)
    q, scales = torch.empty(7, k, dtype=torch.int8, device="cuda"), torch.empty(7, device="cuda")
    run(gg, torch, "quant", _type(gg, kind), 7, k, x.data_ptr(), q.data_ptr(), scales.data_ptr())
    want, want_scales = quant_ref(x.float().cpu().numpy())
    assert np.array_equal(q.cpu().numpy(), want)
    assert np.array_equal(scales.cpu().numpy(), want_scales, equal_nan=True)


# ---- 8-bit products -----------------------------------------------------------------------------------

I8 = [
    # rows of each expert, n, k, type, gather (top_k or 0), rows of no expert at the end, x in 8 bits
    ([1], 8, 16, "bf16", 0, 0, True),
    ([1], 8, 16, "bf16", 0, 0, False),
    ([0, 1, 0], 16, 64, "fp16", 0, 0, True),
    ([1, 0, 2, 8], 40, 128, "bf16", 2, 0, False),
    ([9, 16, 17, 0, 33, 1], 264, 384, "bf16", 3, 2, True),
    ([5, 100], 72, 2880, "fp16", 1, 3, False),
    ([7, 3], 2880, 2880, "bf16", 0, 0, True),
    ([0, 0, 0], 64, 64, "bf16", 0, 4, True),
    ([31, 32, 64, 65], 512, 384, "fp16", 0, 1, True),
    ([1] * 8, 4096, 7168, "bf16", 8, 0, False),
    ([2, 0, 11], 1000, 1040, "bf16", 1, 0, False),
    ([257, 600, 0, 255], 520, 272, "fp16", 2, 5, True),
    ([1 if i % 7 == 0 else 0 for i in range(1024)], 24, 160, "bf16", 0, 0, True),
    ([300], 1000, 2048, "fp16", 1, 0, False),
    ([1000, 513, 40, 770], 2880, 2880, "bf16", 2, 7, False),
    ([4096, 100, 3000], 512, 384, "bf16", 0, 0, True),
    ([20, 30], 256, 131056, "bf16", 0, 0, True),
    # items that are cut along k: narrow and wide chunks, all items and those of the last rounds, experts of uneven rows
    ([1] * 5, 4096, 7168, "fp16", 5, 0, False),
    ([1280], 4096, 7168, "bf16", 0, 0, True),
    ([1, 30, 0, 7, 64], 1032, 8192, "fp16", 1, 2, True),
    ([900, 0, 1300], 2056, 9216, "bf16", 2, 1, False),
    ([40], 8, 16384, "bf16", 0, 0, False),
    ([4000, 300], 136, 2064, "bf16", 33, 0, False),  # more places a token than are put in order by tokens
]


def i8_case(torch, counts, n, k, kind, top_k, extra, eight, seed=1):
    e, rows = len(counts), sum(counts) + extra
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(rows=rows, kind=kind, n=n, k=k, top_k=top_k, counts=counts,
             offsets=torch.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), device="cuda"))
    c["tokens"] = tokens = max(-(-rows // top_k) if top_k else rows, 1)
    c["src"] = None
    if top_k:
        src = torch.randperm(tokens * top_k, generator=g, device="cuda")[:rows].int()
        src[sum(counts):] = -1
        c["src"] = src
    if eight:
        c["x"] = torch.randint(-128, 128, (tokens, k), dtype=torch.int8, generator=g, device="cuda")
        c["x_scales"] = torch.rand(tokens, generator=g, device="cuda") * 0.02 + 0.001
        c["q"], c["qs"] = c["x"], c["x_scales"]
    else:
        c["x"], c["x_scales"] = rows_of(torch, g, tokens, k, kind, 0.0), None
        q, qs = quant_ref(c["x"].float().cpu().numpy())
        c["q"], c["qs"] = torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda()
    c["weight"] = torch.randint(-128, 128, (e, n, k), dtype=torch.int8, generator=g, device="cuda")
    c["scales"] = torch.rand(e, n, generator=g, device="cuda") * 2e-3 - 1e-3
    return c


def prepare_i8(gg, torch, c, out, b=None):
    b, stream = b or gg.make_b200_backend(), torch.cuda.current_stream().cuda_stream
    ptr = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
    why = b.prepare_i8(_type(gg, c["kind"]), len(c["counts"]), c["n"], c["k"], c["rows"], ptr(c["x"]), ptr(c["weight"]), ptr(c["scales"]),
                       ptr(c["offsets"]), out.data_ptr(), x_scales_ptr=ptr(c["x_scales"]), src_ptr=ptr(c["src"]), tokens=c["tokens"],
                       top_k=c["top_k"] or 1, stream=stream)
    assert why == "", why
    return b


def run_i8(gg, torch, c, status=0):
    out = Guarded(torch, (c["rows"], c["n"]), _dtype(torch, c["kind"]))
    b = prepare_i8(gg, torch, c, out.all)
    stream = torch.cuda.current_stream().cuda_stream
    b.run(stream)
    assert b.device_status(stream) == status
    out.check(torch)
    return out, b


def check_i8(torch, c, out):
    at, kind = 0, c["kind"]
    for e, m in enumerate(c["counts"]):
        if not m:
            continue
        r = torch.arange(at, at + m, device="cuda")
        token = c["src"][r].long() // c["top_k"] if c["top_k"] else r
        whole = c["q"][token].double() @ c["weight"][e].double().t()  # exact: below 2^53
        ref = whole * c["qs"][token].double()[:, None] * c["scales"][e].double()
        tol = 3 * U * ref.abs()
        tol = tol + HALF_ULP[kind] * (ref.abs() + tol) + TINY[kind]
        close(_np(out[r]), _np(ref), _np(tol))
        at += m
    assert (out[at:] == 0).all()


@pytest.mark.parametrize("counts,n,k,kind,top_k,extra,eight", I8)
def test_i8(gg, counts, n, k, kind, top_k, extra, eight):
    torch = _torch()
    c = i8_case(torch, counts, n, k, kind, top_k, extra, eight)
    out, b = run_i8(gg, torch, c)
    check_i8(torch, c, out.t)
    first = out.t.clone()
    for _ in range(3):
        b.run(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(first.view(torch.int16), out.t.view(torch.int16))


@pytest.mark.parametrize("kind,top_k,eight", [("bf16", 2, False), ("fp16", 2, True), ("bf16", 7, True), ("fp16", 32, False), ("bf16", 1, False)])
def test_i8_rows_by_tokens(gg, kind, top_k, eight):
    """Enough rows that each token is rounded once for all its places: with tokens that have none or some of them, and in further runs, whose
    routing the places of the run before do not fit: one that names slots twice, one with entries that are no slots."""
    torch = _torch()
    counts = [3000, 0, 1100, 77]
    c = i8_case(torch, counts, 264, 2064, kind, top_k, 300, eight)
    assert c["rows"] * c["k"] >= 1 << 23
    out, b = run_i8(gg, torch, c)
    check_i8(torch, c, out.t)
    stream = torch.cuda.current_stream().cuda_stream
    src = c["src"].clone()
    for change in ("other", "fewer", "twice", "bad"):
        if change == "other":
            c["src"].copy_(torch.randperm(c["tokens"] * top_k, device="cuda")[: c["rows"]].int())
        elif change == "fewer":
            c["counts"] = [500, 40, 0, 0]
            c["offsets"].copy_(torch.tensor([0, 500, 540, 540, 540], dtype=torch.int32))
            c["src"][540:] = -1
        elif change == "twice":
            c["counts"] = counts
            c["offsets"].copy_(torch.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)))
            c["src"].copy_(src)
            c["src"][5:4000:7] = c["src"][4:3999:7]
            c["src"][100:140] = c["src"][99]
        else:
            c["src"].copy_(src)
            c["src"][17], c["src"][3100] = -9, c["tokens"] * top_k
        out.t.fill_(3)
        b.run(stream)
        assert b.device_status(stream) == (0x2011 if change == "bad" else 0)
        if change == "bad":
            assert (out.t[17] == 0).all() and (out.t[3100] == 0).all()
            c["src"][17] = c["src"][3100] = 0  # what the reference takes for them is not compared
            keep = out.t.clone()
            ref_rows = torch.ones(c["rows"], dtype=torch.bool, device="cuda")
            ref_rows[17] = ref_rows[3100] = False
            c["src"].copy_(src)
            b.run(stream)
            torch.cuda.synchronize()
            assert torch.equal(out.t[ref_rows], keep[ref_rows])
        check_i8(torch, c, out.t)


@pytest.mark.parametrize("kind,eight", [("bf16", False), ("fp16", True)])
@pytest.mark.parametrize("more", [0.9, 2.3, 8])
def test_i8_rows_of_few_tokens(gg, kind, eight, more):
    """Rows of some of the slots only, as where other experts' rows are elsewhere: from more than two rows a token to a fraction of one."""
    torch = _torch()
    c = i8_case(torch, [2900, 0, 1201], 136, 2064, kind, 4, 33, eight)
    tokens, g = int(c["tokens"] * 2 * more), torch.Generator(device="cuda").manual_seed(11)
    pick = torch.randint(0, c["tokens"], (tokens,), generator=g, device="cuda")
    c["x"], c["q"], c["qs"] = c["x"][pick].contiguous(), c["q"][pick], c["qs"][pick].contiguous()
    c["x_scales"] = c["qs"] if eight else None
    c["tokens"] = tokens
    c["src"] = torch.randperm(4 * tokens, generator=g, device="cuda")[: c["rows"]].int()
    c["src"][-33:] = -1
    out, _ = run_i8(gg, torch, c)
    check_i8(torch, c, out.t)


def test_i8_largest_sums(gg):
    """All factors -128 at the longest k: the sum is 2^31 less one factor's share, and still exact."""
    torch = _torch()
    c = i8_case(torch, [3, 40], 264, 131056, "bf16", 0, 0, True)
    c["x"].fill_(-128)
    c["weight"].fill_(-128)
    c["weight"][:, 1::2] = 127
    out, _ = run_i8(gg, torch, c)
    check_i8(torch, c, out.t)


def test_i8_scales_of_any_size(gg):
    """Products with a very large and a very small scale, whose result is in range, and a row of zeros beside them."""
    torch = _torch()
    c = i8_case(torch, [3, 6], 40, 256, "bf16", 0, 0, True)
    c["x_scales"].fill_(1e36)
    c["scales"].fill_(-1e-36)
    c["x_scales"][4:] = 1e-37
    c["scales"][1] = 3e37
    c["x"][2] = 0
    c["x_scales"][2] = 3e38
    c["scales"][0, 5] = 3e38
    out, _ = run_i8(gg, torch, c)
    assert (out.t[2] == 0).all()
    ref = torch.cat([(c["x"][r].double() @ c["weight"][e].double().t()) * c["x_scales"][r].double()[:, None] * c["scales"][e].double()
                     for e, r in ((0, slice(0, 3)), (1, slice(3, 9)))])
    ok = ref.abs() < 3e38
    close(_np(out.t)[ok.cpu().numpy()], _np(ref[ok]), _np((3 * U + HALF_ULP["bf16"] * (1 + 3 * U)) * ref[ok].abs()) + TINY["bf16"])
    assert torch.isinf(out.t[~ok].float()).all()


def test_i8_special_values(gg):
    """NaN and infinities of a token stay in its rows, those of a weight row's scale in its column."""
    torch = _torch()
    c = i8_case(torch, [3, 12], 48, 256, "bf16", 0, 0, False)
    clean, _ = run_i8(gg, torch, c)
    c["x"][4, 7] = math.nan
    c["x"][6, 100] = math.inf
    c["scales"][1, 5] = math.nan
    out, _ = run_i8(gg, torch, c)
    assert torch.isnan(out.t[4]).all() and torch.isnan(out.t[6]).all() and torch.isnan(out.t[3:, 5]).all()
    rest = torch.ones(15, 48, dtype=torch.bool, device="cuda")
    rest[4] = rest[6] = False
    rest[3:, 5] = False
    assert torch.equal(out.t[rest], clean.t[rest])


@pytest.mark.parametrize("eight", [True, False])
def test_i8_bad_indices(gg, eight):
    """A src that is no slot gives a zero row and a report; offsets out of range are held to the rows; falling ones leave no rows."""
    torch = _torch()
    counts = [5, 0, 40, 3]
    c = i8_case(torch, counts, 520, 272, "bf16", 2, 4, eight)
    good, _ = run_i8(gg, torch, c)
    src, offsets = c["src"].clone(), c["offsets"].clone()
    for bad in (-7, c["tokens"] * 2, 2 ** 31 - 1, -2 ** 31):
        c["src"] = src.clone()
        c["src"][9] = bad
        out, _ = run_i8(gg, torch, c, status=0x2011)
        assert (out.t[9] == 0).all()
        keep = torch.arange(c["rows"], device="cuda") != 9
        assert torch.equal(out.t[keep], good.t[keep])
    c["src"] = src
    c["offsets"] = offsets.clone()
    c["offsets"][4] = c["rows"] + 1000
    out, _ = run_i8(gg, torch, c, status=0x2012)
    for places in ((1, 100), (2, 3), (0, 20)):
        c["offsets"] = offsets.clone()
        c["offsets"][places[0]] = places[1]
        out, _ = run_i8(gg, torch, c, status=0x2012)
        assert (out.t == 0).all()
    c["offsets"] = offsets.clone()
    c["offsets"][0] = 2  # the first two rows belong to no expert
    out, _ = run_i8(gg, torch, c)
    assert (out.t[:2] == 0).all() and torch.equal(out.t[2:], good.t[2:])


def test_i8_contents_change_between_runs(gg):
    """One prepared handle over routings from nothing to all rows on one expert, as the counts on the device say."""
    torch = _torch()
    e, rows = 16, 700
    c = i8_case(torch, [rows] + [0] * (e - 1), 776, 400, "bf16", 1, 0, False)
    out = torch.empty(rows, c["n"], dtype=torch.bfloat16, device="cuda")
    b, stream = prepare_i8(gg, torch, c, out), torch.cuda.current_stream().cuda_stream
    r = np.random.RandomState(3)
    for counts in ([rows] + [0] * (e - 1), [0] * e, [0] * (e - 1) + [1], list(r.multinomial(rows, r.dirichlet([0.3] * e))), [40] * e):
        c["counts"] = counts
        c["offsets"].copy_(torch.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)))
        c["src"].copy_(torch.randperm(rows, device="cuda").int())
        c["x"].copy_(rows_of(torch, torch.Generator(device="cuda").manual_seed(int(sum(counts[:3]))), rows, c["k"], "bf16", 0.0))
        q, qs = quant_ref(c["x"].float().cpu().numpy())
        c["q"], c["qs"] = torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda()
        out.fill_(7)
        b.run(stream)
        assert b.device_status(stream) == 0
        check_i8(torch, c, out)


def test_i8_other_stream_and_graph(gg):
    """On a stream of its own, and captured with the norm and the rounding before it and replayed on new contents."""
    torch = _torch()
    t, e, k, n = 50, 4, 1024, 264
    counts = [20, 0, 25, 5]
    c = i8_case(torch, counts, n, k, "bf16", 1, 0, False)
    rows, scales, y = torch.empty(t, k, dtype=torch.int8, device="cuda"), torch.empty(t, device="cuda"), torch.empty_like(c["x"])
    x = c["x"].clone()
    c.update(x=rows, x_scales=scales)
    out = torch.empty(t, n, dtype=torch.bfloat16, device="cuda")
    norm = gg.make_b200_backend()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert norm.prepare_norm(gg.BF16, t, k, x.data_ptr(), y.data_ptr(), q_ptr=rows.data_ptr(), q_scales_ptr=scales.data_ptr(),
                                 stream=side.cuda_stream) == ""
        b = prepare_i8(gg, torch, c, out)
        norm.run(side.cuda_stream)
        b.run(side.cuda_stream)
        side.synchronize()

        def check():
            q, qs = quant_ref(y.float().cpu().numpy())
            c["q"], c["qs"] = torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda()
            assert torch.equal(c["q"], rows)
            check_i8(torch, c, out)

        check()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            norm.run(side.cuda_stream)
            b.run(side.cuda_stream)
        for seed in (4, 5):
            x.copy_(rows_of(torch, torch.Generator(device="cuda").manual_seed(seed), t, k, "bf16"))
            graph.replay()
            side.synchronize()
            check()
    assert norm.device_status(side.cuda_stream) == 0 and b.device_status(side.cuda_stream) == 0


def test_i8_offsets_beyond_32_bits(gg):
    """An output of more than 2^31 elements: its last rows are right, and so is one in the middle."""
    torch = _torch()
    n, k, rows = 16384, 128, 140000
    assert n * rows > 1 << 31
    c = i8_case(torch, [rows - 60000, 60000], n, k, "bf16", 0, 0, True)
    out = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    b, stream = prepare_i8(gg, torch, c, out), torch.cuda.current_stream().cuda_stream
    b.run(stream)
    assert b.device_status(stream) == 0
    for r in (0, rows - 60001, rows - 60000, rows // 2, rows - 1):
        e = int(r >= rows - 60000)
        ref = (c["x"][r].double() @ c["weight"][e].double().t()) * c["x_scales"][r].double() * c["scales"][e].double()
        tol = 3 * U * ref.abs()
        close(_np(out[r]), _np(ref), _np(tol + HALF_ULP["bf16"] * (ref.abs() + tol) + TINY["bf16"]))


def test_a_handle_takes_one_operator_after_another(gg):
    """One handle prepared for each operator in turn, small and large, gives what a new one gives."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(2)
    b, stream = gg.make_b200_backend(), torch.cuda.current_stream().cuda_stream
    for h in (16384, 64, 2880):
        x, y = rows_of(torch, g, 200, h, "bf16"), torch.empty(200, h, dtype=torch.bfloat16, device="cuda")
        assert b.prepare_norm(gg.BF16, 200, h, x.data_ptr(), y.data_ptr(), stream=stream) == ""
        b.run(stream)
        ref, _, _, t_y, _, _ = norm_ref(_np(x), f64(1.0), f64(0.0), 1e-5)
        close(_np(y), ref, t_y + HALF_ULP["bf16"] * (np.abs(ref) + t_y) + TINY["bf16"])
        c = i8_case(torch, [3, h // 32], 136, 176, "fp16", 0, 0, False)
        out = torch.empty(c["rows"], 136, dtype=torch.float16, device="cuda")
        prepare_i8(gg, torch, c, out, b)
        b.run(stream)
        assert b.device_status(stream) == 0
        check_i8(torch, c, out)
