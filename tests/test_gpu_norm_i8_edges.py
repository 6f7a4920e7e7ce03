"""The layer norm and its gradients at the ends of fp32's range, against the definitions in 64 bits. Tolerances as derived in test_gpu_norm_i8.py
where nothing else is said."""
import re

import numpy as np
import pytest

from test_gpu_moe_ops import HALF_ULP, TINY, U, _dtype, _torch, _type, close
from test_gpu_norm_i8 import _np, grad_ref, norm_ref, quant_ref, rows_of, run

pytestmark = pytest.mark.gpu


def far_rows(torch, g, hidden, kind):
    """Rows whose squares around the mean pass fp32's largest value and whose sum does not, between ordinary ones (the first and the last): a value
    of 1e38 in the columns of the first warp, of one in the middle and of the last, and the first, middle or last columns at 3e34."""
    at = [0, 5, 37, hidden // 3, hidden // 2, hidden - 9, hidden - 1]
    x = rows_of(torch, g, 2 * len(at) + 5, hidden, kind)
    for i, col in enumerate(at):
        x[1 + i, col] = 1e38
        x[1 + len(at) + i, col] = -1e38
    some = max(8, min(1024, hidden // 4))
    x[-4, :some], x[-3, hidden // 2: hidden // 2 + some], x[-2, -some:] = 3e34, -3e34, 3e34
    return x


RANGE = [(64, "bf16", False), (1024, "bf16", False), (2880, "f32", True), (4096, "f32", False), (7168, "bf16", False), (7168, "bf16", True),
         (8200, "bf16", True), (16384, "bf16", False), (16384, "f32", True)]


@pytest.mark.parametrize("hidden,kind,q", RANGE)
def test_norm_of_far_values_wherever_they_are(gg, hidden, kind, q):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(hidden)
    dt = _dtype(torch, kind)
    x = far_rows(torch, g, hidden, kind)
    t = x.shape[0]
    gamma, beta = (1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")).to(dt), torch.randn(hidden, generator=g, device="cuda").to(dt)
    y, mean, rstd = torch.empty_like(x), torch.empty(t, device="cuda"), torch.empty(t, device="cuda")
    rows, scales = torch.empty(t, hidden, dtype=torch.int8, device="cuda"), torch.empty(t, device="cuda")
    run(gg, torch, "norm", _type(gg, kind), t, hidden, x.data_ptr(), y.data_ptr(), gamma_ptr=gamma.data_ptr(), beta_ptr=beta.data_ptr(),
        mean_ptr=mean.data_ptr(), rstd_ptr=rstd.data_ptr(), q_ptr=rows.data_ptr() if q else 0, q_scales_ptr=scales.data_ptr() if q else 0)
    ref, m, r, t_y, t_m, t_r = norm_ref(_np(x), _np(gamma), _np(beta), 1e-5)
    close(_np(mean), m, t_m)
    assert (rstd[1:-1] == 0).all()
    assert torch.equal(y[1:-1], beta.expand(t - 2, hidden))
    ends = [0, -1]
    close(_np(rstd)[ends], r[ends], t_r[ends])
    close(_np(y)[ends], ref[ends], (t_y + HALF_ULP[kind] * (np.abs(ref) + t_y) + TINY[kind])[ends])
    if q:
        want, want_scales = quant_ref(y.float().cpu().numpy())
        assert np.array_equal(rows.cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), want_scales)


@pytest.mark.parametrize("hidden", [64, 128])
def test_norm_of_a_value_further_from_the_mean_than_fp32_reaches(gg, hidden):
    """The type's lowest value and a mean above 0 whose difference passes fp32 (the sum, and those of its parts, do not)."""
    torch = _torch()
    low = torch.finfo(torch.bfloat16).min
    x = torch.zeros(3, hidden, device="cuda")
    x[0, 0], x[0, 1:8], x[0, 8:40:8] = low, 4e37, 4e37 * hidden / 64
    x[1:] = x[0].flip(0)
    x[2, 0] = 2e36
    x = x.bfloat16()
    s = _np(x)
    assert (s.sum(1) < 3e38).all() and (s.mean(1) - float(low) > 3.403e38).all()
    beta = torch.randn(hidden, device="cuda").bfloat16()
    y, mean, rstd = torch.empty_like(x), torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
    run(gg, torch, "norm", gg.BF16, 3, hidden, x.data_ptr(), y.data_ptr(), beta_ptr=beta.data_ptr(), mean_ptr=mean.data_ptr(), rstd_ptr=rstd.data_ptr())
    close(_np(mean), s.mean(1), 48 * U * np.abs(s).mean(1))
    assert not rstd.any() and torch.equal(y, beta.expand(3, hidden))


def detail(b, name):
    """A number of the handle's description, as in groups=2."""
    return int(re.search(name + r"=(\d+)", b.detail()).group(1))


def columns_of_warp(torch, w, warps, hidden, kind):
    """A mask of the columns whose sums a group's warp w forms: vectors of eight values, in turn over the group's threads; in fp32 four of them are
    in the row's second half."""
    col = torch.arange(hidden, device="cuda")
    vec = col % (hidden // 2) // 4 if kind == "f32" else col // 8
    return vec % (32 * warps) // 32 == w


@pytest.mark.parametrize("hidden,kind", [(16384, "bf16"), (4096, "f32"), (7168, "bf16")])
def test_norm_of_rows_whose_squares_are_just_in_range(gg, hidden, kind):
    """Squares around the row's mean within fp32, around the first warp's mean beyond it: rstd is that of the definition. The squares of up to 16
    warps are joined around the first one's mean: shares, products and sums 8 u, twice that and the shares' own for the squared distance to the
    mean, times 16 warps, half of it in rstd: 200 u; of y that and norm_ref's own."""
    torch = _torch()
    dt = _dtype(torch, kind)
    gamma = (1 + 0.3 * torch.randn(hidden, device="cuda")).to(dt)
    x = torch.zeros(4, hidden, dtype=dt, device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    args = (_type(gg, kind), 4, hidden, x.data_ptr(), y.data_ptr())
    kw = dict(gamma_ptr=gamma.data_ptr(), mean_ptr=mean.data_ptr(), rstd_ptr=rstd.data_ptr())
    warps = detail(run(gg, torch, "norm", *args, **kw), "warps")
    assert warps >= 8
    a = (0.5 * 3.4e38 * warps / (hidden * (1 - 1 / warps))) ** 0.5
    for r, (w, v) in enumerate(((0, a), (0, -a), (warps // 2, a), (warps - 1, -a))):
        x[r, columns_of_warp(torch, w, warps, hidden, kind)] = v
    run(gg, torch, "norm", *args, **kw)
    s = _np(x)
    assert (((s - s.mean(1, keepdims=True)) ** 2).sum(1) < 3.4e38).all() and hidden * (1 - 1 / warps) * a * a > 3.5e38
    ref, m, r, t_y, t_m, _ = norm_ref(s, _np(gamma), 0.0, 1e-5)
    close(_np(mean), m, t_m)
    close(_np(rstd), r, 200 * U * r)
    t_y = t_y + 200 * U * np.abs(ref)
    close(_np(y), ref, t_y + HALF_ULP[kind] * (np.abs(ref) + t_y) + TINY[kind])


@pytest.mark.parametrize("dsum", [False, True])
@pytest.mark.parametrize("hidden,kind,_", RANGE)
def test_norm_grad_of_rows_without_spread(gg, hidden, kind, _, dsum):
    """Rows whose squares pass fp32 have rstd 0: their dx is dsum to the last bit, they add nothing to dgamma, and the rows beside them are as ever."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(hidden + 1)
    dt = _dtype(torch, kind)
    x = far_rows(torch, g, hidden, kind)
    t = x.shape[0]
    dy, more = (torch.randn(t, hidden, generator=g, device="cuda").to(dt) for _ in range(2))
    gamma = (1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")).to(dt)
    y, mean, rstd = torch.empty_like(x), torch.empty(t, device="cuda"), torch.empty(t, device="cuda")
    run(gg, torch, "norm", _type(gg, kind), t, hidden, x.data_ptr(), y.data_ptr(), gamma_ptr=gamma.data_ptr(), mean_ptr=mean.data_ptr(),
        rstd_ptr=rstd.data_ptr())
    assert (rstd[1:-1] == 0).all() and torch.isfinite(mean).all()
    check_grad(gg, torch, kind, x, mean, rstd, gamma, dy, more if dsum else None)
    dx = torch.empty_like(x)
    run(gg, torch, "norm_grad", _type(gg, kind), t, hidden, x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), dx.data_ptr(),
        gamma_ptr=gamma.data_ptr(), dsum_ptr=more.data_ptr() if dsum else 0)
    assert torch.equal(dx[1:-1], more[1:-1] if dsum else torch.zeros_like(dx[1:-1]))


def check_grad(gg, torch, kind, x, mean, rstd, gamma, dy, more):
    t, hidden = x.shape
    dx = torch.empty_like(x)
    dgamma, dbeta = torch.empty(hidden, device="cuda"), torch.empty(hidden, device="cuda")
    run(gg, torch, "norm_grad", _type(gg, kind), t, hidden, x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), dx.data_ptr(),
        gamma_ptr=gamma.data_ptr(), dsum_ptr=more.data_ptr() if more is not None else 0, dgamma_ptr=dgamma.data_ptr(), dbeta_ptr=dbeta.data_ptr())
    ref, tol, dg, a_dg, db, a_db = grad_ref(_np(x), _np(dy), _np(mean), _np(rstd), _np(gamma), _np(more) if more is not None else 0.0)
    close(_np(dx), ref, tol + HALF_ULP[kind] * (np.abs(ref) + tol) + TINY[kind])
    many = (t // 148 + 48) * U
    close(_np(dgamma), dg, many * a_dg + 1e-37)
    close(_np(dbeta), db, many * a_db + 1e-37)


@pytest.mark.parametrize("hidden,kind", [(64, "bf16"), (1024, "f32"), (7168, "bf16"), (8200, "f32"), (16384, "bf16")])
def test_norm_grad_of_large_values_and_gradients(gg, hidden, kind):
    """Rows and gradients whose products pass fp32, which the gradient's own terms do not: rstd times a value is about 1."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(hidden + 2)
    dt = _dtype(torch, kind)
    x = (torch.randn(20, hidden, generator=g, device="cuda") * 1e14).to(dt)
    dy = (torch.randn(20, hidden, generator=g, device="cuda") * 1e28).to(dt)
    x[::2], dy[1::2] = rows_of(torch, g, 10, hidden, kind), torch.randn(10, hidden, generator=g, device="cuda").to(dt)
    x[::3], dy[::3] = (x[::3].float() * 1e-12).to(dt), (dy[::3].float() * 1e-12).to(dt)
    gamma = (1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")).to(dt)
    x[5], dy[5] = (torch.randn(hidden, generator=g, device="cuda") * 1e14).to(dt), (torch.randn(hidden, generator=g, device="cuda") * 1e28).to(dt)
    mean = x.double().mean(1).float()
    rstd = (x.double().var(1, unbiased=False) + 1e-5).rsqrt().float()
    check_grad(gg, torch, kind, x, mean, rstd, gamma, dy, None)
