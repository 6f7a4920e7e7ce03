"""Arrays of more than 2^31 elements through the layer norm, its gradients, the rounding and the rows' kernels of the 8-bit products: some rows from each
end and the middle against plain implementations, as in test_gpu_norm_i8.py."""
import numpy as np
import pytest

from test_gpu_moe_ops import HALF_ULP, TINY, U, _torch, close
from test_gpu_norm_i8 import _np, grad_ref, norm_ref, quant_ref, run

pytestmark = pytest.mark.gpu


def large(torch, tokens, hidden, seed):
    """Rows that differ: one block of random ones, over and over with another factor each time."""
    x = torch.empty(tokens, hidden, dtype=torch.bfloat16, device="cuda")
    block = torch.randn(1000, hidden, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    for i in range(0, tokens, 1000):
        rows = x[i: i + 1000]
        rows.copy_(block[: rows.shape[0]] * (1 + 0.01 * (i // 1000)))
    return x


def test_norm_and_its_gradients(gg):
    torch = _torch()
    t, h = 132000, 16384
    assert t * h > 1 << 31
    at = [0, 1, t // 2, 131071, 131072, t - 1]  # 2^31 elements are 131072 rows
    x = large(torch, t, h, 1)
    gamma, beta = (torch.randn(h, device="cuda") for _ in range(2))
    y, q = torch.empty_like(x), torch.empty(t, h, dtype=torch.int8, device="cuda")
    mean, rstd, scales = (torch.empty(t, device="cuda") for _ in range(3))
    run(gg, torch, "norm", gg.BF16, t, h, x.data_ptr(), y.data_ptr(), gamma_ptr=gamma.data_ptr(), beta_ptr=beta.data_ptr(), param_type=gg.F32,
        mean_ptr=mean.data_ptr(), rstd_ptr=rstd.data_ptr(), q_ptr=q.data_ptr(), q_scales_ptr=scales.data_ptr())
    ref, m, r, t_y, t_m, t_r = norm_ref(_np(x[at]), _np(gamma), _np(beta), 1e-5)
    close(_np(mean[at]), m, t_m)
    close(_np(rstd[at]), r, t_r)
    close(_np(y[at]), ref, t_y + HALF_ULP["bf16"] * (np.abs(ref) + t_y) + TINY["bf16"])
    want, want_scales = quant_ref(y[at].float().cpu().numpy())
    assert np.array_equal(q[at].cpu().numpy(), want) and np.array_equal(scales[at].cpu().numpy(), want_scales)
    q.zero_()
    run(gg, torch, "quant", gg.BF16, t, h, y.data_ptr(), q.data_ptr(), scales.data_ptr())
    assert np.array_equal(q[at].cpu().numpy(), want) and np.array_equal(scales[at].cpu().numpy(), want_scales)
    del q
    dx = torch.empty_like(x)
    dgamma, dbeta = torch.empty(h, device="cuda"), torch.empty(h, device="cuda")
    run(gg, torch, "norm_grad", gg.BF16, t, h, x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), y.data_ptr(), dx.data_ptr(), gamma_ptr=gamma.data_ptr(),
        param_type=gg.F32, dsum_ptr=x.data_ptr(), dgamma_ptr=dgamma.data_ptr(), dbeta_ptr=dbeta.data_ptr())
    ref, tol, *_ = grad_ref(_np(x[at]), _np(y[at]), _np(mean[at]), _np(rstd[at]), _np(gamma), _np(x[at]))
    close(_np(dx[at]), ref, tol + HALF_ULP["bf16"] * (np.abs(ref) + tol) + TINY["bf16"])
    total, size = torch.zeros(h, dtype=torch.float64, device="cuda"), torch.zeros(h, dtype=torch.float64, device="cuda")
    for i in range(0, t, 4000):
        rows = y[i: i + 4000].double()
        total += rows.sum(0)
        size += rows.abs().sum(0)
    close(_np(dbeta), _np(total), (t // 148 + 48) * U * _np(size))


@pytest.mark.parametrize("by_token,eight", [(True, False), (True, True), (False, False), (False, True)])
def test_i8_rows(gg, by_token, eight):
    """Of 2 places a token, rounded or copied by tokens, and of one by places."""
    torch = _torch()
    top_k, k, n = (2 if by_token else 1), 16384, 8
    tokens = 134000 // top_k
    rows = tokens * top_k
    assert rows * k > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(5)
    x = large(torch, tokens, k, 2)
    qs = None
    if eight:
        x, qs = (x * 20).clamp(-127, 127).to(torch.int8), torch.rand(tokens, generator=g, device="cuda") + 0.1
    src = torch.randperm(rows, generator=g, device="cuda").int()
    offsets = torch.tensor([0, rows - 5000, rows], dtype=torch.int32, device="cuda")
    weight = torch.randint(-127, 128, (2, n, k), dtype=torch.int8, generator=g, device="cuda")
    scales = torch.rand(2, n, generator=g, device="cuda") * 1e-3
    out = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    run(gg, torch, "i8", gg.BF16, 2, n, k, rows, x.data_ptr(), weight.data_ptr(), scales.data_ptr(), offsets.data_ptr(), out.data_ptr(),
        x_scales_ptr=qs.data_ptr() if eight else 0, src_ptr=src.data_ptr(), tokens=tokens, top_k=top_k)
    for r in (0, rows // 3, 131071, 131072, rows - 5001, rows - 5000, rows - 1):
        token, e = int(src[r]) // top_k, int(r >= rows - 5000)
        if eight:
            q, s = x[token].double(), qs[token].double()
        else:
            q, s = (torch.from_numpy(v).cuda().double() for v in quant_ref(x[token: token + 1].float().cpu().numpy()))
        ref = ((q.view(1, -1) @ weight[e].double().t()) * s * scales[e].double()).view(-1)
        tol = 3 * U * ref.abs()
        close(_np(out[r]), _np(ref), _np(tol + HALF_ULP["bf16"] * (ref.abs() + tol) + TINY["bf16"]))


def test_i8_weights(gg):
    """The last expert's weights begin behind 2^31 elements."""
    torch = _torch()
    e, n, k = 80, 4096, 7168
    assert (e - 1) * n * k > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(6)
    weight = torch.randint(-127, 128, (e, n, k), dtype=torch.int8, generator=g, device="cuda")
    scales = torch.rand(e, n, generator=g, device="cuda") * 1e-3
    x, qs = torch.randint(-127, 128, (3 * e, k), dtype=torch.int8, generator=g, device="cuda"), torch.rand(3 * e, generator=g, device="cuda")
    offsets = torch.arange(0, 3 * e + 1, 3, dtype=torch.int32, device="cuda")
    out = torch.empty(3 * e, n, dtype=torch.float16, device="cuda")
    run(gg, torch, "i8", gg.FP16, e, n, k, 3 * e, x.data_ptr(), weight.data_ptr(), scales.data_ptr(), offsets.data_ptr(), out.data_ptr(), x_scales_ptr=qs.data_ptr())
    for i in (0, e // 2, e - 1):
        r = slice(3 * i, 3 * i + 3)
        ref = (x[r].double() @ weight[i].double().t()) * qs[r].double()[:, None] * scales[i].double()
        tol = 3 * U * ref.abs()
        close(_np(out[r]), _np(ref), _np(tol + HALF_ULP["fp16"] * (ref.abs() + tol) + TINY["fp16"]))
