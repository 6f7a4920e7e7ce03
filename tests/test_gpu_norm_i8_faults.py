"""Waits of the layer norm, its gradients and the 8-bit products that run out, without faulting the GPU: "test_stall" makes one barrier wait for an
arrival that never comes. The kernel records it after timeout_ms and returns; the same handle then gives what a new one gives."""
import time

import pytest

from test_gpu_moe_ops import _torch, _type
from test_gpu_norm_i8 import i8_case, prepare_i8, rows_of

pytestmark = pytest.mark.gpu


def stalls(gg, torch, prepare, outputs):
    """prepare(b): of a handle. Runs it with a wait that runs out, then as it should be, and a new handle."""
    stream = torch.cuda.current_stream().cuda_stream
    b, other = gg.make_b200_backend(), gg.make_b200_backend()
    b.set_option("timeout_ms", 200)
    b.set_option("test_stall", 1)
    prepare(b)
    for _ in range(2):  # a second launch after the first one's report: it clears what that left
        t0 = time.time()
        b.run(stream)
        status = b.device_status(stream)
        assert status & 0x1000 and status & 0xf00 in (0x100, 0x200, 0x300), hex(status)
        assert time.time() - t0 < 10
        assert b.device_status(stream) == 0
    b.set_option("test_stall", 0)
    prepare(b)
    prepare(other)
    got = []
    for handle in (b, other):
        for o in outputs:
            o.view(torch.uint8).fill_(0x5A)
        handle.run(stream)
        assert handle.device_status(stream) == 0
        got.append([o.clone().view(torch.uint8) for o in outputs])
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("tokens,hidden,kind,q", [(1, 64, "bf16", False), (1500, 7168, "bf16", True), (900, 4096, "f32", False), (500, 16384, "f32", True)])
def test_norm_wait_runs_out(gg, tokens, hidden, kind, q):
    torch = _torch()
    x = rows_of(torch, torch.Generator(device="cuda").manual_seed(1), tokens, hidden, kind)
    y, rows, scales = torch.empty_like(x), torch.empty(tokens, hidden, dtype=torch.int8, device="cuda"), torch.empty(tokens, device="cuda")
    mean, rstd = torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda")

    def prepare(b):
        assert b.prepare_norm(_type(gg, kind), tokens, hidden, x.data_ptr(), y.data_ptr(), mean_ptr=mean.data_ptr(), rstd_ptr=rstd.data_ptr(),
                              q_ptr=rows.data_ptr() if q else 0, q_scales_ptr=scales.data_ptr() if q else 0) == ""

    stalls(gg, torch, prepare, [y, mean, rstd] + ([rows, scales] if q else []))


@pytest.mark.parametrize("tokens,hidden,kind", [(1, 64, "bf16"), (1500, 7168, "bf16"), (2000, 1024, "fp16"), (500, 16384, "f32")])
def test_norm_grad_wait_runs_out(gg, tokens, hidden, kind):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(2)
    x, dy, more = (rows_of(torch, g, tokens, hidden, kind) for _ in range(3))
    mean, rstd = x.float().mean(1), (x.float().var(1, unbiased=False) + 1e-5).rsqrt()
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty(hidden, device="cuda"), torch.empty(hidden, device="cuda")

    def prepare(b):
        assert b.prepare_norm_grad(_type(gg, kind), tokens, hidden, x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), dx.data_ptr(),
                                   dsum_ptr=more.data_ptr(), dgamma_ptr=dgamma.data_ptr(), dbeta_ptr=dbeta.data_ptr()) == ""

    stalls(gg, torch, prepare, [dx, dgamma, dbeta])


@pytest.mark.parametrize("counts,n,k,kind,top_k,extra,eight", [
    ([1] * 5, 4096, 7168, "bf16", 5, 0, False),         # all items cut along k
    ([900, 0, 1300], 2056, 9216, "fp16", 2, 1, False),  # those of the last round
    ([700, 300], 2880, 1024, "bf16", 0, 3, True),       # none
    ([1], 8, 16, "bf16", 0, 0, True),
])
def test_i8_wait_runs_out(gg, counts, n, k, kind, top_k, extra, eight):
    torch = _torch()
    c = i8_case(torch, counts, n, k, kind, top_k, extra, eight)
    out = torch.empty(c["rows"], n, dtype=c["x"].dtype if not eight else torch.bfloat16, device="cuda")
    stalls(gg, torch, lambda b: prepare_i8(gg, torch, c, out, b), [out])
