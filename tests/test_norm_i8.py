"""CPU tests of the layer norm's, the 8-bit rounding's and the 8-bit products' entry points: what they refuse, before any CUDA call, and
how the products' work is dealt out (tests/i8_plan_check.cu walks the kernel's own plan on the host)."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG_DIR, ROOT

P = 0x10000  # an aligned address that is never read

NORM = dict(dtype=0, tokens=4, hidden=64, x_ptr=P, y_ptr=P)
NORM_GRAD = dict(dtype=0, tokens=4, hidden=64, x_ptr=P, mean_ptr=P, rstd_ptr=P, dy_ptr=P, dx_ptr=P)
QUANT = dict(dtype=0, rows=4, k=64, x_ptr=P, q_ptr=P, scales_ptr=P)
I8 = dict(dtype=0, experts=8, n=64, k=256, rows=4, x_ptr=P, weight_ptr=P, scales_ptr=P, offsets_ptr=P, out_ptr=P)
BASE = dict(norm=NORM, norm_grad=NORM_GRAD, quant=QUANT, i8=I8)


@pytest.mark.parametrize("op,kw,reason", [
    ("norm", dict(dtype=3), "dtype"),
    ("norm", dict(param_type=1), "param_type"),
    ("norm", dict(tokens=-1), "tokens"),
    ("norm", dict(tokens=1 << 31), "tokens"),
    ("norm", dict(hidden=60), "hidden"),
    ("norm", dict(hidden=0), "hidden"),
    ("norm", dict(hidden=16392), "hidden"),
    ("norm", dict(eps=-1e-5), "eps"),
    ("norm", dict(eps=float("nan")), "eps"),
    ("norm", dict(eps=float("inf")), "eps"),
    ("norm", dict(x_ptr=0), "non-null"),
    ("norm", dict(y_ptr=0), "non-null"),
    ("norm", dict(q_ptr=P), "go together"),
    ("norm", dict(q_scales_ptr=P), "go together"),
    ("norm", dict(sum_ptr=P), "residual"),
    ("norm", dict(x_ptr=P + 8), "16-byte"),
    ("norm", dict(gamma_ptr=P + 2), "16-byte"),
    ("norm", dict(mean_ptr=P + 2), "4-byte"),
    ("norm_grad", dict(dtype=-1), "dtype"),
    ("norm_grad", dict(param_type=1), "param_type"),
    ("norm_grad", dict(hidden=12), "hidden"),
    ("norm_grad", dict(mean_ptr=0), "non-null"),
    ("norm_grad", dict(dx_ptr=0), "non-null"),
    ("norm_grad", dict(dsum_ptr=P + 8), "16-byte"),
    ("norm_grad", dict(dgamma_ptr=P + 1), "4-byte"),
    ("quant", dict(dtype=4), "dtype"),
    ("quant", dict(rows=-1), "rows"),
    ("quant", dict(k=12), "multiple of 8"),
    ("quant", dict(scales_ptr=0), "non-null"),
    ("quant", dict(q_ptr=P + 8), "16-byte"),
    ("i8", dict(dtype=2), "dtype"),
    ("i8", dict(experts=0), "experts"),
    ("i8", dict(experts=1025), "experts"),
    ("i8", dict(n=60), "n must be a multiple of 8"),
    ("i8", dict(k=40), "k must be a multiple of 16"),
    ("i8", dict(k=131072), "131056"),
    ("i8", dict(rows=-1), "rows"),
    ("i8", dict(rows=1 << 31), "rows"),
    ("i8", dict(src_ptr=P, tokens=-1), "tokens"),
    ("i8", dict(src_ptr=P, tokens=4, top_k=0), "top_k"),
    ("i8", dict(src_ptr=P, tokens=0), "without tokens"),
    ("i8", dict(weight_ptr=0), "non-null"),
    ("i8", dict(weight_ptr=P + 8), "16-byte"),
    ("i8", dict(scales_ptr=P + 2), "4-byte"),
    ("i8", dict(n=1 << 23, k=1 << 16), "TMA"),
    ("i8", dict(n=1 << 20, k=16, rows=(1 << 31) - 1, experts=1024), "too many"),
])
def test_refusals(gg, op, kw, reason):
    b = gg.B200Backend()
    why = getattr(b, "prepare_" + op)(**dict(BASE[op], **kw))
    assert reason in why, why
    assert reason in b.last_error()
    with pytest.raises(gg.GGError):
        b.run()  # nothing is prepared


@pytest.mark.parametrize("op", sorted(BASE))
def test_prepare_without_gpu_fails_loudly(gg, op):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(gg.GGError) as e:
        getattr(gg.B200Backend(), "prepare_" + op)(**BASE[op])
    assert e.value.code == gg.GG_ERR_CUDA


@pytest.mark.parametrize("op", sorted(BASE))
def test_null_arguments(gg, op):
    fn = getattr(gg.load_library(), "gg_prepare_" + op)
    b = gg.B200Backend()
    assert fn(None, None, None, None, 0) == gg.GG_ERR_ARG
    assert fn(b._h, None, None, None, 0) == gg.GG_ERR_ARG


def test_plan_covers_every_step_once(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not available")
    exe = tmp_path / "i8_plan_check"
    build = subprocess.run([nvcc, "-std=c++17", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "-I", os.path.join(ROOT, "include"), "-I",
                            os.path.join(PKG_DIR, "csrc"), "-o", str(exe), os.path.join(ROOT, "tests", "i8_plan_check.cu")],
                           capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr[-2000:]
    run = subprocess.run([str(exe), "4000"], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0 and run.stdout.startswith("ok "), run.stdout + run.stderr
