"""CPU tests of the layer operators' entry points: what they refuse, before any CUDA call."""
import ctypes

import pytest

P = 0x10000  # an aligned address that is never read

ROUTE = dict(logits_type=2, tokens=4, experts=8, top_k=2, logits_ptr=P, ids_ptr=P, weights_ptr=P, counts_ptr=P, offsets_ptr=P, live_ptr=P,
             dest_ptr=P, src_ptr=P)
ROUTE_GRAD = dict(logits_type=2, tokens=4, experts=8, top_k=2, logits_ptr=P, dlogits_ptr=P, ids_ptr=P, lse_ptr=P, counts_ptr=P, live_ptr=P)
DISPATCH = dict(dtype=0, tokens=4, top_k=2, experts=8, hidden=64, x_ptr=P, dest_ptr=P, offsets_ptr=P, rows_ptr=P)
COMBINE = dict(dtype=0, tokens=4, top_k=2, experts=8, hidden=64, rows_ptr=P, dest_ptr=P, y_ptr=P)
COMBINE_GRAD = dict(dtype=0, tokens=4, top_k=2, experts=8, hidden=64, dy_ptr=P, rows_ptr=P, dest_ptr=P, offsets_ptr=P, drows_ptr=P,
                    dweights_ptr=P)
W4 = dict(dtype=0, experts=8, n=64, k=256, group_size=128, rows=4, x_ptr=P, qweight_ptr=P, scales_ptr=P, offsets_ptr=P, out_ptr=P)
BASE = dict(route=ROUTE, route_grad=ROUTE_GRAD, dispatch=DISPATCH, combine=COMBINE, combine_grad=COMBINE_GRAD, w4=W4)


@pytest.mark.parametrize("op,kw,reason", [
    ("route", dict(logits_type=3), "logits_type"),
    ("route", dict(tokens=-1), "tokens must be"),
    ("route", dict(tokens=1 << 40), "tokens must be"),
    ("route", dict(experts=0), "experts must be 1..1024"),
    ("route", dict(experts=1025), "experts must be 1..1024"),
    ("route", dict(top_k=0), "top_k"),
    ("route", dict(top_k=9), "top_k"),
    ("route", dict(experts=64, top_k=33), "top_k"),
    ("route", dict(tokens=1 << 30), "below 2^31"),
    ("route", dict(logits_ptr=0), "non-null"),
    ("route", dict(src_ptr=0), "non-null"),
    ("route", dict(tokens=0, counts_ptr=0), "non-null"),
    ("route", dict(logits_ptr=P + 4), "16-byte"),
    ("route", dict(weights_ptr=P + 2), "4-byte"),
    ("route_grad", dict(logits_type=-1), "logits_type"),
    ("route_grad", dict(lse_ptr=0), "non-null"),
    ("route_grad", dict(dlogits_ptr=P + 8), "16-byte"),
    ("dispatch", dict(dtype=2), "dtype"),
    ("dispatch", dict(hidden=60), "hidden"),
    ("dispatch", dict(hidden=0), "hidden"),
    ("dispatch", dict(top_k=33), "top_k"),
    ("dispatch", dict(experts=0), "experts"),
    ("dispatch", dict(rows_ptr=0), "non-null"),
    ("dispatch", dict(offsets_ptr=0), "non-null"),
    ("dispatch", dict(x_ptr=P + 8), "16-byte"),
    ("combine", dict(tokens=-1), "tokens"),
    ("combine", dict(y_ptr=0), "non-null"),
    ("combine", dict(weights_ptr=P + 1), "4-byte"),
    ("combine_grad", dict(rows_ptr=0), "non-null"),
    ("combine_grad", dict(drows_ptr=P + 2), "16-byte"),
    ("w4", dict(dtype=2), "dtype"),
    ("w4", dict(experts=1025), "experts"),
    ("w4", dict(n=60), "n must be a multiple of 8"),
    ("w4", dict(k=40), "k must be a multiple of 32"),
    ("w4", dict(group_size=48), "group_size"),
    ("w4", dict(rows=-1), "rows"),
    ("w4", dict(src_ptr=P, tokens=-1), "tokens"),
    ("w4", dict(src_ptr=P, tokens=4, top_k=0), "top_k"),
    ("w4", dict(qweight_ptr=0), "non-null"),
    ("w4", dict(scales_ptr=P + 2), "16-byte"),
    ("w4", dict(offsets_ptr=P + 2), "4-byte"),
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


def test_null_arguments(gg):
    lib = gg.load_library()
    b = gg.B200Backend()
    for name, extra in (("route", ()), ("route_grad", ()), ("permute", (gg.OP_DISPATCH,)), ("w4", ())):
        fn = getattr(lib, "gg_prepare_" + name)
        assert fn(None, None, *extra, None, None, 0) == gg.GG_ERR_ARG
        assert fn(b._h, None, *extra, None, None, 0) == gg.GG_ERR_ARG
    prob = gg.GGPermuteProblem()
    assert lib.gg_prepare_permute(b._h, ctypes.byref(prob), 7, None, None, 0) == gg.GG_ERR_ARG
    assert "op must be" in b.last_error()
