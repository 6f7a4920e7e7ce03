"""Workloads of the operators around the experts' products of a mixture-of-experts layer.

Each case names one operator and its sizes. `run` computes it either in plain torch operations
(`own` false) or through the B200 library's entry points (`own` true), on the same inputs.

  route          logits -> top-k experts, weights, expert order, per-expert counts, balance losses
  route_grad     gradient of the weights and of the losses with respect to the logits
  dispatch       tokens into expert order (one row for each chosen expert)
  combine        weighted sum of each token's rows, back in token order
  dispatch_grad  the same sum without weights: the gradient of dispatch
  combine_grad   gradients of combine with respect to the rows and to the weights
  w4             rows in expert order times their expert's 4-bit weights with group scales

Sizes: 256 experts, hidden 7168, N 4096 and 131072 rows are the largest expert-parallel workload of
bench.py; 32 experts with N 7168 and K 2048 its down projection; 2880 its padded one; N 512 and K 384 the tiny one.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one step of single-stream decoding: the router's answer for one token
        dict(name="route-1", op="route", tokens=1, experts=256, top_k=8, logits="f32", normalize=True, pad=0.0, closed=0.0),
        # a ragged training micro-batch with padding tokens, experts that are closed to some tokens, and an odd number of experts
        dict(name="route-1000", op="route", tokens=1000, experts=33, top_k=3, logits="bf16", normalize=False, pad=0.1, closed=0.1),
        # the router of the 256-expert workload: 131072 rows are 16384 tokens times 8
        dict(name="route-16384", op="route", tokens=16384, experts=256, top_k=8, logits="f32", normalize=True, pad=0.02, closed=0.0),
        # the same router's backward pass
        dict(name="route_grad-16384", op="route_grad", tokens=16384, experts=256, top_k=8, logits="f32", normalize=True, pad=0.02, closed=0.0),
        # backward pass of the ragged micro-batch, 16-bit logits
        dict(name="route_grad-1000", op="route_grad", tokens=1000, experts=33, top_k=3, logits="bf16", normalize=False, pad=0.1, closed=0.1),
        # tokens into expert order for the 256-expert workload's gate/up product
        dict(name="dispatch-16384", op="dispatch", tokens=16384, experts=256, top_k=8, hidden=7168, dtype="bf16", pad=0.02),
        # a decoding batch's rows back to its tokens
        dict(name="combine-64", op="combine", tokens=64, experts=32, top_k=4, hidden=7168, dtype="fp16", pad=0.0),
        # training: the rows of the 256-expert workload's product (N 4096) back to its tokens
        dict(name="combine-16384", op="combine", tokens=16384, experts=256, top_k=8, hidden=4096, dtype="bf16", pad=0.02),
        # the combine's backward pass on the padded workload's width, a ragged number of tokens
        dict(name="combine_grad-7999", op="combine_grad", tokens=7999, experts=16, top_k=2, hidden=2880, dtype="bf16", pad=0.05),
        # one decoded token through 8 of 64 experts (gate/up projection)
        dict(name="w4-1", op="w4", tokens=1, experts=64, top_k=8, n=4096, k=7168, group=128, zeros=False, dtype="bf16"),
        # a small decoding batch through the down projection, with zero points
        dict(name="w4-37", op="w4", tokens=37, experts=32, top_k=4, n=7168, k=2048, group=64, zeros=True, dtype="fp16"),
        # a large decoding batch: 1024 rows over 64 experts, 16 rows an expert on average and more where they are popular
        dict(name="w4-128", op="w4", tokens=128, experts=64, top_k=8, n=4096, k=7168, group=128, zeros=False, dtype="bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["route", "route_grad", "dispatch", "combine", "dispatch_grad", "combine_grad", "w4", "w4"])
    experts = rng.choice([4, 7, 8, 16, 32, 33, 64, 100, 128, 256])
    top_k = min(experts, rng.randint(1, 8))
    if op in ("route", "route_grad"):
        return dict(op=op, tokens=_spread(rng, 1, 16384), experts=experts, top_k=top_k, logits=rng.choice(sorted(TYPES)),
                    normalize=rng.random() < 0.5, pad=rng.choice([0.0, 0.1]), closed=rng.choice([0.0, 0.2]))
    dtype = rng.choice(["bf16", "fp16"])
    if op != "w4":
        return dict(op=op, tokens=_spread(rng, 1, 16384), experts=experts, top_k=top_k,
                    hidden=8 * _spread(rng, 16, 896), dtype=dtype, pad=rng.choice([0.0, 0.1]))
    n, k = 8 * _spread(rng, 16, 896), 32 * _spread(rng, 8, 224)
    while experts * n * k > 64 * 4096 * 7168:
        experts //= 2
    top_k = min(top_k, experts)
    return dict(op=op, tokens=_spread(rng, 1, max(1, 1024 // top_k)), experts=experts, top_k=top_k, n=n, k=k,
                group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5, dtype=dtype)


# ---- inputs -----------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _pad_mask(case, g):
    """1 for a token, 0 for padding: a fixed share of the tokens, at random places."""
    t = case["tokens"]
    m = torch.ones(t, dtype=torch.uint8, device="cuda")
    m[torch.randperm(t, generator=g, device="cuda")[: int(t * case["pad"])]] = 0
    return m


def _logits(case, g):
    """Router outputs: normal with popular experts among them; closed experts at -inf."""
    t, e = case["tokens"], case["experts"]
    x = torch.randn(t, e, generator=g, device="cuda") * 1.5 + torch.randn(e, generator=g, device="cuda") * 0.7
    x = x.to(TYPES[case["logits"]])
    if case["closed"]:
        x[torch.rand(t, e, generator=g, device="cuda") < case["closed"]] = -math.inf
    return x


def _slots(case, g):
    """Tokens' experts under uneven popularity, as route returns them: ids, dest, src, offsets."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    popular = torch.randn(e, generator=g, device="cuda") * 0.7
    u = torch.rand(t, e, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
    ids = (popular - torch.log(-torch.log(u))).topk(k, dim=1).indices
    ids[_pad_mask(case, g) == 0] = -1
    return _expert_order(ids, e)


def _expert_order(ids, experts):
    key = torch.where(ids < 0, experts, ids).flatten()
    sorted_key, order = torch.sort(key, stable=True)
    slots = key.numel()
    dest = torch.empty(slots, dtype=torch.int32, device=ids.device)
    dest[order] = torch.arange(slots, dtype=torch.int32, device=ids.device)
    dest = torch.where(key < experts, dest, -1).view(ids.shape)
    src = torch.where(sorted_key < experts, order, -1).int()
    counts = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    counts.scatter_add_(0, key, torch.ones_like(key, dtype=torch.int32))
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = torch.cumsum(counts[:experts], 0)
    return dict(ids=ids.int(), dest=dest, src=src, counts=counts[:experts].clone(), offsets=offsets)


def _w4_ids(case):
    """The experts of each token [tokens, top_k]: by the case alone, so that what a pass reads is known."""
    r = np.random.RandomState(case["tokens"] * 7 + case["experts"] * 3 + case["top_k"])
    score = r.randn(case["experts"]) * 0.7 + r.gumbel(size=(case["tokens"], case["experts"]))
    return np.argsort(-score, axis=1)[:, : case["top_k"]]


def prepare(case, seed):
    g = _generator(seed)
    op, t, k = case["op"], case["tokens"], case["top_k"]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = dict(case=dict(case))
    if op in ("route", "route_grad"):
        s["logits"] = _logits(case, g)
        s["mask"] = _pad_mask(case, g)
        if op == "route_grad":
            s.update(_route(s["logits"], s["mask"], case))
            s["dweights"] = rand(t, k)
            s["dlosses"] = torch.tensor([0.01, 0.001], device="cuda")
    elif op == "w4":
        e, n, kk = case["experts"], case["n"], case["k"]
        relabel = torch.randperm(e, generator=g, device="cuda")
        s.update(_expert_order(relabel[torch.from_numpy(_w4_ids(case)).cuda()], e))
        groups = -(-kk // case["group"])
        s["x"] = rand(t, kk).to(TYPES[case["dtype"]])
        s["qweight"] = torch.randint(0, 256, (e, n, kk // 2), dtype=torch.uint8, generator=g, device="cuda")
        s["scales"] = (torch.rand(e, n, groups, generator=g, device="cuda") * 0.01 + 0.002).to(TYPES[case["dtype"]])
        s["zeros"] = torch.randint(0, 16, (e, n, groups), dtype=torch.uint8, generator=g, device="cuda") if case["zeros"] else None
    else:
        s.update(_slots(case, g))
        h, dt = case["hidden"], TYPES[case["dtype"]]
        if op == "dispatch":
            s["x"] = rand(t, h).to(dt)
        else:
            s["rows"] = rand(t * k, h).to(dt)
            s["weights"] = torch.softmax(rand(t, k), dim=1) if op != "dispatch_grad" else None
            if op == "combine_grad":
                s["dy"] = rand(t, h).to(dt)
    if own:
        _handle(s)
    return s


# ---- the framework's operators ------------------------------------------------------------------


def _package():
    if "gg_b200" not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        path = os.path.join(root, "groupgemm-cktile-optimized_b200", "__init__.py")
        spec = importlib.util.spec_from_file_location("gg_b200", path)
        mod = importlib.util.module_from_spec(spec)
        sys.modules["gg_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["gg_b200"]


def _handle(s):
    """The prepared handle of the state's operator and the buffers that it writes."""
    gg, case = _package(), s["case"]
    op, t, k, e = case["op"], case["tokens"], case["top_k"], case["experts"]
    dt = {"f32": gg.F32, "bf16": gg.BF16, "fp16": gg.FP16}
    new = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    ptr = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
    ints = dict(dtype=torch.int32)
    b, stream = gg.make_b200_backend(), torch.cuda.current_stream().cuda_stream
    if op == "route":
        o = dict(ids=new(t, k, **ints), weights=new(t, k), lse=new(t), counts=new(e, **ints), offsets=new(e + 1, **ints),
                 live=new(1, **ints), dest=new(t, k, **ints), src=new(t * k, **ints), prob=new(e), losses=new(2))
        why = b.prepare_route(dt[case["logits"]], t, e, k, ptr(s["logits"]), mask_ptr=ptr(s["mask"]), normalize=case["normalize"],
                              stream=stream, **{n + "_ptr": ptr(v) for n, v in o.items()})
    elif op == "route_grad":
        o = dict(dlogits=torch.empty_like(s["logits"]))
        why = b.prepare_route_grad(dt[case["logits"]], t, e, k, ptr(s["logits"]), ptr(o["dlogits"]), ids_ptr=ptr(s["ids"]),
                                   lse_ptr=ptr(s["lse"]), counts_ptr=ptr(s["counts"]), live_ptr=ptr(s["live"]), mask_ptr=ptr(s["mask"]),
                                   dweights_ptr=ptr(s["dweights"]), dlosses_ptr=ptr(s["dlosses"]), normalize=case["normalize"], stream=stream)
    elif op == "w4":
        o = dict(out=new(t * k, case["n"], dtype=s["x"].dtype))
        why = b.prepare_w4(dt[case["dtype"]], e, case["n"], case["k"], case["group"], t * k, ptr(s["x"]), ptr(s["qweight"]), ptr(s["scales"]),
                           ptr(s["offsets"]), ptr(o["out"]), zeros_ptr=ptr(s["zeros"]), src_ptr=ptr(s["src"]), tokens=t, top_k=k, stream=stream)
    elif op == "dispatch":
        o = dict(rows=new(t * k, case["hidden"], dtype=s["x"].dtype))
        why = b.prepare_dispatch(dt[case["dtype"]], t, k, e, case["hidden"], ptr(s["x"]), ptr(s["dest"]), ptr(s["offsets"]), ptr(o["rows"]),
                                 stream=stream)
    elif op == "combine_grad":
        o = dict(drows=torch.empty_like(s["rows"]), dweights=new(t, k))
        why = b.prepare_combine_grad(dt[case["dtype"]], t, k, e, case["hidden"], ptr(s["dy"]), ptr(s["rows"]), ptr(s["dest"]), ptr(s["offsets"]),
                                     ptr(o["drows"]), weights_ptr=ptr(s["weights"]), dweights_ptr=ptr(o["dweights"]), stream=stream)
    else:
        o = dict(y=new(t, case["hidden"], dtype=s["rows"].dtype))
        why = b.prepare_combine(dt[case["dtype"]], t, k, e, case["hidden"], ptr(s["rows"]), ptr(s["dest"]), ptr(o["y"]),
                                weights_ptr=ptr(s["weights"]), stream=stream)
    if why:
        raise ValueError(why)
    s["backend"], s["out"] = b, o


# ---- plain forms ---------------------------------------------------------------------------------


def _route(logits, mask, case):
    t, e = logits.shape
    k = case["top_k"]
    l = torch.where(mask[:, None] != 0, logits.float(), -math.inf)
    top = l.amax(1, keepdim=True)
    alive = top[:, 0] > -math.inf
    top = torch.where(alive[:, None], top, 0.0)
    ex = torch.exp(l - top)
    total = ex.sum(1, keepdim=True)
    lse = torch.where(alive, top[:, 0] + torch.log(total[:, 0]), -math.inf)
    p = torch.where(alive[:, None], ex / total, 0.0)
    best, index = torch.sort(l, dim=1, descending=True, stable=True)
    best, index = best[:, :k], index[:, :k]
    there = best > -math.inf
    ids = torch.where(there, index, -1)
    chosen = torch.exp(best - top)
    weights = chosen / chosen.sum(1, keepdim=True) if case["normalize"] else chosen / total
    weights = torch.where(there, weights, 0.0)
    order = _expert_order(ids, e)
    live = alive.sum()
    n = live.clamp(min=1).float()
    prob = p.sum(0) / n
    balance = e * (order["counts"].float() / (k * n) * prob).sum()
    z = torch.where(alive, lse, 0.0).square().sum() / n
    return dict(order, weights=weights, lse=lse, live=live.int().view(1), prob=prob, losses=torch.stack([balance, z]))


def _route_grad(s):
    case, logits = s["case"], s["logits"]
    t, e = logits.shape
    k = case["top_k"]
    l = torch.where(s["mask"][:, None] != 0, logits.float(), -math.inf)
    alive = (s["lse"] > -math.inf)[:, None]
    p = torch.where(alive, torch.exp(l - torch.where(alive, s["lse"][:, None], 0.0)), 0.0)
    n = s["live"].clamp(min=1).float()
    dp = (s["dlosses"][0] * e / (k * n * n) * s["counts"].float()).expand(t, e)
    there = s["ids"] >= 0
    at = torch.where(there, s["ids"], 0).long()
    dw = torch.where(there, s["dweights"], 0.0)
    if case["normalize"]:
        q = torch.where(there, p.gather(1, at), 0.0)
        q = q / torch.where(there.any(1, keepdim=True), q.sum(1, keepdim=True), 1.0)
        dq = q * (dw - (q * dw).sum(1, keepdim=True))
        d = torch.zeros_like(p).scatter_add_(1, at, dq)
    else:
        dp = dp.scatter_add(1, at, dw)
        d = 0.0
    d = d + p * (dp - (p * dp).sum(1, keepdim=True))
    d = d + p * (2 * s["dlosses"][1] / n * torch.where(alive, s["lse"][:, None], 0.0))
    return dict(dlogits=d.to(logits.dtype))


def _w4(s):
    case = s["case"]
    e, n, k, rows = case["experts"], case["n"], case["k"], s["src"].numel()
    expert = torch.searchsorted(s["offsets"][1:].contiguous(), torch.arange(rows, dtype=torch.int32, device="cuda"), right=True)
    active, which = torch.unique(expert, return_inverse=True)
    q = s["qweight"][active]
    group = torch.arange(k, device="cuda") // case["group"]
    w = torch.stack([q & 15, q >> 4], dim=3).view(active.numel(), n, k).float()
    w -= s["zeros"][active][:, :, group] if case["zeros"] else 8
    w *= s["scales"][active][:, :, group].float()
    place = torch.arange(rows, device="cuda") - s["offsets"][expert]
    x = torch.zeros(active.numel(), int(place.max()) + 1, k, device="cuda")
    x[which, place] = s["x"][(s["src"] // case["top_k"]).long()].float()
    return dict(out=torch.bmm(x, w.transpose(1, 2))[which, place].to(s["x"].dtype))


def _gathered(s):
    """The rows of each token [tokens, top_k, hidden] in 32 bits, zero where a slot has none."""
    there = s["dest"] >= 0
    rows = s["rows"][torch.where(there, s["dest"], 0).long()].float()
    return torch.where(there[..., None], rows, 0.0), there


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "route":
        return _route(s["logits"], s["mask"], case)
    if op == "route_grad":
        return _route_grad(s)
    if op == "w4":
        return _w4(s)
    if op == "dispatch":
        there = s["src"] >= 0
        token = torch.where(there, s["src"], 0) // case["top_k"]
        return dict(rows=torch.where(there[:, None], s["x"][token.long()], 0.0))
    rows, there = _gathered(s)
    if op == "combine":
        return dict(y=(rows * s["weights"][..., None]).sum(1).to(s["rows"].dtype))
    if op == "dispatch_grad":
        return dict(y=rows.sum(1).to(s["rows"].dtype))
    dy = s["dy"].float()
    slot = torch.where(s["src"] >= 0, s["src"], 0).long()
    drows = dy[slot // case["top_k"]] * s["weights"].flatten()[slot][:, None]
    drows = torch.where(s["src"][:, None] >= 0, drows, 0.0).to(s["dy"].dtype)
    return dict(drows=drows, dweights=torch.where(there, (rows * dy[:, None]).sum(2), 0.0))


def run(state):
    if not own:
        return _plain(state)
    state["backend"].run(torch.cuda.current_stream().cuda_stream)
    return state["out"]


# ---- work and the definition in 64 bits ------------------------------------------------------------


def work(case):
    op, t, k, e = case["op"], case["tokens"], case["top_k"], case["experts"]
    live = t - int(t * case.get("pad", 0.0))
    if op == "route":
        # logits and mask in; ids, weights, dest, src; lse; counts, offsets, prob, losses, live
        return {"bytes": t * e * SIZE[case["logits"]] + t + 16 * t * k + 4 * t + 12 * e + 16, "flops": 4 * t * e}
    if op == "route_grad":
        return {"bytes": 2 * t * e * SIZE[case["logits"]] + t + 8 * t * k + 4 * t + 4 * e + 12, "flops": 8 * t * e}
    if op == "w4":
        n, kk = case["n"], case["k"]
        active = len(np.unique(_w4_ids(case)))
        groups = -(-kk // case["group"])
        weights = active * n * (kk // 2 + groups * (3 if case["zeros"] else 2))
        return {"bytes": weights + 2 * t * kk + 2 * t * k * n + 4 * t * k + 4 * (e + 1), "flops": 2 * t * k * n * kk}
    row = 2 * case["hidden"]
    if op == "dispatch":  # padding tokens' rows are not read; every output row is written
        return {"bytes": live * row + t * k * row + 4 * t * k, "flops": 0}
    if op in ("combine", "dispatch_grad"):
        return {"bytes": live * k * row + t * row + (8 if op == "combine" else 4) * t * k, "flops": 2 * live * k * case["hidden"]}
    return {"bytes": live * row + live * k * row + t * k * row + 12 * t * k, "flops": 3 * live * k * case["hidden"]}


def exact(case, seed):
    """From the definitions, token by token or expert by expert where that is how they read, in 64 bits."""
    s = prepare(case, seed)
    s = {n: v for n, v in s.items() if n not in ("backend", "out")}
    op, k = case["op"], case["top_k"]
    if op in ("route", "route_grad"):
        l = s["logits"].double().cpu().numpy()
        l = np.where(s["mask"].cpu().numpy()[:, None] != 0, l, -np.inf)
        t, e = l.shape
        alive = np.isfinite(l).any(1)
        with np.errstate(all="ignore"):
            peak = np.where(alive, l.max(1), 0.0)
            lse = np.where(alive, peak + np.log(np.exp(l - peak[:, None]).sum(1)), -np.inf)
            p = np.where(alive[:, None], np.exp(l - np.where(alive, lse, 0.0)[:, None]), 0.0)
        pick = np.argsort(-l, axis=1, kind="stable")[:, :k]
        there = np.take_along_axis(l, pick, 1) > -np.inf
        q = np.where(there, np.take_along_axis(p, pick, 1), 0.0)
        share = q / np.where(alive, q.sum(1), 1.0)[:, None]
        counts = np.bincount(pick[there], minlength=e)
        n = max(1, int(alive.sum()))
        if op == "route":
            prob = p.sum(0) / n
            balance = e * float((counts / (k * n) * prob).sum())
            z = float((lse[alive] ** 2).sum()) / n
            return dict(ids=None, counts=None, offsets=None, live=None, dest=None, src=None, weights=share if case["normalize"] else q,
                        lse=lse, prob=prob, losses=np.array([balance, z]))
        db, dz = (float(v) for v in s["dlosses"].cpu())
        dw = np.where(there, s["dweights"].double().cpu().numpy(), 0.0)
        d = p * (2 * dz / n * np.where(alive, lse, 0.0))[:, None]
        gb = np.broadcast_to(db * e * counts / (k * n * n), (t, e)).copy()
        if case["normalize"]:
            np.put_along_axis(d, pick, np.take_along_axis(d, pick, 1) + share * (dw - (share * dw).sum(1, keepdims=True)), 1)
        else:
            np.put_along_axis(gb, pick, np.take_along_axis(gb, pick, 1) + dw, 1)
        return dict(dlogits=d + p * (gb - (p * gb).sum(1, keepdims=True)))
    if op == "w4":
        offsets = s["offsets"].tolist()
        src = s["src"].long()
        out = torch.zeros(src.numel(), case["n"], dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            if offsets[e] == offsets[e + 1]:
                continue
            q = s["qweight"][e].int()
            w = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = (q % 16).double(), (q // 16).double()
            grow = lambda v: v.double().repeat_interleave(case["group"], 1)[:, : case["k"]]  # noqa: E731
            w = (w - (grow(s["zeros"][e]) if case["zeros"] else 8.0)) * grow(s["scales"][e])
            rows = slice(offsets[e], offsets[e + 1])
            out[rows] = s["x"][src[rows] // k].double() @ w.t()
        return dict(out=out)
    dest = s["dest"].long()
    if op == "dispatch":
        rows = torch.zeros(dest.numel(), case["hidden"], dtype=torch.float64, device="cuda")
        for j in range(k):
            at = dest[:, j] >= 0
            rows[dest[at, j]] = s["x"][at].double()
        return dict(rows=rows)
    weights = s["weights"].double() if s["weights"] is not None else torch.ones(dest.shape, dtype=torch.float64, device="cuda")
    if op in ("combine", "dispatch_grad"):
        y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
        for j in range(k):
            at = dest[:, j] >= 0
            y[at] += s["rows"][dest[at, j]].double() * weights[at, j, None]
        return dict(y=y)
    drows = torch.zeros(dest.numel(), case["hidden"], dtype=torch.float64, device="cuda")
    dweights = torch.zeros(dest.shape, dtype=torch.float64, device="cuda")
    for j in range(k):
        at = dest[:, j] >= 0
        drows[dest[at, j]] = s["dy"][at].double() * weights[at, j, None]
        dweights[at, j] = (s["dy"][at].double() * s["rows"][dest[at, j]].double()).sum(1)
    return dict(drows=drows, dweights=dweights)
