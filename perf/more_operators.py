"""Workloads of the layer norm in front of a mixture-of-experts layer and of the experts' products in 8-bit integers.

Each case names one operator and its sizes. `run` computes it either in plain torch operations
(`own` false) or through the B200 library's entry points (`own` true), on the same inputs.

  norm       layer norm of each token, after adding the block's residual where there is one
  norm_grad  its gradients with respect to the input, the weight and the bias
  i8         rows in expert order times their expert's 8-bit weights: each token is rounded to 8-bit integers with
             a scale of its own, each weight row has a scale, sums are whole numbers. With `norm`, the tokens'
             layer norm makes the 8-bit rows.

Sizes: hidden 7168, N 4096 and 16384 tokens (131072 rows over 8) belong to the largest expert-parallel workload of
bench.py, 8 experts of 4096 rows are its gate/up projection; 32 experts with N 7168 and K 2048 its down projection;
2880 its padded one.
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
EPS = 1e-5


def listed():
    return [
        # one decoded token enters the layer: latency
        dict(name="norm-1", op="norm", tokens=1, hidden=7168, dtype="bf16", params="bf16", residual=True),
        # a ragged micro-batch of the padded workload's width, the first norm of a model (no residual yet)
        dict(name="norm-1000", op="norm", tokens=1000, hidden=2880, dtype="fp16", params="f32", residual=False),
        # a training step's tokens at the largest workload's width
        dict(name="norm-16384", op="norm", tokens=16384, hidden=7168, dtype="bf16", params="bf16", residual=True),
        # backward pass of the ragged micro-batch
        dict(name="norm_grad-1000", op="norm_grad", tokens=1000, hidden=2880, dtype="fp16", params="f32", residual=False),
        # a residual stream kept in 32 bits
        dict(name="norm_grad-2048", op="norm_grad", tokens=2048, hidden=4096, dtype="f32", params="f32", residual=True),
        # backward pass of the training step
        dict(name="norm_grad-16384", op="norm_grad", tokens=16384, hidden=7168, dtype="bf16", params="bf16", residual=True),
        # one decoded token through 8 of 64 experts (gate/up projection)
        dict(name="i8-1", op="i8", tokens=1, experts=64, top_k=8, n=4096, k=7168, dtype="bf16", pad=0.0, norm=False),
        # a small decoding batch through the down projection
        dict(name="i8-37", op="i8", tokens=37, experts=32, top_k=4, n=7168, k=2048, dtype="fp16", pad=0.0, norm=False),
        # a large decoding batch from its norm on: 1024 rows over 64 experts
        dict(name="i8-128", op="i8", tokens=128, experts=64, top_k=8, n=4096, k=7168, dtype="bf16", pad=0.0, norm=True),
        # a short prompt through one expert's odd width (a dense layer)
        dict(name="i8-300", op="i8", tokens=300, experts=1, top_k=1, n=1000, k=2048, dtype="fp16", pad=0.0, norm=False),
        # prompts with padding on the padded workload: 16 experts, 1000 rows each on average
        dict(name="i8-8000", op="i8", tokens=8000, experts=16, top_k=2, n=2880, k=2880, dtype="bf16", pad=0.05, norm=False),
        # long prompts through the gate/up projection: 8 experts, 4096 rows each on average, from their norm on
        dict(name="i8-16384", op="i8", tokens=16384, experts=8, top_k=2, n=4096, k=7168, dtype="bf16", pad=0.0, norm=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "i8", "i8"])
    if op != "i8":
        dtype = rng.choice(sorted(TYPES))
        hidden = 8 * _spread(rng, 8, 896)
        return dict(op=op, tokens=_spread(rng, 1, 16384 // (SIZE[dtype] // 2)), hidden=hidden, dtype=dtype,
                    params=rng.choice(["f32", dtype]), residual=rng.random() < 0.5)
    experts = rng.choice([1, 2, 4, 7, 8, 16, 32, 33, 64])
    n, k = 8 * _spread(rng, 16, 896), 16 * _spread(rng, 16, 448)
    while experts * n * k > 64 * 4096 * 7168:
        experts //= 2
    top_k = min(experts, rng.randint(1, 8))
    most = min(16384, 32768 * 4096 * 7168 // (n * k)) // top_k
    return dict(op=op, tokens=_spread(rng, 1, max(1, most)), experts=experts, top_k=top_k, n=n, k=k, dtype=rng.choice(["bf16", "fp16"]),
                pad=rng.choice([0.0, 0.1]), norm=rng.random() < 0.3)


# ---- inputs -----------------------------------------------------------------------------------


def _ids(case):
    """The experts of each token [tokens, top_k], -1 for padding: by the case alone, so that what a pass reads is known."""
    r = np.random.RandomState(case["tokens"] * 7 + case["experts"] * 3 + case["top_k"])
    score = r.randn(case["experts"]) * 0.5 + r.gumbel(size=(case["tokens"], case["experts"]))
    ids = np.argsort(-score, axis=1)[:, : case["top_k"]]
    ids[r.permutation(case["tokens"])[: int(case["tokens"] * case["pad"])]] = -1
    return ids


def _expert_order(ids, experts):
    """src and offsets as the router gives them: the slots in expert order, -1 behind the last."""
    key = torch.where(ids < 0, experts, ids).flatten()
    sorted_key, order = torch.sort(key, stable=True)
    src = torch.where(sorted_key < experts, order, -1).int()
    offsets = torch.searchsorted(sorted_key, torch.arange(experts + 1, device=ids.device)).int()
    return dict(src=src, offsets=offsets)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    op, t, dt = case["op"], case["tokens"], TYPES[case["dtype"]]
    h = case["k"] if op == "i8" else case["hidden"]
    s = dict(case=dict(case))
    # a residual stream: tokens of uneven size, a mean, and a few channels much larger than the others
    channels = torch.where(torch.rand(h, generator=g, device="cuda") < 0.005, 8.0, 1.0)
    stream = lambda: (rand(t, h) * channels * torch.exp(0.3 * rand(t, 1)) + 0.2 * rand(t, 1)).to(dt)  # noqa: E731
    s["x"] = stream()
    if op != "i8" or case["norm"]:
        pt = TYPES[case["params"]] if op != "i8" else dt
        s["gamma"], s["beta"] = (1 + 0.2 * rand(h)).to(pt), (0.1 * rand(h)).to(pt)
    if op == "norm":
        s["residual"] = stream() if case["residual"] else None
    elif op == "norm_grad":
        s["mean"], s["rstd"] = _statistics(s["x"].float())
        s["dy"] = rand(t, h).to(dt)
        s["dsum"] = rand(t, h).to(dt) if case["residual"] else None  # the residual's own gradient
    else:
        e, n = case["experts"], case["n"]
        relabel = torch.cat([torch.randperm(e, generator=g, device="cuda"), torch.tensor([-1], device="cuda")])
        s.update(_expert_order(relabel[torch.from_numpy(_ids(case)).cuda()], e))
        s["weight"] = torch.empty(e, n, h, dtype=torch.int8, device="cuda")
        for w in s["weight"]:
            w.copy_((rand(n, h) * 32).round_().clamp_(-127, 127))
        s["scales"] = torch.rand(e, n, generator=g, device="cuda") * 4e-4 + 2e-4
    if own:
        _handles(s)
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


def _handles(s):
    """The prepared handles of the state's operator, in order, and the buffers that they write."""
    gg, case = _package(), s["case"]
    op, t = case["op"], case["tokens"]
    types = {"f32": gg.F32, "bf16": gg.BF16, "fp16": gg.FP16}
    dt, stream = types[case["dtype"]], torch.cuda.current_stream().cuda_stream
    new = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    ptr = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
    x, backends, reasons = s["x"], [], []

    def add(prepare, *args, **kw):
        backends.append(gg.make_b200_backend())
        reasons.append(getattr(backends[-1], prepare)(*args, stream=stream, **kw))

    if op == "norm":
        o = dict(y=torch.empty_like(x), mean=new(t), rstd=new(t))
        if case["residual"]:
            o["sum"] = torch.empty_like(x)
        add("prepare_norm", dt, t, case["hidden"], ptr(x), ptr(o["y"]), gamma_ptr=ptr(s["gamma"]), beta_ptr=ptr(s["beta"]),
            param_type=types[case["params"]], residual_ptr=ptr(s["residual"]), sum_ptr=ptr(o.get("sum")), mean_ptr=ptr(o["mean"]),
            rstd_ptr=ptr(o["rstd"]), eps=EPS)
    elif op == "norm_grad":
        o = dict(dx=torch.empty_like(x), dgamma=new(case["hidden"]), dbeta=new(case["hidden"]))
        add("prepare_norm_grad", dt, t, case["hidden"], ptr(x), ptr(s["mean"]), ptr(s["rstd"]), ptr(s["dy"]), ptr(o["dx"]),
            gamma_ptr=ptr(s["gamma"]), param_type=types[case["params"]], dsum_ptr=ptr(s["dsum"]), dgamma_ptr=ptr(o["dgamma"]),
            dbeta_ptr=ptr(o["dbeta"]))
    else:
        e, n, k, rows = case["experts"], case["n"], case["k"], t * case["top_k"]
        o = dict(out=new(rows, n, dtype=x.dtype))
        rows_in = dict(x=x, scales=None)
        if case["norm"]:
            o["y"] = torch.empty_like(x)
            rows_in = dict(x=new(t, k, dtype=torch.int8), scales=new(t))
            s["rows_in"] = rows_in
            add("prepare_norm", dt, t, k, ptr(x), ptr(o["y"]), gamma_ptr=ptr(s["gamma"]), beta_ptr=ptr(s["beta"]), param_type=dt,
                q_ptr=ptr(rows_in["x"]), q_scales_ptr=ptr(rows_in["scales"]), eps=EPS)
        add("prepare_i8", dt, e, n, k, rows, ptr(rows_in["x"]), ptr(s["weight"]), ptr(s["scales"]), ptr(s["offsets"]), ptr(o["out"]),
            x_scales_ptr=ptr(rows_in["scales"]), src_ptr=ptr(s["src"]), tokens=t, top_k=case["top_k"])
    if any(reasons):
        raise ValueError("; ".join(r for r in reasons if r))
    s["backends"], s["out"] = backends, o


# ---- plain forms ---------------------------------------------------------------------------------


def _statistics(v):
    mean = v.mean(1)
    return mean, torch.rsqrt((v - mean[:, None]).square().mean(1) + EPS)


def _norm(v, s):
    mean, rstd = _statistics(v)
    y = (v - mean[:, None]) * rstd[:, None] * s["gamma"].float() + s["beta"].float()
    return y.to(s["x"].dtype), mean, rstd


def _rounded(v):
    """Each row's nearest whole numbers from -127 to 127, in 64 bits as halves are near, and its scale."""
    top = v.float().abs().amax(1)
    q = (v.double() * 127 / torch.where(top > 0, top, 1).double()[:, None]).round()
    return q.float(), top / 127


def _plain(s):
    case = s["case"]
    x = s["x"].float()
    if case["op"] == "norm":
        if s["residual"] is None:
            y, mean, rstd = _norm(x, s)
            return dict(y=y, mean=mean, rstd=rstd)
        total = (x + s["residual"].float()).to(s["x"].dtype)
        y, mean, rstd = _norm(total.float(), s)
        return dict(y=y, mean=mean, rstd=rstd, sum=total)
    if case["op"] == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xhat = (x - s["mean"][:, None]) * rstd
        d = dy * s["gamma"].float()
        dx = rstd * (d - d.mean(1, keepdim=True) - xhat * (d * xhat).mean(1, keepdim=True))
        if s["dsum"] is not None:
            dx = dx + s["dsum"].float()
        return dict(dx=dx.to(s["x"].dtype), dgamma=(dy * xhat).sum(0), dbeta=dy.sum(0))
    o = {}
    rows, k = s["src"].numel(), case["top_k"]
    if case["norm"]:
        o["y"] = _norm(x, s)[0]
    q, qs = _rounded(o["y"] if case["norm"] else s["x"])
    there = s["src"] >= 0
    token = (torch.where(there, s["src"], 0) // k).long()
    expert = torch.searchsorted(s["offsets"][1:].contiguous(), torch.arange(rows, dtype=torch.int32, device="cuda"), right=True)
    expert = torch.where(there, expert, s["offsets"].numel() - 2)
    active, which = torch.unique(expert, return_inverse=True)
    place = torch.arange(rows, device="cuda") - s["offsets"][expert]
    xs = torch.zeros(active.numel(), int(place.max()) + 1, case["k"], device="cuda")
    xs[which, place] = q[token]
    out = torch.bmm(xs, s["weight"][active].float().transpose(1, 2))[which, place]
    out = out * qs[token][:, None] * s["scales"][expert]
    o["out"] = torch.where(there[:, None], out, 0.0).to(s["x"].dtype)
    return o


def run(state):
    if not own:
        return _plain(state)
    stream = torch.cuda.current_stream().cuda_stream
    for b in state["backends"]:
        b.run(stream)
    return state["out"]


# ---- work and the definition in 64 bits ------------------------------------------------------------


def work(case):
    op, t = case["op"], case["tokens"]
    size = SIZE[case["dtype"]]
    if op == "norm":  # x and the residual in, y and the sum out; weight, bias; statistics
        return {"bytes": (4 if case["residual"] else 2) * t * case["hidden"] * size + 2 * case["hidden"] * SIZE[case["params"]] + 8 * t,
                "flops": 8 * t * case["hidden"]}
    if op == "norm_grad":  # x, dy and the sum's gradient in, dx out; weight, its and the bias's gradients; statistics
        return {"bytes": (4 if case["residual"] else 3) * t * case["hidden"] * size + case["hidden"] * (SIZE[case["params"]] + 8) + 8 * t,
                "flops": 14 * t * case["hidden"]}
    ids, n, k, rows = _ids(case), case["n"], case["k"], t * case["top_k"]
    active, slots = len(np.unique(ids[ids >= 0])), int((ids >= 0).sum())
    moved = active * n * (k + 4) + t * k * size + rows * n * size + 4 * rows + 4 * (case["experts"] + 1)
    return {"bytes": moved + (t * k * size + 2 * k * size if case["norm"] else 0), "flops": 2 * slots * n * k}


def exact(case, seed):
    """From the definitions in 64 bits, expert by expert where that is how they read."""
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "norm_grad":
        h = case["hidden"]
        dy = s["dy"].double()
        c = (x - s["mean"].double()[:, None]) * s["rstd"].double()[:, None]
        d = dy * s["gamma"].double()
        along, level = torch.einsum("th,th->t", d, c) / h, d.sum(1) / h
        dx = (d - level[:, None] - c * along[:, None]) * s["rstd"].double()[:, None]
        if s["dsum"] is not None:
            dx += s["dsum"].double()
        return dict(dx=dx, dgamma=torch.einsum("th,th->h", dy, c), dbeta=dy.sum(0))

    def norm(v):
        var, mean = torch.var_mean(v, 1, correction=0)
        rstd = 1 / torch.sqrt(var + EPS)
        return torch.addcmul(s["beta"].double(), (v - mean[:, None]) * rstd[:, None], s["gamma"].double()), mean, rstd

    if case["op"] == "norm":
        o = {}
        if s["residual"] is not None:
            o["sum"] = x + s["residual"].double()
            x = o["sum"].to(s["x"].dtype).double()  # the sum as it is handed on is what is normalised
        o["y"], o["mean"], o["rstd"] = norm(x)
        return o
    o = {}
    if case["norm"]:
        o["y"] = norm(x)[0]
        x = o["y"].to(s["x"].dtype).double()
    top = x.abs().amax(1, keepdim=True)
    q = torch.round(127 * x / torch.where(top == 0, 1.0, top))
    offsets, src = s["offsets"].tolist(), s["src"].long()
    out = torch.zeros(src.numel(), case["n"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        rows = slice(offsets[e], offsets[e + 1])
        token = src[rows] // case["top_k"]
        out[rows] = (q[token] @ s["weight"][e].double().t()) * (top[token] / 127) * s["scales"][e].double()
    o["out"] = out
    return o
