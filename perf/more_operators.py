"""The operators of a feed-forward layer with 8-bit weights, as cases that can be timed: tokens quantised to 8 bits
(`quantize`), a linear layer on them with scales for each token and channel (`linear`), tokens routed to experts and
sorted by them (`route`), the experts' layers (`experts`), and their results weighted and summed (`combine`).

`run` computes them in plain torch operations in 32 bits (the choice of experts and the rounding to 8 bits, where a
value next to a border counts, in 64), or, with `own` set, by the calls that a user of lava_hip makes.  Tokens are rows.
A layer's weights are (channels, K), one scale a channel; a gated layer has its gate's channels first, then as many
others, and gives act(gate) * other.  The tokens of an expert are a run of the T * top_k assignments (token * top_k +
rank) sorted by expert: `order`, with the runs' ends in `offsets`.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _linear(T, N, K, dtype, act="none", gated=False, bias=False):
    return {"op": "linear", "T": T, "N": N, "K": K, "dtype": dtype, "act": act, "gated": gated, "bias": bias}


def _experts(T, E, top_k, N, K, dtype, act="none", gated=False, bias=False, back=False, skew=0.5):
    """back: rows in the experts' order in, each assignment's own row out; else the tokens' rows in, the experts' order out."""
    return {"op": "experts", "T": T, "E": E, "top_k": top_k, "N": N, "K": K, "dtype": dtype, "act": act, "gated": gated,
            "bias": bias, "back": back, "skew": skew}


def _route(T, E, top_k, dtype, score, bias=False, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0):
    return {"op": "route", "T": T, "E": E, "top_k": top_k, "dtype": dtype, "score": score, "bias": bias,
            "groups": groups, "top_groups": top_groups, "group_best": group_best, "renormalize": renormalize,
            "scale": scale}


def listed():
    return [
        # the step of one token in front of a projection: latency is all there is
        {"name": "quantize_token", "op": "quantize", "T": 1, "K": 4096, "dtype": "f16"},
        # the experts' hidden rows of a batch of prompts, an odd number of them: bound by HBM
        {"name": "quantize_hidden", "op": "quantize", "T": 40961, "K": 1408, "dtype": "bf16"},
        # one token through a square projection: the weights' bytes in a few microseconds
        {"name": "linear_token", **_linear(1, 4096, 4096, "f16")},
        # the benchmark's decode step with 8-bit weights, its tokens in 8 bits too
        {"name": "linear_decode16", **_linear(16, 14336, 4096, "bf16", bias=True)},
        # a ragged batch of chunks: between the weights' bytes and the matrix cores
        {"name": "linear_chunks_gelu", **_linear(333, 14336, 4096, "f16", act="gelu_tanh", bias=True)},
        # prompts through the gate and up projections of the benchmark's layer at once: bound by the matrix cores
        {"name": "linear_prompts_gated", **_linear(8192, 28672, 4096, "bf16", act="silu", gated=True)},
        # a decode step's 32 tokens: most experts get a few rows, all weights are read
        {"name": "experts_decode", **_experts(32, 64, 8, 2816, 2048, "f16", act="silu", gated=True)},
        # prompts' hidden rows back through the experts, an odd number of tokens, uneven experts
        {"name": "experts_prompts", **_experts(5003, 60, 4, 2048, 1408, "bf16", back=True, skew=1.0)},
        # a decode step's tokens: one small launch
        {"name": "route_decode", **_route(64, 64, 8, "bf16", "softmax")},
        # prompts, the best 4 of 8 groups, a bias that balances the experts
        {"name": "route_prompts_groups", **_route(16384, 256, 8, "f32", "sigmoid", bias=True, groups=8, top_groups=4,
                                                  group_best=2, scale=2.5)},
        # a decode step's results
        {"name": "combine_decode", "op": "combine", "T": 64, "top_k": 8, "N": 2048, "dtype": "f16", "base": False},
        # prompts' results onto what came in
        {"name": "combine_prompts", "op": "combine", "T": 8191, "top_k": 6, "N": 2048, "dtype": "bf16", "base": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: most are multiples of 64, some of 16, a few any number."""
    n, r = _log(rng, lo, hi), rng.random()
    return max(64, n // 64 * 64) if r < 0.6 else max(16, n // 16 * 16) if r < 0.9 else n


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "route", "experts", "experts", "combine"])
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    act, gated = rng.choice([("none", False), ("none", False), ("silu", True), ("gelu_tanh", True), ("gelu_erf", False),
                             ("relu", False), ("silu", False)])
    T = _log(rng, 1, 16384)
    if op == "quantize":
        got = {"op": op, "T": T, "K": _width(rng, 64, 20000), "dtype": dtype}
    elif op == "linear":
        got = _linear(T, _width(rng, 64, 30000) * (2 if gated else 1), _width(rng, 64, 16384), dtype, act, gated,
                      rng.random() < 0.3)
    elif op == "combine":
        got = {"op": op, "T": T, "top_k": rng.randint(1, 10), "N": _width(rng, 64, 8192), "dtype": dtype,
               "base": rng.random() < 0.5}
    else:
        E = rng.choice([8, 16, 32, 60, 64, 96, 128, 160, 256, rng.randint(2, 384)])
        top_k = rng.randint(1, min(10, E))
        if op == "route":
            groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0])
            top_groups = rng.randint(max(1, groups // 2), groups)
            best = rng.choice([b for b in (1, 2) if b <= E // groups])
            top_k = min(top_k, top_groups * (E // groups))
            got = _route(T, E, top_k, dtype, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups, top_groups,
                         best, rng.random() < 0.7, rng.choice([1.0, 2.5]))
        else:
            got = _experts(T, E, top_k, _width(rng, 64, 6000) * (2 if gated else 1), _width(rng, 64, 6000), dtype, act,
                           gated, rng.random() < 0.3, rng.random() < 0.5, rng.choice([0.0, 0.5, 1.0]))
    # no more than the largest listed call of the operator
    bytes_, flops = {"quantize": (1.7e8, 1e12), "linear": (3.8e8, 1.9e12), "route": (1.8e7, 1e12),
                     "experts": (3.7e8, 1.15e11), "combine": (2.3e8, 1e12)}[op]
    while work(got)["bytes"] > bytes_ or work(got)["flops"] > flops:
        if got["T"] > 1 and rng.random() < 0.6:
            got["T"] = max(1, got["T"] * 2 // 3)
        elif "N" in got and got["N"] > 128:
            got["N"] = max(128, got["N"] // 256 * 128)
        elif "K" in got and got["K"] > 128:
            got["K"] = got["K"] // 128 * 64
        else:
            got["T"] = max(1, got["T"] // 2)
    return got


def work(case):
    T, size = case["T"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "quantize":
        return {"bytes": T * case["K"] * (size + 1) + 4 * T, "flops": 3 * T * case["K"]}
    if case["op"] == "combine":
        rows = case["top_k"] + 1 + case["base"]
        return {"bytes": T * case["N"] * rows * size + 8 * T * case["top_k"], "flops": 2 * T * case["top_k"] * case["N"]}
    if case["op"] == "route":
        E, k = case["E"], case["top_k"]
        return {"bytes": T * E * size + T * k * 12 + 4 * (E + 1) + 4 * E * case["bias"], "flops": 6 * T * E}
    N, K = case["N"], case["K"]
    out = N // 2 if case["gated"] else N
    per_channel = 8 if case["bias"] else 4
    if case["op"] == "linear":
        return {"bytes": T * (K + 4) + N * (K + per_channel) + T * out * size, "flops": 2 * T * N * K}
    rows = T * case["top_k"]
    met = case["E"] * (1.0 - (1.0 - case["top_k"] / case["E"]) ** T)   # experts that some token goes to
    read = rows if case["back"] else T
    return {"bytes": int(read * (K + 4) + met * N * (K + per_channel) + rows * (out * size + 4)), "flops": 2 * rows * N * K}


# ---- what a program has in hand -------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, dtype=dtype, device="cuda", generator=g)


def _bytes(g, *shape):
    """What rows of normal values are in 8 bits, their largest near 127."""
    x = torch.empty(shape, dtype=torch.int8, device="cuda")
    for part in x.view(shape[0], -1).chunk(8):   # a piece at a time: the normal values take four times the room
        part.copy_(_normal(g, *part.shape).mul_(34.0).round_().clamp_(-127, 127))
    return x


def _tokens(g, T, K, dtype):
    """A layer's input: tokens of different sizes, a few channels larger than the rest."""
    size = torch.exp(_normal(g, T, 1))
    channel = torch.where(torch.rand(1, K, device="cuda", generator=g) < 0.01, 8.0, 1.0)
    return (_normal(g, T, K) * size * channel).to(_TORCH[dtype])


def _layer(g, case, *experts):
    N, K = case["N"], case["K"]
    return {"w": _bytes(g, *experts, N, K),
            "w_scale": (torch.rand(*experts, N, device="cuda", generator=g) + 0.5) / (34.0 * math.sqrt(K)),
            "bias": _normal(g, *experts, N) * 0.2 if case["bias"] else None}


def _rows(g, T, K):
    return {"x": _bytes(g, T, K), "x_scale": torch.exp(_normal(g, T) * 0.5) / 34.0}


def _sorted_by_expert(ids, E):
    flat = ids.reshape(-1).long()
    order = torch.sort(flat, stable=True).indices.to(torch.int32)
    ends = torch.cumsum(torch.bincount(flat, minlength=E), 0)
    return order, torch.cat((ends.new_zeros(1), ends)).to(torch.int32)


def _inputs(case, seed):
    g, T = _generator(seed), case["T"]
    if case["op"] == "quantize":
        return {"x": _tokens(g, T, case["K"], case["dtype"])}
    if case["op"] == "linear":
        return {**_rows(g, T, case["K"]), **_layer(g, case)}
    if case["op"] == "route":
        logits = (_normal(g, T, case["E"]) * 1.5 + _normal(g, 1, case["E"]) * 0.5).to(_TORCH[case["dtype"]])
        return {"logits": logits, "bias": _normal(g, case["E"]) * 0.1 if case["bias"] else None}
    k = case["top_k"]
    if case["op"] == "combine":
        ids = torch.rand(T, max(k, 64), device="cuda", generator=g).topk(k).indices.to(torch.int32)
        w = torch.rand(T, k, device="cuda", generator=g) + 0.1
        dt = _TORCH[case["dtype"]]
        return {"ids": ids, "weights": w / w.sum(dim=1, keepdim=True), "y": _normal(g, T * k, case["N"], dtype=dt),
                "base": _normal(g, T, case["N"], dtype=dt) if case["base"] else None}
    liked = _normal(g, 1, case["E"]) * case["skew"]   # some experts are chosen more often than others
    ids = (_normal(g, T, case["E"]) + liked).topk(k).indices.to(torch.int32)
    order, offsets = _sorted_by_expert(ids, case["E"])
    return {**_rows(g, T * k if case["back"] else T, case["K"]), **_layer(g, case, case["E"]), "order": order,
            "offsets": offsets}


def _outputs(case):
    """Where a program has an operator's results."""
    T, dt = case["T"], _TORCH[case["dtype"]]
    empty = lambda *shape, dtype=dt: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if case["op"] == "quantize":
        return {"q": empty(T, case["K"], dtype=torch.int8), "scale": empty(T, dtype=torch.float32)}
    if case["op"] == "combine":
        return {"out": empty(T, case["N"])}
    if case["op"] == "route":
        k = case["top_k"]
        return {"ids": empty(T, k, dtype=torch.int32), "weights": empty(T, k, dtype=torch.float32),
                "order": empty(T * k, dtype=torch.int32), "offsets": empty(case["E"] + 1, dtype=torch.int32)}
    rows = T * case["top_k"] if case["op"] == "experts" else T
    return {"y": empty(rows, case["N"] // 2 if case["gated"] else case["N"])}


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed), "result": _outputs(case)}
    if case["op"] == "experts":
        state["most"] = int((state["offsets"][1:] - state["offsets"][:-1]).max())   # rows of an expert
    if own:
        _describe(state)
    return state


def _describe(state):
    """The descriptors of the layer, the router and the plan that a program keeps."""
    package = str(Path(__file__).resolve().parents[1] / "lava.jl_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    import lava_hip as lh
    lh.init()
    case, res = state["case"], state["result"]
    state["lh"] = lh
    if case["op"] in ("linear", "experts"):
        bias = state["bias"].data_ptr() if state["bias"] is not None else 0
        state["layer"] = lh.w8_layer_raw(state["w"].data_ptr(), state["w_scale"].data_ptr(), case["N"], case["K"],
                                         case["K"], bias=bias, act=case["act"], gated=case["gated"],
                                         experts=case.get("E", 1), expert_stride=case["N"] * case["K"])
    if case["op"] == "route":
        state["router"] = lh.moe_router_raw(case["E"], case["top_k"], case["score"],
                                            bias=state["bias"].data_ptr() if state["bias"] is not None else 0,
                                            groups=case["groups"], top_groups=case["top_groups"],
                                            group_best=case["group_best"], renormalize=case["renormalize"],
                                            scale=case["scale"])
        n = lh.moe_plan_workspace_bytes(case["T"], case["E"], case["top_k"])
        state["workspace"] = torch.zeros(max(n, 4), dtype=torch.uint8, device="cuda")
        state["plan"] = lh.moe_plan_raw(case["T"], case["E"], case["top_k"], res["offsets"].data_ptr(),
                                        res["order"].data_ptr(), state["workspace"].data_ptr(), n)
    if case["op"] == "experts":
        state["plan"] = lh.moe_plan_raw(case["T"], case["E"], case["top_k"], state["offsets"].data_ptr(),
                                        state["order"].data_ptr())


def run(state):
    case, res = state["case"], state["result"]
    if not own:
        return {"quantize": _plain_quantize, "linear": _plain_linear, "experts": _plain_experts, "route": _plain_route,
                "combine": _plain_combine}[case["op"]](state)
    lh, stream, dtype, T = state["lh"], torch.cuda.current_stream().cuda_stream, case["dtype"], case["T"]
    if case["op"] == "quantize":
        lh.quantize_i8_raw(dtype, state["x"].data_ptr(), res["q"].data_ptr(), res["scale"].data_ptr(), case["K"], T,
                           case["K"], case["K"], stream=stream)
    elif case["op"] == "linear":
        lh.w8a8_raw(state["layer"], state["x"].data_ptr(), state["x_scale"].data_ptr(), T, case["K"], dtype,
                    res["y"].data_ptr(), res["y"].shape[1], stream=stream)
    elif case["op"] == "experts":
        lh.experts_w8a8_raw(state["plan"], state["layer"], state["x"].data_ptr(), state["x_scale"].data_ptr(), case["K"],
                            dtype, res["y"].data_ptr(), res["y"].shape[1], x_sorted=case["back"],
                            y_sorted=not case["back"], stream=stream)
    elif case["op"] == "route":
        lh.moe_route_raw(state["router"], dtype, state["logits"].data_ptr(), case["E"], T, res["ids"].data_ptr(),
                         res["weights"].data_ptr(), plan=state["plan"], stream=stream)
    else:
        lh.moe_combine_raw(dtype, state["y"].data_ptr(), case["N"], state["ids"].data_ptr(), state["weights"].data_ptr(),
                           T, case["top_k"], case["N"], res["out"].data_ptr(), case["N"],
                           base=state["base"].data_ptr() if state["base"] is not None else 0, ldb=case["N"],
                           stream=stream)
    return res


# ---- the plain form -------------------------------------------------------------------

def _plain_quantize(state):
    x, res = state["x"], state["result"]
    top = x.abs().amax(dim=1).double()
    res["scale"].copy_(top / 127.0)
    # the nearest integer to x / (top / 127), the quotient's border between two integers included
    res["q"].copy_(torch.round(x.double() * 127.0 / torch.where(top == 0, 1.0, top)[:, None]))
    return res


def _activate(act, x):
    if act == "relu":
        return torch.clamp(x, min=0.0)
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    if act == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))
    if act == "gelu_erf":
        return 0.5 * x * torch.erfc(x * -math.sqrt(0.5))
    return x


def _finish(case, y):
    """Activation and gate of the finished sums, (rows, N) in 32 bits."""
    if not case["gated"]:
        return _activate(case["act"], y)
    half = case["N"] // 2
    return _activate(case["act"], y[..., :half]) * y[..., half:]


def _plain_linear(state):
    y = (state["x"].float() @ state["w"].float().t()) * state["x_scale"][:, None] * state["w_scale"]
    if state["bias"] is not None:
        y = y + state["bias"]
    state["result"]["y"].copy_(_finish(state["case"], y))
    return state["result"]


def _plain_experts(state):
    case, E = state["case"], state["case"]["E"]
    start, end = state["offsets"][:-1].long(), state["offsets"][1:].long()
    place = start[:, None] + torch.arange(state["most"], device="cuda")   # of each expert's rows, padded to the most
    real = place < end[:, None]
    slot = state["order"].long()[torch.where(real, place, 0)]
    row = torch.where(real, place, 0) if case["back"] else slot // case["top_k"]
    x, x_scale = state["x"].float()[row], state["x_scale"][row]
    y = torch.bmm(x, state["w"].float().transpose(1, 2).contiguous()) * x_scale[:, :, None] * state["w_scale"][:, None, :]
    if state["bias"] is not None:
        y = y + state["bias"][:, None, :]
    y = _finish(case, y)
    to = slot if case["back"] else place
    state["result"]["y"][to[real]] = y[real].to(state["result"]["y"].dtype)
    return state["result"]


def _plain_route(state):
    case, res = state["case"], state["result"]
    E, k, G = case["E"], case["top_k"], case["groups"]
    x = state["logits"].double()
    p = 1.0 / (1.0 + torch.exp(-x))
    if case["score"] == "softmax":
        e = torch.exp(x - x.amax(dim=1, keepdim=True))
        p = e / e.sum(dim=1, keepdim=True)
    choice = p if state["bias"] is None else p + state["bias"].double()
    if case["top_groups"] < G:
        best = torch.sort(choice.view(-1, G, E // G), dim=2, descending=True).values[:, :, :case["group_best"]].sum(dim=2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = torch.where(open_[:, :, None], choice.view(-1, G, E // G), -math.inf).view(-1, E)
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, ids)
    if case["renormalize"]:
        w = w / w.sum(dim=1, keepdim=True)
    res["ids"].copy_(ids)
    res["weights"].copy_(w * case["scale"])
    order, offsets = _sorted_by_expert(ids, E)
    res["order"].copy_(order)
    res["offsets"].copy_(offsets)
    return res


def _plain_combine(state):
    case = state["case"]
    y = state["y"].float().view(case["T"], case["top_k"], case["N"])
    total = (y * state["weights"][:, :, None]).sum(dim=1)
    if state["base"] is not None:
        total = total + state["base"].float()
    state["result"]["out"].copy_(total)
    return state["result"]


# ---- the definition, in 64 bits -------------------------------------------------------

def exact(case, seed):
    x = _inputs(case, seed)
    return {"quantize": _exact_quantize, "linear": _exact_linear, "experts": _exact_experts, "route": _exact_route,
            "combine": _exact_combine}[case["op"]](case, x)


def _exact_quantize(case, x):
    q = torch.empty(x["x"].shape, dtype=torch.int8, device="cuda")
    scale = torch.empty(case["T"], dtype=torch.float64, device="cuda")
    for at in range(0, case["T"], 4096):
        rows = x["x"][at:at + 4096].double()
        most = torch.maximum(rows.amax(dim=1), -rows.amin(dim=1))
        # n is nearest where 127 |x| lies within half of `most` from n * most: whole products, no quotient
        a = 127.0 * rows.abs()
        n = torch.floor(a / most.clamp(min=1e-300)[:, None])
        rest = a - n * most[:, None]
        n = torch.where(rest >= most[:, None], n + 1, torch.where(rest < 0, n - 1, n))
        rest = 2.0 * (a - n * most[:, None]) - most[:, None]
        n = torch.where((rest > 0) | ((rest == 0) & (n % 2 == 1)), n + 1, n)
        q[at:at + 4096] = torch.where(most[:, None] > 0, n * torch.sign(rows), 0.0).to(torch.int8)
        scale[at:at + 4096] = most / 127.0
    return {"q": q, "scale": scale}


def _exact_act(case, y):
    f = {"none": lambda t: t, "relu": lambda t: t * (t > 0), "silu": lambda t: t * torch.sigmoid(t),
         "gelu_tanh": lambda t: t * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (t + 0.044715 * t ** 3)),
         "gelu_erf": lambda t: t * torch.special.ndtr(t)}[case["act"]]
    if not case["gated"]:
        return f(y)
    gate, other = y.split(case["N"] // 2, dim=-1)
    return f(gate) * other


def _exact_rows(case, x, rows, w, w_scale, bias):
    sums = x["x"][rows].double() @ w.double().t().contiguous()
    y = sums * torch.outer(x["x_scale"][rows].double(), w_scale.double())
    return _exact_act(case, y if bias is None else y + bias.double())


def _exact_linear(case, x):
    y = torch.empty(case["T"], case["N"] // 2 if case["gated"] else case["N"], dtype=torch.float64, device="cuda")
    for at in range(0, case["T"], 1024):
        rows = torch.arange(at, min(at + 1024, case["T"]), device="cuda")
        y[rows] = _exact_rows(case, x, rows, x["w"], x["w_scale"], x["bias"])
    return {"y": y}


def _exact_experts(case, x):
    y = torch.empty(case["T"] * case["top_k"], case["N"] // 2 if case["gated"] else case["N"], dtype=torch.float64,
                    device="cuda")
    ends = x["offsets"].tolist()
    for e in range(case["E"]):
        at = torch.arange(ends[e], ends[e + 1], device="cuda")
        if not len(at):
            continue
        slots = x["order"][at].long()
        rows, to = (at, slots) if case["back"] else (torch.div(slots, case["top_k"], rounding_mode="floor"), at)
        y[to] = _exact_rows(case, x, rows, x["w"][e], x["w_scale"][e], x["bias"][e] if x["bias"] is not None else None)
    return {"y": y}


def _exact_route(case, x):
    T, E, k, G = case["T"], case["E"], case["top_k"], case["groups"]
    logits = x["logits"].double()
    p = torch.softmax(logits, dim=1) if case["score"] == "softmax" else torch.sigmoid(logits)
    left = p.clone() if x["bias"] is None else p + x["bias"].double()
    number = torch.arange(E, device="cuda")

    def highest(v):
        """The highest of each row, and the first place that has it."""
        top = v.amax(dim=1)
        return top, torch.where(v == top[:, None], number[:v.shape[1]], E).amin(dim=1)

    if case["top_groups"] < G:
        best = torch.zeros(T, G, dtype=torch.float64, device="cuda")
        inside = left.reshape(T * G, E // G).clone()
        for _ in range(case["group_best"]):
            top, at = highest(inside)
            best += top.view(T, G)
            inside[torch.arange(T * G, device="cuda"), at] = -math.inf
        closed = torch.ones(T, G, dtype=torch.bool, device="cuda")
        for _ in range(case["top_groups"]):
            _, at = highest(best)
            closed[torch.arange(T, device="cuda"), at] = False
            best[torch.arange(T, device="cuda"), at] = -math.inf
        left[closed.repeat_interleave(E // G, dim=1)] = -math.inf
    ids = torch.empty(T, k, dtype=torch.int64, device="cuda")
    for j in range(k):
        ids[:, j] = highest(left)[1]
        left[torch.arange(T, device="cuda"), ids[:, j]] = -math.inf
    w = p[torch.arange(T, device="cuda")[:, None], ids]
    w = case["scale"] * (w / w.sum(dim=1, keepdim=True) if case["renormalize"] else w)
    # an assignment's place: the assignments of lower experts, and those of its own in front of it
    flat = ids.reshape(-1)
    ahead = torch.zeros(E, dtype=torch.int64, device="cuda")
    within = torch.empty_like(flat)
    for at in range(0, len(flat), 1 << 16):
        hit = torch.nn.functional.one_hot(flat[at:at + (1 << 16)], E).to(torch.int32)
        within[at:at + (1 << 16)] = ((hit.cumsum(dim=0) - hit) * hit).sum(dim=1) + ahead[flat[at:at + (1 << 16)]]
        ahead += hit.sum(dim=0)
    offsets = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = ahead.cumsum(dim=0)
    order = torch.empty_like(flat)
    order[offsets[flat] + within] = torch.arange(len(flat), device="cuda")
    return {"ids": ids.to(torch.int32), "weights": w, "order": order.to(torch.int32), "offsets": offsets.to(torch.int32)}


def _exact_combine(case, x):
    y = x["y"].view(case["T"], case["top_k"], case["N"])
    out = x["base"].double() if x["base"] is not None else torch.zeros(case["T"], case["N"], dtype=torch.float64,
                                                                      device="cuda")
    for j in range(case["top_k"]):
        out = out + x["weights"][:, j, None].double() * y[:, j].double()
    return {"out": out}
