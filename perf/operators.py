"""The operators of a serving step over a paged key/value cache, as cases that can be timed: keys and values
appended to the cache with their rotation (`kv_append`), attention of new tokens over it (`paged_attn`), and the
same for sequences that share a long prefix (`shared_prefix_attn`).

`run` computes them in plain torch operations in 32 bits, or, with `own` set, by the calls that a user of
lava_hip makes.  A cache is a pair of tensors of pages, (pages, heads, page_size, D) ("hl") or
(pages, page_size, heads, D) ("lh"); tokens of a batch are packed, (tokens, heads, D).
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16}


def _case(op, dtype, Hq, Hkv, D, page, B, q, kv, **more):
    """q, kv: [least, most] new tokens and tokens in the cache (those of the call included) of a sequence."""
    case = {"op": op, "dtype": dtype, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "order": "hl", "B": B,
            "q_lo": q[0], "q_hi": q[1], "kv_lo": kv[0], "kv_hi": kv[1], "lengths": 1,
            "causal": True, "window": 0, "cap": 0.0, "slopes": False, "bidir": 0.0, "prefix": 0,
            "rot": 0, "interleaved": False}
    case.update(more)
    return case


def listed():
    return [
        # one decode step's tokens of 64 sequences: a few hundred kilobytes, latency is all there is
        {"name": "append_decode64", **_case("append", "f16", 32, 8, 128, 16, 64, (1, 1), (1, 4096), rot=128)},
        # prompts' tokens, half of each head rotated in adjacent pairs: bound by HBM
        {"name": "append_prompts", **_case("append", "bf16", 32, 8, 128, 64, 16, (333, 4096), (333, 4096), rot=64,
                                           interleaved=True, order="lh")},
        # one user's decode step over a short context: the smallest attention call
        {"name": "decode_single", **_case("attn", "f16", 32, 8, 128, 16, 1, (1, 1), (777, 777))},
        # a served batch of ragged contexts: bound by the cache's bytes
        {"name": "decode_batch64", **_case("attn", "bf16", 32, 8, 128, 16, 64, (1, 1), (100, 8192))},
        # few very long contexts, capped scores: work split along the keys
        {"name": "decode_long_capped", **_case("attn", "f16", 16, 2, 128, 64, 3, (1, 1), (30000, 131071), cap=50.0)},
        # four drafted tokens a sequence checked at once, a head for a head, windows and distance bias
        {"name": "decode_drafts_window", **_case("attn", "f16", 12, 12, 64, 32, 32, (1, 4), (5, 4096), window=1024,
                                                 slopes=True)},
        # the attention benchmark's prompts, with grouped heads, through the cache
        {"name": "prompt_4096", **_case("attn", "f16", 32, 8, 128, 64, 4, (4096, 4096), (4096, 4096))},
        # chunks of prompts behind what the cache holds already, beside sequences that decode; capped scores
        {"name": "prompt_chunks_capped", **_case("attn", "bf16", 32, 8, 128, 16, 12, (1, 777), (777, 6000), cap=30.0)},
        # an instruction read both ways, then causal; odd lengths, D = 64
        {"name": "prompt_bidirectional", **_case("attn", "bf16", 12, 12, 64, 32, 8, (301, 1537), (301, 1537), bidir=0.4,
                                                 order="lh")},
        # a few answers to one prompt, small
        {"name": "shared_samples8", **_case("shared", "f16", 32, 8, 128, 16, 8, (1, 1), (1, 64), prefix=1024)},
        # a served batch behind one long system prompt
        {"name": "shared_batch64", **_case("shared", "bf16", 32, 8, 128, 16, 64, (1, 1), (1, 1000), prefix=8192)},
        # a long document asked about by many, a few tokens each
        {"name": "shared_document", **_case("shared", "f16", 32, 4, 128, 64, 48, (1, 6), (6, 300), prefix=32768,
                                            cap=50.0)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "attn", "shared"])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (32, 32), (12, 12), (16, 2), (28, 4), (64, 8), (8, 1)])
    D = rng.choice([64, 64, 80, 96, 128, 128, 128, 128, 256])
    common = {"page": rng.choice([16, 16, 32, 64, 128, 8 * rng.randint(1, 40)]), "dtype": rng.choice(["f16", "bf16"]),
              "order": rng.choice(["hl", "lh"]), "lengths": rng.randrange(1 << 20)}
    mods = {"cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "slopes": rng.random() < 0.25,
            "window": _log(rng, 16, 4096) if rng.random() < 0.25 else 0}

    def case(q, kv, B, **more):
        return _case(op, common["dtype"], Hq, Hkv, D, common["page"], B, q, kv,
                     **{"order": common["order"], "lengths": common["lengths"], **more})

    if op == "append":
        top = _log(rng, 1, 4096)
        got = case((rng.randint(1, top), top), (top, _log(rng, top, 3 * top)), _log(rng, 1, 64),
                   rot=rng.choice([D, D, D // 2]), interleaved=rng.random() < 0.5)
    elif op == "shared":
        top = rng.choice([1, 1, 1, 4, 16])
        got = case((1, top), (top, _log(rng, top, 2000)), _log(rng, 2, 64), prefix=_log(rng, 100, 32768), **mods)
    elif rng.random() < 0.5:   # decode
        top = rng.choice([1, 1, 1, 2, 4])
        hi = _log(rng, top, 65536)
        got = case((rng.randint(0, 1), top), (min(hi, _log(rng, top, hi)), hi), _log(rng, 1, 64), **mods)
    else:
        top = _log(rng, 8, 4096)
        causal = rng.random() < 0.85
        if causal and rng.random() < 0.25:
            mods["bidir"] = 0.4
        hi = _log(rng, top, max(top, 8192))
        got = case((rng.randint(1, top), top), (top, hi), _log(rng, 1, 8), causal=causal, **mods)
    # no more than the largest listed call of the operator
    bytes_, flops = {"append": (6.5e8, 1e12), "attn": (1.1e9, 5e11), "shared": (1.1e9, 1e11)}[op]
    while work(got)["bytes"] > bytes_ or work(got)["flops"] > flops:
        if got["B"] > 1:
            got["B"] = got["B"] * 2 // 3
        else:
            for n in ("q_lo", "q_hi", "kv_lo", "kv_hi"):
                got[n] = max(1, got[n] * 2 // 3)
    return got


# ---- lengths: given by the case alone -------------------------------------------------

def _lengths(case):
    """(new tokens, tokens in the cache) of each sequence; for shared prefixes the cache's own part."""
    rng = random.Random(case["lengths"])
    got = []
    for b in range(case["B"]):
        kv = rng.randint(case["kv_lo"], case["kv_hi"])
        n = min(kv, rng.randint(case["q_lo"], case["q_hi"]))
        got.append((max(1, n) if b == 0 else n, kv))   # some sequences may wait, not all of them
    return got


def _bidir(case, kv):
    """How many leading keys every query of a sequence of kv tokens sees."""
    return int(case["bidir"] * kv)


def _visible(case):
    """Query-key pairs, and keys that some query of their sequence sees (a shared prefix counted once)."""
    pairs = keys = 0
    low = case["prefix"]
    for n, kv in _lengths(case):
        if n == 0:
            continue
        end = case["prefix"] + kv
        first = end - n   # position of the first query
        bid, w = _bidir(case, kv), case["window"]
        for pos in range(first, end):
            hi = max(pos, bid - 1) if case["causal"] else end - 1
            lo = max(0, pos - w + 1) if w else 0
            pairs += max(0, hi - lo + 1)
        lo = max(0, first - w + 1) if w else 0
        keys += end - max(lo, case["prefix"])
        low = min(low, lo)
    return pairs, keys + case["prefix"] - low


def work(case):
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    tokens = sum(n for n, _ in _lengths(case))
    if case["op"] == "append":
        rotated = tokens * (Hq + Hkv) * case["rot"]
        return {"bytes": 2 * 2 * tokens * (Hq + 2 * Hkv) * D, "flops": 3 * rotated}
    pairs, keys = _visible(case)
    return {"bytes": 2 * 2 * keys * Hkv * D + 2 * 2 * tokens * Hq * D, "flops": 4 * pairs * Hq * D}


# ---- what a program has in hand -------------------------------------------------------

def _cache_shape(case, pages):
    h, l = case["Hkv"], case["page"]
    return (pages, h, l, case["D"]) if case["order"] == "hl" else (pages, l, h, case["D"])


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, page = _TORCH[case["dtype"]], case["page"]
    lens = _lengths(case)
    counts = [-(-kv // page) for _, kv in lens]
    shared = -(-case["prefix"] // page)
    pages = sum(counts) + shared + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((case["B"], max(counts + [1])), -1, dtype=torch.int32, device="cuda")
    at = shared
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    q_start = [0]
    for n, _ in lens:
        q_start.append(q_start[-1] + n)

    def normal(*shape):
        return torch.randn(shape, dtype=dt, device="cuda", generator=g)

    got = {"k": normal(*_cache_shape(case, pages)), "v": normal(*_cache_shape(case, pages)), "table": table,
           "prefix_pages": order[:shared].contiguous(), "tokens": q_start[-1],
           "q_start": torch.tensor(q_start, dtype=torch.int32, device="cuda"),
           "kv_len": torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")}
    if case["op"] == "append":   # the projections' result, Q, K and V side by side
        got["qkv"] = normal(got["tokens"], case["Hq"] + 2 * case["Hkv"], case["D"])
        half = case["rot"] // 2
        got["inv_freq"] = 10000.0 ** (-torch.arange(half, dtype=torch.float32, device="cuda") / half)
    else:
        # keys and queries of a trained layer agree with a few tokens more than with the rest
        got["q"] = normal(got["tokens"], case["Hq"], case["D"]) * 1.5
        got["slopes"] = (2.0 ** (-8.0 * torch.arange(1, case["Hq"] + 1, dtype=torch.float32, device="cuda") / case["Hq"])
                         if case["slopes"] else None)
        got["bidir"] = (torch.tensor([_bidir(case, kv) for _, kv in lens], dtype=torch.int32, device="cuda")
                        if case["bidir"] else None)
    return got


def prepare(case, seed):
    state = {"case": case, "lens": _lengths(case), **_inputs(case, seed)}
    state["out"] = torch.empty((state["tokens"], case["Hq"], case["D"]), dtype=_TORCH[case["dtype"]], device="cuda")
    if own:
        _describe(state)
    return state


def _describe(state):
    """The descriptors of the cache, the batch and the scores that a serving program keeps."""
    package = str(Path(__file__).resolve().parents[1] / "lava.jl_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    import lava_hip as lh
    lh.init()
    case = state["case"]
    h, l, d = case["Hkv"], case["page"], case["D"]
    strides = (1, d, l * d, h * l * d) if case["order"] == "hl" else (1, h * d, d, h * l * d)   # of (E, L, H, P)
    state["lh"] = lh
    state["cache"] = lh.paged_cache_raw(case["dtype"], state["k"].data_ptr(), state["v"].data_ptr(), d, l, h,
                                        state["k"].shape[0], strides)
    state["batch"] = lh.paged_batch_raw(case["B"], state["tokens"], state["q_start"].data_ptr(),
                                        state["kv_len"].data_ptr(), state["table"].data_ptr(), state["table"].shape[1],
                                        max_q=max(n for n, _ in state["lens"]))
    if case["op"] == "append":
        state["rope"] = lh.rope_raw(state["inv_freq"].data_ptr(), case["rot"], interleaved=case["interleaved"])
        return
    state["score"] = lh.attn_score_raw(1.0 / math.sqrt(d), causal=case["causal"], window=case["window"],
                                       cap=case["cap"],
                                       slopes=state["slopes"].data_ptr() if state["slopes"] is not None else 0,
                                       bidirectional=state["bidir"].data_ptr() if state["bidir"] is not None else 0)


def run(state):
    case = state["case"]
    if not own:
        return {"append": _plain_append, "attn": _plain_attn, "shared": _plain_shared}[case["op"]](state)
    lh, out, d, Hq = state["lh"], state["out"], case["D"], case["Hq"]
    stream = torch.cuda.current_stream().cuda_stream
    packed = (1, d, Hq * d)   # of (E, H, T)
    if case["op"] == "append":
        q = state["qkv"].data_ptr()
        fused = (1, d, (Hq + 2 * case["Hkv"]) * d)
        lh.kv_append_raw(state["cache"], state["batch"], q + 2 * Hq * d, q + 2 * (Hq + case["Hkv"]) * d, fused, Q=q,
                         Q_out=out.data_ptr(), q_heads=Hq, q_strides=fused, qo_strides=packed, rope=state["rope"],
                         stream=stream)
        return {"q": out, "k": state["k"], "v": state["v"]}
    if case["op"] == "attn":
        lh.paged_attn_raw(state["cache"], state["batch"], state["score"], state["q"].data_ptr(), out.data_ptr(), Hq,
                          packed, packed, stream=stream)
    else:
        lh.shared_prefix_attn_raw(state["cache"], state["batch"], state["score"], state["prefix_pages"].data_ptr(),
                                  case["prefix"], state["q"].data_ptr(), out.data_ptr(), Hq, packed, packed,
                                  stream=stream)
    return out


# ---- the plain form -------------------------------------------------------------------

def _plain_append(state):
    case, page = state["case"], state["case"]["page"]
    Hq, Hkv, rot = case["Hq"], case["Hkv"], case["rot"]
    q_len = state["q_start"][1:].long() - state["q_start"][:-1].long()
    seq = torch.repeat_interleave(torch.arange(case["B"], device="cuda"), q_len, output_size=state["tokens"])
    pos = torch.arange(state["tokens"], device="cuda") - state["q_start"].long()[seq] + (state["kv_len"].long() - q_len)[seq]
    angle = pos.double()[:, None] * state["inv_freq"].double()[None, :]
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]

    def rotate(x):
        x = x.float()
        if case["interleaved"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        else:
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        return torch.cat((turned, x[..., rot:]), dim=-1).to(state["out"].dtype)

    qkv = state["qkv"]
    state["out"].copy_(rotate(qkv[:, :Hq]))
    where, row = state["table"].long()[seq, pos // page], pos % page
    for cache, x in ((state["k"], rotate(qkv[:, Hq:Hq + Hkv])), (state["v"], qkv[:, Hq + Hkv:])):
        if case["order"] == "hl":
            cache[where, :, row] = x
        else:
            cache[where, row] = x
    return {"q": state["out"], "k": state["k"], "v": state["v"]}


def _gather(state, cache, pages, n):
    """The first n keys (values) of the listed pages, (heads, n, D) in 32 bits."""
    got = cache[pages.long()]
    if state["case"]["order"] == "lh":
        got = got.transpose(1, 2)
    return got.transpose(0, 1).reshape(state["case"]["Hkv"], -1, state["case"]["D"])[:, :n].float()


def _plain_sequence(state, q, k, v, first, bid):
    """softmax attention of q (n, Hq, D), the first at position `first`, over k and v (Hkv, L, D)."""
    case = state["case"]
    n, L, Hkv = q.shape[0], k.shape[1], case["Hkv"]
    G = case["Hq"] // Hkv
    rows = q.float().reshape(n, Hkv, G, -1).permute(1, 2, 0, 3).reshape(Hkv, G * n, -1)
    s = torch.bmm(rows, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(case["D"]))
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    s = s.view(Hkv, G, n, L)
    pos = torch.arange(first, first + n, device="cuda")[:, None]
    key = torch.arange(L, device="cuda")[None, :]
    if state["slopes"] is not None:
        s = s - state["slopes"].view(Hkv, G, 1, 1) * (pos - key).abs().float()
    keep = (key <= pos) | (key < bid) if case["causal"] else torch.ones_like(key <= pos)
    if case["window"]:
        keep = keep & (key > pos - case["window"])
    s = s.masked_fill(~keep, -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.bmm(p.view(Hkv, G * n, L), v).view(Hkv, G, n, -1) / torch.where(total == 0, 1.0, total)
    return o.permute(2, 0, 1, 3).reshape(n, case["Hq"], -1)


def _plain_attn(state):
    at = 0
    for b, (n, kv) in enumerate(state["lens"]):
        if n:
            pages = state["table"][b, :-(-kv // state["case"]["page"])]
            k, v = _gather(state, state["k"], pages, kv), _gather(state, state["v"], pages, kv)
            state["out"][at:at + n] = _plain_sequence(state, state["q"][at:at + n], k, v, kv - n,
                                                      _bidir(state["case"], kv)).to(state["out"].dtype)
        at += n
    return state["out"]


def _plain_shared(state):
    case, at = state["case"], 0
    P = case["prefix"]
    k0, v0 = _gather(state, state["k"], state["prefix_pages"], P), _gather(state, state["v"], state["prefix_pages"], P)
    for b, (n, kv) in enumerate(state["lens"]):
        if n:
            pages = state["table"][b, :-(-kv // case["page"])]
            k = torch.cat((k0, _gather(state, state["k"], pages, kv)), dim=1)
            v = torch.cat((v0, _gather(state, state["v"], pages, kv)), dim=1)
            state["out"][at:at + n] = _plain_sequence(state, state["q"][at:at + n], k, v, P + kv - n,
                                                      0).to(state["out"].dtype)
        at += n
    return state["out"]


# ---- the definition, in 64 bits -------------------------------------------------------

def exact(case, seed):
    x = _inputs(case, seed)
    return _exact_append(case, x) if case["op"] == "append" else _exact_attn(case, x)


def _exact_append(case, x):
    Hq, Hkv, rot, page = case["Hq"], case["Hkv"], case["rot"], case["page"]
    k, v = x["k"].double(), x["v"].double()
    q = torch.empty((x["tokens"], Hq, case["D"]), dtype=torch.float64, device="cuda")
    j = torch.arange(rot // 2, device="cuda")
    first, second = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + rot // 2)
    at = 0
    for b, (n, kv) in enumerate(_lengths(case)):
        if n == 0:
            continue
        pos = torch.arange(kv - n, kv, device="cuda")
        part = x["qkv"][at:at + n].double()
        turn = torch.polar(torch.ones(n, rot // 2, dtype=torch.float64, device="cuda"),
                           torch.outer(pos.double(), x["inv_freq"].double()))[:, None, :]
        heads = part[:, :Hq + Hkv]
        z = torch.complex(heads[:, :, first], heads[:, :, second]) * turn
        heads[:, :, first], heads[:, :, second] = z.real, z.imag
        q[at:at + n] = heads[:, :Hq]
        pages = x["table"][b].long()[torch.div(pos, page, rounding_mode="floor")]
        for i in range(Hkv):   # one head at a time: (n, D) rows
            if case["order"] == "hl":
                k[pages, i, pos % page] = heads[:, Hq + i]
                v[pages, i, pos % page] = part[:, Hq + Hkv + i]
            else:
                k[pages, pos % page, i] = heads[:, Hq + i]
                v[pages, pos % page, i] = part[:, Hq + Hkv + i]
        at += n
    return {"q": q, "k": k, "v": v}


def _exact_attn(case, x):
    G, D, page, P = case["Hq"] // case["Hkv"], case["D"], case["page"], case["prefix"]
    lens = _lengths(case)
    pairs = sum(n * (P + kv) for n, kv in lens) * case["Hq"]
    if pairs * (4 * D + 60) > 2e13 or sum(1 for n, _ in lens if n) * case["Hq"] > 30000:
        return None
    out = torch.empty((x["tokens"], case["Hq"], D), dtype=torch.float64, device="cuda")

    def head(cache, b, i, kv):
        """Keys (values) of sequence b and key head i in order, token by token."""
        own_keys = torch.arange(kv, device="cuda")
        both = [(x["table"][b].long()[own_keys // page], own_keys % page)]
        if P:
            j = torch.arange(P, device="cuda")
            both.insert(0, (x["prefix_pages"].long()[j // page], j % page))
        at_page, row = (torch.cat(t) for t in zip(*both))
        return (cache[at_page, i, row] if case["order"] == "hl" else cache[at_page, row, i]).double()

    at = 0
    for b, (n, kv) in enumerate(lens):
        if n == 0:
            continue
        end = P + kv
        for i in range(case["Hkv"]):
            k, v = head(x["k"], b, i, kv), head(x["v"], b, i, kv)
            kt = k.t().contiguous()
            for r0 in range(0, n, 2048):   # rows of scores that fit
                rows = slice(r0, min(n, r0 + 2048))
                dist = (torch.arange(end - n + rows.start, end - n + rows.stop, device="cuda")[:, None]
                        - torch.arange(end, device="cuda")[None, :])
                seen = torch.ones_like(dist, dtype=torch.bool)
                if case["causal"]:
                    seen = dist >= 0
                    seen[:, :_bidir(case, kv)] = True
                if case["window"]:
                    seen &= dist < case["window"]
                for h in range(i * G, (i + 1) * G):
                    t = x["q"][at + rows.start:at + rows.stop, h].double() @ kt / math.sqrt(D)
                    if case["cap"]:
                        t = torch.tanh(t / case["cap"]) * case["cap"]
                    if x["slopes"] is not None:
                        t -= dist.abs() * x["slopes"][h].double()
                    w = torch.softmax(torch.where(seen, t, -math.inf), dim=-1)
                    out[at + rows.start:at + rows.stop, h] = torch.nan_to_num(w) @ v
        at += n
    return out
