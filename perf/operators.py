"""The operators between the products that this library is measured on: their plain forms in torch,
the calls that a program makes of them (include/q8_mix.h), and their answers in 64 bits.

  conv   the short causal convolution of each channel with SiLU, behind a DeltaNet layer's QKV product
  delta  the gated delta rule with its output norm and gate, one token or many, from and to a state
  rope   the norm of each head of queries and keys with the rotation of positions, and the keys' and
         values' way into a paged cache
  attn   attention of each sequence's newest tokens over the paged cache, with the output gate

The head counts and sizes are those of the layers whose products the library runs: on a hidden size
of 4096, 16 key and 32 value heads of 128 for the delta rule (QKV 8192 wide) and 16 query heads on 4
key-value heads of 256, 64 of which turn; on 2048, 16 key and 16 value heads of 128, and 8 query
heads on 2 key-value heads.
"""
import ctypes as c
import importlib.util
import math
import os
import random
import sys

import torch

own = False
_SHARED = {}
EPS = 1e-6
CHUNK = 64


def listed():
    nine = {"kind": "delta", "k_heads": 16, "v_heads": 32, "k_dim": 128, "v_dim": 128, "tiled": True, "gated": True}
    attn = {"kind": "attn", "q_heads": 16, "kv_heads": 4, "dim": 256, "gated": True}
    return [
        # one step of decoding for four users: latency alone
        {"name": "conv_decode_4", "kind": "conv", "ch": 8192, "taps": 4, "n": 4, "low": 1, "high": 1},
        # prompts of three requests in one call
        {"name": "conv_prompt", "kind": "conv", "ch": 8192, "taps": 4, "n": 3, "low": 301, "high": 2048},
        # a decode step of one sequence, and of a serving batch
        {"name": "delta_decode_1", **nine, "n": 1, "low": 1, "high": 1},
        {"name": "delta_decode_64", **nine, "n": 64, "low": 1, "high": 1},
        # a token and its three drafts, as speculative decoding checks them
        {"name": "delta_verify_8", **nine, "n": 8, "low": 4, "high": 4},
        # prompts of odd lengths on the small model's heads, the plain rule without its output norm
        {"name": "delta_prompt_2b", **nine, "v_heads": 16, "tiled": False, "gated": False, "n": 3, "low": 77, "high": 1003},
        # a long prompt of one request
        {"name": "delta_prompt_long", **nine, "n": 1, "low": 8192, "high": 8192},
        # heads of one new token, late in a long sequence; and of prompts
        {"name": "rope_decode_1", "kind": "rope", "q_heads": 16, "kv_heads": 4, "dim": 256, "rot": 64, "pairs": False, "norm": True, "type": "f16",
         "n": 1, "low": 1, "high": 1, "past": 100003, "page": 64},
        {"name": "rope_prompt", "kind": "rope", "q_heads": 16, "kv_heads": 4, "dim": 256, "rot": 64, "pairs": False, "norm": True, "type": "bf16",
         "n": 3, "low": 300, "high": 2048, "past": 1000, "page": 16},
        # one user's next token on a short history in the engine's own type
        {"name": "attn_decode_1", **attn, "type": "f32", "page": 64, "n": 1, "tokens": 1, "low": 777, "high": 777},
        # a serving batch of mixed lengths
        {"name": "attn_decode_32", **attn, "type": "f16", "page": 16, "n": 32, "tokens": 1, "low": 100, "high": 16384},
        # a token and its drafts at the end of a very long history
        {"name": "attn_verify_long", **attn, "type": "bf16", "page": 64, "n": 1, "tokens": 4, "low": 131072, "high": 131072},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["conv", "delta", "delta", "rope", "attn", "attn"])
    if kind == "conv":
        n = _log(rng, 1, 64)
        high = _log(rng, 1, 6000 // n)
        return {"kind": "conv", "ch": 4 * _log(rng, 128, 2048), "taps": rng.choice([2, 3, 4, 4, 4]), "n": n, "low": max(1, high // rng.randint(1, 8)), "high": high}
    if kind == "delta":
        kh = rng.choice([4, 8, 16])
        case = {"kind": "delta", "k_heads": kh, "v_heads": kh * rng.choice([1, 2]), "k_dim": rng.choice([64, 128, 128, 128, 256]), "v_dim": rng.choice([48, 64, 128, 128, 128]),
                "tiled": rng.random() < 0.5, "gated": rng.random() < 0.7}
        if rng.random() < 0.5:
            high = rng.choice([1, 1, rng.randint(2, 8)])
            return {**case, "n": _log(rng, 1, 96), "low": 1, "high": high}
        n = _log(rng, 1, 6)
        high = _log(rng, 20, 6000 // n)
        return {**case, "k_dim": min(case["k_dim"], 128), "n": n, "low": max(1, high // rng.randint(1, 6)), "high": high}
    kv = rng.choice([1, 2, 4, 8])
    case = {"kind": kind, "q_heads": kv * rng.choice([1, 2, 4, 4, 6, 8]), "kv_heads": kv, "dim": rng.choice([64, 96, 128, 128, 256, 256]), "type": rng.choice(["f32", "f16", "bf16"]),
            "page": rng.choice([16, 16, 24, 64, 256])}
    if kind == "rope":
        n = _log(rng, 1, 64)
        high = rng.choice([1, _log(rng, 1, max(1, 4000 // n))])
        return {**case, "rot": rng.choice([case["dim"], case["dim"] // 2, 32]), "pairs": rng.random() < 0.3, "norm": rng.random() < 0.8, "n": n,
                "low": max(1, high // rng.randint(1, 8)), "high": high, "past": _log(rng, 1, 200000 // n)}
    n = _log(rng, 1, 64)
    high = _log(rng, 17, min(100000, 400000 // n) // max(1, kv * case["dim"] // 512) // (2 if case["type"] == "f32" else 1))
    return {**case, "gated": rng.random() < 0.7, "n": n, "tokens": rng.choice([1, 1, 1, 2, 3, 4, 6]), "low": max(8, high // rng.randint(1, 20)), "high": high}


def _lengths(case):
    """Each sequence's tokens (of an attention case: its cached positions), odd and even, between low and high; one of them high."""
    rng = random.Random(case["n"] * 7919 + case["high"] * 31 + case["low"])
    return [case["high"]] + [rng.randint(case["low"], case["high"]) for _ in range(case["n"] - 1)]


TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the inputs


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
    start = [0]
    for v in counts:
        start.append(start[-1] + v)
    return start


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale)

    def uniform(*shape, low=0.0, high=1.0):
        return torch.rand(*shape, generator=gen, device="cuda").mul_(high - low).add_(low)

    n, kind = case["n"], case["kind"]
    lengths = _lengths(case)
    new = [case["tokens"]] * n if kind == "attn" else lengths
    start = _starts(new)
    t = start[-1]
    s = {"case": case, "t": t, "longest": max(new), "start": _ints(start)}
    if kind == "conv":
        s["x"], s["w"], s["s_in"] = normal(t, case["ch"]), normal(case["ch"], case["taps"], scale=0.5), normal(n, case["taps"] - 1, case["ch"])
        s["s_out"], s["y"] = torch.empty_like(s["s_in"]), torch.empty_like(s["x"])
    elif kind == "delta":
        hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
        # the convolution's outputs: queries, keys and values of a token side by side
        s["x"] = torch.nn.functional.silu(normal(t, 2 * hk * dk + hv * dv))
        s["a"], s["b"] = normal(t, hv), normal(t, hv)
        # decays as they are trained: rates of 1 to 16 times steps of 0.001 to 0.1
        s["decay"] = -torch.exp(uniform(hv, high=math.log(16.0)))
        s["dt"] = torch.log(torch.expm1(torch.exp(uniform(hv, low=math.log(1e-3), high=math.log(0.1)))))
        s["s_in"] = normal(n, hv, dk, dv, scale=0.2)
        s["s_out"], s["o"] = torch.empty_like(s["s_in"]), torch.empty(t, hv * dv, device="cuda")
        if case["gated"]:
            s["z"], s["nw"] = normal(t, hv * dv), 1.0 + 0.1 * normal(dv)
    else:
        hq, hk, d, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
        if kind == "rope":
            total = [case["past"] + v for v in new]
        else:
            total = [max(v, case["tokens"]) for v in lengths]
        s["past"] = _ints([a - b for a, b in zip(total, new)])
        s["most"] = max(total)
        s["freq"] = (1e7 ** (-torch.arange(0, case.get("rot", 2), 2, dtype=torch.float64) / max(1, case.get("rot", 2)))).cuda()
        # each query's gate lies beside it, as the query product gives them
        s["qg"] = normal(t, hq, 2 * d)
        # the rotation's call touches the new tokens' pages alone, so only those are there for it
        first = [(b - a) // page if kind == "rope" else 0 for a, b in zip(new, total)]
        need = [-(-v // page) - f for v, f in zip(total, first)]
        s["pages"] = sum(need) + 1
        order = torch.randperm(s["pages"], generator=gen, device="cuda").int()
        s["table"] = torch.full((n, max(f + m for f, m in zip(first, need))), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, (f, m) in enumerate(zip(first, need)):
            s["table"][i, f:f + m] = order[at:at + m]
            at += m
        shape, kind_of = (s["pages"], hk, page, d), TYPES[case["type"]]
        if kind == "rope":
            s["k"], s["v"] = normal(t, hk, d), normal(t, hk, d)
            s["q_norm"], s["k_norm"] = 1.0 + 0.1 * normal(d), 1.0 + 0.1 * normal(d)
            s["ck"], s["cv"] = torch.zeros(shape, dtype=kind_of, device="cuda"), torch.zeros(shape, dtype=kind_of, device="cuda")
            s["out"] = torch.empty(t, hq, d, device="cuda")
        else:
            s["ck"], s["cv"] = (torch.empty(shape, dtype=kind_of, device="cuda").normal_(generator=gen) for _ in range(2))
            s["qg"][:, :, :d] *= 1.5
            s["o"] = torch.empty(t, hq * d, device="cuda")
    return s


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _bind(state)
        fn, args, out = state["call"]
        fn(*args)
        return out
    return {"conv": _conv, "delta": _delta, "rope": _rope, "attn": _attn}[state["case"]["kind"]](state)


# ---- the library's calls


def _runtime():
    if "rt" not in _SHARED:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        if "q8rt" not in sys.modules:
            spec = importlib.util.spec_from_file_location("q8rt", os.path.join(root, "intel-phi-apl_amd", "__init__.py"))
            sys.modules["q8rt"] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules["q8rt"])
        _SHARED["rt"] = sys.modules["q8rt"].Runtime()
    return _SHARED["rt"], sys.modules["q8rt"]


def _bind(s):
    """(the entry point, its arguments, its outputs): the structures that a program fills once for its buffers."""
    rt, m = _runtime()
    case = s["case"]
    kind, n = case["kind"], case["n"]

    def p(name):
        return s[name].data_ptr() if name in s else None

    seqs = m.Seqs(n=n, t=s["t"], longest=s["longest"], start=p("start"), past=p("past"))
    if kind == "conv":
        return rt.lib.rt_conv_silu_dev, (rt.R, c.byref(seqs), p("x"), case["ch"], case["ch"], p("w"), case["taps"], p("s_in"), p("s_out"), p("y"), case["ch"]), \
            {"y": s["y"], "state": s["s_out"]}
    if kind == "delta":
        hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
        ld, x = 2 * hk * dk + hv * dv, p("x")
        a = m.Delta(k_heads=hk, v_heads=hv, k_dim=dk, v_dim=dv, tiled=case["tiled"], q=x, q_ld=ld, k=x + 4 * hk * dk, k_ld=ld, v=x + 8 * hk * dk, v_ld=ld,
                    a=p("a"), a_ld=hv, b=p("b"), b_ld=hv, decay=p("decay"), dt=p("dt"), eps=EPS, scale=dk ** -0.5, s_in=p("s_in"), s_out=p("s_out"),
                    z=p("z"), z_ld=hv * dv, nw=p("nw"), nw_eps=EPS, o=p("o"), o_ld=hv * dv)
        return rt.lib.rt_delta_rule_dev, (rt.R, c.byref(seqs), c.byref(a)), {"o": s["o"], "state": s["s_out"]}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    kv = m.Kv(k=p("ck"), v=p("cv"), type=m.TYPES[case["type"]], dim=d, heads=hk, page=case["page"], pages=s["pages"], table=p("table"), table_ld=s["table"].shape[1])
    if kind == "rope":
        a = m.Rope(q=p("qg"), q_ld=2 * hq * d, q_hd=2 * d, q_heads=hq, k=p("k"), k_ld=hk * d, k_hd=d, v=p("v"), v_ld=hk * d, v_hd=d,
                   q_norm=p("q_norm") if case["norm"] else None, k_norm=p("k_norm") if case["norm"] else None, eps=EPS, rot=case["rot"], pairs=case["pairs"],
                   freq=p("freq"), out=p("out"), out_ld=hq * d, out_hd=d)
        return rt.lib.rt_rope_kv_dev, (rt.R, c.byref(seqs), c.byref(kv), c.byref(a)), {"q": s["out"], "k": s["ck"], "v": s["cv"]}
    a = m.Attn(q=p("qg"), q_ld=2 * hq * d, q_hd=2 * d, q_heads=hq, scale=d ** -0.5, gate=p("qg") + 4 * d if case["gated"] else None, gate_ld=2 * hq * d, gate_hd=2 * d,
               o=p("o"), o_ld=hq * d)
    return rt.lib.rt_attn_kv_dev, (rt.R, c.byref(seqs), c.byref(kv), c.byref(a)), {"o": s["o"]}


# ---- the plain forms, in 32 bits


def _sequence(s):
    """The sequence of each token and its place in it."""
    i = torch.arange(s["t"], device="cuda")
    seq = torch.searchsorted(s["start"].long(), i, right=True) - 1
    return seq, i - s["start"][seq].long()


def _conv(s):
    taps, n = s["case"]["taps"], s["case"]["n"]
    seq, at = _sequence(s)
    # every sequence's inputs behind one another, the state's rows before each one's own
    pool = torch.empty(s["t"] + n * (taps - 1), s["case"]["ch"], device="cuda")
    place = torch.arange(s["t"], device="cuda") + (seq + 1) * (taps - 1)
    first = s["start"][:-1].long() + torch.arange(n, device="cuda") * (taps - 1)
    pool[place] = s["x"]
    pool[first[:, None] + torch.arange(taps - 1, device="cuda")] = s["s_in"]
    y = sum(pool[place - (taps - 1) + j] * s["w"][:, j] for j in range(taps))
    last = s["start"][1:].long() + torch.arange(n, device="cuda") * (taps - 1)
    return {"y": y * torch.sigmoid(y), "state": pool[last[:, None] + torch.arange(taps - 1, device="cuda")]}


def _delta(s):
    case = s["case"]
    n, hk, hv, dk, dv = case["n"], case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    size = min(CHUNK, s["longest"])
    padded = -(-s["longest"] // size) * size
    count = (s["start"][1:] - s["start"][:-1]).long()
    place = torch.arange(padded, device="cuda")
    live = place < count[:, None]
    token = torch.where(live, s["start"][:-1, None].long() + place, 0)

    def heads(x, h, d):  # [n, h, padded, d]
        return x[token].view(n, padded, h, d).transpose(1, 2)

    of = torch.arange(hv, device="cuda")
    of = of % hk if case["tiled"] else of // (hv // hk)
    q, k, v = heads(s["x"][:, :hk * dk], hk, dk), heads(s["x"][:, hk * dk:2 * hk * dk], hk, dk), heads(s["x"][:, 2 * hk * dk:], hv, dv)
    q = (q * (torch.rsqrt(q.square().sum(-1, keepdim=True) + EPS) * dk ** -0.5))[:, of]
    k = (k * torch.rsqrt(k.square().sum(-1, keepdim=True) + EPS))[:, of]
    a = s["a"] + s["dt"]
    g = s["decay"] * (a.clamp_min(0) + torch.log1p(torch.exp(-a.abs())))
    g = torch.where(live[:, :, None], g[token], 0.0).transpose(1, 2)
    beta = torch.where(live[:, :, None], torch.sigmoid(s["b"])[token], 0.0).transpose(1, 2)
    state, outs = s["s_in"], []
    below = torch.ones(size, size, device="cuda", dtype=torch.bool).tril()
    # a chunk of tokens at a time: within it the rule is a triangular system, between chunks a recurrence
    for i in range(0, padded, size):
        qc, kc, vc, bc = q[:, :, i:i + size], k[:, :, i:i + size], v[:, :, i:i + size], beta[:, :, i:i + size, None]
        sums = g[:, :, i:i + size].double().cumsum(-1)
        between = torch.exp(torch.where(below, sums[..., :, None] - sums[..., None, :], -math.inf)).float()
        since = torch.exp(sums).float()[..., None]
        left = torch.tril(bc * (kc @ kc.transpose(-1, -2)) * between, -1)
        delta = torch.linalg.solve_triangular(left, bc * (vc - since * (kc @ state)), upper=False, unitriangular=True)
        outs.append(since * (qc @ state) + ((qc @ kc.transpose(-1, -2)) * between) @ delta)
        state = since[:, :, -1:] * state + (kc * between[:, :, -1, :, None]).transpose(-1, -2) @ delta
    o = torch.cat(outs, 2).transpose(1, 2)[live].view(s["t"], hv, dv)
    if case["gated"]:
        z = s["z"].view(s["t"], hv, dv)
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS) * s["nw"] * (z * torch.sigmoid(z))
    return {"o": o.reshape(s["t"], hv * dv), "state": state}


def _rope(s):
    case = s["case"]
    rot, d, page = case["rot"], case["dim"], case["page"]
    seq, at = _sequence(s)
    at = at + s["past"][seq].long()
    angle = at.double()[:, None, None] * s["freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def turned(x, nw):
        if case["norm"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * nw
        x = x.clone()
        i, j = (slice(0, rot, 2), slice(1, rot, 2)) if case["pairs"] else (slice(0, rot // 2), slice(rot // 2, rot))
        a, b = x[..., i].clone(), x[..., j].clone()
        x[..., i], x[..., j] = a * cos - b * sin, b * cos + a * sin
        return x

    where = s["table"][seq, at // page].long()
    s["ck"][where, :, at % page] = turned(s["k"], s["k_norm"]).to(s["ck"].dtype)
    s["cv"][where, :, at % page] = s["v"].to(s["cv"].dtype)
    return {"q": turned(s["qg"][..., :d], s["q_norm"]), "k": s["ck"], "v": s["cv"]}


def _attn(s):
    case = s["case"]
    n, m, hq, hk, d, page, most = case["n"], case["tokens"], case["q_heads"], case["kv_heads"], case["dim"], case["page"], s["most"]
    where = s["table"].clamp_min(0).long()

    def cached(x):  # [n, hk, positions, d]
        return x[where].transpose(1, 2).reshape(n, hk, -1, d)[:, :, :most].float()

    q = s["qg"][..., :d].view(n, m, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
    scores = (q * d ** -0.5) @ cached(s["ck"]).transpose(-1, -2)
    last = s["past"][:, None].long() + torch.arange(m, device="cuda")
    seen = torch.arange(most, device="cuda") <= last[:, :, None]
    scores = torch.where(seen.repeat_interleave(hq // hk, 1)[:, None], scores, -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    values = cached(s["cv"])
    o = (scores @ values) / scores.sum(-1, keepdim=True)
    o = o.view(n, hk, m, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(s["t"], hq, d)
    if case["gated"]:
        o = o * torch.sigmoid(s["qg"][..., d:])
    return {"o": o.reshape(s["t"], hq * d)}


# ---- what a pass cannot do without


def work(case):
    lengths, n, kind = _lengths(case), case["n"], case["kind"]
    t = n * case["tokens"] if kind == "attn" else sum(lengths)
    if kind == "conv":
        ch, taps = case["ch"], case["taps"]
        return {"bytes": 4 * ch * (2 * t + taps + 2 * n * (taps - 1)), "flops": 2.0 * t * ch * taps}
    if kind == "delta":
        hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
        row = 2 * hk * dk + 2 * hv * dv + 2 * hv + (hv * dv if case["gated"] else 0)
        # a token decays the state, reads it twice and adds to it once
        return {"bytes": 4 * t * row + 8 * n * hv * dk * dv, "flops": 7.0 * t * hv * dk * dv}
    hq, hk, d, size = case["q_heads"], case["kv_heads"], case["dim"], 4 if case["type"] == "f32" else 2
    if kind == "rope":
        return {"bytes": t * d * (8 * hq + 2 * hk * (4 + size)), "flops": 8.0 * t * d * (hq + hk)}
    seen = sum(max(v, case["tokens"]) for v in lengths)
    return {"bytes": 2 * seen * hk * d * size + 4 * t * hq * d * (3 if case["gated"] else 2), "flops": 4.0 * seen * case["tokens"] * hq * d}


# ---- the answers in 64 bits, from the operators' definitions


def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "delta": _exact_delta, "rope": _exact_rope, "attn": _exact_attn}[case["kind"]](s)


def _each(s):
    start = s["start"].tolist()
    return [(i, start[i], start[i + 1]) for i in range(s["case"]["n"])]


def _exact_conv(s):
    ys, states = [], []
    for i, a, b in _each(s):
        u = torch.cat([s["s_in"][i], s["x"][a:b]]).double().T[None]
        y = torch.nn.functional.conv1d(u, s["w"].double()[:, None], groups=s["case"]["ch"])[0].T
        ys.append(y / (1 + torch.exp(-y)))
        states.append(u[0].T[b - a:])
    return {"y": torch.cat(ys), "state": torch.stack(states)}


def _exact_delta(s):
    """Token by token, every sequence and head at once."""
    case = s["case"]
    n, hk, hv, dk, dv, t = case["n"], case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"], s["t"]
    x = s["x"].double()
    q, k, v = x[:, :hk * dk].view(t, hk, dk), x[:, hk * dk:2 * hk * dk].view(t, hk, dk), x[:, 2 * hk * dk:].view(t, hv, dv)
    q, k = (u / (u * u).sum(2, keepdim=True).add(EPS).sqrt() for u in (q, k))
    q, k = (u.repeat(1, hv // hk, 1) if case["tiled"] else u.repeat_interleave(hv // hk, 1) for u in (q, k))
    q = q / math.sqrt(dk)
    alpha = torch.exp(s["decay"].double() * torch.nn.functional.softplus(s["a"].double() + s["dt"].double(), threshold=50.0))
    beta = 1 / (1 + torch.exp(-s["b"].double()))
    state, o = s["s_in"].double(), torch.empty(t, hv, dv, dtype=torch.float64, device="cuda")
    first, count = s["start"][:-1].long(), s["start"].diff().long()
    for j in range(s["longest"]):
        at = (count > j).nonzero()[:, 0] if n > 1 else slice(None)
        i = first[at] + j
        m = alpha[i][..., None, None] * state[at]
        d = beta[i][..., None] * (v[i] - (k[i][..., None, :] @ m)[..., 0, :])
        m = m + k[i][..., :, None] * d[..., None, :]
        o[i] = (q[i][..., None, :] @ m)[..., 0, :]
        if n > 1:
            state[at] = m
        else:
            state = m
    if case["gated"]:
        z = s["z"].double().view(t, hv, dv)
        o = s["nw"].double() * o / ((o * o).mean(2, keepdim=True) + EPS).sqrt() * z / (1 + torch.exp(-z))
    return {"o": o.reshape(t, hv * dv), "state": state}


def _exact_rope(s):
    case = s["case"]
    rot, d, page = case["rot"], case["dim"], case["page"]
    past, table = s["past"].tolist(), s["table"].tolist()
    at = torch.cat([torch.arange(past[i], past[i] + b - a) for i, a, b in _each(s)]).cuda()
    page_of = torch.cat([torch.tensor(table[i])[torch.arange(past[i], past[i] + b - a) // page] for i, a, b in _each(s)]).cuda()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), at.double()[:, None] * s["freq"])[:, None]

    def turned(x, nw):
        x = x.double()
        if case["norm"]:
            x = nw.double() * x / ((x * x).mean(2, keepdim=True) + EPS).sqrt()
        r, rest = x[..., :rot], x[..., rot:]
        r = r.unflatten(2, (rot // 2, 2)) if case["pairs"] else r.unflatten(2, (2, rot // 2)).transpose(2, 3)
        r = torch.view_as_real(torch.view_as_complex(r.contiguous()) * turn)
        r = r if case["pairs"] else r.transpose(2, 3)
        return torch.cat([r.flatten(2), rest], 2)

    out = {"q": turned(s["qg"][..., :d], s["q_norm"])}
    for name, cache, x in (("k", s["ck"], turned(s["k"], s["k_norm"])), ("v", s["cv"], s["v"].double())):
        full = cache.double().transpose(1, 2).flatten(0, 1)
        full[page_of * page + at % page] = x
        out[name] = full.unflatten(0, (s["pages"], page)).transpose(1, 2).contiguous()
    return out


def _exact_attn(s):
    case = s["case"]
    hq, hk, d, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    o = torch.empty(s["t"], hq, d, dtype=torch.float64, device="cuda")
    past = s["past"].tolist()
    for i, a, b in _each(s):
        for h in range(hk):
            kc, vc = (x[s["table"][i, :-(-(past[i] + b - a) // page)].long(), h].double().flatten(0, 1) for x in (s["ck"], s["cv"]))
            for j in range(b - a):
                m = past[i] + j + 1
                rows = slice(h * (hq // hk), (h + 1) * (hq // hk))
                p = torch.softmax(s["qg"][a + j, rows, :d].double() @ kc[:m].T / math.sqrt(d), 1)
                o[a + j, rows] = p @ vc[:m]
    if case["gated"]:
        o = o / (1 + torch.exp(-s["qg"][..., d:].double()))
    return {"o": o.reshape(s["t"], hq * d)}
