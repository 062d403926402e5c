"""The operators of long histories in little memory: their plain forms in torch, the calls that a program makes
of them (include/q8_mix.h), and their answers in 64 bits.

  store   the heads' norms and the rotation with the keys' and values' way into a cache of 8 bits, a scale for
          each position and head, and those rows read back from it as 16-bit values
  read    a range of positions of each sequence read back from a cache of any type
  attn8   attention over the cache of 8 bits: single tokens, drafts, prompts
  window  attention with a sliding window and a few first positions that stay visible, over a cache of any type

The head counts and sizes are those of the layers whose products the library runs: 16 query heads on 4
key-value heads of 256, 64 of which turn, on a hidden size of 4096, and 8 on 2 on one of 2048.
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
BLOCK = 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    nine = {"q_heads": 16, "kv_heads": 4, "dim": 256}
    two = {"q_heads": 8, "kv_heads": 2, "dim": 256}
    store = {"kind": "store", "type": "q8", "rot": 64, "pairs": False, "norm": True, "to": "f16"}
    attn8 = {"kind": "attn8", "type": "q8", "gated": True}
    window = {"kind": "window", "gated": True}
    return [
        # one decode step of a serving batch: latency
        {"name": "store_decode_32", **store, **nine, "page": 16, "n": 32, "new_low": 1, "new_high": 1, "past_low": 100, "past_high": 16384},
        # prompts of three requests in one call
        {"name": "store_prompt", **store, **nine, "page": 64, "n": 3, "new_low": 301, "new_high": 2048, "past_low": 0, "past_high": 0},
        # the newest rows of a few sequences, for a check on the host
        {"name": "read_few", "kind": "read", "type": "q8", "to": "f32", **nine, "page": 16, "n": 4, "new_low": 17, "new_high": 100, "past_low": 0, "past_high": 5000},
        # a prefix of odd length on its way into another cache
        {"name": "read_prefix", "kind": "read", "type": "q8", "to": "bf16", **nine, "page": 64, "n": 1, "new_low": 32767, "new_high": 32767, "past_low": 0, "past_high": 0},
        # one user's next token on a short history
        {"name": "attn8_decode_1", **attn8, **nine, "page": 64, "n": 1, "new_low": 1, "new_high": 1, "past_low": 776, "past_high": 776},
        # a serving batch of mixed lengths
        {"name": "attn8_decode_32", **attn8, **nine, "page": 16, "n": 32, "new_low": 1, "new_high": 1, "past_low": 100, "past_high": 16383},
        # a token and its drafts at the end of a very long history
        {"name": "attn8_verify_long", **attn8, **nine, "page": 64, "n": 1, "new_low": 4, "new_high": 4, "past_low": 131068, "past_high": 131068},
        # a request's prompt
        {"name": "attn8_prompt", **attn8, **nine, "page": 16, "n": 1, "new_low": 2048, "new_high": 2048, "past_low": 0, "past_high": 0},
        # a serving batch whose layers look back 1024 positions and at the first 4
        {"name": "window_decode_32", **window, **nine, "type": "f16", "page": 16, "n": 32, "new_low": 1, "new_high": 1, "past_low": 100, "past_high": 30000,
         "window": 1024, "sinks": 4},
        # one user's next token, far into a conversation without end, in 8 bits
        {"name": "window_decode_far", **window, **nine, "type": "q8", "page": 64, "n": 1, "new_low": 1, "new_high": 1, "past_low": 1000003, "past_high": 1000003,
         "window": 4096, "sinks": 4},
        # prompts of two requests through a short window on the smaller model
        {"name": "window_prompt_2b", **window, **two, "type": "bf16", "page": 64, "n": 2, "new_low": 1500, "new_high": 4001, "past_low": 0, "past_high": 0, "window": 512,
         "sinks": 4},
        # a part of a very long prompt, in 8 bits, behind what came before
        {"name": "window_prompt_long", **window, **nine, "type": "q8", "page": 16, "n": 1, "new_low": 8192, "new_high": 8192, "past_low": 20000, "past_high": 20000,
         "window": 1024, "sinks": 16},
    ]


def _log(rng, low, high):
    high = max(low, high)
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["store", "read", "attn8", "attn8", "window", "window"])
    kv = rng.choice([1, 2, 4, 8])
    case = {"kind": kind, "type": "q8", "q_heads": kv * rng.choice([1, 2, 4, 4, 6, 8]), "kv_heads": kv, "dim": rng.choice([64, 96, 128, 128, 256, 256]),
            "page": rng.choice([16, 16, 24, 64, 256])}
    n = _log(rng, 1, 64)
    if kind == "store":
        high = rng.choice([1, _log(rng, 1, 4000 // n)])
        return {**case, "rot": rng.choice([case["dim"], case["dim"] // 2, 32]), "pairs": rng.random() < 0.3, "norm": rng.random() < 0.8, "to": rng.choice(["f16", "bf16"]),
                "n": n, "new_low": max(1, high // rng.randint(1, 8)), "new_high": high, "past_low": 0, "past_high": _log(rng, 1, 200000)}
    if kind == "read":
        high = _log(rng, 1, 32000 * 1024 // (n * max(512, kv * case["dim"])))
        return {**case, "type": rng.choice(["q8", "q8", "f16", "bf16", "f32"]), "to": rng.choice(["f32", "f16", "bf16"]), "n": n, "new_low": max(1, high // rng.randint(1, 8)),
                "new_high": high, "past_low": 0, "past_high": _log(rng, 1, 200000)}
    case["gated"] = rng.random() < 0.7
    if kind == "window":
        case |= {"type": rng.choice(["q8", "q8", "f16", "bf16", "f32"]), "window": _log(rng, 16, 8192), "sinks": rng.choice([0, 1, 4, 4, 16, 100])}
    if rng.random() < 0.3:
        # prompts, a few or one, at the start or behind a history
        n = _log(rng, 1, 6)
        high = _log(rng, 20, 2000 // n)
        past = rng.choice([0, _log(rng, 1, 100000 if kind == "window" else 2000 // n)])
        return {**case, "n": n, "new_low": max(1, high // rng.randint(1, 6)), "new_high": high, "past_low": past // rng.randint(1, 4), "past_high": past}
    if kind == "window":
        n = min(n, max(1, 32 * 1024 * 1024 // (case["window"] * kv * case["dim"])))
        high = _log(rng, 17, 1000000)
    else:
        high = _log(rng, 17, min(100000, 400000 // n) // max(1, kv * case["dim"] // 1024))
    new = rng.choice([1, 1, 1, 2, 3, 4, 6])
    return {**case, "n": n, "new_low": new, "new_high": new, "past_low": max(8, high // rng.randint(1, 20)), "past_high": high}


def _lengths(case):
    """Each sequence's new tokens and the positions before them, odd and even, between low and high; one of each high."""
    rng = random.Random(case["n"] * 7919 + case["new_high"] * 31 + case["past_high"])
    many = range(case["n"] - 1)
    new = [case["new_high"]] + [rng.randint(case["new_low"], case["new_high"]) for _ in many]
    return new, [case["past_high"]] + [rng.randint(case["past_low"], max(case["past_low"], case["past_high"])) for _ in many]


def _needed(case, new, past):
    """The pages of a sequence that the call touches, as (first, one behind the last) of one or two runs."""
    page, total = case["page"], past + new
    if case["kind"] in ("store", "read"):
        return [(past // page, -(-total // page))]
    if case["kind"] == "attn8":
        return [(0, -(-total // page))]
    first = max(0, past - case["window"] + 1)
    sinks = -(-min(case["sinks"], first) // page)
    return [(0, min(sinks, first // page)), (first // page, -(-total // page))]


# ---- the inputs


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pool(shape, kind, gen):
    """A cache's keys or values, and for 8 bits its scales: (all of its memory, the values, the scales)"""
    if kind != "q8":
        x = torch.empty(shape, dtype=TYPES[kind], device="cuda").normal_(generator=gen)
        return x, x, None
    rows, d = math.prod(shape[:-1]), shape[-1]
    # the scales lie behind the values
    mem = torch.empty(rows * (d + 4), dtype=torch.uint8, device="cuda")
    q, scale = mem[:rows * d].view(torch.int8).view(shape), mem[rows * d:].view(torch.float32).view(shape[:-1])
    x = torch.randn(shape, generator=gen, device="cuda")
    top = x.abs().amax(-1)
    scale.copy_(top / 127)
    q.copy_(torch.round(x / scale[..., None]))
    return mem, q, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale)

    n, kind, hk, d, page = case["n"], case["kind"], case["kv_heads"], case["dim"], case["page"]
    hq = case["q_heads"]
    new, past = _lengths(case)
    start = [0]
    for v in new:
        start.append(start[-1] + v)
    t = start[-1]
    s = {"case": case, "t": t, "longest": max(new), "start": _ints(start), "past": _ints(past), "most": max(a + b for a, b in zip(new, past))}
    # the pages that the call touches are there, in any order, the others are not
    need = [_needed(case, a, b) for a, b in zip(new, past)]
    s["pages"] = sum(b - a for runs in need for a, b in runs) + 1
    order, at = torch.randperm(s["pages"], generator=gen, device="cuda").int(), 0
    s["table"] = torch.full((n, max(runs[-1][1] for runs in need)), -1, dtype=torch.int32, device="cuda")
    for i, runs in enumerate(need):
        for a, b in runs:
            s["table"][i, a:b] = order[at:at + b - a]
            at += b - a
    for name in ("k", "v"):
        s["c" + name], s["q" + name], s["d" + name] = _pool((s["pages"], hk, page, d), case["type"], gen)
    if kind == "read":
        s["k_out"], s["v_out"] = (torch.empty(t, hk, d, dtype=TYPES[case["to"]], device="cuda") for _ in range(2))
        return s
    # each query's gate lies beside it, as the query product gives them
    s["qg"] = normal(t, hq, 2 * d)
    if kind == "store":
        s["freq"] = (1e7 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])).cuda()
        s["k"], s["v"] = normal(t, hk, d), normal(t, hk, d)
        s["q_norm"], s["k_norm"] = 1.0 + 0.1 * normal(d), 1.0 + 0.1 * normal(d)
        s["out"] = torch.empty(t, hq, d, device="cuda")
        s["k_out"], s["v_out"] = (torch.empty(t, hk, d, dtype=TYPES[case["to"]], device="cuda") for _ in range(2))
    else:
        s["qg"][:, :, :d] *= 1.5
        s["o"] = torch.empty(t, hq * d, device="cuda")
    return s


def run(state):
    if own:
        if "calls" not in state:
            state["calls"] = _bind(state)
        calls, out = state["calls"]
        for fn, args in calls:
            fn(*args)
        return out
    return {"store": _store, "read": _read, "attn8": _attend, "window": _attend}[state["case"]["kind"]](state)


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
    """([(an entry point, its arguments)], the outputs): the structures that a program fills once for its buffers."""
    rt, m = _runtime()
    case = s["case"]
    kind, hq, hk, d = case["kind"], case["q_heads"], case["kv_heads"], case["dim"]

    def p(name):
        return s[name].data_ptr() if name in s else None

    seqs = m.Seqs(n=case["n"], t=s["t"], longest=s["longest"], start=p("start"), past=p("past"))
    kv = m.Kv(k=p("ck"), v=p("cv"), type=m.TYPES[case["type"]], dim=d, heads=hk, page=case["page"], pages=s["pages"], table=p("table"), table_ld=s["table"].shape[1])
    first = (rt.R, c.byref(seqs), c.byref(kv))
    if kind in ("store", "read"):
        rows = m.KvRows(type=m.TYPES[case["to"]], k=p("k_out"), k_ld=hk * d, k_hd=d, v=p("v_out"), v_ld=hk * d, v_hd=d)
        read, out = (rt.lib.rt_kv_read_dev, (*first, c.byref(rows))), {"k": s["k_out"], "v": s["v_out"]}
        if kind == "read":
            return [read], out
        a = m.Rope(q=p("qg"), q_ld=2 * hq * d, q_hd=2 * d, q_heads=hq, k=p("k"), k_ld=hk * d, k_hd=d, v=p("v"), v_ld=hk * d, v_hd=d,
                   q_norm=p("q_norm") if case["norm"] else None, k_norm=p("k_norm") if case["norm"] else None, eps=EPS, rot=case["rot"], pairs=case["pairs"],
                   freq=p("freq"), out=p("out"), out_ld=hq * d, out_hd=d)
        return [(rt.lib.rt_rope_kv_dev, (*first, c.byref(a))), read], {"q": s["out"], **out}
    a = m.Attn(q=p("qg"), q_ld=2 * hq * d, q_hd=2 * d, q_heads=hq, scale=d ** -0.5, gate=p("qg") + 4 * d if case["gated"] else None, gate_ld=2 * hq * d, gate_hd=2 * d,
               o=p("o"), o_ld=hq * d)
    if kind == "attn8":
        return [(rt.lib.rt_attn_kv_dev, (*first, c.byref(a)))], {"o": s["o"]}
    return [(rt.lib.rt_attn_window_dev, (*first, c.byref(a), case["window"], case["sinks"]))], {"o": s["o"]}


# ---- the plain forms, in 32 bits


def _places(s):
    """Each token's sequence, position, and its row's page and place in the cache."""
    i = torch.arange(s["t"], device="cuda")
    seq = torch.searchsorted(s["start"].long(), i, right=True) - 1
    at = i - s["start"][seq].long() + s["past"][seq].long()
    return at, s["table"][seq, at // s["case"]["page"]].long(), at % s["case"]["page"]


def _cached(s, name, where, row):
    """The cache's rows of these pages and places in 32 bits, heads behind them"""
    x = s["q" + name][where, :, row].float()
    return x if s["d" + name] is None else x * s["d" + name][where, :, row][..., None]


def _read(s):
    _, where, row = _places(s)
    return {name: _cached(s, name, where, row).to(TYPES[s["case"]["to"]]) for name in ("k", "v")}


def _store(s):
    case = s["case"]
    rot, d = case["rot"], case["dim"]
    at, where, row = _places(s)
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

    for name, x in (("k", turned(s["k"], s["k_norm"])), ("v", s["v"])):
        scale = x.abs().amax(-1) / 127
        s["d" + name][where, :, row] = scale
        s["q" + name][where, :, row] = torch.round(x / scale[..., None]).to(torch.int8)
    return {"q": turned(s["qg"][..., :d], s["q_norm"]), **_read(s)}


def _attend(s):
    """Blocks of a sequence's tokens, each with the positions that it sees."""
    case = s["case"]
    n, hq, hk, d, page = case["n"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    size = min(BLOCK, s["longest"])
    new, past = (s["start"][1:] - s["start"][:-1]).long(), s["past"].long()
    blocks = (s["longest"] + size - 1) // size
    seq = torch.arange(n, device="cuda").repeat_interleave(blocks)
    place = torch.arange(blocks, device="cuda").repeat(n)[:, None] * size + torch.arange(size, device="cuda")  # [blocks, size], in the sequence
    some = place[:, 0] < new[seq]
    seq, place = seq[some], place[some]
    live = place < new[seq][:, None]
    token = torch.where(live, s["start"][seq].long()[:, None] + place, 0)
    at = past[seq][:, None] + place
    if case["kind"] == "window":
        reach, sinks = case["window"], case["sinks"]
        near = at[:, :1] - reach + 1 + torch.arange(reach - 1 + size, device="cuda")
        far = torch.arange(sinks, device="cuda").expand(len(seq), sinks)
        pos = torch.cat([far, torch.where(near >= sinks, near, -1)], 1)
        seen = (pos[:, None] >= 0) & (pos[:, None] <= at[..., None]) & ((pos[:, None] < sinks) | (pos[:, None] > at[..., None] - reach))
    else:
        pos = torch.arange(s["most"], device="cuda").expand(len(seq), -1)
        seen = pos[:, None] <= at[..., None]
    # what no token sees is read from anywhere
    inside = pos.clamp(0, s["table"].shape[1] * page - 1)
    where, row = s["table"][seq[:, None], inside // page].clamp_min(0).long(), inside % page
    keys, values = (_cached(s, name, where, row).transpose(1, 2) for name in ("k", "v"))  # [blocks, hk, positions, d]
    group = hq // hk
    q = s["qg"][..., :d][token].view(-1, size, hk, group, d).permute(0, 2, 3, 1, 4).reshape(len(seq), hk, group * size, d)
    scores = ((q * d ** -0.5) @ keys.transpose(-1, -2)).view(len(seq), hk, group, size, -1)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_().view(len(seq), hk, group * size, -1)
    o = (scores @ values) / scores.sum(-1, keepdim=True)
    o = o.view(len(seq), hk, group, size, d).permute(0, 3, 1, 2, 4)[live].reshape(s["t"], hq, d)
    if case["gated"]:
        o = o * torch.sigmoid(s["qg"][..., d:])
    return {"o": o.reshape(s["t"], hq * d)}


# ---- what a pass cannot do without


def _seen(case, new, past):
    """The positions that a sequence's tokens see: of all of them together, and summed over them"""
    if case["kind"] == "attn8":
        return past + new, new * past + new * (new + 1) // 2
    w, sinks = case["window"], case["sinks"]
    first = max(0, past - w + 1)
    each = sum(min(p + 1, w) + max(0, min(sinks, p + 1 - w)) for p in range(past, past + new))
    return past + new - first + min(sinks, first), each


def work(case):
    new, past = _lengths(case)
    hq, hk, d, t = case["q_heads"], case["kv_heads"], case["dim"], sum(new)
    held = d + 4 if case["type"] == "q8" else d * TYPES[case["type"]].itemsize
    if case["kind"] == "store":
        return {"bytes": t * (8 * d * hq + 2 * hk * (4 * d + held + 2 * d)), "flops": 8.0 * t * d * (hq + 2 * hk)}
    if case["kind"] == "read":
        return {"bytes": 2 * t * hk * (held + d * TYPES[case["to"]].itemsize), "flops": 2.0 * t * hk * d}
    seen = [_seen(case, a, b) for a, b in zip(new, past)]
    return {"bytes": 2 * hk * held * sum(a for a, _ in seen) + 4 * t * hq * d * (3 if case["gated"] else 2), "flops": 4.0 * d * hq * sum(b for _, b in seen)}


# ---- the answers in 64 bits, from the operators' definitions


def exact(case, seed):
    s = prepare(case, seed)
    new, past = _lengths(case)
    if case["kind"] in ("attn8", "window"):
        return _exact_attn(s, new, past)
    page, table = case["page"], s["table"].tolist()
    at = [p + j for m, p in zip(new, past) for j in range(m)]
    rows = [table[i][(p + j) // page] * page + (p + j) % page for i, (m, p) in enumerate(zip(new, past)) for j in range(m)]
    if case["kind"] == "read":
        rows = torch.tensor(rows, device="cuda")
        return {name: _all(s, name).transpose(1, 2).flatten(0, 1)[rows] for name in ("k", "v")}
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.tensor(at, device="cuda").double()[:, None] * s["freq"])[:, None]
    rot, d = case["rot"], case["dim"]

    def turned(x, nw):
        x = x.double()
        if case["norm"]:
            x = nw.double() * x / ((x * x).mean(2, keepdim=True) + EPS).sqrt()
        r, rest = x[..., :rot], x[..., rot:]
        r = r.unflatten(2, (rot // 2, 2)) if case["pairs"] else r.unflatten(2, (2, rot // 2)).transpose(2, 3)
        r = torch.view_as_real(torch.view_as_complex(r.contiguous()) * turn)
        return torch.cat([(r if case["pairs"] else r.transpose(2, 3)).flatten(2), rest], 2)

    def held(x):
        step = x.abs().amax(2, keepdim=True) / 127
        return torch.round(x / step) * step

    return {"q": turned(s["qg"][..., :d], s["q_norm"]), "k": held(turned(s["k"], s["k_norm"])), "v": held(s["v"].double())}


def _all(s, name):
    x = s["q" + name].double()
    return x if s["d" + name] is None else x * s["d" + name].double()[..., None]


def _exact_attn(s, new, past):
    """A sequence, a key-value head and some tokens at a time."""
    case = s["case"]
    hq, hk, d, page, w, sinks = case["q_heads"], case["kv_heads"], case["dim"], case["page"], case.get("window"), case.get("sinks")
    o = torch.empty(s["t"], hq, d, dtype=torch.float64, device="cuda")
    group, a = hq // hk, 0
    for i, (m, p) in enumerate(zip(new, past)):
        for j in range(0, m, 512):
            at = torch.arange(p + j, min(p + j + 512, p + m), device="cuda")
            pos = torch.arange(0, p + m, device="cuda")
            if w is not None:
                pos = pos[(pos < sinks) | (pos > p + j - w)]
            pos = pos[pos <= at[-1]]
            seen = pos <= at[:, None]
            if w is not None:
                seen &= (pos < sinks) | (pos > at[:, None] - w)
            where = s["table"][i].long()[pos // page]
            for h in range(hk):
                k, v = (s["q" + name][where, h, pos % page].double() * (1.0 if s["d" + name] is None else s["d" + name][where, h, pos % page].double()[:, None])
                        for name in ("k", "v"))
                rows = slice(h * group, (h + 1) * group)
                q = s["qg"][a + j:a + j + len(at), rows, :d].double()
                x = torch.where(seen[:, None], q.flatten(0, 1).matmul(k.T).view(len(at), group, -1) / math.sqrt(d), -math.inf)
                o[a + j:a + j + len(at), rows] = (torch.softmax(x, 2).flatten(0, 1) @ v).view(len(at), group, d)
        a += m
    if case["gated"]:
        o = o / (1 + torch.exp(-s["qg"][..., d:].double()))
    return {"o": o.reshape(s["t"], hq * d)}
