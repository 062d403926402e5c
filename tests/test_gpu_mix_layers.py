"""The operators of include/q8_mix.h between the products, as a layer's mixer runs them on activations in
HBM: a prompt, then single tokens and a token with its drafts, against the same layers in 64 bits on the
dequantised weights. DeltaNet: the quartet on the RMS norm, the convolution, the delta rule with its norm
and gate, W_OUT onto a residual. Attention: Q (with its gates), K and V on the norm, the heads to the cache, the
attention, W_O onto a residual. The bar is the products' own (tests/parity.py) on what each layer adds (to a residual
of 0, which hides none of it)."""
import ctypes as c

import numpy as np
import pytest

import mix_ref as ref
import synth
from mix_ref import Call
from parity import assert_parity

pytestmark = pytest.mark.gpu
EPS = 1e-6
H = 512  # hidden


class Weights:
    def __init__(self, rt, rng, shapes):
        self.rt, self.h, self.f = rt, {}, {}
        for name, (rows, cols) in shapes.items():
            q8 = synth.q8_rows(rng, rows, cols)
            self.h[name] = rt.upload(q8, rows, cols)
            blk = q8.reshape(rows, cols // 32, 34)
            d = blk[:, :, :2].copy().view(np.float16).astype(np.float64)
            self.f[name] = (blk[:, :, 2:].copy().view(np.int8) * d).reshape(rows, cols)

    def free(self):
        for h in self.h.values():
            self.rt.lib.rt_q8_free(self.rt.R, c.c_void_p(h))


def rms(x, nw):
    return nw * x / np.sqrt((x * x).mean(1, keepdims=True) + EPS)


def round_norm(rt, w, names, x, nw, t, ys):
    rt.lib.rt_gemv_round_norm_dev(rt.R, len(names), (c.c_void_p * len(names))(*[w.h[k] for k in names]), (c.c_long * len(names))(*[w.f[k].shape[0] for k in names]), H,
                                  c.c_void_p(x), H, t, c.c_void_p(nw), EPS, (c.c_void_p * len(names))(*ys))


STEPS = [[70, 5], [1, 1], [4, 1]]  # the new tokens of two sequences, call by call


def inputs(rng):
    return [rng.standard_normal((sum(n), H)).astype(np.float32) for n in STEPS]


def test_deltanet_layer(rt, q8rt):
    rng = np.random.default_rng(31)
    hk, hv, dk, dv = 2, 4, 64, 128
    qkv, vw = 2 * hk * dk + hv * dv, hv * dv
    w = Weights(rt, rng, {"qkv": (qkv, H), "z": (vw, H), "b": (32, H), "a": (32, H), "out": (H, vw)})
    anorm, nw = (1 + 0.1 * rng.standard_normal(n).astype(np.float32) for n in (H, dv))
    taps = rng.standard_normal((qkv, 4)).astype(np.float32)
    decay, dt = -np.exp(rng.uniform(0, 2, hv)).astype(np.float32), rng.uniform(-4, -1, hv).astype(np.float32)
    conv, state = np.zeros((2, 3, qkv)), np.zeros((2, hv, dk, dv))
    try:
        with Call(rt, q8rt) as d:
            dev = {k: d.put(v) for k, v in dict(anorm=anorm, nw=nw, taps=taps, decay=decay, dt=dt).items()}
            cs, ss = d.put(conv.astype(np.float32)), d.put(state.astype(np.float32))
            for news, x in zip(STEPS, inputs(rng)):
                t, start = sum(news), ref.starts(news)
                s = d.seqs(start)
                px, py, pz, pb, pa = d.put(x), *(d.put(np.zeros((t, n), np.float32)) for n in (qkv, vw, 32, 32))
                pu, po, pr = d.put(np.zeros((t, qkv), np.float32)), d.put(np.zeros((t, vw), np.float32)), d.out("x", (t, H), np.float32)
                round_norm(rt, w, ("qkv", "z", "b", "a"), px, dev["anorm"], t, (py, pz, pb, pa))
                rt.lib.rt_conv_silu_dev(rt.R, c.byref(s), py, qkv, qkv, dev["taps"], 4, cs, cs, pu, qkv)
                arg = q8rt.Delta(k_heads=hk, v_heads=hv, k_dim=dk, v_dim=dv, tiled=1, q=pu, q_ld=qkv, k=pu + 4 * hk * dk, k_ld=qkv, v=pu + 8 * hk * dk, v_ld=qkv, a=pa,
                                 a_ld=32, b=pb, b_ld=32, decay=dev["decay"], dt=dev["dt"], eps=EPS, scale=dk ** -0.5, s_in=ss, s_out=ss, z=pz, z_ld=vw,
                                 nw=dev["nw"], nw_eps=EPS, o=po, o_ld=vw)
                rt.lib.rt_delta_rule_dev(rt.R, c.byref(s), c.byref(arg))
                rt.lib.rt_gemm_residual_dev(rt.R, c.c_void_p(w.h["out"]), H, vw, c.c_void_p(po), vw, t, c.c_void_p(d.put(np.zeros((t, H), np.float32))), c.c_void_p(pr))
                got = d.get("x")
                xn = rms(x.astype(np.float64), anorm)
                y, conv, _ = ref.conv(xn @ w.f["qkv"].T, taps, conv, start)
                q, k, v = (u.reshape(t, -1, n) for u, n in zip(np.split(y, [hk * dk, 2 * hk * dk], 1), (dk, dk, dv)))
                o, state, _ = ref.delta(q, k, v, (xn @ w.f["a"].T)[:, :hv], (xn @ w.f["b"].T)[:, :hv], decay, dt, EPS, dk ** -0.5, state, start, True,
                                        (xn @ w.f["z"].T).reshape(t, hv, dv), nw, EPS)
                assert_parity(got, o.reshape(t, vw) @ w.f["out"].T, f"DeltaNet layer, {news} tokens")
    finally:
        w.free()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_attention_layer(rt, q8rt, kind):
    rng = np.random.default_rng(32)
    hq, hk, dim, page, rot = 4, 2, 128, 16, 32
    w = Weights(rt, rng, {"q": (2 * hq * dim, H), "k": (hk * dim, H), "v": (hk * dim, H), "o": (H, hq * dim)})
    anorm, qn, kn = (1 + 0.1 * rng.standard_normal(n).astype(np.float32) for n in (H, dim, dim))
    freq = 1e7 ** (-np.arange(0, rot, 2) / rot)
    total = [sum(n[i] for n in STEPS) for i in range(2)]
    cache = ref.Paged(rng, kind, total, hk, dim, page, k=[np.zeros((n, hk, dim)) for n in total], v=[np.zeros((n, hk, dim)) for n in total])
    seq_k, seq_v, past = [np.zeros((0, hk, dim)) for _ in total], [np.zeros((0, hk, dim)) for _ in total], [0, 0]
    try:
        with Call(rt, q8rt) as d:
            kv, dn, dq, dk, df = cache.struct(d, written=True), d.put(anorm), d.put(qn), d.put(kn), d.put(freq)
            for news, x in zip(STEPS, inputs(rng)):
                t, start = sum(news), ref.starts(news)
                s = d.seqs(start, past)
                px, pq, pk, pv = d.put(x), *(d.put(np.zeros((t, n), np.float32)) for n in (2 * hq * dim, hk * dim, hk * dim))
                pt, po, pr = d.put(np.zeros((t, hq * dim), np.float32)), d.put(np.zeros((t, hq * dim), np.float32)), d.out("x", (t, H), np.float32)
                round_norm(rt, w, ("q", "k", "v"), px, dn, t, (pq, pk, pv))
                rope = q8rt.Rope(q=pq, q_ld=2 * hq * dim, q_hd=2 * dim, q_heads=hq, k=pk, k_ld=hk * dim, k_hd=dim, v=pv, v_ld=hk * dim, v_hd=dim, q_norm=dq, k_norm=dk,
                                 eps=EPS, rot=rot, freq=df, out=pt, out_ld=hq * dim, out_hd=dim)
                rt.lib.rt_rope_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(rope))
                attn = q8rt.Attn(q=pt, q_ld=hq * dim, q_hd=dim, q_heads=hq, scale=dim ** -0.5, gate=pq + 4 * dim, gate_ld=2 * hq * dim, gate_hd=2 * dim, o=po,
                                 o_ld=hq * dim)
                rt.lib.rt_attn_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(attn))
                rt.lib.rt_gemm_residual_dev(rt.R, c.c_void_p(w.h["o"]), H, hq * dim, c.c_void_p(po), hq * dim, t, c.c_void_p(d.put(np.zeros((t, H), np.float32))), c.c_void_p(pr))
                got = d.get("x")
                xn = rms(x.astype(np.float64), anorm)
                q, k, v = ((xn @ w.f[n].T).reshape(t, -1, m) for n, m in (("q", 2 * dim), ("k", dim), ("v", dim)))
                pos = np.concatenate([past[i] + np.arange(news[i]) for i in range(2)])
                q, gate = ref.turn(ref.head_norm(q[..., :dim], qn, EPS), pos, freq, rot, False), q[..., dim:]
                k = ref.turn(ref.head_norm(k, kn, EPS), pos, freq, rot, False)
                for i in range(2):
                    rows = slice(start[i], start[i + 1])
                    # as the cache holds them: what the library rounded is taken from its cache, within half a step of the exact
                    seq_k[i], seq_v[i] = np.concatenate([seq_k[i], k[rows]]), np.concatenate([seq_v[i], v[rows]])
                    at = np.arange(past[i] + news[i])
                    for name, mine in (("ck", seq_k), ("cv", seq_v)):
                        held = ref.of_cache(d.get(name)[cache.table[i, at // page], :, at % page], kind)
                        assert (np.abs(held - mine[i]) <= 1.001 * ref.HALF[kind] * np.abs(mine[i]) + 1e-5 * np.abs(mine[i]).max()).all()
                        mine[i] = held
                o, _ = ref.attn(q, seq_k, seq_v, dim ** -0.5, start, past, gate)
                assert_parity(got, o.reshape(t, hq * dim) @ w.f["o"].T, f"attention layer, {news} tokens, {kind}")
                past = [a + b for a, b in zip(past, news)]
    finally:
        w.free()
