"""The operators of include/q8_mix.h at the edges of their ranges, against their definitions in 64 bits: rows that see
nothing in sequences that are cut, weights far below a row's largest, decays near 1, the
most sequences; and what the workspace holds."""
import ctypes as c

import numpy as np
import pytest

import mix_ref as ref
from mix_ref import Call, Paged, starts
from test_gpu_mix import EPS, check_delta, delta_bound, delta_inputs, run_attn, run_delta, say

pytestmark = pytest.mark.gpu


# ---- rows that see nothing


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("hq,hk,dim,news,pasts", [
    (2, 1, 64, [200], [-2]), (16, 4, 64, [200], [-8]), (4, 2, 128, [400], [-2]), (4, 2, 256, [330, 200], [0, -70]), (2, 1, 32, [300, 1, 90], [-17, 500, -90])])
def test_attn_rows_before_position_0_of_cut_sequences(rt, q8rt, kind, gated, hq, hk, dim, news, pasts):
    """Prompts with padding before them, long enough that their positions go to several workgroups and are joined: zeros
    where a token sees nothing, its values elsewhere."""
    say("attn before 0", kind, gated, hq, hk, dim, news, pasts)
    rng = np.random.default_rng(hq + dim + news[0])
    start, t = starts(news), sum(news)
    cache = Paged(rng, kind, [max(0, a + b) for a, b in zip(news, pasts)], hk, dim, 16)
    q = rng.standard_normal((t, hq, dim)).astype(np.float32)
    gate = rng.standard_normal((t, hq, dim)).astype(np.float32) if gated else None
    want, tol = ref.attn(q, cache.seq_k, cache.seq_v, dim ** -0.5, start, pasts, gate)
    got = run_attn(rt, q8rt, cache, q, start, pasts, dim ** -0.5, gate)[:, :hq * dim].reshape(t, hq, dim)
    for s, past in enumerate(pasts):
        empty = min(news[s], max(0, -past))
        assert (got[start[s]:start[s] + empty] == 0).all()
    assert (np.abs(got - want) <= tol).all()


# ---- weights far below a row's largest


def sink_case(rng, kind, hq, hk, dim, n, new, nats, at):
    """One sequence whose position `at` has a score of `nats` above every other, in every row, and half of whose values there
    are 0: those elements of the output are the other positions' weights alone"""
    k, v = (rng.standard_normal((n, hk, dim)) for _ in range(2))
    q = rng.standard_normal((new, hq, dim)).astype(np.float32)
    q[..., -1], k[..., -1] = 8.0, 0.0
    top = max((q[:, h].astype(np.float64) @ k[:, h // (hq // hk)].T).max() for h in range(hq))
    k[at], v[at, :, ::2] = 0.0, 0.0
    k[at, :, -1] = (top + nats * dim ** 0.5) / 8.0
    return Paged(rng, kind, [n], hk, dim, 16, k=[k], v=[v]), q


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nats", [3, 8, 14, 20, 30, 60])
@pytest.mark.parametrize("hq,hk,dim,n,new,at", [
    (4, 1, 64, 16384, 1, 0), (4, 1, 64, 5000, 2, 2500), (6, 2, 128, 700, 3, 0), (16, 4, 256, 40, 1, 0), (2, 1, 96, 3000, 6, 2990), (2, 1, 32, 30, 2, 7),
    (4, 2, 128, 300, 300, 0), (8, 2, 256, 400, 70, 100)])
def test_attn_small_weights(rt, q8rt, kind, nats, hq, hk, dim, n, new, at):
    """A position that takes nearly all of the softmax and has values of 0, as the first of a sequence often does: the other
    positions' weights, however small, count as exactly as F32 holds them."""
    say("attn small weights", kind, nats, hq, hk, dim, n, new, at)
    rng = np.random.default_rng(n + nats + dim)
    cache, q = sink_case(rng, kind, hq, hk, dim, n, new, nats, at)
    start, pasts = starts([new]), [n - new]
    want, tol = ref.attn(q, cache.seq_k, cache.seq_v, dim ** -0.5, start, pasts)
    got = run_attn(rt, q8rt, cache, q, start, pasts, dim ** -0.5)[:, :hq * dim].reshape(new, hq, dim)
    worst = (np.abs(got - want) / tol).max()
    say("worst of the tolerance", worst)
    assert worst <= 1


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nats", [14, 30, 60])
@pytest.mark.parametrize("hq,hk,dim,n,new", [(4, 1, 64, 3000, 1), (4, 2, 128, 90, 4), (8, 2, 256, 200, 40)])
def test_attn_infinite_values_of_small_weights(rt, q8rt, kind, nats, hq, hk, dim, n, new):
    """An infinite or NaN value shows however small its weight, in its own element, and no other one changes."""
    say("attn infinite values", kind, nats, hq, hk, dim, n, new)
    rng = np.random.default_rng(n + nats)
    cache, q = sink_case(rng, kind, hq, hk, dim, n, new, nats, 5)
    spare = cache.table[0]
    for pos, e, x in ((20, 3, np.inf), (n - new, 6, -np.inf), (33, 9, np.nan), (n - 2, 12, np.inf)):
        cache.v[spare[pos // 16], :, pos % 16, e] = ref.to_cache(np.array([x]), kind)[0]
        cache.seq_v[0][pos, :, e] = x
    start, pasts = starts([new]), [n - new]
    want, tol = ref.attn(q, cache.seq_k, cache.seq_v, dim ** -0.5, start, pasts)
    got = run_attn(rt, q8rt, cache, q, start, pasts, dim ** -0.5)[:, :hq * dim].reshape(new, hq, dim)
    fine = np.isfinite(want)
    assert (np.abs(got - want)[fine] <= tol[fine]).all()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])


# ---- decays near 1


@pytest.mark.parametrize("count,longest", [(8192, None), (4000, 1), (100, None)])  # in chunks, token by token, a short prompt
@pytest.mark.parametrize("a,b", [(-5.5, -5.0), (-6.9, -5.0), (-8.0, -7.0), (-10.0, -3.0), (0.5, -5.0)])
def test_delta_constant_slow_gates(rt, q8rt, count, longest, a, b):
    """The same gate at every token, its decay near 1: what the decay is off by is off the same way at every token, and adds up
    over the 1 / (1 - decay) tokens that a state remembers, so it has to be far below a half step of F32."""
    say("delta slow gate", count, longest, a, b)
    rng = np.random.default_rng(count)
    hv, dk, dv, start = 3, 128, 32, starts([count])
    q, k, v, ga, gb, decay, dt, s_in = delta_inputs(rng, count, 1, hv, dk, dv, 1)
    ga[:], gb[:], decay[:], dt[:] = a, b, np.float32([-1.0, -0.7, -1.9]), 0.0
    x = (q, k, v, ga, gb, decay, dt, s_in)
    got, state = run_delta(rt, q8rt, x, start, False, longest=longest)
    want, wstate, size = ref.delta(*x[:7], EPS, dk ** -0.5, s_in, start, False)
    say("state", [float(np.sqrt(((state[0, h] - wstate[0, h]) ** 2).mean() / (wstate[0, h] ** 2).mean())) for h in range(hv)], "bound", delta_bound(dk, count))
    check_delta(got, state, want, wstate, size, start, dk, hv * dv)


# ---- workspaces


def test_growing_prompts_keep_little_memory(q8rt):
    """Prompts that get longer call by call: what the runtime holds stays within a few times the largest call's need, whatever
    it replaced on the way."""
    r = q8rt.Runtime()
    hk, hv, dk, dv, most = 16, 32, 128, 128, 4096
    part = 4 * (hv * (2 * 10 * 256 + 256) + hk * 2 * 64 * dk)  # bytes a chunk of 64 tokens
    try:
        with Call(r, q8rt) as d:
            x, ab = d.put(np.zeros((most, 2 * hk * dk + hv * dv), np.float32)), d.put(np.zeros((most, 2 * hv), np.float32))
            state, o, head = d.put(np.zeros((hv, dk, dv), np.float32)), d.put(np.zeros((most, hv * dv), np.float32)), d.put(np.zeros(hv, np.float32))
            ld = 2 * hk * dk + hv * dv
            arg = q8rt.Delta(k_heads=hk, v_heads=hv, k_dim=dk, v_dim=dv, q=x, q_ld=ld, k=x + 4 * hk * dk, k_ld=ld, v=x + 8 * hk * dk, v_ld=ld, a=ab, a_ld=2 * hv,
                             b=ab + 4 * hv, b_ld=2 * hv, decay=head, dt=head, eps=EPS, scale=1.0, s_in=state, s_out=state, o=o, o_ld=hv * dv)
            free, total = c.c_size_t(), c.c_size_t()

            def call(t):
                s = d.seqs(starts([t]))
                r.lib.rt_delta_rule_dev(r.R, c.byref(s), c.byref(arg))
                r.lib.rt_dev_sync(r.R)
                assert r.lib.hipMemGetInfo(c.byref(free), c.byref(total)) == 0
                return free.value

            first = call(64)
            held = first - min(call(t) for t in range(128, most + 1, 64))
            say("held", held / 2 ** 20, "MB, a call's need", part * (most // 64 + 1) / 2 ** 20)
            assert held <= 4 * part * (most // 64 + 1)
    finally:
        r.close()


# ---- the most sequences and heads


def test_delta_more_workgroups_than_a_launch_has_along_x(rt, q8rt):
    """65535 sequences of 5 heads of 32 x 416, 17 GB of state in place: the first and last sequence's tokens in chunks, the
    others, which have none, as they were."""
    n, hk, hv, dk, dv, count = 65535, 1, 5, 32, 416, 70
    rng = np.random.default_rng(1)
    x = delta_inputs(rng, 2 * count, hk, hv, dk, dv, 4)
    q, k, v, a, b, decay, dt, s_in = x
    place = [0, n - 1, 1, n // 2]  # of s_in's four states
    start = np.full(n + 1, count, np.int32)
    start[0], start[n] = 0, 2 * count
    size = hv * dk * dv * 4
    with Call(rt, q8rt) as d:
        state = rt.alloc(n * size)
        d.bufs.append(state)
        for i, s in zip(place, s_in):
            rt.to_dev(state + i * size, s)
        seqs = q8rt.Seqs(n=n, t=2 * count, longest=count, start=d.put(start))
        arg = q8rt.Delta(k_heads=hk, v_heads=hv, k_dim=dk, v_dim=dv, q=d.put(q), q_ld=hk * dk, k=d.put(k), k_ld=hk * dk, v=d.put(v), v_ld=hv * dv, a=d.put(a), a_ld=hv,
                         b=d.put(b), b_ld=hv, decay=d.put(decay), dt=d.put(dt), eps=EPS, scale=dk ** -0.5, s_in=state, s_out=state,
                         o=d.out("o", (2 * count, hv * dv), np.float32), o_ld=hv * dv)
        say("delta, sequences", n)
        rt.lib.rt_delta_rule_dev(rt.R, c.byref(seqs), c.byref(arg))
        got, after = d.get("o"), np.empty_like(s_in)
        for i, s in zip(place, after):
            rt.from_dev(s, state + i * size)
    few = starts([count, count])
    want, wstate, width = ref.delta(*x[:7], EPS, dk ** -0.5, s_in[:2], few, False)
    check_delta(got, after[:2], want, wstate, width, few, dk, hv * dv)
    assert np.array_equal(after[2:], s_in[2:])
