"""The operators of include/q8_mix.h at the edges of their ranges, against their definitions in 64 bits: rows that see
nothing in sequences that are cut, weights far below a row's largest."""
import numpy as np
import pytest

import mix_ref as ref
from mix_ref import Paged, starts
from test_gpu_mix import run_attn, say

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
