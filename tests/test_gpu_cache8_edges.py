"""Attention over the 8-bit cache and through windows on the GPU at the edges of F32: gates that are infinite, NaN or far from 0, in
every kernel and in row tiles that are cut and that are not."""
import numpy as np
import pytest

import cache8_ref as ref8
import mix_ref as ref
from cache8_ref import F, paged
from mix_ref import starts
from test_gpu_cache8 import run_attn
from test_gpu_mix import say

pytestmark = pytest.mark.gpu

# positions of a sequence, new tokens of it, window, sinks: single tokens and drafts; prompts whose row tiles are one chunk each
# (the table reaches so little, or the window), and are cut; a part of a prompt behind a history
CALLS = [([300, 40], [1, 3], None, 0), ([90], [90], None, 0), ([70, 64], [70, 33], 30, 3), ([3000], [40], None, 0), ([3000], [40], 1500, 4), ([900], [300], 60, 0)]
GATES = [np.inf, -np.inf, np.nan, 3e38, -3e38, 2.37e38, -2.37e38, 1e30, -1e30, 105, -105, 100, -100, 88, -88, 80, -80, 1.5, -1.5, 0.0, -0.0]


@pytest.mark.parametrize("kind", ["q8", "f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 96, 256])
@pytest.mark.parametrize("lens,news,window,sinks", CALLS)
def test_gates_far_from_0(rt, q8rt, kind, dim, lens, news, window, sinks):
    """o / (1 + exp(-gate)): 0 and o where the gate is infinite or far below and above 0, NaN where it is NaN, whichever kernel has
    the row. A factor below 2^-126, F32's smallest with all its bits, may be 0: |o| 2^-126."""
    say("gates", kind, dim, lens, news, window, sinks)
    rng = np.random.default_rng(dim + lens[0])
    hq, hk, t = 8, 2, sum(news)
    cache = paged(rng, kind, lens, hk, dim, 8)
    q = (2 * rng.standard_normal((t, hq, dim))).astype(F)
    gate = rng.choice(np.array(GATES, F), (t, hq, dim))
    pasts = [a - b for a, b in zip(lens, news)]
    o, tol = ref8.attn(q, cache.seq_k, cache.seq_v, dim ** -0.5, starts(news), pasts, window or 0, sinks)
    with np.errstate(invalid="ignore"):
        g = ref.sigmoid(gate.astype(np.float64))
        want, tol = o * g, tol * g + 4 * ref.U * np.abs(o * g) + 2.0 ** -126 * np.abs(o) + 2.0 ** -140
    got = run_attn(rt, q8rt, cache, q, starts(news), pasts, dim ** -0.5, window, sinks, gate)[:, :hq * dim].reshape(t, hq, dim)
    assert np.isfinite(o).all() and np.array_equal(np.isnan(gate), np.isnan(want))
    assert np.array_equal(np.isnan(got), np.isnan(want))
    there = ~np.isnan(want)
    assert (np.abs(got - want)[there] <= tol[there]).all()
    assert (got[gate < -150] == 0).all()


@pytest.mark.parametrize("what", ["far keys", "huge", "tiny", "inf", "nan", "values", "small values", "spike", "zero"])
@pytest.mark.parametrize("new,window,sinks", [(5, None, 0), (90, None, 0), (90, 70, 3)])
def test_range_of_queries_and_scales(rt, q8rt, what, new, window, sinks):
    """Single rows and prompts alike: scores that are ordinary numbers though keys are near 2^103 and queries near 2^-97, or the other
    way round; queries of zeros, not finite, with one element above all others; values' scales from 2^-100 to 2^100, or near 2^-105.

    Far below 1 a weight's product with its value's scale d has few bits left. The weights are taken 2^-8 to 1 for the largest, so
    that they add up to 2^-8 at least; one below 2^-126 is 0, and a product is held to 2^-133, the least step of the bf16 limbs. So a
    position adds up to 127 (2^-126 d + 2^-133) / 2^-8, which is below 2^-118 (127 d + 1), whatever the kernel."""
    say("range", what, new, window, sinks)
    rng = np.random.default_rng(17)
    hq, hk, dim, n = 4, 2, 64, 300
    k, v = (rng.standard_normal((n, hk, dim)) for _ in range(2))
    q = rng.standard_normal((new, hq, dim))
    if what == "far keys":
        q, k = q * 2.0 ** -97, k * 2.0 ** 103  # scores of some 60 either way
    elif what == "huge":
        q, k = q * 2.0 ** 100, k * 2.0 ** -100
    elif what == "tiny":
        q, k = q * 2.0 ** -60, k * 2.0 ** 60
    elif what in ("inf", "nan"):
        q[new // 2, 1, 3] = float(what)
    elif what == "values":
        v *= 2.0 ** rng.integers(-100, 100, (n, hk, 1))
    elif what == "small values":
        v *= 2.0 ** -100
    elif what == "spike":
        q[..., 7] = 300.0
        k[..., 7] *= 0.01
    else:
        q[:] = 0
    cache = paged(rng, "q8", [n], hk, dim, 16, k=[k], v=[v])
    q = q.astype(F)
    want, tol = ref8.attn(q, cache.seq_k, cache.seq_v, 0.125, starts([new]), [n - new], window or 0, sinks)
    tol += 2.0 ** -118 * n * (1 + np.abs(cache.seq_v[0]).max())
    got = run_attn(rt, q8rt, cache, q, starts([new]), [n - new], 0.125, window, sinks)[:, :hq * dim].reshape(new, hq, dim)
    if what in ("inf", "nan"):
        at = new // 2, 1
        assert np.isnan(got[at]).all()
        want[at], got[at], tol[at] = 0, 0, 0
    assert (np.abs(got - want) <= tol).all()
