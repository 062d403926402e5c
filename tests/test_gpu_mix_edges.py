"""The operators of include/q8_mix.h at the edges of their ranges, against their definitions in 64 bits: rows that see
nothing in sequences that are cut."""
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
