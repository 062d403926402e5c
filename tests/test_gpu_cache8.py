"""The 8-bit cache, reading caches back, and attention through a window on the GPU against their definitions
(cache8_ref.py): odd sizes and pages, ragged and empty sequences, rows that see nothing, pages and positions that are not
there, masked NaN, weights far below a row's largest, far offsets, recordings, and a run of them as a layer uses them."""
import ctypes as c

import numpy as np
import pytest

import cache8_ref as ref8
import mix_ref as ref
from cache8_ref import F, Paged8, paged, quantise, value
from mix_ref import Call, U, starts, untouched
from test_gpu_mix import ATTN, EPS, PROMPTS, rows_of, say
from test_gpu_mix_edges import sink_case

pytestmark = pytest.mark.gpu


# ---- writing


def run_store(rt, m, cache, q, k, v, start, past, rot=0, pairs=False, norms=(None, None), freq=None, t=None):
    """rt_rope_kv_dev into an 8-bit cache: q, and the cache's values and scales of k and v"""
    rows, hq, dim = q.shape
    hk = cache.heads
    with Call(rt, m) as d:
        s = d.seqs(start, past, t=rows if t is None else t)
        kv = cache.struct(d, written=True)
        a = m.Rope(q=d.put(q), q_ld=hq * dim, q_hd=dim, q_heads=hq, k=d.put(k), k_ld=hk * dim, k_hd=dim, v=d.put(v), v_ld=hk * dim, v_hd=dim,
                   q_norm=None if norms[0] is None else d.put(norms[0]), k_norm=None if norms[1] is None else d.put(norms[1]), eps=EPS, rot=rot, pairs=pairs,
                   freq=None if freq is None else d.put(freq), out=d.out("q", q.shape, F), out_ld=hq * dim, out_hd=dim)
        rt.lib.rt_rope_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
        return d.get("q"), cache.held(d, "k"), cache.held(d, "v")


STORE = [
    # hq, hk, dim, page, positions before, new tokens, first
    (1, 1, 32, 16, [0], [1], 0),
    (16, 4, 256, 16, [5, 100, 47], [1, 1, 1], 0),
    (16, 4, 256, 64, [0, 3], [130, 70], 2),
    (3, 3, 96, 7, [6, 0, 20], [3, 0, 9], 1),
    (4, 2, 160, 1, [2], [5], 0),
    (8, 1, 64, 24, [23], [50], 0),
    (2, 2, 192, 5, [0], [11], 0),
    (5, 1, 224, 16, [15], [2], 0),
    (32, 8, 128, 256, [200], [700], 0),
]


@pytest.mark.parametrize("hq,hk,dim,page,pasts,news,first", STORE)
def test_store_values(rt, q8rt, hq, hk, dim, page, pasts, news, first):
    """Rows without norm and rotation: values and scales bit for bit, and every other row of the cache as it was."""
    say("store", hq, hk, dim, page, pasts, news, first)
    rng = np.random.default_rng(hq + dim + page)
    start = starts(news, first)
    t = int(start[-1]) + 2
    q = rng.standard_normal((t, hq, dim)).astype(F)
    k, v = ((rng.standard_normal((t, hk, dim)) * np.exp(rng.uniform(-30, 30, (t, hk, 1)))).astype(F) for _ in range(2))
    cache = Paged8(rng, [a + b for a, b in zip(pasts, news)], hk, dim, page)
    got, *held = run_store(rt, q8rt, cache, q, k, v, start, pasts, t=t)
    live = rows_of(start, t)
    assert np.array_equal(got[live], q[live]) and untouched(got[~live]).all()
    for name, x, (hq8, hd) in zip("kv", (k, v), held):
        want_q, want_d = cache.q[name].copy(), cache.d[name].copy()
        for s, p in enumerate(pasts):
            pos = p + np.arange(news[s])
            where = cache.table[s, pos // page], slice(None), pos % page
            want_q[where], want_d[where] = quantise(x[start[s]:start[s + 1]])
        assert np.array_equal(hq8, want_q) and np.array_equal(hd.view(np.uint32), want_d.view(np.uint32))


@pytest.mark.parametrize("hq,hk,dim,page,pasts,news,first", STORE)
@pytest.mark.parametrize("pairs", [False, True])
def test_store_norm_and_rotation(rt, q8rt, hq, hk, dim, page, pasts, news, first, pairs):
    """A held key is within half a step of the exact one, and what F32 adds to a norm and a rotation: 16 half steps of the
    row's largest (the norm's sum and root 6, its two products, the angle's factors 3, two products and a sum)."""
    rng = np.random.default_rng(hq + dim + page + 1)
    start = starts(news, first)
    t = int(start[-1]) + 2
    q, k, v = (rng.standard_normal((t, h, dim)).astype(F) for h in (hq, hk, hk))
    qn, kn = ((1 + 0.1 * rng.standard_normal(dim)).astype(F) for _ in range(2))
    rot = dim // 2
    freq = 1e6 ** (-np.arange(0, rot, 2) / rot)
    cache = Paged8(rng, [a + b for a, b in zip(pasts, news)], hk, dim, page)
    got, (kq, kd), (vq, vd) = run_store(rt, q8rt, cache, q, k, v, start, pasts, rot, pairs, (qn, kn), freq, t)
    for s, p in enumerate(pasts):
        rows, pos = slice(start[s], start[s + 1]), p + np.arange(news[s])
        want = ref.turn(ref.head_norm(k[rows], kn, EPS), pos, freq, rot, pairs)
        where = cache.table[s, pos // page], slice(None), pos % page
        most = np.abs(want).max(-1)
        assert (np.abs(kd[where] * 127.0 - most) <= 18 * U * most).all()
        assert (np.abs(value(kq[where], kd[where]) - want) <= 0.5 * kd[where][..., None] + 18 * U * most[..., None]).all()
        wq, wd = quantise(v[rows])
        assert np.array_equal(vq[where], wq) and np.array_equal(vd[where], wd)
        qq = ref.turn(ref.head_norm(q[rows], qn, EPS), pos, freq, rot, pairs)
        assert (np.abs(got[rows] - qq) <= 16 * U * np.abs(qq).max(-1, keepdims=True)).all()


def test_store_extremes(rt, q8rt):
    """Rows of zeros, of the largest and smallest numbers, of one large element, ties between two steps, infinities and NaN."""
    dim, page = 64, 16
    rng = np.random.default_rng(3)
    rows = [np.zeros(dim), np.full(dim, 3.4e38), np.r_[1e-44, np.zeros(dim - 1)], np.r_[127.0, np.arange(dim - 1) + 0.5], np.r_[-127.0, -np.arange(dim - 1) - 0.5],
            np.r_[1e30, rng.standard_normal(dim - 1)], np.full(dim, 127 * 2.0 ** -126), np.full(dim, 126.9 * 2.0 ** -126), np.r_[np.inf, np.ones(dim - 1)],
            np.r_[np.ones(dim - 1), -np.inf], np.r_[np.ones(5), np.nan, np.ones(dim - 6)], -rng.standard_normal(dim), np.full(dim, -0.0)]
    x = np.array(rows, F)[:, None]
    t = len(rows)
    cache = Paged8(rng, [t], 1, dim, page)
    _, (kq, kd), (vq, vd) = run_store(rt, q8rt, cache, x, x, x[::-1].copy(), starts([t]), [0])
    pos = np.arange(t)
    where = cache.table[0, pos // page], slice(None), pos % page
    for (gq, gd), y in (((kq, kd), x), ((vq, vd), x[::-1])):
        wq, wd = quantise(y)
        assert np.array_equal(gq[where], wq)
        assert np.array_equal(gd[where], wd, equal_nan=True)


def test_store_places_that_are_not_there(rt, q8rt):
    """Positions before 0, behind the table and on pages outside the cache are not stored, and nothing else moves."""
    rng = np.random.default_rng(4)
    hk, dim, page = 2, 64, 4
    cache = Paged8(rng, [8, 8, 8], hk, dim, page, spare=3)
    cache.table[1, 1] = cache.pages
    cache.table[2, 0] = -1
    news, pasts = [6, 9, 20], [-3, 1, 0]
    t, start = sum(news), starts(news)
    x = rng.standard_normal((t, hk, dim)).astype(F)
    _, *held = run_store(rt, q8rt, cache, x, x, x, start, pasts)
    for name, (gq, gd) in zip("kv", held):
        want_q, want_d = cache.q[name].copy(), cache.d[name].copy()
        for s in range(3):
            for j in range(news[s]):
                p = pasts[s] + j
                if 0 <= p < page * cache.ld and 0 <= cache.table[s, p // page] < cache.pages:
                    q, d = quantise(x[start[s] + j])
                    want_q[cache.table[s, p // page], :, p % page], want_d[cache.table[s, p // page], :, p % page] = q, d
        assert np.array_equal(gq, want_q) and np.array_equal(gd.view(np.uint32), want_d.view(np.uint32))


# ---- reading


NP = {"f32": F, "f16": np.float16, "bf16": np.uint16}


def to_rows(x, to):
    """F32 values as rows of a type hold them, as bits"""
    return ref.to_cache(x, to).view(np.uint32 if to == "f32" else np.uint16)


@pytest.mark.parametrize("kind", ["q8", "f32", "f16", "bf16"])
@pytest.mark.parametrize("to", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hk,dim,page,pasts,news,first", [
    (1, 32, 16, [0], [1], 0), (4, 256, 16, [100, 3, 77], [20, 0, 50], 2), (3, 96, 7, [5, 6], [30, 2], 0), (2, 224, 24, [0], [333], 1), (8, 128, 64, [0, 1], [700, 1], 0),
    (1, 64, 1, [3], [9], 0)])
def test_read(rt, q8rt, kind, to, hk, dim, page, pasts, news, first):
    """Every row's bits; rows that no sequence has, and what lies between the heads, as they were."""
    say("read", kind, to, hk, dim, page, pasts, news, first)
    rng = np.random.default_rng(hk + dim + page)
    start = starts(news, first)
    t = int(start[-1]) + 2
    cache = paged(rng, kind, [a + b for a, b in zip(pasts, news)], hk, dim, page)
    hd, ld = dim + 8, hk * (dim + 8) + 8
    with Call(rt, q8rt) as d:
        s = d.seqs(start, pasts, t=t)
        kv = cache.struct(d)
        a = q8rt.KvRows(type=q8rt.TYPES[to], k=d.out("k", (t, ld), NP[to]), k_ld=ld, k_hd=hd, v=d.out("v", (t, ld), NP[to]), v_ld=ld, v_hd=hd)
        rt.lib.rt_kv_read_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
        got = [d.get("k"), d.get("v")]
    fill = ref.FILL if to == "f32" else None
    for x, mine in zip(got, (cache.seq_k, cache.seq_v)):
        bits = x.view(np.uint32 if to == "f32" else np.uint16)
        want = np.tile(np.array([ref.FILL], np.uint32).view(bits.dtype), t * ld // (1 if to == "f32" else 2)).reshape(t, ld)
        assert fill is None or want[0, 0] == fill
        for i, p in enumerate(pasts):
            for h in range(hk):
                want[start[i]:start[i + 1], h * hd:h * hd + dim] = to_rows(mine[i][p:p + news[i], h].astype(F), to)
        assert np.array_equal(bits, want)


def test_read_one_of_two_heads_first_and_places_that_are_not_there(rt, q8rt):
    """Only v, head by head; NaN before position 0, behind the table and on pages outside the cache."""
    rng = np.random.default_rng(5)
    hk, dim, page, t = 3, 64, 8, 40
    cache = Paged8(rng, [24], hk, dim, page)
    cache.table[0, 1] = cache.pages + 5
    with Call(rt, q8rt) as d:
        s = d.seqs(starts([t]), [-4])
        kv = cache.struct(d)
        a = q8rt.KvRows(type=0, v=d.out("v", (hk, t, dim), F), v_ld=dim, v_hd=t * dim)
        rt.lib.rt_kv_read_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
        got = d.get("v")
    want = np.full((hk, t, dim), np.nan)
    for j in range(t):
        p = j - 4
        if 0 <= p < 8 or 16 <= p < 24:
            want[:, j] = cache.seq_v[0][p]
    assert np.array_equal(got, want.astype(F), equal_nan=True)


# ---- attention


def run_attn(rt, m, cache, q, start, pasts, scale, window=None, sinks=0, gate=None, t=None, longest=None):
    rows, hq, dim = q.shape
    with Call(rt, m) as d:
        s = d.seqs(start, pasts, longest=longest, t=rows if t is None else t)
        kv = cache.struct(d)
        p = d.put(np.concatenate([q, np.zeros_like(q) if gate is None else gate], 2))  # a head's gate beside its query
        a = m.Attn(q=p, q_ld=2 * hq * dim, q_hd=2 * dim, q_heads=hq, scale=scale, gate=None if gate is None else p + 4 * dim, gate_ld=2 * hq * dim, gate_hd=2 * dim,
                   o=d.out("o", (rows, hq * dim + 4), F), o_ld=hq * dim + 4)
        if window is None:
            rt.lib.rt_attn_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
        else:
            rt.lib.rt_attn_window_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a), window, sinks)
        return d.get("o")


def check_attn(rt, m, kind, hq, hk, dim, page, lens, news, first, window, sinks, longests=(None, 1)):
    rng = np.random.default_rng(hq + dim + page + len(lens))
    start = starts(news, first)
    t = int(start[-1]) + 2
    cache = paged(rng, kind, lens, hk, dim, page)
    q = (2 * rng.standard_normal((t, hq, dim))).astype(F)
    gate = rng.standard_normal((t, hq, dim)).astype(F) if hq % 2 == 0 else None
    pasts = [a - b for a, b in zip(lens, news)]
    live = rows_of(start, t)
    want, tol = ref8.attn(q, cache.seq_k, cache.seq_v, dim ** -0.5, start, pasts, window or 0, sinks, gate)
    for longest in longests:
        got = run_attn(rt, m, cache, q, start, pasts, dim ** -0.5, window, sinks, gate, t, longest)
        assert untouched(got[~live]).all() and untouched(got[:, hq * dim:]).all()
        worst = (np.abs(got[live, :hq * dim].reshape(-1, hq, dim) - want[live]) / tol[live]).max() if live.any() else 0.0
        say("worst of the tolerance", worst)
        assert worst <= 1


@pytest.mark.parametrize("hq,hk,dim,page,lens,news,first", ATTN + PROMPTS)
def test_attn8(rt, q8rt, hq, hk, dim, page, lens, news, first):
    say("attn8", hq, hk, dim, page, lens[:5], news[:5], first)
    check_attn(rt, q8rt, "q8", hq, hk, dim, page, lens, news, first, None, 0)


@pytest.mark.parametrize("kind", ["q8", "f32", "f16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 1), (64, 0), (100, 4), (513, 17), (33, 70), (4096, 4)])
@pytest.mark.parametrize("hq,hk,dim,page,lens,news,first", ATTN)
def test_window(rt, q8rt, kind, window, sinks, hq, hk, dim, page, lens, news, first):
    say("window", kind, window, sinks, hq, hk, dim, page, lens[:5], news[:5], first)
    check_attn(rt, q8rt, kind, hq, hk, dim, page, lens, news, first, window, sinks, (None,))


@pytest.mark.parametrize("kind", ["q8", "f32", "f16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 1), (130, 0), (300, 65)])
@pytest.mark.parametrize("hq,hk,dim,page,lens,news,first", PROMPTS + [(6, 2, 96, 7, [333, 40], [290, 40], 1)])
def test_window_prompts(rt, q8rt, kind, window, sinks, hq, hk, dim, page, lens, news, first):
    say("window", kind, window, sinks, hq, hk, dim, page, lens[:5], news[:5], first)
    check_attn(rt, q8rt, kind, hq, hk, dim, page, lens, news, first, window, sinks, (None,))


@pytest.mark.parametrize("kind", ["q8", "f16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(33, 1), (96, 31), (200, 40)])
@pytest.mark.parametrize("dim", range(32, 257, 32))
def test_window_prompts_of_every_head_size(rt, q8rt, kind, window, sinks, dim):
    """The kernels of many rows at each size of a head: their threads' shares of a tile are odd at some."""
    say("window", kind, window, sinks, dim)
    check_attn(rt, q8rt, kind, 8, 2, dim, 9, [430, 150, 77], [390, 77, 77], 0, window, sinks, (None,))


@pytest.mark.parametrize("kind", ["q8", "f32", "f16", "bf16"])
def test_window_of_everything(rt, q8rt, kind):
    """A window or sinks as long as the table, or the longest there are, are no window: the bits of the call without."""
    rng = np.random.default_rng(6)
    hq, hk, dim, lens, news = 8, 2, 128, [700, 90], [1, 40]
    cache = paged(rng, kind, lens, hk, dim, 16)
    q = rng.standard_normal((41, hq, dim)).astype(F)
    start, pasts = starts(news), [699, 50]
    plain = run_attn(rt, q8rt, cache, q, start, pasts, 0.1)
    for window, sinks in ((16 * cache.ld, 0), (2 ** 62, 0), (5, 16 * cache.ld), (1, 2 ** 62)):
        assert np.array_equal(run_attn(rt, q8rt, cache, q, start, pasts, 0.1, window, sinks).view(np.uint32), plain.view(np.uint32))


@pytest.mark.parametrize("kind", ["q8", "f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hk,dim,page,lens,news,window,sinks", [
    (16, 4, 256, 16, [5000, 300], [1, 4], 100, 4), (4, 2, 128, 64, [3000], [150], 200, 0), (2, 1, 64, 5, [999, 20], [20, 20], 64, 11), (8, 8, 96, 24, [400], [3], 1, 1)])
def test_window_pages_that_are_gone(rt, q8rt, kind, hq, hk, dim, page, lens, news, window, sinks):
    """Pages of which no token sees anything: their table entries are anything (pages of others, none, outside), and on the
    pages that stay the positions that nobody sees hold NaN and infinities."""
    say("gone", kind, hq, hk, dim, page, lens, news, window, sinks)
    rng = np.random.default_rng(dim + page)
    pasts = [a - b for a, b in zip(lens, news)]
    k, v = ([rng.standard_normal((n, hk, dim)) for n in lens] for _ in range(2))
    want_k, want_v = [x.copy() for x in k], [x.copy() for x in v]
    for s, n in enumerate(lens):
        unseen = np.ones(n, bool)
        for j in range(news[s]):
            unseen[ref8.seen(pasts[s] + j, window, sinks)] = False
        k[s][unseen], v[s][unseen] = np.inf, np.nan
        k[s][unseen & (np.arange(n) % 3 == 0)], v[s][unseen & (np.arange(n) % 2 == 0)] = np.nan, -np.inf
    cache = paged(rng, kind, lens, hk, dim, page, k=k, v=v)
    for s, n in enumerate(lens):
        for i in range(-(-n // page)):
            pos = np.arange(i * page, min(n, (i + 1) * page))
            if np.isnan(v[s][pos, 0, 0]).sum() + np.isinf(v[s][pos, 0, 0]).sum() == len(pos):
                cache.table[s, i] = (-1, cache.pages, 2 ** 31 - 1, -2 ** 31, 0)[i % 5]
    q = rng.standard_normal((sum(news), hq, dim)).astype(F)
    want, tol = ref8.attn(q, cache.seq_k, cache.seq_v, dim ** -0.5, starts(news), pasts, window, sinks)
    assert np.isfinite(want).all()
    got = run_attn(rt, q8rt, cache, q, starts(news), pasts, dim ** -0.5, window, sinks)[:, :hq * dim].reshape(-1, hq, dim)
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("kind", ["q8", "f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,news,window,sinks", [([2100], [70], 40, 3), ([90], [90], 9, 0), ([40], [6], 5, 2)])
def test_window_masked_places(rt, q8rt, kind, lens, news, window, sinks, dim=64):
    """NaN and infinities in a key and in values that some tokens of a tile see and others do not: in the rows that see
    them as the definition has it, in no other."""
    rng = np.random.default_rng(7)
    hq, hk, n, new = 4, 2, lens[0], news[0]
    k, v = (rng.standard_normal((n, hk, dim)) for _ in range(2))
    if kind == "q8":
        k[n - 3, 0, 5], v[n - new + 2, 1, 3], v[sinks, 0, 1] = np.nan, np.inf, np.nan  # a row's scale: all of its elements
    else:
        k[n - 3, 0], v[n - new + 2, :, 3], v[n - 5, 1, 7], v[sinks, 0, 1] = np.nan, np.inf, -np.inf, np.nan
    cache = paged(rng, kind, lens, hk, dim, 16, k=[k], v=[v])
    q = rng.standard_normal((new, hq, dim)).astype(F)
    start, pasts = starts(news), [n - new]
    want, tol = ref8.attn(q, cache.seq_k, cache.seq_v, 0.125, start, pasts, window, sinks)
    got = run_attn(rt, q8rt, cache, q, start, pasts, 0.125, window, sinks)[:, :hq * dim].reshape(new, hq, dim)
    fine = np.isfinite(want)
    assert fine.any() and not fine.all()
    assert (np.abs(got - want)[fine] <= tol[fine]).all()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])


@pytest.mark.parametrize("kind", ["q8", "f16", "bf16"])
@pytest.mark.parametrize("dim", [160, 224, 256])
def test_window_prompts_of_large_heads_over_what_is_not_there(rt, q8rt, kind, dim):
    """The two tests above for the kernels of many rows on heads of more than 128, whose tiles are shorter."""
    for page, lens, news, window, sinks in [(5, [600, 90], [120, 80], 70, 3), (64, [3000], [150], 200, 0), (24, [400], [60], 33, 40)]:
        test_window_pages_that_are_gone(rt, q8rt, kind, 8, 2, dim, page, lens, news, window, sinks)
    for lens, news, window, sinks in [([2100], [70], 40, 3), ([90], [90], 9, 0), ([700], [300], 65, 30)]:
        test_window_masked_places(rt, q8rt, kind, lens, news, window, sinks, dim)


@pytest.mark.parametrize("kind", ["q8", "f32", "f16", "bf16"])
@pytest.mark.parametrize("news,pasts,window,sinks", [([200], [-8], 50, 4), ([400, 3], [-70, -2], 20, 0), ([30], [-40], 5, 5)])
def test_window_rows_before_position_0(rt, q8rt, kind, news, pasts, window, sinks):
    """Prompts with padding before them: zeros where a token sees nothing, its values elsewhere."""
    rng = np.random.default_rng(8)
    hq, hk, dim = 4, 1, 128
    cache = paged(rng, kind, [max(0, a + b) for a, b in zip(news, pasts)], hk, dim, 16)
    q = rng.standard_normal((sum(news), hq, dim)).astype(F)
    start = starts(news)
    want, tol = ref8.attn(q, cache.seq_k, cache.seq_v, 0.1, start, pasts, window, sinks)
    got = run_attn(rt, q8rt, cache, q, start, pasts, 0.1, window, sinks)[:, :hq * dim].reshape(-1, hq, dim)
    for s, p in enumerate(pasts):
        assert (got[start[s]:start[s] + min(news[s], -p)] == 0).all()
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("window", [None, 20])
def test_pages_that_are_not_there(rt, q8rt, kind, window):
    """A token behind the table, or that sees a page outside the cache, gives NaN; the others their values."""
    rng = np.random.default_rng(9)
    hq, hk, dim, page = 2, 1, 64, 16
    lens, news = [100, 60, 30], [1, 2, 40]
    cache = paged(rng, kind, lens, hk, dim, page)
    start, t, pasts = starts(news), sum(news), [99, 58, 27]
    q = rng.standard_normal((t, hq, dim)).astype(F)
    cache.table[1, 3 if window else 2] = cache.pages
    table = cache.ld * page
    for s in range(3):  # what the table reaches and the sequence does not have is NaN
        for x in (cache.seq_k, cache.seq_v):
            x[s] = np.concatenate([x[s], np.full((table - len(x[s]), hk, dim), np.nan)])
    cache.seq_k[1][(48 if window else 32):(64 if window else 48)] = np.nan
    want, tol = ref8.attn(q, cache.seq_k, cache.seq_v, 0.125, start, pasts, window or 0, 0)
    got = run_attn(rt, q8rt, cache, q, start, pasts, 0.125, window)[:, :hq * dim].reshape(t, hq, dim)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert fine[0].all() and not fine[1:3].any() and (np.abs(got - want)[fine] <= tol[fine]).all()


@pytest.mark.parametrize("nats", [3, 14, 30, 60])
@pytest.mark.parametrize("hq,hk,dim,n,new,at,window", [
    (4, 1, 64, 5000, 2, 2500, None), (6, 2, 128, 700, 3, 0, None), (16, 4, 256, 40, 1, 0, None), (2, 1, 96, 3000, 6, 2990, 200), (4, 2, 128, 300, 300, 0, 50),
    (8, 2, 256, 400, 70, 0, 100)])
def test_attn8_small_weights(rt, q8rt, nats, hq, hk, dim, n, new, at, window):
    """A position that takes nearly all of the softmax and has zeros in half of its values, as the first of a sequence often
    does: there the other positions' weights, however small, count as exactly as F32 holds them."""
    say("small weights", nats, hq, hk, dim, n, new, at, window)
    rng = np.random.default_rng(n + nats + dim)
    plain, q = sink_case(rng, "f32", hq, hk, dim, n, new, nats, at)
    cache = Paged8(rng, [n], hk, dim, 16, k=plain.seq_k, v=plain.seq_v)
    start, pasts = starts([new]), [n - new]
    want, tol = ref8.attn(q, cache.seq_k, cache.seq_v, dim ** -0.5, start, pasts, window or 0, 1 if window else 0)
    got = run_attn(rt, q8rt, cache, q, start, pasts, dim ** -0.5, window, 1 if window else 0)[:, :hq * dim].reshape(new, hq, dim)
    worst = (np.abs(got - want) / tol).max()
    say("worst of the tolerance", worst)
    assert worst <= 1


@pytest.mark.parametrize("what", ["zero", "huge", "tiny", "inf", "nan", "scale", "spike"])
def test_attn8_extremes(rt, q8rt, what):
    """Queries of zeros, of very large and small numbers, not finite, with one element above all others; rows' scales from
    2^-100 to 2^100."""
    rng = np.random.default_rng(10)
    hq, hk, dim, n, new = 4, 2, 64, 300, 5
    k, v = (rng.standard_normal((n, hk, dim)) for _ in range(2))
    q, scale = rng.standard_normal((new, hq, dim)), 0.125
    if what == "zero":
        q[:] = 0
    elif what == "huge":
        q, k, scale = q * 2.0 ** 60, k * 2.0 ** -60, 0.125
    elif what == "tiny":
        q, k = q * 2.0 ** -60, k * 2.0 ** 60
    elif what == "inf":
        q[2, 1, 3] = np.inf
    elif what == "nan":
        q[2, 1, 3] = np.nan
    elif what == "scale":
        v *= 2.0 ** rng.integers(-100, 100, (n, hk, 1))
    else:
        q[..., 7] = 300.0
        k[..., 7] *= 0.01
    cache = Paged8(rng, [n], hk, dim, 16, k=[k], v=[v])
    q = q.astype(F)
    start, pasts = starts([new]), [n - new]
    want, tol = ref8.attn(q, cache.seq_k, cache.seq_v, scale, start, pasts)
    got = run_attn(rt, q8rt, cache, q, start, pasts, scale)[:, :hq * dim].reshape(new, hq, dim)
    if what in ("inf", "nan"):
        assert np.isnan(got[2, 1]).all()
        want[2, 1], got[2, 1], tol[2, 1] = 0, 0, 0
    assert (np.abs(got - want) <= tol).all()


def test_far_rows(rt, q8rt):
    """A cache of 5.4 GB each: rows and scales behind 2^32 bytes, written, read back and attended."""
    say("far rows")
    rng = np.random.default_rng(11)
    hq, hk, dim, page, pages, n = 8, 4, 256, 64, 81000, 200
    size = pages * hk * page * (dim + 4)
    table = np.array([[pages - 1, pages - 3, 0, pages // 2]], np.int32)
    with Call(rt, q8rt) as d:
        ck, cv = (rt.alloc(size) for _ in range(2))
        d.bufs += [ck, cv]
        kv = q8rt.Kv(k=ck, v=cv, type=q8rt.TYPES["q8"], dim=dim, heads=hk, page=page, pages=pages, table=d.put(table), table_ld=4)
        assert rt.lib.rt_kv_bytes(c.byref(kv)) == size
        q, k, v = (rng.standard_normal((n, h, dim)).astype(F) for h in (hq, hk, hk))
        s, pq = d.seqs(starts([n]), [0]), d.put(q)
        a = q8rt.Rope(q=pq, q_ld=hq * dim, q_hd=dim, q_heads=hq, k=d.put(k), k_ld=hk * dim, k_hd=dim, v=d.put(v), v_ld=hk * dim, v_hd=dim, out=d.out("q", q.shape, F),
                      out_ld=hq * dim, out_hd=dim)
        rt.lib.rt_rope_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
        rows = q8rt.KvRows(type=0, k=d.out("k", k.shape, F), k_ld=hk * dim, k_hd=dim, v=d.out("v", v.shape, F), v_ld=hk * dim, v_hd=dim)
        rt.lib.rt_kv_read_dev(rt.R, c.byref(s), c.byref(kv), c.byref(rows))
        held = [value(*quantise(x)) for x in (k, v)]
        assert np.array_equal(d.get("k"), held[0].astype(F)) and np.array_equal(d.get("v"), held[1].astype(F))
        at = q8rt.Attn(q=pq, q_ld=hq * dim, q_hd=dim, q_heads=hq, scale=0.0625, o=d.out("o", (n, hq * dim), F), o_ld=hq * dim)
        for window, sinks in ((0, 0), (33, 5)):
            if window:
                rt.lib.rt_attn_window_dev(rt.R, c.byref(s), c.byref(kv), c.byref(at), window, sinks)
            else:
                rt.lib.rt_attn_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(at))
            want, tol = ref8.attn(q, [held[0]], [held[1]], 0.0625, starts([n]), [0], window, sinks)
            assert (np.abs(d.get("o").reshape(n, hq, dim) - want) <= tol).all()


MANY = [
    # hq, hk, dim, page, positions a sequence, new tokens
    (16, 4, 256, 16, [20000], [70]),  # a few row tiles on a long history: cut, and joined by rows
    (8, 4, 128, 24, [9000, 40, 3000], [50, 40, 33]),
    (6, 2, 96, 7, [5000], [43]),
    (4, 1, 32, 64, [4000, 64], [64, 64]),
    (16, 2, 224, 16, [1500, 900, 2], [40, 8, 2]),
    (4, 2, 128, 16, list(range(1, 2000, 45)), [1] * 45),  # chunks by rounds, over one and two of them
    (8, 8, 64, 16, [3000, 0, 17, 900, 2999, 64], [1, 0, 2, 1, 3, 1]),
    (4, 1, 256, 16, [700] * 33, [1] * 33),
    (2, 1, 128, 16, [37 * i % 1500 + 1 for i in range(150)], [1] * 150),  # more sequences than a wave has lanes
    (8, 1, 64, 16, [60 + 5 * i for i in range(70)], [40 + i % 20 for i in range(70)]),
    (16, 8, 64, 16, [1000], [1000]),  # several heads an XCD
    (6, 3, 64, 16, [500, 700], [500, 90]),  # three heads, which 8 XCDs do not divide into
]


@pytest.mark.parametrize("kind,window,sinks", [("q8", None, 0), ("q8", 700, 5), ("bf16", 700, 5), ("f16", 1500, 33), ("f32", 300, 0), ("bf16", 5000, 0)])
@pytest.mark.parametrize("hq,hk,dim,page,lens,news", MANY)
def test_many_and_long(rt, q8rt, kind, window, sinks, hq, hk, dim, page, lens, news):
    """Calls that are cut and joined in every way: row tiles of 64 on long histories, batches in one and two rounds of chunks,
    more sequences than lanes, head counts that do and do not divide the XCDs."""
    say("many and long", kind, window, sinks, hq, hk, dim, page, lens[:5], news[:5])
    check_attn(rt, q8rt, kind, hq, hk, dim, page, lens, news, 0, window, sinks, (None,))


@pytest.mark.parametrize("kind", ["q8", "bf16", "f16"])
def test_the_same_bits_again(rt, q8rt, kind):
    """A call's bits are the same every time, cut and joined or not."""
    rng = np.random.default_rng(14)
    hq, hk, dim = 8, 2, 128
    for lens, news in (([9000], [60]), ([700, 3000, 90], [1, 1, 1]), ([1200], [1200])):
        cache = paged(rng, kind, lens, hk, dim, 16)
        q = rng.standard_normal((sum(news), hq, dim)).astype(F)
        pasts = [a - b for a, b in zip(lens, news)]
        first = run_attn(rt, q8rt, cache, q, starts(news), pasts, 0.1, 600, 4)
        for _ in range(3):
            assert np.array_equal(run_attn(rt, q8rt, cache, q, starts(news), pasts, 0.1, 600, 4).view(np.uint32), first.view(np.uint32))


@pytest.mark.parametrize("kind", ["q8", "f32", "f16", "bf16"])
@pytest.mark.parametrize("past,new", [(10 ** 9 + 7, 1), (10 ** 9 + 7, 5), (10 ** 9 + 7, 40), (2 ** 31 - 2 ** 21 - 100, 30)])
def test_window_at_far_positions(rt, q8rt, kind, past, new):
    """A thousand million positions behind the sequence's first, of which the pages of the window and the sinks are there."""
    say("far", kind, past, new)
    rng = np.random.default_rng(15)
    hq, hk, dim, page, window, sinks = 4, 1, 32, 1 << 18, 100, 3
    ld = (past + new) // page + 1
    first = (past - window + 1) // page
    table = np.full((1, ld), -1, np.int32)
    table[0, first:], table[0, 0] = np.arange(ld - first) + 1, 0
    pages = ld - first + 1
    pos = np.r_[np.arange(sinks), np.arange(past - window + 1, past + new)]
    rows = np.where(pos < sinks, pos, table[0, pos // page].astype(np.int64) * page + pos % page)
    x = {n: rng.standard_normal((len(pos), dim)).astype(F) for n in "kv"}
    held = {}
    with Call(rt, q8rt) as d:
        ptr = {}
        for n in "kv":
            if kind == "q8":
                q, s = quantise(x[n])
                held[n] = value(q, s)
                mem = np.full(pages * page * (dim + 4), 0x7F, np.uint8)
                mem[:pages * page * dim].reshape(-1, dim)[rows] = q.view(np.uint8)
                mem[pages * page * dim:].view(F)[rows] = s
            else:
                raw = ref.to_cache(x[n], kind)
                held[n] = ref.of_cache(raw, kind)
                mem = ref.to_cache(np.full((pages * page, dim), np.nan), kind)
                mem[rows] = raw
            ptr[n] = d.put(mem)
        q = rng.standard_normal((new, hq, dim)).astype(F)
        s = d.seqs(starts([new]), [past])
        kv = q8rt.Kv(k=ptr["k"], v=ptr["v"], type=q8rt.TYPES[kind], dim=dim, heads=hk, page=page, pages=pages, table=d.put(table), table_ld=ld)
        a = q8rt.Attn(q=d.put(q), q_ld=hq * dim, q_hd=dim, q_heads=hq, scale=0.2, o=d.out("o", (new, hq * dim), F), o_ld=hq * dim)
        rt.lib.rt_attn_window_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a), window, sinks)
        got = d.get("o").reshape(new, hq, dim)
    for j in range(new):
        at = (pos < sinks) | ((pos > past + j - window) & (pos <= past + j))
        k, v = (np.concatenate([held[n][at][:, None], np.zeros((0, 1, dim))]) for n in "kv")
        want, tol = ref8.attn(q[j:j + 1], [k], [v], 0.2, [0, 1], [int(at.sum()) - 1])
        assert (np.abs(got[j] - want[0]) <= tol[0]).all(), j



# ---- as a layer uses them


@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 3)])
def test_a_conversation(rt, q8rt, window, sinks):
    """Prompts of two sequences, single tokens, four drafts of which two are taken back and written over, tokens again: each
    call's attention against 64 bits on what the cache holds, and the cache the same as one written at once."""
    rng = np.random.default_rng(12)
    hq, hk, dim, page, rot = 8, 2, 128, 16, 64
    total = [150, 90]
    steps = [([130, 70], [0, 0]), ([1, 1], [130, 70]), ([4, 4], [131, 71]), ([4, 1], [133, 73]), ([1, 0], [137, 74])]
    freq = 1e6 ** (-np.arange(0, rot, 2) / rot)
    kn = (1 + 0.1 * rng.standard_normal(dim)).astype(F)
    cache = Paged8(rng, total, hk, dim, page, k=[np.zeros((n, hk, dim)) for n in total], v=[np.zeros((n, hk, dim)) for n in total])
    k_all, v_all = ([np.zeros((n, hk, dim), F) for n in total] for _ in range(2))
    with Call(rt, q8rt) as d:
        kv, dkn, df = cache.struct(d, written=True), d.put(kn), d.put(freq)
        pos = [np.arange(n) for n in total]
        where = [(cache.table[s, pos[s] // page], slice(None), pos[s] % page) for s in range(2)]
        for news, pasts in steps:
            t, start = sum(news), starts(news)
            q, k, v = (rng.standard_normal((t, h, dim)).astype(F) for h in (hq, hk, hk))
            for s in range(2):
                rows = slice(pasts[s], pasts[s] + news[s])
                k_all[s][rows], v_all[s][rows] = k[start[s]:start[s + 1]], v[start[s]:start[s + 1]]
            s = d.seqs(start, pasts)
            turned = d.out("q", q.shape, F)
            a = q8rt.Rope(q=d.put(q), q_ld=hq * dim, q_hd=dim, q_heads=hq, k=d.put(k), k_ld=hk * dim, k_hd=dim, v=d.put(v), v_ld=hk * dim, v_hd=dim, k_norm=dkn, eps=EPS,
                          rot=rot, freq=df, out=turned, out_ld=hq * dim, out_hd=dim)
            rt.lib.rt_rope_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
            at = q8rt.Attn(q=turned, q_ld=hq * dim, q_hd=dim, q_heads=hq, scale=dim ** -0.5, o=d.out("o", (t, hq * dim), F), o_ld=hq * dim)
            if window:
                rt.lib.rt_attn_window_dev(rt.R, c.byref(s), c.byref(kv), c.byref(at), window, sinks)
            else:
                rt.lib.rt_attn_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(at))
            held = [[value(x[w], y[w]) for w in where] for x, y in (cache.held(d, "k"), cache.held(d, "v"))]
            want, tol = ref8.attn(d.get("q"), held[0], held[1], dim ** -0.5, start, pasts, window, sinks)
            assert (np.abs(d.get("o").reshape(t, hq, dim) - want) <= tol).all(), (news, pasts)
        ends = [a + b for a, b in zip(*steps[-1])]
        apart = [cache.held(d, "k"), cache.held(d, "v")]
        # the same rows in one call, over what is there
        t, start = sum(ends), starts(ends)
        s = d.seqs(start, [0, 0])
        q = np.zeros((t, hq, dim), F)
        a = q8rt.Rope(q=d.put(q), q_ld=hq * dim, q_hd=dim, q_heads=hq, k=d.put(np.concatenate([x[:e] for x, e in zip(k_all, ends)])), k_ld=hk * dim, k_hd=dim,
                      v=d.put(np.concatenate([x[:e] for x, e in zip(v_all, ends)])), v_ld=hk * dim, v_hd=dim, k_norm=dkn, eps=EPS, rot=rot, freq=df,
                      out=d.out("q", q.shape, F), out_ld=hq * dim, out_hd=dim)
        rt.lib.rt_rope_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
        for (q8, d8), (o8, od) in zip(apart, (cache.held(d, "k"), cache.held(d, "v"))):
            assert np.array_equal(q8, o8) and np.array_equal(d8.view(np.uint32), od.view(np.uint32))


@pytest.mark.parametrize("kind", ["q8", "f16"])
def test_recorded_steps(rt, q8rt, kind):
    """A decode step (store, attention through a window, reading the new rows back) recorded once and replayed as positions
    move on, with eager calls of other sizes between the replays: every replay's bits are the eager step's."""
    rng = np.random.default_rng(13)
    hq, hk, dim, page, n, w, sinks = 8, 2, 128, 16, 3, 500, 4
    lens = [1500, 700, 90]
    cache = paged(rng, kind, lens, hk, dim, page)
    freq = 1e6 ** (-np.arange(0, dim, 2) / dim)
    with Call(rt, q8rt) as d:
        kv, df = cache.struct(d, written=True), d.put(freq)
        s = d.seqs(starts([1] * n), [x - 10 for x in lens])
        q, k, v = (d.put(np.zeros((n, h, dim), F)) for h in (hq, hk, hk))
        turned, o, back = d.out("q", (n, hq, dim), F), d.out("o", (n, hq * dim), F), d.out("k", (n, hk, dim), F)
        a = q8rt.Rope(q=q, q_ld=hq * dim, q_hd=dim, q_heads=hq, k=k, k_ld=hk * dim, k_hd=dim, v=v, v_ld=hk * dim, v_hd=dim, rot=dim, freq=df, out=turned, out_ld=hq * dim,
                      out_hd=dim)
        at = q8rt.Attn(q=turned, q_ld=hq * dim, q_hd=dim, q_heads=hq, scale=dim ** -0.5, o=o, o_ld=hq * dim)
        rows = q8rt.KvRows(type=0, k=back, k_ld=hk * dim, k_hd=dim)
        # a prompt of other sizes between the replays, in the same workspace
        big = d.seqs(starts([200]), [0])
        bq, bo = d.put(rng.standard_normal((200, hq, dim)).astype(F)), d.put(np.zeros((200, hq * dim), F))
        other = q8rt.Attn(q=bq, q_ld=hq * dim, q_hd=dim, q_heads=hq, scale=dim ** -0.5, o=bo, o_ld=hq * dim)

        def step():
            rt.lib.rt_rope_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
            rt.lib.rt_attn_window_dev(rt.R, c.byref(s), c.byref(kv), c.byref(at), w, sinks)
            rt.lib.rt_kv_read_dev(rt.R, c.byref(s), c.byref(kv), c.byref(rows))

        step()
        rt.lib.rt_graph_begin(rt.R)
        step()
        graph = rt.lib.rt_graph_end(rt.R)
        for i in range(6):
            past = np.array([x - 10 + i for x in lens], np.int32)
            rt.to_dev(s.past, past)
            for p, h in ((q, hq), (k, hk), (v, hk)):
                rt.to_dev(p, rng.standard_normal((n, h, dim)).astype(F))
            step()
            eager = [d.get(x) for x in ("o", "k", "ck", "cv")]
            rt.lib.rt_attn_kv_dev(rt.R, c.byref(big), c.byref(kv), c.byref(other))
            rt.to_dev(o, np.zeros((n, hq * dim), F))
            rt.lib.rt_graph_launch(rt.R, c.c_void_p(graph))
            for x, y in zip(eager, (d.get(x) for x in ("o", "k", "ck", "cv"))):
                assert np.array_equal(x.view(np.uint8), y.view(np.uint8))
        rt.lib.rt_graph_free(rt.R, c.c_void_p(graph))


def test_two_runtimes(rt, q8rt):
    """Calls of two runtimes on one cache, one behind the other without a wait between them, each with a workspace of its own:
    each one's bits alone."""
    rng = np.random.default_rng(16)
    hq, hk, dim, lens = 8, 2, 128, [5000, 900]
    cache = Paged8(rng, lens, hk, dim, 16)
    other = q8rt.Runtime()
    try:
        with Call(rt, q8rt) as d:
            kv = cache.struct(d)
            calls = []
            for r, news, window in ((rt, [1, 1], 800), (other, [70, 30], 300), (rt, [40, 200], 2000), (other, [2, 1], 4000)):
                s = d.seqs(starts(news), [a - b for a, b in zip(lens, news)])
                q = d.put(rng.standard_normal((sum(news), hq, dim)).astype(F))
                name = f"o{len(calls)}"
                a = q8rt.Attn(q=q, q_ld=hq * dim, q_hd=dim, q_heads=hq, scale=0.1, o=d.out(name, (sum(news), hq * dim), F), o_ld=hq * dim)
                calls.append((r, s, a, window, name))

            def run(r, s, a, window, name):
                r.lib.rt_attn_window_dev(r.R, c.byref(s), c.byref(kv), c.byref(a), window, 4)

            alone = []
            for call in calls:
                run(*call)
                call[0].sync()
                alone.append(d.get(call[4]))
            for _ in range(5):
                for call in calls:
                    run(*call)
                rt.sync()
                other.sync()
                for call, x in zip(calls, alone):
                    assert np.array_equal(d.get(call[4]).view(np.uint32), x.view(np.uint32))
    finally:
        other.close()
