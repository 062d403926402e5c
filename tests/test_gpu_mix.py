"""The operators between the products (include/q8_mix.h) on the GPU against their definitions in 64 bits
(mix_ref.py), where they can go wrong: ragged and empty sequences, rows that no sequence has, hints
that are too small, odd sizes, states in place, decays of zero, repeated keys, pages that end inside a
tile, pages that are not there, and NaN and infinities where a mask hides them. Every tolerance counts F32
roundings (mix_ref.py); a state's and an output's of the delta rule are said at their test."""
import ctypes as c

import numpy as np
import pytest

import mix_ref as ref
from mix_ref import Call, Paged, U, starts, untouched

pytestmark = pytest.mark.gpu
EPS = 1e-6


def say(*a):
    print(*a, flush=True)


def rows_of(start, t):
    live = np.zeros(t, bool)
    for a, b in zip(start[:-1], start[1:]):
        live[a:b] = True
    return live


# ---- the short convolution


@pytest.mark.parametrize("taps,ch,lens,first,longest", [
    (4, 64, [1], 0, None), (4, 1036, [1, 0, 3, 17], 0, None), (2, 8, [5, 2], 3, None), (8, 260, [3, 0, 40, 7, 1], 2, None), (3, 2048, [33], 0, 1),
    (5, 20, [100, 3], 0, 2), (6, 512, [9, 8, 7], 1, None), (7, 4, [64], 0, 64), (4, 128, [1] * 70, 0, None)])
@pytest.mark.parametrize("in_place", [False, True])
def test_conv(rt, q8rt, taps, ch, lens, first, longest, in_place):
    say("conv", taps, ch, lens, first, longest, in_place)
    rng = np.random.default_rng(taps * ch + len(lens))
    start = starts(lens, first)
    t = int(start[-1]) + 2  # two rows behind the last sequence
    x = rng.standard_normal((t, ch + 8)).astype(np.float32)
    w = rng.standard_normal((ch, taps)).astype(np.float32)
    s_in = rng.standard_normal((len(lens), taps - 1, ch)).astype(np.float32)
    with Call(rt, q8rt) as d:
        s = d.seqs(start, longest=longest, t=t)
        y = d.out("y", (t, ch + 4), np.float32)
        s_out = d.out("s", s_in.shape, np.float32, s_in if in_place else None)
        rt.lib.rt_conv_silu_dev(rt.R, c.byref(s), d.put(x), ch + 8, ch, d.put(w), taps, s_out if in_place else d.put(s_in), s_out, y, ch + 4)
        got, state = d.get("y"), d.get("s")
    want, wstate, tol = ref.conv(x[:, :ch], w, s_in, start)
    live = rows_of(start, t)
    assert (np.abs(got[live, :ch] - want[live]) <= tol[live]).all()
    assert np.array_equal(state, wstate.astype(np.float32))
    assert untouched(got[~live]).all() and untouched(got[:, ch:]).all()


def test_conv_extremes(rt, q8rt):
    """SiLU far from zero, infinities, NaN: each in its own channel and within reach of its taps alone."""
    ch, t = 16, 12
    x = np.ones((t, ch), np.float32)
    x[:, 0], x[:, 1], x[3, 2], x[3, 3], x[5, 4] = 200.0, -200.0, np.inf, -np.inf, np.nan
    w, s_in = np.ones((ch, 4), np.float32), np.zeros((1, 3, ch), np.float32)
    start = starts([t])
    with Call(rt, q8rt) as d:
        s = d.seqs(start)
        y, s_out = d.out("y", (t, ch), np.float32), d.out("s", s_in.shape, np.float32)
        rt.lib.rt_conv_silu_dev(rt.R, c.byref(s), d.put(x), ch, ch, d.put(w), 4, d.put(s_in), s_out, y, ch)
        got = d.get("y")
    with np.errstate(invalid="ignore"):
        want, _, tol = ref.conv(x, w, s_in, start)
    fine = np.isfinite(want)
    assert (np.abs(got[fine] - want[fine]) <= tol[fine] + 1e-37).all()
    assert np.isposinf(got[3:7, 2]).all() and np.isnan(got[5:9, 4]).all() and np.isfinite(got[:, 5:]).all()
    assert np.isfinite(got[:3, :5]).all() and np.isfinite(got[9:, :5]).all()


# ---- the gated delta rule


def delta_inputs(rng, t, hk, hv, dk, dv, n):
    q, k = (rng.standard_normal((t, hk, dk)).astype(np.float32) for _ in range(2))
    v = rng.standard_normal((t, hv, dv)).astype(np.float32)
    a, b = (rng.standard_normal((t, hv)).astype(np.float32) for _ in range(2))
    decay = -np.exp(rng.uniform(0, np.log(16), hv)).astype(np.float32)
    dt = np.log(np.expm1(np.exp(rng.uniform(np.log(1e-3), np.log(0.1), hv)))).astype(np.float32)
    s_in = (0.2 * rng.standard_normal((n, hv, dk, dv))).astype(np.float32)
    return q, k, v, a, b, decay, dt, s_in


def run_delta(rt, m, x, start, tiled, eps=EPS, scale=None, z=None, nw=None, t=None, longest=None, in_place=False, graph=False):
    q, k, v, a, b, decay, dt, s_in = x
    rows, hk, dk = q.shape
    hv, dv = v.shape[1:]
    scale = dk ** -0.5 if scale is None else scale
    # q, k and v side by side in a row, as the convolution gives them, with a gap
    ld = 2 * hk * dk + hv * dv + 4
    xs = np.zeros((rows, ld), np.float32)
    xs[:, :hk * dk], xs[:, hk * dk:2 * hk * dk], xs[:, 2 * hk * dk:-4] = q.reshape(rows, -1), k.reshape(rows, -1), v.reshape(rows, -1)
    ab = np.concatenate([a, b, a[:, :1]], 1)  # a stride that is no multiple of 4, an address of any alignment
    with Call(rt, m) as d:
        s = d.seqs(start, longest=longest, t=rows if t is None else t)
        px, pab = d.put(xs), d.put(ab)
        s_out = d.out("s", s_in.shape, np.float32, s_in if in_place else None)
        arg = m.Delta(k_heads=hk, v_heads=hv, k_dim=dk, v_dim=dv, tiled=tiled, q=px, q_ld=ld, k=px + 4 * hk * dk, k_ld=ld, v=px + 8 * hk * dk, v_ld=ld,
                      a=pab, a_ld=2 * hv + 1, b=pab + 4 * hv, b_ld=2 * hv + 1, decay=d.put(decay), dt=d.put(dt), eps=eps, scale=scale,
                      s_in=s_out if in_place else d.put(s_in), s_out=s_out, z=None if z is None else d.put(z), z_ld=hv * dv,
                      nw=None if nw is None else d.put(nw), nw_eps=EPS, o=d.out("o", (rows, hv * dv + 8), np.float32), o_ld=hv * dv + 8)
        rt.lib.rt_delta_rule_dev(rt.R, c.byref(s), c.byref(arg))
        return d.get("o"), d.get("s")


def delta_bound(dk, count):
    """A token's two dot products over dk elements round as random steps, 2 sqrt(dk) + 8 half steps of the
    state's size; what earlier tokens added dies away with the decays and the rule itself (each key's part is
    replaced), so the sum over tokens grows as a random walk of at most some 100: times sqrt(1 + count / 10)
    up to 100 tokens."""
    return U * (2 * np.sqrt(dk) + 8) * np.sqrt(1 + min(count, 100) / 10)


def check_delta(got, state, want, wstate, size, start, dk, width):
    live = rows_of(start, len(got))
    for s in range(len(start) - 1):
        n = start[s + 1] - start[s]
        b = delta_bound(dk, n)
        if n == 0:
            assert np.array_equal(state[s], wstate[s].astype(np.float32))
            continue
        e = np.sqrt(((state[s] - wstate[s]) ** 2).mean((1, 2)) / (wstate[s] ** 2).mean((1, 2)))
        assert (e <= b).all(), ("state", s, e.max(), b)
        r = slice(start[s], start[s + 1])
        err = got[r, :width].reshape(want[r].shape) - want[r]
        assert np.isfinite(err).all()
        # an element's error: within 6 of the random walk's standard deviations (never by chance)
        worst = (np.abs(err) / (size[r] + np.abs(want[r]) + 1e-30)).max()
        assert worst <= 6 * b, ("o", s, worst, b)
    assert untouched(got[~live]).all() and untouched(got[:, width:]).all()


DELTA = [
    # hk, hv, dk, dv, tiled, lens, first, longest
    (1, 1, 32, 16, False, [1], 0, None),
    (2, 4, 64, 48, True, [1, 0, 1, 2], 1, None),
    (16, 32, 128, 128, True, [1], 0, None),
    (2, 6, 96, 80, False, [3, 1, 4], 0, None),
    (2, 2, 192, 112, True, [2, 5], 2, None),
    (1, 2, 256, 64, False, [4, 1], 0, None),
    (1, 1, 128, 512, False, [2], 0, None),
    (2, 4, 128, 128, True, [1] * 67, 0, None),
    # longer runs, about the chunks' borders
    (2, 4, 128, 128, True, [63, 64, 65, 0, 1], 0, None),
    (2, 2, 64, 32, False, [129, 17, 300], 5, None),
    (1, 2, 96, 48, True, [100, 7], 0, None),
    (1, 1, 32, 16, False, [33], 0, None),
    (1, 2, 192, 64, False, [70], 0, None),
    (1, 1, 256, 128, False, [130], 0, None),
    (1, 1, 128, 272, False, [66], 0, None),
    (2, 4, 128, 64, False, [400, 1, 90], 0, 1),
    (2, 2, 128, 64, False, [1, 200, 16, 17, 31, 32, 33], 0, 200),
    (1, 1, 128, 128, False, [1500], 0, None),
]


@pytest.mark.parametrize("hk,hv,dk,dv,tiled,lens,first,longest", DELTA)
@pytest.mark.parametrize("gated,in_place", [(False, True), (True, False)])
def test_delta(rt, q8rt, hk, hv, dk, dv, tiled, lens, first, longest, gated, in_place):
    say("delta", hk, hv, dk, dv, tiled, lens, first, longest, gated, in_place)
    rng = np.random.default_rng(hk + hv + dk + dv + len(lens) + gated)
    start = starts(lens, first)
    t = int(start[-1]) + 3
    x = delta_inputs(rng, t, hk, hv, dk, dv, len(lens))
    z = rng.standard_normal((t, hv, dv)).astype(np.float32) if gated else None
    nw = (1 + 0.1 * rng.standard_normal(dv)).astype(np.float32) if gated else None
    got, state = run_delta(rt, q8rt, x, start, tiled, z=z, nw=nw, t=t, longest=longest, in_place=in_place)
    want, wstate, size = ref.delta(*x[:7], EPS, dk ** -0.5, x[7], start, tiled, z, nw, EPS)
    check_delta(got, state, want, wstate, size, start, dk, hv * dv)


@pytest.mark.parametrize("hk,hv,dk,dv,lens,in_place", [(256, 256, 32, 16, [1100, 20, 900, 40], True), (32, 256, 128, 16, [2500, 33], False)])
def test_delta_alternating(rt, q8rt, hk, hv, dk, dv, lens, in_place):
    """So many heads that the chunks' parts do not fit the workspace at once: runs of chunks are made and taken in turn,
    and a sequence's state goes from one to the next."""
    test_delta(rt, q8rt, hk, hv, dk, dv, False, lens, 0, None, in_place, in_place)


@pytest.mark.parametrize("n", [1, 5, 64, 150])
@pytest.mark.parametrize("what", ["forget", "keep", "write", "one_key", "zero", "alternate", "plain"])
def test_delta_extremes(rt, q8rt, what, n):
    """Decays of exactly 0 (also on some tokens alone) and of 1, gates at their ends, the same key at every
    token with beta near 1 (the triangular system's worst), zero keys and queries, q and k as they are."""
    rng = np.random.default_rng(n)
    hk, hv, dk, dv, start = 1, 2, 128, 32, starts([n, 3])
    q, k, v, a, b, decay, dt, s_in = delta_inputs(rng, n + 3, hk, hv, dk, dv, 2)
    eps = EPS
    if what == "forget":
        a[:] = 1e6
    elif what == "keep":
        a[:], b[:] = -200.0, -200.0
    elif what == "write":
        b[:] = 200.0
    elif what == "one_key":
        k[:], b[:], a[:] = k[:1], 8.0, -50.0
    elif what == "zero":
        k[::2], q[1::3] = 0.0, 0.0
    elif what == "alternate":
        a[::7], decay[:] = 3e4, -16.0
    elif what == "plain":
        eps = -1.0
        k /= np.sqrt((k * k).sum(2, keepdims=True))
    x = (q, k, v, a, b, decay, dt, s_in)
    got, state = run_delta(rt, q8rt, x, start, False, eps=eps)
    want, wstate, size = ref.delta(q, k, v, a, b, decay, dt, eps, dk ** -0.5, s_in, start, False)
    check_delta(got, state, want, wstate, size, start, dk, hv * dv)


@pytest.mark.parametrize("n", [2, 70, 130])
def test_delta_nan_stays_in_its_head(rt, q8rt, n):
    """A NaN of one head's value reaches that head from its token on, and no other head, sequence or earlier token."""
    rng = np.random.default_rng(n)
    start = starts([n, n])
    x = delta_inputs(rng, 2 * n, 2, 2, 64, 32, 2)
    x[2][n // 2, 1, 5] = np.nan
    got, state = run_delta(rt, q8rt, x, start, False)
    got = got[:, :64].reshape(2 * n, 2, 32)
    assert np.isnan(got[n // 2:n, 1, 5]).all() and np.isnan(state[0, 1, :, 5]).all()
    got[n // 2:n, 1, 5], state[0, 1, :, 5] = 0, 0
    assert np.isfinite(got).all() and np.isfinite(state).all()


@pytest.mark.parametrize("lens,hk,hv,dv", [([260], 2, 4, 32), ([260, 33, 64, 65, 200], 8, 8, 128)])  # one workgroup a compute unit, or more
@pytest.mark.parametrize("bad", [None, 0, 70, 150, 259])
def test_delta_chunks_around_a_nan(rt, q8rt, lens, hk, hv, dv, bad):
    """The chunks before, with and after a value that is NaN: all that it does not reach is as without it."""
    say("delta nan", lens, hk, hv, dv, bad)
    rng = np.random.default_rng(len(lens))
    start = starts(lens)
    t = int(start[-1])
    x = delta_inputs(rng, t, hk, hv, 128, dv, len(lens))
    want, wstate, size = ref.delta(*x[:7], EPS, 128 ** -0.5, x[7], start, False)
    if bad is not None:
        x[2][bad, 1, 5] = np.nan
    got, state = run_delta(rt, q8rt, x, start, False)
    if bad is not None:
        o = got[:, :hv * dv].reshape(t, hv, dv)
        assert np.isnan(o[bad:lens[0], 1, 5]).all() and np.isnan(state[0, 1, :, 5]).all()
        o[bad:lens[0], 1, 5], state[0, 1, :, 5] = want[bad:lens[0], 1, 5], wstate[0, 1, :, 5]
    check_delta(got, state, want, wstate, size, start, 128, hv * dv)


# ---- heads: norm, rotation, append


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hk,dim,rot,pairs,norm,page,news,pasts,first", [
    (4, 1, 256, 64, False, True, 16, [1], [5], 0), (3, 2, 96, 96, False, True, 7, [3, 0, 10], [0, 4, 13], 1), (2, 2, 32, 30, False, True, 1, [4, 2], [1, 0], 0),
    (8, 2, 128, 128, True, True, 64, [1] * 66, list(range(66)), 0), (1, 1, 224, 10, True, False, 5, [9], [1000003], 0), (2, 1, 64, 0, False, True, 16, [2], [15], 0),
    (5, 1, 160, 42, True, True, 48, [50, 1], [30, 47], 2), (2, 1, 192, 192, False, False, 3, [4], [2], 0)])
def test_rope(rt, q8rt, kind, hq, hk, dim, rot, pairs, norm, page, news, pasts, first):
    say("rope", kind, hq, hk, dim, rot, pairs, norm, page, news, first)
    rng = np.random.default_rng(hq + dim + rot + page)
    start = starts(news, first)
    t, n = int(start[-1]) + 2, len(news)
    far = max(pasts) > 10000  # a far position: a table whose last page alone is there
    q, k, v = (rng.standard_normal((t, h, dim + 4)).astype(np.float32) for h in (hq, hk, hk))
    qn, kn = ((1 + 0.1 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2))
    freq = 1e6 ** (-np.arange(0, rot, 2) / max(rot, 1))
    total = [a + b for a, b in zip(pasts, news)]
    need = [-(-x // page) for x in total]
    ld, pages = max(need), sum(min(x, 40) for x in need) + 1
    table, order, at = np.full((n, ld), -1, np.int32), rng.permutation(pages).astype(np.int32), 0
    for s in range(n):
        m = min(need[s], 40)
        table[s, need[s] - m:need[s]] = order[at:at + m]
        at += m
    dtype = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[kind]
    old = ref.to_cache(rng.standard_normal((pages, hk, page, dim)), kind)
    with Call(rt, q8rt) as d:
        s = d.seqs(start, pasts, t=t)
        kv = q8rt.Kv(k=d.out("ck", old.shape, dtype, old), v=d.out("cv", old.shape, dtype, old), type=q8rt.TYPES[kind], dim=dim, heads=hk, page=page, pages=pages,
                     table=d.put(table), table_ld=ld)
        a = q8rt.Rope(q=d.put(q), q_ld=hq * (dim + 4), q_hd=dim + 4, q_heads=hq, k=d.put(k), k_ld=hk * (dim + 4), k_hd=dim + 4, v=d.put(v),
                      v_ld=hk * (dim + 4), v_hd=dim + 4, q_norm=d.put(qn) if norm else None, k_norm=d.put(kn) if norm else None, eps=EPS, rot=rot, pairs=pairs,
                      freq=d.put(freq) if rot else None, out=d.out("q", (t, hq, dim), np.float32), out_ld=hq * dim, out_hd=dim)
        rt.lib.rt_rope_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
        got, ck, cv = d.get("q"), d.get("ck"), d.get("cv")
    live = rows_of(start, t)
    pos = np.zeros(t, np.int64)
    for i in range(n):
        pos[start[i]:start[i + 1]] = pasts[i] + np.arange(news[i])

    def tol(x, y):
        # the norm: 12 half steps on each of the two elements that an output mixes; the angle's sine and cosine 2 more, the sums
        m = np.abs(x).copy()
        if rot:
            i, j = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
            m[..., i] = m[..., j] = m[..., i] + m[..., j]
        return 18 * U * m + 1e-30

    qw = ref.head_norm(q[..., :dim], qn if norm else None, EPS)
    want = ref.turn(qw, pos, freq, rot, pairs)
    assert (np.abs(got[live] - want[live]) <= tol(qw, want)[live]).all()
    assert untouched(got[~live]).all()
    kw = ref.head_norm(k[..., :dim], kn if norm else None, EPS)
    kt = ref.turn(kw, pos, freq, rot, pairs)
    written = np.zeros((pages, page), bool)
    for i in range(n):
        for r in range(start[i], start[i + 1]):
            p = pos[r]
            where = table[i, p // page]
            written[where, p % page] = True
            e = ref.of_cache(ck[where, :, p % page], kind) - kt[r]
            assert (np.abs(e) <= tol(kw, kt)[r] + ref.HALF[kind] * np.abs(kt[r]) * (1 + 1e-4) + 2.0 ** -25).all()
            assert np.array_equal(cv[where, :, p % page], ref.to_cache(v[r, :, :dim], kind))
    keep = np.broadcast_to(~written[:, None, :, None], old.shape)
    assert np.array_equal(ck[keep], old[keep]) and np.array_equal(cv[keep], old[keep])
    assert far or written.sum() == sum(news)


def test_rope_in_place_and_pages_that_are_not_there(rt, q8rt):
    """q turned in place; positions before 0, behind the table and in pages that the cache lacks are not stored, and the rest is."""
    rng = np.random.default_rng(5)
    hq, hk, dim, page, pages = 2, 1, 64, 4, 3
    start, pasts = starts([6, 6, 2]), [-2, 5, 8]
    table = np.array([[0, 3], [-1, 2], [1, 1]], np.int32)  # 3 and -1: not there; the third sequence's position 8 lies behind the table
    t = int(start[-1])
    q, k, v = (rng.standard_normal((t, h, dim)).astype(np.float32) for h in (hq, hk, hk))
    freq = 1e4 ** (-np.arange(0, dim, 2) / dim)
    old = np.zeros((pages, hk, page, dim), np.float32)
    with Call(rt, q8rt) as d:
        s = d.seqs(start, pasts)
        kv = q8rt.Kv(k=d.out("ck", old.shape, np.float32, old), v=d.out("cv", old.shape, np.float32, old), type=0, dim=dim, heads=hk, page=page, pages=pages,
                     table=d.put(table), table_ld=2)
        p = d.out("q", q.shape, np.float32, q)
        a = q8rt.Rope(q=p, q_ld=hq * dim, q_hd=dim, q_heads=hq, k=d.put(k), k_ld=hk * dim, k_hd=dim, v=d.put(v), v_ld=hk * dim, v_hd=dim, eps=EPS, rot=dim,
                      freq=d.put(freq), out=p, out_ld=hq * dim, out_hd=dim)
        rt.lib.rt_rope_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
        got, cv = d.get("q"), d.get("cv")
    pos = np.concatenate([np.arange(6) - 2, np.arange(6) + 5, np.arange(2) + 8])
    want = ref.turn(q.astype(np.float64), pos, freq, dim, False)
    assert (np.abs(got - want) <= 12 * U * 2 * np.abs(q).max()).all()
    expect = old.copy()
    for r, (seq, p) in enumerate(zip([0] * 6 + [1] * 6 + [2] * 2, pos)):
        if 0 <= p < 2 * page and 0 <= table[seq, p // page] < pages:
            expect[table[seq, p // page], :, p % page] = v[r]
    assert np.array_equal(cv, expect)


# ---- attention over the cache


def run_attn(rt, m, cache, q, start, pasts, scale, gate=None, t=None, longest=None, pages=None):
    rows, hq, dim = q.shape
    with Call(rt, m) as d:
        s = d.seqs(start, pasts, longest=longest, t=rows if t is None else t)
        kv = cache.struct(d)
        if pages is not None:
            kv.pages = pages
        qg = np.concatenate([q, np.zeros_like(q) if gate is None else gate], 2)  # a head's gate beside its query
        p = d.put(qg)
        a = m.Attn(q=p, q_ld=2 * hq * dim, q_hd=2 * dim, q_heads=hq, scale=scale, gate=None if gate is None else p + 4 * dim, gate_ld=2 * hq * dim, gate_hd=2 * dim,
                   o=d.out("o", (rows, hq * dim + 4), np.float32), o_ld=hq * dim + 4)
        rt.lib.rt_attn_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
        return d.get("o")


ATTN = [
    # hq, hk, dim, page, positions a sequence (its new tokens with them), new tokens, first
    (1, 1, 32, 16, [1], [1], 0),
    (4, 1, 256, 16, [17, 1, 5], [1, 1, 1], 0),
    (16, 4, 256, 64, [777], [1], 0),
    (16, 4, 256, 16, [300, 31], [4, 4], 0),
    (6, 2, 96, 7, [100, 0, 3, 16], [3, 0, 3, 1], 2),
    (8, 8, 64, 24, [65, 64, 63], [1, 2, 1], 0),
    (8, 1, 128, 1, [50], [2], 0),
    (12, 2, 160, 5, [33, 200], [5, 6], 1),
    (40, 2, 64, 16, [130], [1], 0),
    (3, 1, 192, 16, [48, 47, 49], [1, 1, 1], 0),
    (2, 1, 224, 100, [250], [2], 0),
    (4, 2, 128, 16, [90, 40], [37, 40], 0),
    (16, 1, 64, 256, [5000], [1], 0),
    (4, 1, 128, 16, [3000, 10, 2049], [2, 1, 1], 0),
    (2, 1, 64, 16, [20] * 70, [1] * 70, 0),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hk,dim,page,lens,news,first", ATTN)
def test_attn(rt, q8rt, kind, hq, hk, dim, page, lens, news, first):
    say("attn", kind, hq, hk, dim, page, lens[:5], news[:5], first)
    rng = np.random.default_rng(hq + dim + page + len(lens))
    start = starts(news, first)
    t = int(start[-1]) + 2
    cache = Paged(rng, kind, lens, hk, dim, page)
    q = (2 * rng.standard_normal((t, hq, dim))).astype(np.float32)
    gate = rng.standard_normal((t, hq, dim)).astype(np.float32) if hq % 2 == 0 else None
    pasts = [a - b for a, b in zip(lens, news)]
    live = rows_of(start, t)
    want, tol = ref.attn(q, cache.seq_k, cache.seq_v, dim ** -0.5, start, pasts, gate)
    for longest in (None, 1):
        got = run_attn(rt, q8rt, cache, q, start, pasts, dim ** -0.5, gate, t=t, longest=longest)
        assert untouched(got[~live]).all() and untouched(got[:, hq * dim:]).all()
        assert (np.abs(got[live, :hq * dim].reshape(-1, hq, dim) - want[live]) <= tol[live]).all()


PROMPTS = [
    # prompts that fill the GPU by themselves, alone and with a sequence that is longer or shorter: cut, or not
    (16, 8, 64, 16, [600], [600], 0),
    (16, 8, 64, 16, [3001, 600], [1, 600], 3),
    (8, 8, 256, 64, [900, 520, 5], [20, 520, 5], 0),
    (16, 4, 128, 24, [270, 2100], [270, 33], 1),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hk,dim,page,lens,news,first", PROMPTS)
def test_attn_prompts(rt, q8rt, kind, hq, hk, dim, page, lens, news, first):
    test_attn(rt, q8rt, kind, hq, hk, dim, page, lens, news, first)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_attn_large_scores(rt, q8rt, kind):
    """Scores of hundreds (their exponentials overflow without the maximum), negative scales, one key far above the rest."""
    rng = np.random.default_rng(9)
    lens, news, dim = [700, 90], [2, 1], 64
    for scale in (8.0, -8.0, 0.0):
        cache = Paged(rng, kind, lens, 2, dim, 16)
        q = (4 * rng.standard_normal((3, 4, dim))).astype(np.float32)
        start, pasts = starts(news), [698, 89]
        want, tol = ref.attn(q, cache.seq_k, cache.seq_v, scale, start, pasts)
        got = run_attn(rt, q8rt, cache, q, start, pasts, scale)[:, :4 * dim].reshape(3, 4, dim)
        assert (np.abs(got - want) <= tol).all(), scale


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("lens", [[40], [2100]])
def test_attn_masked_places(rt, q8rt, kind, bad, lens):
    """NaN and infinities in the keys and values of later new tokens do not reach earlier ones, those of another
    head not this one; the tokens that do see them show them as the definition does."""
    rng = np.random.default_rng(11)
    hq, hk, dim, new = 4, 2, 64, 6
    n = lens[0]
    k, v = (rng.standard_normal((n, hk, dim)) for _ in range(2))
    k[n - 3, 0], v[n - 2, :, 3], v[n - 5, 1, 7] = bad, bad, bad
    cache = Paged(rng, kind, lens, hk, dim, 16, k=[k], v=[v])
    q = rng.standard_normal((new, hq, dim)).astype(np.float32)
    start, pasts = starts([new]), [n - new]
    want, tol = ref.attn(q, cache.seq_k, cache.seq_v, 0.125, start, pasts)
    got = run_attn(rt, q8rt, cache, q, start, pasts, 0.125)[:, :hq * dim].reshape(new, hq, dim)
    fine = np.isfinite(want)
    assert fine[:new - 3, :2].all() and fine[0].all()
    assert (np.abs(got - want)[fine] <= tol[fine]).all()
    # a value's infinity stays one unless a NaN joins it; a key's makes scores of either sign
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])


def test_attn_empty_rows_and_pages_that_are_not_there(rt, q8rt):
    """Tokens before position 0 give zeros; behind the table, or on a page outside the cache, NaN; the others their values."""
    rng = np.random.default_rng(12)
    hq, hk, dim, page = 2, 1, 64, 16
    lens, news = [100, 60, 40, 30], [1, 2, 4, 3]
    cache = Paged(rng, "f16", lens, hk, dim, page)
    start, t = starts(news), sum(news)
    q = rng.standard_normal((t, hq, dim)).astype(np.float32)
    pasts = [99, 58, -2, 27]
    cache.table[1, 2] = cache.pages  # positions 32 to 47 of the second sequence
    want, tol = ref.attn(q, cache.seq_k, cache.seq_v, 0.125, start, pasts)
    got = run_attn(rt, q8rt, cache, q, start, pasts, 0.125)[:, :hq * dim].reshape(t, hq, dim)
    assert np.isnan(got[1:3]).all()
    ok = np.r_[0, 3:t]
    assert (got[3:5] == 0).all() and (np.abs(got - want)[ok] <= tol[ok]).all()
    cache.table[1, 2] = -1
    assert np.isnan(run_attn(rt, q8rt, cache, q, start, pasts, 0.125)[1:3, :hq * dim]).all()
    pasts = [cache.ld * page, 58, 0, -(2 ** 31)]
    got = run_attn(rt, q8rt, cache, q, start, pasts, 0.125)[:, :hq * dim]
    assert np.isnan(got[:3]).all() and np.isfinite(got[3:7]).all() and (got[7:] == 0).all()


@pytest.mark.parametrize("kind,small", [("f16", 2.0 ** -18), ("bf16", 2.0 ** -100), ("f32", 2.0 ** -100)])
def test_attn_small_values(rt, q8rt, kind, small):
    """Keys and values far below 1 (in F16 among its subnormals, which count in full), queries as far above."""
    rng = np.random.default_rng(16)
    n, hq, dim = 300, 4, 64
    cache = Paged(rng, kind, [n], 1, dim, 16, k=[small * rng.standard_normal((n, 1, dim))], v=[small * rng.standard_normal((n, 1, dim))])
    q = (rng.standard_normal((1, hq, dim)) / small).astype(np.float32)
    want, tol = ref.attn(q, cache.seq_k, cache.seq_v, 0.125, starts([1]), [n - 1])
    got = run_attn(rt, q8rt, cache, q, starts([1]), [n - 1], 0.125)[:, :hq * dim].reshape(1, hq, dim)
    assert (np.abs(got - want) <= tol).all()


# ---- starts that make no sense, several calls, graphs


def test_starts_out_of_range_stay_inside(rt, q8rt):
    """starts that descend, or reach before 0 and behind t: nothing outside the arrays is written."""
    rng = np.random.default_rng(13)
    t, hq, dim = 20, 2, 64
    for start in ([-5, 3, 2, 50], [0, 100, -100, 7], [30, 40, 50, 60], [2 ** 31 - 1, -2 ** 31, 5, 9]):
        start = np.array(start)
        x = delta_inputs(rng, t, 1, 1, 32, 16, 3)
        run_delta(rt, q8rt, x, start, False, t=t, longest=t)
        cache = Paged(rng, "f32", [30, 30, 30], 1, dim, 16)
        run_attn(rt, q8rt, cache, rng.standard_normal((t, hq, dim)).astype(np.float32), start, [5, 6, 7], 0.1, t=t, longest=t)
        with Call(rt, q8rt) as d:
            s = d.seqs(start, t=t, longest=t)
            w, s_in = np.ones((8, 4), np.float32), np.ones((3, 3, 8), np.float32)
            rt.lib.rt_conv_silu_dev(rt.R, c.byref(s), d.put(np.ones((t, 8), np.float32)), 8, 8, d.put(w), 4, d.put(s_in), d.out("s", s_in.shape, np.float32),
                                    d.out("y", (t, 8), np.float32), 8)
            d.get("s"), d.get("y")


def test_calls_repeat_bit_for_bit(rt, q8rt):
    """The same call again, other calls between: the same bits."""
    rng = np.random.default_rng(14)
    x, start = delta_inputs(rng, 300, 2, 4, 128, 128, 2), starts([200, 100])
    cache = Paged(rng, "bf16", [3000, 70], 2, 128, 16)
    q = rng.standard_normal((2, 8, 128)).astype(np.float32)
    first = run_delta(rt, q8rt, x, start, True), run_attn(rt, q8rt, cache, q, starts([1, 1]), [2999, 69], 0.1)
    run_delta(rt, q8rt, delta_inputs(rng, 700, 1, 2, 128, 64, 1), starts([700]), True)
    again = run_delta(rt, q8rt, x, start, True), run_attn(rt, q8rt, cache, q, starts([1, 1]), [2999, 69], 0.1)
    for a, b in zip((*first[0], first[1]), (*again[0], again[1])):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


# ---- recorded steps


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_recorded_decode_steps_go_on(rt, q8rt, kind):
    """A decode step of all four operators, recorded once and replayed as positions, pages and states move on in
    device memory: every replay's outputs and states bit for bit an eager run's, with eager work and waits
    between the replays."""
    rng = np.random.default_rng(21)
    n, ch, hk, hv, dk, dv, hq, kvh, dim, page, steps = 3, 384, 1, 2, 128, 64, 4, 2, 64, 8, 4
    lens = [5, 40, 300]
    start = starts([1] * n)
    cache = Paged(rng, kind, [v + steps for v in lens], kvh, dim, page)
    xs = rng.standard_normal((steps, n, ch)).astype(np.float32)
    w, conv_in = rng.standard_normal((ch, 4)).astype(np.float32), rng.standard_normal((n, 3, ch)).astype(np.float32)
    a, b = (rng.standard_normal((n, hv)).astype(np.float32) for _ in range(2))
    decay, dt = -np.ones(hv, np.float32), np.zeros(hv, np.float32)
    state = (0.1 * rng.standard_normal((n, hv, dk, dv))).astype(np.float32)
    qkv = rng.standard_normal((steps, n, (hq + 2 * kvh) * dim)).astype(np.float32)
    freq = 1e4 ** (-np.arange(0, dim, 2) / dim)

    def run(recorded):
        with Call(rt, q8rt) as d:
            lib, R = rt.lib, rt.R
            past = d.put(np.array(lens, np.int32))
            s = q8rt.Seqs(n=n, t=n, longest=1, start=d.put(start.astype(np.int32)), past=past)
            x, y = d.put(xs[0]), d.out("y", (n, ch), np.float32)
            cs, ss = d.out("cs", conv_in.shape, np.float32, conv_in), d.out("ss", state.shape, np.float32, state)
            kv = cache.struct(d, written=True)
            src, q, o, da = d.put(qkv[0]), d.out("q", (n, hq, dim), np.float32), d.out("o", (n, hq * dim), np.float32), d.out("do", (n, hv * dv), np.float32)
            width = (hq + 2 * kvh) * dim
            delta = q8rt.Delta(k_heads=hk, v_heads=hv, k_dim=dk, v_dim=dv, q=y, q_ld=ch, k=y + 4 * dk, k_ld=ch, v=y + 8 * dk, v_ld=ch, a=d.put(a), a_ld=hv, b=d.put(b),
                               b_ld=hv, decay=d.put(decay), dt=d.put(dt), eps=EPS, scale=dk ** -0.5, s_in=ss, s_out=ss, o=da, o_ld=hv * dv)
            rope = q8rt.Rope(q=src, q_ld=width, q_hd=dim, q_heads=hq, k=src + 4 * hq * dim, k_ld=width, k_hd=dim, v=src + 4 * (hq + kvh) * dim, v_ld=width, v_hd=dim,
                             eps=EPS, rot=dim, freq=d.put(freq), out=q, out_ld=hq * dim, out_hd=dim)
            attn = q8rt.Attn(q=q, q_ld=hq * dim, q_hd=dim, q_heads=hq, scale=0.125, o=o, o_ld=hq * dim)
            taps = d.put(w)

            def step():
                lib.rt_conv_silu_dev(R, c.byref(s), x, ch, ch, taps, 4, cs, cs, y, ch)
                lib.rt_delta_rule_dev(R, c.byref(s), c.byref(delta))
                lib.rt_rope_kv_dev(R, c.byref(s), c.byref(kv), c.byref(rope))
                lib.rt_attn_kv_dev(R, c.byref(s), c.byref(kv), c.byref(attn))

            graph = None
            if recorded:
                step()  # the workspaces; then the states as they were
                for name, p, data in (("cs", cs, conv_in), ("ss", ss, state)):
                    rt.to_dev(p, data)
                lib.rt_graph_begin(R)
                step()
                graph = c.c_void_p(lib.rt_graph_end(R))
            got = []
            for i in range(steps):
                rt.to_dev(x, xs[i])
                rt.to_dev(src, qkv[i])
                rt.to_dev(past, np.array(lens, np.int32) + i)
                if graph:
                    lib.rt_graph_launch(R, graph)
                else:
                    step()
                got.append([d.get(k) for k in ("y", "do", "q", "o", "cs", "ss")])
                if graph:  # eager work of the same operators between the replays
                    run_attn(rt, q8rt, Paged(rng, kind, [900], 1, 128, 16), np.ones((1, 2, 128), np.float32), starts([1]), [899], 0.1)
            if graph:
                lib.rt_graph_free(R, graph)
            return got

    for i, (x, y) in enumerate(zip(run(False), run(True))):
        for p, q in zip(x, y):
            assert np.isfinite(p).all() and np.array_equal(p.view(np.uint32), q.view(np.uint32)), i


def test_recorded_prompts(rt, q8rt):
    """The chunks of a prompt and attention split over positions, recorded: three replays give the eager bits."""
    rng = np.random.default_rng(22)
    hk, hv, dk, dv, start = 1, 2, 128, 64, starts([300, 70])
    x = delta_inputs(rng, 370, hk, hv, dk, dv, 2)
    cache, q = Paged(rng, "bf16", [2000, 90], 2, 128, 16), rng.standard_normal((2, 8, 128)).astype(np.float32)
    want = run_delta(rt, q8rt, x, start, True), run_attn(rt, q8rt, cache, q, starts([1, 1]), [1999, 89], 0.1)
    real, records = rt.lib, []

    class Recorded:
        """The library with its calls recorded first, then replayed three times, an eager wait between."""

        def __getattr__(self, name):
            fn = getattr(real, name)
            if name not in ("rt_delta_rule_dev", "rt_attn_kv_dev"):
                return fn

            def call(*args):
                real.rt_graph_begin(rt.R)
                fn(*args)
                g = c.c_void_p(real.rt_graph_end(rt.R))
                for _ in range(3):
                    real.rt_graph_launch(rt.R, g)
                    real.rt_dev_sync(rt.R)
                records.append(name)
                real.rt_graph_free(rt.R, g)

            return call

    rt.lib = Recorded()
    try:
        got = run_delta(rt, q8rt, x, start, True), run_attn(rt, q8rt, cache, q, starts([1, 1]), [1999, 89], 0.1)
    finally:
        rt.lib = real
    assert len(records) == 2
    for a, b in zip((*want[0], want[1][:, :1024]), (*got[0], got[1][:, :1024])):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_two_runtimes_side_by_side(q8rt, rt):
    """A second runtime's calls (a stream and workspaces of its own) between this one's, none waited for: both right."""
    rng = np.random.default_rng(23)
    cache = Paged(rng, "f16", [3000], 1, 128, 16)
    q = rng.standard_normal((1, 4, 128)).astype(np.float32)
    want, tol = ref.attn(q, cache.seq_k, cache.seq_v, 0.1, starts([1]), [2999])
    other = q8rt.Runtime()
    try:
        calls = []
        for r in (rt, other, rt, other):
            d = Call(r, q8rt)
            s, kv = d.seqs(starts([1]), [2999]), cache.struct(d)
            a = q8rt.Attn(q=d.put(q), q_ld=512, q_hd=128, q_heads=4, scale=0.1, o=d.out("o", (1, 512), np.float32), o_ld=512)
            calls.append((r, d, s, kv, a))
        for r, d, s, kv, a in calls:
            r.lib.rt_attn_kv_dev(r.R, c.byref(s), c.byref(kv), c.byref(a))
        for r, d, *_ in calls:
            assert (np.abs(d.get("o").reshape(1, 4, 128) - want) <= tol).all()
            d.__exit__()
    finally:
        other.close()


def test_first_call_of_a_size_while_recording_is_refused(q8rt):
    """A recording may not grow the workspace: the call says so and ends the process (a child here, which never replays)."""
    import os
    import subprocess
    import sys

    code = """
import ctypes as c, sys
sys.path.insert(0, "tests")
import numpy as np
from conftest import load_package
m = load_package()
import mix_ref as ref
rt = m.Runtime()
cache = ref.Paged(np.random.default_rng(1), "f16", [500], 1, 64, 16)
with ref.Call(rt, m) as d:
    s, kv = d.seqs(ref.starts([1]), [499]), cache.struct(d)
    a = m.Attn(q=d.put(np.ones((1, 2, 64), np.float32)), q_ld=128, q_hd=64, q_heads=2, scale=0.1, o=d.out("o", (1, 128), np.float32), o_ld=128)
    rt.lib.rt_graph_begin(rt.R)
    print("child: recording", flush=True)
    rt.lib.rt_attn_kv_dev(rt.R, c.byref(s), c.byref(kv), c.byref(a))
    print("child: returned", flush=True)
"""
    p = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, Q8_ABORT_EXIT="43"), capture_output=True, text=True, timeout=120,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert p.returncode == 43 and "child: recording" in p.stdout and "child: returned" not in p.stdout, (p.returncode, p.stdout, p.stderr)
    assert "must grow while a graph is being recorded" in p.stderr
