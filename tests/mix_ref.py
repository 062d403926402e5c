"""The operators of include/q8_mix.h in 64 bits, from their definitions (numpy, token by token), and the
calls of the library on the same numpy arrays. Outputs come back with what lies around them checked:
every output buffer has a margin of a known pattern on both sides, and starts out filled with it."""
import ctypes as c

import numpy as np

U = 2.0 ** -24  # half a step of F32, relative
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
MARGIN = 1024
FILL = np.uint32(0x7FC0DEAD)  # a NaN of its own


def sigmoid(x):
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1.0, e) / (1.0 + e)


# ---- the definitions


def conv(x, w, s_in, start):
    """(y [t ch], state [n taps-1 ch], a bound on |y|'s F32 error)"""
    x, w, s_in = (a.astype(np.float64) for a in (x, w, s_in))
    n, taps = s_in.shape[0], w.shape[1]
    y, size = np.full(x.shape, np.nan), np.zeros(x.shape)
    state = s_in.copy()
    for s in range(n):
        u = np.concatenate([s_in[s], x[start[s]:start[s + 1]]])
        for i in range(start[s + 1] - start[s]):
            y[start[s] + i] = (w.T * u[i:i + taps]).sum(0)
            size[start[s] + i] = np.abs(w.T * u[i:i + taps]).sum(0)
        state[s] = u[len(u) - (taps - 1):]
    # the sum: taps roundings, through SiLU's slope of at most 1.1; SiLU itself: exp, the sum, the quotient, the product
    return y * sigmoid(y), state, U * (1.1 * taps * size + 8 * np.abs(y))


def delta(q, k, v, a, b, decay, dt, eps, scale, s_in, start, tiled, z=None, nw=None, nw_eps=0.0):
    """q, k [t hk dk], v [t hv dv], a, b [t hv], s_in [n hv dk dv]: (o [t hv dv], state, the size that o's error is relative to)"""
    q, k, v, a, b, decay, dt, s_in = (x.astype(np.float64) for x in (q, k, v, a, b, decay, dt, s_in))
    hk, hv = q.shape[1], v.shape[1]
    of = np.arange(hv) % hk if tiled else np.arange(hv) // (hv // hk)
    if eps >= 0:
        q, k = (x / np.sqrt((x * x).sum(2, keepdims=True) + eps) for x in (q, k))
    with np.errstate(over="ignore"):
        alpha = np.exp(decay * np.logaddexp(0.0, a + dt))
    beta = sigmoid(b)
    o, size, state = np.full(v.shape, np.nan), np.zeros(v.shape), s_in.copy()
    for s in range(s_in.shape[0]):
        m = state[s]
        for i in range(start[s], start[s + 1]):
            m *= alpha[i][:, None, None]
            d = beta[i][:, None] * (v[i] - np.einsum("hkv,hk->hv", m, k[i, of]))
            m += k[i, of][:, :, None] * d[:, None, :]
            o[i] = scale * np.einsum("hkv,hk->hv", m, q[i, of])
            size[i] = abs(scale) * np.sqrt((m * m).sum(1)) * np.sqrt((q[i, of] ** 2).sum(1))[:, None]
    if z is not None:
        r = 1 / np.sqrt((o * o).mean(2, keepdims=True) + nw_eps)
        g = np.abs(nw * z * sigmoid(z.astype(np.float64)))
        # an error of o reaches the normed o through its own element and through the norm
        size = r * g * (size + np.abs(o) * r * np.sqrt((size * size).mean(2, keepdims=True)))
        o = o * r * nw * z * sigmoid(z.astype(np.float64))
    return o, state, size


def turn(x, pos, freq, rot, pairs):
    """x [t h d] turned by pos [t]"""
    x = x.copy()
    ang = pos.astype(np.float64)[:, None, None] * freq
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., i].copy(), x[..., j].copy()
    x[..., i], x[..., j] = a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)
    return x


def head_norm(x, nw, eps):
    x = x.astype(np.float64)
    return x if nw is None else nw.astype(np.float64) * x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def attn(q, k, v, scale, start, past, gate=None):
    """q [t hq d]; k, v: per sequence [positions hk d] in 64 bits, a page that is not there as NaN. (o, a bound on its F32 error)"""
    t, hq, d = q.shape
    o, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for s in range(len(past)):
        for i in range(start[s], start[s + 1]):
            m = past[s] + i - start[s] + 1
            if m <= 0:
                o[i] = 0.0
                continue
            for h in range(hq):
                kh = h // (hq // k[s].shape[1])
                kk, vv = k[s][:m, kh], v[s][:m, kh]
                if len(kk) < m:
                    continue  # behind the table: NaN
                with np.errstate(invalid="ignore", over="ignore"):
                    x = scale * (kk @ q[i, h].astype(np.float64))
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    o[i, h] = p @ vv
                    # the scores' sums of d products, rounding as random steps, and the sum over the positions
                    ds = U * (2 * np.sqrt(d) + 8) * (np.abs(kk) @ np.abs(q[i, h].astype(np.float64)) * abs(scale)).max()
                    tol[i, h] = (2 * ds + U * (2 * np.sqrt(m) + 16)) * (p @ np.abs(vv))
    if gate is not None:
        g = sigmoid(gate.astype(np.float64))
        o, tol = o * g, tol * g + 4 * U * np.abs(o * g)
    return o, tol + 2.0 ** -140


# ---- the cache's types


def to_cache(x, kind):
    """64- or 32-bit values as the cache's bytes (to nearest, ties to even)"""
    x = np.asarray(x, np.float32)
    if kind == "f32":
        return x.copy()
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def of_cache(x, kind):
    if kind == "bf16":
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return x.astype(np.float64)


# ---- the library


class Call:
    """Device buffers of one call: inputs, and outputs with margins."""

    def __init__(self, rt, m):
        self.rt, self.m, self.bufs, self.outs = rt, m, [], {}

    def __enter__(self):
        return self

    def __exit__(self, *e):
        for p in self.bufs:
            self.rt.free(p)

    def put(self, a):
        a = np.ascontiguousarray(a)
        p = self.rt.alloc(max(a.nbytes, 16))
        if a.nbytes:
            self.rt.to_dev(p, a)
        self.bufs.append(p)
        return p

    def out(self, name, shape, dtype, data=None):
        """An output of the call, filled with the pattern, or with data where the call also reads it"""
        n = int(np.prod(shape)) * np.dtype(dtype).itemsize
        raw = np.full((2 * MARGIN + (n + 3) // 4 * 4) // 4, FILL, np.uint32).view(np.uint8)
        if data is not None:
            raw[MARGIN:MARGIN + n] = np.ascontiguousarray(data, dtype).view(np.uint8).reshape(-1)
        p = self.put(raw)
        self.outs[name] = (p, shape, dtype, n, len(raw))
        return p + MARGIN

    def get(self, name):
        p, shape, dtype, n, full = self.outs[name]
        raw = np.empty(full, np.uint8)
        self.rt.from_dev(raw, p)
        assert (raw[:MARGIN].view(np.uint32) == FILL).all() and (raw[MARGIN + (n + 3) // 4 * 4:].view(np.uint32) == FILL).all(), f"{name}: written outside"
        return raw[MARGIN:MARGIN + n].copy().view(dtype).reshape(shape)

    def seqs(self, start, past=None, longest=None, t=None):
        n = len(start) - 1
        t = int(start[-1]) if t is None else t
        longest = max(1, int(np.diff(start).max())) if longest is None else longest
        self.keep = self.m.Seqs(n=n, t=t, longest=longest, start=self.put(np.asarray(start, np.int32)),
                                past=None if past is None else self.put(np.asarray(past, np.int32)))
        return self.keep


def untouched(a):
    return np.ascontiguousarray(a).view(np.uint32) == FILL


def starts(lens, first=0):
    return np.concatenate([[first], first + np.cumsum(lens)]).astype(np.int64)


class Paged:
    """A paged cache of sequences: the pages of k and v, the table, and per sequence their values in 64 bits."""

    def __init__(self, rng, kind, lens, heads, dim, page, spare=2, k=None, v=None):
        self.kind, self.heads, self.dim, self.page = kind, heads, dim, page
        need = [-(-n // page) for n in lens]
        self.pages, self.ld = sum(need) + spare, max(need + [1]) + 1
        self.table = np.full((len(lens), self.ld), -7, np.int32)
        order, at = rng.permutation(self.pages).astype(np.int32), 0
        shape = (self.pages, heads, page, dim)
        # what no sequence has is NaN: nothing of it may reach an output
        self.k, self.v = (to_cache(np.full(shape, np.nan), kind) for _ in range(2))
        self.seq_k, self.seq_v = [], []
        for s, n in enumerate(lens):
            self.table[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            for pool, mine, given in ((self.k, self.seq_k, k), (self.v, self.seq_v, v)):
                x = rng.standard_normal((n, heads, dim)) if given is None else given[s]
                pos = np.arange(n)
                raw = to_cache(x, kind)
                pool[self.table[s, pos // page], :, pos % page] = raw
                mine.append(of_cache(raw, kind))

    def struct(self, call, written=False):
        a = self.k.dtype
        k = call.out("ck", self.k.shape, a, self.k) if written else call.put(self.k)
        v = call.out("cv", self.v.shape, a, self.v) if written else call.put(self.v)
        m = call.m
        self.keep = m.Kv(k=k, v=v, type=m.TYPES[self.kind], dim=self.dim, heads=self.heads, page=self.page, pages=self.pages, table=call.put(self.table),
                         table_ld=self.ld)
        return self.keep
