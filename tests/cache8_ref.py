"""The 8-bit cache, reading a cache back, and attention through a window (include/q8_mix.h) from their definitions:
a row's quantisation in F32 as it is defined, the rest in 64 bits, on mix_ref.py's paged caches."""
import numpy as np

import mix_ref as ref
from mix_ref import U, Paged

F = np.float32


def quantise(x):
    """F32 rows [..., d] as (int8 values, F32 scales)"""
    x = np.asarray(x, F)
    with np.errstate(all="ignore"):
        most = np.abs(x).max(-1)
        d = most / F(127)
        bad, small = ~np.isfinite(x).all(-1), d < F(2.0 ** -126)
        q = np.rint(x / d[..., None])
    q[bad | small] = 0
    return q.astype(np.int8), np.where(bad, F(np.nan), np.where(small, F(0), d)).astype(F)


def value(q, d):
    """The values that they stand for, in 64 bits"""
    return q.astype(np.float64) * d.astype(np.float64)[..., None]


class Paged8(Paged):
    """A paged cache of 8 bits: values and scales of k and v; rows that no sequence has hold NaN."""

    kind = "q8"

    def __init__(self, rng, lens, heads, dim, page, spare=2, k=None, v=None):
        self.heads, self.dim, self.page = heads, dim, page
        need = [-(-n // page) for n in lens]
        self.pages, self.ld = sum(need) + spare, max(need + [1]) + 1
        self.table = np.full((len(lens), self.ld), -7, np.int32)
        order, at = rng.permutation(self.pages).astype(np.int32), 0
        shape = (self.pages, heads, page, dim)
        self.q = {name: np.full(shape, 55, np.int8) for name in "kv"}
        self.d = {name: np.full(shape[:-1], np.nan, F) for name in "kv"}
        self.seq = {"k": [], "v": []}
        for s, n in enumerate(lens):
            self.table[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            pos = np.arange(n)
            for name, given in (("k", k), ("v", v)):
                q, d = quantise(rng.standard_normal((n, heads, dim)) if given is None else given[s])
                where = self.table[s, pos // page], slice(None), pos % page
                self.q[name][where], self.d[name][where] = q, d
                self.seq[name].append(value(q, d))
        self.seq_k, self.seq_v = self.seq["k"], self.seq["v"]

    def memory(self, name):
        return np.concatenate([self.q[name].view(np.uint8).reshape(-1), self.d[name].view(np.uint8).reshape(-1)])

    def struct(self, call, written=False):
        k, v = (call.out("c" + n, (self.memory(n).size,), np.uint8, self.memory(n)) if written else call.put(self.memory(n)) for n in "kv")
        m = call.m
        self.keep = m.Kv(k=k, v=v, type=m.TYPES["q8"], dim=self.dim, heads=self.heads, page=self.page, pages=self.pages, table=call.put(self.table), table_ld=self.ld)
        assert m.load().rt_kv_bytes(m.ctypes.byref(self.keep)) == self.memory("k").size
        return self.keep

    def held(self, call, name):
        """(values, scales) as the call left them"""
        raw, rows = call.get("c" + name), self.pages * self.heads * self.page
        return raw[:rows * self.dim].copy().view(np.int8).reshape(self.q[name].shape), raw[rows * self.dim:].copy().view(F).reshape(self.d[name].shape)


def paged(rng, kind, lens, heads, dim, page, **more):
    return Paged8(rng, lens, heads, dim, page, **more) if kind == "q8" else Paged(rng, kind, lens, heads, dim, page, **more)


def seen(p, window, sinks):
    """The positions that the token at position p sees"""
    pos = np.arange(p + 1)
    return pos if not window else pos[(pos > p - window) | (pos < sinks)]


def attn(q, k, v, scale, start, past, window=0, sinks=0, gate=None):
    """q [t hq d]; k, v: per sequence [positions hk d] in 64 bits, a position that is not there as NaN: (o, a bound on its F32 error).

    The bound is mix_ref.attn's, of F32 sums, and for queries that are held in 24 bits of their row's largest element half
    such a step, U max|q|, times each |k|."""
    t, hq, d = q.shape
    o, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for s in range(len(past)):
        for i in range(start[s], start[s + 1]):
            p = past[s] + i - start[s]
            if p < 0:
                o[i] = 0.0
                continue
            at = seen(p, window, sinks)
            if at[-1] >= len(k[s]):
                continue  # behind the table: NaN
            for h in range(hq):
                kh = h // (hq // k[s].shape[1])
                kk, vv, qq = k[s][at, kh], v[s][at, kh], q[i, h].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    x = scale * (kk @ qq)
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    o[i, h] = w @ vv
                    ds = U * abs(scale) * ((2 * np.sqrt(d) + 8) * (np.abs(kk) @ np.abs(qq)).max() + 2 * np.abs(qq).max() * np.abs(kk).sum(1).max())
                    tol[i, h] = (2 * ds + U * (2 * np.sqrt(len(at)) + 16)) * (w @ np.abs(vv))
    if gate is not None:
        g = ref.sigmoid(gate.astype(np.float64))
        o, tol = o * g, tol * g + 4 * U * np.abs(o * g)
    return o, tol + 2.0 ** -140
