"""The paged cache, its appends with rotation, attention and acceptance in numpy and 64 bits, from
their definitions."""
import math

import numpy as np

NONE = -1  # an entry of the table without a page


def stored(x, fmt):
    """float32 values as a cache of this format holds them, in float32: one rounding to nearest, ties
    to even (an fp16 overflow is an infinity)."""
    x = np.asarray(x, np.float32)
    if fmt == "f32":
        return x.copy()
    if fmt == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7fff + ((b >> 16) & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r).astype(np.float32)


def words(x, fmt):
    """Values that a cache of this format can hold as its array's elements."""
    if fmt == "f32":
        return np.asarray(x, np.float32)
    if fmt == "f16":
        with np.errstate(over="ignore"):
            return np.asarray(x, np.float32).astype(np.float16).view(np.uint16)
    return (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def values(w, fmt):
    """The other way round, in float32."""
    if fmt == "f32":
        return w.view(np.float32)
    if fmt == "f16":
        return w.view(np.float16).astype(np.float32)
    return (w.astype(np.uint32) << 16).view(np.float32)


def turned(x, positions, inv_freq, interleaved):
    """Rows x [n][heads][d] (float32) turned by position * inv_freq, in 64 bits."""
    half = len(inv_freq)
    y = x.astype(np.float64)
    a = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved \
        else (slice(0, half), slice(half, 2 * half))
    x0, x1 = y[..., i].copy(), y[..., j].copy()
    y[..., i], y[..., j] = x0 * c - x1 * s, x1 * c + x0 * s
    return y


def turned_bound(x, inv_freq, interleaved):
    """How far fp32 work may be from turned(): cos and sin are within 2^-22 (the angle is reduced in
    64 bits and rounded once, the series adds under four roundings), and the two products and their
    sum add three roundings more of at most |x0| + |x1| in size."""
    half = len(inv_freq)
    y = np.zeros(x.shape)
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved \
        else (slice(0, half), slice(half, 2 * half))
    size = np.abs(x[..., i].astype(np.float64)) + np.abs(x[..., j].astype(np.float64))
    y[..., i] = y[..., j] = size * (2.0 ** -22 + 3 * 2.0 ** -24)
    return y


STEP = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a unit in the last place, relative


def depths(parents, count):
    """Depths and paths (with the row itself) of a tree's rows."""
    path = []
    for i in range(count):
        p = parents[i]
        path.append((path[p] if 0 <= p < i else []) + [i])
    return [len(p) - 1 for p in path], path


def sight(ln, count, n_tokens, there, window=0, prefix=0, first=None, parents=None):
    """Which tokens each row sees [count][ln], and |difference of positions|."""
    base = ln - count
    t, place = np.arange(ln), base + np.arange(count)
    pos_q, pos_k, kin = place, t, t[None] <= place[:, None]
    if parents is not None:
        deep, path = depths(parents, count)
        pos_q, pos_k = base + np.array(deep, int), t.copy()
        kin = np.repeat((t < base)[None], count, 0)
        for i, p in enumerate(path):
            for j in p:
                if base + j >= 0:
                    kin[i, base + j] = True
                    pos_k[base + j] = base + deep[j]
    far = pos_q[:, None] - pos_k[None]
    sees = kin & ((far < window) if window else True)
    early = (t < prefix)[None] & (kin | (t < base)[None] if parents is not None else True)
    sees = sees | early
    if first is not None:
        sees = sees & (t[None] >= np.asarray(first)[:count, None])
    return sees & there[None, :ln] & (place >= 0)[:, None], np.abs(far)


class RefPaged:
    """Values by sequence and place; pages are the device's affair (there: tokens with a page)."""

    def __init__(self, n_seqs, kv, d, cap, fmt):
        self.fmt, self.shape = fmt, (n_seqs, kv, cap, d)
        self.k = np.zeros(self.shape, np.float32)
        self.v = np.zeros(self.shape, np.float32)
        self.there = np.ones((n_seqs, cap), bool)
        self.lens = [0] * n_seqs

    def attend(self, q, counts, scale, cap=0.0, slopes=None, window=0, prefix=None, first=None,
               parents=None):
        """out [s][n][heads][d], lse [s][heads][n] and the errors that fp32 work may leave.

        A score is a sum of d products whose operands are off by 2^-22 at most (q is rounded once
        with the scale and taken in pieces) and the roundings of the sum, d of 2^-24; capping
        shrinks those and adds under 8 roundings of the capped score, the bias two of its own, and
        the way to the exponent under 8 of the score.  A weight adds under 64 roundings of its
        value (exp2, pieces, sums over tokens, the division); in pieces of fp16 it is off by up to
        2^-37 of the row's largest as well."""
        s_, n, heads, d = q.shape
        group = heads // self.shape[1]
        out, lse = np.zeros(q.shape), np.full((s_, heads, n), -np.inf)
        tol, lse_tol = np.zeros(q.shape), np.zeros((s_, heads, n))
        u = 2.0 ** -24
        for s in range(s_):
            ln, c = self.lens[s], counts[s]
            if not c or not ln:
                continue
            sees, far = sight(ln, c, self.shape[2], self.there[s], window,
                              prefix[s] if prefix is not None else 0,
                              first[s] if first is not None else None,
                              parents[s] if parents is not None else None)
            some = sees.any(1)
            for h in range(heads):
                keys = np.where(self.there[s, :ln, None], self.k[s, h // group, :ln], 0).astype(np.float64)
                vals = np.where(self.there[s, :ln, None], self.v[s, h // group, :ln], 0).astype(np.float64)
                qs = q[s, :c, h].astype(np.float64) * scale
                x = qs @ keys.T
                e = (np.abs(qs) @ np.abs(keys).T) * (2.0 ** -22 + (d + 8) * u)
                if cap:
                    x = cap * np.tanh(x / cap)
                    e = e + 8 * u * np.abs(x)
                if slopes is not None:
                    bias = float(slopes[h]) * far
                    x = x - bias
                    e = e + 4 * u * np.abs(bias)
                e = e + 8 * u * np.abs(x) + (64 + 16) * u
                x = np.where(sees, x, -np.inf)
                m = np.where(some, x.max(1), 0.0)
                p = np.where(sees, np.exp(x - m[:, None]), 0.0)
                z = np.where(some, p.sum(1), 1.0)
                o = p @ vals / z[:, None]
                out[s, :c, h] = o
                pe = np.where(sees, p * e, 0)
                lost = 2.0 ** -37 * (sees @ np.abs(vals))
                tol[s, :c, h] = (pe @ np.abs(vals) + lost) / z[:, None] \
                    + np.abs(o) * (pe.sum(1) / z)[:, None]
                with np.errstate(divide="ignore"):
                    lse[s, h, :c] = np.where(some, m + np.log(z), -np.inf)
                lse_tol[s, h, :c] = np.where(some, pe.sum(1) / z + 2.0 ** -22 * (1 + np.abs(m + np.log(z))), 0)
        return out, lse, tol, lse_tol


def accept(parents, tokens, choices, ln, count):
    """path, next id and length of one sequence."""
    if count < 1 or count > ln:
        return [], -1, ln
    path, node = [], 0
    while node is not None:
        path.append(node)
        node = next((j for j in range(node + 1, count)
                     if parents[j] == node and tokens[j] == choices[node]), None)
    return path, int(choices[path[-1]]), ln - count + len(path)
