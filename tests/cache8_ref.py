"""The 8-bit cache, its attention, accounts and eviction, and token log probabilities in numpy and
64 bits, from their definitions."""
import math

import numpy as np

CODE_MAX = {"i8": 127.0, "e4m3": 448.0}
FLOOR = 2.0 ** -60


def e4m3_values():
    """The 127 values of a positive e4m3 code, in code order."""
    v = []
    for b in range(127):
        e, m = b >> 3, b & 7
        v.append((m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return np.array(v)


_E4 = e4m3_values()
_E4_MID = (_E4[1:] + _E4[:-1]) / 2


def encode(y, fmt):
    """Codes (bytes) of quotients y in 64 bits: the nearest, ties to the even code."""
    if fmt == "i8":
        return np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    a = np.abs(y)
    i = np.searchsorted(_E4_MID, a, side="left")  # up to a middle: the lower neighbour
    tie = (i < len(_E4_MID)) & (a == _E4_MID[np.minimum(i, len(_E4_MID) - 1)])
    i = i + (tie & (i % 2 == 1))
    return (i | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def whole(codes, fmt):
    """What codes stand for before the scale, as float32."""
    if fmt == "i8":
        return codes.view(np.int8).astype(np.float32)
    c = codes.astype(np.int64)
    return (np.where(c >= 128, -1.0, 1.0) * np.append(_E4, np.nan)[c & 127]).astype(np.float32)


def scale_of(x, fmt):
    """A block's scale, one rounding; NaN where something is not finite."""
    if not np.isfinite(x).all():
        return np.float32(np.nan)
    top = float(np.abs(x).max()) if x.size else 0.0
    return np.maximum(np.float32(top / CODE_MAX[fmt]), np.float32(FLOOR))


class RefCache:
    def __init__(self, n_seqs, kv, d, cap, block, fmt):
        self.shape, self.block, self.fmt = (n_seqs, kv, cap, d), block, fmt
        self.codes = {t: np.zeros(self.shape, np.uint8) for t in "kv"}
        self.scales = {t: np.zeros((n_seqs, kv, cap // block), np.float32) for t in "kv"}
        self.lens = [0] * n_seqs

    def _put(self, t, s, h, a, x):
        """Rows x (float32) as tokens a.. of a head."""
        end, B, fmt = a + len(x), self.block, self.fmt
        for b in range(a // B, -(-end // B)):
            lo, hi, t0 = max(a, b * B), min(end, (b + 1) * B), b * B
            if lo >= hi:
                continue
            codes, scales = self.codes[t][s, h], self.scales[t][s, h]
            rows, now, was = x[lo - a:hi - a], scale_of(x[lo - a:hi - a], fmt), scales[b]
            if lo > t0:
                now = np.float32(np.nan) if np.isnan(was) or np.isnan(now) else max(now, was)
                if now > was:
                    old = whole(codes[t0:lo], fmt) * was
                    codes[t0:lo] = encode(old.astype(np.float64) / np.float64(now), fmt)
            scales[b] = now
            codes[lo:hi] = 0 if np.isnan(now) else encode(
                rows.astype(np.float64) / np.float64(now), fmt)

    def append(self, k, v, lens, counts):
        """k, v [n_seqs][n][kv][d]; lens: tokens held afterwards."""
        self.lens = list(lens)
        for s, (ln, c) in enumerate(zip(lens, counts)):
            skip = max(0, c - ln)
            for h in range(self.shape[1]):
                self._put("k", s, h, ln - c + skip, k[s, skip:c, h])
                self._put("v", s, h, ln - c + skip, v[s, skip:c, h])

    def values(self, t, s, h, n=None):
        """The tokens a head holds, float32 [n, d]."""
        n = self.lens[s] if n is None else n
        each = self.scales[t][s, h][np.arange(n) // self.block]
        return whole(self.codes[t][s, h, :n], self.fmt) * each[:, None]

    def read(self, t, n):
        out = np.zeros((*self.shape[:2], n, self.shape[3]), np.float32)
        for s, ln in enumerate(self.lens):
            m = min(n, ln)
            for h in range(self.shape[1]):
                if m:
                    out[s, h, n - m:] = self.values(t, s, h)[ln - m:]
        return out

    def v_layout(self):
        s, kv, cap, d = self.shape
        return self.codes["v"].reshape(s, kv, cap // 64, 64, d).transpose(0, 1, 2, 4, 3).copy()

    def evict(self, weights, keep, recent, dst):
        kept = np.full((*self.shape[:2], keep), -1, np.int32)
        acc = np.zeros((*self.shape[:2], dst.shape[2]), np.float32)
        dst.lens = [min(ln, keep) for ln in self.lens]
        for s, ln in enumerate(self.lens):
            for h in range(self.shape[1]):
                w = weights[s, h, :ln].astype(np.float64)
                ids = np.arange(ln)
                if ln > keep:
                    old = w[:ln - recent]
                    key = np.where(np.isnan(old), -np.inf, old)
                    # larger first, NaN behind minus infinity, then the lower place
                    order = np.lexsort((np.arange(len(old)), np.isnan(old), -key))
                    ids = np.sort(np.concatenate([order[:keep - recent],
                                                  np.arange(ln - recent, ln)]))
                kept[s, h, :len(ids)] = ids
                acc[s, h, :len(ids)] = weights[s, h, ids]
                for t in "kv":
                    dst._put(t, s, h, 0, self.values(t, s, h)[ids])
        return kept, acc


def attend(ref, q, counts, scale, acc=None, lse_in=None):
    """out [s][n][heads][d], lse [s][heads][n], and for each output an estimate of the error that
    fp32 work may leave: see `bound` below.  With lse_in: the accounts instead."""
    s_, n, heads, d = q.shape
    kv = ref.shape[1]
    group = heads // kv
    out, lse = np.zeros(q.shape), np.full((s_, heads, n), -np.inf)
    tol, lse_tol = np.zeros(q.shape), np.zeros((s_, heads, n))
    got = None if lse_in is None else np.zeros((s_, kv, ref.shape[2]))
    got_tol = None if lse_in is None else np.zeros(got.shape)
    for s, (ln, c) in enumerate(zip(ref.lens, counts)):
        for h in range(kv):
            keys = ref.values("k", s, h).astype(np.float64)
            vals = ref.values("v", s, h).astype(np.float64)
            for i in range(c):
                sees = max(0, ln - c + i + 1)
                if sees == 0:
                    continue
                for j in range(h * group, (h + 1) * group):
                    x = keys[:sees] @ (q[s, i, j].astype(np.float64) * scale)
                    size = np.abs(keys[:sees]) @ np.abs(q[s, i, j].astype(np.float64) * scale)
                    e = bound(size, d)
                    if lse_in is not None:
                        w = np.exp(x - lse_in[s, j, i])
                        got[s, h, :sees] += w
                        got_tol[s, h, :sees] += w * (e + 2.0 ** -22 * (1 + abs(lse_in[s, j, i])))
                        continue
                    m = x.max()
                    p = np.exp(x - m)
                    z = p.sum()
                    out[s, i, j] = p @ vals[:sees] / z
                    lse[s, j, i] = m + math.log(z)
                    rel = np.max(e)
                    tol[s, i, j] = 2 * rel * (p @ np.abs(vals[:sees])) / z
                    lse_tol[s, j, i] = rel + 2.0 ** -22 * (1 + abs(lse[s, j, i]))
    if lse_in is not None:
        return got, got_tol
    return out, lse, tol, lse_tol


def bound(size, d):
    """Relative error of a weight exp(s - m) from fp32 work, `size` = sum |q_d k_d| scale.

    A score is a sum of d products whose operands are off by 2^-22 (q in two fp16 pieces of 11
    bits, q times the scale rounded once) plus the roundings of the sum, d of 2^-24 at most; its
    scaling, the log of V's scale and the difference with the maximum add roundings of the score's
    own size, under 8 in all.  The weight itself (exp2, the pieces, the sums over tokens, the
    division) adds under 64 roundings of its value."""
    return size * (2.0 ** -22 + d * 2.0 ** -24 + 8 * 2.0 ** -24) + (64 + 16) * 2.0 ** -24


def logprobs(x, targets, top):
    """x float32 [rows][vocab]: logprob, entropy, ids, their log probabilities."""
    x = x.astype(np.float64)
    rows, vocab = x.shape
    lp, ent = np.full(rows, np.nan), np.full(rows, np.nan)
    ids, tops = np.zeros((rows, top), np.int32), np.full((rows, top), np.nan)
    for r in range(rows):
        key = np.where(np.isnan(x[r]), -np.inf, x[r])
        ids[r] = np.lexsort((np.arange(vocab), np.isnan(x[r]), -key))[:top]
        if np.isnan(x[r]).any() or (x[r] == np.inf).any() or (x[r] == -np.inf).all():
            continue
        m = x[r].max()
        e = np.exp(x[r] - m)
        z = e.sum()
        d = np.where(e > 0, x[r] - m, 0.0)
        t = targets[r]
        lp[r] = x[r, t] - m - math.log(z) if 0 <= t < vocab else -np.inf
        ent[r] = math.log(z) - (e * d).sum() / z
        tops[r] = x[r, ids[r]] - m - math.log(z)
    return lp, ent, ids, tops
