"""The 8-bit cache on the GPU against tests/cache8_ref.py.

Codes, scales and what eviction keeps are compared bit for bit; attention and accounts within the
bounds that cache8_ref.bound derives from the operations' roundings."""
import ctypes as C

import numpy as np
import pytest

import cache8_ref as R
from spirv_inference_amd import Cache8, Context, DeviceTensor, ShpError
from spirv_inference_amd._lib import check, lib

pytestmark = pytest.mark.gpu

SENTINEL = 0xFF  # a NaN code of e4m3: what lies behind a length must not be used


class Pair:
    """A device cache, filled with codes and scales that would show, and the reference."""

    def __init__(self, ctx, n_seqs, kv, d, cap, block, fmt):
        self.ctx, self.dims = ctx, (n_seqs, kv, d, cap)
        self.ref = R.RefCache(n_seqs, kv, d, cap, block, fmt)
        self.dev = Cache8(ctx, n_seqs, kv, d, cap, block, fmt)
        for t in (self.dev.k, self.dev.v):
            t.upload(np.full(t.n, SENTINEL, np.uint8))
        for t in (self.dev.k_scale, self.dev.v_scale):
            t.upload(np.full(t.n, np.nan, np.float32))
        self.temp = []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for t in self.temp:
            t.free()
        self.dev.close()

    def up(self, a, dtype=np.float32):
        t = self.ctx.tensor(np.ascontiguousarray(a), dtype)
        self.temp.append(t)
        return t

    def new(self, n, dtype=np.float32, fill=None):
        return self.up(np.full(n, 0 if fill is None else fill, dtype), dtype)

    def append(self, k, v, lens, counts=None):
        n = k.shape[1]
        self.dev.set_lengths(lens)
        c = [n] * len(lens) if counts is None else counts
        self.dev.append(self.up(k), self.up(v), n,
                        counts=None if counts is None else self.up(counts, np.int32))
        self.ref.append(k, v, lens, c)

    def check_content(self):
        s_, kv, d, cap = self.dims
        n = max(max(self.ref.lens), 1)
        ko, vo = self.new(s_ * kv * n * d, fill=7), self.new(s_ * kv * n * d, fill=7)
        self.dev.read(n, ko, vo)
        self.ctx.sync()
        for t, o in (("k", ko), ("v", vo)):
            got, want = o.download().reshape(s_, kv, n, d), self.ref.read(t, n)
            np.testing.assert_array_equal(got, want, err_msg=t)
        # the bytes, and those behind the lengths as they were
        k = self.dev.k.download().reshape(s_, kv, cap, d)
        v = self.dev.v.download().reshape(s_, kv, cap // 64, d, 64).transpose(0, 1, 2, 4, 3) \
            .reshape(s_, kv, cap, d)
        for s, ln in enumerate(self.ref.lens):
            for t, got in (("k", k), ("v", v)):
                want, have = self.ref.codes[t][s, :, :ln], got[s, :, :ln]
                zero = (have & 127 == 0) & (want & 127 == 0)  # the sign of a zero is nobody's
                assert (zero | (have == want)).all() if self.ref.fmt == "e4m3" \
                    else (have == want).all()
                assert (got[s, :, ln:] == SENTINEL).all(), f"{t}: bytes behind sequence {s}"
        for t, dev in (("k", self.dev.k_scale), ("v", self.dev.v_scale)):
            got = dev.download().reshape(self.ref.scales[t].shape)
            for s, ln in enumerate(self.ref.lens):
                b = -(-ln // self.ref.block)
                np.testing.assert_array_equal(got[s, :, :b], self.ref.scales[t][s, :, :b])
                assert np.isnan(got[s, :, b:]).all()

    def attend(self, q, counts=None, scale=None, lse=True):
        s_, n, heads, d = q.shape
        out, l = self.new(q.size, fill=-3), self.new(s_ * heads * n, fill=-3)
        self.dev.attend(self.up(q), out, heads, n, lse=l if lse else None, scale=scale,
                        counts=None if counts is None else self.up(counts, np.int32))
        self.ctx.sync()
        return out.download().reshape(q.shape), l.download().reshape(s_, heads, n), l

    def check_attend(self, q, counts=None, scale=None):
        s_, n, heads, d = q.shape
        out, lse, _ = self.attend(q, counts, scale)
        c = [n] * s_ if counts is None else [max(0, min(n, x)) for x in counts]
        want, wl, tol, ltol = R.attend(self.ref, q, c, d ** -0.5 if scale is None else scale)
        for s in range(s_):
            assert (out[s, c[s]:] == -3).all() and (lse[s, :, c[s]:] == -3).all(), "rows behind"
            o, w = out[s, :c[s]].astype(np.float64), want[s, :c[s]]
            assert np.isfinite(o).all()
            assert (np.abs(o - w) <= tol[s, :c[s]] + 1e-30).all(), \
                np.max(np.abs(o - w) - tol[s, :c[s]])
            g, wg = lse[s, :, :c[s]].astype(np.float64), wl[s, :, :c[s]]
            np.testing.assert_array_equal(np.isinf(g), np.isinf(wg))
            f = np.isfinite(wg)
            assert (np.abs(g[f] - wg[f]) <= ltol[s, :, :c[s]][f]).all()
        return out, lse


def rows(rng, *shape, spread=0.0):
    x = rng.standard_normal(shape)
    return (x * np.exp(spread * rng.standard_normal(shape[:-1]))[..., None]).astype(np.float32)


def filled(ctx, rng, n_seqs, kv, d, cap, block, fmt, lens, spread=0.0):
    """A pair that holds lens[s] tokens, written by one ragged append."""
    p = Pair(ctx, n_seqs, kv, d, cap, block, fmt)
    n = max(max(lens), 1)
    p.append(rows(rng, n_seqs, n, kv, d, spread=spread), rows(rng, n_seqs, n, kv, d, spread=spread),
             lens, lens)
    return p


# ---- append and read ------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("d,block", [(64, 16), (64, 128), (128, 32), (128, 64)])
def test_append_token_by_token_and_in_chunks(ctx, fmt, d, block):
    """Chunks of many lengths, ragged over the sequences, that begin and end inside blocks and
    tiles; scales grow on the way, so codes are rounded again."""
    rng = np.random.default_rng(1)
    with Pair(ctx, 3, 2, d, 384, block, fmt) as p:
        lens = [0, 0, 0]
        for step, n in enumerate([1, 1, 1, 5, 16, 1, 64, 63, 2, 1, 130, 1]):
            counts = [n, max(0, n - 1 - step % 3), n // 2]
            lens = [a + b for a, b in zip(lens, counts)]
            p.append(rows(rng, 3, n, 2, d, spread=1.0), rows(rng, 3, n, 2, d, spread=1.0), lens,
                     counts)
        p.check_content()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_append_to_the_last_slot_and_over_an_old_end(ctx, fmt):
    """A full cache, and a sequence that goes back to an earlier length and on from there."""
    rng = np.random.default_rng(2)
    with filled(ctx, rng, 2, 1, 64, 128, 64, fmt, [128, 128]) as p:
        p.check_content()
        p.append(rows(rng, 2, 3, 1, 64), rows(rng, 2, 3, 1, 64), [67, 34])
        np.testing.assert_array_equal(p.ref.lens, [67, 34])
        ko = p.new(2 * 67 * 64)
        p.dev.read(67, ko, None)
        ctx.sync()
        np.testing.assert_array_equal(ko.download().reshape(2, 1, 67, 64), p.ref.read("k", 67))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_append_rounds_the_exact_quotient(ctx, fmt):
    """Quotients at and next to the middle of two codes, in blocks whose scales are no powers of
    two: rounding the fp32 quotient again would send some the other way."""
    rng = np.random.default_rng(3)
    top = np.float32(R.CODE_MAX[fmt])
    n, d = 64, 64
    k = np.empty((1, n, 1, d), np.float32)
    for t in range(0, n, 16):
        scale = np.float32(rng.uniform(0.01, 0.02))
        amax = np.float32(scale * top)
        s = R.scale_of(np.array([amax]), fmt)
        vals = np.arange(0, 127) if fmt == "i8" else R.e4m3_values()
        mids = (vals[1:] + vals[:-1]) / 2
        x = (rng.choice(mids, (16, d)) * np.float64(s)).astype(np.float32)
        x = np.nextafter(x, np.where(rng.random(x.shape) < 0.5, np.inf, -np.inf).astype(np.float32)) \
            if t % 32 else x
        x = np.minimum(x, amax) * np.where(rng.random(x.shape) < 0.5, -1, 1).astype(np.float32)
        x[0, 0] = amax
        k[0, t:t + 16, 0] = x
    with Pair(ctx, 1, 1, d, 64, 16, fmt) as p:
        p.append(k, k[:, ::-1].copy(), [n])
        p.check_content()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_append_of_zeros_tiny_and_huge_values(ctx, fmt):
    x = np.zeros((1, 80, 1, 64), np.float32)
    x[0, 16:32] = np.float32(1e-44)                       # below the smallest scale
    x[0, 32:48] = np.linspace(-1e-18, 1e-18, 64)          # about it
    x[0, 48:64] = np.linspace(-3.4e38, 3.4e38, 64)        # the top of the range
    x[0, 64:80] = np.linspace(-1, 1, 64) * 2.0 ** -57
    with Pair(ctx, 1, 1, 64, 128, 16, fmt) as p:
        p.append(x, -x, [80])
        p.check_content()


def test_rows_of_tokens_before_the_first_are_dropped(ctx):
    rng = np.random.default_rng(5)
    with Pair(ctx, 3, 1, 64, 64, 16, "i8") as p:
        p.append(rows(rng, 3, 9, 1, 64), rows(rng, 3, 9, 1, 64), [4, 0, 9])
        p.check_content()


def test_lengths_and_counts_out_of_range_stay_in_bounds(ctx):
    """They count as the nearest length and count that can be."""
    rng = np.random.default_rng(6)
    k, v = rows(rng, 4, 3, 1, 64), rows(rng, 4, 3, 1, 64)
    with Pair(ctx, 4, 1, 64, 64, 16, "i8") as p:
        for t in (p.dev.k, p.dev.v, p.dev.k_scale, p.dev.v_scale):
            t.upload(np.zeros(t.n))  # sequence 1 claims tokens that nobody wrote
        p.dev.set_lengths([-5, 1 << 30, 3, 3])
        p.dev.append(p.up(k), p.up(v), 3, counts=p.up([3, 3, -1, 1 << 30], np.int32))
        p.ref.append(k, v, [0, 64, 3, 3], [3, 3, 0, 3])
        got = p.new(4 * 3 * 64)
        p.dev.read(3, got, None)
        ctx.sync()
        got, want = got.download().reshape(4, 1, 3, 64), p.ref.read("k", 3)
        for s in (0, 1, 3):
            np.testing.assert_array_equal(got[s], want[s])
        q = rows(rng, 4, 1, 2, 64)
        out, l, _ = p.attend(q)
        assert (out[0] == 0).all() and (l[0] == -np.inf).all()


def test_nothing_to_do(ctx):
    with Pair(ctx, 1, 1, 64, 64, 16, "i8") as p:
        t = p.new(64, fill=5)
        p.dev.append(t, t, 0)
        p.dev.read(0, t, t)
        p.dev.read(3, None, None)
        p.dev.attend(t, t, 1, 0)
        ctx.sync()
        assert (t.download() == 5).all()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_what_is_not_finite_spoils_its_own_block_only(ctx, fmt, bad):
    """Rows that see a token of the block get NaN, the rows before it what they would have got, and
    a block begun again is sound."""
    rng = np.random.default_rng(7)
    k, v = rows(rng, 1, 48, 1, 64), rows(rng, 1, 48, 1, 64)
    k[0, 20, 0, 3] = bad
    v[0, 40, 0, 5] = bad
    with Pair(ctx, 1, 1, 64, 64, 16, fmt) as p:
        p.append(k, v, [48])
        p.check_content()
        q = rows(rng, 1, 48, 2, 64)
        out, lse, _ = p.attend(q)
        clean = R.RefCache(1, 1, 64, 64, 16, fmt)
        clean.append(k[:, :16], v[:, :16], [16], [16])
        want, wl, tol, _ = R.attend(clean, q[:, :16], [16], 0.125)
        assert (np.abs(out[0, :16] - want[0]) <= tol[0] + 1e-30).all()
        assert np.isnan(out[0, 16:]).all()
        # one more token does not make it sound; beginning the blocks again does
        p.append(rows(rng, 1, 1, 1, 64), rows(rng, 1, 1, 1, 64), [21])
        assert np.isnan(p.dev.k_scale.download()[1])
        p.append(rows(rng, 1, 10, 1, 64), rows(rng, 1, 10, 1, 64), [26])
        p.check_attend(rows(rng, 1, 1, 2, 64))


# ---- attention ------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kv,group,n,block,lens", [
    (1, 1, 1, 16, [1, 2]),
    (2, 4, 1, 32, [63, 64]),
    (2, 8, 1, 64, [65, 300]),
    (1, 16, 1, 128, [700, 0]),
    (3, 5, 1, 16, [129, 17]),
    (2, 3, 7, 32, [90, 7]),          # 21 rows
    (1, 8, 5, 64, [200, 3]),         # 40 rows; a sequence shorter than its rows
    (2, 4, 33, 64, [33, 161]),       # 132 rows, a prompt from the start
    (1, 7, 64, 16, [500, 64])])      # 448 rows
def test_attention(ctx, fmt, d, kv, group, n, block, lens):
    rng = np.random.default_rng(11 + n)
    with filled(ctx, rng, 2, kv, d, 768, block, fmt, lens, spread=0.3) as p:
        p.check_attend(rows(rng, 2, n, kv * group, d))


# So many pairs of rows and tiles, by the capacity, that a workgroup takes 32 rows; their tokens in one
# share or several.
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("d,kv,group,n,counts,lens", [
    (64, 4, 4, 64, None, [70]),
    (64, 4, 4, 61, [59], [1500]),
    (128, 2, 4, 33, [33], [1234]),
    (128, 2, 3, 43, None, [40])])
def test_attention_of_many_rows_in_a_long_cache(ctx, fmt, d, kv, group, n, counts, lens):
    rng = np.random.default_rng(17 + n)
    with filled(ctx, rng, 1, kv, d, 65536, 32, fmt, lens, spread=0.3) as p:
        p.check_attend(rows(rng, 1, n, kv * group, d), counts=counts)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_attention_of_prompts_that_fill_the_gpu(ctx, fmt):
    rng = np.random.default_rng(16)
    with filled(ctx, rng, 5, 8, 128, 128, 64, fmt, [90, 128, 3, 85, 0]) as p:
        p.check_attend(rows(rng, 5, 90, 32, 128), counts=[90, 88, 90, 1, 7])


def test_attention_of_padded_rows(ctx):
    rng = np.random.default_rng(12)
    with filled(ctx, rng, 4, 2, 64, 256, 32, "e4m3", [100, 256, 5, 0]) as p:
        p.check_attend(rows(rng, 4, 6, 8, 64), counts=[6, 1, 0, 3])
        p.check_attend(rows(rng, 4, 40, 8, 64), counts=[40, 17, 2, 0])
        p.check_attend(rows(rng, 4, 2, 8, 64), counts=[9, -1, 2, 1])


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e-30])
def test_attention_scales(ctx, fmt, scale):
    """Uniform, reversed and nearly one-hot weights."""
    rng = np.random.default_rng(13)
    with filled(ctx, rng, 1, 1, 64, 256, 64, fmt, [200]) as p:
        p.check_attend(rows(rng, 1, 3, 4, 64), scale=scale)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_attention_where_scales_differ_by_many_orders(ctx, fmt):
    """Blocks from 2^-40 to 2^40: the tokens with small values have to come out as exactly as in a
    cache of their own."""
    rng = np.random.default_rng(14)
    k = np.zeros((1, 128, 1, 64), np.float32)
    v = rows(rng, 1, 128, 1, 64)
    k[0, :, 0, 0] = np.where(np.arange(128) // 16 % 2, 40, -40)  # every other block is not attended
    v *= np.where(np.arange(128) // 16 % 2, 2.0 ** -40, 2.0 ** 40)[None, :, None, None].astype(np.float32)
    v[0, 48:64] = 0.0  # a block of zeros that takes weight
    with Pair(ctx, 1, 1, 64, 128, 16, fmt) as p:
        p.append(k, v, [128])
        q = np.zeros((1, 2, 1, 64), np.float32)
        q[..., 0] = 30.0
        p.check_attend(q, scale=0.5)
        q[..., 0] = 1e-3
        p.check_attend(q, scale=0.5)


# Blocks of 16 tokens whose V is all zeros (the smallest scale, 2^-60) or 1e-12 beside blocks of very
# large V: in one tile, in the tiles of different wavefronts, in the shares of different workgroups.
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("huge", [1e24, 1e30, 3e38])
@pytest.mark.parametrize("small", [0.0, 1e-12])
@pytest.mark.parametrize("n,length,run", [(1, 32, 16), (1, 128, 64), (40, 320, 16), (1, 2000, 1024)])
def test_attention_weighs_tokens_whatever_their_values(ctx, fmt, d, huge, small, n, length, run):
    """Tokens of all magnitudes share the weight; how large a value is does not change its weight."""
    rng = np.random.default_rng(21)
    k, v = rows(rng, 1, length, 1, d), rng.uniform(-1, 1, (1, length, 1, d))
    v = v * np.where(np.arange(length) // run % 2, huge, small)[None, :, None, None]
    with Pair(ctx, 1, 1, d, -(-length // 128) * 128, 16, fmt) as p:
        p.append(k, v.astype(np.float32), [length])
        p.check_attend(rows(rng, 1, n, 2, d))
        p.check_attend(np.zeros((1, n, 2, d), np.float32))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("gap", [60.0, 80.0, 86.0])
@pytest.mark.parametrize("length,run", [(32, 16), (128, 64), (2000, 1024)])
def test_attention_of_large_values_with_little_weight(ctx, fmt, gap, length, run):
    """Weights of e^-60 to e^-86 on values of 1e36 beside weights of one on values of 0.01 and zero."""
    rng = np.random.default_rng(22)
    big = np.arange(length) // run % 2 == 1
    k = np.zeros((1, length, 1, 64), np.float32)
    k[0, big, 0, 0] = -1.0
    v = rng.uniform(0.5, 1, (1, length, 1, 64))
    v[0, ~big] *= 0.01
    v[0, big] *= 1e36
    v[0, :8] = 0.0
    with Pair(ctx, 1, 1, 64, -(-length // 128) * 128, 16, fmt) as p:
        p.append(k, v.astype(np.float32), [length])
        q = np.zeros((1, 1, 4, 64), np.float32)
        q[..., 0] = gap
        p.check_attend(q, scale=1.0)


def test_attention_of_zero_tiny_and_huge_queries(ctx):
    rng = np.random.default_rng(15)
    with filled(ctx, rng, 1, 1, 64, 128, 32, "i8", [100]) as p:
        q = rows(rng, 1, 4, 1, 64)
        q[0, 0] = 0.0
        q[0, 1] *= np.float32(1e-38)
        q[0, 2] *= np.float32(1e20)
        q[0, 3, 0, :32] *= np.float32(1e-9)  # small next to large
        out, _, _ = p.attend(q, scale=1.0)
        q2 = q.copy()
        q2[0, 2] = 1.0
        want, _, tol, _ = R.attend(p.ref, q2, [4], 1.0)
        for i in (0, 1, 3):
            assert (np.abs(out[0, i] - want[0, i]) <= tol[0, i]).all()
        best = np.argmax(p.ref.values("k", 0, 0)[:99].astype(np.float64) @ q[0, 2, 0])
        np.testing.assert_allclose(out[0, 2, 0], p.ref.values("v", 0, 0)[best], rtol=1e-6)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 40])
def test_attention_of_huge_queries_to_huge_keys_across_them(ctx, fmt, d, n):
    """q and K whose products would overflow, but of which none meets another: scores of zero."""
    rng = np.random.default_rng(24)
    k, q = np.zeros((1, 100, 1, d), np.float32), np.zeros((1, n, 2, d), np.float32)
    k[..., ::2], q[..., 1::2] = 1e30, 1e32
    with Pair(ctx, 1, 1, d, 128, 32, fmt) as p:
        p.append(k, rows(rng, 1, 100, 1, d), [100])
        _, lse = p.check_attend(q)
        t = p.up(lse)
        acc = p.new(128)
        p.dev.weights(p.up(q), t, None, acc, 2, n)
        ctx.sync()
        got = acc.download()[:100]
        want, tol = R.attend(p.ref, q, [n], d ** -0.5, lse_in=lse.astype(np.float64))
        assert (np.abs(got - want[0, 0, :100]) <= tol[0, 0, :100] + want[0, 0, :100] * (2 * n + 2) * 2.0 ** -24).all()


def test_a_row_that_is_not_finite_spoils_only_itself(ctx):
    rng = np.random.default_rng(16)
    with filled(ctx, rng, 1, 1, 64, 128, 32, "i8", [100]) as p:
        q = rows(rng, 1, 1, 8, 64)
        clean, _, _ = p.attend(q)
        q[0, 0, 3, 7] = np.nan
        q[0, 0, 5, 7] = np.inf
        out, _, _ = p.attend(q)
        for j in range(8):
            if j in (3, 5):
                assert np.isnan(out[0, 0, j]).all()
            else:
                np.testing.assert_array_equal(out[0, 0, j], clean[0, 0, j])


def test_strides(ctx):
    """Q, K and V inside one projection's rows, as a fused QKV product leaves them; the output with
    the heads outermost."""
    rng = np.random.default_rng(17)
    kv, heads, d, n = 2, 6, 64, 5
    w = (heads + 2 * kv) * d
    qkv = rng.standard_normal((2, n, w)).astype(np.float32)
    with Pair(ctx, 2, kv, d, 64, 16, "i8") as p:
        t = p.up(qkv)
        at = lambda o: DeviceTensor(ctx, t.n - o, ptr=t.ptr + 4 * o, owned=False)
        p.dev.set_lengths([n, n])
        st = (n * w, w, d)
        p.dev.append(at(heads * d), at((heads + kv) * d), n, k_strides=st, v_strides=st)
        q, k, v = (x.reshape(2, n, -1, d) for x in np.split(qkv, [heads * d, (heads + kv) * d], 2))
        p.ref.append(k, v, [n, n], [n, n])
        p.check_content()
        out = p.new(2 * heads * n * d)
        p.dev.attend(at(0), out, heads, n, q_strides=st, o_strides=(heads * n * d, d, n * d))
        ctx.sync()
        want, _, tol, _ = R.attend(p.ref, q, [n, n], d ** -0.5)
        got = out.download().reshape(2, heads, n, d).transpose(0, 2, 1, 3)
        assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("d,fmt", [(64, "i8"), (128, "e4m3")])
def test_attention_over_a_long_cache(ctx, d, fmt):
    """Tokens over many workgroups, with a length that no split divides."""
    rng = np.random.default_rng(18)
    with filled(ctx, rng, 1, 2, d, 16384, 64, fmt, [16001]) as p:
        p.check_attend(rows(rng, 1, 2, 8, d))


def test_offsets_past_32_bits(ctx):
    """The last head of a cache of more than 4 GiB."""
    rng = np.random.default_rng(19)
    cap, kv, d, n = 1 << 22, 9, 128, 70
    k, v = rows(rng, 1, n, 1, d), rows(rng, 1, n, 1, d)
    ref = R.RefCache(1, 1, d, 128, 32, "i8")
    ref.append(k, v, [n], [n])
    with Cache8(ctx, 1, kv, d, cap, 32, "i8") as c:
        c.set_lengths([n])
        t = [ctx.tensor(np.repeat(x, kv, 2)) for x in (k, v)]
        c.append(*t, n)
        ko, vo, out = (ctx.empty(kv * n * d) for _ in range(3))
        c.read(n, ko, vo)
        q = rows(rng, 1, 1, kv, d)
        tq = ctx.tensor(q)
        c.attend(tq, out, kv, 1)
        ctx.sync()
        for name, o in (("k", ko), ("v", vo)):
            got = o.download().reshape(kv, n, d)
            np.testing.assert_array_equal(got, np.broadcast_to(ref.read(name, n)[0], got.shape))
        got = out.download()[:kv * d].reshape(kv, d)
        for j in range(kv):
            want, _, tol, _ = R.attend(ref, q[:, :, j:j + 1], [1], d ** -0.5)
            assert (np.abs(got[j] - want[0, 0, 0]) <= tol[0, 0, 0]).all()
        for x in (*t, ko, vo, out, tq):
            x.free()


def test_results_do_not_change_from_call_to_call(ctx):
    rng = np.random.default_rng(20)
    with filled(ctx, rng, 2, 2, 128, 4096, 64, "i8", [4000, 1234]) as p:
        q = rows(rng, 2, 3, 8, 128)
        first = p.attend(q)[:2]
        for _ in range(3):
            for a, b in zip(first, p.attend(q)[:2]):
                np.testing.assert_array_equal(a, b)


# ---- accounts and eviction ------------------------------------------------------------------

def check_accounts(ctx, fmt, d, kv, group, n, counts, lens, cap):
    rng = np.random.default_rng(30 + n)
    with filled(ctx, rng, 2, kv, d, cap, 16, fmt, lens) as p:
        q = rows(rng, 2, n, kv * group, d)
        tq, tc = p.up(q), None if counts is None else p.up(counts, np.int32)
        out, lse = p.new(q.size), p.new(2 * kv * group * n)
        p.dev.attend(tq, out, kv * group, n, counts=tc, lse=lse)
        start = rng.uniform(0, 2, (2, kv, cap)).astype(np.float32)
        acc, res = p.up(start), p.new(start.size, fill=-3)
        p.dev.weights(tq, lse, acc, res, kv * group, n, counts=tc)
        p.dev.weights(tq, lse, acc, acc, kv * group, n, counts=tc)   # in place
        only = p.new(start.size, fill=-3)
        p.dev.weights(tq, lse, None, only, kv * group, n, counts=tc)
        ctx.sync()
        c = [n, n] if counts is None else counts
        l64 = lse.download().reshape(2, kv * group, n).astype(np.float64)
        want, tol = R.attend(p.ref, q, c, d ** -0.5, lse_in=l64)
        got, place, bare = (t.download().reshape(start.shape) for t in (res, acc, only))
        for s, ln in enumerate(lens):
            # one rounding of the sum of all rows' weights and of what was there
            t = tol[s, :, :ln] + (want[s, :, :ln] + start[s, :, :ln]) * (c[s] * group + 2) * 2.0 ** -24
            assert (np.abs(got[s, :, :ln] - want[s, :, :ln] - start[s, :, :ln]) <= t).all()
            assert (np.abs(bare[s, :, :ln] - want[s, :, :ln]) <= t).all()
            assert (got[s, :, ln:] == -3).all() and (bare[s, :, ln:] == -3).all()
            np.testing.assert_array_equal(place[s, :, ln:], start[s, :, ln:])
            np.testing.assert_array_equal(place[s, :, :ln], got[s, :, :ln])


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("d,kv,group,n,counts,lens", [
    (64, 2, 8, 1, None, [300, 64]),
    (64, 1, 3, 50, [50, 11], [130, 11]),
    (128, 2, 4, 9, [0, 9], [77, 5]),
    (128, 1, 1, 1, None, [1, 0])])
def test_accounts(ctx, fmt, d, kv, group, n, counts, lens):
    check_accounts(ctx, fmt, d, kv, group, n, counts, lens, 320)


# a capacity of which so many tiles could be held that a wavefront takes 64 rows
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("d,n,counts,lens", [
    (64, 67, [67, 30], [300, 65]), (128, 67, [67, 30], [300, 65]), (128, 100, None, [64, 129])])
def test_accounts_of_many_rows_in_a_long_cache(ctx, fmt, d, n, counts, lens):
    check_accounts(ctx, fmt, d, 2, 3, n, counts, lens, 65536)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("counts", [[0, 1], [1, 0], [0, 0]])
def test_accounts_of_a_decode_step_with_idle_slots(ctx, fmt, counts):
    """One row group a head: where a sequence has no row, its accounts are copied."""
    check_accounts(ctx, fmt, 64, 2, 4, 1, counts, [200, 77], 320)


def test_accounts_of_no_rows_are_copied(ctx):
    rng = np.random.default_rng(31)
    with filled(ctx, rng, 2, 1, 64, 128, 32, "i8", [100, 0]) as p:
        start = rng.uniform(0, 2, (2, 1, 128)).astype(np.float32)
        acc, res, bare, t = p.up(start), p.new(256, fill=-3), p.new(256, fill=-3), p.new(64)
        p.dev.weights(t, t, acc, res, 2, 0)
        p.dev.weights(t, t, acc, acc, 2, 0)
        p.dev.weights(t, t, None, bare, 2, 0)
        ctx.sync()
        np.testing.assert_array_equal(acc.download(), start.reshape(-1))
        for got, want in ((res, start), (bare, 0 * start)):
            want[0, :, 100:], want[1] = -3, -3
            np.testing.assert_array_equal(got.download().reshape(start.shape), want)


@pytest.mark.parametrize("d,fmt", [(64, "i8"), (128, "e4m3")])
def test_accounts_of_row_groups_of_several_chunks(d, fmt):
    """So many rows over so large a cache that the row groups whose sums find room each take several
    chunks of 64 rows, the later ones adding to what the earlier left."""
    kv, group, n, cap, counts, lens = 4, 3, 350, 131072, [350, 30], [400, 65]
    one = 2 * kv * cap * 4  # bytes of a group's sums
    with Context("any") as own:
        check_accounts(own, fmt, d, kv, group, n, counts, lens, cap)
        ptr, size = C.c_void_p(), C.c_uint64()
        check(lib().shp_workspace_info(own.handle, C.byref(ptr), C.byref(size)), "workspace_info")
        # several groups, but fewer than there are chunks
        assert 2 * one <= size.value < n * group // 64 * one


def evict_both(p, q, weights, keep, recent):
    s_, kv, d, cap = q.dims
    kept, acc = p.new(s_ * kv * keep, np.int32, 99), p.new(s_ * kv * cap, fill=-3)
    p.dev.evict(q.dev, p.up(weights), keep, recent, kept, acc)
    p.ctx.sync()
    want, wacc = p.ref.evict(weights, keep, recent, q.ref)
    np.testing.assert_array_equal(kept.download().reshape(want.shape), want)
    np.testing.assert_array_equal(acc.download().reshape(wacc.shape), wacc)
    np.testing.assert_array_equal(q.dev.lengths.download(), q.ref.lens)
    q.check_content()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("d,block,lens,keep,recent", [
    (64, 16, [200, 100, 99], 100, 20),
    (64, 64, [500, 65, 0], 64, 0),
    (128, 32, [300, 301, 1], 37, 37),     # only the newest
    (128, 128, [512, 129, 128], 128, 1),
    (64, 16, [70, 2, 1], 1, 0),
    (64, 32, [450, 512, 448], 449, 448)])
def test_eviction(ctx, fmt, d, block, lens, keep, recent):
    rng = np.random.default_rng(keep)
    w = rng.exponential(size=(3, 2, 512)).astype(np.float32)
    with filled(ctx, rng, 3, 2, d, 512, block, fmt, lens, spread=0.5) as p, \
            Pair(ctx, 3, 2, d, -(-keep // 128) * 128, block, fmt) as q:
        evict_both(p, q, w, keep, recent)


@pytest.mark.parametrize("kind", ["equal", "few", "signs", "strange"])
def test_eviction_orders_weights(ctx, kind):
    """Equal weights: the oldest stay. Zeros of both signs are equal, NaN is below everything."""
    rng = np.random.default_rng(40)
    w = np.ones((1, 2, 2112), np.float32)
    if kind == "few":
        w = rng.integers(0, 3, w.shape).astype(np.float32)
    elif kind == "signs":
        w = rng.choice([-1.0, -0.0, 0.0, 1e-45, -1e-45], w.shape).astype(np.float32)
    elif kind == "strange":
        w = rng.choice([np.nan, -np.nan, -np.inf, np.inf, 0.0, -3.4e38], w.shape).astype(np.float32)
    with filled(ctx, rng, 1, 2, 64, 2112, 64, "i8", [2100]) as p, \
            Pair(ctx, 1, 2, 64, 1536, 64, "i8") as q:
        for keep, recent in ((700, 5), (1500, 0), (6, 5)):
            evict_both(p, q, w, keep, recent)
            for t in (q.dev.k, q.dev.v):
                t.upload(np.full(t.n, SENTINEL, np.uint8))
            for t in (q.dev.k_scale, q.dev.v_scale):
                t.upload(np.full(t.n, np.nan, np.float32))
            q.ref = R.RefCache(1, 2, 64, 1536, 64, "i8")


@pytest.mark.parametrize("n", [1000, 1030, 8200, 8230, 20000, 32800, 40000])
def test_eviction_from_long_sequences(ctx, n):
    """Weights by the thousand: those a workgroup holds one, 8 or 32 a thread, and those it reads
    again for each digit; with plateaus, so that a digit's count decides."""
    rng = np.random.default_rng(n)
    cap = -(-n // 64) * 64
    w = np.round(rng.exponential(size=(1, 1, cap)) * 40).astype(np.float32) / 40
    keep = 500
    with filled(ctx, rng, 1, 1, 64, cap, 64, "i8", [n]) as p, \
            Pair(ctx, 1, 1, 64, 512, 64, "i8") as q:
        evict_both(p, q, w, keep, 7)


def test_eviction_of_a_spoiled_block_spoils_where_its_tokens_go(ctx):
    rng = np.random.default_rng(41)
    k, v = rows(rng, 1, 100, 1, 64), rows(rng, 1, 100, 1, 64)
    k[0, 50, 0, 0] = np.nan
    with Pair(ctx, 1, 1, 64, 128, 16, "i8") as p, Pair(ctx, 1, 1, 64, 64, 16, "i8") as q:
        p.append(k, v, [100])
        evict_both(p, q, np.arange(128, dtype=np.float32)[None, None], 60, 0)


# ---- all together, streams and graphs --------------------------------------------------------

def test_a_serving_loop_within_a_budget(ctx):
    """Prompts of two sequences, their accounts, eviction to a budget, decode steps until the
    budget is reached again, and eviction back into the first cache."""
    rng = np.random.default_rng(50)
    kv, group, d, block, fmt = 2, 4, 64, 32, "i8"
    heads, keep, recent = kv * group, 96, 16
    with Pair(ctx, 2, kv, d, 256, block, fmt) as a, Pair(ctx, 2, kv, d, 128, block, fmt) as b:
        def attend_and_account(p, acc, want_acc, q, counts):
            tq, n = p.up(q), q.shape[1]
            tc = None if counts is None else p.up(counts, np.int32)
            out, lse = p.new(q.size), p.new(2 * heads * n)
            p.dev.attend(tq, out, heads, n, counts=tc, lse=lse)
            p.dev.weights(tq, lse, acc, acc, heads, n, counts=tc)
            ctx.sync()
            c = [n, n] if counts is None else counts
            want, _, tol, _ = R.attend(p.ref, q, c, d ** -0.5)
            got = out.download().reshape(q.shape)
            for s in range(2):
                assert (np.abs(got[s, :c[s]] - want[s, :c[s]]) <= tol[s, :c[s]]).all()
            l64 = lse.download().reshape(2, heads, n).astype(np.float64)
            w, wt = R.attend(p.ref, q, c, d ** -0.5, lse_in=l64)
            got = acc.download().reshape(w.shape)
            assert (np.abs(got - want_acc - w) <=
                    wt + (want_acc + w) * (n * group + 2) * 2.0 ** -24).all()
            return got

        lens = [200, 150]
        a.append(rows(rng, 2, 200, kv, d), rows(rng, 2, 200, kv, d), lens, lens)
        acc = a.new(2 * kv * 256)
        got = attend_and_account(a, acc, np.zeros((2, kv, 256)), rows(rng, 2, 200, heads, d), lens)
        kept, bacc = a.new(2 * kv * keep, np.int32), a.new(2 * kv * 128, fill=-3)
        a.dev.evict(b.dev, acc, keep, recent, kept, bacc)
        ctx.sync()
        ids, want = a.ref.evict(got, keep, recent, b.ref)
        np.testing.assert_array_equal(kept.download().reshape(ids.shape), ids)
        np.testing.assert_array_equal(bacc.download().reshape(want.shape), want)
        b.check_content()
        lens = [keep, keep]
        for _ in range(5):
            lens = [x + 1 for x in lens]
            b.append(rows(rng, 2, 1, kv, d), rows(rng, 2, 1, kv, d), lens)
            want = attend_and_account(b, bacc, want, rows(rng, 2, 1, heads, d), None)
        aacc = a.new(2 * kv * 256)
        b.dev.evict(a.dev, bacc, keep, recent, kept, aacc)
        a.ref = R.RefCache(2, kv, d, 256, block, fmt)
        ctx.sync()
        ids, _ = b.ref.evict(want, keep, recent, a.ref)
        np.testing.assert_array_equal(kept.download().reshape(ids.shape), ids)
        a.check_attend(rows(rng, 2, 1, heads, d))


def test_captured_decode_steps_follow_the_lengths(ctx):
    """One graph of append, attend and accounts, replayed while the host moves the lengths on:
    every replay as the eager calls. A second graph of the same context takes turns with it."""
    rng = np.random.default_rng(51)
    kv, heads, d = 2, 8, 128
    with Context("any") as own, filled(own, rng, 2, kv, d, 1024, 32, "e4m3", [700, 0]) as p:
        k, v = p.new(2 * kv * d), p.new(2 * kv * d)
        tq, out, lse = p.new(2 * heads * d), p.new(2 * heads * d), p.new(2 * heads)
        acc, zero = p.new(2 * kv * 1024), p.new(2 * kv * 1024)

        def step(o, l):
            p.dev.append(k, v, 1)
            p.dev.attend(tq, o, heads, 1, lse=l)
            p.dev.weights(tq, l, zero, acc, heads, 1)

        lens = [700, 0]
        p.dev.set_lengths([701, 1])
        eo, el = p.new(2 * heads * d), p.new(2 * heads)
        step(eo, el)          # sizes the workspace
        own.sync()
        p.dev.set_lengths(lens)
        graphs = []
        for o, l in ((out, lse), (p.new(2 * heads * d), p.new(2 * heads))):
            own.capture_begin()
            step(o, l)
            graphs.append((own.capture_end(), o, l))
        for i in range(6):
            lens = [x + 1 for x in lens]
            kn, vn, q = rows(rng, 2, 1, kv, d), rows(rng, 2, 1, kv, d), rows(rng, 2, 1, heads, d)
            k.upload(kn), v.upload(vn), tq.upload(q)
            p.dev.set_lengths(lens)
            g, o, l = graphs[i % 2]
            g.launch()
            own.sync()
            p.ref.append(kn, vn, lens, [1, 1])
            p.check_content()
            want, _, tol, _ = R.attend(p.ref, q, [1, 1], d ** -0.5)
            got = o.download().reshape(q.shape)
            assert (np.abs(got - want) <= tol).all()
            graph_acc = acc.download()
            p.dev.attend(tq, eo, heads, 1, lse=el)
            p.dev.weights(tq, el, zero, acc, heads, 1)
            own.sync()
            np.testing.assert_array_equal(eo.download(), o.download())
            np.testing.assert_array_equal(acc.download(), graph_acc)
        for g, _, _ in graphs:
            g.destroy()


def test_a_capture_without_workspace_runs_unsplit(ctx):
    rng = np.random.default_rng(52)
    with Context("any") as own, filled(own, rng, 1, 1, 64, 8192, 64, "i8", [8000]) as p:
        q = rows(rng, 1, 1, 4, 64)
        tq, out = p.up(q), p.new(4 * 64)
        own.capture_begin()
        p.dev.attend(tq, out, 4, 1)
        g = own.capture_end()
        want, _, tol, _ = R.attend(p.ref, q, [1], 0.125)
        for _ in range(3):
            g.launch()
            own.sync()
            assert (np.abs(out.download().reshape(q.shape) - want) <= tol).all()
            out.upload(np.zeros(4 * 64, np.float32))
        g.destroy()


def test_accounts_captured_without_workspace(ctx):
    """Row groups cannot leave their sums anywhere: one wavefront after the other adds its rows."""
    rng = np.random.default_rng(56)
    n, heads, cap, lens = 60, 8, 384, [300, 61]
    with Context("any") as own, filled(own, rng, 2, 1, 64, cap, 32, "e4m3", lens) as p:
        q = rows(rng, 2, n, heads, 64)
        tq, out, lse = p.up(q), p.new(q.size), p.new(2 * heads * n)
        start = rng.uniform(0, 2, (2, 1, cap)).astype(np.float32)
        acc, res = p.up(start), p.new(start.size, fill=-3)
        own.capture_begin()
        p.dev.attend(tq, out, heads, n, lse=lse)
        p.dev.weights(tq, lse, acc, res, heads, n)
        g = own.capture_end()
        for _ in range(3):
            g.launch()
            own.sync()
            l64 = lse.download().reshape(2, heads, n).astype(np.float64)
            want, tol = R.attend(p.ref, q, [n, n], 0.125, lse_in=l64)
            got = res.download().reshape(start.shape)
            for s, ln in enumerate(lens):
                t = tol[s, :, :ln] + (want[s, :, :ln] + start[s, :, :ln]) * (n * heads + 2) * 2.0 ** -24
                assert (np.abs(got[s, :, :ln] - want[s, :, :ln] - start[s, :, :ln]) <= t).all()
                assert (got[s, :, ln:] == -3).all()
            res.upload(np.full(start.size, -3))
        g.destroy()


def test_eviction_and_read_in_a_graph(ctx):
    rng = np.random.default_rng(53)
    with filled(ctx, rng, 2, 1, 64, 256, 16, "i8", [250, 90]) as p, \
            Pair(ctx, 2, 1, 64, 128, 16, "i8") as q:
        w, kept = p.new(2 * 256), p.new(2 * 100, np.int32)
        ko = p.new(2 * 100 * 64)
        ctx.capture_begin()
        p.dev.evict(q.dev, w, 100, 10, kept)
        q.dev.read(100, ko, None)
        g = ctx.capture_end()
        for _ in range(3):
            x = rng.exponential(size=(2, 1, 256)).astype(np.float32)
            w.upload(x)
            g.launch()
            ctx.sync()
            q.ref = R.RefCache(2, 1, 64, 128, 16, "i8")
            ids, _ = p.ref.evict(x, 100, 10, q.ref)
            np.testing.assert_array_equal(kept.download().reshape(ids.shape), ids)
            np.testing.assert_array_equal(ko.download().reshape(2, 1, 100, 64),
                                          q.ref.read("k", 100))
        g.destroy()


def test_calls_run_on_the_adopted_stream(ctx):
    """The context's work goes to the stream it was given, in the order there: behind the copies
    that bring q, before the one that spoils it."""
    rng = np.random.default_rng(54)
    with Context("any") as other, Context("any") as own, \
            filled(own, rng, 1, 2, 64, 4096, 64, "i8", [4000]) as p:
        q = rows(rng, 1, 1, 8, 64)
        good, bad = p.up(q), p.new(512, fill=np.nan)
        big, tq, out = p.new(1 << 24), p.new(512), p.new(512)
        own.sync()
        check(lib().shp_set_stream(own.handle, lib().shp_get_stream(other.handle)), "set_stream")
        for _ in range(20):
            other.launch("add", big, big, big, [big.n])
        other.launch("reshape", good, None, tq, [512])
        p.dev.attend(tq, out, 8, 1)
        other.launch("reshape", bad, None, tq, [512])
        other.sync()
        got = out.download().reshape(q.shape)
        check(lib().shp_set_stream(own.handle, None), "set_stream")
        want, _, tol, _ = R.attend(p.ref, q, [1], 0.125)
        assert (np.abs(got - want) <= tol).all()


def test_calls_are_timed_by_name(ctx):
    rng = np.random.default_rng(55)
    with Context("any") as own, filled(own, rng, 1, 1, 64, 64, 16, "i8", [60]) as p:
        own.timing(True)
        p.attend(rows(rng, 1, 1, 2, 64))
        p.check_content()
        rep = own.timing_report()
        assert rep["cache8_attend"][1] == 1 and rep["cache8_read"][1] == 1
        own.timing(False)


def test_refusals_name_the_call(ctx):
    with Cache8(ctx, 1, 1, 64, 64) as c, Cache8(ctx, 1, 1, 64, 128) as dst:
        t = ctx.empty(4096)
        with pytest.raises(ShpError, match="shp_cache8_attend.*n_heads"):
            c.attend(t, t, 0, 1)
        with pytest.raises(ShpError, match="shp_cache8_evict.*keep"):
            c.evict(dst, t, 129, 0, t)
        with pytest.raises(ValueError, match="bytes where the cache needs"):
            Cache8(ctx, 1, 1, 64, 128, k=ctx.empty(4, np.uint8))
        t.free()


def test_a_closed_cache_refuses_calls(ctx):
    c, open_one = Cache8(ctx, 1, 1, 64, 64), Cache8(ctx, 1, 1, 64, 64)
    c.close()
    t = ctx.empty(4096)
    for call in (lambda: c.append(t, t, 1), lambda: c.read(1, t, t), lambda: c.attend(t, t, 1, 1),
                 lambda: c.weights(t, t, None, t, 1, 1), lambda: c.evict(open_one, t, 1, 0, t),
                 lambda: open_one.evict(c, t, 1, 0, t)):
        with pytest.raises(ShpError, match="null array in the cache"):
            call()
    c.close()
    open_one.close()
    t.free()
