"""The paged cache on the GPU against tests/paged_ref.py.

What is stored unturned and what acceptance moves are compared bit for bit; rotation and attention
within the bounds that paged_ref derives from the operations' roundings."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from spirv_inference_amd import Context, DeviceTensor, PagedCache, ShpError
from spirv_inference_amd._lib import check, lib

pytestmark = pytest.mark.gpu

FORMATS = ["f32", "f16", "bf16"]


class Pair:
    """A device cache whose pages lie in any order and hold NaN until they are written, and the
    reference."""

    def __init__(self, ctx, n_seqs, kv, d, max_pages, page, fmt, seed=0, spare=3):
        self.ctx, self.dims, self.page, self.fmt = ctx, (n_seqs, kv, d, max_pages * page), page, fmt
        self.ref = R.RefPaged(n_seqs, kv, d, max_pages * page, fmt)
        self.n_pages = n_seqs * max_pages + spare
        self.dev = PagedCache(ctx, n_seqs, kv, d, self.n_pages, page, max_pages, fmt)
        self.fill = np.nan if fmt == "f32" else 0xFFFF  # NaN as fp16 and as bf16
        for t in (self.dev.k, self.dev.v):
            t.upload(np.full(t.n, self.fill, t.dtype))
        order = np.random.default_rng(seed).permutation(self.n_pages)[:n_seqs * max_pages]
        self.table = order.reshape(n_seqs, max_pages).astype(np.int32)
        self.dev.set_table(self.table)
        self.temp = []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for t in self.temp:
            t.free()
        self.dev.close()

    def up(self, a, dtype=np.float32):
        if a is None:
            return None
        t = self.ctx.tensor(np.ascontiguousarray(a), dtype)
        self.temp.append(t)
        return t

    def new(self, n, dtype=np.float32, fill=0):
        return self.up(np.full(n, fill, dtype), dtype)

    def drop(self, s, page, entry=-1):
        """Takes a page from a sequence: its table has `entry` there."""
        self.table[s, page] = entry
        self.dev.set_table(self.table)
        self.ref.there[s, page * self.page:(page + 1) * self.page] = False

    def put(self, lens, k, v):
        """Fills the device and the reference with lens[s] tokens of k, v [s][kv][tokens][d]."""
        self.ref.lens = list(lens)
        self.dev.set_lengths(lens)
        s_, kv, d, cap = self.dims
        for name, x in (("k", k), ("v", v)):
            x = R.stored(x, self.fmt)
            w = np.full((self.n_pages, kv, self.page, d), self.fill, getattr(self.dev, name).dtype)
            for s, ln in enumerate(lens):
                getattr(self.ref, name)[s, :, :ln] = x[s, :, :ln]
                for p in range(-(-ln // self.page)):
                    a, b = p * self.page, min(ln, (p + 1) * self.page)
                    w[self.table[s, p], :, :b - a] = R.words(x[s, :, a:b], self.fmt)
            getattr(self.dev, name).upload(w)

    def content(self, name):
        """What the device holds, [s][kv][cap][d], words."""
        s_, kv, d, cap = self.dims
        w = getattr(self.dev, name).download().reshape(self.n_pages, kv, self.page, d)
        return w[self.table].transpose(0, 2, 1, 3, 4).reshape(s_, kv, cap, d)

    def attend(self, q, counts=None, lse=True, **how):
        s_, n, heads, d = q.shape
        out, l = self.new(q.size, fill=-3), self.new(s_ * heads * n, fill=-3)
        arrays = {x: self.up(how.get(x), np.int32) for x in ("prefix", "first", "parents")}
        self.dev.attend(self.up(q), out, heads, n, counts=self.up(counts, np.int32),
                        lse=l if lse else None, scale=how.get("scale"), cap=how.get("cap"),
                        slopes=self.up(how.get("slopes")), window=how.get("window"), **arrays)
        self.ctx.sync()
        return out.download().reshape(q.shape), l.download().reshape(s_, heads, n)

    def check_attend(self, q, counts=None, **how):
        s_, n, heads, d = q.shape
        out, lse = self.attend(q, counts, **how)
        c = [n] * s_ if counts is None else [max(0, min(n, x)) for x in counts]
        with np.errstate(invalid="ignore"):
            want, wl, tol, ltol = self.ref.attend(
                q, c, how.get("scale") or d ** -0.5, how.get("cap") or 0.0, how.get("slopes"),
                how.get("window") or 0, how.get("prefix"), how.get("first"), how.get("parents"))
        for s in range(s_):
            assert (out[s, c[s]:] == -3).all() and (lse[s, :, c[s]:] == -3).all(), "rows behind"
            o, w = out[s, :c[s]].astype(np.float64), want[s, :c[s]]
            assert np.isfinite(o).all()
            over = np.abs(o - w) - tol[s, :c[s]] - 1e-30
            assert (over <= 0).all(), (s, np.argwhere(over > 0)[:5], over.max())
            g, wg = lse[s, :, :c[s]].astype(np.float64), wl[s, :, :c[s]]
            np.testing.assert_array_equal(g == -np.inf, wg == -np.inf)
            f = np.isfinite(wg)
            assert np.isfinite(g[f]).all()
            assert (np.abs(g[f] - wg[f]) <= ltol[s, :, :c[s]][f]).all()
        return out, lse


def rows(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def filled(ctx, rng, n_seqs, kv, d, max_pages, page, fmt, lens):
    p = Pair(ctx, n_seqs, kv, d, max_pages, page, fmt, seed=len(lens) + page)
    n = max(max(lens), 1)
    p.put(lens, rows(rng, n_seqs, kv, n, d), rows(rng, n_seqs, kv, n, d))
    return p


# ---- append ---------------------------------------------------------------------------------

def freqs(rot):
    return (10000.0 ** (-np.arange(rot // 2) / max(rot // 2, 1))).astype(np.float32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,kv,group,n,page,rot,inter", [
    (64, 1, 1, 1, 16, 64, False), (64, 3, 7, 5, 16, 64, True), (128, 2, 4, 33, 64, 128, False),
    (128, 8, 4, 17, 256, 24, False), (64, 4, 8, 3, 32, 8, True), (128, 1, 1, 70, 128, 0, False),
    (128, 2, 1, 9, 32, 56, True)])
def test_append(ctx, fmt, d, kv, group, n, page, rot, inter):
    """Rows at the start, in the middle and over the edge of pages; ragged counts; what lies in front
    and behind stays."""
    rng = np.random.default_rng(n)
    lens, counts = [n, 77, 150], [n, max(0, n - 2), min(n, 3)]
    heads = kv * group
    with Pair(ctx, 3, kv, d, -(-160 // page), page, fmt) as p:
        k, v, q = rows(rng, 3, n, kv, d), rows(rng, 3, n, kv, d), rows(rng, 3, n, heads, d)
        out = p.new(q.size, fill=-3)
        p.dev.set_lengths(lens)
        p.dev.append(p.up(k), p.up(v), n, counts=p.up(counts, np.int32), q=p.up(q), q_out=out,
                     n_heads=heads, inv_freq=p.up(freqs(rot)) if rot else None, interleaved=inter,
                     rot=rot)
        ctx.sync()
        out, kc, vc = out.download().reshape(q.shape), p.content("k"), p.content("v")
        for s in range(3):
            c, base = counts[s], lens[s] - counts[s]
            pos = base + np.arange(c)
            bound = R.turned_bound(q[s, :c], freqs(rot), inter)
            assert (np.abs(out[s, :c] - R.turned(q[s, :c], pos, freqs(rot), inter)) <= bound).all()
            assert (out[s, c:] == -3).all()
            np.testing.assert_array_equal(vc[s, :, base:lens[s]],
                                          R.words(R.stored(v[s, :c], fmt), fmt).transpose(1, 0, 2))
            want = R.turned(k[s, :c], pos, freqs(rot), inter).transpose(1, 0, 2)
            got = R.values(kc[s, :, base:lens[s]].copy(), fmt)
            bound = R.turned_bound(k[s, :c], freqs(rot), inter).transpose(1, 0, 2)
            least = 0.0 if fmt == "f32" else 2.0 ** -25 if fmt == "f16" else 2.0 ** -134
            assert (np.abs(got - want) <= bound + (np.abs(want) + bound) * R.STEP[fmt] + least).all()
            for x in (kc, vc):
                x = R.values(x.copy(), fmt)
                assert np.isnan(x[s, :, :base]).all() and np.isnan(x[s, :, lens[s]:]).all()


def test_append_far_positions(ctx):
    """Positions of millions, where an angle in fp32 would have lost its fraction, quarter turns and
    negative positions, in place."""
    rng = np.random.default_rng(3)
    n, d = 64, 64
    offsets = np.concatenate([np.arange(16), 131071 + np.arange(16), 4194303 - np.arange(16),
                              -np.arange(8), [2 ** 31 - 1 - 64, -2 ** 31, 10 ** 9, 7, 22, 355, 710, 103993]])
    with Pair(ctx, 1, 1, d, 4, 16, "f32") as p:
        for f in (freqs(d), np.full(32, np.float32(np.pi / 2)), np.geomspace(1e-8, 3, 32).astype(np.float32)):
            q, k = rows(rng, 1, n, 2, d), rows(rng, 1, n, 1, d)
            dq = p.up(q)
            p.dev.set_lengths([n])
            p.dev.append(p.up(k), p.up(k), n, q=dq, q_out=dq, n_heads=2, inv_freq=p.up(f),
                         offsets=p.up(offsets, np.int32))
            ctx.sync()
            got = dq.download().reshape(q.shape)[0]
            # the quarter turns are taken off to 2^-53 of up to 2^33, which adds 2^-19 of the size there
            far = 2.0 ** -52 * np.abs(offsets[:, None] * f.astype(np.float64))
            extra = (np.abs(q[0, ..., :32]) + np.abs(q[0, ..., 32:])) * far[:, None]
            bound = R.turned_bound(q[0], f, False) + np.concatenate([extra, extra], -1)
            assert (np.abs(got - R.turned(q[0], offsets, f, False)) <= bound).all()
            kc = p.content("k")[0, 0]
            extra = (np.abs(k[0, :, 0, :32]) + np.abs(k[0, :, 0, 32:])) * far
            bound = R.turned_bound(k[0], f, False)[:, 0] + np.concatenate([extra, extra], -1)
            assert (np.abs(kc - R.turned(k[0], offsets, f, False)[:, 0]) <= bound).all()


def test_far_offsets_behind_a_context(ctx):
    """Sums of length and offset that pass 32 bits."""
    rng = np.random.default_rng(51)
    d = 64
    offsets = np.array([2 ** 31 - 1, 2 ** 31 - 1 - 300, 2 ** 31 - 200, 2 ** 31 - 1000, 5, -2 ** 31])
    n = len(offsets)
    with Pair(ctx, 1, 1, d, 64, 16, "f32") as p:
        f = np.geomspace(1e-9, 1e-3, 32).astype(np.float32)
        q, k = rows(rng, 1, n, 2, d), rows(rng, 1, n, 1, d)
        dq = p.up(q)
        p.dev.set_lengths([1000])
        p.dev.append(p.up(k), p.up(k), n, q=dq, q_out=dq, n_heads=2, inv_freq=p.up(f), offsets=p.up(offsets, np.int32))
        ctx.sync()
        got = dq.download().reshape(q.shape)[0]
        pos = 1000 - n + offsets
        # two roundings in 64 bits, of the product and of its quarter turns, and one of the quarter turns' length
        far = 3 * 2.0 ** -53 * np.abs(pos[:, None] * f.astype(np.float64))
        extra = (np.abs(q[0, ..., :32]) + np.abs(q[0, ..., 32:])) * far[:, None]
        bound = R.turned_bound(q[0], f, False) + np.concatenate([extra, extra], -1)
        assert (np.abs(got - R.turned(q[0], pos, f, False)) <= bound).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_of_strided_rows(ctx, fmt):
    """q, k and v side by side in one tensor, as a fused projection leaves them; q in place."""
    rng = np.random.default_rng(4)
    n, d, width = 6, 64, (4 + 2 + 2) * 64 + 4
    x = rows(rng, 2, n, width)
    with Pair(ctx, 2, 2, d, 2, 16, fmt) as p:
        t = p.up(x)
        part = [DeviceTensor(ctx, 1, np.float32, ptr=t.ptr + 4 * d * o, owned=False) for o in (0, 4, 6)]
        st = (n * width, width, d)
        p.dev.set_lengths([n, 20])
        p.dev.append(part[1], part[2], n, q=part[0], q_out=part[0], n_heads=4, inv_freq=p.up(freqs(64)),
                     k_strides=st, v_strides=st, q_strides=st, o_strides=st)
        ctx.sync()
        got = t.download().reshape(x.shape)
        np.testing.assert_array_equal(got[..., 4 * d:], x[..., 4 * d:])
        for s, base in enumerate((0, 20 - n)):
            q = x[s, :, :4 * d].reshape(n, 4, d)
            assert (np.abs(got[s, :, :4 * d].reshape(n, 4, d)
                           - R.turned(q, base + np.arange(n), freqs(64), False))
                    <= R.turned_bound(q, freqs(64), False)).all()
            v = x[s, :, 6 * d:8 * d].reshape(n, 2, d).transpose(1, 0, 2)
            np.testing.assert_array_equal(p.content("v")[s, :, base:base + n],
                                          R.words(R.stored(v, fmt), fmt))


@pytest.mark.parametrize("fmt", ["f16", "bf16"])
def test_append_rounds_to_nearest_even(ctx, fmt):
    bits = 10 if fmt == "f16" else 7
    x = np.array([1 + 2.0 ** -(bits + 1), 1 + 3 * 2.0 ** -(bits + 1), -1 - 2.0 ** -(bits + 1) - 2.0 ** -20,
                  65504, 65519, 65520, 3.4e38, -3.4e38, 1e-8, 6e-8, 2.0 ** -25, 3 * 2.0 ** -25, 1e-40, 0,
                  -0.0, np.inf, -np.inf, np.nan], np.float32)
    v = np.resize(x, (1, 2, 1, 64)).astype(np.float32)
    with Pair(ctx, 1, 1, 64, 1, 16, fmt) as p:
        p.dev.set_lengths([2])
        p.dev.append(p.up(v), p.up(v), 2)
        ctx.sync()
        for name in "kv":
            got = R.values(p.content(name)[0, 0, :2].copy(), fmt)
            np.testing.assert_array_equal(got, R.stored(v[0, :, 0], fmt))


def test_appends_without_pages_or_before_the_first_token_are_dropped(ctx):
    rng = np.random.default_rng(5)
    k = rows(rng, 4, 40, 1, 64)
    with Pair(ctx, 4, 1, 64, 3, 16, "f32") as p:
        for s, bad in enumerate((-1, p.n_pages, 2 ** 31 - 1, -2 ** 31)):
            p.table[s, 1] = bad
        p.dev.set_table(p.table)
        before = p.dev.k.download()
        p.dev.set_lengths([40, 48, 17, 0])
        p.dev.append(p.up(k), p.up(k), 40, counts=p.up([40, 40, 40, 40], np.int32))
        ctx.sync()
        got = p.dev.k.download().reshape(p.n_pages, 16, 64)
        want = before.reshape(p.n_pages, 16, 64).copy()
        for s, ln in enumerate((40, 48, 17, 0)):
            for i in range(40):
                t = ln - 40 + i
                if t >= 0 and t // 16 != 1:
                    want[p.table[s, t // 16], t % 16] = k[s, i, 0]
        np.testing.assert_array_equal(got, want)


def test_lengths_and_counts_out_of_range_stay_in_bounds(ctx):
    rng = np.random.default_rng(6)
    k = rows(rng, 4, 3, 1, 64)
    with Pair(ctx, 4, 1, 64, 4, 16, "f32") as p:
        for t in (p.dev.k, p.dev.v):
            t.upload(np.zeros(t.n))
        p.dev.set_lengths([-5, 1 << 30, 3, 3])
        counts = p.up([3, 3, -1, 1 << 30], np.int32)
        p.dev.append(p.up(k), p.up(k), 3, counts=counts)
        ctx.sync()
        got = p.content("k")[:, 0]
        np.testing.assert_array_equal(got[1, 61:], k[1, :, 0])
        np.testing.assert_array_equal(got[3, :3], k[3, :, 0])
        assert (got[0] == 0).all() and (got[1, :61] == 0).all() and (got[2] == 0).all()
        out, l = p.attend(rows(rng, 4, 1, 2, 64))
        assert (out[0] == 0).all() and (l[0] == -np.inf).all() and np.isfinite(out).all()


# ---- attention ------------------------------------------------------------------------------

SHAPES = [
    (1, 1, 1, 16, [1, 2]),
    (2, 4, 1, 16, [63, 64]),
    (2, 8, 1, 64, [65, 300]),
    (1, 16, 1, 32, [700, 0]),
    (3, 5, 1, 256, [129, 17]),
    (1, 33, 1, 16, [40, 555]),       # 33 heads on one
    (2, 3, 7, 32, [90, 7]),          # 21 rows
    (1, 8, 5, 64, [200, 3]),         # 40 rows; a sequence shorter than its rows
    (2, 4, 33, 128, [33, 161]),      # 132 rows, a prompt from the start
    (1, 7, 64, 16, [500, 64])]       # 448 rows


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kv,group,n,page,lens", SHAPES)
def test_attention(ctx, fmt, d, kv, group, n, page, lens):
    rng = np.random.default_rng(11 + n)
    with filled(ctx, rng, 2, kv, d, -(-max(lens) // page) + 1, page, fmt, lens) as p:
        p.check_attend(rows(rng, 2, n, kv * group, d))


HOW = {
    "cap": dict(cap=5.0), "bias": dict(bias=True), "window": dict(window=37), "window1": dict(window=1),
    "window of all": dict(window=100000), "prefix": dict(prefix=[100, 3]),
    "prefix and window": dict(prefix=[17, 70], window=64), "first": dict(first=True),
    "all": dict(cap=3.0, bias=True, window=50, prefix=[20, 5], first=True)}


def options(how, rng, n, heads, lens):
    how = dict(how)
    if how.pop("bias", False):
        how["slopes"] = np.exp2(-8.0 * np.arange(1, heads + 1) / heads).astype(np.float32)
    if how.pop("first", False):
        how["first"] = np.stack([np.sort(rng.integers(0, max(ln, 1), n)) for ln in lens])
    return how


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("d,kv,group,n,page,lens", [
    (64, 2, 4, 1, 16, [300, 129]), (128, 1, 8, 33, 32, [33, 211]), (64, 1, 3, 150, 64, [150, 400]),
    (128, 2, 1, 3, 128, [700, 2])])
def test_attention_forms(ctx, fmt, how, d, kv, group, n, page, lens):
    rng = np.random.default_rng(12 + n)
    with filled(ctx, rng, 2, kv, d, -(-max(lens) // page), page, fmt, lens) as p:
        p.check_attend(rows(rng, 2, n, kv * group, d), **options(HOW[how], rng, n, kv * group, lens))


def trees(rng, n_seqs, n):
    """Recursive trees; some rows that name no earlier row hang on the context."""
    out = np.zeros((n_seqs, n), np.int64)
    for s in range(n_seqs):
        for i in range(n):
            out[s, i] = rng.integers(0, i) if i and rng.random() < 0.9 else rng.choice([-1, i, i + 3, -7, 2 ** 30])
    return out


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,kv,group,n,page,lens,counts", [
    (64, 2, 4, 1, 16, [300, 1], None), (64, 1, 8, 24, 16, [24, 331], None), (128, 2, 4, 60, 64, [500, 161], [60, 31]),
    (64, 1, 1, 256, 32, [700, 256], [256, 255]), (128, 1, 5, 130, 128, [200, 129], [100, 130])])
@pytest.mark.parametrize("how", [{}, dict(window=3), dict(bias=True, cap=4.0), dict(prefix=[10, 260], window=40),
                                 dict(first=True, bias=True)])
def test_attention_of_trees(ctx, fmt, d, kv, group, n, page, lens, counts, how):
    rng = np.random.default_rng(13 + n)
    with filled(ctx, rng, 2, kv, d, -(-max(lens) // page), page, fmt, lens) as p:
        p.check_attend(rows(rng, 2, n, kv * group, d), counts=counts, parents=trees(rng, 2, n),
                       **options(how, rng, n, kv * group, lens))


@pytest.mark.parametrize("fmt", FORMATS)
def test_trees_of_sequences_that_are_shorter(ctx, fmt):
    """Rows before the first token see nothing, and their places are nobody's."""
    rng = np.random.default_rng(29)
    with filled(ctx, rng, 3, 1, 64, 6, 16, fmt, [20, 90, 1]) as p:
        for n in (33, 70, 128):
            for how in ({}, dict(window=4), dict(prefix=[5, 80, 1], bias=True)):
                p.check_attend(rows(rng, 3, n, 3, 64), parents=trees(rng, 3, n), **options(how, rng, n, 3, [20, 90, 1]))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("first", [0, 63, 64, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 64, 1 << 30])
def test_first_tokens_of_any_size(ctx, fmt, first):
    rng = np.random.default_rng(30)
    with filled(ctx, rng, 2, 1, 64, 8, 16, fmt, [128, 70]) as p:
        for n in (1, 20, 70):
            f = np.full((2, n), first, np.int64)
            p.check_attend(rows(rng, 2, n, 3, 64), first=f)
            f[:, ::2] = 5
            p.check_attend(rows(rng, 2, n, 3, 64), first=f, window=2 ** 31 - 1, prefix=[2 ** 31 - 1, -2 ** 31])


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_table_with_room_for_millions(ctx, fmt):
    """Most of the table names no page, and most workgroups have nothing to do."""
    rng = np.random.default_rng(34)
    with PagedCache(ctx, 2, 2, 64, 20, 16, 1 << 18, fmt=fmt) as dev:
        table = np.full((2, 1 << 18), -1, np.int32)
        table[0, :10], table[1, :10] = np.arange(10), np.arange(10, 20)
        dev.set_table(table)
        for lens in ([150, 33], [1 << 22, 5]):  # the second: of four million tokens 160 are there
            dev.set_lengths([150, 33])
            k, v = rows(rng, 2, 150, 2, 64), rows(rng, 2, 150, 2, 64)
            ts = [ctx.tensor(x) for x in (k, v)]
            counts = ctx.tensor(np.array([150, 33]), np.int32)
            dev.append(ts[0], ts[1], 150, counts=counts)
            dev.set_lengths(lens)
            ref = R.RefPaged(2, 2, 64, 160, fmt)
            for s, ln in enumerate((150, 33)):
                ref.k[s, :, :ln] = R.stored(k[s, :ln], fmt).transpose(1, 0, 2)
                ref.v[s, :, :ln] = R.stored(v[s, :ln], fmt).transpose(1, 0, 2)
            ref.lens = [150, lens[1]]
            if lens[0] > 160:  # places 150 .. 159 hold zeros
                ref.lens[0] = 160
                w = np.zeros((20, 2, 16, 64), dev.k.dtype)
                for name in "kv":
                    t = getattr(dev, name)
                    w = t.download().reshape(20, 2, 16, 64)
                    w[9, :, 6:] = 0
                    t.upload(w)
            q = rows(rng, 2, 1, 6, 64)
            out, dq = ctx.empty(q.size), ctx.tensor(q)
            dev.attend(dq, out, 6, 1)
            ctx.sync()
            want, _, tol, _ = ref.attend(q, [1, 1], 0.125)
            assert (np.abs(out.download().reshape(q.shape) - want) <= tol).all()
            for t in (*ts, counts, out, dq):
                t.free()


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_chain_of_rows_is_a_deep_tree(ctx, fmt):
    """Row i on row i - 1: 256 levels, the same as causal rows."""
    rng = np.random.default_rng(14)
    with filled(ctx, rng, 1, 1, 64, 30, 16, fmt, [450]) as p:
        q = rows(rng, 1, 256, 2, 64)
        chain = np.arange(-1, 255)[None]
        for how in ({}, dict(window=20), dict(slopes=np.float32([0.1, 0.02]))):
            a = p.check_attend(q, parents=chain, **how)
            b = p.check_attend(q, **how)
            np.testing.assert_allclose(a[1], b[1], rtol=1e-5)


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_over_missing_pages(ctx, fmt):
    """Entries that name no page, inside a tile, at its edges and for a whole sequence."""
    rng = np.random.default_rng(15)
    with filled(ctx, rng, 3, 2, 64, 10, 16, fmt, [150, 160, 33]) as p:
        p.drop(0, 0)
        p.drop(0, 5, p.n_pages)
        p.drop(1, 9, -2 ** 31)
        p.drop(1, 3, 2 ** 31 - 1)
        for x in range(3):
            p.drop(2, x)
        for n in (1, 9):
            q = rows(rng, 3, n, 8, 64)
            out, lse = p.check_attend(q)
            assert (out[2] == 0).all() and (lse[2] == -np.inf).all()
            p.check_attend(q, window=30, prefix=[20, 20, 20])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_what_a_row_does_not_see_has_no_part(ctx, fmt, bad):
    """Keys and values that are not finite spoil the rows that see them and no others: behind a row,
    out of its window, of another document, of another branch."""
    rng = np.random.default_rng(16)
    ln, n, d = 90, 40, 64
    k, v = rows(rng, 1, 1, ln, d), rows(rng, 1, 1, ln, d)
    k[0, 0, 70, 3] = bad
    v[0, 0, 70, 5] = bad
    v[0, 0, 20, 6] = bad
    q = rows(rng, 1, n, 2, d)
    parents = trees(rng, 1, n)
    for how in (dict(first=np.full((1, n), 21)), dict(window=30), dict(window=5, prefix=[9]),
                dict(parents=parents, first=np.full((1, n), 21)),
                dict(first=np.where(np.arange(n) < 20, 0, 71)[None])):
        with Pair(ctx, 1, 1, d, 6, 16, fmt) as p:
            p.put([ln], k, v)
            out, lse = p.attend(q, **how)
            sees, _ = R.sight(ln, n, 96, np.ones(96, bool), how.get("window", 0),
                              how.get("prefix", [0])[0], how["first"][0] if "first" in how else None,
                              parents[0] if "parents" in how else None)
            clean = Pair(ctx, 1, 1, d, 6, 16, fmt)
            with clean:
                k2, v2 = k.copy(), v.copy()
                k2[0, 0, 70, 3] = v2[0, 0, 70, 5] = v2[0, 0, 20, 6] = 0.0
                clean.put([ln], k2, v2)
                with np.errstate(invalid="ignore"):
                    want, wl, tol, _ = clean.ref.attend(q, [n], d ** -0.5, 0.0, None, how.get("window", 0),
                                                        how.get("prefix"), how.get("first"), how.get("parents"))
            hit20, hit70 = sees[:, 20], sees[:, 70]
            free = ~hit20 & ~hit70
            assert free.any() and (hit20.any() or hit70.any())
            assert (np.abs(out[0, free] - want[0, free]) <= tol[0, free] + 1e-30).all()
            only = hit20 & ~hit70  # its values are as without it but for the dimension
            ok = np.abs(out[0, only] - want[0, only]) <= tol[0, only] + 1e-30
            ok[..., 6] = ~np.isfinite(out[0, only][..., 6])
            assert ok.all()
            assert not np.isfinite(out[0, hit70][..., 5]).any() or bad == -np.inf


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("scale", [-0.3, 3.0, 1e-30])
def test_attention_scales(ctx, fmt, scale):
    """Uniform, reversed and nearly one-hot weights, and caps that bend most scores."""
    rng = np.random.default_rng(17)
    with filled(ctx, rng, 1, 1, 64, 13, 16, fmt, [200]) as p:
        p.check_attend(rows(rng, 1, 3, 4, 64), scale=scale)
        p.check_attend(rows(rng, 1, 3, 4, 64), scale=scale, cap=1.0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_caps_from_small_to_large(ctx, fmt):
    rng = np.random.default_rng(18)
    with filled(ctx, rng, 1, 1, 128, 8, 32, fmt, [250]) as p:
        for cap in (1e-6, 0.3, 50.0, 1e6, 1e30):
            p.check_attend(rows(rng, 1, 2, 4, 128), cap=cap)


FLT_MAX = float(np.finfo(np.float32).max)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("cap", [1e9, 1e18, 1e27, 1e33, 1e36, 2.0 ** 126, 2.3e38, 2.4e38, FLT_MAX])
@pytest.mark.parametrize("scale", [0.125, 3.0, 1e-3])
def test_caps_up_to_the_largest(ctx, fmt, cap, scale):
    """Such caps bend nothing: out and lse are those of the scores themselves."""
    rng = np.random.default_rng(49)
    with filled(ctx, rng, 2, 2, 64, 13, 16, fmt, [200, 65]) as p:
        p.check_attend(rows(rng, 2, 3, 8, 64), cap=cap, scale=scale)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,kv,group,n,ln,how", [
    (64, 1, 4, 1, 3001, {}), (128, 2, 4, 33, 700, HOW["all"]), (128, 1, 8, 60, 500, dict(tree=True, bias=True)),
    (64, 72, 4, 101, 130, dict(window=37))])
def test_large_caps_in_every_form(ctx, fmt, d, kv, group, n, ln, how):
    """Split over shares, with masks, in trees and of many blocks, on both sides of the caps that are large."""
    rng = np.random.default_rng(52)
    with filled(ctx, rng, 2, kv, d, -(-ln // 16), 16, fmt, [ln, n]) as p:
        opts = {**how, **(dict(parents=trees(rng, 2, n)) if how.get("tree") else {})}
        opts.pop("tree", None)
        opts = options(opts, rng, n, kv * group, [ln, n])
        q = rows(rng, 2, n, kv * group, d)
        for cap in (float(np.nextafter(np.float32(2.0 ** 64), np.float32(0))), 2.0 ** 64, FLT_MAX):
            p.check_attend(q, **{**opts, "cap": cap})


def test_large_caps_bend_large_scores(ctx):
    """Scores of the cap's own size: out is finite and lse the largest capped score within fp32's roundings."""
    rng = np.random.default_rng(53)
    for fmt in ("f32", "bf16"):
        with Pair(ctx, 1, 1, 64, 13, 16, fmt) as p:
            k = rows(rng, 1, 1, 200, 64) * np.float32(2.0 ** 50)
            p.put([200], k, rows(rng, 1, 1, 200, 64))
            q = rows(rng, 1, 3, 4, 64) * np.float32(2.0 ** 50)
            for cap in (2.0 ** 63, 2.0 ** 100, 2.0 ** 101):
                p.check_attend(q, cap=cap)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("scale,cap", [(2.0 ** 126, None), (-2.0 ** 126, None), (2.35e38, None), (-2.35e38, None),
                                       (3.4e38, 30.0), (3.4e38, 2.0 ** 64), (2.0 ** 126, FLT_MAX)])
def test_scales_up_to_the_largest(ctx, fmt, scale, cap):
    """Over queries that are as small."""
    rng = np.random.default_rng(50)
    with filled(ctx, rng, 1, 1, 64, 13, 16, fmt, [200]) as p:
        p.check_attend(rows(rng, 1, 3, 4, 64) * np.float32(2.0 ** -125), scale=scale, cap=cap)


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_of_large_and_small_values(ctx, fmt):
    """Weights times values near the ends of the range."""
    rng = np.random.default_rng(19)
    top = {"f32": 3.4e38, "f16": 65504.0, "bf16": 3.3e38}[fmt]
    k, v = rows(rng, 1, 1, 100, 64), rng.uniform(0.5, 1, (1, 1, 100, 64)).astype(np.float32) * np.float32(top)
    with Pair(ctx, 1, 1, 64, 7, 16, fmt) as p:
        p.put([100], k, v)
        p.check_attend(rows(rng, 1, 3, 4, 64))
        p.put([100], k, v * np.float32(2.0 ** -126 if fmt != "f16" else 2.0 ** -30))
        p.check_attend(rows(rng, 1, 3, 4, 64))
        p.put([100], k * 0, v * 0)
        out, lse = p.check_attend(rows(rng, 1, 3, 4, 64))
        assert (out == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_scores_that_are_far_apart(ctx, fmt):
    """A first tile of small scores, one large score later; distances that leave one token."""
    rng = np.random.default_rng(20)
    k, v = rows(rng, 1, 1, 300, 64), rows(rng, 1, 1, 300, 64)
    k[0, 0, 257] *= 60
    k[0, 0, 130] *= 30
    with Pair(ctx, 1, 1, 64, 19, 16, fmt) as p:
        p.put([300], k, v)
        q = rows(rng, 1, 5, 4, 64)
        p.check_attend(q)
        p.check_attend(-q)
        p.check_attend(q, slopes=np.float32([100.0, 0.0, 3.0, -0.05]))


@pytest.mark.parametrize("fmt", FORMATS)
def test_padded_and_strided_rows(ctx, fmt):
    rng = np.random.default_rng(21)
    with filled(ctx, rng, 4, 2, 64, 16, 16, fmt, [100, 256, 5, 0]) as p:
        p.check_attend(rows(rng, 4, 6, 8, 64), counts=[6, 1, 0, 3])
        p.check_attend(rows(rng, 4, 40, 8, 64), counts=[40, 17, 2, 0], window=9)
        p.check_attend(rows(rng, 4, 2, 8, 64), counts=[9, -1, 2, 1])
        # heads before rows, out with gaps
        q = rows(rng, 4, 8, 3, 64)
        out = p.new(4 * 3 * (8 * 64 + 8), fill=-3)
        p.dev.attend(p.up(q), out, 8, 3, q_strides=(8 * 3 * 64, 64, 3 * 64),
                     o_strides=(3 * (8 * 64 + 8), 8 * 64 + 8, 64))
        ctx.sync()
        got = out.download().reshape(4, 3, 8 * 64 + 8)
        assert (got[..., 8 * 64:] == -3).all()
        want = p.attend(q.transpose(0, 2, 1, 3))[0]
        np.testing.assert_array_equal(got[..., :8 * 64].reshape(want.shape), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,kv,group,n,ln,page", [(128, 1, 4, 1, 5000, 64), (64, 2, 1, 2, 3001, 16),
                                                  (64, 1, 8, 40, 2500, 256)])
def test_long_sequences(ctx, fmt, d, kv, group, n, ln, page):
    rng = np.random.default_rng(22)
    with filled(ctx, rng, 1, kv, d, -(-ln // page), page, fmt, [ln]) as p:
        q = rows(rng, 1, n, kv * group, d)
        p.check_attend(q)
        p.check_attend(q, window=ln // 2, prefix=[200])


# So many blocks of rows that their tokens are not shared out.
@pytest.mark.parametrize("fmt", ["f16", "bf16"])
@pytest.mark.parametrize("d,kv,group,n,lens,counts", [
    (64, 56, 4, 101, [101, 230], None), (128, 75, 3, 90, [77, 90], [77, 3]), (64, 224, 1, 70, [70, 4], None)])
@pytest.mark.parametrize("how", ["cap", "window", "prefix and window", "first", "all", "tree"])
def test_attention_of_many_blocks(ctx, fmt, d, kv, group, n, lens, counts, how):
    rng = np.random.default_rng(25 + n)
    with filled(ctx, rng, 2, kv, d, 16, 16, fmt, lens) as p:
        opts = dict(parents=trees(rng, 2, n), bias=True) if how == "tree" else HOW[how]
        if how == "first":
            p.drop(0, 1)
        p.check_attend(rows(rng, 2, n, kv * group, d), counts=counts,
                       **options(opts, rng, n, kv * group, lens))


@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_many_blocks_do_not_see_what_is_masked(ctx, bad):
    rng = np.random.default_rng(26)
    n, ln = 64, 100
    k, v = rows(rng, 1, 224, ln, 64), rows(rng, 1, 224, ln, 64)
    v[0, :, 90, 7] = bad
    with Pair(ctx, 1, 224, 64, 7, 16, "bf16") as p:
        p.put([ln], k, v)
        q = rows(rng, 1, n, 448, 64)
        out, _ = p.attend(q)
        hit = np.arange(n) + ln - n >= 90
        p.ref.v[0, :, 90, 7] = 0
        want, _, tol, _ = p.ref.attend(q, [n], 0.125)
        assert (np.abs(out[0, ~hit] - want[0, ~hit]) <= tol[0, ~hit]).all()
        got, ok = out[0, hit], np.ones(64, bool)
        ok[7] = False
        assert not np.isfinite(got[..., 7]).any()
        assert (np.abs(got - want[0, hit]) <= tol[0, hit])[..., ok].all()


# So many blocks of rows that a wavefront takes one by itself.
WAVES = [(64, 72, 4, 101, [101, 230], None), (128, 100, 3, 90, [77, 90], [77, 3]), (64, 300, 1, 70, [70, 4], None),
         (128, 180, 1, 160, [160, 171], [111, 160])]


def takes_waves(p, n, heads):
    out = (C.c_int32 * 4)()
    check(lib().shp_paged_attend_plan(p.ctx.handle, C.byref(p.dev._struct), n, heads, out), "shp_paged_attend_plan")
    return out[1] == 1


@pytest.mark.parametrize("fmt", ["f16", "bf16"])
@pytest.mark.parametrize("d,kv,group,n,lens,counts", WAVES)
@pytest.mark.parametrize("how", ["plain", "cap", "bias", "window", "prefix and window", "first", "all", "tree", "tree of all"])
def test_attention_of_a_wavefront_a_block(ctx, fmt, d, kv, group, n, lens, counts, how):
    rng = np.random.default_rng(46 + n)
    with filled(ctx, rng, 2, kv, d, 16, 16, fmt, lens) as p:
        assert takes_waves(p, n, kv * group)
        opts = {"plain": {}, "tree": dict(parents=trees(rng, 2, n), bias=True),
                "tree of all": dict(parents=trees(rng, 2, n), **HOW["all"])}.get(how) or HOW.get(how, {})
        if how in ("first", "tree"):
            p.drop(0, 1)
        p.check_attend(rows(rng, 2, n, kv * group, d), counts=counts, **options(opts, rng, n, kv * group, lens))


@pytest.mark.parametrize("fmt", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_wavefront_a_block_does_not_see_what_is_masked(ctx, fmt, d, bad):
    rng = np.random.default_rng(47)
    n, ln, kv = 64, 100, 448
    k, v = rows(rng, 1, kv, ln, d), rows(rng, 1, kv, ln, d)
    k[0, :, 95, 3] = v[0, :, 90, 7] = bad
    with Pair(ctx, 1, kv, d, 7, 16, fmt) as p:
        assert takes_waves(p, n, 2 * kv)
        p.put([ln], k, v)
        q = rows(rng, 1, n, 2 * kv, d)
        out, _ = p.attend(q)
        place = np.arange(n) + ln - n
        free, hit = place < 90, (place >= 90) & (place < 95)
        p.ref.v[0, :, 90, 7] = p.ref.k[0, :, 95, 3] = 0
        want, _, tol, _ = p.ref.attend(q, [n], d ** -0.5)
        assert (np.abs(out[0, free] - want[0, free]) <= tol[0, free]).all()
        got, ok = out[0, hit], np.ones(d, bool)
        ok[7] = False
        assert not np.isfinite(got[..., 7]).any()
        assert (np.abs(got - want[0, hit]) <= tol[0, hit])[..., ok].all()


@pytest.mark.parametrize("fmt", ["f16", "bf16"])
@pytest.mark.parametrize("d,kv,group,n,lens", [(64, 72, 4, 101, [130, 101]), (128, 100, 3, 90, [90, 200])])
def test_a_wavefront_a_block_in_place_and_replayed(ctx, fmt, d, kv, group, n, lens):
    """out in place of q gives the same bits; so does every replay of a captured call."""
    rng = np.random.default_rng(48)
    with filled(ctx, rng, 2, kv, d, 13, 16, fmt, lens) as p:
        assert takes_waves(p, n, kv * group)
        q = rows(rng, 2, n, kv * group, d)
        want, t = p.attend(q)[0], p.up(q)
        p.dev.attend(t, t, kv * group, n)
        ctx.sync()
        np.testing.assert_array_equal(t.download().reshape(q.shape), want)
        t.upload(q)
        out = p.new(q.size)
        ctx.capture_begin()
        p.dev.attend(t, out, kv * group, n)
        g = ctx.capture_end()
        for _ in range(3):
            out.upload(np.full(out.n, -3))
            g.launch()
            ctx.sync()
            np.testing.assert_array_equal(out.download().reshape(q.shape), want)
            p.attend(rows(rng, 2, 3, kv * group, d))
        g.destroy()


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("n_seqs,kv,group,n", [(65, 1, 2, 1), (130, 2, 1, 2), (300, 1, 4, 5), (600, 1, 1, 1)])
def test_attention_of_many_sequences(ctx, fmt, n_seqs, kv, group, n):
    rng = np.random.default_rng(27)
    lens = rng.integers(0, 200, n_seqs).tolist()
    lens[3] = 0
    with filled(ctx, rng, n_seqs, kv, 64, 13, 16, fmt, lens) as p:
        counts = rng.integers(0, n + 1, n_seqs).tolist()
        p.check_attend(rows(rng, n_seqs, n, kv * group, 64), counts=counts)
        p.check_attend(rows(rng, n_seqs, n, kv * group, 64), window=20)


# Lengths so different that a sequence has many shares and others none, and shares that end where a sequence does.
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kv,group,n,lens", [(1, 4, 1, [5000, 1, 0, 640, 641, 33]), (2, 8, 5, [4096, 100, 5, 2049])])
def test_attention_of_uneven_sequences(ctx, fmt, kv, group, n, lens):
    rng = np.random.default_rng(28)
    with filled(ctx, rng, len(lens), kv, 64, 320, 16, fmt, lens) as p:
        q = rows(rng, len(lens), n, kv * group, 64)
        p.check_attend(q)
        p.check_attend(q, window=700, slopes=np.float32(rng.uniform(0, 0.1, kv * group)))
        p.check_attend(q, window=64, prefix=[40] * len(lens))


@pytest.mark.parametrize("kv,n,how", [(1, 4000, {}), (29, 2000, dict(window=150)), (2, 3999, dict(prefix=[700]))])
def test_long_prompts(ctx, kv, n, how):
    """Blocks of rows that see from one to 4,000 tokens, in any order."""
    rng = np.random.default_rng(35)
    with filled(ctx, rng, 1, kv, 64, 4000 // 64 + 1, 64, "bf16", [n]) as p:
        p.check_attend(rows(rng, 1, n, kv, 64), **how)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kv,group,n,lens", [(2, 4, 1, [3000, 5]), (2, 8, 9, [900, 40]), (56, 4, 101, [130, 101])])
def test_out_in_place_of_q(ctx, fmt, kv, group, n, lens):
    rng = np.random.default_rng(36)
    with filled(ctx, rng, 2, kv, 64, 190, 16, fmt, lens) as p:
        q = rows(rng, 2, n, kv * group, 64)
        want, t = p.attend(q)[0], p.up(q)
        p.dev.attend(t, t, kv * group, n)
        ctx.sync()
        np.testing.assert_array_equal(t.download().reshape(q.shape), want)


def test_results_do_not_depend_on_chance(ctx):
    """The same call gives the same bits, whatever else ran in between."""
    rng = np.random.default_rng(23)
    with filled(ctx, rng, 2, 2, 64, 250, 16, "bf16", [4000, 1700]) as p:
        q = rows(rng, 2, 3, 8, 64)
        first = p.attend(q, window=3000)
        for _ in range(3):
            p.attend(rows(rng, 2, 9, 8, 64))
            again = p.attend(q, window=3000)
            np.testing.assert_array_equal(first[0], again[0])
            np.testing.assert_array_equal(first[1], again[1])


def test_offsets_past_32_bits(ctx):
    """A cache of 5 GiB a tensor whose last pages are in use."""
    kv, d, page = 8, 128, 256
    n_pages = 5 * 2 ** 30 // (kv * page * d * 2)
    rng = np.random.default_rng(24)
    with PagedCache(ctx, 1, kv, d, n_pages, page, 3, fmt="bf16") as dev:
        table = [n_pages - 1, 1, n_pages - 2]
        dev.set_table(table)
        dev.set_lengths([600])
        k, v, q = rows(rng, 1, 600, kv, d), rows(rng, 1, 600, kv, d), rows(rng, 1, 2, kv, d)
        ts = [ctx.tensor(x) for x in (k, v, q)]
        out = ctx.empty(q.size)
        dev.append(ts[0], ts[1], 600)
        dev.attend(ts[2], out, kv, 2)
        ctx.sync()
        ref = R.RefPaged(1, kv, d, 768, "bf16")
        ref.lens = [600]
        ref.k[0, :, :600] = R.stored(k[0].transpose(1, 0, 2), "bf16")
        ref.v[0, :, :600] = R.stored(v[0].transpose(1, 0, 2), "bf16")
        want, _, tol, _ = ref.attend(q, [2], d ** -0.5)
        assert (np.abs(out.download().reshape(q.shape) - want) <= tol).all()
        for t in (*ts, out):
            t.free()


def test_nothing_to_do(ctx):
    with Pair(ctx, 1, 1, 64, 1, 16, "f32") as p:
        t = p.new(64, fill=5)
        p.dev.append(t, t, 0)
        p.dev.attend(t, t, 1, 0)
        ctx.sync()
        assert (t.download() == 5).all()


# ---- acceptance -----------------------------------------------------------------------------

def draft(rng, n_seqs, n, vocab, agree):
    parents = np.array([[-1] + [int(rng.integers(0, i)) for i in range(1, n)] for _ in range(n_seqs)])
    tokens, choices = rng.integers(0, vocab, (n_seqs, n)), rng.integers(0, vocab, (n_seqs, n))
    for s in range(n_seqs):
        for i in range(1, n):
            if rng.random() < agree:
                choices[s, parents[s, i]] = tokens[s, i]
    return parents, tokens, choices


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,kv,n,page,lens,counts,vocab,agree", [
    (64, 4, 1, 16, [1, 20], None, 9, 1.0), (64, 2, 24, 16, [700, 30], None, 1000, 0.7),
    (128, 8, 60, 64, [100, 60], [60, 17], 3, 0.5), (64, 1, 256, 32, [300, 256], [256, 200], 2, 0.0),
    (128, 3, 33, 256, [33, 400], [0, 33], 50, 0.9), (64, 1, 9, 16, [5, 40], [9, 9], 4, 0.5)])
def test_acceptance(ctx, fmt, d, kv, n, page, lens, counts, vocab, agree):
    rng = np.random.default_rng(31 + n)
    parents, tokens, choices = draft(rng, 2, n, vocab, agree)
    with filled(ctx, rng, 2, kv, d, -(-max(lens) // page), page, fmt, lens) as p:
        path, acc, nxt = p.new(2 * n, np.int32, 7), p.new(2, np.int32, 7), p.new(2, np.int32, 7)
        before = {x: p.content(x) for x in "kv"}
        t = [p.up(x, np.int32) for x in (parents, tokens, choices)]
        p.dev.accept(*t, n, path, acc, nxt, counts=p.up(counts, np.int32))
        ctx.sync()
        for s in range(2):
            c = n if counts is None else counts[s]
            want, follow, ln = R.accept(parents[s], tokens[s], choices[s], lens[s], c)
            assert path.download().reshape(2, n)[s].tolist() == want + [-1] * (n - len(want))
            assert acc.download()[s] == len(want) and nxt.download()[s] == follow
            assert p.dev.lengths.download()[s] == ln
            base = lens[s] - c
            for x in "kv":
                got = p.content(x)[s]
                np.testing.assert_array_equal(got[:, :max(base, 0)], before[x][s][:, :max(base, 0)])
                np.testing.assert_array_equal(got[:, max(base, 0):ln] if want else got,
                                              before[x][s][:, [base + i for i in want]] if want else before[x][s])


def test_acceptance_of_a_long_path(ctx):
    """Every other row of 256 on one path: rows move past places that are read for later ones."""
    rng = np.random.default_rng(32)
    n = 256
    parents = np.array([[-1] + [max(0, (i - 1) // 2 * 2 - (0 if i % 2 else 0)) for i in range(1, n)]])
    parents[0, 2::2] = np.arange(0, n - 2, 2)
    tokens, choices = np.arange(n)[None] % 2, np.zeros((1, n), int)
    with filled(ctx, rng, 1, 2, 64, 20, 16, "bf16", [300]) as p:
        path, acc, nxt, ln = (p.new(k, np.int32) for k in (n, 1, 1, 1))
        before = p.content("k")[0]
        p.dev.accept(*[p.up(x, np.int32) for x in (parents, tokens, choices)], n, path, acc, nxt, lengths_out=ln)
        ctx.sync()
        want = R.accept(parents[0], tokens[0], choices[0], 300, n)
        assert acc.download()[0] == len(want[0]) == 128 and ln.download()[0] == want[2] == 44 + 128
        assert p.dev.lengths.download()[0] == 300
        np.testing.assert_array_equal(p.content("k")[0, :, 44:172], before[:, [44 + i for i in want[0]]])


def test_acceptance_over_missing_pages(ctx):
    """Rows whose page is not there, at either end, are not moved; nothing else is touched."""
    rng = np.random.default_rng(33)
    n = 40
    parents = np.array([[-1] + [max(0, i - 2) for i in range(1, n)]])
    tokens, choices = np.zeros((1, n), int), np.zeros((1, n), int)
    tokens[0, 1::2] = 1
    for page, entry in ((0, -1), (2, 2 ** 30)):
        with filled(ctx, rng, 1, 1, 64, 3, 16, "f32", [48]) as p:
            path, acc, nxt, ln = (p.new(k, np.int32) for k in (n, 1, 1, 1))
            before = p.content("v")[0, 0]
            p.drop(0, page, entry)
            p.dev.accept(*[p.up(x, np.int32) for x in (parents, tokens, choices)], n, path, acc, nxt, lengths_out=ln)
            ctx.sync()
            want = R.accept(parents[0], tokens[0], choices[0], 48, n)[0]
            assert acc.download()[0] == len(want)
            p.table[0, page] = 0
            there = [t for t in range(48) if t // 16 != page]
            exp, base = before.copy(), 48 - n
            for j, i in enumerate(want):
                if (base + i) // 16 != page and (base + j) // 16 != page:
                    exp[base + j] = before[base + i]
            np.testing.assert_array_equal(p.content("v")[0, 0][there], exp[there])


# ---- together -------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FORMATS)
def test_drafting_gives_what_single_tokens_give(ctx, fmt):
    """A model of one layer (fixed projections of an id's embedding) decodes token by token, and again
    by drafted trees that hold the right continuation among wrong ones: the same ids, and the same
    keys and values in the cache."""
    rng = np.random.default_rng(41)
    vocab, kv, heads, d, steps = 50, 2, 4, 64, 24
    emb = {x: rows(rng, vocab, (heads if x == "q" else kv) * d) for x in "qkv"}
    head = rows(rng, heads * d, vocab)
    inv = freqs(d)

    def step(p, ids, base, parents=None):
        """Appends the ids as the tokens base .., attends, and gives the id chosen behind each."""
        n = len(ids)
        q, k, v = (p.up(emb[x][ids]) for x in "qkv")
        qo, out = p.new(n * heads * d), p.new(n * heads * d)
        p.dev.set_lengths([base + n])
        off = None if parents is None else p.up(R.depths(parents, n)[0], np.int32)
        par = None if parents is None else p.up(parents, np.int32)
        f = p.up(inv)
        p.dev.append(k, v, n, q=q, q_out=qo, n_heads=heads, inv_freq=f, offsets=off)
        p.dev.attend(qo, out, heads, n, parents=par)
        ctx.sync()
        return (out.download().reshape(n, -1).astype(np.float64) @ head).argmax(1)

    prompt = [3, 14, 15, 9, 26]
    with Pair(ctx, 1, kv, d, 4, 16, fmt) as a, Pair(ctx, 1, kv, d, 4, 16, fmt, seed=1) as b:
        ids = prompt + [int(step(a, prompt, 0)[-1])]
        while len(ids) < len(prompt) + steps:
            ids.append(int(step(a, [ids[-1]], len(ids) - 1)[0]))
        got = prompt + [int(step(b, prompt, 0)[-1])]
        calls = 0
        while len(got) < len(ids):
            # the settled token, two right ones in a row, wrong ones beside each
            right = (ids[len(got):] + [0, 0])[:2]
            tree = [got[-1], (right[0] + 1) % vocab, right[0], (right[1] + 1) % vocab, right[1], right[0]]
            parents = [-1, 0, 0, 2, 2, 1]
            pick = step(b, tree, len(got) - 1, parents)
            path, acc, nxt = (b.new(k, np.int32) for k in (6, 1, 1))
            b.dev.accept(b.up(parents, np.int32), b.up(tree, np.int32), b.up(pick, np.int32), 6, path, acc, nxt)
            ctx.sync()
            m = acc.download()[0]
            taken = path.download()[:m]
            assert b.dev.lengths.download()[0] == len(got) - 1 + m
            got += [tree[i] for i in taken[1:]] + [int(nxt.download()[0])]
            calls += 1
        assert got[:len(ids)] == ids and calls <= steps // 2
        held = len(ids) - 1
        for x in "kv":
            np.testing.assert_array_equal(a.content(x)[..., :held, :], b.content(x)[..., :held, :])


def test_captured_step_replays(ctx):
    """A step of append, attention and acceptance is recorded once and replayed on other rows, with the
    program's own calls in between; every replay is compared with the calls made one by one."""
    rng = np.random.default_rng(42)
    n, heads, kv, d = 12, 8, 2, 64
    parents = np.array([[-1] + [int(rng.integers(0, i)) for i in range(1, n)] for _ in range(2)])
    off = np.array([R.depths(x, n)[0] for x in parents])
    with filled(ctx, rng, 2, kv, d, 40, 16, "bf16", [600, 300]) as p:
        ins = {x: p.new(2 * n * (heads if x == "q" else kv) * d) for x in "qkv"}
        ids = {x: p.new(2 * n, np.int32) for x in ("tokens", "choices")}
        outs = {x: p.new(2 * n * heads * d) for x in ("q", "out")}
        ints = {x: p.new(k, np.int32) for x, k in (("path", 2 * n), ("acc", 2), ("next", 2), ("len", 2))}
        par, offs, inv = p.up(parents, np.int32), p.up(off, np.int32), p.up(freqs(d))
        lse = p.new(2 * heads * n)

        def step():
            p.dev.append(ins["k"], ins["v"], n, q=ins["q"], q_out=outs["q"], n_heads=heads, inv_freq=inv,
                         offsets=offs)
            p.dev.attend(outs["q"], outs["out"], heads, n, lse=lse, parents=par)
            p.dev.accept(par, ids["tokens"], ids["choices"], n, ints["path"], ints["acc"], ints["next"],
                         lengths_out=ints["len"])

        def state():
            ctx.sync()
            return [t.download() for t in (*outs.values(), lse, *ints.values())] + [p.content(x) for x in "kv"]

        def load(seed):
            r = np.random.default_rng(seed)
            for x, t in ins.items():
                t.upload(rows(r, t.n))
            _, tok, pick = draft(r, 2, n, 30, 0.6)
            ids["tokens"].upload(tok)
            ids["choices"].upload(pick)
            p.dev.set_lengths([600 - seed, 300 + seed])

        load(0)
        step()
        ctx.sync()
        ctx.capture_begin()
        step()
        g = ctx.capture_end()
        for seed in range(1, 5):
            load(seed)
            g.launch()
            got = state()
            p.attend(rows(rng, 2, 3, heads, d))  # the program's own work
            load(seed)
            step()
            for a, b in zip(got, state()):
                np.testing.assert_array_equal(a, b)
        g.destroy()


def test_a_long_call_captured_before_it_ever_ran(ctx):
    """A fresh context has no workspace: a captured call runs without one, and eager calls later do not
    disturb the replay."""
    rng = np.random.default_rng(43)
    with Context("any") as own, filled(own, rng, 1, 1, 64, 400, 16, "f16", [6000]) as p:
        q, out = rows(rng, 1, 2, 4, 64), p.new(2 * 4 * 64, fill=-3)
        dq = p.up(q)
        own.capture_begin()
        p.dev.attend(dq, out, 4, 2)
        g = own.capture_end()
        want, _, tol, _ = p.ref.attend(q, [2], 0.125)
        for _ in range(3):
            out.upload(np.full(out.n, -3))
            g.launch()
            own.sync()
            assert (np.abs(out.download().reshape(q.shape) - want) <= tol).all()
            p.check_attend(rows(rng, 1, 5, 4, 64))
        g.destroy()


@pytest.mark.parametrize("fmt", FORMATS)
def test_two_graphs_share_a_workspace_that_grows(ctx, fmt):
    """Two captured calls whose tokens are shared out, and an eager one that needs more workspace than both: replays of
    the two, in turn and one behind the other, give the eager calls' bits."""
    rng = np.random.default_rng(54)
    with Context("any") as own, filled(own, rng, 2, 2, 64, 190, 16, fmt, [3000, 700]) as p:
        calls = []
        for n in (1, 3):
            q = rows(rng, 2, n, 4, 64)
            want, t, out = p.attend(q)[0], p.up(q), p.new(q.size)
            own.capture_begin()
            p.dev.attend(t, out, 4, n)
            calls.append((own.capture_end(), out, want))
        size = C.c_uint64()
        where = C.c_void_p()
        check(lib().shp_workspace_info(own.handle, C.byref(where), C.byref(size)), "shp_workspace_info")
        before = where.value
        check(lib().shp_reserve_workspace(own.handle, 2 * size.value), "shp_reserve_workspace")
        check(lib().shp_workspace_info(own.handle, C.byref(where), C.byref(size)), "shp_workspace_info")
        assert before and where.value != before
        for _ in range(3):
            p.attend(rows(rng, 2, 30, 4, 64))
            for g, out, _ in calls:
                out.upload(np.full(out.n, -3))
                g.launch()
            own.sync()
            for _, out, want in calls:
                np.testing.assert_array_equal(out.download().reshape(want.shape), want)
        for g, _, _ in calls:
            g.destroy()


def test_calls_on_another_stream(ctx):
    rng = np.random.default_rng(44)
    with Context("any") as other, Context("any") as own, filled(own, rng, 2, 2, 64, 20, 16, "f32", [300, 77]) as p:
        q = rows(rng, 2, 4, 8, 64)
        want = p.attend(q)
        stream = lib().shp_get_stream(other.handle)
        assert stream and stream != lib().shp_get_stream(own.handle)
        check(lib().shp_set_stream(own.handle, stream), "shp_set_stream")
        got = p.attend(q)
        check(lib().shp_set_stream(own.handle, None), "shp_set_stream")
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])


def test_timing_names_the_calls(ctx):
    rng = np.random.default_rng(45)
    with Context("any") as own, filled(own, rng, 1, 1, 64, 4, 16, "f32", [40]) as p:
        own.timing(True)
        p.attend(rows(rng, 1, 1, 2, 64))
        t = p.up(rows(rng, 1, 1, 1, 64))
        p.dev.append(t, t, 1)
        i = [p.new(1, np.int32) for _ in range(6)]
        p.dev.accept(*i[:3], 1, *i[3:])
        assert set(own.timing_report()) == {"paged_attend", "paged_append", "paged_accept"}


def test_closed_caches_are_refused(ctx):
    p = Pair(ctx, 1, 1, 64, 1, 16, "f32")
    t = p.new(64)
    p.dev.close()
    with pytest.raises(ShpError, match="null array"):
        p.dev.attend(t, t, 1, 1)
    p.__exit__()
