"""Token log probabilities, entropies and top alternatives on the GPU against numpy in 64 bits.

Bounds: x - m is rounded once (2^-24 of its size), the sums of exp(x - m) over a row are off by
under 64 roundings relative to themselves plus 2^-23 of |x - m| per weight, which stays under 2^-23 *
max over weights of exp(d) |d| < 2^-23; logf and the last differences add roundings of their own size."""
import ctypes as C

import numpy as np
import pytest

import cache8_ref as R
from conftest import assert_close
from spirv_inference_amd import Context, DeviceTensor, ShpError
from spirv_inference_amd._lib import lib
from spirv_inference_amd.models import Llama

pytestmark = pytest.mark.gpu


def run(ctx, x, targets, top, stride=None, offset=0, parts=("lp", "ent")):
    rows, vocab = x.shape
    stride = vocab if stride is None else stride
    flat = np.full(offset + rows * stride, np.nan, np.float32)  # what lies between rows
    np.lib.stride_tricks.as_strided(flat[offset:], x.shape, (4 * stride, 4))[:] = x
    t = ctx.tensor(flat)
    logits = DeviceTensor(ctx, flat.size - offset, ptr=t.ptr + 4 * offset, owned=False)
    tg = ctx.tensor(targets, np.int32)
    lp, ent = ctx.tensor(np.full(rows, 7)), ctx.tensor(np.full(rows, 7))
    ids, tops = ctx.tensor(np.full(max(1, rows * top), 7), np.int32), ctx.empty(max(1, rows * top))
    ctx.token_logprobs(logits, tg if "lp" in parts else None, lp if "lp" in parts else None,
                       ent if "ent" in parts else None, ids if top else None,
                       tops if top else None, rows, vocab, top, row_stride=stride)
    ctx.sync()
    out = (lp.download(), ent.download(), ids.download()[:rows * top].reshape(rows, top),
           tops.download()[:rows * top].reshape(rows, top))
    for b in (t, tg, lp, ent, ids, tops):
        b.free()
    return out


def check(got, x, targets, top):
    want = R.logprobs(x, targets, top)
    np.testing.assert_array_equal(got[2], want[2])
    for i in (0, 1, 3):
        g, w = got[i].astype(np.float64), want[i]
        np.testing.assert_array_equal(np.isnan(g), np.isnan(w))
        np.testing.assert_array_equal(g == -np.inf, w == -np.inf)
        f = np.isfinite(w)
        assert (np.abs(g[f] - w[f]) <= (64 + 8) * 2.0 ** -24 + 4 * 2.0 ** -24 * np.abs(w[f])).all(), \
            i


@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 1, 0), (3, 2, 2), (5, 63, 5), (2, 64, 64), (7, 65, 64), (4, 1000, 20),
    (3, 4097, 1), (2, 32000, 5), (1, 32768, 64), (2, 32769, 64), (3, 100003, 33), (1, 300000, 20),
    (600, 777, 3), (256, 8192, 20), (257, 8193, 64), (255, 33000, 5), (300, 30001, 20)])
@pytest.mark.parametrize("std", [0.1, 4.0])
def test_logprobs(ctx, rows, vocab, top, std):
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((rows, vocab)) * std).astype(np.float32)
    targets = rng.integers(0, vocab, rows)
    check(run(ctx, x, targets, top), x, targets, top)


# so many rows that each takes a workgroup of 128, with one chunk of logits or several
@pytest.mark.parametrize("rows,vocab,top", [
    (1024, 4096, 64), (1025, 4097, 5), (1100, 300, 64), (1030, 12345, 20), (1500, 1, 1)])
def test_logprobs_of_many_rows(ctx, rows, vocab, top):
    rng = np.random.default_rng(rows)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    targets = rng.integers(0, vocab, rows)
    check(run(ctx, x, targets, top), x, targets, top)


# so many parts of a row that the best of all do not fit into the memory of the workgroup that joins them
@pytest.mark.parametrize("kind", ["normal", "few", "equal"])
def test_logprobs_of_more_than_a_million_logits(ctx, kind):
    rng = np.random.default_rng(14)
    shape = (2, 1_100_003)
    x = {"normal": rng.standard_normal(shape), "few": rng.integers(0, 50000, shape) * 1e-4,
         "equal": np.full(shape, -2.5)}[kind].astype(np.float32)
    check(run(ctx, x, [7, 1_100_002], 64), x, [7, 1_100_002], 64)


@pytest.mark.parametrize("vocab", [200, 32000, 70001])
@pytest.mark.parametrize("kind", ["equal", "few", "ascending", "descending", "zeros"])
def test_ties_go_to_the_lowest_id(ctx, vocab, kind):
    rng = np.random.default_rng(5)
    x = {"equal": np.full((2, vocab), 0.25), "few": rng.integers(0, 3, (2, vocab)),
         "ascending": np.tile(np.arange(vocab) * 1e-3, (2, 1)),
         "descending": np.tile(np.arange(vocab)[::-1] * 1e-3, (2, 1)),
         "zeros": rng.choice([0.0, -0.0], (2, vocab))}[kind].astype(np.float32)
    check(run(ctx, x, [0, vocab - 1], 64), x, [0, vocab - 1], 64)


def test_plateaus_of_many_rows(ctx):
    test_plateaus_and_chunks_of_one_kind(ctx, 1026, 13000)


@pytest.mark.parametrize("rows,vocab", [(2, 40000), (300, 20000)])
def test_plateaus_and_chunks_of_one_kind(ctx, rows, vocab):
    """Rows in which the best lie in one place, rise, tie, or are all that is allowed: the ways in
    which a row's candidates can be too many or too few."""
    rng = np.random.default_rng(12)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    kinds = [lambda r: np.sort(r), lambda r: np.sort(r)[::-1], lambda r: np.round(r),
             lambda r: np.where(np.arange(vocab) % 977 == 5, r, -np.inf),
             lambda r: np.where(np.arange(vocab) < 3, r, -np.inf),
             lambda r: np.where(np.arange(vocab) > vocab - 40, r, np.nan),
             lambda r: np.where((np.arange(vocab) >= 9000) & (np.arange(vocab) < 9600), 50 + r, r),
             lambda r: np.where(np.arange(vocab) // 4 % 256 == 7, 50 + r, r),
             lambda r: np.minimum(r, 0.5)]
    for i in range(rows):
        x[i] = kinds[i % len(kinds)](x[i])
    t = rng.integers(0, vocab, rows)
    for top in (1, 20, 64):
        check(run(ctx, x, t, top), x, t, top)


@pytest.mark.parametrize("vocab", [50, 40000])
def test_infinities_and_nan(ctx, vocab):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((9, vocab)).astype(np.float32)
    x[0, rng.random(vocab) < 0.5] = -np.inf
    x[1] = -np.inf
    x[1, vocab - 3] = 2.0                       # one token can be
    x[2] = -np.inf                              # none
    x[3, 7] = np.nan
    x[4, 9] = np.inf
    x[5, :] = np.nan
    x[6, :vocab // 2] = -3.4028235e38           # the lowest finite number
    x[7, :] = -3.4028235e38
    x[8, ::3] = 3.4028235e38
    t = [int(np.argmin(x[0])), vocab - 3, 0, 0, 0, 0, 0, 1, 0]
    check(run(ctx, x, t, 10), x, t, 10)


# What is masked: a part of its own for the join, whole chunks at either end, the logits of one
# wavefront of a chunk, all but one logit.
MASKED = [(1, 40000, lambda i: i >= 32768), (3, 100000, lambda i: i < 70000),
          (1, 32000, lambda i: i // 4 % 1024 // 64 == 5), (300, 20000, lambda i: i >= 9000),
          (300, 20000, lambda i: i < 9000), (300, 20000, lambda i: i // 4 % 256 // 64 == 2),
          (1030, 9000, lambda i: i >= 4100), (1030, 9000, lambda i: i < 4100),
          (2, 50, lambda i: i != 17), (2, 40000, lambda i: i != 35000)]


@pytest.mark.parametrize("case", range(len(MASKED)))
@pytest.mark.parametrize("fill", [-3.4028235e38, -1e38, -2e9])
def test_masks_of_very_negative_numbers(ctx, case, fill):
    """Finite logits whose weight is zero: parts of a row that hold nothing else add nothing."""
    rows, vocab, masked = MASKED[case]
    rng = np.random.default_rng(case)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    x[:, masked(np.arange(vocab))] = fill
    t = rng.integers(0, vocab, rows)
    for top in (0, 5):
        check(run(ctx, x, t, top), x, t, top)


@pytest.mark.parametrize("rows,vocab", [(2, 40000), (300, 20000)])
def test_a_nan_among_very_negative_numbers_shows(ctx, rows, vocab):
    rng = np.random.default_rng(13)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    x[:, 9000:] = -3.4028235e38
    x[::2, vocab - 5] = np.nan
    x[1, 9000:] = -np.inf
    t = rng.integers(0, vocab, rows)
    check(run(ctx, x, t, 3), x, t, 3)


def test_large_common_offsets_cancel(ctx):
    rng = np.random.default_rng(7)
    x = (rng.integers(-40, 40, (4, 5000)) * 0.25 + np.array([[1e5], [-1e5], [0], [3e6]])).astype(np.float32)
    t = rng.integers(0, 5000, 4)
    check(run(ctx, x, t, 8), x, t, 8)


def test_ids_outside_the_vocabulary_cannot_be(ctx):
    x = np.zeros((4, 10), np.float32)
    t = [-1, 10, -2147483648, 2147483647]
    got = run(ctx, x, t, 2)
    check(got, x, t, 2)
    assert (got[0] == -np.inf).all()


@pytest.mark.parametrize("offset,stride", [(0, 1003), (1, 1001), (2, 1030), (3, 1000)])
def test_strides_and_alignment(ctx, offset, stride):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((5, 1000)).astype(np.float32)
    t = rng.integers(0, 1000, 5)
    check(run(ctx, x, t, 7, stride=stride, offset=offset), x, t, 7)


def test_parts_that_are_not_asked_for(ctx):
    rng = np.random.default_rng(9)
    x = rng.standard_normal((3, 500)).astype(np.float32)
    got = run(ctx, x, [1, 2, 3], 4, parts=())
    want = R.logprobs(x, [1, 2, 3], 4)
    assert (got[0] == 7).all() and (got[1] == 7).all()
    np.testing.assert_array_equal(got[2], want[2])
    got = run(ctx, x, [1, 2, 3], 0, parts=("ent",))
    assert (got[0] == 7).all() and np.allclose(got[1], want[1], atol=1e-5)


def test_offsets_past_31_bits(ctx):
    """Rows whose stride takes the last of them past 2^32 bytes."""
    rows, vocab, stride = 3, 1000, 600_000_000
    big = ctx.empty((rows - 1) * stride + vocab)
    rng = np.random.default_rng(10)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    for r in range(rows):
        DeviceTensor(ctx, vocab, ptr=big.ptr + 4 * r * stride, owned=False).upload(x[r])
    tg, lp = ctx.tensor([5, 6, 7], np.int32), ctx.empty(rows)
    ids, tops = ctx.empty(rows * 3, np.int32), ctx.empty(rows * 3)
    ctx.token_logprobs(big, tg, lp, None, ids, tops, rows, vocab, 3, row_stride=stride)
    ctx.sync()
    want = R.logprobs(x, [5, 6, 7], 3)
    np.testing.assert_array_equal(ids.download().reshape(rows, 3), want[2])
    assert np.allclose(lp.download(), want[0], atol=1e-5)
    for t in (big, tg, lp, ids, tops):
        t.free()


def test_captured_calls(ctx):
    """Replays follow the logits; a capture that would have to grow the workspace is refused."""
    rng = np.random.default_rng(11)
    rows, vocab, top = 2, 90000, 6
    with Context("any") as own:
        x, tg = own.empty(rows * vocab), own.tensor([3, 4], np.int32)
        lp, ent = own.empty(rows), own.empty(rows)
        ids, tops = own.empty(rows * top, np.int32), own.empty(rows * top)
        args = (x, tg, lp, ent, ids, tops, rows, vocab, top)
        own.capture_begin()
        with pytest.raises(ShpError, match="run the call once before"):
            own.token_logprobs(*args)
        own.capture_end().destroy()
        own.token_logprobs(*args)
        own.sync()
        own.capture_begin()
        own.token_logprobs(*args)
        g = own.capture_end()
        for _ in range(3):
            v = rng.standard_normal((rows, vocab)).astype(np.float32)
            x.upload(v)
            g.launch()
            own.sync()
            check((lp.download(), ent.download(), ids.download().reshape(rows, top),
                   tops.download().reshape(rows, top)), v, [3, 4], top)
        g.destroy()


def test_the_workspace_grows_seldom():
    """Outgrown buffers live as long as their context (a graph may hold them): calls that grow one row
    at a time leave few of them, smaller together than the one in use."""
    vocab = 70001
    with Context("any") as own:
        x, tg, lp = own.empty(255 * vocab), own.tensor(np.zeros(255), np.int32), own.empty(255)
        seen = {}
        for rows in range(1, 256):
            own.token_logprobs(x, tg, lp, None, None, None, rows, vocab)
            ptr, size = C.c_void_p(), C.c_uint64()
            assert lib().shp_workspace_info(own.handle, C.byref(ptr), C.byref(size)) == 0
            seen[ptr.value] = size.value
        own.sync()
        sizes = sorted(seen.values())
        assert sum(sizes[:-1]) <= sizes[-1] and len(sizes) < 10, sizes


# ---- the decoder scores a text -----------------------------------------------------------------

SMALL = dict(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=1000,
             max_seq=200)


@pytest.mark.parametrize("engine", ["persistent", "graph", "kernels"])
@pytest.mark.parametrize("n,top", [(1, 3), (2, 0), (3, 64), (40, 5), (150, 1)])
def test_scores_are_those_of_the_token_steps(ctx, engine, n, top):
    """The prompt pass adds up its products in another order than the token steps, so the two are
    held to each other by the gate of the decoder's own tests (1e-4 + 1e-4 of the value)."""
    ids = [int(t) for t in np.random.default_rng(n).integers(3, SMALL["vocab"], n)]
    with Llama(ctx, seed=5, **SMALL) as lm:
        lm.set_engine(engine)
        lp, ent, tid, tlp = lm.score(ids, top)
        on = lm.decode(4) or lm.tokens()[n - 1:n + 4]
        lm.reset()
        x = []
        for t in ids:
            lm.step(t)
            ctx.sync()
            x.append(lm.logits())
        lm.decode(4)
        assert lm.tokens()[n - 1:n + 4] == on
    x = np.array(x)
    want = R.logprobs(x, ids[1:] + [0], 0)
    assert lp.shape == (n - 1,) and tid.shape == tlp.shape == (n, top)
    assert_close(lp, want[0][:-1], what="logprob")
    assert_close(ent, want[1], what="entropy")
    full = x.astype(np.float64) - x.max(1, keepdims=True)
    full -= np.log(np.exp(full).sum(1, keepdims=True))
    for i in range(n):
        assert_close(tlp[i], full[i, tid[i]], what="top")
        assert len(set(tid[i])) == top and (np.diff(tlp[i]) <= 0).all()
        if top:
            rest = np.delete(full[i], tid[i]).max()
            assert rest <= tlp[i, -1] + 1e-4 + 1e-4 * abs(rest)


def test_scores_refuse_bad_texts(ctx):
    with Llama(ctx, seed=5, **SMALL) as lm:
        for ids, top in (([], 0), ([3, 1000], 0), ([3, -1], 0), ([3] * 201, 0), ([3], 65), ([3], -1)):
            with pytest.raises(ShpError, match="shp_llama_score"):
                lm.score(ids, top)
        lm.score([3] * 200, 1)
