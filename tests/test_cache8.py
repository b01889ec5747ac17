"""Refusals of the 8-bit cache's and the log probabilities' entry points: arguments are checked
before the context, so all of them show without a device."""
import ctypes as C

import numpy as np
import pytest

import cache8_ref as R
from spirv_inference_amd import Cache8, _lib, cache8
from spirv_inference_amd._lib import (Cache8AppendArgs, Cache8AttendArgs, Cache8EvictArgs,
                                      Cache8Struct, Cache8WeightsArgs, LogprobsArgs)

P = 0x1000  # an aligned address that no call gets to use


def cache(**over):
    f = dict(k=P, v=P + 0x1000, k_scale=P + 0x2000, v_scale=P + 0x3000, lengths=P + 0x4000,
             n_seqs=2, n_kv_heads=2, head_dim=64, capacity=128, block=64, format=0)
    f.update(over)
    return Cache8Struct(*(f[n] for n, _ in Cache8Struct._fields_))


def args(cls, **over):
    f = {n: (P if t is C.c_void_p else 64) for n, t in cls._fields_}
    f.update({n: v for n, v in dict(counts=0, n=1, n_heads=4, scale=0.125, rows=2, vocab=64,
                                    row_stride=64, n_top=4, keep=64, recent=8,
                                    weights=P, kept=P, dst_weights=0).items() if n in f})
    f.update(over)
    return cls(*(f[n] for n, _ in cls._fields_))


def call(name, *structs):
    rc = getattr(_lib.lib(), name)(None, *[C.byref(s) if isinstance(s, C.Structure) else s
                                           for s in structs])
    return rc, _lib.lib().shp_last_error().decode()


CALLS = {"shp_cache8_append": Cache8AppendArgs, "shp_cache8_attend": Cache8AttendArgs,
         "shp_cache8_weights": Cache8WeightsArgs}


@pytest.mark.parametrize("name", CALLS)
def test_good_arguments_get_as_far_as_the_context(name):
    assert call(name, cache(), args(CALLS[name])) == (_lib.SHP_ERR_INVALID, f"{name}: null ctx")
    assert call(name, cache(head_dim=128, block=128, format=1), args(CALLS[name], n=0))[1] \
        == f"{name}: null ctx"


def test_good_arguments_of_the_other_calls():
    other = cache(k=P + 0x5000, v=P + 0x6000, k_scale=P + 0x7000, v_scale=P + 0x8000,
                  lengths=P + 0x9000, capacity=64)
    for name, a in (("shp_cache8_read", (cache(), 5, P, P)),
                    ("shp_cache8_read", (cache(), 0, None, None)),
                    ("shp_cache8_evict", (cache(), other, args(Cache8EvictArgs))),
                    ("shp_token_logprobs", (args(LogprobsArgs),)),
                    ("shp_token_logprobs", (args(LogprobsArgs, rows=0),)),
                    ("shp_token_logprobs", (args(LogprobsArgs, n_top=0, top_ids=0, top_logprobs=0,
                                                 targets=0, logprob=0),))):
        assert call(name, *a) == (_lib.SHP_ERR_INVALID, f"{name}: null ctx")


@pytest.mark.parametrize("over,code,what", [
    (dict(k=0), _lib.SHP_ERR_INVALID, "null array"),
    (dict(v=0), _lib.SHP_ERR_INVALID, "null array"),
    (dict(k_scale=0), _lib.SHP_ERR_INVALID, "null array"),
    (dict(v_scale=0), _lib.SHP_ERR_INVALID, "null array"),
    (dict(lengths=0), _lib.SHP_ERR_INVALID, "null array"),
    (dict(format=2), _lib.SHP_ERR_UNSUPPORTED, "format"),
    (dict(format=-1), _lib.SHP_ERR_UNSUPPORTED, "format"),
    (dict(head_dim=96), _lib.SHP_ERR_UNSUPPORTED, "head_dim"),
    (dict(head_dim=0), _lib.SHP_ERR_UNSUPPORTED, "head_dim"),
    (dict(block=8), _lib.SHP_ERR_UNSUPPORTED, "block"),
    (dict(block=48), _lib.SHP_ERR_UNSUPPORTED, "block"),
    (dict(block=256), _lib.SHP_ERR_UNSUPPORTED, "block"),
    (dict(block=0), _lib.SHP_ERR_UNSUPPORTED, "block"),
    (dict(n_seqs=0), _lib.SHP_ERR_SHAPE, "n_seqs"),
    (dict(n_kv_heads=-1), _lib.SHP_ERR_SHAPE, "n_seqs"),
    (dict(n_seqs=40000), _lib.SHP_ERR_SHAPE, "n_seqs"),
    (dict(capacity=0), _lib.SHP_ERR_SHAPE, "capacity"),
    (dict(capacity=96), _lib.SHP_ERR_SHAPE, "capacity"),
    (dict(capacity=192, block=128), _lib.SHP_ERR_SHAPE, "capacity"),
    (dict(capacity=(1 << 22) + 64), _lib.SHP_ERR_SHAPE, "capacity"),
    (dict(k=P + 8), _lib.SHP_ERR_INVALID, "16-byte"),
    (dict(v=P + 4), _lib.SHP_ERR_INVALID, "16-byte"),
    (dict(k_scale=P + 2), _lib.SHP_ERR_INVALID, "4-byte"),
    (dict(lengths=P + 1), _lib.SHP_ERR_INVALID, "4-byte")])
def test_bad_caches_are_refused(over, code, what):
    c = cache(**over)
    good = cache(k=P + 0x5000, v=P + 0x6000, k_scale=P + 0x7000, v_scale=P + 0x8000,
                 lengths=P + 0x9000)
    for name, rest in (*((n, (args(t),)) for n, t in CALLS.items()),
                       ("shp_cache8_read", (1, P, P))):
        rc, msg = call(name, c, *rest)
        assert rc == code and what in msg and msg.startswith(name), (name, rc, msg)
    for pair in ((c, good), (good, c)):
        rc, msg = call("shp_cache8_evict", *pair, args(Cache8EvictArgs))
        assert rc == code and what in msg, msg


@pytest.mark.parametrize("name,over,what", [
    ("shp_cache8_append", dict(n=-1), "n < 0"),
    ("shp_cache8_append", dict(k=0), "null k"),
    ("shp_cache8_append", dict(v=0), "null v"),
    ("shp_cache8_append", dict(k=P + 4), "k rows"),
    ("shp_cache8_append", dict(v_row=66), "v rows"),
    ("shp_cache8_append", dict(k_head=1), "k rows"),
    ("shp_cache8_attend", dict(n=-1), "n < 0"),
    ("shp_cache8_attend", dict(q=0), "null q"),
    ("shp_cache8_attend", dict(out=0), "null out"),
    ("shp_cache8_attend", dict(q=P + 8), "q rows"),
    ("shp_cache8_attend", dict(o_seq=2), "out rows"),
    ("shp_cache8_attend", dict(n_heads=3), "n_heads"),
    ("shp_cache8_attend", dict(n_heads=0), "n_heads"),
    ("shp_cache8_attend", dict(scale=float("nan")), "scale"),
    ("shp_cache8_attend", dict(scale=float("inf")), "scale"),
    ("shp_cache8_attend", dict(n=300000), "500000"),
    ("shp_cache8_weights", dict(n=-1), "n < 0"),
    ("shp_cache8_weights", dict(q=0), "null q"),
    ("shp_cache8_weights", dict(lse=0), "null lse"),
    ("shp_cache8_weights", dict(acc_out=0), "null lse or acc_out"),
    ("shp_cache8_weights", dict(n_heads=5), "n_heads")])
def test_bad_arguments_are_refused(name, over, what):
    rc, msg = call(name, cache(), args(CALLS[name], **over))
    assert rc != 0 and what in msg and "ctx" not in msg, (rc, msg)


@pytest.mark.parametrize("name,cls,fields", [
    ("shp_cache8_append", Cache8AppendArgs, ["counts"]),
    ("shp_cache8_attend", Cache8AttendArgs, ["counts", "lse"]),
    ("shp_cache8_weights", Cache8WeightsArgs, ["counts", "lse", "acc_in", "acc_out"]),
    ("shp_cache8_evict", Cache8EvictArgs, ["weights", "kept", "dst_weights"]),
    ("shp_token_logprobs", LogprobsArgs, ["targets", "logprob", "entropy", "top_ids", "top_logprobs"])])
def test_arrays_of_numbers_that_are_not_aligned_are_refused(name, cls, fields):
    far = cache(k=P + 0x50000, v=P + 0x60000, k_scale=P + 0x70000, v_scale=P + 0x80000,
                lengths=P + 0x90000)
    first = () if cls is LogprobsArgs else (cache(), far) if cls is Cache8EvictArgs else (cache(),)
    for f in fields:
        for off in (1, 2, 3):
            rc, msg = call(name, *first, args(cls, **{f: 0x100000 + off}))
            assert rc == _lib.SHP_ERR_INVALID and "4-byte aligned" in msg, (f, msg)
        rc, msg = call(name, *first, args(cls, **{f: 0x100004}))
        assert msg == f"{name}: null ctx"


def test_null_structures_are_refused():
    for name in (*CALLS, "shp_cache8_evict"):
        rest = (cache(k=P + 64),) if name == "shp_cache8_evict" else ()
        assert call(name, None, *rest, None)[1] == f"{name}: null cache"
        assert call(name, cache(), *rest, None)[1].startswith(name)
    assert call("shp_token_logprobs", None)[1] == "shp_token_logprobs: null arguments"


def test_bad_reads_and_evictions_are_refused():
    for n, k in ((-1, P), (129, P), (4, P + 4)):
        rc, msg = call("shp_cache8_read", cache(), n, k, P)
        assert rc != 0 and "ctx" not in msg, msg
    far = dict(k=P + 0x5000, v=P + 0x6000, k_scale=P + 0x7000, v_scale=P + 0x8000,
               lengths=P + 0x9000)
    for dst, over, what in (
            (dict(), dict(), "share"),
            ({**far, "lengths": P + 0x4000}, dict(), "share"),
            ({**far, "block": 32}, dict(), "differ"),
            ({**far, "format": 1}, dict(), "differ"),
            ({**far, "n_seqs": 1}, dict(), "differ"),
            ({**far, "head_dim": 128}, dict(), "differ"),
            (far, dict(keep=0), "keep"),
            (far, dict(keep=129), "keep"),
            (far, dict(recent=65), "recent"),
            (far, dict(recent=-1), "recent"),
            (far, dict(weights=0), "null"),
            (far, dict(kept=0), "null"),
            (far, dict(dst_weights=P), "dst_weights")):
        rc, msg = call("shp_cache8_evict", cache(), cache(**dst), args(Cache8EvictArgs, **over))
        assert rc != 0 and what in msg, (dst, over, msg)


def test_evictions_into_their_own_arrays_are_refused():
    """By the arrays' sizes, not only where they begin.  The context is memory that a refused call
    does not touch: calls without an overlap get as far as asking for its device."""
    ctx = C.create_string_buffer(1 << 16)
    # 2 x 2 heads of 128 (src) and 64 (dst) tokens x 64, blocks of 64, 64 kept
    size = dict(k=32768, v=32768, k_scale=32, v_scale=32, lengths=8, weights=2048)
    dsize = dict(k=16384, v=16384, k_scale=16, v_scale=16, lengths=8, kept=1024, dst_weights=1024)
    at, where = 1 << 20, {}
    for n, b in (*(("s." + n, b) for n, b in size.items()), *(("d." + n, b) for n, b in dsize.items())):
        where[n] = at
        at += -(-b // 16) * 16

    def evict(**moved):
        w = {**where, **{n.replace("_", ".", 1): p for n, p in moved.items()}}
        names = ("k", "v", "k_scale", "v_scale", "lengths")
        s, d = (cache(capacity=c, **{n: w[f"{o}.{n}"] for n in names}) for o, c in (("s", 128), ("d", 64)))
        rc = _lib.lib().shp_cache8_evict(ctx, C.byref(s), C.byref(d), C.byref(args(
            Cache8EvictArgs, weights=w["s.weights"], kept=w["d.kept"], dst_weights=w["d.dst_weights"])))
        return "shares memory" in _lib.lib().shp_last_error().decode(), rc

    for n, b in dsize.items():
        for o, ob in (*(("s." + m, x) for m, x in size.items()), *(("d." + m, x) for m, x in dsize.items())):
            if o == "d." + n:
                continue
            step = 16 if n in "kv" else 4
            for p in (where[o] + ob - step, where[o] - b + step):  # the last bytes, the first bytes
                p = p // step * step
                overlap, rc = evict(**{"d_" + n: p})
                assert overlap and rc == _lib.SHP_ERR_INVALID, (n, o)
    far = 1 << 22
    for n in dsize:
        # next to each other is not an overlap
        assert not evict(**{"d_" + n: far})[0] and not evict(**{"d_" + n: at})[0], n
    assert not evict(d_dst_weights=0)[0]


@pytest.mark.parametrize("over,what", [
    (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(logits=0), "logits"),
    (dict(logits=P + 2), "logits"), (dict(row_stride=63), "row_stride"),
    (dict(n_top=-1), "n_top"), (dict(n_top=65, vocab=100, row_stride=100), "n_top"),
    (dict(n_top=9, vocab=8), "n_top"), (dict(targets=0), "targets"), (dict(logprob=0), "targets"),
    (dict(top_ids=0), "top_ids"), (dict(top_logprobs=0), "top_ids"),
    (dict(rows=16000001), "16000000"), (dict(vocab=(1 << 30) + 1, row_stride=1 << 31), "2^30")])
def test_bad_logprobs_are_refused(over, what):
    rc, msg = call("shp_token_logprobs", args(LogprobsArgs, **over))
    assert rc != 0 and what in msg and "ctx" not in msg, msg


def test_the_mirror_refuses_unknown_formats_and_blocks():
    with pytest.raises(ValueError, match="i8, e4m3"):
        Cache8(None, 1, 1, 64, 64, fmt="int8")
    for block in (0, 8, 48, 256):
        with pytest.raises(ValueError, match="16, 32, 64 or 128"):
            Cache8(None, 1, 1, 64, 64, block=block)


@pytest.mark.parametrize("over,what", [
    (dict(head_dim=96), "head_dim"), (dict(n_seqs=0), "heads"), (dict(n_kv_heads=-1), "heads"),
    (dict(n_seqs=40000, n_kv_heads=2), "heads"), (dict(capacity=0), "capacity"),
    (dict(capacity=96), "capacity"), (dict(capacity=192, block=128), "capacity"),
    (dict(capacity=(1 << 22) + 64), "capacity"), (dict(given="k_scale"), "array of 4 bytes"),
    (dict(given="v_scale"), "array of 4 bytes"), (dict(given="lengths"), "array of 4 bytes"),
    (dict(fails_at=1), "no memory"), (dict(fails_at=5), "no memory"), (dict(fails_at=6), "no copy")])
def test_a_cache_that_cannot_be_made_holds_no_memory(monkeypatch, over, what):
    """Geometry and given arrays are looked at first, and what was allocated before a failure is
    freed: the caller gets no object to close."""
    made, freed = [], []

    class Tensor:
        nbytes = 4

        def __init__(self, ctx, n, dtype):
            if len(made) + 1 == fails_at:
                raise MemoryError("no memory")
            made.append(self)

        def upload(self, a):
            raise MemoryError("no copy")

        def free(self):
            freed.append(self)

    dims = dict(n_seqs=2, n_kv_heads=2, head_dim=64, capacity=128, block=64)
    fails_at, given = over.get("fails_at"), over.get("given")
    dims.update({k: v for k, v in over.items() if k in dims})
    small = object.__new__(Tensor)
    monkeypatch.setattr(cache8, "DeviceTensor", Tensor)
    with pytest.raises(MemoryError if fails_at else ValueError, match=what):
        Cache8(None, **dims, **({given: small} if given else {}))
    assert made == freed and len(made) == (fails_at - 1 if fails_at else 0)


# ---- the reference itself -------------------------------------------------------------------

def test_reference_rounds_to_the_nearest_code():
    for fmt in ("i8", "e4m3"):
        values = np.arange(0, 128.0) if fmt == "i8" else R.e4m3_values()
        y = np.concatenate([values, (values[1:] + values[:-1]) / 2,
                            np.random.default_rng(1).uniform(0, values[-1], 1000)])
        got = R.whole(R.encode(y, fmt), fmt).astype(np.float64)
        off = np.abs(got - y)
        best = np.abs(values[None] - y[:, None]).min(1)
        assert (off == best).all()
        assert (R.whole(R.encode(-y, fmt), fmt) == -got).all()
    # ties go to the even code
    assert list(R.encode(np.array([0.5, 1.5, 2.5, -0.5, -1.5]), "i8").view(np.int8)) \
        == [0, 2, 2, 0, -2]
    assert list(R.whole(R.encode(np.array([17.0, 19.0, 2.0 ** -10]), "e4m3"), "e4m3")) \
        == [16.0, 20.0, 0.0]


def test_reference_attention_of_equal_keys_is_the_mean():
    ref = R.RefCache(1, 1, 64, 64, 16, "i8")
    rng = np.random.default_rng(0)
    v = rng.standard_normal((1, 5, 1, 64)).astype(np.float32)
    ref.append(np.ones((1, 5, 1, 64), np.float32), v, [5], [5])
    q = rng.standard_normal((1, 1, 2, 64)).astype(np.float32)
    out, lse, _, _ = R.attend(ref, q, [1], 0.125)
    mean = ref.values("v", 0, 0).astype(np.float64).mean(0)
    assert np.allclose(out[0, 0], mean[None], atol=1e-12)
    assert np.allclose(lse[0, :, 0], q[0, 0].astype(np.float64).sum(1) * 0.125 + np.log(5))
