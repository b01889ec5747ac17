"""Refusals of the paged cache's entry points: arguments are checked before the context, so all of
them show without a device."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from spirv_inference_amd import PagedCache, _lib, paged
from spirv_inference_amd._lib import (PagedAcceptArgs, PagedAppendArgs, PagedAttendArgs, PagedStruct)

P = 0x1000  # an aligned address that no call gets to use
PAGES = 0x1000000


def cache(**over):
    f = dict(k=PAGES, v=2 * PAGES, table=3 * PAGES, lengths=4 * PAGES, n_seqs=2, n_kv_heads=2,
             head_dim=64, n_pages=9, page_size=16, max_pages=4, format=0)
    f.update(over)
    return PagedStruct(*(f[n] for n, _ in PagedStruct._fields_))


def args(cls, **over):
    ptrs = [n for n, t in cls._fields_ if t is C.c_void_p]
    f = {n: (P * (1 + ptrs.index(n)) if t is C.c_void_p else 64) for n, t in cls._fields_}
    f.update({n: v for n, v in dict(counts=0, offsets=0, n=1, n_heads=4, rot=64, interleaved=0,
                                    window=0, scale=0.125, cap=0.0, slopes=0, prefix=0, first=0,
                                    parents=f.get("parents") if cls is PagedAcceptArgs else 0).items()
              if n in f})
    f.update(over)
    return cls(*(f[n] for n, _ in cls._fields_))


def call(name, *structs):
    rc = getattr(_lib.lib(), name)(None, *[C.byref(s) if isinstance(s, C.Structure) else s
                                           for s in structs])
    return rc, _lib.lib().shp_last_error().decode()


CALLS = {"shp_paged_append": PagedAppendArgs, "shp_paged_attend": PagedAttendArgs,
         "shp_paged_accept": PagedAcceptArgs}


@pytest.mark.parametrize("name", CALLS)
def test_good_arguments_get_as_far_as_the_context(name):
    good = (_lib.SHP_ERR_INVALID, f"{name}: null ctx")
    assert call(name, cache(), args(CALLS[name])) == good
    for page in (16, 32, 64, 128, 256):
        assert call(name, cache(head_dim=128, page_size=page, format=2, max_pages=(1 << 22) // page),
                    args(CALLS[name])) == good
    if name != "shp_paged_accept":
        assert call(name, cache(format=1), args(CALLS[name], n=0)) == good
    else:
        assert call(name, cache(), args(PagedAcceptArgs, n=256)) == good
        assert call(name, cache(), args(PagedAcceptArgs, lengths_out=4 * PAGES)) == good


def test_good_arguments_of_appends_and_attention():
    for over in (dict(q=0, q_out=0, n_heads=0), dict(rot=0, inv_freq=0), dict(q=P, q_out=P),
                 dict(rot=8, interleaved=1, offsets=P)):
        assert call("shp_paged_append", cache(), args(PagedAppendArgs, **over))[1].endswith("null ctx")
    for over in (dict(lse=0), dict(window=5, cap=30.0, slopes=P, prefix=P, first=P, parents=P, n=256),
                 dict(n=100000, scale=-1.0), dict(scale=2.35e38), dict(scale=-2.35e38),
                 dict(scale=3.4e38, cap=30.0), dict(cap=3.4028234663852886e38)):
        assert call("shp_paged_attend", cache(), args(PagedAttendArgs, **over))[1].endswith("null ctx")


@pytest.mark.parametrize("over,code,what", [
    (dict(k=0), _lib.SHP_ERR_INVALID, "null array"),
    (dict(v=0), _lib.SHP_ERR_INVALID, "null array"),
    (dict(table=0), _lib.SHP_ERR_INVALID, "null array"),
    (dict(lengths=0), _lib.SHP_ERR_INVALID, "null array"),
    (dict(format=3), _lib.SHP_ERR_UNSUPPORTED, "format"),
    (dict(format=-1), _lib.SHP_ERR_UNSUPPORTED, "format"),
    (dict(head_dim=96), _lib.SHP_ERR_UNSUPPORTED, "head_dim"),
    (dict(head_dim=0), _lib.SHP_ERR_UNSUPPORTED, "head_dim"),
    (dict(page_size=8), _lib.SHP_ERR_UNSUPPORTED, "page_size"),
    (dict(page_size=48), _lib.SHP_ERR_UNSUPPORTED, "page_size"),
    (dict(page_size=512), _lib.SHP_ERR_UNSUPPORTED, "page_size"),
    (dict(page_size=0), _lib.SHP_ERR_UNSUPPORTED, "page_size"),
    (dict(page_size=-16), _lib.SHP_ERR_UNSUPPORTED, "page_size"),
    (dict(n_seqs=0), _lib.SHP_ERR_SHAPE, "n_seqs"),
    (dict(n_kv_heads=-1), _lib.SHP_ERR_SHAPE, "n_seqs"),
    (dict(n_seqs=40000), _lib.SHP_ERR_SHAPE, "n_seqs"),
    (dict(n_pages=0), _lib.SHP_ERR_SHAPE, "n_pages"),
    (dict(n_pages=-4), _lib.SHP_ERR_SHAPE, "n_pages"),
    (dict(max_pages=0), _lib.SHP_ERR_SHAPE, "max_pages"),
    (dict(max_pages=(1 << 18) + 1), _lib.SHP_ERR_SHAPE, "max_pages"),
    (dict(max_pages=2 ** 31 - 1, page_size=256), _lib.SHP_ERR_SHAPE, "max_pages"),
    (dict(k=PAGES + 8), _lib.SHP_ERR_INVALID, "16-byte"),
    (dict(v=PAGES + 4), _lib.SHP_ERR_INVALID, "16-byte"),
    (dict(table=PAGES + 2), _lib.SHP_ERR_INVALID, "4-byte"),
    (dict(lengths=PAGES + 1), _lib.SHP_ERR_INVALID, "4-byte")])
def test_bad_caches_are_refused(over, code, what):
    for name, cls in CALLS.items():
        rc, msg = call(name, cache(**over), args(cls))
        assert rc == code and what in msg and msg.startswith(name), (name, rc, msg)


@pytest.mark.parametrize("name,over,what", [
    ("shp_paged_append", dict(n=-1), "n < 0"),
    ("shp_paged_append", dict(k=0), "null k"),
    ("shp_paged_append", dict(v=0), "null v"),
    ("shp_paged_append", dict(k=P + 4), "k rows"),
    ("shp_paged_append", dict(v_row=66), "v rows"),
    ("shp_paged_append", dict(k_head=1), "k rows"),
    ("shp_paged_append", dict(q=0), "q and q_out"),
    ("shp_paged_append", dict(q_out=0), "q and q_out"),
    ("shp_paged_append", dict(q=P + 8), "q rows"),
    ("shp_paged_append", dict(o_head=2), "q_out rows"),
    ("shp_paged_append", dict(n_heads=3), "n_heads"),
    ("shp_paged_append", dict(n_heads=0), "n_heads"),
    ("shp_paged_append", dict(q=P, q_out=P, o_row=128), "other strides"),
    ("shp_paged_append", dict(rot=-8), "rot"),
    ("shp_paged_append", dict(rot=12), "rot"),
    ("shp_paged_append", dict(rot=72), "rot"),
    ("shp_paged_append", dict(inv_freq=0), "inv_freq"),
    ("shp_paged_append", dict(n=600000), "500000"),
    ("shp_paged_attend", dict(q=P, out=P, o_seq=128), "other strides"),
    ("shp_paged_attend", dict(cap=1e-45, scale=1.0), "cap"),
    ("shp_paged_attend", dict(cap=1e-3, scale=1e37), "cap"),
    ("shp_paged_attend", dict(n=-1), "n < 0"),
    ("shp_paged_attend", dict(q=0), "null q"),
    ("shp_paged_attend", dict(out=0), "null out"),
    ("shp_paged_attend", dict(q=P + 8), "q rows"),
    ("shp_paged_attend", dict(o_seq=2), "out rows"),
    ("shp_paged_attend", dict(n_heads=3), "n_heads"),
    ("shp_paged_attend", dict(n_heads=0), "n_heads"),
    ("shp_paged_attend", dict(scale=float("nan")), "scale"),
    ("shp_paged_attend", dict(scale=float("inf")), "scale"),
    ("shp_paged_attend", dict(scale=2.4e38), "scale times log2 e"),
    ("shp_paged_attend", dict(scale=-3.4028234663852886e38), "scale times log2 e"),
    ("shp_paged_attend", dict(cap=-1.0), "cap"),
    ("shp_paged_attend", dict(cap=float("inf")), "cap"),
    ("shp_paged_attend", dict(cap=float("nan")), "cap"),
    ("shp_paged_attend", dict(window=-1), "window"),
    ("shp_paged_attend", dict(n=300000), "500000"),
    ("shp_paged_attend", dict(parents=P, n=257), "256"),
    ("shp_paged_accept", dict(n=0), "n < 1"),
    ("shp_paged_accept", dict(n=257), "256"),
    ("shp_paged_accept", dict(parents=0), "null parents"),
    ("shp_paged_accept", dict(tokens=0), "null parents"),
    ("shp_paged_accept", dict(choices=0), "null parents"),
    ("shp_paged_accept", dict(path=0), "null path"),
    ("shp_paged_accept", dict(accepted=0), "null path"),
    ("shp_paged_accept", dict(next=0), "null path"),
    ("shp_paged_accept", dict(lengths_out=0), "null path")])
def test_bad_arguments_are_refused(name, over, what):
    rc, msg = call(name, cache(), args(CALLS[name], **over))
    assert rc != 0 and what in msg and "ctx" not in msg, (rc, msg)


def test_appends_of_too_many_rows_are_refused():
    rc, msg = call("shp_paged_append", cache(n_seqs=40, n_kv_heads=1), args(PagedAppendArgs, n=400001, n_heads=1))
    assert rc == _lib.SHP_ERR_UNSUPPORTED and "16000000" in msg
    assert call("shp_paged_append", cache(n_seqs=40, n_kv_heads=1),
                args(PagedAppendArgs, n=400000, n_heads=1))[1].endswith("null ctx")


@pytest.mark.parametrize("name,fields", [
    ("shp_paged_append", ["counts", "offsets", "inv_freq"]),
    ("shp_paged_attend", ["counts", "lse", "slopes", "prefix", "first", "parents"]),
    ("shp_paged_accept", ["counts", "parents", "tokens", "choices", "path", "accepted", "next",
                          "lengths_out"])])
def test_arrays_of_numbers_that_are_not_aligned_are_refused(name, fields):
    for f in fields:
        for off in (1, 2, 3):
            rc, msg = call(name, cache(), args(CALLS[name], **{f: 0x80000 + off}))
            assert rc == _lib.SHP_ERR_INVALID and "4-byte aligned" in msg, (f, msg)


def test_acceptance_refuses_arrays_that_overlap():
    """Everything that is written against everything else, at its first and at its last word; only the
    cache's own lengths may be where the new ones go."""
    n, size = 5, {"counts": 8, "accepted": 8, "next": 8, "lengths_out": 8}
    names = [f for f, t in PagedAcceptArgs._fields_ if t is C.c_void_p]
    for out in ("path", "accepted", "next", "lengths_out"):
        for other in names:
            if other == out:
                continue
            base = 0x80000
            for at in (base - size.get(out, 2 * n * 4) + 4, base, base + size.get(other, 2 * n * 4) - 4):
                rc, msg = call("shp_paged_accept", cache(),
                               args(PagedAcceptArgs, n=n, **{other: base, out: at}))
                assert rc == _lib.SHP_ERR_INVALID and "shares memory" in msg, (out, other, msg)
        for field, bytes_ in (("k", 9 * 2 * 16 * 64 * 4), ("v", 9 * 2 * 16 * 64 * 4), ("table", 32),
                              ("lengths", 8)):
            base = getattr(cache(), field)
            for at in (base - size.get(out, 2 * n * 4) + 4, base + bytes_ - 4):
                rc, msg = call("shp_paged_accept", cache(), args(PagedAcceptArgs, n=n, **{out: at}))
                assert rc == _lib.SHP_ERR_INVALID and "shares memory" in msg, (out, field, msg)


@pytest.mark.parametrize("form,n,heads,want", [
    # rows of a block, a wavefront by itself, tokens shared out
    (dict(format=2, n_kv_heads=112), 101, 112 * 4, (32, 1, 0)),    # 2 x 112 x 13 blocks
    (dict(format=2, n_kv_heads=896), 64, 896, (32, 0, 0)),         # 64 rows of a KV head: never
    (dict(format=2, n_kv_heads=896), 65, 896, (32, 1, 0)),
    (dict(format=2, n_kv_heads=298, max_pages=8), 70, 298, (32, 0, 0)),  # 3 x 596 = 1,788 blocks: not quite
    (dict(format=1, n_kv_heads=299, max_pages=8), 70, 299, (32, 1, 0)),  # 1,794 of at least 7 x 256
    (dict(format=0, n_kv_heads=896), 65, 896, (32, 0, 0)),         # fp32: never
    (dict(format=1, max_pages=64), 1, 2, (16, 0, 1)),
    (dict(format=1, max_pages=4), 1, 2, (16, 0, 0)),               # a tile
    (dict(format=1, max_pages=64, n_kv_heads=512), 1, 512, (16, 0, 0)),   # 16 tiles, a share has 32 with 1,024 blocks
    (dict(format=1, max_pages=128, n_kv_heads=512), 1, 512, (16, 0, 0)),
    (dict(format=1, max_pages=129, n_kv_heads=512), 1, 512, (16, 0, 1)),
    (dict(format=1, max_pages=129, n_kv_heads=513), 1, 513, (16, 0, 0)),  # more than 1,024 blocks
    (dict(format=0, max_pages=64, n_seqs=512, n_kv_heads=1), 1, 1, (16, 0, 0)),  # 32 tiles
    (dict(format=0, max_pages=65, n_seqs=512, n_kv_heads=1), 1, 1, (16, 0, 1)),
    (dict(format=0, max_pages=65, n_seqs=513, n_kv_heads=1), 1, 1, (16, 0, 0))])  # more than 512 sequences
def test_attention_plans(form, n, heads, want):
    """Which variant a call takes on 256 CUs, on both sides of each line."""
    out = (C.c_int32 * 4)()
    rc = _lib.lib().shp_paged_attend_plan(None, C.byref(cache(**form)), n, heads, out)
    assert rc == 0 and tuple(out[:3]) == want, _lib.lib().shp_last_error()


class FakeTensor:
    def __init__(self, nbytes, ptr=P):
        self.nbytes, self.ptr = nbytes, ptr


@pytest.mark.parametrize("bad,what", [
    (dict(fmt="i8"), "format"), (dict(page_size=24), "pages of 24"), (dict(head_dim=80), "head_dim"),
    (dict(n_seqs=0), "sequences"), (dict(n_kv_heads=70000), "sequences"), (dict(n_pages=0), "0 pages"),
    (dict(max_pages=0), "0 pages a sequence"), (dict(max_pages=1 << 19), "pages a sequence"),
    (dict(k=FakeTensor(100)), "an array of 100 bytes"), (dict(lengths=FakeTensor(4)), "an array of 4"),
    (dict(table=FakeTensor(8)), "an array of 8")])
def test_the_mirror_looks_at_shapes_and_arrays_before_it_allocates(monkeypatch, bad, what):
    def no(*a, **k):
        raise AssertionError("allocated")
    monkeypatch.setattr(paged, "DeviceTensor", no)
    f = dict(n_seqs=2, n_kv_heads=2, head_dim=64, n_pages=3, page_size=16, max_pages=2)
    f.update(bad)
    with pytest.raises(ValueError, match=what):
        PagedCache(None, f.pop("n_seqs"), f.pop("n_kv_heads"), f.pop("head_dim"), f.pop("n_pages"),
                   f.pop("page_size"), f.pop("max_pages"), **f)


def test_a_failed_allocation_frees_what_was_allocated(monkeypatch):
    made, freed = [], []

    class T:
        def __init__(self, ctx, n, dtype):
            if len(made) == 2:
                raise MemoryError
            made.append(self)

        def free(self):
            freed.append(self)
    monkeypatch.setattr(paged, "DeviceTensor", T)
    with pytest.raises(MemoryError):
        PagedCache(None, 1, 1, 64, 4, 16, 2)
    assert freed == made and len(made) == 2


def test_a_closed_cache_is_refused():
    t = FakeTensor(1 << 20)
    c = PagedCache.__new__(PagedCache)
    c._own, c._struct = [], cache()
    c.close()
    for name, cls in CALLS.items():
        rc, msg = call(name, c._struct, args(cls))
        assert rc == _lib.SHP_ERR_INVALID and "null array" in msg


# ---- the reference itself -----------------------------------------------------------------------

def test_reference_rounding_and_words():
    x = np.array([1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -1 - 2.0 ** -9, 3.4e38, 70000.0, np.inf, 0.0],
                 np.float32)
    np.testing.assert_array_equal(R.stored(x, "bf16")[:4], np.float32([1, 1, 1 + 2.0 ** -6, -1]))
    assert np.isinf(R.stored(x, "f16")[5]) and np.isinf(R.stored(x, "bf16")[4])
    for fmt in ("f32", "f16", "bf16"):
        y = R.stored(x, fmt)
        np.testing.assert_array_equal(R.values(R.words(y, fmt), fmt), y)


def test_reference_sight():
    there = np.ones(16, bool)
    sees, far = R.sight(6, 2, 16, there)
    assert sees.tolist() == [[True] * 5 + [False], [True] * 6]
    sees, _ = R.sight(6, 2, 16, there, window=2, prefix=1)
    assert sees.tolist() == [[True, False, False, True, True, False], [True] + [False] * 3 + [True] * 2]
    sees, _ = R.sight(4, 4, 16, there, prefix=2)
    assert sees[0].tolist() == [True, True, False, False]
    sees, _ = R.sight(4, 4, 16, there, first=[0, 1, 1, 9])
    assert sees[2].tolist() == [False, True, True, False] and not sees[3].any()
    # a chain is causal; two rows on one parent do not see each other
    a, _ = R.sight(9, 4, 16, there, parents=[-1, 0, 1, 2])
    np.testing.assert_array_equal(a, R.sight(9, 4, 16, there)[0])
    sees, far = R.sight(5, 3, 16, there, parents=[-1, 0, 0])
    assert sees[2].tolist() == [True, True, True, False, True] and far[2].tolist() == [3, 2, 1, 0, 0]
    assert not R.sight(2, 3, 16, there)[0][0].any()


def test_reference_acceptance():
    par, ids, pick = [-1, 0, 0, 1, 1, 4], [5, 7, 8, 9, 9, 4], [7, 9, 1, 2, 3, 6]
    assert R.accept(par, ids, pick, 20, 6) == ([0, 1, 3], 2, 17)
    assert R.accept(par, ids, [8] + pick[1:], 20, 6) == ([0, 2], 1, 16)
    assert R.accept(par, ids, [1] + pick[1:], 6, 6) == ([0], 1, 1)
    assert R.accept(par, ids, pick, 5, 6) == ([], -1, 5) and R.accept(par, ids, pick, 5, 0) == ([], -1, 5)


def test_reference_rotation_is_a_rotation():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 2, 64)).astype(np.float32)
    f = (10000.0 ** (-np.arange(12) / 12)).astype(np.float32)
    for inter in (False, True):
        y = R.turned(x, [0, 5, 131071], f, inter)
        np.testing.assert_allclose(y[0], x[0])
        np.testing.assert_allclose((y ** 2).sum(-1), (x.astype(np.float64) ** 2).sum(-1), rtol=1e-12)
        np.testing.assert_array_equal(y[..., 24:], x[..., 24:])
