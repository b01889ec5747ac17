"""The serving operators around an 8-bit key/value cache, as cases that can be timed and checked.

Each case is one call (or a call and the read of what it wrote) on resident tensors of one GPU:

* `append`   - new K and V rows are quantised into the cache, and the newest tokens read back;
* `attend`   - attention of new queries over the cached tokens;
* `weigh`    - the attention weight each cached token got is added to its account;
* `evict`    - the tokens with the least weight leave: the rest is compacted into another cache;
* `logprobs` - log probabilities of given tokens, with the entropy and the likeliest alternatives.

`own` chooses between the framework's calls and the plain form in elementary torch operations;
`exact` states the definition again in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
TILE = 64            # tokens of one V tile in the cache
FLOOR = 2.0 ** -60   # smallest scale of a block
CODE_MAX = {"i8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # one decode step of the TinyLlama-shaped decoder early in a chat: latency
        {"name": "attend_b1_300", "kind": "attend", "seqs": 1, "heads": 32, "kv": 4, "d": 64,
         "cap": 512, "lo": 300, "hi": 300, "n": 1, "ragged": False, "fmt": "i8", "block": 64},
        # a decode step of a batch whose conversations differ in length; one slot is empty
        {"name": "attend_b24_ragged", "kind": "attend", "seqs": 24, "heads": 32, "kv": 8, "d": 128,
         "cap": 8192, "lo": 0, "hi": 8100, "n": 1, "ragged": False, "fmt": "e4m3", "block": 32},
        # a decode step over long documents: a cache of more than 4 GiB
        {"name": "attend_b16_131k", "kind": "attend", "seqs": 16, "heads": 32, "kv": 8, "d": 128,
         "cap": 131072, "lo": 128001, "hi": 131072, "n": 1, "ragged": False, "fmt": "i8",
         "block": 64},
        # a chunk of a prompt behind what is cached already: matrix work
        {"name": "attend_chunk_512", "kind": "attend", "seqs": 1, "heads": 32, "kv": 8, "d": 128,
         "cap": 8192, "lo": 8190, "hi": 8190, "n": 512, "ragged": False, "fmt": "i8", "block": 64},
        # the token each sequence of a batch just made, into small blocks
        {"name": "append_b64_step", "kind": "append", "seqs": 64, "kv": 4, "d": 64, "cap": 1024,
         "lo": 3, "hi": 1020, "n": 1, "ragged": False, "fmt": "i8", "block": 16},
        # prompts of a batch, of different lengths
        {"name": "append_b4_prompt", "kind": "append", "seqs": 4, "kv": 8, "d": 128, "cap": 4096,
         "lo": 2001, "hi": 4000, "n": 2000, "ragged": True, "fmt": "e4m3", "block": 64},
        # the weights of a batch's decode step
        {"name": "weigh_b24_step", "kind": "weigh", "seqs": 24, "heads": 32, "kv": 8, "d": 128,
         "cap": 8192, "lo": 500, "hi": 8100, "n": 1, "ragged": False, "fmt": "i8", "block": 64},
        # the weights of a prompt's last chunk, which eviction goes by
        {"name": "weigh_chunk_512", "kind": "weigh", "seqs": 1, "heads": 32, "kv": 4, "d": 64,
         "cap": 8192, "lo": 8190, "hi": 8190, "n": 512, "ragged": False, "fmt": "i8", "block": 64},
        # one conversation shrinks to half
        {"name": "evict_b1_1000", "kind": "evict", "seqs": 1, "kv": 4, "d": 64, "cap": 1024,
         "lo": 1000, "hi": 1000, "keep": 512, "recent": 64, "fmt": "i8", "block": 64},
        # a batch of prompts shrinks to the budget that decoding goes on with
        {"name": "evict_b16_8k", "kind": "evict", "seqs": 16, "kv": 8, "d": 128, "cap": 8192,
         "lo": 1900, "hi": 8190, "keep": 2048, "recent": 256, "fmt": "i8", "block": 32},
        # the token just decoded, with five alternatives
        {"name": "logprobs_1x32000", "kind": "logprobs", "rows": 1, "vocab": 32000, "top": 5},
        # a scored document over a large vocabulary of odd size
        {"name": "logprobs_1500x131071", "kind": "logprobs", "rows": 1500, "vocab": 131071,
         "top": 20},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "weigh", "evict", "logprobs"])
    if kind == "logprobs":
        vocab = _log(rng, 1000, 160000)
        return {"kind": kind, "rows": _log(rng, 1, min(4000, 190_000_000 // vocab)),
                "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 32])}
    fmt, block = rng.choice(["i8", "i8", "e4m3"]), rng.choice([16, 32, 64, 64, 128])
    kv, d = rng.choice([(4, 64), (8, 128), (8, 64), (2, 128)])
    case = {"kind": kind, "kv": kv, "d": d, "fmt": fmt, "block": block}
    if kind == "append":
        n = rng.choice([1, 1, _log(rng, 2, 2000)])
        hi = n + _log(rng, 1, 2000)
        return {**case, "seqs": _log(rng, 1, 64 if n < 64 else 4), "n": n, "lo": n, "hi": hi,
                "cap": -(-hi // 128) * 128, "ragged": rng.random() < 0.5}
    if kind == "evict":
        hi = _log(rng, 200, 8190)
        keep = rng.randint(64, max(65, hi // 2))
        return {**case, "seqs": _log(rng, 1, 16), "lo": max(1, hi // 4), "hi": hi, "keep": keep,
                "recent": rng.randint(0, keep), "cap": -(-hi // 128) * 128}
    case["heads"] = kv * rng.choice([1, 4, 4, 8 if kv < 8 else 4])
    if kind == "attend" and rng.random() < 0.5:  # decode steps, or a few tokens at a time
        n, seqs = rng.choice([1, 1, 1, rng.randint(2, 8)]), _log(rng, 1, 64)
        hi = max(n, _log(rng, 16, 400_000 // seqs))
        lo = rng.choice([0, hi // 3, hi])
    else:
        n, seqs = _log(rng, 1, 512), 1 + (rng.random() < 0.4)
        hi = n + _log(rng, 1, 7600)
        lo = rng.choice([n, hi])
    return {**case, "seqs": seqs, "n": n, "lo": lo, "hi": hi, "cap": -(-hi // 128) * 128,
            "ragged": n > 1 and rng.random() < 0.5}


# ---- what the cases hold -----------------------------------------------------------------

def _lens(case):
    """Tokens held by each sequence: spread over [lo, hi], the same for every seed."""
    s, lo, hi = case["seqs"], case["lo"], case["hi"]
    if s == 1:
        return [hi]
    r = random.Random(7 * s + hi)
    lens = [lo + (hi - lo) * i // (s - 1) for i in range(s)]
    r.shuffle(lens)
    return lens


def _counts(case):
    """New rows of each sequence, at most those it holds."""
    s, n = case["seqs"], case["n"]
    r = random.Random(3 * s + n)
    return [min(ln, r.randint(1, n) if case["ragged"] else n) for ln in _lens(case)]


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        r, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": 4.0 * r * v + r * (12 + 8 * k), "flops": 6.0 * r * v}
    kv, d, lens = case["kv"], case["d"], _lens(case)
    tokens = sum(lens)
    scales = 8.0 * kv * sum(-(-ln // case["block"]) for ln in lens)
    if kind == "evict":
        kept = sum(min(ln, case["keep"]) for ln in lens)
        # the weights; kept codes in and out; slots and weights out; the values read back
        return {"bytes": kv * (4.0 * tokens + kept * (4.0 * d + 8) + kept * 8.0 * d) + scales,
                "flops": 4.0 * kept * kv * d}
    counts = _counts(case)
    new = sum(counts)
    if kind == "append":
        back = sum(min(ln, _back(case)) for ln in lens)
        return {"bytes": kv * d * (8.0 * new + 2.0 * new + 10.0 * back), "flops": 4.0 * new * kv * d}
    h = case["heads"]
    seen = sum(c * ln - c * (c - 1) // 2 for c, ln in zip(counts, lens)) * h  # (row, token) pairs
    if kind == "attend":
        return {"bytes": 2.0 * tokens * kv * d + scales + new * h * (8.0 * d + 4),
                "flops": 4.0 * d * seen}
    return {"bytes": kv * tokens * (d + 8.0) + scales / 2 + new * h * (4.0 * d + 4),
            "flops": 2.0 * d * seen}


def _back(case):
    """Newest tokens that an `append` case reads back: the new ones and the rest of their first
    block, whose codes change when its scale grows."""
    return min(case["cap"], case["n"] + case["block"] - 1)


def _codes(shape, fmt, g):
    """Codes as a trained model's rows give them: about normal, a few at the end of the range."""
    x = torch.empty(shape, device=DEV, dtype=torch.float16).normal_(0, 0.27, generator=g)
    if fmt == "i8":
        return x.mul_(127).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    return x.mul_(448).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1009 + 17)

    def randn(*shape, std=1.0):
        return torch.empty(shape, device=DEV).normal_(0, std, generator=g)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    st = {"case": case}
    if case["kind"] == "logprobs":
        r, v, k = case["rows"], case["vocab"], case["top"]
        st["logits"] = randn(r, v, std=3.0)
        st["targets"] = torch.randint(0, v, (r,), device=DEV, generator=g, dtype=torch.int32)
        st["logprob"], st["entropy"] = torch.zeros(r, device=DEV), torch.zeros(r, device=DEV)
        st["top_ids"] = torch.zeros(r, k, device=DEV, dtype=torch.int32)
        st["top_logprobs"] = torch.zeros(r, k, device=DEV)
        if own:
            _hold(st)
        return st
    s, kv, d, cap, block, fmt = (case[x] for x in ("seqs", "kv", "d", "cap", "block", "fmt"))
    st["k"] = _codes((s, kv, cap, d), fmt, g)
    st["v"] = _codes((s, kv, cap // TILE, d, TILE), fmt, g)
    for t in ("k_scale", "v_scale"):  # absolute maxima near 3.5, as of normal rows
        st[t] = torch.empty(s, kv, cap // block, device=DEV).uniform_(
            2.5 / CODE_MAX[fmt], 4.5 / CODE_MAX[fmt], generator=g)
    st["lens"] = ints(_lens(case))
    if case["kind"] == "evict":
        keep = case["keep"]
        dcap = -(-keep // 128) * 128
        # accounts as attention leaves them: a few tokens hold most of the weight
        st["acc"] = randn(s, kv, cap).mul_(2.0).exp_()
        st["dk"] = torch.zeros(s, kv, dcap, d, dtype=torch.uint8, device=DEV)
        st["dv"] = torch.zeros(s, kv, dcap // TILE, d, TILE, dtype=torch.uint8, device=DEV)
        st["dk_scale"] = torch.zeros(s, kv, dcap // block, device=DEV)
        st["dv_scale"] = torch.zeros(s, kv, dcap // block, device=DEV)
        st["dlens"] = torch.zeros(s, dtype=torch.int32, device=DEV)
        st["kept"] = torch.zeros(s, kv, keep, dtype=torch.int32, device=DEV)
        st["dacc"] = torch.zeros(s, kv, dcap, device=DEV)
        st["k_back"] = torch.zeros(s, kv, keep, d, device=DEV)
        st["v_back"] = torch.zeros(s, kv, keep, d, device=DEV)
    else:
        n = case["n"]
        st["counts"] = ints(_counts(case))
        if case["kind"] == "append":
            st["k_new"], st["v_new"] = randn(s, n, kv, d), randn(s, n, kv, d)
            st["k_back"] = torch.zeros(s, kv, _back(case), d, device=DEV)
            st["v_back"] = torch.zeros(s, kv, _back(case), d, device=DEV)
        else:
            h = case["heads"]
            st["q"] = randn(s, n, h, d)
            st["lse"] = torch.full((s, h, n), -math.inf, device=DEV)
            if case["kind"] == "attend":
                st["out"] = torch.zeros(s, n, h, d, device=DEV)
            else:  # the call before gave the rows' log sums
                st["lse"] = _softmax(st)[2].reshape(s, kv, n, h // kv).transpose(2, 3) \
                    .reshape(s, h, n).contiguous()
                st["acc"] = randn(s, kv, cap).abs_()
                st["acc_out"] = torch.zeros(s, kv, cap, device=DEV)
    if own:
        _hold(st)
    return st


def _hold(st):
    """What a program keeps for its calls: the context, the cache and its tensors."""
    from spirv_inference_amd import Cache8, Context, DeviceTensor
    global _CTX
    if _CTX is None:
        _CTX = Context("any")
    kinds = {torch.float32: "<f4", torch.int32: "<i4", torch.uint8: "u1"}
    t = {n: DeviceTensor(_CTX, x.numel(), kinds[x.dtype], ptr=x.data_ptr(), owned=False)
         for n, x in st.items() if isinstance(x, torch.Tensor)}
    c = st["case"]
    st["t"], st["ctx"] = t, _CTX
    if c["kind"] == "logprobs":
        return
    shape = (c["seqs"], c["kv"], c["d"])
    st["cache"] = Cache8(_CTX, *shape, c["cap"], block=c["block"], fmt=c["fmt"], k=t["k"], v=t["v"],
                         k_scale=t["k_scale"], v_scale=t["v_scale"], lengths=t["lens"])
    if c["kind"] == "evict":
        st["to"] = Cache8(_CTX, *shape, st["dk"].shape[2], block=c["block"], fmt=c["fmt"],
                          k=t["dk"], v=t["dv"], k_scale=t["dk_scale"], v_scale=t["dv_scale"],
                          lengths=t["dlens"])


_CTX = None


def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    c, t = st["case"], st["t"]
    kind = c["kind"]
    if kind == "attend":
        st["cache"].attend(t["q"], t["out"], c["heads"], c["n"], counts=t["counts"], lse=t["lse"])
        return {"out": st["out"], "lse": st["lse"]}
    if kind == "append":
        st["cache"].append(t["k_new"], t["v_new"], c["n"], counts=t["counts"])
        st["cache"].read(_back(c), t["k_back"], t["v_back"])
        return {"k": st["k_back"], "v": st["v_back"], "k_scale": st["k_scale"],
                "v_scale": st["v_scale"]}
    if kind == "weigh":
        st["cache"].weights(t["q"], t["lse"], t["acc"], t["acc_out"], c["heads"], c["n"],
                            counts=t["counts"])
        return {"acc": st["acc_out"]}
    if kind == "evict":
        st["cache"].evict(st["to"], t["acc"], c["keep"], c["recent"], kept=t["kept"],
                          dst_weights=t["dacc"])
        st["to"].read(c["keep"], t["k_back"], t["v_back"])
        return {"k": st["k_back"], "v": st["v_back"], "lens": st["dlens"], "kept": st["kept"],
                "acc": st["dacc"]}
    st["ctx"].token_logprobs(t["logits"], t["targets"], t["logprob"], t["entropy"], t["top_ids"],
                             t["top_logprobs"], c["rows"], c["vocab"], c["top"])
    return {"logprob": st["logprob"], "entropy": st["entropy"], "top_ids": st["top_ids"],
            "top_logprobs": st["top_logprobs"]}


# ---- the plain forms ---------------------------------------------------------------------

def _value(codes, fmt):
    """What codes stand for before the scale."""
    return codes.view(torch.int8 if fmt == "i8" else torch.float8_e4m3fn).float()


def _cached(st):
    """Keys and values [seqs, kv, cap, d] that the cache holds."""
    c = st["case"]
    k = _value(st["k"], c["fmt"]) * st["k_scale"].repeat_interleave(c["block"], 2)[..., None]
    v = _value(st["v"], c["fmt"]).transpose(3, 4).reshape(k.shape) \
        * st["v_scale"].repeat_interleave(c["block"], 2)[..., None]
    return k, v


def _scores(st, k):
    """Scaled scores [seqs, kv, n * group, cap], -inf where a row does not see a token; and which
    rows are real."""
    c = st["case"]
    s, kv, d, n, cap = c["seqs"], c["kv"], c["d"], c["n"], c["cap"]
    group = c["heads"] // kv
    q = st["q"].reshape(s, n, kv, group, d).permute(0, 2, 1, 3, 4).reshape(s, kv, n * group, d)
    x = torch.matmul(q * d ** -0.5, k.transpose(2, 3))
    i = torch.arange(n, device=DEV).repeat_interleave(group)
    sees = (st["lens"] - st["counts"])[:, None] + i + 1
    slot = torch.arange(cap, device=DEV)
    real = (i < st["counts"][:, None])[:, None, :, None]
    x = x.masked_fill_((slot >= sees[:, :, None])[:, None], -math.inf)
    return x, real


def _softmax(st):
    """Weights before they are divided by their sum, that sum, and its log: an empty row's are 0, 0
    and -inf."""
    k, v = _cached(st)
    x, real = _scores(st, k)
    m = x.amax(3, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    p = x.sub_(m).exp_()
    z = p.sum(3, keepdim=True)
    return p, z, torch.where(real, m + z.log(), torch.full_like(m, -math.inf)), v, real


def _plain_attend(st):
    c = st["case"]
    s, n, h, kv, d = c["seqs"], c["n"], c["heads"], c["kv"], c["d"]
    p, z, lse, v, real = _softmax(st)
    o = torch.matmul(p, v) / torch.where(z > 0, z, torch.ones_like(z))
    o = torch.where(real, o, torch.zeros_like(o))
    o = o.reshape(s, kv, n, h // kv, d).permute(0, 2, 1, 3, 4).reshape(s, n, h, d).contiguous()
    lse = lse.reshape(s, kv, n, h // kv).transpose(2, 3).reshape(s, h, n).contiguous()
    return {"out": o, "lse": lse}


def _plain_weigh(st):
    c = st["case"]
    s, n, h, kv = c["seqs"], c["n"], c["heads"], c["kv"]
    k, _ = _cached(st)
    x, real = _scores(st, k)
    lse = st["lse"].reshape(s, kv, h // kv, n).transpose(2, 3).reshape(s, kv, -1, 1)
    p = torch.where(real & torch.isfinite(lse), x - lse, torch.full_like(x, -math.inf)).exp_()
    held = torch.arange(c["cap"], device=DEV) < st["lens"][:, None, None]
    return {"acc": torch.where(held, st["acc"] + p.sum(2), torch.zeros_like(st["acc"]))}


def _scale(top, fmt):
    """A block's scale from its largest absolute value: the quotient rounded once (a product with
    the reciprocal, which torch takes for a plain number, can be the next number)."""
    return (top.double() / CODE_MAX[fmt]).float().clamp(min=FLOOR)


def _encode(x, scale, fmt):
    """Codes of x at a scale: the quotient, to the nearest code (ties to even); in 64 bits, since a
    quotient next to the middle of two codes has to fall on its own side."""
    y = x.double() / scale.double()
    if fmt == "i8":
        return y.round().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y).exponent - 1).clamp_(min=-6) - 3)
    return ((y / step).round() * step).clamp_(-448, 448).float().to(torch.float8_e4m3fn) \
        .view(torch.uint8)


def _plain_append(st):
    c = st["case"]
    s, kv, d, cap, block, n, fmt = (c[x] for x in ("seqs", "kv", "d", "cap", "block", "n", "fmt"))
    back = _back(c)
    start = (st["lens"] - st["counts"])[:, None].long()
    # slots of the newest `back` tokens, and which are new
    slot = st["lens"][:, None].long() - back + torch.arange(back, device=DEV)
    held, new = slot >= 0, slot >= start
    at = slot.clamp(min=0)[:, None, :, None].expand(s, kv, back, d)
    row = (slot - start).clamp(0, n - 1)[:, None, :, None].expand(s, kv, back, d)
    blk = at[..., 0] // block
    got = {}
    for name in ("k", "v"):
        scale = st[name + "_scale"]
        bytes_ = st[name] if name == "k" else st[name].transpose(3, 4).reshape(s, kv, cap, d)
        x = st[name + "_new"].transpose(1, 2).gather(2, row)
        is_new = new[:, None, :].expand(s, kv, back)
        top = torch.where(is_new, x.abs().amax(3), torch.zeros_like(x[..., 0]))
        top = torch.zeros_like(scale).scatter_reduce_(2, blk, top, "amax")
        touched = torch.zeros_like(scale).scatter_reduce_(2, blk, is_new.float(), "amax") > 0
        begun = torch.arange(cap // block, device=DEV) * block < start[:, :, None]
        grown = _scale(top, fmt)
        grown = torch.where(begun, torch.maximum(scale, grown), grown)
        grown = torch.where(touched, grown, scale)
        old = bytes_.gather(2, at)
        was, now = scale.gather(2, blk)[..., None], grown.gather(2, blk)[..., None]
        again = torch.where(now > was, _encode(_value(old, fmt) * was, now, fmt), old)
        code = torch.where(is_new[..., None], _encode(x, now, fmt), again)
        # slots before the first token stand for nothing: they are sent to the newest one's place
        last = (slot[:, -1:])[:, None, :, None].expand(s, kv, back, d)
        put = torch.where(held[:, None, :, None], at, last)
        code = torch.where(held[:, None, :, None], code, code[:, :, -1:])
        if name == "k":
            st["k"].scatter_(2, put, code)
        else:
            bytes_ = bytes_.scatter(2, put, code)
            st["v"].copy_(bytes_.reshape(s, kv, cap // TILE, TILE, d).transpose(3, 4))
        scale.copy_(grown)
        got[name] = torch.where(held[:, None, :, None], _value(code, fmt) * now,
                                torch.zeros_like(x))
        got[name + "_scale"] = scale
    return got


def _order(w):
    """Weights as whole numbers in the same order (both zeros alike)."""
    b = (w + 0.0).view(torch.int32).long()
    return torch.where(b < 0, -(b & 0x7FFFFFFF), b)


def _plain_evict(st):
    c = st["case"]
    s, kv, d, cap, block, fmt = (c[x] for x in ("seqs", "kv", "d", "cap", "block", "fmt"))
    keep, recent = c["keep"], c["recent"]
    slot = torch.arange(cap, device=DEV)
    lens = st["lens"][:, None, None]
    key = (_order(st["acc"]) << 20) + (cap - slot)
    key = torch.where(slot >= lens - recent, torch.full_like(key, 1 << 60) + slot, key)
    key = torch.where(slot >= lens, torch.full_like(key, -(1 << 60)), key)
    keys, kept = key.topk(keep, 2)
    kept = torch.where(keys > -(1 << 60), kept, torch.full_like(kept, cap)).sort(2).values
    held = kept < cap
    at = kept.clamp(max=cap - 1)
    dcap = -(-keep // 128) * 128
    got = {"lens": st["lens"].clamp(max=keep),
           "kept": torch.where(held, kept, torch.full_like(kept, -1)).int(),
           "acc": torch.nn.functional.pad(torch.where(held, st["acc"].gather(2, at),
                                                      torch.zeros_like(st["acc"][..., :1])),
                                          (0, dcap - keep))}
    rows = at[..., None].expand(s, kv, keep, d)
    for name in ("k", "v"):
        bytes_ = st[name] if name == "k" else st[name].transpose(3, 4).reshape(s, kv, cap, d)
        x = _value(bytes_.gather(2, rows), fmt) * st[name + "_scale"].gather(2, at // block)[..., None]
        x = torch.where(held[..., None], x, torch.zeros_like(x))
        top = torch.nn.functional.pad(x.abs().amax(3), (0, dcap - keep))
        scale = _scale(top.reshape(s, kv, dcap // block, block).amax(3), fmt)
        scale = scale.repeat_interleave(block, 2)[:, :, :keep, None]
        y = _value(_encode(x, scale, fmt), fmt) * scale
        # the newest `keep` tokens: a sequence that holds fewer has its own at the end
        move = torch.arange(keep, device=DEV) - (keep - got["lens"][:, None])
        y = y.gather(2, move.clamp(min=0)[:, None, :, None].expand_as(y))
        got[name] = torch.where((move >= 0)[:, None, :, None], y, torch.zeros_like(y))
    return got


def _plain_logprobs(st):
    x, top = st["logits"], st["case"]["top"]
    vocab = x.shape[1]
    e = x - x.amax(1, keepdim=True)
    w = e.exp()
    z = w.sum(1)
    lp = e.gather(1, st["targets"][:, None].long())[:, 0] - z.log()
    key = (_order(x) << 20) + (vocab - torch.arange(vocab, device=DEV))
    ids = key.topk(top, 1).indices if top else key[:, :0]
    return {"logprob": lp, "entropy": z.log() - (w * e).sum(1) / z, "top_ids": ids.int(),
            "top_logprobs": e.gather(1, ids) - z.log()[:, None]}


def _run_plain(st):
    return {"attend": _plain_attend, "append": _plain_append, "weigh": _plain_weigh,
            "evict": _plain_evict, "logprobs": _plain_logprobs}[st["case"]["kind"]](st)


# ---- the definitions in 64 bits ----------------------------------------------------------

def _held64(codes, scales, case, seq, n, is_v):
    """The first n tokens of one sequence, [kv, n, d]: the products that the cache's codes and
    scales stand for, which are fp32 numbers."""
    if is_v:
        tiles = -(-n // TILE)
        codes = codes[seq, :, :tiles].permute(0, 1, 3, 2).reshape(case["kv"], tiles * TILE, -1)
    else:
        codes = codes[seq]
    codes = codes[:, :n].contiguous()
    whole = codes.view(torch.int8 if case["fmt"] == "i8" else torch.float8_e4m3fn)
    each = scales[seq][:, torch.arange(n, device=DEV) // case["block"]]
    return (whole.float() * each[..., None]).double()


def _grid(fmt):
    """Every value a code stands for, in order, with the middles between neighbours."""
    if fmt == "i8":
        v = torch.arange(-127, 128, dtype=torch.float64, device=DEV)
    else:
        m = torch.arange(0, 127, dtype=torch.uint8, device=DEV)  # 127 is NaN
        p = m.view(torch.float8_e4m3fn).double()
        v = torch.cat([-p.flip(0)[:-1], p])
    return v, (v[1:] + v[:-1]) / 2


def _nearest(y, fmt):
    v, mid = _grid(fmt)
    zero = len(v) // 2  # position of 0; a code is even where its distance from it is
    i = torch.bucketize(y.contiguous(), mid)  # values up to a middle go to its lower neighbour
    up = (i < len(mid)) & ((i - zero) % 2 != 0) & (y == mid[i.clamp(max=len(mid) - 1)])
    return v[i + up.long()]


def _exact_scale(top, fmt):
    return torch.clamp((top / CODE_MAX[fmt]).float(), min=FLOOR)


def _exact_append(case, st):
    """Blocks of a sequence one after the other."""
    kv, d, block, fmt, back = case["kv"], case["d"], case["block"], case["fmt"], _back(case)
    out = {"k": [], "v": [], "k_scale": st["k_scale"].clone(), "v_scale": st["v_scale"].clone()}
    for s, (ln, cnt) in enumerate(zip(_lens(case), _counts(case))):
        for name in ("k", "v"):
            old = _held64(st[name], st[name + "_scale"], case, s, ln, name == "v")
            new = st[name + "_new"][s, :cnt].permute(1, 0, 2).double()
            res, start = old.clone(), ln - cnt
            for b in range(start // block, -(-ln // block)):
                t0, t1, a = b * block, min(ln, (b + 1) * block), max(start, b * block)
                x = new[:, a - start:t1 - start]
                sc = _exact_scale(x.abs().amax((1, 2)), fmt)
                if a > t0:
                    was = st[name + "_scale"][s, :, b]
                    sc = torch.maximum(sc, was)
                    z = sc.double()[:, None, None]
                    again = (_nearest(old[:, t0:a] / z, fmt).float() * sc[:, None, None]).double()
                    res[:, t0:a] = torch.where((sc > was)[:, None, None], again, old[:, t0:a])
                y = _nearest(x / sc.double()[:, None, None], fmt).float() * sc[:, None, None]
                res[:, a:t1] = y.double()
                out[name + "_scale"][s, :, b] = sc
            whole = torch.zeros(kv, back, d, dtype=torch.float64, device=DEV)
            m = min(back, ln)
            whole[:, back - m:] = res[:, ln - m:]
            out[name].append(whole)
    return {n: torch.stack(v) if isinstance(v, list) else v.double() for n, v in out.items()}


def _exact_attend(case, st, weigh):
    n, h, kv, cap = case["n"], case["heads"], case["kv"], case["cap"]
    group, d = h // kv, case["d"]
    f64 = {"dtype": torch.float64, "device": DEV}
    out, lse = torch.zeros(case["seqs"], n, h, d, **f64), \
        torch.full((case["seqs"], h, n), -math.inf, **f64)
    acc = torch.zeros(case["seqs"], kv, cap, **f64)
    for s, (ln, cnt) in enumerate(zip(_lens(case), _counts(case))):
        if not ln:
            continue
        keys = _held64(st["k"], st["k_scale"], case, s, ln, False)
        vals = None if weigh else _held64(st["v"], st["v_scale"], case, s, ln, True)
        far = torch.arange(ln, device=DEV)[None] >= \
            ln - cnt + 1 + torch.arange(cnt, device=DEV)[:, None]
        for j in range(h):
            q = st["q"][s, :cnt, j].double()
            x = (q @ keys[j // group].T.contiguous()) / math.sqrt(d)
            x[far] = -math.inf
            if weigh:
                y = x - st["lse"][s, j, :cnt, None].double()
                acc[s, j // group, :ln] += y.exp().sum(0)
            else:
                l = torch.logsumexp(x, 1)
                lse[s, j, :cnt] = l
                out[s, :cnt, j] = (x - l[:, None]).exp() @ vals[j // group]
        if weigh:
            acc[s, :, :ln] += st["acc"][s, :, :ln].double()
    return {"acc": acc} if weigh else {"out": out, "lse": lse}


def _exact_evict(case, st):
    keep, recent, kv, d = case["keep"], case["recent"], case["kv"], case["d"]
    block, fmt = case["block"], case["fmt"]
    s_, f64 = case["seqs"], {"dtype": torch.float64, "device": DEV}
    out = {"k": torch.zeros(s_, kv, keep, d, **f64), "v": torch.zeros(s_, kv, keep, d, **f64),
           "acc": torch.zeros(s_, kv, -(-keep // 128) * 128, **f64), "kept": None, "lens": None}
    for s, ln in enumerate(_lens(case)):
        held = {t: _held64(st[t], st[t + "_scale"], case, s, ln, t == "v") for t in ("k", "v")}
        m = min(ln, keep)
        for j in range(kv):
            w = st["acc"][s, j, :ln].double()
            if ln > keep:
                best = torch.sort(w[:ln - recent], descending=True, stable=True).indices
                ids = torch.cat([best[:keep - recent], torch.arange(ln - recent, ln, device=DEV)])
                ids = ids.sort().values
            else:
                ids = torch.arange(ln, device=DEV)
            out["acc"][s, j, :m] = w[ids]
            for t in ("k", "v"):
                x = torch.zeros(-(-m // block) * block, d, **f64)
                x[:m] = held[t][j, ids]
                x = x.reshape(-1, block, d)
                sc = _exact_scale(x.abs().amax((1, 2)), fmt)[:, None, None]
                y = (_nearest(x / sc.double(), fmt).float() * sc).double().reshape(-1, d)
                out[t][s, j, keep - m:] = y[:m]
    return out


def _exact_logprobs(case, st):
    rows = [[], [], []]
    for x, y in zip(st["logits"].split(64), st["targets"].split(64)):
        lp = torch.log_softmax(x.double(), 1)
        rows[0].append(lp.gather(1, y[:, None].long())[:, 0])
        rows[1].append(-(lp.exp() * lp).sum(1))
        rows[2].append(lp.topk(case["top"], 1).values)
    return {"logprob": torch.cat(rows[0]), "entropy": torch.cat(rows[1]), "top_ids": None,
            "top_logprobs": torch.cat(rows[2])}


def exact(case, seed):
    kind = case["kind"]
    st = prepare(case, seed)
    if kind == "append":
        return _exact_append(case, st)
    if kind in ("attend", "weigh"):
        return _exact_attend(case, st, kind == "weigh")
    return _exact_evict(case, st) if kind == "evict" else _exact_logprobs(case, st)
