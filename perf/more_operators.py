"""The operators of a paged key/value cache, as cases that can be timed and checked.

Each case is a call (or the calls of one step) on resident tensors of one GPU:

* `append` - new K and V rows go into pages, K and Q turned by their positions on the way;
* `attend` - attention of new queries over the pages, with capped scores, a bias by distance, a
  window, a prefix that all rows see, documents side by side or a tree of drafted tokens;
* `accept` - a drafted tree's rows are appended, then the path that the model's choices take is
  kept: its K and V move to the front.

`own` chooses between the framework's calls and the plain form in elementary torch operations;
`exact` states the definition again in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA = 10000.0


def listed():
    small = {"heads": 32, "kv": 4, "d": 64}   # the TinyLlama-shaped decoder
    large = {"heads": 32, "kv": 8, "d": 128}
    return [
        # the token each sequence of a batch just made: latency
        {"name": "append_b64_step", "kind": "append", **small, "seqs": 64, "page": 16, "lo": 3,
         "hi": 1020, "n": 1, "ragged": False, "fmt": "f32", "rot": 64, "inter": False},
        # prompts of a batch, of different lengths, half of each head turned
        {"name": "append_b4_prompt", "kind": "append", **large, "seqs": 4, "page": 64, "lo": 2001,
         "hi": 4000, "n": 2000, "ragged": True, "fmt": "bf16", "rot": 64, "inter": True},
        # one decode step early in a chat: latency
        {"name": "attend_b1_300", "kind": "attend", **small, "seqs": 1, "page": 16, "lo": 300,
         "hi": 300, "n": 1, "ragged": False, "fmt": "f32"},
        # a decode step of a batch whose conversations differ in length, with capped scores; one
        # slot is empty
        {"name": "attend_b24_capped", "kind": "attend", **large, "seqs": 24, "page": 64, "lo": 0,
         "hi": 8100, "n": 1, "ragged": False, "fmt": "bf16", "cap": 30.0},
        # a decode step over long documents: a cache of more than 4 GiB
        {"name": "attend_b16_131k", "kind": "attend", **large, "seqs": 16, "page": 128,
         "lo": 128001, "hi": 131072, "n": 1, "ragged": False, "fmt": "f16"},
        # a chunk of a prompt behind what is cached already: matrix work in fp32
        {"name": "attend_chunk_512", "kind": "attend", **large, "seqs": 1, "page": 64, "lo": 8190,
         "hi": 8190, "n": 512, "ragged": False, "fmt": "f32"},
        # short documents packed into one long prompt, the bias by distance
        {"name": "attend_documents_4k", "kind": "attend", **large, "seqs": 1, "page": 64,
         "lo": 4090, "hi": 4090, "n": 4090, "ragged": False, "fmt": "bf16", "docs": 700,
         "bias": True},
        # prompts whose first part all rows see, the rest within a window
        {"name": "attend_prefix_window", "kind": "attend", **small, "seqs": 3, "page": 32,
         "lo": 500, "hi": 1501, "n": 1501, "ragged": True, "fmt": "f16", "prefix": 257,
         "window": 400},
        # a drafted tree of one conversation: latency
        {"name": "tree_b1_24", "kind": "attend", **small, "seqs": 1, "page": 16, "lo": 700,
         "hi": 700, "n": 24, "ragged": False, "fmt": "f32", "tree": True},
        # the drafted trees of a batch
        {"name": "tree_b16_60", "kind": "attend", **large, "seqs": 16, "page": 64, "lo": 1000,
         "hi": 4100, "n": 60, "ragged": True, "fmt": "bf16", "tree": True},
        # what of a drafted tree is kept: latency
        {"name": "accept_b1_24", "kind": "accept", **small, "seqs": 1, "page": 16, "lo": 700,
         "hi": 700, "n": 24, "ragged": False, "fmt": "f32", "rot": 64, "inter": False},
        {"name": "accept_b64_60", "kind": "accept", **large, "seqs": 64, "page": 64, "lo": 100,
         "hi": 1000, "n": 60, "ragged": True, "fmt": "bf16", "rot": 128, "inter": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "append", "accept"])
    kv, d = rng.choice([(4, 64), (8, 128), (8, 64), (2, 128)])
    case = {"kind": kind, "kv": kv, "d": d, "heads": kv * rng.choice([1, 4, 4, 7, 8 if kv < 8 else 4]),
            "fmt": rng.choice(["f32", "f16", "bf16", "bf16"]),
            "page": rng.choice([16, 16, 32, 64, 128, 256])}
    if kind != "attend":
        case.update(rot=rng.choice([d, d, d // 2, 24]), inter=rng.random() < 0.4)
        if kind == "accept":
            n = _log(rng, 1, 200)
            return {**case, "n": n, "seqs": _log(rng, 1, 64), "lo": n, "hi": n + _log(rng, 1, 1000),
                    "ragged": rng.random() < 0.5}
        n = rng.choice([1, 1, _log(rng, 2, 2000)])
        return {**case, "n": n, "seqs": _log(rng, 1, 64 if n < 64 else 4), "lo": n,
                "hi": n + _log(rng, 1, 2000), "ragged": rng.random() < 0.5}
    form = rng.choice(["step", "step", "chunk", "tree"])
    if form == "step":  # decode steps, or a few tokens at a time
        n, seqs = rng.choice([1, 1, 1, rng.randint(2, 8)]), _log(rng, 1, 64)
        hi = max(n, _log(rng, 16, 400_000 // seqs))
        lo = rng.choice([0, hi // 3, hi])
    elif form == "chunk":
        n, seqs = _log(rng, 1, 512), 1 + (rng.random() < 0.4)
        hi = n + _log(rng, 1, 7600)
        lo = rng.choice([n, hi])
        if rng.random() < 0.4:
            case["docs"] = _log(rng, 16, hi)
        elif rng.random() < 0.4:
            case["prefix"] = rng.randint(1, hi)
    else:
        n, seqs = _log(rng, 1, 200), _log(rng, 1, 16)
        hi = n + _log(rng, 1, 4000)
        lo = rng.choice([n, hi])
        case["tree"] = True
    if rng.random() < 0.3:
        case["window"] = _log(rng, 1, 2 * hi)
        if rng.random() < 0.5 and "docs" not in case:
            case["prefix"] = rng.randint(1, 64)
    if rng.random() < 0.3:
        case["cap"] = rng.choice([5.0, 30.0, 50.0])
    if rng.random() < 0.3:
        case["bias"] = True
    return {**case, "n": n, "seqs": seqs, "lo": lo, "hi": hi, "ragged": n > 1 and rng.random() < 0.5}


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


def _pages(case):
    """Pages of a sequence's table, and pages in all: what is held and a few that are free."""
    page = case["page"]
    return -(-case["hi"] // page), sum(-(-ln // page) for ln in _lens(case)) + 3


def _parents(case):
    """Each sequence's tree: node 0 is the token that is settled, the others hang on earlier ones."""
    r = random.Random(11 * case["seqs"] + case["n"])
    return [[-1] + [r.randrange(i) for i in range(1, case["n"])] for _ in range(case["seqs"])]


def _depths(parents):
    out = []
    for p in parents:
        d = [0] * len(p)
        for i in range(1, len(p)):
            d[i] = d[p[i]] + 1
        out.append(d)
    return out


def _firsts(case):
    """The first token each row sees: its document's, documents being of 1 to 2 * docs tokens."""
    out = []
    for ln, cnt in zip(_lens(case), _counts(case)):
        r, starts = random.Random(ln + 5 * case["docs"]), [0]
        while starts[-1] < ln:
            starts.append(starts[-1] + r.randint(1, 2 * case["docs"]))
        own_, j = [], 0
        for t in range(ln):
            if starts[j + 1] <= t:
                j += 1
            own_.append(starts[j])
        out.append((own_[ln - cnt:] + [0] * case["n"])[:case["n"]])
    return out


def _seen(case):
    """(row, token) pairs, and tokens that any row of their sequence sees."""
    window, pairs, tokens = case.get("window") or 1 << 30, 0, 0
    depths = _depths(_parents(case)) if case.get("tree") else None
    firsts = _firsts(case) if case.get("docs") else None
    for s, (ln, cnt) in enumerate(zip(_lens(case), _counts(case))):
        base, prefix, low = ln - cnt, min(case.get("prefix") or 0, ln), ln
        for i in range(cnt):
            at = base + (depths[s][i] if depths else i)
            first = firsts[s][i] if firsts else 0
            lo = max(first, at - window + 1)
            low = min(low, lo)
            got = max(0, at + 1 - lo)  # a tree's row: the context and its path
            if prefix > lo:  # the window begins within the prefix
                got += max(0, (base if depths else prefix) - (at + 1)) if prefix > at else 0
                lo = max(first, 0)
                got += max(0, min(prefix, at - window + 1) - lo)
            else:
                got += max(0, prefix - first)
            pairs += got
        if cnt:
            tokens += ln - max(0, low) + max(0, min(prefix, low))
    return pairs, tokens


def work(case):
    kv, d, h = case["kv"], case["d"], case["heads"]
    size = TYPES[case["fmt"]].itemsize
    new = sum(_counts(case))
    if case["kind"] == "attend":
        pairs, tokens = _seen(case)
        return {"bytes": 2.0 * tokens * kv * d * size + new * h * (8.0 * d + 4),
                "flops": 4.0 * d * h * pairs}
    rows = {"bytes": new * d * (kv * (8.0 + 2 * size) + 8.0 * h),
            "flops": 3.0 * new * case["rot"] * (kv + h)}
    if case["kind"] == "accept":  # a path's rows twice, and the trees
        rows["bytes"] += 4.0 * kv * d * size * sum(c > 0 for c in _counts(case)) * 2 + 16.0 * new
    return rows


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1013 + 29)
    s, kv, d, page, n, h = (case[x] for x in ("seqs", "kv", "d", "page", "n", "heads"))

    def randn(*shape, dtype=torch.float32):
        return torch.empty(shape, device=DEV, dtype=dtype).normal_(generator=g)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    per, total = _pages(case)
    lens = _lens(case)
    st = {"case": case, "k": randn(total, kv, page, d, dtype=TYPES[case["fmt"]]),
          "v": randn(total, kv, page, d, dtype=TYPES[case["fmt"]]), "lens": ints(lens),
          "counts": ints(_counts(case)), "q": randn(s, n, h, d), "out": torch.zeros(s, n, h, d, device=DEV)}
    # pages in the order in which a running server hands them out; behind the last there is none
    free, table = torch.randperm(total, generator=g, device=DEV).tolist(), []
    for ln in lens:
        held = -(-ln // page)
        table.append([free.pop() for _ in range(held)] + [-1] * (per - held))
    st["table"] = ints(table)
    if case["kind"] == "attend":
        st["lse"] = torch.full((s, h, n), -math.inf, device=DEV)
        if case.get("bias"):
            st["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device=DEV) / h)
        if case.get("prefix"):
            st["prefix"] = ints([case["prefix"]] * s)
        if case.get("docs"):
            st["first"] = ints(_firsts(case))
        if case.get("tree"):
            st["parents"] = ints(_parents(case))
    else:
        st["k_new"], st["v_new"] = randn(s, n, kv, d), randn(s, n, kv, d)
        j = torch.arange(0, case["rot"], 2, dtype=torch.float64, device=DEV)
        st["inv_freq"] = (THETA ** (-j / case["rot"])).float()
        if case["kind"] == "accept":
            parents = _parents(case)
            st["parents"], st["offsets"] = ints(parents), ints(_depths(parents))
            # drafted ids, and what the model chose behind each: often the first child's id
            r = random.Random(seed)
            ids = [[r.randrange(32000) for _ in range(n)] for _ in range(s)]
            picks = []
            for p, t in zip(parents, ids):
                child = {}
                for i in range(n - 1, 0, -1):
                    child[p[i]] = t[i]
                picks.append([child[i] if i in child and r.random() < 0.8 else r.randrange(32000)
                              for i in range(n)])
            st["tokens"], st["choices"] = ints(ids), ints(picks)
            st["path"] = ints([[0] * n] * s)
            st["accepted"], st["next"], st["lens_out"] = ints([0] * s), ints([0] * s), ints([0] * s)
    if own:
        _hold(st)
    return st


def _hold(st):
    """What a program keeps for its calls: the context, the cache and its tensors."""
    from spirv_inference_amd import Context, DeviceTensor, PagedCache
    global _CTX
    if _CTX is None:
        _CTX = Context("any")
    kinds = {torch.float32: "<f4", torch.int32: "<i4", torch.float16: "<u2", torch.bfloat16: "<u2"}
    t = {n: DeviceTensor(_CTX, x.numel(), kinds[x.dtype], ptr=x.data_ptr(), owned=False)
         for n, x in st.items() if isinstance(x, torch.Tensor)}
    c = st["case"]
    st["t"] = t
    st["cache"] = PagedCache(_CTX, c["seqs"], c["kv"], c["d"], st["k"].shape[0], c["page"],
                             st["table"].shape[1], fmt=c["fmt"], k=t["k"], v=t["v"],
                             table=t["table"], lengths=t["lens"])


_CTX = None


def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    c, t, cache = st["case"], st["t"], st["cache"]
    if c["kind"] == "attend":
        cache.attend(t["q"], t["out"], c["heads"], c["n"], counts=t["counts"], lse=t["lse"],
                     cap=c.get("cap"), slopes=t.get("slopes"), window=c.get("window"),
                     prefix=t.get("prefix"), first=t.get("first"), parents=t.get("parents"))
        return {"out": st["out"], "lse": st["lse"]}
    cache.append(t["k_new"], t["v_new"], c["n"], counts=t["counts"], q=t["q"], q_out=t["out"],
                 n_heads=c["heads"], inv_freq=t["inv_freq"], rot=c["rot"], interleaved=c["inter"],
                 offsets=t.get("offsets"))
    got = {"q": st["out"], "k": st["k"], "v": st["v"]}
    if c["kind"] == "append":
        return got
    cache.accept(t["parents"], t["tokens"], t["choices"], c["n"], t["path"], t["accepted"],
                 t["next"], counts=t["counts"], lengths_out=t["lens_out"])
    return {**got, "path": st["path"], "accepted": st["accepted"], "next": st["next"],
            "lens": st["lens_out"]}


# ---- the plain forms ---------------------------------------------------------------------

def _held(pages, st):
    """What the pages hold of each sequence, [seqs, kv, tokens, d]; zeros where there is no page."""
    x = pages[st["table"].clamp(min=0).long()].float()
    x = x.masked_fill_((st["table"] < 0)[:, :, None, None, None], 0)
    s, per, kv, page, d = x.shape
    return x.transpose(1, 2).reshape(s, kv, per * page, d)


def _ancestors(parents):
    """[seqs, n, n]: whether row i is node j or hangs below it."""
    n = parents.shape[1]
    step = torch.nn.functional.one_hot(parents.long() + 1, n + 1)[..., 1:].double()
    paths = torch.linalg.matrix_power(step + torch.eye(n, device=DEV, dtype=torch.float64), n)
    return paths > 0


def _plain_attend(st):
    c = st["case"]
    s, n, h, kv, d = c["seqs"], c["n"], c["heads"], c["kv"], c["d"]
    k, v = _held(st["k"], st), _held(st["v"], st)
    cap = k.shape[2]
    q = st["q"].reshape(s, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(s, kv, h // kv * n, d)
    x = torch.matmul(q * d ** -0.5, k.transpose(2, 3).contiguous()).reshape(s, h, n, cap)
    if c.get("cap"):
        x = torch.tanh(x / c["cap"]) * c["cap"]
    i = torch.arange(n, device=DEV)
    t = torch.arange(cap, device=DEV)
    base = (st["lens"] - st["counts"])[:, None]
    at, where = base + i, t.expand(s, cap)  # positions of rows and tokens
    if c.get("tree"):
        kin = _ancestors(st["parents"])
        depth = (kin.sum(2) - 1).int()
        new = (t - base).clamp(0, n - 1)
        at = base + depth
        where = torch.where(t >= base, base + depth.gather(1, new), t)
        own_ = kin.gather(2, new[:, None].expand(s, n, cap).long()) | (t < base)[:, None]
    else:
        own_ = t <= at[:, :, None]
    far = at[:, :, None] - where[:, None, :]
    sees = own_ & (far < (c.get("window") or 1 << 30))
    if c.get("prefix"):
        head = t < st["prefix"][:, None]
        sees = sees | (head[:, None] & ((t < base)[:, None] | own_ if c.get("tree") else True))
    if c.get("docs"):
        sees = sees & (t >= st["first"][:, :, None])
    sees = sees & (t < st["lens"][:, None])[:, None] & (i < st["counts"][:, None])[:, :, None]
    if c.get("bias"):
        x = x - st["slopes"][:, None, None] * far.abs()[:, None].float()
    x = x.masked_fill_(~sees[:, None], -math.inf)
    m = x.amax(3, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    p = x.sub_(m).exp_()
    z = p.sum(3, keepdim=True)
    o = torch.matmul(p.reshape(s, kv, -1, cap), v).reshape(s, h, n, d)
    o = o / torch.where(z > 0, z, torch.ones_like(z))
    return {"out": o.transpose(1, 2).contiguous(), "lse": (m + z.log())[..., 0]}


def _turn(x, angle, inter):
    """Rows x [..., d] turned by angles [seqs, n, rot / 2] in 64 bits, over all heads."""
    rot = 2 * angle.shape[2]
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    y0, y1 = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([y0, y1], -1).flatten(-2) if inter else torch.cat([y0, y1], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_append(st):
    c = st["case"]
    s, n, page = c["seqs"], c["n"], c["page"]
    i = torch.arange(n, device=DEV)
    base = (st["lens"] - st["counts"])[:, None]
    pos = base + st.get("offsets", i)
    angle = pos.double()[:, :, None] * st["inv_freq"].double()
    real = i < st["counts"][:, None]
    place = base + i
    own_page = st["table"].gather(1, (place // page).clamp(max=st["table"].shape[1] - 1).long())
    to = (own_page[real].long(), slice(None), (place % page)[real].long())
    st["k"][to] = _turn(st["k_new"], angle, c["inter"])[real].to(st["k"].dtype)
    st["v"][to] = st["v_new"][real].to(st["v"].dtype)
    q = torch.where(real[:, :, None, None], _turn(st["q"], angle, c["inter"]), st["out"])
    return {"q": q, "k": st["k"], "v": st["v"]}


def _plain_accept(st):
    c = st["case"]
    got = _plain_append(st)
    s, n, page = c["seqs"], c["n"], c["page"]
    i = torch.arange(n, device=DEV)
    real = i < st["counts"][:, None]
    # a node is taken if it is the first of its siblings with the id chosen behind its parent, and
    # all nodes above it are
    up = st["parents"].clamp(min=0).long()
    good = (st["tokens"] == st["choices"].gather(1, up)) & real
    twin = (up[:, :, None] == up[:, None]) & (i[:, None] > i) & good[:, None, :]
    good = good & ~(twin & (i > 0)).any(2)
    good[:, 0] = real[:, 0]
    taken = ~(_ancestors(st["parents"]) & ~good[:, None]).any(2)
    accepted = taken.sum(1).int()
    path = torch.where(taken, i, n).sort(1).values
    last = path.gather(1, (accepted - 1).clamp(min=0).long()[:, None]).clamp(max=n - 1)
    nxt = torch.where(accepted > 0, st["choices"].gather(1, last.long())[:, 0], -1)
    base = (st["lens"] - st["counts"])[:, None]
    keep = path < n
    src, dst = base + path.clamp(max=n - 1), base + i
    last_page = st["table"].shape[1] - 1
    from_page = st["table"].gather(1, (src // page).clamp(max=last_page).long())[keep].long()
    to_page = st["table"].gather(1, (dst // page).clamp(max=last_page).long())[keep].long()
    to, source = (dst % page)[keep].long(), (src % page)[keep].long()
    st["k"][to_page, :, to] = st["k"][from_page, :, source]
    st["v"][to_page, :, to] = st["v"][from_page, :, source]
    return {**got, "path": torch.where(keep, path, -1).int(), "accepted": accepted,
            "next": nxt.int(), "lens": (base[:, 0] + accepted).int()}


def _run_plain(st):
    return {"attend": _plain_attend, "append": _plain_append,
            "accept": _plain_accept}[st["case"]["kind"]](st)


# ---- the definitions in 64 bits ----------------------------------------------------------

def _tokens64(pages, st, seq, n):
    """The first n tokens of one sequence, [kv, n, d]."""
    own_ = st["table"][seq, :-(-n // st["case"]["page"])].long()
    x = pages[own_].double().permute(1, 0, 2, 3)
    return x.reshape(x.shape[0], -1, x.shape[3])[:, :n].contiguous()


def _exact_attend(case, st):
    n, h, kv, d = case["n"], case["heads"], case["kv"], case["d"]
    f64 = {"dtype": torch.float64, "device": DEV}
    out = torch.zeros(case["seqs"], n, h, d, **f64)
    lse = torch.full((case["seqs"], h, n), -math.inf, **f64)
    parents = _parents(case) if case.get("tree") else None
    firsts = _firsts(case) if case.get("docs") else None
    for s, (ln, cnt) in enumerate(zip(_lens(case), _counts(case))):
        if not ln:
            continue
        base, t = ln - cnt, torch.arange(ln, device=DEV)
        pos_q, pos_k = base + torch.arange(cnt, device=DEV), t
        if parents:
            path = []
            for i in range(cnt):
                path.append((path[parents[s][i]] if i else []) + [i])
            sees = torch.zeros(cnt, ln, dtype=torch.bool)
            sees[:, :base] = True
            for i, nodes in enumerate(path):
                sees[i, [base + j for j in nodes]] = True
            sees = sees.to(DEV)
            deep = torch.tensor([len(p) - 1 for p in path], device=DEV)
            pos_q, pos_k = base + deep, torch.cat([t[:base], base + deep])
        else:
            sees = t[None] <= pos_q[:, None]
        gap = (pos_q[:, None] - pos_k[None]).double()
        kin = sees
        if case.get("window"):
            sees = sees & (gap < case["window"])
        if case.get("prefix"):
            sees = sees | ((t < case["prefix"])[None] & (kin if parents else True))
        if firsts:
            sees = sees & (t[None] >= torch.tensor(firsts[s][:cnt], device=DEV)[:, None])
        keys, vals = _tokens64(st["k"], st, s, ln), _tokens64(st["v"], st, s, ln)
        for j in range(h):
            x = (st["q"][s, :cnt, j].double() @ keys[j // (h // kv)].T.contiguous()) / math.sqrt(d)
            if case.get("cap"):
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case.get("bias"):
                x = x - float(st["slopes"][j]) * gap.abs()
            x = torch.where(sees, x, torch.full_like(x, -math.inf))
            l = torch.logsumexp(x, 1)
            lse[s, j, :cnt] = l
            w = torch.exp(x - torch.where(torch.isfinite(l), l, torch.zeros_like(l))[:, None])
            out[s, :cnt, j] = w @ vals[j // (h // kv)]
    return {"out": out, "lse": lse}


def _exact_append(case, st):
    """Row by row of a sequence's new tokens, heads together, as complex products."""
    half = case["rot"] // 2
    res = {"q": st["out"].double(), "k": st["k"].double(), "v": st["v"].double()}
    freq = st["inv_freq"].double()
    for s, (ln, cnt) in enumerate(zip(_lens(case), _counts(case))):
        rows = torch.arange(cnt, device=DEV)
        off = st["offsets"][s, :cnt].double() if "offsets" in st else rows.double()
        turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV),
                           (ln - cnt + off)[:, None, None] * freq)
        at = ln - cnt + rows
        page, slot = st["table"][s][at // case["page"]].long(), at % case["page"]
        for name, x in (("q", st["q"]), ("k", st["k_new"])):
            x = x[s, :cnt].double()
            y, head = x.clone(), x[..., :case["rot"]]
            if case["inter"]:
                z = torch.view_as_complex(head.reshape(*head.shape[:-1], half, 2).contiguous()) * turn
                y[..., :case["rot"]] = torch.view_as_real(z).reshape(head.shape)
            else:
                z = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) * turn
                y[..., :half], y[..., half:case["rot"]] = z.real, z.imag
            if name == "q":
                res["q"][s, :cnt] = y
            else:
                res["k"][page, :, slot] = y
        res["v"][page, :, slot] = st["v_new"][s, :cnt].double()
    return res


def _exact_accept(case, st):
    res = _exact_append(case, st)
    par, ids, picks = _parents(case), st["tokens"].tolist(), st["choices"].tolist()
    table, page = st["table"].tolist(), case["page"]
    for s, (ln, cnt) in enumerate(zip(_lens(case), _counts(case))):
        node, depth = (0, 0) if cnt else (None, 0)
        while node is not None:
            a, b = ln - cnt + node, ln - cnt + depth
            for x in (res["k"], res["v"]):
                x[table[s][b // page], :, b % page] = x[table[s][a // page], :, a % page].clone()
            here = node
            node = next((j for j in range(here + 1, cnt)
                         if par[s][j] == here and ids[s][j] == picks[s][here]), None)
            depth += 1
    return {**res, "path": None, "accepted": None, "next": None, "lens": None}


def exact(case, seed):
    st = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append,
            "accept": _exact_accept}[case["kind"]](case, st)
