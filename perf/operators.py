"""Cases of the paged key/value cache operators: what is run, on which inputs, and what it has to move and compute.

The cache keeps keys and values in pages [layers][pages][kv_heads][page_size][head_dim]; a sequence owns the pages that its
row of the page table lists, `seq_len` tokens of them.  Three operators work on it:

  append     the norms of queries and keys per head and the rotation by position, the keys and values written to their pages
  attention  new tokens of each sequence (one, or a chunk) attend to the sequence's pages
  pages      the bookkeeping on the device and the page moves: extend, fork, free, compact, copy

`run` computes them in plain torch operations, or, with `own` set, through the package's `kv_cache.KVCache`.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


# ---- cases --------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one user's decode step: the smallest call, latency alone
        dict(name="append decode 1", op="append", type="bf16", q_heads=28, kv_heads=4, dim=128, page=16, seqs=1,
             q_min=1, q_max=1, kv_min=1000, kv_max=1000, norm=True, rot=128, interleaved=False),
        # a full decode batch on long contexts
        dict(name="append decode 64", op="append", type="f16", q_heads=32, kv_heads=8, dim=128, page=32, seqs=64,
             q_min=1, q_max=1, kv_min=1000, kv_max=100000, norm=True, rot=64, interleaved=True),
        # prompts being read in, of odd lengths
        dict(name="append prompts", op="append", type="bf16", q_heads=28, kv_heads=4, dim=128, page=16, seqs=5,
             q_min=777, q_max=2500, kv_min=2600, kv_max=9000, norm=True, rot=128, interleaved=False),
        # one user's decode step on a short context
        dict(name="attention decode 1", op="attention", type="bf16", q_heads=28, kv_heads=4, dim=128, page=16, seqs=1,
             q_min=1, q_max=1, kv_min=1000, kv_max=1000, causal=True, window=0),
        # a full decode batch, ragged contexts: the cache's bytes are the work
        dict(name="attention decode 64", op="attention", type="bf16", q_heads=32, kv_heads=8, dim=128, page=16, seqs=64,
             q_min=1, q_max=1, kv_min=2000, kv_max=15000, causal=True, window=0),
        # one user, one very long context: few rows, a long axis to split
        dict(name="attention decode long", op="attention", type="f16", q_heads=28, kv_heads=4, dim=128, page=64, seqs=1,
             q_min=1, q_max=1, kv_min=131071, kv_max=131071, causal=True, window=0),
        # chunks of long prompts: the matrix products are the work
        dict(name="attention chunks", op="attention", type="bf16", q_heads=32, kv_heads=8, dim=128, page=16, seqs=2,
             q_min=1900, q_max=2048, kv_min=14000, kv_max=16000, causal=True, window=0),
        # what a serving step holds in earnest: one chunk among decoding sequences
        dict(name="attention mixed", op="attention", type="f16", q_heads=16, kv_heads=4, dim=64, page=32, seqs=32,
             q_min=1, q_max=1, first=512, kv_min=700, kv_max=4000, causal=True, window=1000),
        # the f32 decoder's shape (12 heads of 64, contexts to 1024), prompts being read in
        dict(name="attention prompts f32", op="attention", type="f32", q_heads=12, kv_heads=12, dim=64, page=16, seqs=8,
             q_min=300, q_max=777, kv_min=800, kv_max=1000, causal=True, window=0),
        # room for the next token of a decode batch
        dict(name="pages extend 64", op="pages", kind="extend", type="bf16", kv_heads=4, dim=128, page=16, layers=2,
             pages=8192, seqs=64, kv_min=100, kv_max=1500, live=0.6, count=1),
        # several samples from each prompt: the pages are shared, the last one copied over all layers
        dict(name="pages fork 64", op="pages", kind="fork", type="bf16", kv_heads=4, dim=128, page=16, layers=28,
             pages=1536, seqs=16, kv_min=100, kv_max=1500, live=0.6, count=4),
        # a pool with holes, made dense again
        dict(name="pages compact", op="pages", kind="compact", type="bf16", kv_heads=4, dim=128, page=16, layers=8,
             pages=2048, seqs=24, kv_min=100, kv_max=1500, live=0.55, count=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "pages"])
    kind = rng.choice(["f32", "f16", "bf16", "bf16"])
    q_heads, kv_heads, dim = rng.choice([(12, 12, 64), (28, 4, 128), (32, 8, 128), (16, 2, 64), (16, 16, 80), (8, 1, 128),
                                         (6, 2, 96), (5, 5, 40), (40, 8, 128), (4, 4, 256), (9, 3, 64)])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if op == "append":
        seqs = _log(rng, 1, 64)
        chunk = rng.random() < 0.5
        q = _log(rng, 1, max(2, 8000 // seqs)) if chunk else 1
        q = min(q, 2500)
        kv = q + _log(rng, 1, 4000)
        return dict(op=op, type=kind, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, seqs=seqs, q_min=max(1, q // 2), q_max=q,
                    kv_min=q, kv_max=kv, norm=rng.random() < 0.8, rot=rng.choice([dim, dim, dim // 2, 0]), interleaved=rng.random() < 0.4)
    if op == "attention":
        mode = rng.choice(["decode", "decode", "chunk", "mixed"])
        seqs = _log(rng, 1, 64) if mode != "chunk" else _log(rng, 1, 8)
        # at most about 0.5 GB of the cache, 2 GB of scores, and 0.2 TFLOP
        kv_most = min(100000, int(5e8 / (seqs * kv_heads * dim * 2 * SIZE[kind])))
        kv = _log(rng, 17, max(40, kv_most))
        c = dict(op=op, type=kind, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, seqs=seqs, q_min=1, q_max=1)
        q = 1
        if mode != "decode":
            most = min(kv, 2048, int(5e8 / (seqs * q_heads * kv)), int(2e11 / (4.0 * seqs * q_heads * kv * dim)))
            q = _log(rng, 2, max(3, most)) if most > 2 else 2
            q = min(q, kv)
            if mode == "chunk":
                c.update(q_min=max(1, q // 2), q_max=q)
            else:
                c.update(first=q)
        c.update(kv_min=max(q, kv // 3), kv_max=max(kv, q), causal=rng.random() < 0.85, window=rng.choice([0, 0, 0, _log(rng, 8, 4000)]))
        return c
    what = rng.choice(["extend", "fork", "free", "compact", "copy"])
    layers = _log(rng, 1, 16)
    each = layers * kv_heads * page * dim * 2 * SIZE[kind]
    pages = max(64, min(_log(rng, 64, 8192), int(1.0e9 / each)))
    seqs = _log(rng, 1, min(64, pages // 16))
    most = max(page, int(pages * page * 0.5 / seqs))
    return dict(op=op, kind=what, type=kind, kv_heads=kv_heads, dim=dim, page=page, layers=layers, pages=pages, seqs=seqs,
                kv_min=max(1, most // 4), kv_max=max(1, most * 3 // 4), live=round(rng.uniform(0.5, 0.8), 2),
                count=rng.randint(1, 3) if what in ("extend", "fork") else 0)


def _spread(lo, hi, n, at=0.0):
    """n lengths between lo and hi, spread evenly in no order: a function of the case alone."""
    return [int(lo + (hi - lo) * ((at + (i + 1) * 0.6180339887498949) % 1.0)) if hi > lo else lo for i in range(n)]


def _lengths(case):
    """New tokens and tokens held (the new ones included) of each sequence."""
    n = case["seqs"]
    new = _spread(case.get("q_min", 1), case.get("q_max", 1), n, 0.3)
    if case.get("first"):
        new[n // 2] = case["first"]
    held = [max(a, b) for a, b in zip(_spread(case["kv_min"], case["kv_max"], n), new)]
    return new, held


def _pages_of(case, held):
    return [-(-h // case["page"]) for h in held]


# ---- inputs -------------------------------------------------------------------------------------------------------


def _normal(gen, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=dtype, device="cuda")
    x.normal_(0.0, scale, generator=gen)
    return x


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tables(case, held, gen, num_pages, max_seqs, room):
    """A page table whose sequences own pages in no order, the lengths and the reference counts."""
    need = _pages_of(case, held)
    order = torch.randperm(num_pages, generator=gen, device="cuda").to(torch.int32)
    rows = torch.full((max_seqs, max(need) + room), -1, dtype=torch.int32, device="cuda")
    ids = torch.randperm(max_seqs, generator=gen, device="cuda")[: len(held)]
    width = rows.shape[1]
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    col = torch.arange(width, device="cuda")
    used = col[None, :] < torch.tensor(need, device="cuda")[:, None]
    rows[ids] = torch.where(used, order[(first[:, None] + col[None, :]).clamp(max=num_pages - 1)], -1)
    lens = torch.zeros(max_seqs, dtype=torch.int32, device="cuda")
    lens[ids] = _ints(held)
    refs = torch.zeros(num_pages, dtype=torch.int32, device="cuda")
    refs[order[: sum(need)].long()] = 1
    return rows, lens, refs, ids.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, hk, d, page = TYPES[case["type"]], case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "pages":
        held = _spread(case["kv_min"], case["kv_max"], case["seqs"])
        most = int(case["pages"] * case["live"])
        while sum(_pages_of(case, held)) > most:  # as many sequences as the pool's live share holds
            held = [max(1, int(h * 0.9)) for h in held]
        max_seqs = case["seqs"] * (1 + max(1, case["count"]))
        rows, lens, refs, ids = _tables(case, held, gen, case["pages"], max_seqs, 2)
        shape = (case["layers"], case["pages"], hk, page, d)
        s = dict(case=case, k=_normal(gen, shape, dt), v=_normal(gen, shape, dt), rows0=rows, lens0=lens, refs0=refs, ids=ids,
                 rows=rows.clone(), lens=lens.clone(), refs=refs.clone(), status=torch.zeros(1, dtype=torch.int32, device="cuda"))
        rest = torch.ones(max_seqs, dtype=torch.bool, device="cuda")
        rest[ids.long()] = False
        empty = torch.argsort(rest.int(), descending=True, stable=True).to(torch.int32)  # ids of sequences that hold nothing first
        if case["kind"] == "extend":
            s["counts"] = _ints([case["count"]] * case["seqs"])
        elif case["kind"] == "fork":
            s["parents"] = ids.repeat_interleave(case["count"])
            s["children"] = empty[: case["seqs"] * case["count"]].contiguous()
        elif case["kind"] == "copy":
            order = torch.randperm(case["pages"], generator=gen, device="cuda").to(torch.int32)
            half = case["pages"] // 2
            s["src"], s["dst"] = order[:half].contiguous(), order[half: 2 * half].contiguous()
        return s
    new, held = _lengths(case)
    n, hq = case["seqs"], case["q_heads"]
    num_pages = sum(_pages_of(case, held)) + 3
    rows, lens, refs, ids = _tables(case, held, gen, num_pages, n + 2, 1)
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    s = dict(case=case, rows=rows, lens=lens, refs=refs, ids=ids, cu=None if max(new) == 1 else _ints(cu), cu_plain=_ints(cu),
             max_new=max(new), max_held=max(held), status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    shape = (1, num_pages, hk, page, d)
    if case["op"] == "append":
        # one buffer of a fused projection: queries, keys and values of a token side by side
        qkv = _normal(gen, (cu[-1], hq + 2 * hk, d), dt)
        s.update(k=torch.zeros(shape, dtype=dt, device="cuda"), v=torch.zeros(shape, dtype=dt, device="cuda"), qkv=qkv,
                 qw=(1 + _normal(gen, (d,), torch.float32, 0.1)).to(dt) if case["norm"] else None,
                 kw=(1 + _normal(gen, (d,), torch.float32, 0.1)).to(dt) if case["norm"] else None, inv=None)
        if case["rot"]:
            j = torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64)
            s["inv"] = (10000.0 ** (-2.0 * j / case["rot"])).float()
    else:
        s.update(k=_normal(gen, shape, dt), v=_normal(gen, shape, dt), q=_normal(gen, (cu[-1], hq, d), dt, 1.5))
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------


def _tokens(s, total):
    """Of each new token: its place in the list of sequences, its number among the sequence's new ones, its position."""
    cu = s["cu_plain"].long()
    t = torch.arange(total, device=cu.device)
    b = torch.searchsorted(cu[1:], t, right=True)
    i = t - cu[b]
    pos = s["lens"].long()[s["ids"].long()[b]] - (cu[b + 1] - cu[b]) + i
    return b, i, pos


def _rotate(x, angle, interleaved):
    """x [T, H, D] rotated in its first 2 * angle.shape[1] features by angle [T, R / 2] (f64)."""
    c, s = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    half = angle.shape[1]
    head, tail = x[..., : 2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    else:
        a, b = head[..., :half], head[..., half:]
        turned = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    return torch.cat((turned, tail), dim=-1)


def _append_plain(s):
    case, qkv = s["case"], s["qkv"]
    hq, hk = case["q_heads"], case["kv_heads"]
    b, _, pos = _tokens(s, qkv.shape[0])
    x = qkv.float()
    q, k, v = x[:, :hq], x[:, hq: hq + hk], qkv[:, hq + hk:]
    if case["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * s["qw"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * s["kw"].float()
    if case["rot"]:
        angle = pos.double()[:, None] * s["inv"].double()[None, :]
        q, k = _rotate(q, angle, case["interleaved"]), _rotate(k, angle, case["interleaved"])
    page = s["rows"].long()[s["ids"].long()[b], pos // case["page"]]
    s["k"][0][page, :, pos % case["page"]] = k.to(qkv.dtype)
    s["v"][0][page, :, pos % case["page"]] = v
    return [q.to(qkv.dtype), s["k"], s["v"]]


def _attention_plain(s):
    case, q = s["case"], s["q"]
    page, hk, hq, d, n = case["page"], case["kv_heads"], case["q_heads"], case["dim"], case["seqs"]
    ids, cu = s["ids"].long(), s["cu_plain"].long()
    wide = -(-s["max_held"] // page)
    table = s["rows"][ids][:, :wide].long().clamp(min=0)
    held, new = s["lens"][ids].long(), cu[1:] - cu[:-1]
    keys = torch.arange(wide * page, device=q.device)
    there = (keys[None, :] < held[:, None])[:, None, :, None]

    def gathered(pool):  # [n, kv_heads, keys, d] in 32 bits, what no sequence holds as zeros
        x = pool[0][table].permute(0, 2, 1, 3, 4).reshape(n, hk, wide * page, d).float()
        return torch.where(there, x, 0.0)

    k, v = gathered(s["k"]), gathered(s["v"])
    i = torch.arange(s["max_new"], device=q.device)
    rows = (cu[:-1, None] + i[None, :]).clamp(max=q.shape[0] - 1)
    x = q[rows].float().reshape(n, s["max_new"], hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    score = torch.matmul(x, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    pos = (held - new)[:, None] + i[None, :]
    seen = (keys[None, None, :] < held[:, None, None]).expand(n, s["max_new"], -1)
    if case["causal"]:
        seen = seen & (keys <= pos[..., None])
    if case["window"]:
        seen = seen & (keys > pos[..., None] - case["window"])
    score = torch.where(seen[:, None, None].expand(n, hk, hq // hk, -1, -1).reshape(score.shape), score, -math.inf)
    most = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(most == -math.inf, 0.0, most))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total > 0, total, 1.0)
    o = o.reshape(n, hk, hq // hk, s["max_new"], d).permute(0, 3, 1, 2, 4).reshape(n, s["max_new"], hq, d)
    b, i, _ = _tokens(s, q.shape[0])
    return o[b, i].to(q.dtype)


def _free_pages(refs):
    """The pages, those that nobody holds first, lowest first."""
    return torch.argsort((refs != 0).int(), stable=True).to(torch.int32)


def _pages_plain(s):
    case, rows, lens, refs = s["case"], s["rows"], s["lens"], s["refs"]
    page, ids = case["page"], s["ids"].long()
    col = torch.arange(rows.shape[1], device=rows.device)
    if case["kind"] == "extend":
        old = lens[ids]
        had, has = (old + page - 1) // page, (old + s["counts"] + page - 1) // page
        first = torch.cumsum(has - had, 0) - (has - had)
        fresh = (col[None, :] >= had[:, None]) & (col[None, :] < has[:, None])
        at = _free_pages(refs)[(first[:, None] + col[None, :] - had[:, None]).clamp(0, refs.shape[0] - 1).long()]
        rows[ids] = torch.where(fresh, at, rows[ids])
        refs.index_add_(0, torch.where(fresh, at, 0).long().flatten(), fresh.to(refs.dtype).flatten())
        lens[ids] = old + s["counts"]
    elif case["kind"] == "fork":
        parents, children = s["parents"].long(), s["children"].long()
        held = lens[parents]
        full, part = held // page, (held % page != 0)
        nth = torch.cumsum(part.int(), 0) - part.int()
        at = _free_pages(refs)[nth.long()]
        theirs = rows[parents]
        last = theirs.gather(1, full[:, None].long().clamp(max=rows.shape[1] - 1))[:, 0]
        src = torch.where(part, last, theirs[:, 0]).long()  # nothing left over: a page copied onto itself
        dst = torch.where(part, at, theirs[:, 0]).long()
        s["k"][:, dst] = s["k"][:, src]
        s["v"][:, dst] = s["v"][:, src]
        shared = col[None, :] < full[:, None]
        refs.index_add_(0, torch.where(shared, theirs, 0).long().flatten(), shared.to(refs.dtype).flatten())
        refs.index_add_(0, dst, part.to(refs.dtype))
        rows[children] = torch.where(shared, theirs, torch.where((col[None, :] == full[:, None]) & part[:, None], at[:, None], -1))
        lens[children] = held
    elif case["kind"] == "free":
        theirs = rows[ids]
        refs.index_add_(0, theirs.clamp(min=0).long().flatten(), -(theirs >= 0).to(refs.dtype).flatten())
        rows[ids] = -1
        lens[ids] = 0
    elif case["kind"] == "compact":
        live = refs > 0
        index = torch.arange(refs.shape[0], device=refs.device)
        low = index < live.sum()
        dst, src = torch.nonzero(low & ~live)[:, 0], torch.nonzero(~low & live)[:, 0]
        s["k"][:, dst] = s["k"][:, src]
        s["v"][:, dst] = s["v"][:, src]
        to = index.to(torch.int32)
        to[src] = dst.to(torch.int32)
        rows.copy_(torch.where(rows >= 0, to[rows.clamp(min=0).long()], -1))
        refs[dst] = refs[src]
        refs[src] = 0
    else:
        src, dst = s["src"].long(), s["dst"].long()
        s["k"][:, dst] = s["k"][:, src]
        s["v"][:, dst] = s["v"][:, src]
    return [rows, lens, refs, s["k"], s["v"]]


# ---- the package's operators --------------------------------------------------------------------------------------


def _cache(s):
    """The cache object that a program makes of its pools and tables once."""
    if "cache" not in s:
        package = os.path.join(ROOT, "open-cuda_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        import kv_cache
        s["cache"] = kv_cache.KVCache(s["k"], s["v"], s["rows"], s["lens"], s["refs"], s["status"])
    return s["cache"]


def run(s):
    case = s["case"]
    if case["op"] == "pages":  # the tables as they were, so that each pass finds the same work
        s["rows"].copy_(s["rows0"])
        s["lens"].copy_(s["lens0"])
        s["refs"].copy_(s["refs0"])
        if not own:
            return _pages_plain(s)
        c = _cache(s)
        if case["kind"] == "extend":
            c.extend(s["ids"], s["counts"])
        elif case["kind"] == "fork":
            c.fork(s["parents"], s["children"])
        elif case["kind"] == "free":
            c.free(s["ids"])
        elif case["kind"] == "compact":
            c.compact()
        else:
            c.copy_pages(s["src"], s["dst"])
        return [s["rows"], s["lens"], s["refs"], s["k"], s["v"]]
    if case["op"] == "append":
        if not own:
            return _append_plain(s)
        hq, hk, x = case["q_heads"], case["kv_heads"], s["qkv"]
        q = _cache(s).append(0, x[:, :hq], x[:, hq: hq + hk], x[:, hq + hk:], s["cu"], s["ids"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                             inv_freq=s["inv"], interleaved=case["interleaved"])
        return [q, s["k"], s["v"]]
    if not own:
        return _attention_plain(s)
    return _cache(s).attention(0, s["q"], s["cu"], s["ids"], causal=case["causal"], window=case["window"])


# ---- what a pass cannot do without --------------------------------------------------------------------------------


def _visible(case, new, held):
    """Pairs of a new token and a key that it sees, and keys that any new token sees, of one sequence."""
    w = case["window"]
    if not case["causal"]:
        if not w:
            return new * held, held
        first = max(0, held - new - w + 1)
        return sum(held - max(0, p - w + 1) for p in range(held - new, held)), held - first
    if not w:
        return new * (held - new) + new * (new + 1) // 2, held
    return sum(min(p + 1, w) for p in range(held - new, held)), held - max(0, held - new - w + 1)


def work(case):
    size, hk, d = SIZE[case["type"]], case["kv_heads"], case["dim"]
    if case["op"] == "pages":
        each = case["layers"] * hk * case["page"] * d * size * 2
        held = _spread(case["kv_min"], case["kv_max"], case["seqs"])
        most = int(case["pages"] * case["live"])
        while sum(_pages_of(case, held)) > most:
            held = [max(1, int(h * 0.9)) for h in held]
        need = _pages_of(case, held)
        tables = 4 * case["pages"] + 8 * sum(need)
        if case["kind"] == "fork":
            return {"bytes": tables + 2 * each * case["count"] * sum(h % case["page"] != 0 for h in held), "flops": 0}
        if case["kind"] == "compact":  # pages in no order: the dense part's holes are what is not live of it
            live = sum(need)
            return {"bytes": tables + 2 * each * int(live * (1 - live / case["pages"])), "flops": 0}
        if case["kind"] == "copy":
            return {"bytes": 2 * each * (case["pages"] // 2), "flops": 0}
        return {"bytes": tables, "flops": 0}
    new, held = _lengths(case)
    hq, total = case["q_heads"], sum(new)
    if case["op"] == "append":
        return {"bytes": 2 * total * (hq + 2 * hk) * d * size, "flops": total * (hq + hk) * d * 8}
    seen = [_visible(case, a, b) for a, b in zip(new, held)]
    return {"bytes": 2 * total * hq * d * size + sum(k for _, k in seen) * hk * d * 2 * size, "flops": 4 * d * hq * sum(p for p, _ in seen)}


# ---- the definition in 64 bits, a sequence at a time --------------------------------------------------------------


def _exact_append(case, s):
    hq, hk, page = case["q_heads"], case["kv_heads"], case["page"]
    new, held = _lengths(case)
    rows, ids = s["rows"].tolist(), s["ids"].tolist()
    k, v = s["k"].double(), s["v"].double()
    out, at = [], 0
    for b, (m, h) in enumerate(zip(new, held)):
        x = s["qkv"][at: at + m].double()
        at += m
        pos = torch.arange(h - m, h, device=x.device)
        done = []
        for y, w in ((x[:, :hq], s["qw"]), (x[:, hq: hq + hk], s["kw"])):
            if w is not None:
                y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * w.double()
            r = case["rot"]
            if r:
                turn = torch.polar(torch.ones(m, r // 2, dtype=torch.float64, device=x.device), pos[:, None] * s["inv"].double())[:, None]
                if case["interleaved"]:
                    z = torch.complex(y[..., 0:r:2].contiguous(), y[..., 1:r:2].contiguous()) * turn
                    y = torch.cat((torch.view_as_real(z).reshape(m, -1, r), y[..., r:]), -1)
                else:
                    z = torch.complex(y[..., : r // 2].contiguous(), y[..., r // 2: r].contiguous()) * turn
                    y = torch.cat((z.real, z.imag, y[..., r:]), -1)
            done.append(y)
        out.append(done[0])
        where = torch.tensor(rows[ids[b]], device=x.device)[pos // page]
        k[0, where, :, pos % page] = done[1]
        v[0, where, :, pos % page] = x[:, hq + hk:]
    return [torch.cat(out), k, v]


def _exact_attention(case, s):
    hq, hk, d, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    new, held = _lengths(case)
    rows, ids = s["rows"].tolist(), s["ids"].tolist()
    out, at = [], 0
    for b, (m, h) in enumerate(zip(new, held)):
        own_pages = rows[ids[b]][: -(-h // page)]
        k = torch.cat([s["k"][0, p] for p in own_pages], 1)[:, :h].double()
        v = torch.cat([s["v"][0, p] for p in own_pages], 1)[:, :h].double()
        o = torch.empty(m, hq, d, dtype=torch.float64, device=k.device)
        pos = torch.arange(h - m, h, device=k.device)[:, None]
        key = torch.arange(h, device=k.device)[None, :]
        hidden = torch.zeros(m, h, dtype=torch.bool, device=k.device)
        if case["causal"]:
            hidden |= key > pos
        if case["window"]:
            hidden |= key <= pos - case["window"]
        for g in range(hq):
            a = s["q"][at: at + m, g].double() @ k[g // (hq // hk)].T / d ** 0.5
            o[:, g] = torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v[g // (hq // hk)]
        out.append(o)
        at += m
    return torch.cat(out)


def exact(case, seed):
    if case["op"] == "pages":
        return None  # whole numbers and copies: nothing is computed
    if case["op"] == "attention" and work(case)["flops"] > 2e13:
        return None
    s = prepare(case, seed)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attention(case, s)
