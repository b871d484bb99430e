"""The paged key/value cache on the GPU against plain 64-bit implementations.

Whatever no sequence holds is NaN in these tests' pools: free pages, and the
rest of a last page.

Tolerances.  eps/2 is half a step of the type (bf16 2^-8, f16 2^-11, f32
2^-24).  Attention, element by element: the output is rounded once,
eps/2 * |o|.  A score is a sum of d products, each off by 2^-24 of its size,
and the exponent's argument by a few more units of 2^-24 of it: with S the
largest scale * sum |q_i k_i|, at most e = (d + 8) * 2^-24 * S, so a weight is
off by a factor exp(e) - 1 and 2^-21 for the exponential; the sums over n keys
add n * 2^-24.  Numerator and denominator both: twice that, times A = the
weighted mean of |v|.  Kernels that feed weights to 16-bit tensor cores may
round each weight once more: eps/2 * A.  Of f32, the products may be carried
as pairs of f16 terms (22 bits each operand): 3 * 2^-22 * S more in a score,
3 * 2^-22 * A more in the output."""
import math
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import kv_cache  # noqa: E402
from kv_cache import KVCache  # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
# below 2^-14 f16 steps by 2^-24 whatever the value: half of that, not 2^-11 of the value, is what a rounding is off by there
SMALLEST = {F32: 1e-30, F16: 2.0 ** -25, BF16: 1e-30}


def close(got, want, tol):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    at = int((off / tol).nan_to_num(math.inf).argmax())
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst at {at}: got {float(got.flatten()[at]):.9g}, want "
                           f"{float(want.flatten()[at]):.9g}, off {float(off.flatten()[at]):.3g}, allowed {float(tol.flatten()[at]):.3g}")


def ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def filled(dtype, hk, d, page, lens, layers=1, layer=0, seed=0, spare=3, k_scale=1.0):
    """A cache whose sequences hold random keys and values in scattered pages.
    Returns it and the sequences' [hk, len, d] keys and values of `layer`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages, seqs = sum(need) + spare, len(lens) + 1
    shape = (layers, pages, hk, page, d)
    k = torch.full(shape, math.nan, dtype=dtype, device="cuda")
    v = torch.full(shape, math.nan, dtype=dtype, device="cuda")
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((seqs, max(need + [1]) + 1), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    ks, vs, at = [], [], 0
    for s, n in enumerate(lens):
        kk = (torch.randn(hk, n, d, generator=g, device="cuda") * k_scale).to(dtype)
        vv = torch.randn(hk, n, d, generator=g, device="cuda").to(dtype)
        for p in range(need[s]):
            page_no = order[at]
            at += 1
            table[s, p], refs[page_no] = page_no, 1
            part = kk[:, p * page:(p + 1) * page]
            k[layer, page_no, :, :part.shape[1]] = part
            v[layer, page_no, :, :part.shape[1]] = vv[:, p * page:(p + 1) * page]
        ks.append(kk)
        vs.append(vv)
    c = KVCache(k, v, table.cuda(), ints(list(lens) + [0]), refs.cuda())
    return c, ks, vs


def expected(q, ks, vs, ids, new, scale, causal, window):
    """Output and allowed error of each row, [tokens, heads, d] in 64 bits."""
    hq, d = q.shape[1:]
    outs, tols, at = [], [], 0
    u = HALF_STEP[q.dtype]
    for s, m in zip(ids, new):
        k, v = ks[s].double(), vs[s].double()
        hk, n = k.shape[:2]
        x = q[at:at + m].double().reshape(m, hk, hq // hk, d)
        at += m
        pos = torch.arange(n - m, n, device=q.device)[:, None]
        key = torch.arange(n, device=q.device)[None, :]
        seen = torch.ones(m, n, dtype=torch.bool, device=q.device)
        if causal:
            seen &= key <= pos
        if window:
            seen &= key > pos - window
        seen = seen[:, None, None, :]
        sc = torch.einsum("mhgd,hnd->mhgn", x, k) * scale
        size = torch.einsum("mhgd,hnd->mhgn", x.abs(), k.abs()) * abs(scale)
        sc = torch.where(seen, sc, -math.inf)
        big = (torch.where(seen, size, 0.0).amax(-1, keepdim=True) if n else torch.zeros(m, hk, hq // hk, 1, dtype=torch.float64, device=q.device))
        top = sc.amax(-1, keepdim=True) if n else torch.full_like(big, -math.inf)
        e = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
        tot = e.sum(-1, keepdim=True)
        w = e / torch.where(tot > 0, tot, 1.0)
        o = torch.einsum("mhgn,hnd->mhgd", w, torch.nan_to_num(v, 0, 0, 0))
        a = torch.einsum("mhgn,hnd->mhgd", w, torch.nan_to_num(v, 0, 0, 0).abs())
        err = (d + 8) * 2.0 ** -24 * big
        extra = u * a
        if q.dtype == F32:
            err, extra = err + 3 * 2.0 ** -22 * big, 3 * 2.0 ** -22 * a
        tol = u * o.abs() + a * 2 * (torch.expm1(err) + 2.0 ** -21 + n * 2.0 ** -24) + extra + SMALLEST[q.dtype]
        outs.append(o.reshape(m, hq, d))
        tols.append(tol.reshape(m, hq, d))
    return torch.cat(outs), torch.cat(tols)


def attend(c, q, ids, new, layer=0, scale=None, causal=True, window=0, plain_ids=False, one_each=False, out=None):
    cu = None if one_each else ints(np.concatenate([[0], np.cumsum(new)]))
    return c.attention(layer, q, cu, None if plain_ids else ints(ids), scale=scale, causal=causal, window=window, out=out)


def check(dtype, hq, hk, d, page, lens, new, causal=True, window=0, layers=1, layer=0, seed=0, scale=None, one_each=False, k_scale=1.0):
    c, ks, vs = filled(dtype, hk, d, page, lens, layers, layer, seed, k_scale=k_scale)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(sum(new), hq, d, generator=g, device="cuda").to(dtype)
    ids = list(np.random.default_rng(seed).permutation(len(lens)))
    new = [new[i] for i in range(len(lens))]
    o = attend(c, q, ids, new, layer, scale, causal, window, one_each=one_each)
    want, tol = expected(q, ks, vs, ids, new, 1 / math.sqrt(d) if scale is None else scale, causal, window)
    close(o, want, tol)
    c.check()
    return c, q, o


SHAPES = [  # q heads, kv heads, head_dim
    (1, 1, 64), (28, 4, 128), (32, 8, 128), (12, 12, 64), (6, 2, 96), (16, 2, 80), (5, 5, 40), (4, 4, 256), (16, 1, 128), (3, 3, 17), (2, 1, 250),
    (4, 2, 8), (40, 1, 64),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hq, hk, d", SHAPES)
def test_decode(dtype, hq, hk, d):
    check(dtype, hq, hk, d, 16, [1, 2, 15, 16, 17, 63, 64, 65, 200, 1000], [1] * 10, one_each=True, seed=hq + d)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("page", [1, 2, 8, 32, 64, 128, 256, 1024])
def test_page_sizes(dtype, page):
    check(dtype, 8, 2, 64, page, [1, 127, 128, 129, 700], [1, 3, 128, 1, 130], seed=page)
    check(dtype, 4, 2, 128, page, [5, 300], [1, 260], seed=page + 1)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hq, hk, d", SHAPES)
@pytest.mark.parametrize("causal, window", [(True, 0), (False, 0), (True, 37), (False, 100), (True, 1)])
def test_chunks(dtype, hq, hk, d, causal, window):
    check(dtype, hq, hk, d, 16, [1, 5, 64, 129, 300, 411], [1, 2, 64, 100, 33, 257], causal=causal, window=window, seed=d + window)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_mixed_batch(dtype, d):
    """Chunks among single tokens, entries without new tokens among both."""
    check(dtype, 8, 2, d, 32, [900, 3, 513, 77, 1, 1500], [1, 0, 300, 1, 1, 17], seed=d)
    check(dtype, 8, 2, d, 32, [900, 3, 513, 77, 1, 1500], [1, 0, 300, 1, 1, 17], window=200, seed=d)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_fewer_tokens_than_sequences(dtype, d):
    """One sequence has several new tokens, the others none."""
    check(dtype, 8, 2, d, 32, [30, 20, 9000, 77, 1, 15], [0, 0, 5, 0, 0, 0], seed=d)
    check(dtype, 8, 2, d, 32, [9000], [9], seed=d)
    check(dtype, 8, 2, d, 32, [9000, 40], [9, 1], seed=d)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq, hk", [(1, 1), (7, 1), (8, 2), (9, 3), (40, 1)])
def test_tiles_of_every_shape(dtype, d, hq, hk):
    """Items with one sub-tile and two, with one tile of keys and many, cut and whole."""
    for lens, new in (([33], [33]), ([128], [128]), ([129, 127], [129, 127]), ([256], [256]), ([257, 4000], [257, 130]), ([5000], [600]),
                      ([6000, 70, 300, 2000, 1], [40, 70, 299, 1000, 1])):
        check(dtype, hq, hk, d, 16, lens, new, seed=sum(lens))
        check(dtype, hq, hk, d, 16, lens, new, seed=sum(lens), window=150)
        check(dtype, hq, hk, d, 16, lens, new, seed=sum(lens), causal=False)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_many_short_sequences(dtype):
    lens = [1 + (7 * i) % 50 for i in range(400)]
    check(dtype, 4, 2, 64, 16, lens, [1] * 400, one_each=True)
    check(dtype, 4, 2, 64, 16, lens, [1 + i % min(9, n) for i, n in enumerate(lens)])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("apart", [31, 32, 2500])
def test_chunks_far_apart_in_the_batch(dtype, apart):
    """Chunks of dozens of row blocks with single tokens and entries without
    any between them, more than a block has threads."""
    lens = [900] + [1 + i % 9 for i in range(apart)] + [40, 1200, 33]
    new = [700] + [int(i % 3 > 0) for i in range(apart)] + [0, 650, 30]
    c, ks, vs = filled(dtype, 1, 64, 16, lens, seed=apart)
    q = torch.randn(sum(new), 16, 64, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    o = attend(c, q, range(len(lens)), new)
    want, tol = expected(q, ks, vs, range(len(lens)), new, 0.125, True, 0)
    close(o, want, tol)
    c.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new", [1, 3, 70])
def test_one_long_sequence_is_split(dtype, new):
    c, q, o = check(dtype, 8, 2, 128, 64, [40000], [new], seed=new)
    for _ in range(3):
        assert torch.equal(o, attend(c, q, [0], [new]))  # the same bits each time


def block_values(n, d, device="cuda"):
    """[1, n, d]: feature f is 1 for the keys of the f-th of d equal blocks, 0
    for the others, so output f is the weight of block f.  Nothing cancels: what
    expected() allows is a fraction of that weight, and a piece of the keys that
    is lost shows in the features of its blocks."""
    return (torch.arange(n, device=device)[:, None] * d // n == torch.arange(d, device=device)[None, :]).double()[None]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hq, hk, d", [(8, 2, 128), (4, 4, 64), (6, 2, 96), (2, 1, 256), (28, 4, 128), (3, 1, 33)])
@pytest.mark.parametrize("new, n", [(1, 40000), (3, 40000), (70, 12000), (300, 7000)])
@pytest.mark.parametrize("scale", [None, 1.0])
def test_every_key_counts(dtype, hq, hk, d, new, n, scale):
    """Long contexts in pieces, joined: none is lost, and none counts twice.
    With a scale of 1 a few keys have the weight, and f32 queries, keys or
    weights of fewer bits would show.

    f32 tiles carry a weight as two f16 terms of 2^15 times it, the largest of
    the row being 1: half a step of f16's subnormals in each, so 2^-24 of the
    scaled weight, 2^-39 of the largest a key, however small the weight itself;
    the sum that divides is at least the largest.  expected() has relative
    errors of weights alone, so 2^-39 sum |v| is added for features that have
    next to no weight."""
    c, ks, vs = filled(dtype, hk, d, 64, [n, 200], seed=new)
    rows = block_values(n, d).to(dtype).expand(hk, n, d)
    at = torch.arange(n, device="cuda")
    c.v[0, c.page_table[0].long()[at // 64], :, at % 64] = rows.transpose(0, 1)
    q = torch.randn(new + 1, hq, d, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").to(dtype)
    scale = 1 / math.sqrt(d) if scale is None else scale
    o = attend(c, q, [0, 1], [new, 1], scale=scale)
    want, tol = expected(q, ks, [rows, vs[1]], [0, 1], [new, 1], scale, True, 0)
    if dtype == F32:
        tol[:new] += 2.0 ** -39 * rows[0].double().sum(0)
    close(o, want, tol)
    c.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_layers_strides_and_scales(dtype):
    c, ks, vs = filled(dtype, 2, 64, 16, [50, 130], layers=3, layer=1)
    wide = torch.randn(131, 13, 64, device="cuda").to(dtype)
    q, new = wide[:, 3:11], [1, 130]
    for scale in (0.3, -0.2, 0.0):
        buf = torch.full((131, 9, 64), 7.0, dtype=dtype, device="cuda")
        o = attend(c, q, [0, 1], new, layer=1, scale=scale, out=buf[:, :8])
        want, tol = expected(q, ks, vs, [0, 1], new, scale, True, 0)
        close(o, want, tol)
        assert (buf[:, 8] == 7).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_unaligned_queries_and_pools(dtype):
    """Rows that no vector load can take."""
    c, ks, vs = filled(dtype, 2, 64, 16, [40, 99])
    raw = torch.randn(4 * (8 * 64 + 1) + 1, device="cuda").to(dtype)
    q = raw[1:].as_strided((4, 8, 64), (8 * 64 + 1, 64, 1), 1)
    o = attend(c, q, [0, 1], [1, 3])
    want, tol = expected(q, ks, vs, [0, 1], [1, 3], 0.125, True, 0)
    close(o, want, tol)
    flat = [torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(x.shape).copy_(x) for x in (c.k, c.v)]
    moved = KVCache(*flat, c.page_table, c.seq_len, c.refcount)
    close(attend(moved, q, [0, 1], [1, 3]), want, tol)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hq, hk, d", [(4, 2, 40), (6, 2, 72), (3, 3, 80), (10, 2, 96), (2, 1, 120), (4, 2, 24), (3, 1, 33)])
@pytest.mark.parametrize("page", [4, 16, 128])
def test_padded_heads_in_one_call(dtype, hq, hk, d, page):
    """Head sizes between the tiles' widths: single tokens and chunks side by
    side, both with items that cuts go through, and pages that end in a tile."""
    check(dtype, hq, hk, d, page, [3000, 700, 2501, 129], [1, 300, 1, 129], seed=d, layers=2, layer=1)
    check(dtype, hq, hk, d, page, [1500, 900], [5, 260], causal=False, window=333, seed=d + 1)


@pytest.mark.parametrize("dtype, big", [(F32, 3e38), (F16, 65504.0), (BF16, torch.finfo(BF16).max)])
@pytest.mark.parametrize("hq, hk, d", [(8, 2, 64), (4, 2, 128), (4, 2, 80), (2, 2, 256), (3, 1, 17)])
@pytest.mark.parametrize("lens, new", [([9, 40], [1, 1]), ([3000], [1]), ([300, 1500], [20, 100]), ([2100], [260])])
def test_values_near_the_largest(dtype, big, hq, hk, d, lens, new):
    """Sums of weights times values overflow, the outputs do not: in whole
    items, joined ones and chunks.  Every value of a feature is plus or minus
    `big`, and so is the output (weights sum to one)."""
    c, ks, vs = filled(dtype, hk, d, 16, lens, seed=d)
    sign = torch.where(torch.arange(d, device="cuda") % 3 == 0, -1.0, 1.0).double()
    c.v.copy_((sign * big).to(dtype).expand(c.v.shape))
    q = torch.randn(sum(new), hq, d, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(dtype)
    o = attend(c, q, range(len(lens)), new)
    want, tol = expected(q, ks, [x.copy_((sign * big).to(dtype).expand(x.shape)) for x in vs], range(len(lens)), new, 1 / math.sqrt(d), True, 0)
    assert torch.isfinite(o).all()
    close(o, want, tol)
    c.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hq, hk, d", [(1, 1, 64), (8, 2, 128), (4, 2, 256), (3, 1, 17), (40, 1, 64)])
@pytest.mark.parametrize("small", [2.0 ** -100, 2.0 ** -112])
@pytest.mark.parametrize("new", [1, 70])
def test_values_near_the_smallest(dtype, hq, hk, d, small, new):
    """Sums that f32 holds with all their bits: what is rounded to a subnormal,
    at most 2^-150 at a time, is below 2^-38 of every value's size."""
    c, ks, vs = filled(dtype, hk, d, 16, [40, 900], seed=d)
    c.v.copy_((c.v.double() * small).to(dtype))
    vs = [(x.double() * small).to(dtype) for x in vs]
    q = torch.randn(1 + new, hq, d, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(dtype)
    o = attend(c, q, [0, 1], [1, new])
    want, tol = expected(q, ks, vs, [0, 1], [1, new], 1 / math.sqrt(d), True, 0)
    if dtype == F32:
        tol = two_term_tol(q, ks, vs, [0, 1], [1, new], 1 / math.sqrt(d), tol)
    tol = tol - SMALLEST[dtype] + 940 * 2.0 ** -150
    close(o.double() / small, want / small, tol / small)
    c.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("new", [[1, 1], [1, 90], [90, 200]])
def test_unaligned_outputs(dtype, d, new):
    """Results to rows that no vector store can take, and to odd pairs."""
    c, ks, vs = filled(dtype, 2, d, 16, [400, 999])
    m = sum(new)
    q = torch.randn(m, 4, d, device="cuda").to(dtype)
    want, tol = expected(q, ks, vs, [0, 1], new, 1 / math.sqrt(d), True, 0)
    for gap in (1, 2):
        raw = torch.full((m * (4 * d + gap) + gap,), 7.0, dtype=dtype, device="cuda")
        out = raw.as_strided((m, 4, d), (4 * d + gap, d, 1), gap)
        attend(c, q, [0, 1], new, out=out)
        close(out, want, tol)
        assert (raw[:gap] == 7).all() and (raw[gap:].view(m, 4 * d + gap)[:, 4 * d:] == 7).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_rows_without_keys_are_zero(dtype, d):
    """No keys at all, and more new tokens than the sequence holds: the first
    of them stand before its start."""
    c, ks, vs = filled(dtype, 2, d, 16, [0, 5, 40])
    new = [2, 9, 45]
    q = torch.randn(sum(new), 4, d, device="cuda").to(dtype)
    want, tol = expected(q, ks, vs, [0, 1, 2], new, 1 / math.sqrt(d), True, 0)
    o = attend(c, q, [0, 1, 2], new)
    close(o, want, tol)
    assert (o[:2] == 0).all() and (o[2:6] == 0).all() and (o[11:16] == 0).all() and (o[6:11] != 0).any()
    c.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new", [2, 9, 200])
def test_what_a_row_does_not_see_has_no_part(dtype, d, what, new):
    """The last token's key and value, and the first one's behind a window."""
    n = 260
    c, ks, vs = filled(dtype, 2, d, 16, [n])
    q = torch.randn(new, 4, d, device="cuda").to(dtype)
    want, tol = expected(q, ks, vs, [0], [new], 1 / math.sqrt(d), True, n - new)
    for j in (n - 1, 0):
        page = int(c.page_table[0, j // 16])
        c.k[0, page, :, j % 16], c.v[0, page, :, j % 16] = what, what
    o = attend(c, q, [0], [new], window=n - new)  # the first new token's window ends behind key 0
    close(o[:-1], want[:-1], tol[:-1])
    if math.isnan(what):
        assert torch.isnan(o[-1]).all()  # what a row does see counts


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new, n", [(9, 260), (200, 260), (200, 6000)])
def test_f32_values_of_very_different_size(d, new, n):
    """A value of 1e30 among values of 1e-10: the rows that do not see it, and
    the ones that do."""
    c, ks, vs = filled(F32, 2, d, 16, [n])
    big = vs[0][:, n - 5] * 1e30
    vs[0] = vs[0] * 1e-10
    vs[0][:, n - 5] = big
    for j in range(n):
        page = int(c.page_table[0, j // 16])
        c.v[0, page, :, j % 16] = vs[0][:, j]
    q = torch.randn(new, 4, d, device="cuda")
    o = attend(c, q, [0], [new])
    want, tol = expected(q, ks, vs, [0], [new], 1 / math.sqrt(d), True, 0)
    close(o, want, tol)


def with_values(c, vs, s, at, rows):
    """Puts [hk, m, d] values in place of sequence s's from token `at` on."""
    page = c.page_size
    for j in range(rows.shape[1]):
        number = int(c.page_table[s, (at + j) // page])
        c.v[0, number, :, (at + j) % page] = rows[:, j].to(c.dtype)
    vs[s][:, at:at + rows.shape[1]] = rows.to(c.dtype)


def two_term_tol(q, ks, vs, ids, new, scale, tol):
    """What expected() allows, and what carrying values as two f16 terms of one
    scaling a tile may cost.  The tile's largest is scaled into [2^14, 2^15), so
    a scaled value t is off by half a step of f16's subnormals in each term,
    2^-24, or by 2^-21 |t|.  A row of queries is computed on them when its
    weights p have sum(p (1/4 - r c)) <= 0, r the largest |v| of a key and c the
    scaling: sum(p 2^-24) <= 2^-22 sum(p r c), so any feature is off by at most
    2^-22 times the weighted mean of the keys' largest |v|.  expected() has
    3 * 2^-22 of the weighted mean of the feature's own |v|, which the second
    case (2^-21) takes; a feature that is far below its row's largest needs
    the first."""
    largest, _ = expected(q, ks, [v.abs().amax(-1, keepdim=True).expand(v.shape) for v in vs], ids, new, scale, True, 0)
    return tol + 2.0 ** -22 * largest


@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("new, n", [(200, 260), (260, 260), (130, 3000)])
def test_f32_large_values_of_small_weight(d, new, n):
    """Rows that see a value of 1e12 with a weight of e^-60 beside values near 1."""
    c, ks, vs = filled(F32, 2, d, 16, [n])
    at = n - new + 3
    with_values(c, vs, 0, at, 1e12 * vs[0][:, at:at + 1])
    number = int(c.page_table[0, at // 16])
    ks[0][:, at] = -120.0 / d
    c.k[0, number, :, at % 16] = -120.0 / d
    q = 0.02 * torch.randn(new, 4, d, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") + 0.5
    o = attend(c, q, [0], [new], scale=1.0)
    want, tol = expected(q, ks, vs, [0], [new], 1.0, True, 0)
    close(o, want, two_term_tol(q, ks, vs, [0], [new], 1.0, tol))
    c.check()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bits", [7, 12, 15, 17, 18, 24, 40, 70])
@pytest.mark.parametrize("tiny", [1, 5, 127, 128, 150])
def test_f32_first_values_are_small(d, bits, tiny):
    """The first tokens' values are 2^-bits of the others': the rows that see
    them alone, the ones that see both, and another sequence beside."""
    c, ks, vs = filled(F32, 2, d, 16, [300, 70], seed=bits)
    with_values(c, vs, 0, 0, vs[0][:, :tiny] * 2.0 ** -bits)
    q = torch.randn(370, 4, d, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    o = attend(c, q, [0, 1], [300, 70])
    want, tol = expected(q, ks, vs, [0, 1], [300, 70], 1 / math.sqrt(d), True, 0)
    close(o, want, two_term_tol(q, ks, vs, [0, 1], [300, 70], 1 / math.sqrt(d), tol))
    c.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_nonfinite_values_that_are_seen(dtype):
    c, ks, vs = filled(dtype, 1, 64, 16, [300])
    page = int(c.page_table[0, 100 // 16])
    c.v[0, page, 0, 100 % 16, 7] = math.inf
    for new in (1, 200):
        o = attend(c, torch.randn(new, 2, 64, device="cuda").to(dtype), [0], [new])
        seen = torch.arange(300 - new, 300, device="cuda") >= 100
        assert (o[seen][:, :, 7] == math.inf).all()
        o[seen, :, 7] = 0
        assert torch.isfinite(o).all()


@pytest.mark.parametrize("dtype, hq, hk", [(F32, 12, 12), (F16, 28, 4), (BF16, 28, 4)])
def test_an_infinite_value_in_view_of_a_long_chunk(dtype, hq, hk):
    """Every row of 2048 new tokens over 60000 keys sees one infinite value and
    is computed again; the rows of the sequences beside it, and the other
    features, are what they are without it.  Two results of one row differ by
    what each may be off: A (the weighted mean of |v|) is below 1 over so many
    standard normal values, and expected() is asked for rows all over."""
    n, new, d = 60000, 2048, 64
    c, ks, vs = filled(dtype, hk, d, 64, [400, n, 300])
    parts = [300, new, 5]
    q = torch.randn(sum(parts), hq, d, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(dtype)
    without = attend(c, q, [0, 1, 2], parts)
    page = int(c.page_table[1, 1000 // 64])
    c.v[0, page, :, 1000 % 64, 5] = math.inf
    o = attend(c, q, [0, 1, 2], parts, out=torch.full_like(q, 7.0))
    c.check()
    again = o[300:300 + new]
    assert (again[:, :, 5] == math.inf).all()
    rest = [f for f in range(d) if f != 5]
    for s, at in ((0, 0), (2, 300 + new)):
        rows = slice(at, at + parts[s])
        want, tol = expected(q[rows], ks, vs, [s], [parts[s]], 0.125, True, 0)
        close(o[rows], want, tol)
    u = HALF_STEP[dtype]
    off = (again.double() - without[300:300 + new].double())[:, :, rest].abs()
    assert bool((off <= 2 * u * again[:, :, rest].double().abs() + 2 * (u + 2 ** -20 + n * 2.0 ** -24)).all())
    for t in range(0, new, 157):
        want, tol = expected(q[300 + t:301 + t], [ks[1][:, :n - new + t + 1]], [vs[1][:, :n - new + t + 1]], [0], [1], 0.125, True, 0)
        close(again[t:t + 1, :, rest], want[:, :, rest], tol[:, :, rest])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_large_scores(dtype, d):
    """Scores in the thousands: the softmax stands on one or two keys."""
    check(dtype, 4, 2, d, 16, [700, 300], [1, 200], scale=20.0, seed=3)
    check(dtype, 4, 2, d, 16, [700, 300], [1, 200], scale=1e-20, seed=4)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("below", [24.6, 25.5, 27.0, 30.0])
def test_many_keys_of_small_weight(dtype, d, new, below):
    """One key of most of the weight and a value of 0, and 100000 of 2^-below
    of it each, which make the output; more sequences (that share the pages)
    than blocks, so that one block takes all keys of a sequence."""
    n, seqs = 100000, 600
    c, ks, vs = filled(dtype, 1, d, 64, [n])
    c = KVCache(c.k.zero_(), c.v, c.page_table[:1].expand(seqs, -1).contiguous(), torch.full((seqs,), n, dtype=torch.int32, device="cuda"), c.refcount)
    c.v.copy_((1.0 + torch.arange(d, device="cuda") % 7).to(dtype).expand(c.v.shape))
    ks, vs = [torch.zeros_like(ks[0])], [c.v[0, :1, 0, :1].expand(vs[0].shape).clone()]
    dominant = torch.full((d,), 2.0 * below * math.log(2.0) / d, device="cuda").to(dtype)
    number = int(c.page_table[0, 0])
    c.k[0, number, :, 5], c.v[0, number, :, 5] = dominant, 0.0
    ks[0][:, 5], vs[0][:, 5] = dominant, 0.0
    q = torch.full((seqs * new, 2, d), 0.5, dtype=dtype, device="cuda")
    o = attend(c, q, range(seqs), [new] * seqs, scale=1.0, causal=False)
    want, tol = expected(q[:1], ks, vs, [0], [1], 1.0, False, 0)
    close(o, want.expand(o.shape), tol.expand(o.shape))


@pytest.mark.parametrize("d", [64, 128])
def test_f32_ranges(d):
    check(F32, 4, 2, d, 16, [700, 300], [1, 200], scale=1e-18, k_scale=1e18, seed=3)
    check(F32, 4, 2, d, 16, [700, 300], [1, 200], scale=1e20, k_scale=1e-20, seed=4)


def test_a_falling_and_a_rising_maximum():
    """Running maxima that grow over thousands of keys, and that stand in the first tile."""
    for sign in (1, -1):
        for dtype, d in ((F16, 128), (BF16, 64), (F32, 64)):
            c, ks, vs = filled(dtype, 1, d, 16, [3001])
            ramp = torch.linspace(-30, 30, 3001, device="cuda")[:, None] * sign
            for j0 in range(0, 3001, 16):
                page = int(c.page_table[0, j0 // 16])
                m = min(16, 3001 - j0)
                c.k[0, page, 0, :m] = (ramp[j0:j0 + m] + torch.zeros(1, d, device="cuda")).to(dtype)
            ks[0] = (ramp + torch.zeros(1, d, device="cuda")).to(dtype)[None]
            for new in (1, 150):
                q = torch.full((new, 1, d), 0.5, dtype=dtype, device="cuda")
                o = attend(c, q, [0], [new])
                want, tol = expected(q, ks, vs, [0], [new], 1 / math.sqrt(d), True, 0)
                close(o, want, tol)


def test_rows_behind_the_last_sequence_stay():
    for dtype in (F32, F16, BF16):
        c, _, _ = filled(dtype, 2, 64, 16, [50, 70])
        q = torch.randn(20, 4, 64, device="cuda").to(dtype)
        out = torch.full_like(q, 3.0)
        c.attention(0, q, ints([0, 1, 12]), ints([0, 1]), out=out)
        assert (out[12:] == 3).all() and (out[:12] != 3).any()
        k = torch.randn(20, 2, 64, device="cuda").to(dtype)
        qo = torch.full_like(q, 3.0)
        before = c.k.clone()
        c.append(0, q, k, k, ints([0, 1, 12]), ints([0, 1]), q_out=qo)
        assert (qo[12:] == 3).all() and torch.equal(qo[:12], q[:12])
        changed = (c.k != before) & ~(torch.isnan(c.k) & torch.isnan(before))
        assert int(changed.any(-1).sum()) == 12 * 2


def test_bad_tables_and_ids_are_reported():
    for dtype in (F32, F16, BF16):
        for new in (1, 60):
            c, _, _ = filled(dtype, 2, 64, 16, [100, 64])
            q = torch.randn(2 * new, 4, 64, device="cuda").to(dtype)
            good = attend(c, q, [0, 1], [new, new])

            def as_before(o):  # the work may be cut at other places: f32 sums in another order, and a rounding on each side
                return ((o - good)[new:].float().abs() <= 2 * HALF_STEP[dtype] * good[new:].float().abs() + 2e-6).all()

            o = attend(c, q, [1 << 20, 1], [new, new])
            assert (o[:new] == 0).all() and as_before(o)
            c.page_table[0, 2] = 1 << 28
            o = attend(c, q, [0, 1], [new, new])
            assert as_before(o) and torch.isfinite(o).all()
            with pytest.raises(ValueError, match="page number"):
                c.check()
            c.check()
            c.seq_len[0] = 1 << 30  # more than its row of the table holds
            attend(c, q, [0, 1], [new, new])
            torch.cuda.synchronize()
            bad = torch.full((3,), -(1 << 30), dtype=torch.int32, device="cuda")
            c.attention(0, q, bad, ints([0, 1]))
            c.attention(0, q, -bad, ints([0, 1]))
            torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("bad", [-1, 3, 1 << 20])
def test_attention_reports_bad_ids(dtype, new, bad):
    c, ks, vs = filled(dtype, 2, 64, 16, [100, 64])  # rows 0, 1 and an empty one
    q = torch.randn(2 * new, 4, 64, device="cuda").to(dtype)
    for ids, one in (([bad, 1], False), ([1, bad], False), ([bad], True), ([0, bad] * 300, True)):
        rows = len(ids) * new
        x = q.repeat(-(-rows // (2 * new)), 1, 1)[:rows]
        o = attend(c, x, ids, [new] * len(ids), out=torch.full_like(x, 3.0), one_each=one and new == 1).view(len(ids), new, 4, 64)
        for i in (0, 1, len(ids) - 1):
            if i < len(ids):
                assert bool((o[i] == 0).all()) == (ids[i] == bad)
        with pytest.raises(ValueError, match="sequence id outside"):
            c.check()
    attend(c, q[:new], [bad, 1], [0, new])  # an entry without new tokens is not looked at
    c.check()
    c.attention(0, q[:1].repeat(4, 1, 1))  # without ids: one more entry than there are sequences
    with pytest.raises(ValueError, match="sequence id outside"):
        c.check()


def test_wrong_arguments_raise():
    c, _, _ = filled(F16, 2, 64, 16, [50, 70])
    q = torch.randn(2, 4, 64, device="cuda").half()
    for bad in (q.float(), q[..., :32], q.transpose(0, 1), q.cpu()):
        with pytest.raises(ValueError):
            c.attention(0, bad, None, None)
    with pytest.raises(ValueError):
        c.attention(0, q[:, :3], None, None)
    with pytest.raises(ValueError):
        c.attention(1, q, None, None)
    with pytest.raises(ValueError):
        c.attention(0, q, ints([0, 1, 2]), ints([0]))
    with pytest.raises(ValueError):
        c.attention(0, q, ints([0, 1, 2]).long(), ints([0, 1]))
    with pytest.raises(ValueError):
        c.append(0, q, q[:1, :2], q[:, :2])
    with pytest.raises(ValueError):
        c.append(0, q, q[:, :2], q[:, :2], q_weight=torch.ones(64, device="cuda"))
    with pytest.raises(ValueError):
        c.extend(ints([0]), ints([1, 2]))


def test_outputs_over_the_queries_are_refused():
    c, ks, vs = filled(F16, 2, 64, 16, [50, 70])
    buf = torch.randn(2, 8, 64, device="cuda").half()
    q = buf[:, :4]
    with pytest.raises(ValueError, match="overlaps"):
        c.attention(0, q, out=q)
    with pytest.raises(ValueError, match="overlaps"):
        c.attention(0, q, out=buf[:, 3:7])
    o = c.attention(0, q, out=buf[:, 4:])
    want, tol = expected(q, ks, vs, [0, 1], [1, 1], 0.125, True, 0)
    close(o, want, tol)


# ---- append -------------------------------------------------------------------------------------------------------


def rotated(x, pos, inv, interleaved):
    """x [m, h, d] in 64 bits, and the sum of the sizes that enter each result."""
    r = 2 * inv.numel()
    ang = pos.double()[:, None] * inv.double()[None, :]
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    y, size = x.clone(), x.abs().clone()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2:r])
    ya, yb = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = ya, yb
        size[..., 0:r:2], size[..., 1:r:2] = a.abs() + b.abs(), a.abs() + b.abs()
    else:
        y[..., : r // 2], y[..., r // 2:r] = ya, yb
        size[..., : r // 2] = size[..., r // 2:r] = a.abs() + b.abs()
    return y, size


LENS, NEW = [1, 33, 100, 20000], [1, 20, 0, 7]
MANY = [1, 900, 100, 20000], [1, 700, 0, 60]  # enough tokens for a warp each


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens, new", [(LENS, NEW), MANY])
@pytest.mark.parametrize("hq, hk, d, rot", [(28, 4, 128, 128), (12, 12, 64, 64), (8, 2, 80, 80), (6, 2, 96, 32), (4, 4, 256, 256), (3, 3, 17, 10),
                                            (2, 1, 250, 250), (5, 5, 40, 12), (8, 8, 64, 0), (0, 2, 128, 64), (4, 2, 8, 8), (70, 10, 128, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_append(dtype, lens, new, hq, hk, d, rot, interleaved, norm):
    """Error: one rounding, and in f32 before it d + 10 units of the norm's
    sum and factors, 4 for the rotation and 2^-22 for its cosines (a turn is
    reduced in f64 and given to f32 within 2^-25, times 2 pi): of the sizes
    that are summed."""
    c, _, _ = filled(dtype, hk, d, 16, lens, layers=2, layer=1, seed=d)
    m = sum(new)
    buf = torch.randn(m + 2, hq + 2 * hk + 1, d, device="cuda").to(dtype)[:m]
    q, k, v = buf[:, :hq], buf[:, hq:hq + hk], buf[:, hq + hk:hq + 2 * hk]
    w = [(1 + 0.2 * torch.randn(d, device="cuda")).to(dtype) if norm else None for _ in range(2)]
    inv = (10000.0 ** (-torch.arange(0, rot, 2, device="cuda").double() / max(rot, 1))).float() if rot else None
    ids = [2, 0, 1, 3]
    new_of = [new[i] for i in ids]
    cu = ints(np.concatenate([[0], np.cumsum(new_of)]))
    before = (c.k.clone(), c.v.clone())
    o = c.append(1, q if hq else None, k, v, cu, ints(ids), q_weight=w[0] if hq else None, k_weight=w[1], inv_freq=inv, interleaved=interleaved)
    c.check()
    pos = torch.cat([torch.arange(lens[s] - new[s], lens[s]) for s in ids]).cuda()
    seq = torch.cat([torch.full((new[s],), s) for s in ids]).cuda()
    u = HALF_STEP[dtype]
    for x, weight, got in ((q, w[0], o), (k, w[1], None)):
        if x.shape[1] == 0:
            continue
        y = x.double()
        units = 0
        if norm:
            y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
            units = d + 10
        size = y.abs()
        if rot:
            y, size = rotated(y, pos, inv, interleaved)
            units += 4 + 4
        tol = u * y.abs() + size * units * 2.0 ** -24 * 1.01 + SMALLEST[dtype]
        if got is None:
            page = c.page_table[seq.long(), (pos // 16).long()].long()
            got = c.k[1][page, :, (pos % 16).long()]
            before[0][1][page, :, (pos % 16).long()] = got
            before[1][1][page, :, (pos % 16).long()] = v
        close(got, y, tol)
    for x, y in zip((c.k, c.v), before):  # the values, and nothing else, were written
        assert torch.equal(torch.nan_to_num(x, 9.0), torch.nan_to_num(y, 9.0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens", [40, 900])
def test_append_of_many_sequences(dtype, tokens):
    """More sequences than a warp has lanes, with and without cu, in place."""
    hq, hk, d = 6, 2, 64
    lens = [1 + (5 * i) % 37 for i in range(tokens)]
    c, _, _ = filled(dtype, hk, d, 8, lens, seed=tokens)
    x = torch.randn(tokens, hq + 2 * hk, d, device="cuda").to(dtype)
    ids = list(np.random.default_rng(0).permutation(tokens))
    inv = (10000.0 ** (-torch.arange(0, d, 2, device="cuda").double() / d)).float()
    pos = torch.tensor([lens[s] - 1 for s in ids], device="cuda")
    y, size = rotated(x[:, :hq].double(), pos, inv, False)
    tol = HALF_STEP[dtype] * y.abs() + size * 8.1 * 2.0 ** -24 + SMALLEST[dtype]
    outs = []
    for cu in (None, ints(range(tokens + 1))):
        outs.append(c.append(0, x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], cu, ints(ids), inv_freq=inv))
        close(outs[-1], y, tol)
    assert torch.equal(outs[0], outs[1])
    page = c.page_table[torch.tensor(ids, device="cuda"), pos // 8].long()
    assert torch.equal(c.v[0][page, :, pos % 8], x[:, hq + hk:])
    c.append(0, x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], None, ints(ids), inv_freq=inv, q_out=x[:, :hq])
    assert torch.equal(x[:, :hq], outs[0])
    c.check()


def test_append_in_place_unaligned_and_far():
    for dtype in (F32, F16, BF16):
        c, _, _ = filled(dtype, 2, 64, 1024, [1], spare=0)
        c.page_table = torch.zeros(2, 1 << 15, dtype=torch.int32, device="cuda")  # every page of a far context is page 0
        c.seq_len[:] = ints([(1 << 25) - 5, 0])
        c = KVCache(c.k, c.v, c.page_table, c.seq_len, c.refcount)
        raw = torch.randn(3 * (8 * 64 + 1) + 1, device="cuda").to(dtype)
        x = raw.as_strided((3, 8, 64), (8 * 64 + 1, 64, 1), 1)
        inv = (10000.0 ** (-torch.arange(0, 64, 2, device="cuda").double() / 64)).float()
        y, size = rotated(x[:, :4].double(), torch.arange((1 << 25) - 8, (1 << 25) - 5, device="cuda"), inv, False)
        o = c.append(0, x[:, :4], x[:, 4:6], x[:, 6:], ints([0, 3]), None, inv_freq=inv, q_out=x[:, :4])
        assert o.data_ptr() == x.data_ptr()
        close(x[:, :4], y, HALF_STEP[dtype] * y.abs() + size * 8.1 * 2.0 ** -24 + SMALLEST[dtype])
        c.check()


@pytest.mark.parametrize("behind", [0, 1000])
def test_append_refusals_on_the_device(behind):
    """Few tokens, and the same six in front of a thousand that no sequence has."""
    for dtype, d in ((F16, 64), (F32, 17)):
        c, _, _ = filled(dtype, 2, d, 16, [40, 50])
        x = torch.randn(6 + behind, 6, d, device="cuda").to(dtype)

        def put(cu, ids):
            before, qo = c.k.clone(), torch.full((6 + behind, 2, d), 5.0, dtype=dtype, device="cuda")
            c.append(0, x[:, :2], x[:, 2:4], x[:, 4:], ints(cu), ints(ids), q_out=qo)
            moved = (torch.nan_to_num(c.k, 9.0) != torch.nan_to_num(before, 9.0)).any(-1).any(2)[0]
            return qo, int(moved.sum())

        qo, moved = put([0, 3, 6], [0, 0])  # the second entry of a sequence is refused
        assert (qo[3:] == 5).all() and (qo[:3] != 5).any() and moved == 3
        with pytest.raises(ValueError, match="used twice"):
            c.check()
        qo, moved = put([0, 3, 6], [77, -1])
        assert (qo == 5).all() and moved == 0
        with pytest.raises(ValueError, match="outside the table"):
            c.check()
        c.page_table[0, 2] = -1  # the new tokens' page
        qo, moved = put([0, 3, 6], [0, 1])
        assert moved == 3
        with pytest.raises(ValueError, match="without a page"):
            c.check()
        c.seq_len[0] = 2  # fewer than are new
        put([0, 6, 6], [0, 1])
        with pytest.raises(ValueError, match="without a page"):
            c.check()


# ---- pages --------------------------------------------------------------------------------------------------------


class Book:
    """The bookkeeping, one page at a time, on the host."""

    def __init__(self, pages, page, seqs, row):
        self.page, self.row = page, row
        self.refs, self.table, self.lens = [0] * pages, [[] for _ in range(seqs)], [0] * seqs

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def extend(self, ids, counts):
        for s, n in zip(ids, counts):
            self.lens[s] += n
            while len(self.table[s]) * self.page < self.lens[s]:
                self.table[s].append(self.take())

    def fork(self, parents, children):
        moves = []
        for a, b in zip(parents, children):
            full = self.lens[a] // self.page
            for p in self.table[a][:full]:
                self.refs[p] += 1
            self.table[b] = self.table[a][:full]
            if self.lens[a] % self.page:
                self.table[b].append(self.take())
                moves.append((self.table[a][full], self.table[b][-1]))
            self.lens[b] = self.lens[a]
        return moves

    def free(self, ids):
        for s in ids:
            for p in self.table[s]:
                self.refs[p] -= 1
            self.table[s], self.lens[s] = [], 0

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r]
        holes = [p for p, r in enumerate(self.refs) if not r and p < len(live)]
        to = dict(zip([p for p in live if p >= len(live)], holes))
        for src, dst in to.items():
            self.refs[dst], self.refs[src] = self.refs[src], 0
        self.table = [[to.get(p, p) for p in t] for t in self.table]
        return list(to.items())

    def same(self, c):
        assert c.refcount.tolist() == self.refs
        assert c.seq_len.tolist() == self.lens
        assert c.page_table.tolist() == [t + [-1] * (self.row - len(t)) for t in self.table]


def fresh(pages, page, seqs, row, layers=2, hk=3, d=40, dtype=F16):
    c = KVCache.create(layers, pages, page, hk, d, dtype, seqs, row)
    c.k.copy_(torch.arange(pages, device="cuda")[None, :, None, None, None] + torch.arange(layers, device="cuda")[:, None, None, None, None] * 0.25)
    c.v.copy_(c.k + 0.5)
    return c, Book(pages, page, seqs, row)


@pytest.mark.parametrize("pages, page, seqs, row, layers, hk, d, dtype", [
    (64, 16, 12, 9, 2, 3, 40, F16), (5000, 1, 40, 200, 1, 1, 8, F32), (300, 8, 1500, 20, 3, 1, 17, BF16), (1023, 32, 33, 40, 2, 2, 64, BF16),
    (9000, 4, 64, 150, 1, 1, 3, F16),
])
def test_pages_follow_the_bookkeeping(pages, page, seqs, row, layers, hk, d, dtype):
    """Random calls; each page's contents say where it came from."""
    c, b = fresh(pages, page, seqs, row, layers, hk, d, dtype)
    want = [c.k.clone(), c.v.clone()]
    rng = np.random.default_rng(pages)

    def moved(pairs):
        for x in want:
            old = x.clone()
            for s, t in pairs:
                x[:, t] = old[:, s]

    for step in range(40):
        empty = [s for s in range(seqs) if b.lens[s] == 0]
        held = [s for s in range(seqs) if b.lens[s]]
        left = b.refs.count(0)
        what = rng.choice(["extend", "extend", "fork", "free", "compact"])
        if what == "extend":
            ids = rng.permutation(seqs)[: rng.integers(1, seqs + 1)]
            counts, room = [], left
            for s in ids:
                n = int(rng.integers(0, max(2, row * page // 8)))
                n = min(n, row * page - b.lens[s])
                take = max(0, -(-(b.lens[s] + n) // page) - len(b.table[s]))
                if take > room:
                    n, take = 0, 0
                room -= take
                counts.append(n)
            b.extend(ids, counts)
            c.extend(ints(ids), ints(counts))
        elif what == "fork" and held and empty and left >= len(empty):
            children = rng.permutation(empty)[: rng.integers(1, len(empty) + 1)]
            parents = rng.choice(held, len(children))
            moved(b.fork(parents, children))
            c.fork(ints(parents), ints(children))
        elif what == "free" and held:
            ids = rng.permutation(held)[: rng.integers(1, len(held) // 2 + 2)]
            b.free(ids)
            c.free(ints(list(ids) + [ids[0]]))  # once more: nothing is left to free
        elif what == "compact":
            moved(b.compact())
            c.compact()
        b.same(c)
        assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1])
    c.check()


def state(c):
    return [x.clone() for x in (c.k, c.v, c.page_table, c.seq_len, c.refcount)]


def test_refused_calls_change_nothing():
    c, b = fresh(20, 16, 6, 8)
    c.extend(ints([0, 1, 2]), ints([40, 16, 100]))
    b.extend([0, 1, 2], [40, 16, 100])
    b.same(c)
    before = state(c)

    def refused(match, call):
        call()
        assert all(torch.equal(x, y) for x, y in zip(state(c), before))
        with pytest.raises(ValueError, match=match):
            c.check()

    refused("too few", lambda: c.extend(ints([3, 4]), ints([16 * 5, 16 * 5])))
    refused("more tokens", lambda: c.extend(ints([3, 2]), ints([1, 29])))
    refused("more tokens", lambda: c.extend(ints([3]), ints([2 ** 31 - 1])))
    refused("used twice", lambda: c.extend(ints([3, 3]), ints([1, 1])))
    refused("outside", lambda: c.extend(ints([3, 6]), ints([1, 1])))
    refused("outside", lambda: c.extend(ints([3, -1]), ints([1, 1])))
    refused("outside", lambda: c.extend(ints([3]), ints([-1])))
    refused("not empty", lambda: c.fork(ints([0]), ints([1])))
    refused("used twice", lambda: c.fork(ints([0, 0]), ints([3, 3])))
    refused("used twice", lambda: c.fork(ints([0, 3]), ints([3, 4])))
    refused("outside", lambda: c.fork(ints([6]), ints([3])))
    refused("outside", lambda: c.fork(ints([0]), ints([-7])))
    refused("outside", lambda: c.free(ints([17, -3])))
    refused("page number", lambda: c.copy_pages(ints([0, 1]), ints([2, 2])))
    refused("page number", lambda: c.copy_pages(ints([0, 2]), ints([2, 4])))
    refused("page number", lambda: c.copy_pages(ints([0, 20]), ints([5, 6])))
    refused("page number", lambda: c.copy_pages(ints([0]), ints([-1])))
    c.extend(ints([3, 4]), ints([16 * 8, 0]))  # a whole row, all pages but one
    b.extend([3], [128])
    b.same(c)
    c.extend(ints([4]), ints([16]))
    b.extend([4], [16])
    b.same(c)
    before = state(c)
    refused("too few", lambda: c.fork(ints([0]), ints([5])))  # a partly filled page, none free
    c.fork(ints([1]), ints([5]))  # full pages alone: none is needed
    b.fork([1], [5])
    b.same(c)
    c.check()


def test_more_pages_than_the_pool_has():
    """Lists that need more pages than there are at all: refused before the
    free ones are looked for, by every warp alike."""
    for _ in range(20):
        c, b = fresh(4, 16, 40, 64)
        c.extend(ints([0]), ints([5]))
        b.extend([0], [5])
        before = state(c)
        for call in (lambda: c.extend(ints([1]), ints([16 * 5])), lambda: c.extend(ints(range(1, 40)), ints([1] * 39)),
                     lambda: c.extend(ints([1, 2]), ints([16 * 60, 16 * 60])), lambda: c.fork(ints([0] * 30), ints(range(1, 31)))):
            call()
            assert all(torch.equal(x, y) for x, y in zip(state(c), before))
            with pytest.raises(ValueError, match="too few"):
                c.check()
        c.extend(ints([1]), ints([16 * 3]))
        b.extend([1], [16 * 3])
        b.same(c)
        c.check()


def test_copy_pages():
    c, _ = fresh(50, 8, 4, 4, layers=3)
    k, v = c.k.clone(), c.v.clone()
    src, dst = [3, 7, 7, 49, 11], [0, 1, 2, 48, 11]
    c.copy_pages(ints(src), ints(dst))
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    assert torch.equal(c.k, k) and torch.equal(c.v, v)
    c.check()


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements: its last pages are used."""
    page, hk, d = 64, 8, 128
    pages = (1 << 32) // (page * hk * d) + 8
    k = torch.zeros(1, pages, hk, page, d, dtype=F16, device="cuda")
    v = torch.zeros_like(k)
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[-6:] = 0
    c = KVCache(k, v, torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), ints([0, 0, 0]), refs)
    c.extend(ints([0]), ints([100]))
    assert c.page_table[0, :2].tolist() == [pages - 6, pages - 5]
    x = torch.randn(100, 24, d, device="cuda").half()
    for new, one in ((100, False), (1, True)):
        o = c.append(0, x[:new, :8], x[:new, 8:16], x[:new, 16:], None if one else ints([0, new]), ints([0]))
        o = c.attention(0, o, None if one else ints([0, new]), ints([0]))
        if not one:
            kk, vv = [x[:, 8:16].transpose(0, 1)], [x[:, 16:].transpose(0, 1)]
            want, tol = expected(x[:, :8], kk, vv, [0], [100], 1 / math.sqrt(d), True, 0)
            close(o, want, tol)
    c.fork(ints([0]), ints([1]))
    assert c.page_table[1, :2].tolist() == [pages - 6, pages - 4]
    assert torch.equal(k[0, pages - 4], k[0, pages - 5]) and torch.equal(v[0, pages - 4], v[0, pages - 5]) and bool((k[0, pages - 5] != 0).any())
    c.check()


# ---- together -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype, hq, hk, d", [(BF16, 8, 2, 128), (F16, 12, 12, 64), (F32, 6, 2, 64)])
def test_a_serving_run(dtype, hq, hk, d):
    """Prompts are read in, decoded on, forked, freed and compacted; every
    step's attention equals attention over what each sequence was given."""
    layers, page = 2, 16
    c = KVCache.create(layers, 80, page, hk, d, dtype, 6, 12)
    inv = (10000.0 ** (-torch.arange(0, d, 2, device="cuda").double() / d)).float()
    w = torch.ones(d, dtype=dtype, device="cuda")
    given = {s: [[torch.empty(hk, 0, d, dtype=dtype, device="cuda")] * 2 for _ in range(layers)] for s in range(6)}

    def step(ids, new):
        c.extend(ints(ids), ints(new))
        cu = ints(np.concatenate([[0], np.cumsum(new)]))
        for layer in range(layers):
            x = torch.randn(sum(new), hq + 2 * hk, d, device="cuda").to(dtype)
            q = c.append(layer, x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], cu, ints(ids), q_weight=w, k_weight=w, inv_freq=inv)
            at = 0
            for s, m in zip(ids, new):
                n = given[s][layer][0].shape[1]
                pos = torch.arange(n, n + m, device="cuda")
                page_no = c.page_table[s].long()[pos // page]
                given[s][layer] = [torch.cat([given[s][layer][0], c.k[layer][page_no, :, pos % page].transpose(0, 1)], 1),
                                   torch.cat([given[s][layer][1], x[at:at + m, hq + hk:].transpose(0, 1)], 1)]
                at += m
            o = c.attention(layer, q, cu, ints(ids))
            ks, vs = {s: given[s][layer][0] for s in ids}, {s: given[s][layer][1] for s in ids}
            want, tol = expected(q, ks, vs, ids, new, 1 / math.sqrt(d), True, 0)
            close(o, want, tol)

    step([0, 1], [70, 33])
    for _ in range(3):
        step([0, 1], [1, 1])
    c.fork(ints([0, 0, 1]), ints([2, 3, 4]))
    for s, t in ((0, 2), (0, 3), (1, 4)):
        given[t] = [list(x) for x in given[s]]
    step([4, 2, 0, 3], [1, 1, 1, 20])
    c.free(ints([0, 1]))
    given[0] = [[x[:, :0] for x in layer] for layer in given[0]]
    c.compact()
    used = int((c.refcount > 0).sum())
    assert (c.refcount[:used] > 0).all() and (c.refcount[used:] == 0).all()
    step([2, 3, 4], [5, 1, 1])
    step([0, 2], [90, 1])
    c.check()


def test_graphs_and_streams():
    """A decode step in a CUDA graph, replayed while the sequences grow, and
    two graphs that share nothing but the cache, replayed at once."""
    hq, hk, d = 8, 2, 64
    c = KVCache.create(1, 60, 16, hk, d, F16, 4, 20)
    c.extend(ints([0, 1, 2]), ints([100, 31, 5]))
    x = torch.randn(136, hq + 2 * hk, d, device="cuda").half()
    c.append(0, x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], ints([0, 100, 131, 136]), None)
    ids, one = ints([0, 1, 2]), ints([1, 1, 1])
    y = torch.randn(3, hq + 2 * hk, d, device="cuda").half()

    def decode():
        c.extend(ids, one)
        q = c.append(0, y[:, :hq], y[:, hq:hq + hk], y[:, hq + hk:], None, ids)
        return c.attention(0, q, None, ids)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    before = state(c)
    with torch.cuda.stream(side):
        decode()
    torch.cuda.current_stream().wait_stream(side)
    for x0, x1 in zip((c.k, c.v, c.page_table, c.seq_len, c.refcount), before):
        x0.copy_(x1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = decode()
    for _ in range(40):
        y.copy_(torch.randn_like(y))
        g.replay()
    captured = out.clone()
    after = state(c)
    for x0, x1 in zip((c.k, c.v, c.page_table, c.seq_len, c.refcount), after):
        x0.copy_(x1)
    assert c.seq_len.tolist() == [140, 71, 45, 0]
    q = y[:, :hq].contiguous()
    assert torch.equal(c.attention(0, q, None, ids), captured)
    qa, qb = torch.randn(3, hq, d, device="cuda").half(), torch.randn(3, hq, d, device="cuda").half()
    want = [c.attention(0, qa, None, ids).clone(), c.attention(0, qb, None, ids).clone()]
    graphs, outs = [], []
    for qq in (qa, qb):
        gg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gg):
            outs.append(c.attention(0, qq, None, ids))
        graphs.append(gg)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(50):
        for s, gg in zip(streams, graphs):
            with torch.cuda.stream(s):
                gg.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    c.check()


@pytest.mark.parametrize("dtype", [F32, F16])
def test_threads_on_one_stream(dtype):
    """Four threads call attention on one stream, and two on streams of their
    own, each with a batch of its own: long sequences that many blocks share,
    and chunks."""
    hq, hk, d = 8, 2, 64
    lens = [9000, 90, 5000, 700]
    c, _, _ = filled(dtype, hk, d, 16, lens)
    batches = [([0], [1]), ([2, 1], [1, 60]), ([3, 0], [300, 3]), ([2], [40]), ([0, 1, 2, 3], [1, 1, 1, 1]), ([3], [500])]
    work = []
    for i, (ids, new) in enumerate(batches):
        q = torch.randn(sum(new), hq, d, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").to(dtype)
        work.append((q, ints(np.concatenate([[0], np.cumsum(new)])), ints(ids)))
    want = [c.attention(0, *w) for w in work]
    shared = torch.cuda.Stream()
    torch.cuda.synchronize()
    bad = []

    def run(i):
        with torch.cuda.stream(shared if i < 4 else torch.cuda.Stream()):
            outs = [c.attention(0, *work[i]) for _ in range(200)]
        torch.cuda.synchronize()
        bad.extend(i for o in outs if not torch.equal(o, want[i]))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, f"{len(bad)} calls differ, of threads {sorted(set(bad))}"
    c.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_chunks_in_a_graph(dtype):
    """A mixed batch captured once and replayed while lengths, ids and the
    batch itself change: two graphs of it, beside an eager call."""
    hq, hk, d = 8, 2, 64
    lens = [700, 90, 1500, 40]
    c, ks, vs = filled(dtype, hk, d, 16, lens)
    q = torch.randn(220, hq, d, device="cuda").to(dtype)
    cu, ids = ints([0, 150, 151, 199, 220]), ints([0, 1, 2, 3])
    eager = c.attention(0, q, cu, ids).clone()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.attention(0, q, cu, ids))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        again = c.attention(0, q, cu, ids)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager) and torch.equal(again, eager)
    cu.copy_(ints([0, 1, 1, 180, 200]))
    ids.copy_(ints([3, 0, 2, 0]))
    c.seq_len[0] = 555
    outs[0].fill_(3.0)
    graphs[0].replay()
    short = [k[:, :555] if s == 0 else k for s, k in enumerate(ks)], [v[:, :555] if s == 0 else v for s, v in enumerate(vs)]
    want, tol = expected(q[:200], *short, [3, 0, 2, 0], [1, 0, 179, 20], 1 / math.sqrt(d), True, 0)
    close(outs[0][:200], want, tol)
    assert (outs[0][200:] == 3).all()
    c.check()


def test_python_names_of_the_status_bits():
    assert (kv_cache.NO_PAGES, kv_cache.BAD_SEQUENCE, kv_cache.ROW_FULL, kv_cache.BAD_PAGE) == (1, 2, 4, 8)
