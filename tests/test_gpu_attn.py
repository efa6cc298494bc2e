"""The attention operators through the C ABI against plain forms in 64 bits (numpy): the paged cache's write and read, the
attention of new tokens over it, and causal attention over packed prompts.

Tolerances. The cache is exact: a 16-bit value is the row's nearest, an 8-bit one is the rounded f32 quotient by the f32 step, so
reads are compared for equality. Attention is compared element by element with the bound of its own arithmetic (`_bound`):
  - a score is a sum of D products in f32 (each at most 2^-24 of the sum of their magnitudes, S), of operands whose parts
    drop at most 2^-23 of the largest product: |ds| <= (D + 8) 2^-24 S; the exponential's argument and result are f32: its
    relative error is |ds| + 2^-23 (|s| + 2), |s| <= S in base 2;
  - an output is a quotient of sums of L such weights in f32: relative to sum p |v|, twice the weights' error and
    (L + 16) 2^-24;
  - 16-bit outputs: half a step of the output, half a step of each weight where the weights are rounded (prompts), and what
    fp16 drops of weights under its normal range, 2^-25 of the largest weight's value each.
"""
import ctypes as C

import numpy as np
import pytest

from ijah_amd import synth
from ijah_amd.engine import bf16_to_f32, f32_to_bf16
from test_zz_no_alloc import hip_runtime

pytestmark = pytest.mark.gpu
PAGE = 64
_alive = []  # buffers of calls that may still be running


@pytest.fixture(autouse=True)
def _keep(eng):
    yield
    eng.sync()
    _alive.clear()


def up(eng, x):
    """a buffer that lives until the test has ended (calls only enqueue)"""
    _alive.append(eng.from_numpy(x))
    return _alive[-1]


def batch(eng, *a):
    _alive.append(eng.kv_seqs(*a))
    return _alive[-1]


HALF = {"F32": 2.0 ** -24, "BF16": 2.0 ** -8, "F16": 2.0 ** -11}  # half a step relative to the value


def cast(x, dtype):
    """f32 -> (the bytes to upload, the values they stand for)"""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "F32":
        return x, x
    if dtype == "BF16":
        b = f32_to_bf16(x)
        return b, bf16_to_f32(b)
    with np.errstate(over="ignore"):
        h = x.astype(np.float16)
    return h, h.astype(np.float32)


def values(buf, dtype, shape, offset=0):
    if dtype == "F32":
        return buf.download(np.float32, shape, offset)
    raw = buf.download(np.uint16, shape, offset)
    return bf16_to_f32(raw) if dtype == "BF16" else raw.view(np.float16).astype(np.float32)


def held(x, cache):
    """what the cache holds of f32 rows [..., D]"""
    x = np.asarray(x, np.float32)
    if cache != "I8":
        return cast(x, cache)[1]
    step = np.abs(x).max(-1, keepdims=True) * (np.float32(1) / np.float32(127))
    with np.errstate(all="ignore"):
        q = np.clip(np.rint(np.where(step > 0, x / np.where(step > 0, step, 1), 0)), -127, 127).astype(np.float32)
    return q * step


class Pool:
    """a batch's page tables over a pool whose pages are handed out in a random order"""

    def __init__(self, rng, lens, spare=3):
        self.lens = list(lens)
        per = [-(-v // PAGE) for v in lens]
        self.pages = sum(per) + spare
        ids, at = rng.permutation(self.pages), 0
        self.table = np.full((len(lens), max(max(per), 1)), -7, np.int32)
        for b, p in enumerate(per):
            self.table[b, :p] = ids[at:at + p]
            at += p


def offsets(counts):
    return np.cumsum([0] + list(counts)).astype(np.int32)


def rows_like(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


# ---------------------------------------------------------------------------------------------------- the cache
@pytest.mark.parametrize("cache", ["BF16", "F16", "I8"])
@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("heads,dim", [(1, 64), (4, 128), (3, 256)])
def test_write_then_read(eng, cache, dtype, heads, dim):
    """whole sequences in, single tokens and spans over them, everything back: neighbours in a page keep their values"""
    print(cache, dtype, heads, dim, flush=True)
    rng = np.random.default_rng(dim + heads)
    lens = [1, 63, 64, 65, 200, 17, 128]
    pool = Pool(rng, lens)
    kv = eng.kv_create(2, pool.pages, heads, dim, cache)
    seqs = batch(eng, pool.table, lens, offsets(lens))
    T = sum(lens)
    k, v = rows_like(rng, T, heads, dim), 3 * rows_like(rng, T, heads, dim)
    k[5], v[7] = 0, 0
    want = {}
    for layer in (0, 1):
        kr, kval = cast(k + layer, dtype)
        vr, vval = cast(v - layer, dtype)
        kv.write_bufs(layer, seqs, T, up(eng, kr), up(eng, vr), dtype)
        want[layer] = [held(kval, cache), held(vval, cache)]
    # the newest tokens of each sequence again: 1, 63, 2, 40, 130, 0 and 64 of them
    new = [1, 63, 2, 40, 130, 0, 64]
    n = sum(new)
    k2, v2 = rows_like(rng, n, heads, dim), rows_like(rng, n, heads, dim)
    kr, kval = cast(k2, dtype)
    vr, vval = cast(v2, dtype)
    kv.write_bufs(1, batch(eng, pool.table, lens, offsets(new)), n, up(eng, kr), up(eng, vr), dtype)
    at, o = offsets(lens), offsets(new)
    for b, m in enumerate(new):
        for x, val in zip(want[1], (kval, vval)):
            x[at[b + 1] - m:at[b + 1]] = held(val[o[b]:o[b] + m], cache)
    for layer in (0, 1):
        kb, vb = (eng.alloc(T * heads * dim * (4 if dtype == "F32" else 2)) for _ in range(2))
        kv.read_bufs(layer, seqs, T, kb, vb, dtype)
        for b, x in zip((kb, vb), want[layer]):
            got = values(b, dtype, (T, heads, dim))
            assert np.array_equal(got, cast(x, dtype)[1]), (layer, np.abs(got - x).max())


@pytest.mark.parametrize("cache", ["BF16", "F16", "I8"])
@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("heads,dim", [(1, 64), (9, 64), (5, 128), (2, 256), (3, 256)])
def test_few_rows_of_each_sequence(eng, cache, dtype, heads, dim):
    """no row to five of each sequence, between rows of none, some before token 0, in no page, not finite: the same bytes as
    whole sequences written"""
    print(cache, dtype, heads, dim, flush=True)
    rng = np.random.default_rng(7 * dim + heads)
    lens = [1, 63, 64, 66, 200, 0, 3, 130, 65]
    new = [1, 0, 3, 4, 2, 0, 5, 1, 5]
    pool = Pool(rng, lens)
    table = pool.table.copy()
    table[8, 1] = pool.pages  # the last sequence's token 64
    T, lead = sum(lens), 2
    k, v = rows_like(rng, T, heads, dim), rows_like(rng, T, heads, dim)
    at = offsets(lens)
    k[at[4] - 1, 0, 3], v[at[4] - 2, heads - 1, dim - 1], k[at[3] - 1] = np.inf, np.nan, 0
    (kr, kv_), (vr, vv_) = cast(k, dtype), cast(v, dtype)
    few, full = (eng.kv_create(1, pool.pages, heads, dim, cache) for _ in range(2))
    whole = batch(eng, pool.table, lens, at)
    full.write_bufs(0, whole, T, up(eng, kr), up(eng, vr), dtype)
    few.write_bufs(0, whole, T, up(eng, np.zeros_like(kr)), up(eng, np.zeros_like(vr)), dtype)
    src, mine = [], []
    for b, m in enumerate(new):
        for i in range(m):
            t = lens[b] - m + i
            src.append(at[b] + t if t >= 0 else 0)
            if t >= 0 and not (b == 8 and t == 64):
                mine.append(at[b] + t)
    R = lead + len(src) + 3
    rows_k, rows_v = np.full((R, heads, dim), 9, kr.dtype), np.full((R, heads, dim), 9, vr.dtype)
    rows_k[lead:lead + len(src)], rows_v[lead:lead + len(src)] = kr[src], vr[src]
    few.write_bufs(0, batch(eng, table, lens, offsets(new) + np.int32(lead)), R, up(eng, rows_k), up(eng, rows_v), dtype)
    got = []
    for c in (full, few):
        bufs = [eng.alloc(T * heads * dim * 4) for _ in range(2)]
        c.read_bufs(0, whole, T, *bufs)
        got.append([b.download(np.uint32, (T, heads, dim)) for b in bufs])
    for a, b in zip(*got):
        want = np.zeros_like(a)
        want[mine] = a[mine]
        assert np.array_equal(b, want)


@pytest.mark.parametrize("rows", [12, 700])
def test_eight_bit_values_around_halves(eng, rows):
    """quotients at a half and within a few ulp of one, rows of every magnitude down to the smallest subnormals: as the plain
    form's division and rounding say"""
    rng = np.random.default_rng(rows)
    dim = 64
    top = np.ldexp(np.float32(1), rng.integers(-149, 127, rows)).astype(np.float32) * rng.uniform(1, 2, rows).astype(np.float32)
    top[:4] = [2.0 ** -149, 2.0 ** -126, 3.4e38, 127]
    step = top * (np.float32(1) / np.float32(127))
    x = (step[:, None] * (rng.integers(-127, 127, (rows, dim)) + 0.5).astype(np.float32)).astype(np.float32)
    for i in range(dim):  # up to three ulp off
        for _ in range(i % 4):
            x[:, i] = np.nextafter(x[:, i], np.float32(np.inf if i & 4 else 0))
    x = np.clip(x, -top[:, None], top[:, None])
    x[:, 5] = top
    pool = Pool(rng, [rows])
    kv = eng.kv_create(1, pool.pages, 1, dim, "I8")
    seqs = batch(eng, pool.table, [rows], offsets([rows]))
    kv.write(0, seqs, x, -x)
    k, v = kv.read(0, seqs, rows)
    want = held(x, "I8")
    assert np.array_equal(k.reshape(rows, dim), want) and np.array_equal(v.reshape(rows, dim), -want)


@pytest.mark.parametrize("cache", ["BF16", "I8"])
def test_cache_strides_offsets_and_single_rows(eng, cache):
    """rows inside wider rows (q, k, v side by side), at an offset, one per sequence without a row table; rows that no
    sequence names and the gaps between rows stay as they were"""
    rng = np.random.default_rng(3)
    heads, dim, ld, off = 2, 128, 640, 64
    lens = [5, 64, 129, 1]
    pool = Pool(rng, lens)
    kv = eng.kv_create(1, pool.pages, heads, dim, cache)
    R = len(lens)
    wide = rows_like(rng, R + 1, ld)
    b = up(eng, wide)
    seqs = batch(eng, pool.table, lens)
    kv.write_bufs(0, seqs, R, b, b, k_off=off * 4, v_off=(off + 256) * 4, ldk=ld, ldv=ld)
    out = np.full((R + 2, ld), -99, np.float32)
    ob = up(eng, out)
    kv.read_bufs(0, seqs, R, ob, ob, k_off=off * 4, v_off=(off + 256) * 4, ldk=ld, ldv=ld)
    flat = wide.reshape(-1)
    k = np.stack([flat[off + r * ld:off + r * ld + 256] for r in range(R)]).reshape(R, heads, dim)
    v = np.stack([flat[off + 256 + r * ld:off + 512 + r * ld] for r in range(R)]).reshape(R, heads, dim)
    of = out.reshape(-1)
    for r in range(R):
        of[off + r * ld:off + r * ld + 256] = held(k[r], cache).reshape(-1)
        of[off + 256 + r * ld:off + 512 + r * ld] = held(v[r], cache).reshape(-1)
    assert np.array_equal(ob.download(np.float32, out.shape), out)


def test_rows_before_the_first_token_and_bad_pages(eng):
    """more rows than tokens, empty sequences, page ids outside the pool, lengths outside the table: skipped when written,
    zeros when read, no neighbour touched"""
    rng = np.random.default_rng(4)
    heads, dim = 2, 64
    pool = Pool(rng, [70, 70, 70, 128])
    kv = eng.kv_create(1, pool.pages, heads, dim, "BF16")
    base = rows_like(rng, 338, heads, dim)
    whole = batch(eng, pool.table, [70, 70, 70, 128], offsets([70, 70, 70, 128]))
    kv.write(0, whole, base, base)
    table = pool.table.copy()
    table[1, 0], table[2, 1] = pool.pages, -1
    lens, new = [3, 70, 70, 1 << 30], [5, 70, 4, 130]  # the last is clamped to the table's 128
    R = sum(new)
    x = rows_like(rng, R, heads, dim)
    seqs = batch(eng, table, lens, offsets(new))
    kv.write(0, seqs, x, -x)
    want = held(x, "BF16").copy()
    want[0:2] = 0            # sequence 0: rows at tokens -2, -1
    want[5:69] = 0           # sequence 1: its first page is no page
    want[75:79] = 0          # sequence 2: tokens 66..69 in no page
    want[79:81] = 0          # sequence 3: 130 rows of 128 tokens
    k, v = kv.read(0, seqs, R)
    assert np.array_equal(k, want) and np.array_equal(v, -want)
    k, _ = kv.read(0, whole, 338)
    old = held(base, "BF16").copy()
    old[0:3] = want[2:5]
    old[70 + 64:140] = want[69:75]
    old[210:338] = want[81:]
    assert np.array_equal(k, old)


def test_i8_rows_that_are_not_finite(eng):
    """an infinity or a NaN makes its own row NaN, in its own head; tiny and huge rows keep their steps"""
    rng = np.random.default_rng(5)
    heads, dim, lens = 2, 128, [20]
    pool = Pool(rng, lens)
    kv = eng.kv_create(1, pool.pages, heads, dim, "I8")
    x = rows_like(rng, 20, heads, dim)
    x[3, 0, 5], x[4, 1, 100] = np.inf, np.nan
    x[5] *= np.float32(1e-30)
    x[6] *= np.float32(1e30)
    seqs = batch(eng, pool.table, lens, offsets(lens))
    kv.write(0, seqs, x, x)
    k, v = kv.read(0, seqs, 20)
    want = held(x, "I8")
    want[3, 0], want[4, 1] = np.nan, np.nan
    assert np.array_equal(k, want, equal_nan=True) and np.array_equal(v, want, equal_nan=True)


# ---------------------------------------------------------------------------------------------------- attention
def plain(q, k, v, seen, scale):
    """one sequence in f64: q [m, Hq, D], k, v [L, H, D], seen [m] = the last key each row sees -> out, and what `_bound`
    needs of each row: sum p |v| and the largest sum of a score's magnitudes"""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    m, Hq, D = q.shape
    L, H, _ = k.shape
    out, mag, S, vmax = np.zeros((m, Hq, D)), np.zeros((m, Hq, D)), np.zeros((m, Hq, 1)), np.zeros((m, Hq, D))
    sees = np.arange(L) <= np.asarray(seen)[:, None]
    some = sees.any(1)
    if not some.any():
        return out, mag, S, vmax
    finite = np.isfinite(k).all() and np.isfinite(v).all()
    for h in range(Hq):
        kh, vh = k[:, h // (Hq // H)], v[:, h // (Hq // H)]
        rows = np.nonzero(some)[0]
        for r in np.split(rows, range(256, len(rows), 256)):  # (a few rows at a time; one by one where 0 times a value is not 0)
            for i in ([r] if finite else r[:, None]):
                n = L if finite else int(sees[i[0]].sum())
                on = sees[i][:, :n]
                s = np.where(on, q[i, h] @ kh[:n].T * scale, -np.inf)
                p = np.where(on, np.exp(s - s.max(1, keepdims=True)), 0)
                l = p.sum(1, keepdims=True)
                out[i, h] = p @ vh[:n] / l
                mag[i, h] = p @ np.abs(vh[:n]) / l
                vmax[i, h] = np.abs(vh[:n]).max(0) / l
                S[i, h] = np.where(on, scale * (np.abs(q[i, h]) @ np.abs(kh[:n]).T), 0).max(1, keepdims=True)
    return out, mag, S, vmax


def _bound(out, mag, S, vmax, L, D, dtype, prompt):
    ds = (D + 8) * 2.0 ** -24 * S * 1.4427
    w = ds + 2.0 ** -23 * (1.4427 * S + 2)
    b = (2 * w + (L + 16) * 2.0 ** -24) * mag
    if dtype != "F32":
        b = b + HALF[dtype] * np.abs(out) + (HALF[dtype] * mag if prompt else 0)
        if dtype == "F16":
            b = b + 2.0 ** -25 * (1 + (L * vmax if prompt else 0))
    return b + 1e-37


def check(got, parts, L, D, dtype, prompt, what=""):
    out = parts[0]
    b = _bound(*parts, L, D, dtype, prompt)
    with np.errstate(invalid="ignore"):
        # where the definition gives no number (fp16 has rounded a value to infinity), the kernel must not give one either
        bad = np.where(np.isfinite(out), ~(np.abs(got - out) <= b), np.isfinite(got))
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(np.abs(got - out) / b)))


def decode_case(eng, rng, lens, new, Hq, H, D, cache, dtype, scale=None, garbage=True):
    pool = Pool(rng, [max(v, 1) for v in lens])
    kv = eng.kv_create(1, pool.pages, H, D, cache)
    if garbage:  # every page full of NaN first: nothing behind a sequence's last token may be seen
        all_pages = np.arange(pool.pages, dtype=np.int32)[None]
        n = pool.pages * PAGE
        junk = np.full((n, H, D), np.nan, np.float32)
        kv.write(0, batch(eng, all_pages, [n], [0, n]), junk, junk)
    T = sum(lens)
    k = rows_like(rng, max(T, 1), H, D) * np.exp(0.4 * rows_like(rng, 1, H, D))
    v = rows_like(rng, max(T, 1), H, D)
    if T:
        kv.write(0, batch(eng, pool.table, lens, offsets(lens)), k[:T], v[:T])
    R = sum(new)
    qr, q = cast(rows_like(rng, R, Hq, D), dtype)
    seqs = batch(eng, pool.table, lens, offsets(new))
    qb, ob = up(eng, qr), up(eng, np.full((R + 1) * Hq * D, 7, qr.dtype))
    kv.attend_bufs(0, seqs, R, Hq, qb, ob, dtype, scale)
    got = values(ob, dtype, (R + 1, Hq, D))
    assert np.array_equal(got[R], values(up(eng, np.full(Hq * D, 7, qr.dtype)), dtype, (Hq, D)))
    kh, vh = held(k, cache), held(v, cache)
    at, o = offsets(lens), offsets(new)
    for b in range(len(lens)):
        m = new[b]
        if m:
            parts = plain(q[o[b]:o[b] + m], kh[at[b]:at[b + 1]], vh[at[b]:at[b + 1]], lens[b] - m + np.arange(m),
                          scale or D ** -0.5)
            check(got[o[b]:o[b] + m], parts, lens[b], D, dtype, False, (b, lens[b], m))
    return kv, seqs, qb, ob, R


@pytest.mark.parametrize("cache", ["BF16", "F16", "I8"])
@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("Hq,H,D", [(8, 2, 64), (16, 2, 128), (4, 2, 256)])
def test_decode_lengths(eng, cache, dtype, Hq, H, D):
    """one token of each of a ragged batch, from an empty sequence to one that several workgroups share"""
    print(cache, dtype, Hq, H, D, flush=True)
    lens = [0, 1, 2, 63, 64, 65, 127, 500, 0, 1300]
    decode_case(eng, np.random.default_rng(D + Hq), lens, [1] * len(lens), Hq, H, D, cache, dtype)


@pytest.mark.parametrize("Hq,H,D,cache", [(3, 3, 64, "BF16"), (20, 4, 64, "I8"), (17, 1, 128, "F16"), (80, 5, 128, "BF16"),
                                          (48, 1, 256, "I8"), (1, 1, 256, "BF16"), (24, 2, 128, "I8")])
def test_decode_heads_and_drafts(eng, Hq, H, D, cache):
    """groups of 1 to 48 query heads; between no and seven drafts of a sequence, some with more rows than tokens"""
    print(Hq, H, D, cache, flush=True)
    lens, new = [3, 300, 64, 70, 0, 129, 700], [5, 2, 0, 7, 1, 3, 1]
    decode_case(eng, np.random.default_rng(Hq), lens, new, Hq, H, D, cache, "F32")


@pytest.mark.parametrize("lens,Hq,H,D,cache", [([20000], 8, 1, 128, "BF16"), ([30001], 4, 2, 64, "I8"),
                                               ([9000, 1, 77, 5000], 16, 2, 256, "F16")])
def test_decode_long(eng, lens, Hq, H, D, cache):
    """lengths split over many workgroups; the same call gives the same bits"""
    print(lens, flush=True)
    kv, seqs, qb, ob, R = decode_case(eng, np.random.default_rng(9), lens, [1] * len(lens), Hq, H, D, cache, "F32",
                                      garbage=False)
    first = ob.download(np.uint32)
    for _ in range(5):
        kv.attend_bufs(0, seqs, R, Hq, qb, ob)
        assert np.array_equal(ob.download(np.uint32), first)


def test_decode_many_short_sequences(eng):
    """more groups than workgroups, each far smaller than a share"""
    rng = np.random.default_rng(11)
    lens = [int(x) for x in rng.integers(0, 150, 400)]
    decode_case(eng, rng, lens, [1] * 400, 8, 4, 64, "BF16", "F32")


@pytest.mark.parametrize("cache", ["F16", "I8"])
def test_decode_ranges(eng, cache):
    """rows, keys and values far from 1: fp16 parts must not overflow or lose what f32 keeps"""
    rng = np.random.default_rng(12)
    H, Hq, D, L = 2, 4, 128, 500
    pool = Pool(rng, [L])
    kv = eng.kv_create(1, pool.pages, H, D, cache)
    seqs1 = batch(eng, pool.table, [L], [0, L])
    for qs, ks, vs in ((1e6, 1e-5, 1e3), (1e6, 1e-5, 1e2), (1e-6, 1e4, 1e-3), (1e-3, 1.0, 1e-4 if cache == "F16" else 1e-20)):
        k, v = ks * rows_like(rng, L, H, D), vs * rows_like(rng, L, H, D)
        v[::7] *= 100
        if cache == "I8":
            v[3] *= np.float32(1e-12)
        kv.write(0, seqs1, k, v)
        q = qs * rows_like(rng, 1, Hq, D)
        got = kv.attend(0, batch(eng, pool.table, [L]), q)
        check(got, plain(q, held(k, cache), held(v, cache), [L - 1], D ** -0.5), L, D, "F32", False, (qs, ks, vs))


def test_decode_scores_far_apart(eng):
    """one key far above the others, and rows whose scores lie hundreds apart from page to page"""
    rng = np.random.default_rng(13)
    H, Hq, D, L = 1, 2, 64, 1000
    pool = Pool(rng, [L])
    kv = eng.kv_create(1, pool.pages, H, D, "BF16")
    k, v = rows_like(rng, L, H, D), rows_like(rng, L, H, D)
    k *= (1 + np.arange(L)[:, None, None] % 130).astype(np.float32)
    kv.write(0, batch(eng, pool.table, [L], [0, L]), k, v)
    q = 4 * rows_like(rng, 1, Hq, D)
    got = kv.attend(0, batch(eng, pool.table, [L]), q)
    check(got, plain(q, held(k, "BF16"), held(v, "BF16"), [L - 1], D ** -0.5), L, D, "F32", False)


@pytest.mark.parametrize("cache", ["BF16", "F16", "I8"])
def test_decode_drafts_do_not_see_later_drafts(eng, cache):
    """keys and values that are not finite at later drafts' tokens: earlier drafts are as without them"""
    rng = np.random.default_rng(14)
    H, Hq, D, L, m = 2, 8, 128, 130, 5
    pool = Pool(rng, [L])
    kv = eng.kv_create(1, pool.pages, H, D, cache)
    k, v = rows_like(rng, L, H, D), rows_like(rng, L, H, D)
    whole = batch(eng, pool.table, [L], [0, L])
    q = rows_like(rng, m, Hq, D)
    seqs = batch(eng, pool.table, [L], [0, m])
    kv.write(0, whole, k, v)
    clean = kv.attend(0, seqs, q)
    k[L - 2, 0, 3], v[L - 2, 0, 7], v[L - 1, 1, 9] = np.inf, np.nan, -np.inf
    kv.write(0, whole, k, v)
    got = kv.attend(0, seqs, q)
    assert np.array_equal(got[:3], clean[:3])       # tokens up to L - 3
    assert np.array_equal(got[3, 4:], clean[3, 4:])  # the second key head is clean there
    assert not np.isfinite(got[3, :4, 7]).any() and not np.isfinite(got[4, 4:, 9]).any()
    if cache != "I8":
        assert np.array_equal(np.delete(got[4, 4:], 9, 1), np.delete(clean[4, 4:], 9, 1))


def test_decode_in_place_and_strided(eng):
    """out = q's own rows, inside wider rows; a bad page is a page without tokens"""
    rng = np.random.default_rng(15)
    H, Hq, D, ld = 2, 4, 64, 320
    lens = [200, 64, 90]
    pool = Pool(rng, lens)
    kv = eng.kv_create(1, pool.pages, H, D, "BF16")
    k, v = rows_like(rng, 354, H, D), rows_like(rng, 354, H, D)
    kv.write(0, batch(eng, pool.table, lens, offsets(lens)), k, v)
    table = pool.table.copy()
    table[0, 1], table[1, 0] = 10 ** 6, -1
    want = rows_like(rng, 4 * ld)
    b = up(eng, want)
    kv.attend_bufs(0, batch(eng, table, lens), 3, Hq, b, b, q_off=128, out_off=128, ldq=ld, ldo=ld)
    got = b.download(np.float32)
    kh, vh = held(k, "BF16"), held(v, "BF16")
    keep = [np.r_[0:64, 128:200], np.r_[0:0], np.r_[264:354]]
    for r in range(3):
        lo = 32 + r * ld
        parts = plain(want[lo:lo + 256].reshape(1, Hq, D), kh[keep[r]], vh[keep[r]], [10 ** 6], D ** -0.5)
        check(got[lo:lo + 256].reshape(1, Hq, D), parts, 200, D, "F32", False, r)
        got[lo:lo + 256] = want[lo:lo + 256]
    assert np.array_equal(got, want)


def prompt_case(eng, rng, nq, nk, Hq, H, D, dtype, scale=None, lead=0, q=None, k=None, v=None):
    """packed sequences behind `lead` rows that belong to none"""
    Rq, Rk = lead + sum(nq) + 2, lead + sum(nk) + 1
    q = rows_like(rng, Rq, Hq, D) if q is None else q
    k = rows_like(rng, Rk, H, D) * np.exp(0.3 * rows_like(rng, 1, H, D)) if k is None else k
    v = rows_like(rng, Rk, H, D) if v is None else v
    (qr, q), (kr, k), (vr, v) = (cast(x, dtype) for x in (q, k, v))
    qo, ko = offsets(nq) + lead, offsets(nk) + lead
    ob = up(eng, np.full(Rq * Hq * D, 7, qr.dtype))
    untouched = values(ob, dtype, (Rq, Hq, D))
    eng.attn_prompt_bufs(len(nq), up(eng, qo), up(eng, ko), Rq, Rk, Hq, H, D, up(eng, qr),
                         up(eng, kr), up(eng, vr), ob, dtype, scale)
    got = values(ob, dtype, (Rq, Hq, D))
    assert np.array_equal(got[:lead], untouched[:lead]) and np.array_equal(got[-2:], untouched[-2:])
    for b, (m, n) in enumerate(zip(nq, nk)):
        if m:
            parts = plain(q[qo[b]:qo[b + 1]], k[ko[b]:ko[b + 1]], v[ko[b]:ko[b + 1]], np.arange(m) + n - m, scale or D ** -0.5)
            check(got[qo[b]:qo[b + 1]], parts, n, D, dtype, True, (b, m, n))
    return got


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("Hq,H,D", [(2, 1, 64), (4, 2, 128), (3, 3, 256)])
def test_prompt_lengths(eng, dtype, Hq, H, D):
    print(dtype, Hq, H, D, flush=True)
    nq = [1, 31, 32, 33, 0, 64, 65, 127, 128, 129, 200, 2]
    prompt_case(eng, np.random.default_rng(D), nq, nq, Hq, H, D, dtype)


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
def test_prompt_later_chunks_and_fewer_keys(eng, dtype):
    """keys of earlier chunks in front; sequences with fewer keys than rows, and with none: their first rows are zero"""
    print(dtype, flush=True)
    nq, nk = [70, 1, 5, 130, 40, 3], [300, 129, 0, 64, 39, 500]
    got = prompt_case(eng, np.random.default_rng(21), nq, nk, 4, 1, 128, dtype, lead=3)
    assert not got[3 + 71:3 + 76].any()          # no keys
    assert not got[3 + 76:3 + 76 + 66].any()     # 130 rows, 64 keys


@pytest.mark.parametrize("Hq,H,D", [(8, 8, 64), (17, 1, 128), (10, 2, 256)])
def test_prompt_heads(eng, Hq, H, D):
    prompt_case(eng, np.random.default_rng(Hq), [50, 90], [50, 200], Hq, H, D, "BF16", scale=0.2)


@pytest.mark.parametrize("dtype,D", [("F32", 64), ("F32", 256), ("BF16", 128), ("F16", 128), ("F16", 256)])
def test_prompt_masked_values_that_are_not_finite(eng, dtype, D):
    """infinities and NaN at keys that a row does not see (later ones, other sequences', rows that belong to none) change
    nothing in it"""
    print(dtype, D, flush=True)
    rng = np.random.default_rng(22)
    nq, Hq, H = [70, 200, 33], 2, 1
    R = 1 + sum(nq) + 2
    q, k, v = rows_like(rng, R, Hq, D), rows_like(rng, R - 1, H, D), rows_like(rng, R - 1, H, D)
    clean = prompt_case(eng, rng, nq, nq, Hq, H, D, dtype, lead=1, q=q, k=k, v=v)
    k2, v2 = k.copy(), v.copy()
    k2[0], v2[0] = np.nan, np.inf            # a row of no sequence
    k2[-1], v2[-1] = np.inf, np.nan
    v2[1 + 69, 0, 3] = np.inf                # the first sequence's last key
    k2[71 + 150], v2[71 + 150, 0, 5], v2[71 + 180, 0, 6] = np.nan, np.nan, -np.inf
    (qr, _), (kr, _), (vr, _) = (cast(x, dtype) for x in (q, k2, v2))
    ob = eng.alloc(qr.nbytes)
    qo = up(eng, offsets(nq) + 1)
    eng.attn_prompt_bufs(3, qo, qo, R, R - 1, Hq, H, D, up(eng, qr), up(eng, kr), up(eng, vr), ob, dtype)
    got = values(ob, dtype, (R, Hq, D))
    assert np.array_equal(got[1:70], clean[1:70])
    assert np.array_equal(np.delete(got[70], 3, 1), np.delete(clean[70], 3, 1)) and not np.isfinite(got[70, :, 3]).any()
    assert np.array_equal(got[71:221], clean[71:221])
    assert np.array_equal(got[271:304], clean[271:304])
    assert not np.isfinite(got[71 + 180:271, :, 6]).any()


def test_prompt_strided(eng):
    """q, k, v and out as columns of wider rows"""
    rng = np.random.default_rng(23)
    n, Hq, H, D = 100, 2, 1, 64
    ld = 128 + 64 + 64 + 128
    wide = rows_like(rng, n, ld)
    b = up(eng, wide)
    ob = up(eng, np.full((n, 200), 7, np.float32))
    r = up(eng, np.array([0, n], np.int32))
    eng.attn_prompt_bufs(1, r, None, n, n, Hq, H, D, b, b, b, ob, q_off=0, k_off=512, v_off=768, out_off=64, ldq=ld, ldk=ld,
                         ldv=ld, ldo=180)
    got = ob.download(np.float32)
    at = 16 + np.arange(n)[:, None] * 180 + np.arange(128)
    q, k, v = (wide[:, a:z].reshape(n, -1, D) for a, z in ((0, 128), (128, 192), (192, 256)))
    check(got[at].reshape(n, Hq, D), plain(q, k, v, np.arange(n), D ** -0.5), n, D, "F32", True)
    rest = np.ones(got.size, bool)
    rest[at.reshape(-1)] = False
    assert (got[rest] == 7).all()


def test_prompt_ranges_f32(eng):
    """32-bit rows keep their range and precision: tiny and huge elements side by side"""
    rng = np.random.default_rng(24)
    n, Hq, H, D = 150, 2, 1, 128
    q, k, v = rows_like(rng, n, Hq, D), rows_like(rng, n, H, D), rows_like(rng, n, H, D)
    q *= np.float32(1e8)
    k *= np.float32(1e-8)
    v *= np.exp(8 * rows_like(rng, n, 1, 1))
    got = eng.attn_prompt(q, k, v, [0, n])
    check(got, plain(q, k, v, np.arange(n), D ** -0.5), n, D, "F32", True)


@pytest.mark.parametrize("dtype,Hq,H,D", [("BF16", 64, 8, 64), ("F16", 48, 4, 128), ("BF16", 44, 2, 256)])
def test_prompt_one_stream(eng, dtype, Hq, H, D):
    """more blocks than CUs: a workgroup of four waves takes a block's tiles alone"""
    print(dtype, Hq, D, flush=True)
    prompt_case(eng, np.random.default_rng(D), [700, 130], [740, 130], Hq, H, D, dtype)


@pytest.mark.parametrize("dtype,D", [("F32", 128), ("BF16", 64), ("F16", 128), ("BF16", 256)])
def test_prompt_two_streams_with_values_that_are_not_finite(eng, dtype, D):
    """few blocks and many keys: two streams of tiles, the second without a tile in the last step or with; later keys that are
    not finite change nothing in earlier rows"""
    print(dtype, D, flush=True)
    rng = np.random.default_rng(25)
    for n in (600, 640, 673):
        q, k, v = rows_like(rng, n, 2, D), rows_like(rng, n, 1, D), rows_like(rng, n, 1, D)
        (qr, q), (kr, _), (vr, _) = (cast(x, dtype) for x in (q, k, v))
        r, ob = up(eng, np.array([0, n], np.int32)), eng.alloc(qr.nbytes)
        eng.attn_prompt_bufs(1, r, None, n, n, 2, 1, D, up(eng, qr), up(eng, kr), up(eng, vr), ob, dtype)
        clean = values(ob, dtype, (n, 2, D))
        check(clean, plain(q, cast(k, dtype)[1], cast(v, dtype)[1], np.arange(n), D ** -0.5), n, D, dtype, True, n)
        at = n - 70
        v[at, 0, 1], v[at + 40, 0, 2], k[n - 3] = np.inf, np.nan, np.nan
        (kr, _), (vr, _) = (cast(x, dtype) for x in (k, v))
        eng.attn_prompt_bufs(1, r, None, n, n, 2, 1, D, up(eng, qr), up(eng, kr), up(eng, vr), ob, dtype)
        got = values(ob, dtype, (n, 2, D))
        assert np.array_equal(got[:at], clean[:at])
        assert not np.isfinite(got[at:, :, 1]).any() and not np.isfinite(got[at + 40:, :, 2]).any()
        assert np.array_equal(got[at:n - 3, :, 3:], clean[at:n - 3, :, 3:])


@pytest.mark.parametrize("n", [64, 65, 130, 256, 257, 700])
def test_many_sequences(eng, n):
    """batches around the sizes at which the kernels divide them differently: one lane a sequence, several, all threads"""
    print(n, flush=True)
    rng = np.random.default_rng(n)
    H, Hq, D = 1, 4, 64
    lens = [int(x) for x in rng.integers(0, 200, n)]
    new = [min(v, int(x)) for v, x in zip(lens, rng.integers(0, 3, n))]
    decode_case(eng, rng, lens, new, Hq, H, D, "F16", "F32")  # writes and reads are checked below
    pool = Pool(rng, [max(v, 1) for v in lens])
    kv = eng.kv_create(1, pool.pages, H, D, "BF16")
    T = sum(lens)
    k = rows_like(rng, T, H, D)
    seqs = batch(eng, pool.table, lens, offsets(lens))
    kv.write(0, seqs, k, -k)
    got = kv.read(0, seqs, T)
    assert np.array_equal(got[0], held(k, "BF16")) and np.array_equal(got[1], -held(k, "BF16"))
    prompt_case(eng, rng, new, lens, Hq, H, D, "BF16")
    prompt_case(eng, rng, [v % 37 for v in lens], [v % 41 for v in lens], Hq, H, D, "F32")


def test_offsets_past_32_bits(eng):
    """pages beyond 4 GB of the cache, in its last layer, and rows beyond 4 GB of a prompt's keys"""
    rng = np.random.default_rng(41)
    H, Hq, D, L = 4, 8, 128, 200
    kv = eng.kv_create(2, 40000, H, D, "BF16")  # 5.2 GB a layer
    assert kv.nbytes > 2 * (1 << 32)
    k, v = rows_like(rng, L, H, D), rows_like(rng, L, H, D)
    table = np.array([[39999, 33333, 39000, 2]], np.int32)
    whole = batch(eng, table, [L], [0, L])
    kv.write(1, whole, k, v)
    got = kv.read(1, whole, L)
    assert np.array_equal(got[0], held(k, "BF16")) and np.array_equal(got[1], held(v, "BF16"))
    assert not kv.read(0, whole, L)[0].any()
    q = rows_like(rng, 1, Hq, D)
    check(kv.attend(1, batch(eng, table, [L]), q), plain(q, held(k, "BF16"), held(v, "BF16"), [L - 1], D ** -0.5), L, D, "F32",
          False)
    kv.free()
    n, ld = 1100, 1 << 21  # rows of 4 MB
    (qr, q), (kr, k), (vr, v) = (cast(rows_like(rng, n, 1, D), "BF16") for _ in range(3))
    kb = eng.alloc(n * ld * 2)
    for r in range(n):
        kb.upload(kr[r], offset=r * ld * 2)
        kb.upload(vr[r], offset=r * ld * 2 + 1024)
    ob, rows = eng.alloc(qr.nbytes), up(eng, np.array([0, n], np.int32))
    eng.attn_prompt_bufs(1, rows, None, n, n, 1, 1, D, up(eng, qr), kb, kb, ob, "BF16", v_off=1024, ldk=ld, ldv=ld)
    check(values(ob, "BF16", (n, 1, D)), plain(q, k, v, np.arange(n), D ** -0.5), n, D, "BF16", True)


def test_two_graphs_of_one_cache(eng):
    """two captured decode calls over one cache (and its workspace) replayed in turn, with an eager call in between"""
    hip = hip_runtime()
    rng = np.random.default_rng(42)
    H, Hq, D = 2, 16, 128
    lens = [6000, 900]
    pool = Pool(rng, lens)
    kv = eng.kv_create(1, pool.pages, H, D, "BF16")
    k, v = rows_like(rng, sum(lens), H, D), rows_like(rng, sum(lens), H, D)
    kv.write(0, batch(eng, pool.table, lens, offsets(lens)), k, v)
    qs = [up(eng, rows_like(rng, 2, Hq, D)) for _ in range(2)]
    outs = [eng.alloc(2 * Hq * D * 4) for _ in range(3)]
    seqs = batch(eng, pool.table, lens)
    want = []
    for q in qs:
        kv.attend_bufs(0, seqs, 2, Hq, q, outs[2])
        want.append(outs[2].download(np.uint32))
    s, graphs = eng.lib.ne_stream(), []
    for q, o in zip(qs, outs):
        g, ex = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(s, 1) == 0
        kv.attend_bufs(0, seqs, 2, Hq, q, o)
        assert hip.hipStreamEndCapture(s, C.byref(g)) == 0
        assert hip.hipGraphInstantiate(C.byref(ex), g, None, None, 0) == 0
        graphs.append((g, ex))
    for i in range(6):
        assert hip.hipGraphLaunch(graphs[i % 2][1], s) == 0
        if i % 3 == 0:
            kv.attend_bufs(0, seqs, 2, Hq, qs[0], outs[2])
        assert hip.hipGraphLaunch(graphs[1 - i % 2][1], s) == 0
        assert hip.hipStreamSynchronize(s) == 0
        for o, w in zip(outs, want):
            assert np.array_equal(o.download(np.uint32), w), i
    for g, ex in graphs:
        hip.hipGraphExecDestroy(ex)
        hip.hipGraphDestroy(g)


def test_captured_drafts(eng):
    """a captured decode of drafts, whose parts a second launch joins: replays follow lengths and rows from long sequences to
    one page, none and back, and leave what no sequence names"""
    hip = hip_runtime()
    rng = np.random.default_rng(43)
    H, Hq, D, R = 2, 16, 128, 8
    full = [9000, 700]
    pool = Pool(rng, full)
    kv = eng.kv_create(1, pool.pages, H, D, "F16")
    k, v = rows_like(rng, sum(full), H, D), rows_like(rng, sum(full), H, D)
    kv.write(0, batch(eng, pool.table, full, offsets(full)), k, v)
    kh, vh = held(k, "F16"), held(v, "F16")
    q = rows_like(rng, R, Hq, D)
    qb, ob = up(eng, q), up(eng, np.full((R, Hq, D), -99, np.float32))
    seqs = batch(eng, pool.table, full, offsets([4, 4]))
    eng.sync()
    s, g, ex = eng.lib.ne_stream(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(s, 1) == 0
    try:
        kv.attend_bufs(0, seqs, R, Hq, qb, ob)
    finally:
        assert hip.hipStreamEndCapture(s, C.byref(g)) == 0
    try:
        assert hip.hipGraphInstantiate(C.byref(ex), g, None, None, 0) == 0
        for lens, new in (([9000, 700], [4, 4]), ([60, 3], [5, 3]), ([0, 700], [0, 8]), ([8999, 1], [7, 1]), ([5000, 0], [1, 0]),
                          ([9000, 700], [4, 4])):
            seqs.lens.upload(np.array(lens, np.int32))
            seqs.rows.upload(offsets(new))
            ob.upload(np.full((R, Hq, D), -99, np.float32))
            assert hip.hipGraphLaunch(ex, s) == 0
            assert hip.hipStreamSynchronize(s) == 0
            got = ob.download(np.float32, (R, Hq, D))
            at = 0
            for b, m in enumerate(new):
                if m:
                    o = b * full[0]
                    last = [lens[b] - m + i for i in range(m)]
                    check(got[at:at + m], plain(q[at:at + m], kh[o:o + lens[b]], vh[o:o + lens[b]], last, D ** -0.5), lens[b], D,
                          "F32", False, (lens, new, b))
                at += m
            assert (got[at:] == -99).all()
            eager = up(eng, np.full((R, Hq, D), -99, np.float32))
            kv.attend_bufs(0, seqs, R, Hq, qb, eager)
            assert np.array_equal(eager.download(np.float32, (R, Hq, D)), got)
    finally:
        if ex.value:
            hip.hipGraphExecDestroy(ex)
        hip.hipGraphDestroy(g)


# ---------------------------------------------------------------------------------------------------- together
def test_block_of_a_model(eng):
    """the trunk's q, k, v in one launch, the cache, decode and the o linear, step by step after a prompt: decode gives what
    the prompt attention of the whole sequence gives, chunk by chunk as well through read"""
    rng = np.random.default_rng(31)
    hid, Hq, H, D = 512, 8, 2, 64
    lins = [eng.exl3_linear(*synth.linear(rng, hid, o, 5)) for o in (Hq * D, H * D, H * D)]
    for m in lins:
        assert m.inp == hid
    back = eng.exl3_linear(*synth.linear(rng, Hq * D, hid, 5))
    n, steps = 90, 5
    x = synth.bf16_values(rng, n + steps, hid)
    qs, ks, vs = [], [], []
    for at in range(0, n + steps, 19):  # (a linear takes up to 32 rows)
        a, b, c = eng.lin_run_multi(lins, [x[at:at + 19]] * 3)
        qs.append(a), ks.append(b), vs.append(c)
    q, k, v = (np.concatenate(t).reshape(n + steps, -1, D) / np.float32(hid ** 0.5) for t in (qs, ks, vs))
    pool = Pool(rng, [n + steps])
    kv = eng.kv_create(1, pool.pages, H, D, "F16")
    # the prompt in two chunks: the second one's keys are the first one's, read back, and its own
    kv.write(0, batch(eng, pool.table, [50], [0, 50]), k[:50], v[:50])
    kv.write(0, batch(eng, pool.table, [n], [0, 40]), k[50:n], v[50:n])
    kc, vc = kv.read(0, batch(eng, pool.table, [n], [0, n]), n)
    assert np.array_equal(kc, held(k[:n], "F16"))
    chunk = eng.attn_prompt(q[50:n], kc, vc, [0, 40], [0, n])
    kh, vh = held(k, "F16"), held(v, "F16")
    whole = plain(q, kh, vh, np.arange(n + steps), D ** -0.5)
    check(chunk, [p[50:n] for p in whole], n, D, "F32", True)
    for t in range(n, n + steps):
        seqs = batch(eng, pool.table, [t + 1])
        kv.write(0, seqs, k[t:t + 1], v[t:t + 1])
        o = kv.attend(0, seqs, q[t:t + 1])
        check(o, [p[t:t + 1] for p in whole], t + 1, D, "F32", False, t)
        y = back.run(o.reshape(1, -1))
        assert y.shape == (1, hid) and np.isfinite(y).all()
    drafts = kv.attend(0, batch(eng, pool.table, [n + steps], [0, steps]), q[n:])  # the same tokens verified together
    check(drafts, [p[n:] for p in whole], n + steps, D, "F32", False)


def test_captured_step(eng):
    """a decode step (write, decode, read, prompt) captured on the library's stream: replays follow the lengths, rows and
    values that the buffers hold then, with the program's own calls in between"""
    hip = hip_runtime()
    rng = np.random.default_rng(32)
    Hq, H, D, n = 8, 2, 128, 3
    lens = [700, 64, 9]
    pool = Pool(rng, [v + 40 for v in lens])
    kv = eng.kv_create(1, pool.pages, H, D, "BF16")
    T = sum(lens)
    k, v = rows_like(rng, T, H, D), rows_like(rng, T, H, D)
    kv.write(0, batch(eng, pool.table, lens, offsets(lens)), k, v)
    at = offsets(lens)
    ks, vs = [held(k[at[b]:at[b + 1]], "BF16") for b in range(n)], [held(v[at[b]:at[b + 1]], "BF16") for b in range(n)]
    e = 4 * D
    kb, vb, qb, ob = eng.alloc(n * H * e), eng.alloc(n * H * e), eng.alloc(n * Hq * e), eng.alloc(n * Hq * e)
    kr, vr, po = eng.alloc(n * H * e), eng.alloc(n * H * e), eng.alloc(n * Hq * e)
    seqs = batch(eng, pool.table, lens)
    one = up(eng, np.array([0, n], np.int32))
    eng.sync()
    s, g, ex = eng.lib.ne_stream(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(s, 1) == 0
    try:
        kv.write_bufs(0, seqs, n, kb, vb)
        kv.attend_bufs(0, seqs, n, Hq, qb, ob)
        kv.read_bufs(0, seqs, n, kr, vr)
        eng.attn_prompt_bufs(1, one, None, n, n, Hq, H, D, qb, kr, vr, po)
    finally:
        assert hip.hipStreamEndCapture(s, C.byref(g)) == 0
    try:
        assert hip.hipGraphInstantiate(C.byref(ex), g, None, None, 0) == 0
        for step in range(4):
            lens = [a + 1 for a in lens]
            seqs.lens.upload(np.array(lens, np.int32))
            q, k1, v1 = rows_like(rng, n, Hq, D), rows_like(rng, n, H, D), rows_like(rng, n, H, D)
            for b, x in ((qb, q), (kb, k1), (vb, v1)):
                b.upload(x)
            for b in range(n):
                ks[b], vs[b] = np.concatenate([ks[b], held(k1[b:b + 1], "BF16")]), np.concatenate([vs[b], held(v1[b:b + 1], "BF16")])
            assert hip.hipGraphLaunch(ex, s) == 0
            assert hip.hipStreamSynchronize(s) == 0
            got = ob.download(np.float32, (n, Hq, D))
            for b in range(n):
                check(got[b:b + 1], plain(q[b:b + 1], ks[b], vs[b], [lens[b]], D ** -0.5), lens[b], D, "F32", False, (step, b))
            assert np.array_equal(kr.download(np.float32, (n, H, D)), held(k1, "BF16"))
            check(po.download(np.float32, (n, Hq, D)), plain(q, held(k1, "BF16"), held(v1, "BF16"), np.arange(n), D ** -0.5), n,
                  D, "F32", True)
            eager = eng.alloc(n * Hq * e)
            kv.attend_bufs(0, seqs, n, Hq, qb, eager)
            assert np.array_equal(eager.download(np.float32, (n, Hq, D)), got)
    finally:
        if ex.value:
            hip.hipGraphExecDestroy(ex)
        hip.hipGraphDestroy(g)
