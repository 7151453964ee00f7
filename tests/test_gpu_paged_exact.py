"""Paged attention on data whose scores or sums are exact, so that the tolerance stays that of a few
roundings however long the cache is, and on the shapes that take two query sets per wave.

Tolerance of fp16 and int8 pages, as in test_gpu_paged_kv.py: a probability is rounded to fp16 (2^-11 of
it), scores and sums in fp32 are inside 2^-13 of sum p |v|, the output is rounded once more; a
probability under 2^-14 of the reference is subnormal and off by up to 2^-25 of it."""
from __future__ import annotations

import numpy as np
import pytest

import _serving as sv
from test_gpu_paged_kv import check_attention
from moe_mi355x.paged_kv import PagedKvCache, append_args, attn_args

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[gpu] {msg}", flush=True)


def attend(mi355x, stream, b, q, k, v, ks=None, vs=None, scale=1.0):
    """Outputs [rows, heads, dims] of the call on pools k, v (int8: with scales ks, vs), in float64;
    rows behind the last sequence stay as they were."""
    dtype = np.dtype(k.dtype).name
    nkv, hd = k.shape[1], k.shape[3]
    o = np.full(q.shape, 9.0, q.dtype)
    with sv.Arrays(mi355x, stream) as ar:
        bufs = (ar.put(k), ar.put(v), *(ar.put(s) if s is not None else None for s in (ks, vs)))
        cache = PagedKvCache(mi355x, 1, nkv, hd, b.n_pages, page_size=b.page, dtype=dtype,
                             buffers=[bufs])
        po, db = ar.put(o), b.device(ar)
        n = cache.attn_workspace_bytes(db, q.shape[1])
        work = ar.put(np.full(max(n, 16), 255, np.uint8))
        cache.attend(0, db, attn_args(ar.put(q), po, n_heads=q.shape[1], head_dim=hd, scale=scale),
                     stream, (work, n))
        got = ar.get(po, o)
    assert np.all(got[b.used:] == 9.0)
    return got[:b.used].astype(np.float64)


def rounded(want, mag, big, n):
    return mag * (2.0 ** -11 + 2.0 ** -13) + 2.0 ** -11 * np.abs(want) + n * 2.0 ** -25 * big + 1e-7


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("news,lens", [([1, 1], [600, 70]), ([3], [300]), ([40], [500])])
def test_int8_scores_keep_their_digits_under_a_common_offset(mi355x, stream, hd, news, lens):
    """Queries around 200 in all dims, keys that differ by a few units.  Products and partial sums are
    whole numbers under 2^24 (hd 250 121 < 2^23), so fp32 holds every score exactly, however the sum
    is ordered."""
    say(f"int8 attention, queries with a common offset, hd={hd} {news}")
    nh, nkv = 4, 2
    rng = np.random.default_rng(hd + len(news))
    b = sv.Batch(rng, news, lens, 16, pad=2)
    q = np.repeat(rng.integers(150, 251, (b.rows, nh, hd // 2)), 2, axis=-1).astype(np.float16)
    base = np.repeat(rng.integers(-120, 121, (nkv, 1, hd // 2)), 2, axis=-1)
    base[..., 1::2] *= -1  # pairs that cancel: the scores come from the differences
    k = np.broadcast_to(base, (b.n_pages, nkv, b.page, hd)).astype(np.int8)
    at = rng.integers(0, hd, (4, *k.shape[:3]))
    for i in range(4):
        np.put_along_axis(k, at[i][..., None],
                          np.take_along_axis(k, at[i][..., None], -1) + np.int8(1 - 2 * (i % 2)), -1)
    k = np.clip(k, -121, 121)
    v = rng.integers(-127, 128, k.shape).astype(np.int8)
    ks = np.full(k.shape[:3], 0.05, np.float32)
    vs = rng.uniform(0.005, 0.02, k.shape[:3]).astype(np.float32)
    got = attend(mi355x, stream, b, q, k, v, ks, vs)
    want, mag, big = sv.attention(b, q[:b.used], sv.values(k, ks), sv.values(v, vs), nkv, 1.0)
    assert np.all(np.abs(got - want) <= rounded(want, mag, big, max(lens)))


@pytest.mark.parametrize("news,lens", [([7, 3], [40, 20]), ([40, 9], [100, 9])])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_int8_rows_that_are_not_finite_read_as_nan(mi355x, stream, news, lens, what):
    """A key and a value with one element that is no number, appended to int8 pages: their rows get a
    NaN scale, the tokens that see them are NaN, and all others are as if they were not there."""
    say(f"int8 append and attention with {what}, {news}")
    nh, nkv, hd, page = 4, 2, 64, 16
    rng = np.random.default_rng(21)
    b = sv.Batch(rng, news, lens, page, pad=1)
    k0, ks0 = sv.pool_of(rng, b, nkv, hd, "int8", hole=0.02)
    x = rng.standard_normal((2, b.rows, nkv, hd)).astype(np.float32)
    x[0, news[0] - 2, 0, 5] = what              # a key of the first sequence, head 0
    x[1, news[0] + news[1] - 1, 1, hd - 1] = what  # a value of the second, head 1
    q = (rng.standard_normal((b.rows, nh, hd)) * 1.5).astype(np.float16)
    with sv.Arrays(mi355x, stream) as ar:
        bufs = tuple(ar.put(a) for a in (k0, k0, ks0, ks0))
        cache = PagedKvCache(mi355x, 1, nkv, hd, b.n_pages, page_size=page, dtype="int8",
                             buffers=[bufs])
        cache.append(0, b.device(ar), append_args(k=ar.put(x[0]), v=ar.put(x[1]), n_kv_heads=nkv,
                                                  head_dim=hd), stream)
        k, v, ks, vs = (ar.get(p, a) for p, a in zip(bufs, (k0, k0, ks0, ks0)))
    bad = np.zeros((2, b.n_pages, nkv, page), bool)
    for i, seq, pos, h in ((0, 0, lens[0] - 2, 0), (1, 1, lens[1] - 1, 1)):
        bad[i, b.table[seq, pos // page], h, pos % page] = True
    assert np.array_equal(np.isnan(np.stack([ks, vs])), bad)
    assert np.all(np.isfinite(np.stack([ks, vs])[~bad]))
    got = attend(mi355x, stream, b, q, k, v, ks, vs, hd ** -0.5)
    want, mag, big = sv.attention(b, q[:b.used], sv.values(k, ks), sv.values(v, vs), nkv, hd ** -0.5)
    gone = np.zeros(got.shape, bool)
    gone[news[0] - 2:news[0], :2] = True
    gone[b.used - 1, 2:] = True
    assert np.all(np.isnan(got[gone])) and np.all(np.isfinite(got[~gone]))
    ok = np.abs(got - want) <= rounded(want, mag, big, max(lens))
    assert np.all(ok[~gone])


# ---- chunks of many rows: two query sets per wave --------------------------------------------

def takes_two_sets(b, nh, nkv):
    """The rule of the launch: more than 16 rows of a head, 160 tiles of 64 rows or more."""
    group = nh // nkv
    return b.max_q * group > 16 and (b.rows * group // 64 + len(b.news)) * nkv >= 160


TWO_SETS = [("float16", hd) for hd in (24, 32, 48, 64, 96, 128, 200, 256)] + \
    [("int8", hd) for hd in (32, 48, 64, 112, 128)]


@pytest.mark.parametrize("dtype,hd", TWO_SETS)
@pytest.mark.parametrize("nh,nkv,news,lens,page", [
    (32, 16, [150, 1, 97, 0, 64], [300, 200, 97, 5, 513], 16),
    (24, 8, [450], [2000], 64),
])
def test_chunks_of_many_rows(mi355x, stream, dtype, hd, nh, nkv, news, lens, page):
    b = sv.Batch(np.random.default_rng(hd), news, lens, page, pad=3)
    assert takes_two_sets(b, nh, nkv)
    say(f"attention, two query sets, hd={hd} {dtype} new={news}")
    got, want, tol = check_attention(mi355x, stream, b, nh, nkv, hd, dtype, hd, gate=len(news) == 1)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("dtype", ["float16", "int8"])
def test_chunks_of_many_rows_with_missing_pages_and_strides(mi355x, stream, dtype):
    say(f"attention, two query sets, missing pages, {dtype}")
    b = sv.Batch(np.random.default_rng(2), [70, 90, 1, 0, 200, 6], [140, 100, 100, 0, 450, 3], 16,
                 extra_pages=2)
    b.table[0] = -1
    b.table[1, 2] = -5
    b.table[2, 0], b.table[2, 6] = b.n_pages, 2 ** 31 - 1
    b.table[4, 3:5] = -1
    assert takes_two_sets(b, 32, 16)
    got, want, tol = check_attention(mi355x, stream, b, 32, 16, 64, dtype, 3, gate=True,
                                     pads=(64, 8, 32))
    assert np.all(got[:70] == 0.0) and np.all(got[b.q_start[5]:b.q_start[5] + 3] == 0.0)
    assert np.all(np.abs(got - want) <= tol)


def poison(b, seqs, page):
    """NaN and infinities into the newest token's key and value of some sequences."""
    def poke(k, v, q):
        for n, i in enumerate(seqs):
            p = b.lens[i] - 1
            at = (b.table[i, p // page], slice(None), p % page)
            k[at], v[at] = [(np.nan, np.inf), (0.0, np.nan), (np.inf, -np.inf)][n % 3]
    return poke


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("nh,nkv,hd,news,lens", [
    (32, 16, 64, [150, 97, 1, 64], [300, 97, 40, 513]),       # two query sets
    (16, 16, 256, [400, 300], [500, 300]),
    (4, 2, 64, [3, 1, 4, 1], [50, 33, 200, 20]),              # up to 16 rows of a head, a block an item
    (4, 2, 256, [3, 1, 8], [50, 33, 700]),
    (2, 2, 32, [1, 3, 2] * 50, [33, 50, 200] * 50),           # ... and blocks of several items
])
def test_a_poisoned_newest_token_stays_with_its_row(mi355x, stream, dtype, nh, nkv, hd, news, lens):
    say(f"attention with poisoned newest tokens, hd={hd} {dtype} {len(news)} sequences")
    b = sv.Batch(np.random.default_rng(9), news, lens, 16)
    seqs = [i for i, m in enumerate(news) if m > 1]
    got, want, tol = check_attention(mi355x, stream, b, nh, nkv, hd, dtype, 11, poke=poison(b, seqs, 16))
    last = np.zeros(b.used, bool)
    last[[b.q_start[i + 1] - 1 for i in seqs]] = True
    assert not np.any(np.isfinite(got[last]))
    assert np.all((np.abs(got - want) <= tol)[~last])


@pytest.mark.parametrize("dtype", ["float16", "int8", "float32"])
@pytest.mark.parametrize("nh,nkv,n", [(2, 1, 70), (4, 2, 100), (4, 2, 200)])
def test_chunks_of_more_sequences_than_a_wave_looks_at(mi355x, stream, dtype, nh, nkv, n):
    """70 sequences with one query set per wave, 100 and 200 with two."""
    rng = np.random.default_rng(n)
    news = [int(v) for v in rng.choice([0, 1, 2, 5, 17, 40], n)]
    lens = [int(m + v) for m, v in zip(news, rng.integers(0, 300, n))]
    lens[n // 2] = news[n // 2] + 1500
    b = sv.Batch(rng, news, lens, 16, pad=5)
    assert takes_two_sets(b, nh, nkv) == (n >= 100) and b.max_q * nh // nkv > 16
    say(f"attention of chunks of {n} sequences, {dtype}")
    got, want, tol = check_attention(mi355x, stream, b, nh, nkv, 64, dtype, 3)
    assert np.all(np.abs(got - want) <= tol)


# ---- every range of keys exactly once --------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float16", "int8", "float32"])
@pytest.mark.parametrize("nh,nkv,news,lens", [
    (4, 1, [1], [30000]), (4, 1, [1, 1], [9000, 20000]), (4, 1, [2, 1, 70], [4097, 8193, 4200]),
    (16, 2, [1], [913]), (8, 2, [1] * 90, [40 * i + 1 for i in range(90)]),
    (16, 16, [640], [5000]), (32, 16, [1, 300, 40], [12000, 900, 6001]),
])
def test_every_key_counts_once(mi355x, stream, nh, nkv, news, lens, dtype):
    """Queries of zero weigh all keys alike, and the keys' values are one-hot by blocks of 64
    tokens: an output is the share of the row's keys that lie in the dim's blocks.  Probabilities of 1 and
    sums of them are exact; what is left is the rounding of 1 / sum, of the product and of the
    output: 2^-20 of it with some room, and half a step of the type (2^-25 where subnormal)."""
    say(f"one-hot values, heads={nh}/{nkv} new={news[:3]} cached={lens[:3]} {dtype}")
    hd, page = 64, 32
    rng = np.random.default_rng(5)
    b = sv.Batch(rng, news, lens, page, pad=1)
    k, ks = sv.pool_of(rng, b, nkv, hd, dtype)
    v = np.zeros(k.shape, k.dtype)
    for i in range(len(news)):
        pg, row, ok = b.slots(i, b.n_pages)
        j = np.arange(lens[i])[ok]
        v[pg[ok], :, row[ok], j // 64 % hd] = 1
    vs = np.ones(k.shape[:3], np.float32) if dtype == "int8" else None
    q = np.zeros((b.rows, nh, hd), np.float32 if dtype == "float32" else np.float16)
    got = attend(mi355x, stream, b, q, k, v, ks, vs, hd ** -0.5)
    want = np.zeros((b.used, hd))
    for i in range(len(news)):
        for r, pos in zip(range(b.q_start[i], b.q_start[i + 1]), b.positions(i)):
            want[r] = np.bincount(np.arange(pos + 1) // 64 % hd, minlength=hd) / (pos + 1)
    half = 0 if dtype == "float32" else 2.0 ** -11
    tol = want * (half + 2.0 ** -20) + (0 if dtype == "float32" else 2.0 ** -25)
    assert np.all(np.abs(got - want[:, None]) <= tol[:, None])


@pytest.mark.parametrize("dtype", ["float16", "int8", "float32"])
@pytest.mark.parametrize("nh,nkv,news,lens", [
    (4, 1, [1], [30000]), (4, 1, [2, 1, 70], [4097, 8193, 4200]), (16, 2, [1], [913]),
    (8, 2, [1] * 90, [40 * i + 1 for i in range(90)]), (16, 16, [640], [5000]),
])
def test_ranges_are_joined_by_their_weights(mi355x, stream, nh, nkv, news, lens, dtype):
    """As above with a score for every block of 64 tokens, an eighth's multiple in [-3, 3] that the types hold
    exactly, so that every range of keys has a reference of its own.  Scores are exact up to two fp32
    roundings; probabilities, 2^-8.7 of the reference or more, are rounded once to fp16; the positive
    sums are off by at most 2^-24 for each term; the output is rounded once."""
    say(f"one-hot values, scores by block, heads={nh}/{nkv} cached={lens[:3]} {dtype}")
    hd, page = 64, 32
    rng = np.random.default_rng(6)
    b = sv.Batch(rng, news, lens, page, pad=1)
    k = np.zeros((b.n_pages, nkv, page, hd), sv.DT[dtype])
    v = np.zeros_like(k)
    score = rng.integers(-24, 25, (len(news), max(lens) // 64 + 1))
    for i in range(len(news)):
        pg, row, ok = b.slots(i, b.n_pages)
        j = np.arange(lens[i])[ok]
        v[pg[ok], :, row[ok], j // 64 % hd] = 1
        s = score[i, j // 64][:, None] * (1 if dtype == "int8" else 0.125)
        k[pg[ok], :, row[ok], 7] = s.astype(k.dtype)
    ks = np.full(k.shape[:3], 0.125, np.float32) if dtype == "int8" else None
    vs = np.ones(k.shape[:3], np.float32) if dtype == "int8" else None
    q = np.zeros((b.rows, nh, hd), np.float32 if dtype == "float32" else np.float16)
    q[..., 7] = 1
    got = attend(mi355x, stream, b, q, k, v, ks, vs, 1.0)
    want = np.zeros((b.used, hd))
    for i in range(len(news)):
        for r, pos in zip(range(b.q_start[i], b.q_start[i + 1]), b.positions(i)):
            j = np.arange(pos + 1) // 64
            w = np.exp(score[i, j] / 8)
            want[r] = np.bincount(j % hd, w, minlength=hd) / w.sum()
    half = 0 if dtype == "float32" else 2.0 ** -11
    tol = want * (3 * half + 2 * max(lens) * 2.0 ** -24 + 2.0 ** -18) + (0 if dtype == "float32" else 2.0 ** -25)
    assert np.all(np.abs(got - want[:, None]) <= tol[:, None])


# ---- append ----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float16", "int8"])
@pytest.mark.parametrize("rotary,off", [(32, 0), (30, 0), (32, 2)])
def test_append_with_fp16_norm_weights(mi355x, stream, dtype, rotary, off):
    """Norm weights in fp16, also 2 bytes off a vector's boundary, give what their fp32 copies give,
    bit by bit: the weights are widened before use."""
    say(f"append with fp16 norm weights, {dtype} rotary={rotary} {off} bytes off")
    nh, nkv, hd, page = 4, 2, 64, 16
    rng = np.random.default_rng(rotary)
    b = sv.Batch(rng, [5, 1], [30, 17], page, pad=1)
    k0, ks0 = sv.pool_of(rng, b, nkv, hd, dtype, hole=7.0)
    x = rng.standard_normal((b.rows, (nh + 2 * nkv) * hd)).astype(np.float32)
    w16 = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float16)
    q0 = np.full((b.rows, nh, hd), 3.0, np.float16)
    got = []
    with sv.Arrays(mi355x, stream) as ar:
        px, db = ar.put(x), b.device(ar)
        for w, name in ((w16, "float16"), (w16.astype(np.float32), "float32")):
            shift = np.zeros(off // 2, w.dtype)
            pw = [ar.put(np.concatenate([shift, r])) + shift.nbytes for r in w]
            bufs = tuple(ar.put(a) if a is not None else None for a in (k0, k0, ks0, ks0))
            cache = PagedKvCache(mi355x, 1, nkv, hd, b.n_pages, page_size=page, dtype=dtype,
                                 buffers=[bufs])
            pq = ar.put(q0)
            cache.append(0, db, append_args(
                q=px, k=px + 4 * nh * hd, v=px + 4 * (nh + nkv) * hd, q_out=pq, q_norm=pw[0],
                k_norm=pw[1], n_heads=nh, n_kv_heads=nkv, head_dim=hd, rotary_dim=rotary,
                param_dtype=name, ldq=x.shape[1], ldk=x.shape[1], ldv=x.shape[1]), stream)
            got.append([ar.get(pq, q0)] + [ar.get(p, a) for p, a in zip(bufs, (k0, k0, ks0, ks0)) if p])
    assert not np.array_equal(got[0][0], q0)
    for a, c in zip(*got):
        assert np.array_equal(a, c)
