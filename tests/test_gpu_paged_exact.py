"""Paged attention on data whose scores or sums are exact, so that the tolerance stays that of a few
roundings however long the cache is, and on the shapes that take two query sets per wave.

Tolerance of fp16 and int8 pages, as in test_gpu_paged_kv.py: a probability is rounded to fp16 (2^-11 of
it), scores and sums in fp32 are inside 2^-13 of sum p |v|, the output is rounded once more; a
probability under 2^-14 of the reference is subnormal and off by up to 2^-25 of it."""
from __future__ import annotations

import numpy as np
import pytest

import _serving as sv
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
