"""Append, attention and page copies of the serving cache on the GPU, against float64.

Tolerances.  Append: sum of squares and the norm are a few fp32 roundings, the rotation two products
and a sum: 16 x 2^-24 of the row's largest value, and half a step of the output type.  Int8 rows:
half a quantisation step of the row (and the roundings before it).
Attention over fp16 / int8 pages: a probability is rounded to fp16, 2^-11 of it (2^-25 of the largest
where it is subnormal), scores and sums are fp32 (2^-13 of sum p |v| holds both), and the
output is rounded once more.  Over fp32 pages: scores of hd products and sums over the keys in
fp32, each at most one rounding of 2^-24 per term of a sum of absolute values."""
from __future__ import annotations

import numpy as np
import pytest

import _serving as sv
from moe_mi355x.paged_kv import (PagedKvCache, append_args, attn_args, copy_pages, page_pools)

pytestmark = pytest.mark.gpu

STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11}


def say(msg):
    print(f"[gpu] {msg}", flush=True)


def cache_of(mi355x, ar, b, nkv, hd, dtype, k, ks, v, vs):
    buf = (ar.put(k), ar.put(v), ar.put(ks) if ks is not None else None,
           ar.put(vs) if vs is not None else None)
    return PagedKvCache(mi355x, 1, nkv, hd, b.n_pages, page_size=b.page, dtype=dtype,
                        buffers=[buf]), buf


# ---- append ----------------------------------------------------------------------------------

@pytest.mark.parametrize("nh,nkv,hd,rotary,page,news,lens,xdt,dtype", [
    (4, 2, 64, 16, 16, [1], [1], "float32", "float16"),
    (16, 2, 256, 64, 64, [1, 1, 1], [1, 64, 65], "float32", "float16"),
    (8, 2, 128, 128, 32, [5, 0, 40, 1], [37, 9, 40, 100000], "float32", "float16"),
    (6, 3, 96, 96, 16, [17, 3], [17, 200], "float16", "float16"),
    (4, 1, 24, 24, 128, [130], [131], "float32", "float32"),
    (2, 2, 8, 2, 16, [33], [33], "float32", "float16"),     # a half that is no vector of dims
    (4, 2, 40, 20, 16, [9, 9], [9, 30], "float16", "float32"),
    (4, 4, 64, 0, 64, [3], [70], "float32", "float16"),     # no rotation
    (8, 2, 256, 64, 64, [1, 20], [300, 20], "float32", "int8"),
    (3, 1, 80, 30, 32, [11], [64], "float16", "int8"),
    (4, 2, 64, 32, 16, [600], [1000], "float32", "float16"),  # a block per token
])
def test_append_matches_float64(mi355x, stream, nh, nkv, hd, rotary, page, news, lens, xdt, dtype):
    say(f"append heads={nh}/{nkv} hd={hd} rotary={rotary} page={page} new={news} {xdt}->{dtype}")
    rng = np.random.default_rng(hd + rotary + page)
    b = sv.Batch(rng, news, lens, page, pad=2)
    k0, ks0 = sv.pool_of(rng, b, nkv, hd, dtype, hole=7.0)
    v0, vs0 = sv.pool_of(rng, b, nkv, hd, dtype, hole=7.0)
    x = rng.standard_normal((b.rows, (nh + 2 * nkv) * hd + 4)).astype(sv.DT[xdt])
    qw, kw = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    odt = np.float32 if dtype == "float32" else np.float16
    q0 = np.full((b.rows, nh, hd), 3.0, odt)
    e = x.itemsize
    with sv.Arrays(mi355x, stream) as ar:
        cache, buf = cache_of(mi355x, ar, b, nkv, hd, dtype, k0, ks0, v0, vs0)
        px, pq = ar.put(x), ar.put(q0)
        args = append_args(q=px, k=px + e * nh * hd, v=px + e * (nh + nkv) * hd, q_out=pq,
                           q_norm=ar.put(qw), k_norm=ar.put(kw), n_heads=nh, n_kv_heads=nkv,
                           head_dim=hd, rotary_dim=rotary, rope_theta=10000.0, eps=1e-6, dtype=xdt,
                           ldq=x.shape[1], ldk=x.shape[1], ldv=x.shape[1])
        cache.append(0, b.device(ar), args, stream)
        q, k, v = ar.get(pq, q0), ar.get(buf[0], k0), ar.get(buf[1], v0)
        ks = ar.get(buf[2], ks0) if dtype == "int8" else None
        vs = ar.get(buf[3], vs0) if dtype == "int8" else None
    k64, v64 = sv.values(k0, ks0), sv.values(v0, vs0)
    kg, vg = sv.values(k, ks), sv.values(v, vs)
    fresh = np.zeros((b.n_pages, page), bool)
    tol = 16 * 2.0 ** -24
    for i, m in enumerate(news):
        if not m:
            continue
        r, pos = slice(b.q_start[i], b.q_start[i] + m), b.positions(i)
        xs = x[r].astype(np.float64)
        qx, kx, vx = np.split(xs[:, :(nh + 2 * nkv) * hd], [nh * hd, (nh + nkv) * hd], axis=1)
        want = sv.rotated(qx.reshape(m, nh, hd), qw, pos, rotary, 10000.0, 1e-6)
        top = np.abs(want).max(-1, keepdims=True)
        assert np.all(np.abs(q[r] - want) <= tol * top + STEP[np.dtype(odt).name] * np.abs(want) + 1e-7)
        p, s = b.table[i][pos // page], pos % page
        fresh[p, s] = True
        k64[p, :, s] = sv.rotated(kx.reshape(m, nkv, hd), kw, pos, rotary, 10000.0, 1e-6)
        v64[p, :, s] = vx.reshape(m, nkv, hd)
    for got, want, raw, raw0, sc, sc0 in ((kg, k64, k, k0, ks, ks0), (vg, v64, v, v0, vs, vs0)):
        old = ~fresh[:, None, :, None] & np.ones(raw.shape, bool)
        assert np.array_equal(raw[old], raw0[old])  # nothing else in the pools moved
        if dtype == "int8":
            assert np.array_equal(sc[~fresh[:, None] & np.ones(sc.shape, bool)],
                                  sc0[~fresh[:, None] & np.ones(sc.shape, bool)])
        top = np.abs(want).max(-1, keepdims=True)
        step = np.where(old, 0, (0.5 + 1e-4) * top / 127) if dtype == "int8" else \
            STEP[dtype] * np.abs(want) + 1e-7
        assert np.all(np.abs(got - want) <= tol * top + step)
    assert np.all(q[b.used:] == 3.0)  # rows behind the last sequence


def test_append_without_queries_norms_or_pages(mi355x, stream):
    """Keys and values alone, no norm weights; a page id of -1, one past the pool and a table too
    short for a position: those rows are written nowhere.  A row of zeros in int8: scale 1."""
    rng = np.random.default_rng(5)
    nkv, hd, page = 2, 32, 16
    say("append of keys and values with missing pages")
    for dtype in ("float16", "int8"):
        b = sv.Batch(rng, [20, 20, 2, 3], [20, 36, 2, 2], page, spare=2)  # last: first row before 0
        b.table[1, 1], b.table[2, 0] = -1, b.n_pages
        b.kv_len[0] = 40  # rows 20 .. 39: its table ends at 32 tokens at the latest
        b.lens[0] = 40
        k0, ks0 = sv.pool_of(rng, b, nkv, hd, dtype, hole=7.0)
        x = rng.standard_normal((b.rows, nkv * hd)).astype(np.float32)
        x[1] = 0.0
        with sv.Arrays(mi355x, stream) as ar:
            cache, buf = cache_of(mi355x, ar, b, nkv, hd, dtype, k0, ks0, k0, ks0)
            px = ar.put(x)
            cache.append(0, b.device(ar), append_args(k=px, v=px, n_kv_heads=nkv, head_dim=hd), stream)
            k, v = ar.get(buf[0], k0), ar.get(buf[1], k0)
            ks = ar.get(buf[2], ks0) if dtype == "int8" else None
        want = sv.values(k0, ks0)
        for i, m in enumerate(b.news):
            for n, pos in enumerate(range(int(b.kv_len[i]) - m, int(b.kv_len[i]))):
                pi = pos // page
                if pos < 0 or pi >= b.max_pages or not 0 <= b.table[i, pi] < b.n_pages:
                    continue
                want[b.table[i, pi], :, pos % page] = x[b.q_start[i] + n].reshape(nkv, hd)
        top = np.abs(want).max(-1, keepdims=True)
        tol = 0.51 * top / 127 if dtype == "int8" else 2.0 ** -11 * np.abs(want) + 1e-7
        assert np.all(np.abs(sv.values(k, ks) - want) <= tol) and np.array_equal(k, v)


# ---- attention -------------------------------------------------------------------------------

def check_attention(mi355x, stream, b, nh, nkv, hd, dtype, seed, gate=False, pads=(0, 0, 0),
                    std=1.5, poke=None):
    rng = np.random.default_rng(seed)
    k, ks = sv.pool_of(rng, b, nkv, hd, dtype)
    v, vs = sv.pool_of(rng, b, nkv, hd, dtype)
    xdt = np.float32 if dtype == "float32" else np.float16
    q = (rng.standard_normal((b.rows, nh, hd)) * std).astype(xdt)
    g = rng.standard_normal((b.rows, nh, hd)).astype(np.float32) if gate else None
    if poke:
        poke(k, v, q)
    w = nh * hd
    wide = [np.full((b.rows, w + p), 9.0, d) for p, d in zip(pads, (xdt, xdt, np.float32))]
    wide[0][:, :w] = q.reshape(b.rows, w)
    if gate:
        wide[2][:, :w] = g.reshape(b.rows, w)
    with sv.Arrays(mi355x, stream) as ar:
        cache, _ = cache_of(mi355x, ar, b, nkv, hd, dtype, k, ks, v, vs)
        po = ar.put(wide[1])
        args = attn_args(ar.put(wide[0]), po, n_heads=nh, head_dim=hd, scale=hd ** -0.5,
                         gate=ar.put(wide[2]) if gate else None, ldq=w + pads[0], ldo=w + pads[1],
                         ldg=w + pads[2])
        db = b.device(ar)
        n = cache.attn_workspace_bytes(db, nh)
        work = ar.put(np.full(max(n, 16), 255, np.uint8))  # a used workspace
        cache.attend(0, db, args, stream, (work, n))
        full = ar.get(po, wide[1])
        cache.attend(0, db, args, stream, (work, n))
        assert np.array_equal(full, ar.get(po, wide[1]), equal_nan=True)  # the same every time
    assert np.all(full[:, w:] == 9.0) and np.all(full[b.used:] == 9.0)
    got = full[:b.used, :w].astype(np.float64).reshape(-1, nh, hd)
    kd, vd = sv.values(k, ks), sv.values(v, vs)
    want, mag, big = sv.attention(b, q[:b.used], kd, vd, nkv, hd ** -0.5,
                                  g[:b.used] if gate else None)
    n = max([1, *b.lens])
    if dtype == "float32":
        tol = mag * 2.0 ** -24 * (2 * n ** 0.5 + 8 * hd) + 1e-30
    else:
        tol = mag * (2.0 ** -11 + 2.0 ** -13) + 2.0 ** -11 * np.abs(want) + n * 2.0 ** -25 * big + 1e-7
    return got, want, tol


SHAPES = [  # heads, kv heads, head dim, page, new rows, cached tokens
    (4, 2, 64, 16, [1], [1]),
    (16, 2, 256, 64, [1, 1], [913, 64]),
    (16, 2, 256, 16, [1, 1, 1, 1], [17, 1, 2049, 300]),
    (8, 8, 128, 32, [1, 1], [130, 31]),
    (8, 1, 128, 64, [2, 1, 3], [2, 700, 65]),
    (32, 1, 64, 128, [1, 5], [129, 500]),
    (6, 2, 96, 16, [1, 4, 0, 1], [33, 64, 40, 16]),
    (3, 1, 72, 32, [7, 1], [7, 95]),
    (2, 2, 8, 16, [5], [21]),
    (4, 1, 248, 256, [3, 1], [255, 257]),
    (16, 2, 256, 64, [40, 1, 130], [500, 777, 130]),
    (8, 2, 128, 16, [64, 65, 63], [64, 1000, 127]),
    (4, 4, 32, 64, [300], [301]),
    (12, 4, 96, 32, [33, 200], [400, 200]),
    (16, 2, 256, 128, [257], [2000]),
    (24, 2, 64, 16, [1, 50, 3], [4000, 60, 3]),
]


@pytest.mark.parametrize("dtype", ["float16", "int8", "float32"])
@pytest.mark.parametrize("nh,nkv,hd,page,news,lens", SHAPES)
def test_attention_matches_float64(mi355x, stream, nh, nkv, hd, page, news, lens, dtype):
    if dtype == "int8" and hd % 16:
        hd += 8
    say(f"attention heads={nh}/{nkv} hd={hd} page={page} new={news} cached={lens} {dtype}")
    b = sv.Batch(np.random.default_rng(hd), news, lens, page, pad=3)
    got, want, tol = check_attention(mi355x, stream, b, nh, nkv, hd, dtype, 7 * hd + len(news),
                                     gate=len(news) % 2 == 0)
    bad = np.abs(got - want) > tol
    assert np.all(np.isfinite(got)) and not bad.any(), \
        f"{bad.sum()} off, worst {np.max(np.abs(got - want) / tol):.2f} of the tolerance"


@pytest.mark.parametrize("dtype", ["float16", "int8", "float32"])
def test_rows_that_see_nothing_and_missing_pages(mi355x, stream, dtype):
    """Empty sequences, sequences with no page at all, holes in a table, ids past the pool, more
    rows than cached tokens: zeros where nothing is seen, the rest over what there is."""
    say(f"attention with missing pages, {dtype}")
    b = sv.Batch(np.random.default_rng(2), [1, 1, 4, 0, 20, 6], [40, 100, 100, 0, 150, 3], 16,
                 extra_pages=2)
    b.table[0] = -1
    b.table[1, 2] = -5
    b.table[2, 0], b.table[2, 6] = b.n_pages, 2 ** 31 - 1
    b.table[4, 3:5] = -1
    got, want, tol = check_attention(mi355x, stream, b, 8, 2, 64, dtype, 3, gate=True)
    assert np.all(got[0] == 0.0) and np.all(got[b.q_start[5]:b.q_start[5] + 3] == 0.0)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("dtype", ["float16", "int8", "float32"])
@pytest.mark.parametrize("news,lens", [([1, 1], [300, 45]), ([40, 70], [300, 70])])
def test_strides(mi355x, stream, dtype, news, lens):
    say(f"attention over strided rows, {dtype} {news}")
    b = sv.Batch(np.random.default_rng(4), news, lens, 32, pad=2)
    got, want, tol = check_attention(mi355x, stream, b, 4, 2, 64, dtype, 5, gate=True,
                                     pads=(64, 8, 32))
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("news,lens", [([1, 1], [300, 45]), ([40, 70], [300, 70])])
def test_scores_far_apart(mi355x, stream, dtype, news, lens):
    """Scores over hundreds: one key carries nearly everything, wherever it lies."""
    say(f"attention with large scores, {dtype} {news}")
    b = sv.Batch(np.random.default_rng(6), news, lens, 16)
    got, want, tol = check_attention(mi355x, stream, b, 4, 2, 64, dtype, 8, std=60.0)
    # a score of size S is off by S 2^-24 times the terms of its sum, and its probability by as much
    assert np.all(np.abs(got - want) <= tol + 64 * 300 * 2.0 ** -24 * 2)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_keys_that_a_row_may_not_see_do_not_reach_it(mi355x, stream, dtype):
    """NaN and infinities in the newest token's key and value: only that token's row has them."""
    say(f"attention with a poisoned newest token, {dtype}")
    b = sv.Batch(np.random.default_rng(9), [20, 1, 90], [50, 33, 90], 16)

    def poke(k, v, q):
        for i, (x, y) in enumerate([(np.nan, np.inf), (0.0, 0.0), (np.inf, np.nan)]):
            if x or y:
                p = b.lens[i] - 1
                k[b.table[i, p // 16], :, p % 16] = x
                v[b.table[i, p // 16], :, p % 16] = y

    got, want, tol = check_attention(mi355x, stream, b, 4, 2, 64, dtype, 11, poke=poke)
    last = np.zeros(b.used, bool)
    last[[b.q_start[1] - 1, b.q_start[3] - 1]] = True
    assert np.all(np.isnan(got[last]).any(axis=(1, 2)))
    ok = np.abs(got - want) <= tol
    assert np.all(ok[~last])


# ---- copies ----------------------------------------------------------------------------------

@pytest.mark.parametrize("pools,page_bytes,copies", [
    (1, 16, 1), (3, 1040, 5), (2, 65536, 7), (70, 512, 3), (1, 16384 * 3 + 48, 40), (5, 16, 300)])
def test_page_copies(mi355x, stream, pools, page_bytes, copies):
    say(f"page copies: {pools} pools, {copies} pages of {page_bytes}")
    rng = np.random.default_rng(pools)
    n = 2 * copies + 3
    data = rng.integers(0, 256, (pools, n, page_bytes), dtype=np.uint8)
    ids = rng.permutation(n).astype(np.int32)
    src, dst = ids[:copies].copy(), ids[copies:2 * copies].copy()
    src[0] = src[-1]  # a page may be a source twice
    with sv.Arrays(mi355x, stream) as ar:
        base = ar.put(data)
        want = data.copy()
        want[:, dst] = data[:, src]
        p = page_pools((base + i * n * page_bytes, page_bytes, n) for i in range(pools))
        copy_pages(p, ar.put(src), ar.put(dst), copies, stream)
        assert np.array_equal(ar.get(base, data), want)
        # pairs with an id that is no page are left out
        bad = np.array([-1, n, 2, 5, 1], np.int32)
        to = np.array([0, 1, -7, n, 4], np.int32)
        copy_pages(p, ar.put(bad), ar.put(to), 5, stream)
        want[:, 4] = want[:, 1]
        assert np.array_equal(ar.get(base, data), want)


# ---- together --------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float16", "float32", "int8"])
def test_a_server_of_forking_sequences(mi355x, stream, dtype):
    """Prompts, decode steps, a fork in the middle of a page, a freed sequence and a compaction:
    every step's attention over the cache is that over all the keys and values a sequence was
    given so far."""
    say(f"cache life, {dtype}")
    rng = np.random.default_rng(12)
    nh, nkv, hd, page, rotary = 4, 2, 64, 16, 32
    xdt = np.float32 if dtype == "float32" else np.float16
    cache = PagedKvCache(mi355x, 2, nkv, hd, 24, page_size=page, dtype=dtype)
    seen: dict[int, list[tuple[np.ndarray, np.ndarray]]] = {}
    qw, kw = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)

    def step(growth):
        with sv.Arrays(mi355x, stream) as ar:
            db = cache.batch(growth, stream)
            rows = sum(n for _, n in growth)
            x = rng.standard_normal((2, rows, (nh + 2 * nkv) * hd)).astype(np.float32)
            px, pw, pk = ar.put(x), ar.put(qw), ar.put(kw)
            outs = []
            for layer in range(2):
                q0 = np.zeros((rows, nh, hd), xdt)
                pq, po = ar.put(q0), ar.put(q0)
                at = px + layer * x[0].nbytes
                cache.append(layer, db, append_args(
                    q=at, k=at + 4 * nh * hd, v=at + 4 * (nh + nkv) * hd, q_out=pq, q_norm=pw,
                    k_norm=pk, n_heads=nh, n_kv_heads=nkv, head_dim=hd, rotary_dim=rotary,
                    ldq=x.shape[2], ldk=x.shape[2], ldv=x.shape[2]), stream)
                cache.reserve_attn(db, nh)
                cache.attend(layer, db, attn_args(pq, po, n_heads=nh, head_dim=hd), stream)
                outs.append((ar.get(pq, q0), ar.get(po, q0)))
        r = 0
        for s, n in growth:
            pos = np.arange(cache.tables.length(s) - n, cache.tables.length(s))
            for layer in range(2):
                _, kx, vx = np.split(x[layer, r:r + n], [nh * hd, (nh + nkv) * hd], axis=1)
                kr = sv.rotated(kx.reshape(n, nkv, hd), kw, pos, rotary, 10000.0, 1e-6)
                seen[s][layer][0].extend(kr)
                seen[s][layer][1].extend(vx.reshape(n, nkv, hd))
                k, v = (np.array(a) for a in seen[s][layer])
                assert len(k) == cache.tables.length(s)
                q, o = (a[r:r + n].astype(np.float64) for a in outs[layer])
                for h in range(nh):
                    sc = q[:, h] @ k[:, h // 2].T * hd ** -0.5
                    sc = np.where(np.arange(len(k))[None] <= pos[:, None], sc, -np.inf)
                    p = np.exp(sc - sc.max(1, keepdims=True))
                    want = p @ v[:, h // 2] / p.sum(1, keepdims=True)
                    # keys and values rounded to the cache's type: the scores are off by step |q||k|
                    step_ = {"float32": 2.0 ** -20, "float16": 2.0 ** -11, "int8": 1 / 127}[dtype]
                    off = np.linalg.norm(q[:, h], axis=1).max() * np.linalg.norm(k[:, h // 2], axis=1).max()
                    tol = (step_ * (2 * off * hd ** -0.5 + 4)) * np.abs(v).max()
                    assert np.max(np.abs(o[:, h] - want)) <= tol
            r += n

    try:
        def new(parent=None):
            s = cache.fork(parent) if parent is not None else cache.add()
            seen[s] = [tuple(list(a) for a in seen[parent][i]) if parent is not None else ([], [])
                       for i in range(2)]
            return s

        a, b = new(), new()
        step([(a, 21), (b, 40)])
        step([(a, 1), (b, 1)])
        c = new(a)                  # shares a page that is part filled
        step([(a, 1), (c, 2), (b, 1)])
        d = new(c)
        step([(d, 17), (c, 1), (a, 13)])
        cache.free(b)
        cache.compact(stream)
        step([(a, 1), (c, 1), (d, 1)])
        e = new()
        step([(e, 50), (a, 1), (d, 1)])
        assert cache.tables.free_pages > 0
    finally:
        cache.close()


# ---- many sequences --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float16", "int8", "float32"])
@pytest.mark.parametrize("n,longest", [(100, 900), (4200, 20)])
def test_more_sequences_than_a_wave_looks_at(mi355x, stream, n, longest, dtype):
    """The sequence of a row and the ranges of keys are found 64 sequences at a time."""
    say(f"attention over {n} sequences, {dtype}")
    rng = np.random.default_rng(n)
    news = [int(v) for v in rng.choice([0, 1, 1, 1, 2], n)]
    lens = [int(m + v) for m, v in zip(news, rng.integers(0, longest, n))]
    lens[n // 2] = 3 * longest
    b = sv.Batch(rng, news, lens, 16, pad=5)
    got, want, tol = check_attention(mi355x, stream, b, 2, 1, 32, dtype, 3)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_append_of_more_sequences_than_a_wave_looks_at(mi355x, stream, dtype):
    n, nkv, hd, page = 4200, 1, 16, 16
    say(f"append to {n} sequences, {dtype}")
    rng = np.random.default_rng(3)
    news = [int(v) for v in rng.choice([0, 1, 1, 2], n)]
    lens = [int(m + v) for m, v in zip(news, rng.integers(0, 20, n))]
    b = sv.Batch(rng, news, lens, page, pad=3)
    k0 = np.zeros((b.n_pages, nkv, page, hd), sv.DT[dtype])
    x = rng.standard_normal((b.rows, nkv * hd)).astype(sv.DT[dtype])
    with sv.Arrays(mi355x, stream) as ar:
        cache, buf = cache_of(mi355x, ar, b, nkv, hd, dtype, k0, None, k0, None)
        px = ar.put(x)
        cache.append(0, b.device(ar), append_args(k=px, v=px, n_kv_heads=nkv, head_dim=hd, dtype=dtype),
                     stream)
        k = ar.get(buf[0], k0)
    want = k0.copy()
    for i, m in enumerate(news):
        pos = b.positions(i)
        want[b.table[i, pos // page], 0, pos % page] = x[b.q_start[i]:b.q_start[i] + m]
    assert np.array_equal(k, want)


@pytest.mark.parametrize("dtype", ["float16", "int8", "float32"])
@pytest.mark.parametrize("news,lens", [([1], [30000]), ([1, 1], [9000, 20000]), ([2, 1, 70], [4097, 8193, 4200])])
def test_long_caches(mi355x, stream, news, lens, dtype):
    """More ranges of keys per row than a wave has lanes, and ranges of the largest size."""
    say(f"attention over long caches {lens}, {dtype}")
    b = sv.Batch(np.random.default_rng(1), news, lens, 64)
    got, want, tol = check_attention(mi355x, stream, b, 4, 1, 64, dtype, 2)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("news", [[100], [1]])
def test_pages_behind_four_gigabytes(mi355x, stream, dtype, news):
    """Pages at the end of a pool of more than 2^32 bytes: written by append, copied, attended to."""
    nh, nkv, hd, page = 4, 2, 128, 64
    esz = np.dtype(sv.DT[dtype]).itemsize
    n_pages = (5 << 30) // (nkv * page * hd * esz)
    say(f"attention over the last of {n_pages} pages, {dtype} {news}")
    rng = np.random.default_rng(6)
    b = sv.Batch(rng, news, [100], page, spare=0)
    x = rng.standard_normal((100, nkv * hd)).astype(sv.DT[dtype])
    q = rng.standard_normal((news[0], nh, hd)).astype(sv.DT[dtype])
    pool = np.zeros((b.n_pages, nkv, page, hd), sv.DT[dtype])
    at = np.arange(100)
    pool[b.table[0, at // page], :, at % page] = x.reshape(100, nkv, hd)
    want, mag, big = sv.attention(b, q, pool.astype(np.float64), pool.astype(np.float64), nkv, hd ** -0.5)
    far = n_pages - 2 * b.n_pages  # append there, copy behind, attend to the copies
    bufs = [mi355x.alloc_device(n_pages * nkv * page * hd * esz) for _ in range(2)]
    try:
        with sv.Arrays(mi355x, stream) as ar:
            cache = PagedKvCache(mi355x, 1, nkv, hd, n_pages, page_size=page, dtype=dtype,
                                 buffers=[(int(bufs[0].handle), int(bufs[1].handle), None, None)])
            fill = sv.Batch(rng, [100], [100], page, spare=0)
            fill.table = b.table + far
            px, pq, o = ar.put(x), ar.put(q), np.zeros_like(q)
            po = ar.put(o)
            cache.append(0, fill.device(ar), append_args(k=px, v=px, n_kv_heads=nkv, head_dim=hd, dtype=dtype),
                         stream)
            src = np.arange(far, far + b.n_pages, dtype=np.int32)
            copy_pages(cache.pools, ar.put(src), ar.put(src + b.n_pages), len(src), stream)
            b.table = b.table + far + b.n_pages
            db = b.device(ar)
            cache.reserve_attn(db, nh)
            cache.attend(0, db, attn_args(pq, po, n_heads=nh, head_dim=hd), stream)
            got = ar.get(po, o).astype(np.float64)
            cache.close()
    finally:
        mi355x.synchronize_stream(stream)
        for buf in bufs:
            mi355x.free_device(buf)
    if dtype == "float32":
        tol = mag * 2.0 ** -24 * (2 * 10 + 8 * hd) + 1e-30
    else:
        tol = mag * (2.0 ** -11 + 2.0 ** -13) + 2.0 ** -11 * np.abs(want) + 100 * 2.0 ** -25 * big + 1e-7
    assert np.all(np.abs(got - want) <= tol)
