"""The gated delta rule on the GPU against float64, token by token.

Tolerances: a state or an output is a sum of products over the head dim, formed in fp32 (2^-24 of the
sum of absolute values per rounding, head_dim roundings at most), and the delta rule with beta in
(0, 1) and unit keys does not grow a state: normwise (2 dk + 64) x 2^-24 for a few chunks'
chain.  Fp16 outputs are rounded once more (2^-11 normwise)."""
from __future__ import annotations

import numpy as np
import pytest

import _serving as sv
from moe_mi355x.delta_rule import GatedDeltaRunner, delta_args

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[gpu] {msg}", flush=True)


def make(rng, news, nk, nv, dk, dv, dtype, pad=0, decay=0.3, norm=True):
    rows = sum(news) + pad
    dt = sv.DT[dtype]
    q, k, v = (rng.standard_normal((rows, h, d)) for h, d in ((nk, dk), (nk, dk), (nv, dv)))
    q, k, v = (a / (1 + np.exp(-a)) for a in (q, k, v))  # as behind the short convolution
    if not norm:
        q, k = (a / np.sqrt((a * a).sum(-1, keepdims=True) + 1e-6) for a in (q, k))
    g = (-np.abs(rng.standard_normal((rows, nv))) * decay).astype(np.float32)
    beta = (1 / (1 + np.exp(-rng.standard_normal((rows, nv))))).astype(np.float32)
    return q.astype(dt), k.astype(dt), v.astype(dt), g, beta


def run(mi355x, stream, x, news, nk, nv, dk, dv, dtype, state, slot_in, slot_out, norm=True,
        pads=(0, 0, 0, 0), max_q=None, scale=None):
    q, k, v, g, beta = x
    rows = len(g)

    def wide(a, p, fill=5.0):
        w = np.full((rows, a.shape[1] * a.shape[2] + p), fill, a.dtype)
        w[:, :a.shape[1] * a.shape[2]] = a.reshape(rows, -1)
        return w

    start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    o0 = wide(np.full((rows, nv, dv), 5.0, sv.DT[dtype]), pads[3])
    with sv.Arrays(mi355x, stream) as ar:
        po, ps = ar.put(o0), ar.put(state)
        args = delta_args(q=ar.put(wide(q, pads[0])), k=ar.put(wide(k, pads[1])),
                          v=ar.put(wide(v, pads[2])), g=ar.put(g), beta=ar.put(beta), o=po,
                          state=ps, slot_in=ar.put(np.array(slot_in, np.int32)),
                          slot_out=ar.put(np.array(slot_out, np.int32)), q_start=ar.put(start),
                          n_slots=len(state), n_seqs=len(news), rows=rows,
                          max_q=max_q or max([1, *news]), n_k_heads=nk, n_v_heads=nv, head_dim_k=dk,
                          head_dim_v=dv, dtype=dtype, qk_norm=norm, scale=scale,
                          ldq=nk * dk + pads[0], ldk=nk * dk + pads[1], ldv=nv * dv + pads[2],
                          ldo=nv * dv + pads[3])
        runner = GatedDeltaRunner(mi355x)
        runner.reserve(args)
        try:
            runner.forward_device(args, stream)
            o, s = ar.get(po, o0), ar.get(ps, state)
        finally:
            mi355x.synchronize_stream(stream)
            runner.close()
    assert np.all(o[:, nv * dv:] == 5.0) and np.all(o[start[-1]:] == 5.0)
    return o[:, :nv * dv].reshape(rows, nv, dv), s


def want_of(x, news, nk, nv, dk, dv, state, slot_in, slot_out, scale, norm=True):
    q, k, v, g, beta = x
    o = np.zeros((sum(news), nv, dv))
    s = state.astype(np.float64)
    r = 0
    for b, n in enumerate(news):
        for h in range(nv):
            first = state[slot_in[b], h] if 0 <= slot_in[b] < len(state) else np.zeros((dk, dv))
            at = slice(r, r + n)
            hk = h // (nv // nk)
            o[at, h], last = sv.delta_rule(q[at, hk], k[at, hk], v[at, h], g[at, h], beta[at, h],
                                           first, scale, norm)
            if 0 <= slot_out[b] < len(state):
                s[slot_out[b], h] = last
        r += n
    return o, s


def off(a, b):
    return np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30)


CASES = [  # key heads, value heads, dk, dv, rows per sequence
    (2, 2, 128, 128, [1]),
    (2, 4, 128, 128, [1, 1, 1, 1, 1]),
    (1, 3, 64, 64, [2, 1, 5]),
    (2, 2, 32, 40, [7]),
    (1, 2, 4, 4, [9]),
    (1, 1, 256, 64, [3, 1]),
    (2, 2, 96, 128, [70]),
    (1, 2, 256, 256, [100]),
    (2, 4, 128, 128, [64]),
    (2, 4, 128, 128, [65, 63, 1, 0, 128]),
    (1, 2, 128, 128, [33]),
    (4, 4, 64, 64, [200, 17]),
    (1, 3, 64, 128, [130, 64]),
    (2, 2, 128, 64, [127]),
    (1, 2, 128, 128, [700]),
    (16, 32, 128, 128, [150, 300]),
]


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("nk,nv,dk,dv,news", CASES)
def test_delta_rule_matches_float64(mi355x, stream, nk, nv, dk, dv, news, dtype):
    say(f"delta rule heads={nk}/{nv} dk={dk} dv={dv} rows={news} {dtype}")
    rng = np.random.default_rng(dk + dv + len(news))
    x = make(rng, news, nk, nv, dk, dv, dtype, pad=2)
    n = len(news)
    state = (rng.standard_normal((2 * n + 1, nv, dk, dv)) * 0.3).astype(np.float32)
    ids = rng.permutation(2 * n)
    slot_in, slot_out = list(ids[:n]), list(ids[n:])
    if n > 1:
        slot_in[1] = -1           # a fresh sequence
        slot_out[0] = slot_in[0]  # in place
    o, s = run(mi355x, stream, x, news, nk, nv, dk, dv, dtype, state, slot_in, slot_out)
    wo, ws = want_of(x, news, nk, nv, dk, dv, state, slot_in, slot_out, dk ** -0.5)
    tol = (2 * dk + 64) * 2.0 ** -24
    eo, es = off(o[:sum(news)], wo), off(s, ws)
    print(f"    normwise err o {eo:.2e} state {es:.2e}", flush=True)
    assert es <= tol and eo <= tol + (2.0 ** -11 if dtype == "float16" else 0.0)
    keep = [i for i in range(2 * n + 1) if i not in slot_out]
    assert np.array_equal(s[keep], state[keep])


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("decay,news", [(30.0, [130, 3]), (0.0, [200]), (1e-4, [300]), (400.0, [70])])
def test_decays(mi355x, stream, decay, news, dtype):
    """No decay, hardly any, and decays that wipe the state out in a token."""
    say(f"delta rule, decay scale {decay}, {dtype}")
    nk, nv, dk, dv = 1, 2, 128, 128
    rng = np.random.default_rng(int(decay) + 1)
    x = make(rng, news, nk, nv, dk, dv, dtype, decay=decay)
    if decay == 400.0:
        x[3][5, 0], x[3][20, 1], x[3][64, 0] = -np.inf, -3e38, -np.inf
    state = rng.standard_normal((2, nv, dk, dv)).astype(np.float32)
    io = list(range(len(news)))
    o, s = run(mi355x, stream, x, news, nk, nv, dk, dv, dtype, state, io, io)
    wo, ws = want_of(x, news, nk, nv, dk, dv, state, io, io, dk ** -0.5)
    tol = (2 * dk + 64) * 2.0 ** -24
    assert off(s, ws) <= tol and off(o, wo) <= tol + (2.0 ** -11 if dtype == "float16" else 0.0)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("news", [[1, 3], [90, 200]])
def test_repeated_keys(mi355x, stream, news, dtype):
    """The same key token after token with beta near one: the state holds the newest value, and the
    products within a chunk are as far from small as they come."""
    say(f"delta rule with one key, rows={news} {dtype}")
    nk, nv, dk, dv = 1, 2, 64, 128
    rng = np.random.default_rng(8)
    q, k, v, g, beta = make(rng, news, nk, nv, dk, dv, dtype, decay=0.01)
    k[:] = k[:1]
    beta[:] = 0.999
    state = np.zeros((2, nv, dk, dv), np.float32)
    x = (q, k, v, g, beta)
    o, s = run(mi355x, stream, x, news, nk, nv, dk, dv, dtype, state, [0, 1], [0, 1])
    wo, ws = want_of(x, news, nk, nv, dk, dv, state, [0, 1], [0, 1], dk ** -0.5)
    # each of the chunk's 64 rows is formed from the 63 before it, with factors near one
    tol = 64 * (2 * dk + 64) * 2.0 ** -24
    assert off(s, ws) <= tol and off(o, wo) <= tol + (2.0 ** -11 if dtype == "float16" else 0.0)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("news", [[1, 2], [40, 100]])
def test_strides_scale_and_no_norm(mi355x, stream, news, dtype):
    say(f"delta rule, strided rows={news} {dtype}")
    nk, nv, dk, dv = 2, 4, 64, 64
    rng = np.random.default_rng(4)
    x = make(rng, news, nk, nv, dk, dv, dtype, pad=1, norm=False)
    state = rng.standard_normal((3, nv, dk, dv)).astype(np.float32)
    for pads in ((8, 16, 24, 8), (3, 1, 5, 7)):
        o, s = run(mi355x, stream, x, news, nk, nv, dk, dv, dtype, state, [0, 5], [2, -1], norm=False,
                   pads=pads, scale=0.7)
        wo, ws = want_of(x, news, nk, nv, dk, dv, state, [0, 5], [2, -1], 0.7, norm=False)
        tol = (2 * dk + 64) * 2.0 ** -24
        assert off(s, ws) <= tol
        assert off(o[:sum(news)], wo) <= tol + (2.0 ** -11 if dtype == "float16" else 0.0)


def test_a_prompt_in_pieces_is_the_prompt_at_once(mi355x, stream):
    """Chunks of a prompt and then single tokens, carried through a slot, against one call."""
    say("delta rule, a prompt in pieces")
    nk, nv, dk, dv, T = 2, 4, 128, 128, 260
    rng = np.random.default_rng(13)
    x = make(rng, [T], nk, nv, dk, dv, "float32")
    zero = np.zeros((1, nv, dk, dv), np.float32)
    o, s = run(mi355x, stream, x, [T], nk, nv, dk, dv, "float32", zero, [0], [0])
    st, parts, at = zero, [], 0
    for n in (100, 64, 1, 1, 90, 1, 3):
        po, st = run(mi355x, stream, tuple(a[at:at + n] for a in x), [n], nk, nv, dk, dv, "float32", st,
                     [0], [0])
        parts.append(po)
        at += n
    tol = 2 * (2 * dk + 64) * 2.0 ** -24
    assert at == T and off(np.concatenate(parts), o) <= tol and off(st, s) <= tol


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_many_sequences_of_all_lengths(mi355x, stream, dtype):
    """More sequences than a wave looks at in one go, empty ones and single tokens among prompts: some
    go token by token and some chunk by chunk in the same call."""
    say(f"delta rule, 150 sequences, {dtype}")
    nk, nv, dk, dv = 1, 2, 64, 64
    rng = np.random.default_rng(17)
    news = [0, 1, 23, 24, 25, 63, 64, 65, 128, 0, 2, 129, 1, 0]
    news = news + [int(n) for n in rng.choice([0, 1, 1, 3, 26, 40], 150 - len(news))]
    x = make(rng, news, nk, nv, dk, dv, dtype, pad=70)
    n = len(news)
    state = (rng.standard_normal((n, nv, dk, dv)) * 0.3).astype(np.float32)
    slot_in = rng.permutation(n)
    slot_out = slot_in.copy()
    slot_in[5::7] = n + 3  # afresh
    slot_out[3::11] = -1   # left nowhere
    o, s = run(mi355x, stream, x, news, nk, nv, dk, dv, dtype, state, slot_in, slot_out)
    wo, ws = want_of(x, news, nk, nv, dk, dv, state, slot_in, slot_out, dk ** -0.5)
    tol = (2 * dk + 64) * 2.0 ** -24
    assert off(s, ws) <= tol and off(o[:sum(news)], wo) <= tol + (2.0 ** -11 if dtype == "float16" else 0.0)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("news", [[12], [90, 150]])
def test_magnitudes_far_apart(mi355x, stream, news, dtype):
    """Keys and queries of lengths from 2^-8 to 2^8 (they are normalised), columns of v and of the state
    from 2^-40 to 2^40 (fp16 rows: v 2^-6 to 2^6): every column to its own scale."""
    say(f"delta rule, magnitudes far apart, rows={news} {dtype}")
    nk, nv, dk, dv = 2, 2, 128, 64
    rng = np.random.default_rng(21)
    q, k, v, g, beta = make(rng, news, nk, nv, dk, dv, "float32")
    T = sum(news)
    q *= 2.0 ** rng.integers(-8, 9, (T, nk, 1))
    k *= 2.0 ** rng.integers(-8, 9, (T, nk, 1))
    wide = 40 if dtype == "float32" else 6
    col = 2.0 ** rng.integers(-wide, wide + 1, dv)
    x = tuple(a.astype(sv.DT[dtype]) for a in (q, k, v * col)) + (g, beta)
    state = (rng.standard_normal((2, nv, dk, dv)) * col).astype(np.float32)
    io = list(range(len(news)))
    o, s = run(mi355x, stream, x, news, nk, nv, dk, dv, dtype, state, io, io)
    wo, ws = want_of(x, news, nk, nv, dk, dv, state, io, io, dk ** -0.5)
    tol = (2 * dk + 64) * 2.0 ** -24
    half = 0.0 if dtype == "float32" else 2.0 ** -11
    for c in range(dv):
        assert off(s[..., c], ws[..., c]) <= tol
        # an output under fp16's normal range is off by half its smallest step
        small = 0.0 if dtype == "float32" else 2.0 ** -25 * np.sqrt(wo[..., c].size)
        assert np.linalg.norm(o[..., c] - wo[..., c]) <= (tol + half) * np.linalg.norm(wo[..., c]) + small


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("n,at", [(10, 4), (150, 70), (150, 63), (150, 0), (130, 129)])
def test_a_token_that_is_not_finite_leaves_those_before_it(mi355x, stream, n, at, dtype):
    """NaN or an infinity in one token of v (one column), k, g, beta or q: what comes before it is as it
    was, what follows is not finite, and q's is its own row alone."""
    say(f"delta rule, poisoned token {at} of {n}, {dtype}")
    nk, nv, dk, dv = 1, 1, 64, 32
    rng = np.random.default_rng(n + at)
    news = [n] * 7
    q, k, v, g, beta = x = make(rng, news, nk, nv, dk, dv, dtype)
    v[at, 0, 5] = np.nan
    v[n + at, 0, 7] = np.inf
    k[2 * n + at, 0, 9] = np.nan
    g[3 * n + at] = np.nan
    beta[4 * n + at] = np.nan
    q[5 * n + at, 0, 3] = np.nan
    k[6 * n + at, 0, 3] = -np.inf
    state = rng.standard_normal((7, nv, dk, dv)).astype(np.float32)
    io = list(range(7))
    o, s = run(mi355x, stream, x, news, nk, nv, dk, dv, dtype, state, io, io)
    with np.errstate(invalid="ignore", over="ignore"):
        wo, ws = want_of(x, news, nk, nv, dk, dv, state, io, io, dk ** -0.5)
    assert np.array_equal(np.isfinite(o), np.isfinite(wo)) and np.array_equal(np.isfinite(s), np.isfinite(ws))
    tol = (2 * dk + 64) * 2.0 ** -24
    ok, good = np.isfinite(wo), np.isfinite(ws)
    assert off(s[good], ws[good]) <= tol
    assert off(o[ok], wo[ok]) <= tol + (2.0 ** -11 if dtype == "float16" else 0.0)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("nk,nv,dk,dv,news", [
    (1, 2, 32, 40, [70]), (1, 1, 4, 4, [65]), (3, 3, 100, 12, [30, 90]), (2, 6, 64, 24, [64, 25]),
    (8, 8, 128, 256, [40]), (1, 4, 124, 132, [129])])
def test_chunks_of_odd_heads(mi355x, stream, nk, nv, dk, dv, news, dtype):
    """Head sizes that fill no tile, in sequences that go chunk by chunk."""
    say(f"delta rule heads={nk}/{nv} dk={dk} dv={dv} rows={news} {dtype}")
    rng = np.random.default_rng(dk * dv)
    x = make(rng, news, nk, nv, dk, dv, dtype, pad=1)
    state = (rng.standard_normal((3, nv, dk, dv)) * 0.3).astype(np.float32)
    io = list(range(len(news)))
    o, s = run(mi355x, stream, x, news, nk, nv, dk, dv, dtype, state, io, io, pads=(0, 0, 0, 4))
    wo, ws = want_of(x, news, nk, nv, dk, dv, state, io, io, dk ** -0.5)
    tol = (2 * dk + 64) * 2.0 ** -24
    assert off(s, ws) <= tol and off(o[:sum(news)], wo) <= tol + (2.0 ** -11 if dtype == "float16" else 0.0)
    assert np.array_equal(s[len(news):], state[len(news):])


@pytest.mark.parametrize("news", [[3], [70]])
def test_state_slots_behind_four_gigabytes(mi355x, stream, news):
    """The last slots of more than 2^32 bytes of states, out of one call and into the next."""
    say(f"delta rule, far slots, rows={news}")
    nk, nv, dk, dv = 2, 4, 128, 128
    slots = (5 << 30) // (nv * dk * dv * 4)
    rng = np.random.default_rng(3)
    x = make(rng, [2 * news[0]], nk, nv, dk, dv, "float32")
    n = news[0]
    buf = mi355x.alloc_device(slots * nv * dk * dv * 4)
    runner = GatedDeltaRunner(mi355x)
    try:
        with sv.Arrays(mi355x, stream) as ar:
            o0 = np.zeros((n, nv, dv), np.float32)
            got = []
            for i, (a, b) in enumerate([(-1, slots - 1), (slots - 1, slots - 2)]):
                q, k, v, g, beta = (ar.put(t[i * n:(i + 1) * n]) for t in x)
                po = ar.put(o0)
                ids = np.array([a], np.int32), np.array([b], np.int32)
                args = delta_args(q=q, k=k, v=v, g=g, beta=beta, o=po, state=int(buf.handle),
                                  slot_in=ar.put(ids[0]), slot_out=ar.put(ids[1]),
                                  q_start=ar.put(np.array([0, n], np.int32)), n_slots=slots, n_seqs=1, rows=n,
                                  max_q=n, n_k_heads=nk, n_v_heads=nv, head_dim_k=dk, head_dim_v=dv,
                                  dtype="float32")
                runner.reserve(args)
                runner.forward_device(args, stream)
                got.append(ar.get(po, o0))
    finally:
        mi355x.synchronize_stream(stream)
        runner.close()
        mi355x.free_device(buf)
    zero = np.zeros((1, nv, dk, dv), np.float32)
    wo, _ = want_of(x, [2 * n], nk, nv, dk, dv, zero, [0], [0], dk ** -0.5)
    assert off(np.concatenate(got), wo) <= 2 * (2 * dk + 64) * 2.0 ** -24


def test_a_state_that_faded_keeps_its_digits(mi355x, stream):
    """States of 2^-70, chunks that add nothing to them (beta 0) and chunks that do."""
    say("delta rule, faded states")
    nk, nv, dk, dv, news = 1, 2, 64, 32, [200, 20]
    rng = np.random.default_rng(30)
    q, k, v, g, beta = x = make(rng, news, nk, nv, dk, dv, "float32")
    v *= np.float32(2.0 ** -70)
    beta[:130] = 0.0
    beta[200:210] = 0.0
    g *= np.float32(0.01)
    state = (rng.standard_normal((2, nv, dk, dv)) * 2.0 ** -70).astype(np.float32)
    o, s = run(mi355x, stream, x, news, nk, nv, dk, dv, "float32", state, [0, 1], [0, 1])
    wo, ws = want_of(x, news, nk, nv, dk, dv, state, [0, 1], [0, 1], dk ** -0.5)
    tol = (2 * dk + 64) * 2.0 ** -24
    assert off(s, ws) <= tol and off(o, wo) <= tol
    for r in range(0, 220, 20):  # every stretch to its own size
        assert off(o[r:r + 20], wo[r:r + 20]) <= tol
