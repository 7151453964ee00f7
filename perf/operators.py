"""The serving operators that performance is measured on: what a server does with the memory that its
sequences carry from call to call.

  "attn"    attention of a batch of new tokens (one per sequence, or a chunk) over a paged key/value cache
  "append"  q / k norm and rotary embedding at the cache positions, keys and values into the pages
  "pages"   copies of pages inside the pools of many layers (forks, compaction, snapshots)
  "delta"   the gated delta rule over a ragged batch, from and to the state slots of its sequences

Where ``own`` is false a call runs in elementary torch operations in 32 bits; where it is true it is the
package's call on the same memory.  Lengths of a ragged batch follow from the case alone (``mix`` seeds
them), contents and page numbers from the seed of ``prepare``.  Shapes are Qwen3-Next's attention layers
(16 query heads over 2 key/value heads of 256; 16 key and 32 value heads of 128) and generic ones.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TORCH = {"float32": torch.float32, "float16": torch.float16, "int8": torch.int8}
ESZ = {"float32": 4, "float16": 2, "int8": 1}
EPS = 1e-6
THETA = 5000000.0
CHUNK = 64


# ---- the cases -------------------------------------------------------------------------------

def _attn(name, n_seqs, ctx, new, dtype="float16", heads=(16, 2, 256), page=64, ragged=True, gate=False, mix=1):
    """``ctx`` cached tokens at most, the ``new`` ones of a sequence at most among them."""
    return {"name": name, "kind": "attn", "n_seqs": n_seqs, "ctx": ctx, "new": new, "dtype": dtype, "nh": heads[0],
            "nkv": heads[1], "hd": heads[2], "page": page, "ragged": ragged, "gate": gate, "mix": mix}


def _append(name, n_seqs, ctx, new, dtype="float16", heads=(16, 2, 256), rotary=64, page=64, ragged=True, mix=1):
    return {"name": name, "kind": "append", "n_seqs": n_seqs, "ctx": ctx, "new": new, "dtype": dtype, "nh": heads[0],
            "nkv": heads[1], "hd": heads[2], "rotary": rotary, "page": page, "ragged": ragged, "mix": mix}


def _pages(name, pools, n_pages, copies, page_bytes):
    return {"name": name, "kind": "pages", "pools": pools, "n_pages": n_pages, "copies": copies,
            "page_bytes": page_bytes}


def _delta(name, n_seqs, new, dtype="float16", heads=(16, 32, 128, 128), ragged=True, mix=1):
    return {"name": name, "kind": "delta", "n_seqs": n_seqs, "new": new, "dtype": dtype, "nk": heads[0], "nv": heads[1],
            "dk": heads[2], "dv": heads[3], "ragged": ragged, "mix": mix}


def listed():
    return [
        # Two users' next tokens after short prompts: latency is all there is.
        _attn("attn_decode_2", 2, 913, 1),
        # A full decode batch with contexts from hundreds to twelve thousand tokens, cache in int8.
        _attn("attn_decode_int8_40", 40, 12000, 1, dtype="int8", mix=2),
        # Prompts of all lengths, fed in chunks next to sequences that already decode.
        _attn("attn_mixed", 12, 7001, 401, page=32, mix=3),
        # One long prompt's next chunk behind what is cached already, output gated as in the layer.
        _attn("attn_prefill", 1, 8192, 2048, ragged=False, gate=True),
        # The 32-bit path: a chunk over a 32-bit cache, generic heads of 128.
        _attn("attn_float32", 3, 1500, 130, dtype="float32", heads=(8, 2, 128), page=16, mix=4),
        # The rows of a decode batch: norm, rotation and 64 pages touched for a row each.
        _append("append_decode_64", 64, 9000, 1, mix=5),
        # The rows of a long chunk.
        _append("append_prefill", 2, 8192, 2048, ragged=False),
        # A sequence forks: the part-filled page of each of 12 layers.
        _pages("pages_fork", 24, 96, 2, 65536),
        # Compaction of a busy cache.
        _pages("pages_compact", 24, 640, 250, 65536),
        # One token of one user through the recurrence, 32-bit rows.
        _delta("delta_decode_1", 1, 1, dtype="float32"),
        # A decode batch: two mebibytes of state read and written for each sequence.
        _delta("delta_decode_96", 96, 1),
        # Prompts of uneven length in one call.
        _delta("delta_prefill", 4, 2600, mix=6),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "append", "pages", "delta", "delta"])
    mix = rng.randrange(1, 1 << 20)
    heads = rng.choice([(16, 2, 256), (16, 2, 256), (32, 8, 128), (12, 4, 96), (6, 6, 64), (8, 2, 128)])
    page = rng.choice([16, 32, 64, 128])
    if kind == "attn":
        dtype = rng.choice(["float16", "float16", "int8", "float32"])
        form = rng.choice(["decode", "decode", "chunk", "prefill"])
        if form == "decode":
            n, new = _log_int(rng, 1, 48), rng.choice([1, 1, 1, 2, 4])
            ctx = _log_int(rng, max(new, 17), 12000)
        elif form == "chunk":
            n, new = _log_int(rng, 1, 12), _log_int(rng, 3, 400)
            ctx = _log_int(rng, new + 1, 7000)
        else:
            n, new = 1, _log_int(rng, 200, 2048)
            ctx = min(8192, new + _log_int(rng, 1, 6144))
        if dtype == "float32":  # the 32-bit matrix rate is a sixteenth
            n, new, ctx = min(n, 8), min(new, 300), max(min(new, 300), min(ctx, 2000))
        return {k: v for k, v in _attn("", n, ctx, new, dtype, heads, page, n > 1 and rng.random() < 0.8,
                                       rng.random() < 0.3, mix).items() if k != "name"}
    if kind == "append":
        n = _log_int(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, 4096 // n)
        rotary = rng.choice([heads[2], heads[2] // 2, 32])
        return {k: v for k, v in _append("", n, new + _log_int(rng, 1, 9000), new, rng.choice(["float16", "float16", "float32"]),
                                         heads, rotary, page, rng.random() < 0.7, mix).items() if k != "name"}
    if kind == "pages":
        pools = rng.choice([2, 8, 24, 48])
        size = rng.choice([1024, 8192, 16384, 65536, 131072])
        copies = _log_int(rng, 1, max(2, min(400, (250 * 24 * 65536) // (pools * size))))
        return {k: v for k, v in _pages("", pools, 2 * copies + rng.randrange(1, 40), copies, size).items() if k != "name"}
    dheads = rng.choice([(16, 32, 128, 128), (16, 32, 128, 128), (32, 32, 128, 128), (8, 8, 64, 64), (4, 12, 64, 128)])
    dtype = rng.choice(["float16", "float16", "float32"])
    if rng.random() < 0.4:
        n, new = _log_int(rng, 1, 96), rng.choice([1, 1, 1, 2, 5])
    else:
        n = _log_int(rng, 1, 8)
        new = _log_int(rng, 20, 5000 // n)
    return {k: v for k, v in _delta("", n, new, dtype, dheads, n > 1 and rng.random() < 0.8, mix).items() if k != "name"}


def _lens(case):
    """(new rows, cached tokens) of every sequence; the new rows are among the cached tokens.  The first
    sequence has the most of both, so a case's size is its numbers'."""
    rng = random.Random(case["mix"])
    n, new, ctx = case["n_seqs"], case["new"], case.get("ctx", 0)
    if not case["ragged"]:
        return [new] * n, [max(ctx, new)] * n
    ns, cs = [], []
    for i in range(n):
        m = new if i == 0 or rng.random() < 0.2 else 1 if rng.random() < 0.3 else _log_int(rng, 1, new)
        ns.append(m)
        cs.append(max(ctx, new) if i == 0 else _log_int(rng, m, max(ctx, m)))
    return ns, cs


# ---- inputs ----------------------------------------------------------------------------------

def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + salt)
    return g


def _randn(shape, g, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class State:
    """What a program has in hand before a call; the attributes differ by the kind of case."""


def _batch(case, s, g):
    """The ragged batch over pages that lie anywhere in the pool, as after hours of serving."""
    ns, cs = _lens(case)
    per = [-(-c // case["page"]) for c in cs]
    s.max_pages, s.n_pages = max(per), sum(per) + 3
    ids = torch.randperm(s.n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(ns), s.max_pages), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = ids[at:at + p]
        at += p
    starts = [0]
    for m in ns:
        starts.append(starts[-1] + m)
    s.table, s.q_start, s.kv_len, s.rows = table, _ints(starts), _ints(cs), starts[-1]
    s.max_q, s.max_kv = max(ns), max(cs)


def _pool(case, s, g, std):
    shape = (s.n_pages, case["nkv"], case["page"], case["hd"])
    x = torch.randn(shape, device="cuda", generator=g) * std
    if case["dtype"] != "int8":
        return x.to(TORCH[case["dtype"]]), None
    scale = x.abs().amax(dim=-1) / 127
    return (x / scale[..., None]).round_().clamp_(-127, 127).to(torch.int8), scale


def _stream():
    return torch.cuda.current_stream().cuda_stream or None


def _package():
    import os
    import sys

    path = os.path.abspath("disk-mem-off_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from moe_mi355x.backends import MI355XBackend
    from moe_mi355x import delta_rule, paged_kv

    return MI355XBackend(torch.cuda.current_device()), paged_kv, delta_rule


def _workspace(nbytes):
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device="cuda")


def _own_cache(case, s):
    """The package's cache over this memory, and the batch."""
    s.backend, paged_kv, _ = _package()
    scales = (s.ks.data_ptr(), s.vs.data_ptr()) if case["dtype"] == "int8" else (None, None)
    s.cache = paged_kv.PagedKvCache(s.backend, 1, case["nkv"], case["hd"], s.n_pages, page_size=case["page"],
                                    dtype=case["dtype"], buffers=[(s.k.data_ptr(), s.v.data_ptr(), *scales)])
    s.batch = paged_kv.paged_batch(s.q_start.data_ptr(), s.kv_len.data_ptr(), s.table.data_ptr(),
                                   n_seqs=case["n_seqs"], max_pages=s.max_pages, rows=s.rows, max_q=s.max_q,
                                   max_kv=s.max_kv)
    return paged_kv


def _prepare_attn(case, seed):
    s, g = State(), _gen(seed)
    _batch(case, s, g)
    s.k, s.ks = _pool(case, s, g, 1.0)
    s.v, s.vs = _pool(case, s, g, 1.0)
    dt = torch.float32 if case["dtype"] == "float32" else torch.float16
    s.q = _randn((s.rows, case["nh"], case["hd"]), g, 1.5, dt)
    s.gate = _randn((s.rows, case["nh"], case["hd"]), g) if case["gate"] else None
    s.out = torch.zeros_like(s.q)
    s.scale = case["hd"] ** -0.5
    if own:
        paged_kv = _own_cache(case, s)
        s.args = paged_kv.attn_args(s.q.data_ptr(), s.out.data_ptr(), n_heads=case["nh"], head_dim=case["hd"],
                                    scale=s.scale, gate=s.gate.data_ptr() if case["gate"] else None)
        s.work = _workspace(s.cache.attn_workspace_bytes(s.batch, case["nh"]))
    return s


def _prepare_append(case, seed):
    s, g = State(), _gen(seed)
    _batch(case, s, g)
    s.k, s.ks = _pool(case, s, g, 1.0)
    s.v, s.vs = _pool(case, s, g, 1.0)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    # The projections' rows: queries and their gates side by side, then keys and values.
    s.qg = _randn((s.rows, 2 * nh * hd), g)
    s.kx = _randn((s.rows, nkv * hd), g)
    s.vx = _randn((s.rows, nkv * hd), g)
    s.qw = 1.0 + _randn((hd,), g, 0.1)
    s.kw = 1.0 + _randn((hd,), g, 0.1)
    s.q_out = torch.zeros((s.rows, nh, hd), device="cuda",
                          dtype=torch.float32 if case["dtype"] == "float32" else torch.float16)
    s.freq = THETA ** -(torch.arange(case["rotary"] // 2, dtype=torch.float64, device="cuda") / (case["rotary"] // 2))
    if own:
        paged_kv = _own_cache(case, s)
        s.args = paged_kv.append_args(q=s.qg.data_ptr(), k=s.kx.data_ptr(), v=s.vx.data_ptr(),
                                      q_out=s.q_out.data_ptr(), q_norm=s.qw.data_ptr(), k_norm=s.kw.data_ptr(),
                                      n_heads=nh, n_kv_heads=nkv, head_dim=hd, ldq=2 * nh * hd,
                                      rotary_dim=case["rotary"], rope_theta=THETA, eps=EPS)
    return s


def _prepare_pages(case, seed):
    s, g = State(), _gen(seed)
    s.pool = _randn((case["pools"], case["n_pages"], case["page_bytes"] // 2), g, 1.0, torch.float16)
    ids = torch.randperm(case["n_pages"], device="cuda", generator=g).to(torch.int32)
    s.src, s.dst = ids[:case["copies"]].contiguous(), ids[case["copies"]:2 * case["copies"]].contiguous()
    if own:
        s.backend, paged_kv, _ = _package()
        s.pools = paged_kv.page_pools([(s.pool[i].data_ptr(), case["page_bytes"], case["n_pages"])
                                       for i in range(case["pools"])])
        s.copy_pages = paged_kv.copy_pages
    return s


def _prepare_delta(case, seed):
    s, g = State(), _gen(seed)
    ns, _ = _lens(case)
    starts = [0]
    for m in ns:
        starts.append(starts[-1] + m)
    s.q_start, s.rows, s.max_q = _ints(starts), starts[-1], max(ns)
    nk, nv, dk, dv, n = case["nk"], case["nv"], case["dk"], case["dv"], case["n_seqs"]
    dt = TORCH[case["dtype"]]

    def conv(h, d):  # what comes out of the short convolution and its activation
        x = _randn((s.rows, h, d), g)
        return (x * torch.sigmoid(x)).to(dt)

    s.q, s.k, s.v = conv(nk, dk), conv(nk, dk), conv(nv, dv)
    rate = torch.exp(_randn((nv,), g, 0.5))
    s.g = -rate * torch.log1p(torch.exp(_randn((s.rows, nv), g, 0.7) + torch.linspace(-5.0, 0.0, nv, device="cuda")))
    s.beta = torch.sigmoid(_randn((s.rows, nv), g))
    # A slot to start from and one to leave the state in for each sequence; some begin afresh.
    s.state = _randn((2 * n, nv, dk, dv), g, 0.1)
    ids = torch.randperm(2 * n, device="cuda", generator=g).to(torch.int32)
    s.slot_in, s.slot_out = ids[:n].contiguous(), ids[n:].contiguous()
    if case["new"] > 1:
        s.slot_in[1::3] = -1
    s.o = torch.zeros((s.rows, nv, dv), device="cuda", dtype=dt)
    s.scale = dk ** -0.5
    if own:
        s.backend, _, delta_rule = _package()
        s.args = delta_rule.delta_args(
            q=s.q.data_ptr(), k=s.k.data_ptr(), v=s.v.data_ptr(), g=s.g.data_ptr(), beta=s.beta.data_ptr(),
            o=s.o.data_ptr(), state=s.state.data_ptr(), slot_in=s.slot_in.data_ptr(), slot_out=s.slot_out.data_ptr(),
            q_start=s.q_start.data_ptr(), n_slots=2 * n, n_seqs=n, rows=s.rows, max_q=s.max_q, n_k_heads=nk,
            n_v_heads=nv, head_dim_k=dk, head_dim_v=dv, dtype=case["dtype"], qk_norm=True, scale=s.scale)
        s.runner = delta_rule.GatedDeltaRunner(s.backend)
        s.work = _workspace(delta_rule.workspace_bytes(s.args))
    return s


def prepare(case, seed):
    make = {"attn": _prepare_attn, "append": _prepare_append, "pages": _prepare_pages, "delta": _prepare_delta}
    s = make[case["kind"]](case, seed)
    s.case = case
    return s


# ---- the plain forms -------------------------------------------------------------------------

def _rows_of(s):
    """Sequence of every row, and the row's place among its sequence's rows."""
    row = torch.arange(s.rows, device="cuda")
    seq = (row[:, None] >= s.q_start[None, 1:]).sum(dim=1)
    return seq, row - s.q_start[seq]


def _plain_attn(s):
    c = s.case
    nh, nkv, hd, n = c["nh"], c["nkv"], c["hd"], c["n_seqs"]
    grp = nh // nkv
    pages = s.table.clamp_min(0).long()

    def cached(pool, scale):
        x = pool[pages].float()
        if scale is not None:
            x = x * scale[pages][..., None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, nkv, -1, hd)

    k, v = cached(s.k, s.ks), cached(s.v, s.vs)
    seq, at = _rows_of(s)
    q = torch.zeros((n, s.max_q, nh, hd), device="cuda")
    q[seq, at] = s.q.float()
    q = q.view(n, s.max_q, nkv, grp, hd).permute(0, 2, 1, 3, 4).reshape(n, nkv, s.max_q * grp, hd)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * s.scale
    new = s.q_start[1:] - s.q_start[:-1]
    last = (s.kv_len - new)[:, None] + torch.arange(s.max_q, device="cuda")[None]
    key = torch.arange(k.shape[2], device="cuda")
    seen = key[None, None] <= last[:, :, None]
    scores = scores.view(n, nkv, s.max_q, grp, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    p = (p / p.sum(dim=-1, keepdim=True)).view(n, nkv, s.max_q * grp, -1)
    o = torch.matmul(p, v).view(n, nkv, s.max_q, grp, hd).permute(0, 2, 1, 3, 4).reshape(n, s.max_q, nh, hd)
    o = o[seq, at]
    if s.gate is not None:
        o = o * torch.sigmoid(s.gate)
    s.out.copy_(o)
    return s.out


def _plain_append(s):
    c = s.case
    nh, nkv, hd, half = c["nh"], c["nkv"], c["hd"], c["rotary"] // 2
    seq, at = _rows_of(s)
    pos = (s.kv_len - (s.q_start[1:] - s.q_start[:-1]))[seq] + at
    ang = pos.double()[:, None] * s.freq
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]

    def heads(x, w):
        x = x.view(s.rows, -1, hd)
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], dim=-1)

    s.q_out.copy_(heads(s.qg[:, :nh * hd], s.qw))
    page, slot = s.table[seq, pos // c["page"]].long(), pos % c["page"]
    s.k[page, :, slot] = heads(s.kx, s.kw).to(s.k.dtype)
    s.v[page, :, slot] = s.vx.view(s.rows, nkv, hd).to(s.v.dtype)
    return s.q_out, s.k, s.v


def _plain_pages(s):
    s.pool[:, s.dst.long()] = s.pool[:, s.src.long()]
    return s.pool


def _plain_delta(s):
    c = s.case
    nk, nv, dk, dv, n = c["nk"], c["nv"], c["dk"], c["dv"], c["n_seqs"]
    size = min(CHUNK, 1 << (s.max_q - 1).bit_length())
    chunks = -(-s.max_q // size)
    seq, at = _rows_of(s)

    def heads(x, h):  # [sequence, head, chunk, row of the chunk, ...]; rows past a sequence's end are zero
        y = torch.zeros((n, chunks * size, *x.shape[1:]), device="cuda")
        y[seq, at] = x
        y = y.view(n, chunks, size, *x.shape[1:]).movedim(3, 1)
        return y.repeat_interleave(nv // h, dim=1)

    def unit(x):
        x = x.float()
        return x * torch.rsqrt((x * x).sum(dim=-1, keepdim=True) + EPS)

    q, k, v = heads(unit(s.q) * s.scale, nk), heads(unit(s.k), nk), heads(s.v.float(), nv)
    beta, g = heads(s.beta, nv)[..., None], heads(s.g, nv).double().cumsum(dim=-1)
    low = torch.ones(size, size, dtype=torch.bool, device="cuda").tril()
    decay = torch.exp((g[..., :, None] - g[..., None, :]).masked_fill(~low, -math.inf)).float()
    kt = k.transpose(-1, -2).contiguous()
    a = torch.matmul(k * beta, kt) * decay
    idx = torch.arange(size, device="cuda")
    inv = torch.eye(size, device="cuda").expand_as(a)
    for step in [1 << i for i in range((size - 1).bit_length())]:  # blocks of twice the size from pairs
        pair = (idx[:, None] // (2 * step) == idx[None] // (2 * step)) & (idx[:, None] // step > idx[None] // step)
        inv = inv - torch.matmul(torch.matmul(inv, (a * pair).contiguous()), inv.contiguous())
    eg = torch.exp(g).float()[..., None]
    to_end = torch.exp(g[..., -1:] - g).float()[..., None]
    u0, w = torch.matmul(inv, v * beta), torch.matmul(inv, k * (beta * eg))
    score = torch.matmul(q, kt) * decay
    qg, kend = q * eg, (k * to_end).transpose(-1, -2).contiguous()
    state = s.state[s.slot_in.clamp_min(0).long()] * (s.slot_in >= 0)[:, None, None, None]
    out = torch.empty_like(v)
    for i in range(chunks):
        u = u0[:, :, i] - torch.matmul(w[:, :, i], state)
        out[:, :, i] = torch.matmul(qg[:, :, i], state) + torch.matmul(score[:, :, i], u)
        state = state * eg[:, :, i, -1:] + torch.matmul(kend[:, :, i], u)
    s.o.copy_(out.movedim(1, 3).reshape(n, chunks * size, nv, dv)[seq, at])
    s.state[s.slot_out.long()] = state
    return s.o, s.state


# ---- a pass ----------------------------------------------------------------------------------

def run(s):
    kind = s.case["kind"]
    if own:
        if kind == "attn":
            s.cache.attend(0, s.batch, s.args, _stream(), (s.work.data_ptr(), s.work.numel()))
            return s.out
        if kind == "append":
            s.cache.append(0, s.batch, s.args, _stream())
            return s.q_out, s.k, s.v
        if kind == "pages":
            s.copy_pages(s.pools, s.src.data_ptr(), s.dst.data_ptr(), s.case["copies"], _stream())
            return s.pool
        s.runner.forward_device(s.args, _stream(), (s.work.data_ptr(), s.work.numel()))
        return s.o, s.state
    return {"attn": _plain_attn, "append": _plain_append, "pages": _plain_pages, "delta": _plain_delta}[kind](s)


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    if case["kind"] == "pages":
        return {"bytes": 2.0 * case["pools"] * case["copies"] * case["page_bytes"], "flops": 0.0}
    ns, cs = _lens(case)
    rows = sum(ns)
    if case["kind"] == "attn":
        nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
        row = nkv * (hd * ESZ[case["dtype"]] + (4 if case["dtype"] == "int8" else 0))
        io = rows * nh * hd * ((8 if case["dtype"] == "float32" else 4) + (4 if case["gate"] else 0))
        pairs = sum(m * (c - m) + m * (m + 1) // 2 for m, c in zip(ns, cs))
        return {"bytes": float(2 * row * sum(cs) + io), "flops": 4.0 * nh * hd * pairs}
    if case["kind"] == "append":
        nh, nkv, hd, e = case["nh"], case["nkv"], case["hd"], ESZ[case["dtype"]]
        return {"bytes": float(rows * hd * ((nh + 2 * nkv) * 4 + (nh + 2 * nkv) * e)),
                "flops": float(rows * hd * 8 * (nh + nkv))}
    nk, nv, dk, dv, e = case["nk"], case["nv"], case["dk"], case["dv"], ESZ[case["dtype"]]
    state = 4 * case["n_seqs"] * nv * dk * dv
    return {"bytes": float(2 * state + rows * (e * (2 * nk * dk + 2 * nv * dv) + 8 * nv)),
            "flops": 6.0 * rows * nv * dk * dv}


# ---- the same in 64 bits ---------------------------------------------------------------------

def _exact_attn(case, s):
    nh, nkv, hd, ps = case["nh"], case["nkv"], case["hd"], case["page"]
    ns, cs = _lens(case)
    out = torch.zeros(s.rows, nh, hd, dtype=torch.float64, device="cuda")
    first = 0
    for b, (m, c) in enumerate(zip(ns, cs)):
        ids = s.table[b, :-(-c // ps)].long()
        j = torch.arange(c, device="cuda")
        for h in range(nh):
            kv = h // (nh // nkv)
            k, v = s.k[ids, kv].reshape(-1, hd)[:c].double(), s.v[ids, kv].reshape(-1, hd)[:c].double()
            if case["dtype"] == "int8":
                k = k * s.ks[ids, kv].reshape(-1)[:c, None].double()
                v = v * s.vs[ids, kv].reshape(-1)[:c, None].double()
            w = s.q[first:first + m, h].double() @ k.T.contiguous() * s.scale
            w[j[None] > torch.arange(c - m, c, device="cuda")[:, None]] = -math.inf
            w = torch.exp(w - w.max(dim=1, keepdim=True).values)
            out[first:first + m, h] = (w @ v) / w.sum(dim=1, keepdim=True)
        first += m
    return out / (1.0 + torch.exp(-s.gate.double())) if case["gate"] else out


def _exact_append(case, s):
    nh, nkv, hd, ps, rot = case["nh"], case["nkv"], case["hd"], case["page"], case["rotary"]
    ns, cs = _lens(case)
    k, v = s.k.double(), s.v.double()
    q_out = torch.empty(s.rows, nh, hd, dtype=torch.float64, device="cuda")
    first = 0
    for b, (m, c) in enumerate(zip(ns, cs)):
        pos = torch.arange(c - m, c, dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones(m, 1, rot // 2, dtype=torch.float64, device="cuda"),
                           (pos[:, None] / THETA ** (torch.arange(0, rot, 2, device="cuda").double() / rot))[:, None])

        def rotated(x, w):
            x = x.double().reshape(m, -1, hd)
            x = w.double() * x / torch.sqrt(x.square().mean(dim=2, keepdim=True) + EPS)
            z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * turn
            return torch.cat([z.real, z.imag, x[..., rot:]], dim=2)

        r = slice(first, first + m)
        q_out[r] = rotated(s.qg[r, :nh * hd], s.qw)
        at = torch.arange(c - m, c, device="cuda")
        ids = s.table[b].long()[at // ps]
        k[ids, :, at % ps] = rotated(s.kx[r], s.kw)
        v[ids, :, at % ps] = s.vx[r].double().reshape(m, nkv, hd)
        first += m
    return q_out, k, v


def _exact_pages(s):
    out = s.pool.clone()
    for a, b in zip(s.src.tolist(), s.dst.tolist()):
        out[:, b] = s.pool[:, a]
    return out


def _exact_delta(case, s):
    """Token by token, all sequences side by side."""
    nk, nv, dk, dv, n = case["nk"], case["nv"], case["dk"], case["dv"], case["n_seqs"]
    ns, _ = _lens(case)
    start = s.q_start.tolist()
    state = torch.zeros(n, nv, dk, dv, dtype=torch.float64, device="cuda")
    for b, slot in enumerate(s.slot_in.tolist()):
        if slot >= 0:
            state[b] = s.state[slot].double()
    head = torch.arange(nv, device="cuda") // (nv // nk)
    q, k, v = s.q.double(), s.k.double(), s.v.double()
    q = (q / torch.sqrt(q.square().sum(dim=2, keepdim=True) + EPS) * s.scale)[:, head]
    k = (k / torch.sqrt(k.square().sum(dim=2, keepdim=True) + EPS))[:, head]
    decay, beta = torch.exp(s.g.double()), s.beta.double()
    o = torch.empty(s.rows, nv, dv, dtype=torch.float64, device="cuda")
    order = sorted(range(n), key=lambda b: -ns[b])
    for t in range(max(ns)):
        live = torch.tensor([b for b in order if ns[b] > t], device="cuda")
        r = torch.tensor([start[b] + t for b in order if ns[b] > t], device="cuda")
        x = state[live] * decay[r][:, :, None, None]
        miss = v[r] - (x * k[r][..., None]).sum(dim=2)
        x = x + k[r][..., None] * (beta[r][..., None] * miss)[:, :, None]
        o[r] = (x * q[r][..., None]).sum(dim=2)
        state[live] = x
    whole = s.state.double()
    whole[s.slot_out.long()] = state
    return o, whole


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "attn":
        return _exact_attn(case, s)
    if case["kind"] == "append":
        return _exact_append(case, s)
    return _exact_pages(s) if case["kind"] == "pages" else _exact_delta(case, s)
