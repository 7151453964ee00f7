"""Page bookkeeping of the serving cache, and what the entry points of the serving operators
refuse (all of it decided on the host, before any launch)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from moe_mi355x import _lib, delta_rule, paged_kv
from moe_mi355x.paged_kv import PagedKvCache, PageTables
from moe_mi355x.types import DeviceBuffer

A = 1 << 12  # an aligned address that is never read


def apply(pages, copies):
    """copies as the device makes them: all sources read, then all destinations written."""
    got = {d: pages[s] for s, d in copies}
    assert len(got) == len(copies) and not set(got) & {s for s, _ in copies}
    pages.update(got)


def test_sequences_grow_page_by_page():
    t = PageTables(8, 16)
    a, b = t.add(), t.add()
    assert t.extend([(a, 16), (b, 17)]) == []
    assert len(t.pages(a)) == 1 and len(t.pages(b)) == 2 and t.free_pages == 5
    assert t.extend([(a, 0), (b, 15)]) == [] and len(t.pages(b)) == 2 and t.length(b) == 32
    assert t.extend([(a, 1)]) == [] and len(t.pages(a)) == 2
    assert len(set(t.pages(a) + t.pages(b))) == 4


def test_a_full_cache_changes_nothing():
    t = PageTables(3, 16)
    a, b = t.add(), t.add()
    t.extend([(a, 20)])
    with pytest.raises(RuntimeError, match="full"):
        t.extend([(a, 1), (b, 30)])
    assert t.length(a) == 20 and t.length(b) == 0 and t.free_pages == 1 and not t.pages(b)
    t.extend([(a, 12), (b, 16)])
    assert t.free_pages == 0


@pytest.mark.parametrize("bad", [[(7, 1)], [(0, -1)], [(0, 1), (0, 1)]])
def test_bad_growth_is_refused(bad):
    t = PageTables(4, 16)
    t.add()
    with pytest.raises(ValueError):
        t.extend(bad)


def test_random_life_of_a_cache_keeps_every_sequence_its_tokens():
    """Forks, growth, frees and compactions in any order: every sequence reads back the tokens
    it was given, whatever pages they lie in."""
    rng = np.random.default_rng(3)
    t = PageTables(60, 4)
    pages = {p: [None] * 4 for p in range(60)}
    want: dict[int, list[int]] = {}
    made = moved = copied = 0
    for step in range(4000):
        what = rng.integers(6)
        if what == 0 and len(want) < 9:
            want[t.add()] = []
        elif what == 1 and want and len(want) < 9:
            s = int(rng.choice(list(want)))
            want[t.fork(s)] = list(want[s])
        elif what in (2, 3) and want:
            some = [int(s) for s in rng.permutation(list(want))[:rng.integers(1, 4)]]
            growth = [(s, int(rng.integers(0, 7))) for s in some]
            try:
                copies = t.extend(growth)
            except RuntimeError:
                continue
            apply(pages, [(s, d) for s, d in copies])
            for s, d in copies:
                pages[d] = list(pages[d])
            copied += len(copies)
            for s, n in growth:
                for i in range(len(want[s]), len(want[s]) + n):
                    made += 1
                    page = t.pages(s)[i // 4]
                    for other in want:  # nobody else may own the row that is written
                        if other != s and i // 4 < len(t.pages(other)) and len(want[other]) > i:
                            assert t.pages(other)[i // 4] != page
                    pages[page] = [*pages[page][:i % 4], made, *pages[page][i % 4 + 1:]]
                    want[s].append(made)
        elif what == 4 and want:
            s = int(rng.choice(list(want)))
            t.free(s)
            del want[s]
        elif what == 5:
            moves = t.compact()
            moved += len(moves)
            apply(pages, moves)
            used = {p for s in want for p in t.pages(s)}
            assert used == set(range(len(used))) and t.free_pages == 60 - len(used)
        for s, tokens in want.items():
            assert t.length(s) == len(tokens) and len(t.pages(s)) == -(-len(tokens) // 4)
            assert [pages[t.pages(s)[i // 4]][i % 4] for i in range(len(tokens))] == tokens
    assert made > 500 and moved > 20 and copied > 20


def test_freed_pages_return_once_the_last_owner_goes():
    t = PageTables(4, 16)
    a = t.add()
    t.extend([(a, 33)])
    b = t.fork(a)
    t.free(a)
    assert t.free_pages == 1
    t.free(b)
    assert t.free_pages == 4
    with pytest.raises(ValueError):
        t.free(b)


# ---- refusals --------------------------------------------------------------------------------

def cache(**kw):
    d = dict(k=A, v=A, k_scale=None, v_scale=None, n_pages=4, page_size=16, n_kv_heads=2,
             head_dim=64, dtype=_lib.MX_DT_F16)
    d.update(kw)
    return _lib.MxKvCache(**d)


def batch(**kw):
    d = dict(q_start=A, kv_len=A, pages=A, n_seqs=1, max_pages=2, rows=1, max_q=1, max_kv=20)
    d.update(kw)
    return _lib.MxPagedBatch(**d)


def rows(**kw):
    d = dict(q=A, k=A, v=A, q_out=A, q_norm_w=None, k_norm_w=None, ldq=256, ldk=128, ldv=128,
             ldqo=256, n_heads=4, rotary_dim=32, x_dtype=0, param_dtype=0, rope_theta=1e4, eps=1e-6)
    d.update(kw)
    return _lib.MxKvRows(**d)


def attn(**kw):
    d = dict(q=A, out=A, gate=None, ldq=256, ldo=256, ldg=256, n_heads=4, scale=0.1)
    d.update(kw)
    return _lib.MxPagedAttn(**d)


def delta(**kw):
    d = dict(q=A, k=A, v=A, g=A, beta=A, o=A, state=A, slot_in=A, slot_out=A, q_start=A, ldq=128,
             ldk=128, ldv=256, ldo=256, n_slots=2, n_seqs=1, rows=4, max_q=4, n_k_heads=2,
             n_v_heads=4, head_dim_k=64, head_dim_v=64, x_dtype=1, qk_norm=1, scale=0.1)
    d.update(kw)
    return _lib.MxGatedDelta(**d)


INV, UNS, ALI = _lib.MX_ERR_INVALID, _lib.MX_ERR_UNSUPPORTED, _lib.MX_ERR_ALIGNMENT

BAD_CACHE = [(dict(k=None), INV), (dict(v=None), INV), (dict(n_pages=0), INV),
             (dict(page_size=0), INV), (dict(page_size=8), UNS), (dict(page_size=48), UNS),
             (dict(page_size=512), UNS), (dict(head_dim=260), UNS), (dict(head_dim=260, dtype=0), UNS),
             (dict(head_dim=4), UNS), (dict(head_dim=0), INV), (dict(n_kv_heads=0), INV),
             (dict(dtype=7), INV), (dict(dtype=2), INV),
             (dict(dtype=2, k_scale=A, v_scale=A, head_dim=24), UNS),
             (dict(dtype=2, k_scale=A + 4, v_scale=A), ALI), (dict(k=A + 8), ALI), (dict(v=A + 2), ALI)]
BAD_BATCH = [(dict(q_start=None), INV), (dict(kv_len=None), INV), (dict(pages=None), INV),
             (dict(n_seqs=-1), INV), (dict(rows=-1), INV), (dict(max_pages=0), INV),
             (dict(max_q=0), INV), (dict(max_kv=-1), INV), (dict(n_seqs=65536), UNS),
             (dict(rows=1 << 24), UNS)]


def call_append(c, b, r):
    return _lib.load().mx_kv_append(ctypes.byref(c), ctypes.byref(b), ctypes.byref(r), None)


def call_attn(c, b, a, ws=None, nbytes=0):
    return _lib.load().mx_paged_attn(ctypes.byref(c), ctypes.byref(b), ctypes.byref(a), ws, nbytes,
                                     None)


@pytest.mark.parametrize("kw,rc", BAD_CACHE)
def test_bad_caches_are_refused(kw, rc):
    n = ctypes.c_size_t()
    assert call_append(cache(**kw), batch(), rows(ldk=2048, ldv=2048, ldq=2048, ldqo=2048)) == rc
    assert call_attn(cache(**kw), batch(), attn(ldq=2048, ldo=2048)) == rc
    assert _lib.load().mx_paged_attn_workspace_size(
        ctypes.byref(cache(**kw)), ctypes.byref(batch()), 4, ctypes.byref(n)) == rc


@pytest.mark.parametrize("kw,rc", BAD_BATCH)
def test_bad_batches_are_refused(kw, rc):
    assert call_append(cache(), batch(**kw), rows()) == rc
    assert call_attn(cache(), batch(**kw), attn()) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(k=None), INV), (dict(v=None), INV), (dict(q=None), INV), (dict(q_out=None), INV),
    (dict(n_heads=0), INV), (dict(rotary_dim=33), INV), (dict(rotary_dim=66), INV),
    (dict(rotary_dim=-2), INV), (dict(x_dtype=2), INV), (dict(param_dtype=2), INV),
    (dict(rope_theta=0.0), INV), (dict(rope_theta=float("nan")), INV), (dict(ldq=255), INV),
    (dict(ldk=127), INV), (dict(ldv=100), INV), (dict(ldqo=0), INV), (dict(k=A + 2), ALI),
    (dict(q_out=A + 1), ALI), (dict(q_norm_w=A + 2), ALI)])
def test_bad_rows_are_refused(kw, rc):
    assert call_append(cache(), batch(), rows(**kw)) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), INV), (dict(out=None), INV), (dict(n_heads=3), INV), (dict(n_heads=0), INV),
    (dict(ldq=248), INV), (dict(ldo=0), INV), (dict(gate=A, ldg=255), INV), (dict(q=A + 8), ALI),
    (dict(out=A + 4), ALI), (dict(gate=A + 4), ALI), (dict(ldq=260), ALI), (dict(ldo=257), ALI),
    (dict(gate=A, ldg=258), ALI)])
def test_bad_attention_rows_are_refused(kw, rc):
    assert call_attn(cache(), batch(), attn(**kw)) == rc


@pytest.mark.parametrize("kw,rc", [
    *((dict([(n, None)]), INV) for n in ("q", "k", "v", "g", "beta", "o", "state", "slot_in",
                                         "slot_out", "q_start")),
    (dict(n_seqs=-1), INV), (dict(rows=-1), INV), (dict(max_q=0), INV), (dict(n_slots=-1), INV),
    (dict(n_v_heads=3), INV), (dict(n_k_heads=0), INV), (dict(x_dtype=2), INV),
    (dict(ldq=127), INV), (dict(ldv=255), INV), (dict(head_dim_k=62), UNS),
    (dict(head_dim_v=260, ldv=2048, ldo=2048), UNS), (dict(n_seqs=65536), UNS),
    (dict(rows=1 << 24), UNS), (dict(state=A + 8), ALI), (dict(q=A + 1), ALI)])
def test_bad_delta_arguments_are_refused(kw, rc):
    n = ctypes.c_size_t()
    lib = _lib.load()
    assert lib.mx_gated_delta_rule(ctypes.byref(delta(**kw)), None, 0, None) == rc
    assert lib.mx_gated_delta_rule_workspace_size(ctypes.byref(delta(**kw)), ctypes.byref(n)) == rc


@pytest.mark.parametrize("pool,rc", [((A, 0, 4), INV), ((None, 64, 4), INV), ((A, 64, 0), INV),
                                     ((A, 24, 4), UNS), ((A + 8, 64, 4), ALI)])
def test_bad_pools_are_refused(pool, rc):
    lib = _lib.load()
    p = paged_kv.page_pools([(A, 64, 4), pool])
    assert lib.mx_copy_pages(p, 2, A, A, 1, None) == rc
    assert lib.mx_copy_pages(p, 2, None, A, 1, None) == INV
    assert lib.mx_copy_pages(p, -1, A, A, 1, None) == INV
    assert lib.mx_copy_pages(p, 1, A, A, -1, None) == INV


def test_null_structures_are_refused():
    lib = _lib.load()
    assert lib.mx_kv_append(None, None, None, None) == INV
    assert lib.mx_paged_attn(None, None, None, None, 0, None) == INV
    assert lib.mx_gated_delta_rule(None, None, 0, None) == INV
    assert lib.mx_copy_pages(None, 1, A, A, 1, None) == INV


def test_empty_calls_launch_nothing():
    for b in (batch(n_seqs=0), batch(rows=0)):
        assert call_append(cache(), b, rows()) == 0
    lib = _lib.load()
    assert lib.mx_gated_delta_rule(ctypes.byref(delta(n_seqs=0)), None, 0, None) == 0
    p = paged_kv.page_pools([(A, 64, 4)])
    assert lib.mx_copy_pages(p, 1, A, A, 0, None) == 0
    assert lib.mx_copy_pages(p, 0, A, A, 3, None) == 0


def test_python_arguments_are_checked():
    with pytest.raises(ValueError):
        paged_kv.append_args(k=A, v=A, n_kv_heads=2, head_dim=64, dtype="int8")
    with pytest.raises(ValueError):
        delta_rule.delta_args(q=A, k=A, v=A, g=A, beta=A, o=A, state=A, slot_in=A, slot_out=A,
                              q_start=A, n_slots=1, n_seqs=1, rows=1, max_q=1, n_k_heads=1,
                              n_v_heads=1, head_dim_k=64, head_dim_v=64, dtype="int8")
    with pytest.raises(ValueError):
        PagedKvCache(None, 1, 2, 64, 4, dtype="bfloat16")
    with pytest.raises(ValueError):
        PagedKvCache(None, 2, 2, 64, 4, buffers=[(A, A, None, None)])
    with pytest.raises(ValueError):
        PageTables(0, 16)


def test_delta_workspaces():
    """Token by token there is none; chunk by chunk it has to be there, large enough and aligned."""
    lib, n = _lib.load(), ctypes.c_size_t()

    def size(**kw):
        assert lib.mx_gated_delta_rule_workspace_size(ctypes.byref(delta(**kw)), ctypes.byref(n)) == 0
        return n.value

    long_rows = dict(rows=100, max_q=64)
    assert size() == 0 and size(rows=4, max_q=1000) == 0 and size(rows=1000, max_q=1) == 0
    assert size(head_dim_k=256, ldq=1024, ldk=1024, **long_rows) == 0
    need = size(**long_rows)
    assert need > 0 and size(rows=200, max_q=64) > need
    d = delta(**long_rows)
    assert lib.mx_gated_delta_rule(ctypes.byref(d), None, need, None) == _lib.MX_ERR_WORKSPACE
    assert lib.mx_gated_delta_rule(ctypes.byref(d), A, need - 1, None) == _lib.MX_ERR_WORKSPACE
    assert lib.mx_gated_delta_rule(ctypes.byref(d), A + 8, need, None) == ALI


@pytest.mark.parametrize("b,heads,kv_heads,rc", [
    (dict(max_kv=(1 << 30) + 1), 4, 2, UNS),   # key numbers would pass 32 bits inside the kernels
    (dict(max_kv=2 ** 31 - 1), 4, 2, UNS),
    (dict(rows=1 << 22), 16, 2, UNS),          # 2^26 rows of heads
    (dict(rows=1), 65536, 2, UNS),
    (dict(rows=(1 << 22) - 1), 16, 2, 0), (dict(max_kv=1 << 30), 4, 2, 0), (dict(rows=1), 65535, 1, 0)])
def test_sizes_behind_the_limits_of_attention_are_refused(b, heads, kv_heads, rc):
    """The workspace query and the call agree on what is too large; at the limits the query answers."""
    n = ctypes.c_size_t(77)
    c, ba = cache(n_kv_heads=kv_heads, head_dim=8), batch(**b)
    assert _lib.load().mx_paged_attn_workspace_size(ctypes.byref(c), ctypes.byref(ba), heads,
                                                    ctypes.byref(n)) == rc
    ld = heads * 8
    if rc:
        assert call_attn(c, ba, attn(n_heads=heads, ldq=ld, ldo=ld)) == rc
    else:  # no workspace: refused before any launch
        assert n.value > 0
        assert call_attn(c, ba, attn(n_heads=heads, ldq=ld, ldo=ld)) == _lib.MX_ERR_WORKSPACE


# ---- failing device calls --------------------------------------------------------------------

class FailingBackend:
    """Device calls that work until the ``fail``-th of them."""

    def __init__(self, fail=None):
        self.left, self.live, self.next = fail, {}, 1 << 20

    def _count(self):
        if self.left is not None:
            self.left -= 1
            if self.left < 0:
                raise RuntimeError("device call failed")

    def alloc_device(self, nbytes):
        self._count()
        self.next += -(-nbytes // 256) * 256
        self.live[self.next] = nbytes
        return DeviceBuffer(handle=self.next, nbytes=nbytes, backend="failing")

    def free_device(self, buf):
        del self.live[buf.handle]

    def copy_h2d_ptr_async(self, *args):
        self._count()

    def synchronize_stream(self, stream):
        self._count()


def state(t):
    return (list(t._refs), list(t._free), {s: list(p) for s, p in t._pages.items()}, dict(t._len))


def test_extend_can_be_taken_back():
    """From any state, with shared part-filled pages, whole new pages and growth of nothing."""
    rng = np.random.default_rng(8)
    t = PageTables(40, 4)
    tried = 0
    for _ in range(3000):
        seqs = list(t._pages)
        what = rng.integers(5)
        if what == 0 and len(seqs) < 7:
            t.add()
        elif what == 1 and seqs and len(seqs) < 7:
            t.fork(int(rng.choice(seqs)))
        elif what == 2 and len(seqs) > 2:
            t.free(int(rng.choice(seqs)))
        elif seqs:
            growth = [(int(s), int(rng.integers(0, 9))) for s in rng.permutation(seqs)[:4]]
            before = state(t)
            try:
                copies = t.extend(growth)
            except RuntimeError:
                assert state(t) == before
                continue
            t.take_back(growth, copies)
            assert state(t) == before
            tried += bool(copies)
            t.extend(growth)
    assert tried > 50


@pytest.mark.parametrize("fail", range(12))
def test_a_failing_device_call_leaves_the_sequences_as_they_were(monkeypatch, fail):
    monkeypatch.setattr(paged_kv, "copy_pages", lambda *a: be._count())
    be = FailingBackend()
    c = PagedKvCache(be, 1, 1, 16, 300, page_size=16, buffers=[(A, A, None, None)])
    a = c.add()
    c.batch([(a, 20)], None)
    b = c.fork(a)
    d = c.add()
    before = state(c.tables)
    be.left = fail  # a copied page, new pages, larger tables
    try:
        c.batch([(a, 1), (b, 30), (d, 4000)], None)
    except RuntimeError:
        assert state(c.tables) == before
        be.left = None
        c.batch([(a, 1), (b, 30), (d, 4000)], None)
    else:
        assert be.left >= 0 and c.tables.length(d) == 4000
    be.left = None
    c.close()
    assert not be.live


@pytest.mark.parametrize("fail", range(5))
def test_a_failing_compaction_moves_nothing(monkeypatch, fail):
    monkeypatch.setattr(paged_kv, "copy_pages", lambda *a: be._count())
    be = FailingBackend()
    c = PagedKvCache(be, 1, 1, 16, 30, page_size=16, buffers=[(A, A, None, None)])
    a, b = c.add(), c.add()
    c.batch([(a, 40), (b, 50)], None)
    c.free(a)
    before = state(c.tables)
    be.left = fail
    try:
        c.compact(None)
    except RuntimeError:
        assert state(c.tables) == before
        be.left = None
        c.compact(None)
    assert sorted(c.tables.pages(b)) == [0, 1, 2, 3]


@pytest.mark.parametrize("fail", range(8))
def test_a_cache_that_does_not_fit_leaves_nothing_behind(fail):
    be = FailingBackend(fail)
    with pytest.raises(RuntimeError):
        PagedKvCache(be, 3, 1, 16, 4, page_size=16, dtype="int8")
    assert not be.live
