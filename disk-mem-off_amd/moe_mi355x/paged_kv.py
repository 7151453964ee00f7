"""Paged key/value cache of a server's sequences, on the MI355X.

The reference keeps no cache: each step re-runs the whole prefix.  Here a sequence's keys and
values live in pages of ``page_size`` tokens, one pool of pages per layer, and three device
operators work on them: ``mx_kv_append`` (q / k norm, rotary embedding, new rows into the
pages), ``mx_paged_attn`` (the new rows' attention over everything cached) and
``mx_copy_pages`` (forks, compaction).  ``PageTables`` does the bookkeeping on the host: which
pages a sequence has, shared pages of forked sequences, free pages.

A call takes raw device addresses and a stream, as the package's other runners do; the functions
``paged_batch``, ``append_args``, ``attn_args`` and ``page_pools`` build its argument blocks,
which a program builds once and passes as often as it likes.
"""
from __future__ import annotations

import ctypes
from typing import Any, Iterable, Sequence

import numpy as np

from . import _lib
from .types import DeviceBuffer

_DT = {"float32": _lib.MX_DT_F32, "float16": _lib.MX_DT_F16, "int8": _lib.MX_DT_I8}
_ESZ = {"float32": 4, "float16": 2, "int8": 1}


# ---- argument blocks -------------------------------------------------------------------------

def paged_batch(q_start: int, kv_len: int, pages: int, *, n_seqs: int, max_pages: int, rows: int,
                max_q: int, max_kv: int) -> _lib.MxPagedBatch:
    """The sequences of a call from device arrays (int32) the caller filled."""
    return _lib.MxPagedBatch(q_start, kv_len, pages, n_seqs, max_pages, rows, max_q, max_kv)


def append_args(*, k: int, v: int, n_kv_heads: int, head_dim: int, q: int | None = None,
                q_out: int | None = None, n_heads: int = 0, q_norm: int | None = None,
                k_norm: int | None = None, rotary_dim: int = 0, rope_theta: float = 10000.0,
                eps: float = 1e-6, dtype: str = "float32", param_dtype: str = "float32",
                ldq: int | None = None, ldk: int | None = None, ldv: int | None = None,
                ldqo: int | None = None) -> _lib.MxKvRows:
    """Rows of an append (device addresses of ``dtype`` rows; strides default to contiguous)."""
    for name in (dtype, param_dtype):
        if name not in ("float32", "float16"):
            raise ValueError(f"rows and norm weights must be float32 or float16, got {name!r}")
    qw, kw = n_heads * head_dim, n_kv_heads * head_dim
    return _lib.MxKvRows(q, k, v, q_out, q_norm, k_norm, qw if ldq is None else ldq,
                         kw if ldk is None else ldk, kw if ldv is None else ldv,
                         qw if ldqo is None else ldqo, n_heads, rotary_dim, _DT[dtype],
                         _DT[param_dtype], float(rope_theta), float(eps))


def attn_args(q: int, out: int, *, n_heads: int, head_dim: int, scale: float | None = None,
              gate: int | None = None, ldq: int | None = None, ldo: int | None = None,
              ldg: int | None = None) -> _lib.MxPagedAttn:
    """Rows of an attention call (scale defaults to ``head_dim ** -0.5``)."""
    w = n_heads * head_dim
    return _lib.MxPagedAttn(q, out, gate, w if ldq is None else ldq, w if ldo is None else ldo,
                            w if ldg is None else ldg, n_heads,
                            float(head_dim ** -0.5 if scale is None else scale))


def page_pools(pools: Iterable[tuple[int, int, int]]) -> Any:
    """Pools (base address, bytes per page, pages) for :func:`copy_pages`."""
    items = [_lib.MxPagePool(*p) for p in pools]
    return (_lib.MxPagePool * len(items))(*items)


def copy_pages(pools: Any, src: int, dst: int, n_copies: int, stream: Any) -> None:
    """Page ``dst[i]`` of every pool becomes page ``src[i]`` (device int32 arrays)."""
    _lib.check(_lib.load().mx_copy_pages(pools, len(pools), src, dst, n_copies, stream),
               "mx_copy_pages")


# ---- bookkeeping -----------------------------------------------------------------------------

class PageTables:
    """Which pages every sequence has (host only).

    A page may belong to several sequences after a fork; a sequence that grows into a page it
    shares gets a copy of its own first.  ``extend`` and ``compact`` return the (source,
    destination) copies the pools need, in lists that :func:`copy_pages` accepts: no page is a
    destination twice or a destination and a source.
    """

    def __init__(self, n_pages: int, page_size: int) -> None:
        if n_pages <= 0 or page_size <= 0:
            raise ValueError("n_pages and page_size must be positive")
        self.n_pages = n_pages
        self.page_size = page_size
        self._refs = [0] * n_pages
        self._free = list(range(n_pages - 1, -1, -1))  # lowest page last
        self._pages: dict[int, list[int]] = {}
        self._len: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._len[self._known(seq)]

    def pages(self, seq: int) -> list[int]:
        return list(self._pages[self._known(seq)])

    def _known(self, seq: int) -> int:
        if seq not in self._pages:
            raise ValueError(f"unknown sequence {seq}")
        return seq

    def add(self) -> int:
        """A new, empty sequence."""
        seq = self._next
        self._next += 1
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens; all pages are shared until one side grows."""
        self._known(seq)
        new = self.add()
        self._pages[new], self._len[new] = list(self._pages[seq]), self._len[seq]
        for p in self._pages[new]:
            self._refs[p] += 1
        return new

    def extend(self, growth: Iterable[tuple[int, int]]) -> list[tuple[int, int]]:
        """Room for ``n`` more tokens of each sequence (every sequence at most once); raises
        RuntimeError and changes nothing when the free pages do not suffice."""
        growth = [(self._known(s), int(n)) for s, n in growth]
        if len({s for s, _ in growth}) != len(growth):
            raise ValueError("a sequence may grow once per call")
        refs = dict[int, int]()
        plan = []
        need = 0
        for s, n in growth:
            if n < 0:
                raise ValueError("sequences grow by a non-negative number of tokens")
            have, used = self._pages[s], self._len[s]
            fresh = -(-(used + n) // self.page_size) - len(have)
            last = have[-1] if have else -1
            own = True
            if n and used % self.page_size:  # the part-filled page is written to
                r = refs.get(last, self._refs[last])
                own = r == 1
                if not own:
                    refs[last] = r - 1
            plan.append((s, n, fresh, own))
            need += fresh + (not own)
        if need > len(self._free):
            raise RuntimeError(f"the cache is full: {need} pages needed, {len(self._free)} free")
        copies = []
        for s, n, fresh, own in plan:
            have = self._pages[s]
            if not own:
                copies.append((have[-1], self._take()))
                self._refs[have[-1]] -= 1
                have[-1] = copies[-1][1]
            have.extend(self._take() for _ in range(fresh))
            self._len[s] += n
        return copies

    def _take(self) -> int:
        p = self._free.pop()
        self._refs[p] = 1
        return p

    def take_back(self, growth: Sequence[tuple[int, int]], copies: list[tuple[int, int]]) -> None:
        """Undoes the last ``extend(growth)``, which gave ``copies``."""
        source = {d: s for s, d in copies}
        for seq, n in reversed(growth):
            have = self._pages[seq]
            self._len[seq] -= n
            while len(have) > -(-self._len[seq] // self.page_size):
                self._give(have.pop())
            if have and have[-1] in source:
                self._give(have[-1])
                have[-1] = source[have[-1]]
                self._refs[have[-1]] += 1

    def _give(self, p: int) -> None:
        self._refs[p] = 0
        self._free.append(p)

    def free(self, seq: int) -> None:
        """Forgets the sequence; pages no other sequence has become free."""
        back = []
        for p in self._pages.pop(self._known(seq)):
            self._refs[p] -= 1
            if not self._refs[p]:
                back.append(p)
        del self._len[seq]
        if back:
            self._free = sorted([*self._free, *back], reverse=True)

    def compact(self) -> list[tuple[int, int]]:
        """Moves pages so that the used ones are the first; the copies to make for it."""
        used = [p for p in range(self.n_pages) if self._refs[p]]
        holes = [p for p in range(len(used)) if not self._refs[p]]
        moves = list(zip([p for p in used if p >= len(used)], holes))
        self.move(moves)
        return moves

    def move(self, moves: list[tuple[int, int]]) -> None:
        """Used pages to free places, (from, to), in the tables."""
        to = dict(moves)
        for s, d in moves:
            self._refs[d], self._refs[s] = self._refs[s], 0
        for have in self._pages.values():
            have[:] = [to.get(p, p) for p in have]
        self._free = [p for p in range(self.n_pages - 1, -1, -1) if not self._refs[p]]


# ---- the cache -------------------------------------------------------------------------------

class PagedKvCache:
    """Pools of pages for ``n_layers`` layers, their page tables, and the calls on them.

    ``buffers`` (one (k, v, k_scale, v_scale) of device addresses per layer) puts the pools into
    memory of the caller's; without it the cache allocates them.  All calls on one cache go
    to one stream at a time: a call's device arrays are reused by the next in stream order.
    """

    def __init__(self, backend: Any, n_layers: int, n_kv_heads: int, head_dim: int, n_pages: int,
                 *, page_size: int = 64, dtype: str = "float16",
                 buffers: Sequence[tuple[int, int, int | None, int | None]] | None = None) -> None:
        if dtype not in _DT:
            raise ValueError(f"cache dtype must be one of {sorted(_DT)}, got {dtype!r}")
        if n_layers <= 0 or n_kv_heads <= 0 or head_dim <= 0:
            raise ValueError("n_layers, n_kv_heads and head_dim must be positive")
        if buffers is not None and len(buffers) != n_layers:
            raise ValueError(f"{len(buffers)} buffers for {n_layers} layers")
        self.backend = backend
        self.lib = _lib.load()
        self.tables = PageTables(n_pages, page_size)
        self.dtype = dtype
        self._owned: list[DeviceBuffer] = []
        self._ws: DeviceBuffer | None = None
        self._ids: DeviceBuffer | None = None
        self._lists: DeviceBuffer | None = None
        rows = n_pages * n_kv_heads * page_size
        sizes = [rows * head_dim * _ESZ[dtype]] * 2 + [rows * 4 if dtype == "int8" else 0] * 2
        if buffers is None:
            buffers = []
            try:
                for _ in range(n_layers):
                    got = []
                    for size in sizes:
                        if size:
                            self._owned.append(backend.alloc_device(size))
                        got.append(int(self._owned[-1].handle) if size else None)
                    buffers.append(tuple(got))
            except BaseException:
                self.close()
                raise
        self.layers = [_lib.MxKvCache(*b, n_pages, page_size, n_kv_heads, head_dim, _DT[dtype])
                       for b in buffers]
        per = page_size * n_kv_heads
        page_bytes = [per * head_dim * _ESZ[dtype]] * 2 + [per * 4] * 2
        self.pools = page_pools((p, nb, n_pages) for b in buffers
                                for p, nb in zip(b, page_bytes) if p)

    # -- device calls --
    def append(self, layer: int, batch: _lib.MxPagedBatch, rows: _lib.MxKvRows,
               stream: Any) -> None:
        """The batch's new rows into the layer's pages (and rotated queries out)."""
        _lib.check(self.lib.mx_kv_append(ctypes.byref(self.layers[layer]), ctypes.byref(batch),
                                         ctypes.byref(rows), stream), "mx_kv_append")

    def attn_workspace_bytes(self, batch: _lib.MxPagedBatch, n_heads: int) -> int:
        n = ctypes.c_size_t()
        _lib.check(self.lib.mx_paged_attn_workspace_size(
            ctypes.byref(self.layers[0]), ctypes.byref(batch), n_heads, ctypes.byref(n)),
            "mx_paged_attn_workspace_size")
        return int(n.value)

    def reserve_attn(self, batch: _lib.MxPagedBatch, n_heads: int) -> None:
        """Workspace for this attention call and any that needs no more (not while an earlier
        call still runs)."""
        need = self.attn_workspace_bytes(batch, n_heads)
        if need and (self._ws is None or self._ws.nbytes < need):
            self._drop("_ws")
            self._ws = self.backend.alloc_device(need)

    def attend(self, layer: int, batch: _lib.MxPagedBatch, args: _lib.MxPagedAttn, stream: Any,
               workspace: tuple[int, int] | None = None) -> None:
        """The batch's attention over the layer's pages.  ``workspace`` (address, bytes) stands
        in for the reserved one."""
        ptr, nbytes = workspace or ((self._ws.handle, self._ws.nbytes) if self._ws else (None, 0))
        _lib.check(self.lib.mx_paged_attn(ctypes.byref(self.layers[layer]), ctypes.byref(batch),
                                          ctypes.byref(args), ptr, nbytes, stream),
                   "mx_paged_attn")

    # -- sequences --
    def add(self) -> int:
        return self.tables.add()

    def fork(self, seq: int) -> int:
        return self.tables.fork(seq)

    def free(self, seq: int) -> None:
        self.tables.free(seq)

    def compact(self, stream: Any) -> None:
        """Used pages to the front of the pools; batches made before are void.  Waits for the
        stream; where a device call fails, the tables stay as they were."""
        moves = self.tables.compact()
        try:
            self._copy(moves, stream)
        except BaseException:
            self.tables.move([(d, s) for s, d in moves])
            raise

    def batch(self, growth: Iterable[tuple[int, int]], stream: Any) -> _lib.MxPagedBatch:
        """Grows the sequences by their new rows (copying part-filled pages they share) and
        uploads the tables of a call on them; the last batch of the cache is void then.

        The call waits for the stream, and tables that no longer fit are allocated anew, at another
        address: a graph, or a step that must not stall the host, takes :func:`paged_batch` with
        device arrays of the caller's.  Where a device call fails no sequence has grown."""
        growth = [(s, int(n)) for s, n in growth]
        copies = self.tables.extend(growth)
        try:
            self._copy(copies, stream)
            return self._tables(growth, stream)
        except BaseException:
            self.tables.take_back(growth, copies)
            raise

    def _tables(self, growth: list[tuple[int, int]], stream: Any) -> _lib.MxPagedBatch:
        pages = [self.tables.pages(s) for s, _ in growth]
        n, mp = len(growth), max([1, *(len(p) for p in pages)])
        starts = np.concatenate([[0], np.cumsum([m for _, m in growth])]).astype(np.int32)
        lens = np.array([self.tables.length(s) for s, _ in growth], dtype=np.int32)
        table = np.full((n, mp), -1, dtype=np.int32)
        for row, p in zip(table, pages):
            row[:len(p)] = p
        at = self._upload("_ids", [starts, lens, table.ravel()], stream)
        return paged_batch(at[0], at[1], at[2], n_seqs=n, max_pages=mp, rows=int(starts[-1]),
                           max_q=max([1, *(m for _, m in growth)]),
                           max_kv=max([1, *lens.tolist()]))

    def _copy(self, pairs: list[tuple[int, int]], stream: Any) -> None:
        if pairs:
            src, dst = np.array(pairs, dtype=np.int32).T
            at = self._upload("_lists", [src, dst], stream)
            copy_pages(self.pools, at[0], at[1], len(pairs), stream)

    def _upload(self, name: str, arrays: list[np.ndarray], stream: Any) -> list[int]:
        """Arrays into the named device buffer, each on a 16-byte boundary; their addresses."""
        offs, size = [], 0
        for a in arrays:
            offs.append(size)
            size += -(-a.nbytes // 16) * 16
        size = max(size, 16)
        host = np.zeros(size, dtype=np.uint8)
        for a, o in zip(arrays, offs):
            host[o:o + a.nbytes] = np.ascontiguousarray(a).view(np.uint8).ravel()
        buf = getattr(self, name)
        if buf is None or buf.nbytes < size:
            self.backend.synchronize_stream(stream)
            self._drop(name)
            buf = self.backend.alloc_device(2 * size)
            setattr(self, name, buf)
        self.backend.copy_h2d_ptr_async(buf.handle, host.ctypes.data, size, stream)
        self.backend.synchronize_stream(stream)  # the host array ends with this call
        return [int(buf.handle) + o for o in offs]

    def _drop(self, name: str) -> None:
        buf = getattr(self, name)
        if buf is not None:
            self.backend.free_device(buf)
            setattr(self, name, None)

    def close(self) -> None:
        for name in ("_ws", "_ids", "_lists"):
            self._drop(name)
        while self._owned:
            self.backend.free_device(self._owned.pop())
