"""Serving steps captured into graphs, and on two streams at once; a program of its own, because the
graphs are torch's and torch has to be imported before the library.  Exits with 0 when every
replay left what an eager step left, bit by bit."""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "disk-mem-off_amd"))

from moe_mi355x import delta_rule, paged_kv  # noqa: E402
from moe_mi355x.backends import MI355XBackend  # noqa: E402

NH, NKV, HD, PAGE, PAGES, SEQS, TABLE = 8, 2, 128, 32, 200, 5, 38
NK, NV, DK, DV = 2, 4, 64, 64
GPU = dict(device="cuda")


class Step:
    """A server's step over at most ``rows`` new rows: rows into the cache, attention, the delta rule
    and page copies, on tensors that stay where they are."""

    def __init__(self, backend, dtype, rows, max_q, max_kv, work):
        self.rows, self.max_q, self.max_kv = rows, max_q, max_kv
        dt = {"float16": torch.float16, "int8": torch.int8, "float32": torch.float32}[dtype]
        xdt = torch.float32 if dtype == "float32" else torch.float16
        name = "float32" if dtype == "float32" else "float16"
        z = lambda *s, d=torch.float32: torch.zeros(s, dtype=d, **GPU)  # noqa: E731
        self.kv = [z(PAGES, NKV, PAGE, HD, d=dt) for _ in range(2)]
        self.scales = [z(PAGES, NKV, PAGE) for _ in range(2)] if dtype == "int8" else [None, None]
        self.q, self.k, self.v = z(rows, NH * HD), z(rows, NKV * HD), z(rows, NKV * HD)
        self.q_out, self.out = z(rows, NH * HD, d=xdt), z(rows, NH * HD, d=xdt)
        self.dq, self.dk, self.dv = (z(rows, n, d=xdt) for n in (NK * DK, NK * DK, NV * DV))
        self.g, self.beta = z(rows, NV), z(rows, NV)
        self.do, self.state = z(rows, NV * DV, d=xdt), z(2 * SEQS, NV, DK, DV)
        ints = lambda *s: z(*s, d=torch.int32)  # noqa: E731
        self.q_start, self.kv_len, self.table = ints(SEQS + 1), ints(SEQS), ints(SEQS, TABLE)
        self.slots, self.src, self.dst = ints(2, SEQS), ints(3), ints(3)
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.cache = paged_kv.PagedKvCache(backend, 1, NKV, HD, PAGES, page_size=PAGE, dtype=dtype,
                                           buffers=[(at(self.kv[0]), at(self.kv[1]), *map(at, self.scales))])
        self.batch = paged_kv.paged_batch(at(self.q_start), at(self.kv_len), at(self.table), n_seqs=SEQS,
                                          max_pages=TABLE, rows=rows, max_q=max_q, max_kv=max_kv)
        self.append = paged_kv.append_args(q=at(self.q), k=at(self.k), v=at(self.v), q_out=at(self.q_out),
                                           n_heads=NH, n_kv_heads=NKV, head_dim=HD, rotary_dim=64)
        self.attn = paged_kv.attn_args(at(self.q_out), at(self.out), n_heads=NH, head_dim=HD)
        self.delta = delta_rule.delta_args(
            q=at(self.dq), k=at(self.dk), v=at(self.dv), g=at(self.g), beta=at(self.beta), o=at(self.do),
            state=at(self.state), slot_in=at(self.slots[0]), slot_out=at(self.slots[1]),
            q_start=at(self.q_start), n_slots=2 * SEQS, n_seqs=SEQS, rows=rows, max_q=max_q, n_k_heads=NK,
            n_v_heads=NV, head_dim_k=DK, head_dim_v=DV, dtype=name)
        self.runner = delta_rule.GatedDeltaRunner(backend)
        need = max(self.cache.attn_workspace_bytes(self.batch, NH), delta_rule.workspace_bytes(self.delta), 16)
        self.work = work if work is not None else torch.full((need,), 255, dtype=torch.uint8, **GPU)
        assert self.work.numel() >= need

    def fill(self, seed, news, lens):
        g = torch.Generator().manual_seed(seed)
        for t in (self.q, self.k, self.v, self.dq, self.dk, self.dv, self.out, self.do, self.state, *self.kv):
            if t.dtype == torch.int8:
                t.copy_(torch.randint(-127, 128, t.shape, generator=g, dtype=torch.int8))
            else:
                t.copy_(torch.randn(t.shape, generator=g))
        for t in self.scales:
            if t is not None:
                t.copy_(torch.rand(t.shape, generator=g) * 0.02)
        self.g.copy_(-torch.rand(self.g.shape, generator=g))
        self.beta.copy_(torch.rand(self.beta.shape, generator=g))
        ids = torch.randperm(PAGES - 6, generator=g).to(torch.int32)
        self.table.copy_(ids[:SEQS * TABLE].view(SEQS, TABLE))  # a sequence's pages are its own
        self.q_start.copy_(torch.tensor([0, *torch.tensor(news).cumsum(0).tolist()], dtype=torch.int32))
        self.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        self.slots.copy_(torch.randperm(2 * SEQS, generator=g).to(torch.int32).view(2, SEQS))
        self.src.copy_(ids[:3])
        self.dst.copy_(torch.arange(PAGES - 3, PAGES, dtype=torch.int32))

    def run(self):
        s = torch.cuda.current_stream().cuda_stream
        work = (self.work.data_ptr(), self.work.numel())
        self.cache.append(0, self.batch, self.append, s)
        self.cache.attend(0, self.batch, self.attn, s, work)
        self.runner.forward_device(self.delta, s, work)
        paged_kv.copy_pages(self.cache.pools, self.src.data_ptr(), self.dst.data_ptr(), 3, s)

    def results(self):
        return [*self.kv, *(t for t in self.scales if t is not None), self.q_out, self.out, self.do, self.state]


def same(a, b, what):
    torch.cuda.synchronize()
    for i, (x, y) in enumerate(zip(a.results(), b.results())):
        if not torch.equal(x.view(torch.uint8), y.view(torch.uint8)):
            sys.exit(f"{what}: result {i} differs")


NEWS = {2: [[1, 2, 0, 1, 1], [2, 2, 2, 2, 2], [0, 0, 0, 0, 0], [1, 1, 1, 1, 1]],
        100: [[30, 1, 0, 100, 7], [1, 1, 1, 1, 1], [100, 0, 24, 23, 3], [0, 0, 0, 0, 64]]}
LENS = [[700, 33, 0, 900, 1], [64, 1216, 500, 2, 130], [0, 5, 6, 0, 0], [1000, 1000, 31, 32, 33]]


def main():
    backend = MI355XBackend(torch.cuda.current_device())
    side = torch.cuda.Stream()
    for dtype in ("float16", "int8", "float32"):
        shapes = ((12, 2), (160, 100))
        big = Step(backend, dtype, 160, 100, 1216, None)
        work = big.work  # one workspace for both graphs: their replays are in order
        steps = {q: Step(backend, dtype, r, q, 1216, work) for r, q in shapes}
        eager = {q: Step(backend, dtype, r, q, 1216, None) for r, q in shapes}
        graphs = {}
        for q, st in steps.items():
            st.fill(1, NEWS[q][0], [max(a, b) for a, b in zip(LENS[0], NEWS[q][0])])
            with torch.cuda.stream(side):
                st.run()
                side.synchronize()
                graphs[q] = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graphs[q], stream=side):
                    st.run()
        for i in range(6):
            for q in steps:
                news = NEWS[q][i % 4]
                lens = [max(a, b) for a, b in zip(LENS[(i + q) % 4], news)]
                print(f"[gpu] replay {i}: {dtype}, new {news}, cached {lens}", flush=True)
                steps[q].fill(10 + i, news, lens)
                eager[q].fill(10 + i, news, lens)
                torch.cuda.synchronize()
                graphs[q].replay()
                a = torch.ones(256, 256, **GPU)
                (a @ a).sum().item()  # the program's own work
                eager[q].run()
                same(steps[q], eager[q], f"{dtype}, replay {i}, max_q {q}")
    # Two streams, each with a workspace of its own.
    print("[gpu] two streams at once", flush=True)
    pair = [Step(backend, "float16", 160, 100, 1216, None) for _ in range(2)]
    alone = [Step(backend, "float16", 160, 100, 1216, None) for _ in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        for n in range(2):
            for st in (pair[n], alone[n]):
                st.fill(50 + 2 * i + n, NEWS[100][(i + n) % 4],
                        [max(a, b) for a, b in zip(LENS[(i + n) % 4], NEWS[100][(i + n) % 4])])
        torch.cuda.synchronize()
        for n in range(2):
            with torch.cuda.stream(streams[n]):
                pair[n].run()
        torch.cuda.synchronize()
        for n in range(2):
            alone[n].run()
            torch.cuda.synchronize()
            same(pair[n], alone[n], f"stream {n}, round {i}")
    print("done", flush=True)


if __name__ == "__main__":
    main()
