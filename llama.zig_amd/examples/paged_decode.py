"""Serving with a paged cache: two attention blocks (quantized q/k/v and output
projections, rotary positions, attention, residual) take a prompt, fork it into
several sequences, decode them together in a captured graph, free one, compact
the pool and go on.

    python llama.zig_amd/examples/paged_decode.py

Weights are random, Q8_0.  `Server` is what a program keeps: the caches, the
page table and the lengths on the device, the free pages on the host.
"""
import pathlib
import sys
import time

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))
import ggml_hip as G  # noqa: E402

HEADS, KV_HEADS, DIM, WIDTH, PAGE = 32, 8, 128, 4096, 16


def q8_0(w):
    """f32 [rows, K] as block_q8_0: an f16 scale and 32 int8 codes per block."""
    x = w.view(w.shape[0], -1, 32)
    d = (x.abs().amax(-1, keepdim=True) / 127).half()
    q = (x / d.float().clamp_min(1e-30)).round().clamp(-127, 127).to(torch.int8)
    return torch.cat([d.view(torch.uint8), q.view(torch.uint8)], -1).reshape(w.shape[0], -1).contiguous()


def _norm(x):
    """Root mean square norm; the mean in two short sums, which a graph can hold (one over many blocks clears its
    scratch by a memory-set node)."""
    mean = x.square().view(x.shape[0], 64, -1).mean(-1).mean(-1, keepdim=True)
    return x * torch.rsqrt(mean + 1e-5)


class Server:
    def __init__(self, n_layers=2, n_pages=256, max_seqs=8, max_tokens=1024, seed=1, window=0, sinks=0):
        gen = torch.Generator("cuda").manual_seed(seed)
        rows = (HEADS + 2 * KV_HEADS) * DIM
        self.qkv = [q8_0(torch.randn((rows, WIDTH), generator=gen, device="cuda") * 0.02) for _ in range(n_layers)]
        self.o = [q8_0(torch.randn((WIDTH, HEADS * DIM), generator=gen, device="cuda") * 0.02) for _ in range(n_layers)]
        shape = (n_pages, KV_HEADS, PAGE, DIM)
        self.caches = [G.PagedKV(*(torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2)))
                       for _ in range(n_layers)]
        self.steps, self.mscale = G.rope_steps(DIM, 500000.0)
        self.table = torch.full((max_seqs, max_tokens // PAGE), -1, dtype=torch.int32, device="cuda")
        self.pages = [[] for _ in range(max_seqs)]  # the table's rows, on the host
        self.lens = [0] * max_seqs
        self.used = {}  # page: the sequences that have it
        self.free = list(range(n_pages))[::-1]
        self.window, self.sinks = window, sinks

    # ---- pages, on the host

    def _page(self):
        p = self.free.pop()
        self.used[p] = 1
        return p

    def _write_table(self):
        self.table.fill_(-1)
        for s, row in enumerate(self.pages):
            if row:
                self.table[s, :len(row)] = torch.tensor(row, dtype=torch.int32)

    def grow(self, seq, n):
        """Room for n more tokens of a sequence: their slots, and its new length."""
        first = self.lens[seq]
        self.lens[seq] += n
        while len(self.pages[seq]) * PAGE < self.lens[seq]:
            self.pages[seq].append(self._page())
        return [self.pages[seq][j // PAGE] * PAGE + j % PAGE for j in range(first, first + n)]

    def fork(self, parent, child):
        """The child shares the parent's full pages and has a copy of the last, partly filled one."""
        n = self.lens[parent]
        self.lens[child], self.pages[child] = n, list(self.pages[parent])
        for p in self.pages[child][:n // PAGE]:
            self.used[p] += 1
        if n % PAGE:
            src, dst = self.pages[parent][n // PAGE], self._page()
            self.pages[child][n // PAGE] = dst
            i32 = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")  # noqa: E731
            for kv in self.caches:
                G.copy_pages(kv, i32(src), i32(dst), i32(n % PAGE))
        self._write_table()

    def release(self, seq):
        for p in self.pages[seq]:
            self.used[p] -= 1
            if not self.used[p]:
                del self.used[p]
                self.free.append(p)
        self.pages[seq], self.lens[seq] = [], 0
        self._write_table()

    def compact(self):
        """Pages in use to the front of every layer's pool; the free ones are the rest."""
        lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        for kv in self.caches:
            table, live = G.compact_pages(kv, self.table, lens)
        rows, n = table.tolist(), int(live)
        old, self.used = self.used, {}
        for s, row in enumerate(self.pages):
            for i, p in enumerate(row):
                self.used[rows[s][i]] = old[p]
                row[i] = rows[s][i]
        self.table.copy_(table)
        self.free = list(range(n, self.caches[0].n_pages))[::-1]
        return n

    # ---- the blocks

    def forward(self, x, pos, slots, table, lens, starts=None, max_q=1, max_kv=None):
        """x f32 [tokens, WIDTH] through the blocks: norm, q/k/v, rotation and store, attention, output, residual."""
        n = x.shape[0]
        for qkv, o, kv in zip(self.qkv, self.o, self.caches):
            y = G.mul_mat("Q8_0", qkv, _norm(x))
            q, k, v = (t.unflatten(1, (-1, DIM)) for t in y.split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], 1))
            q = G.rope_kv_store(q, k, v, pos, self.steps, kv, slots, mscale=self.mscale)
            a = G.attn_paged(q, kv, table, lens, q_starts=starts, max_q=max_q, max_kv=max_kv, window=self.window,
                             sinks=self.sinks)
            x = G.add_f32(x, G.mul_mat("Q8_0", o, a.view(n, HEADS * DIM)))
        return x

    def prompt(self, seq, x):
        """A prompt (or more of one) of one sequence; its last token's result."""
        n = x.shape[0]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        first = self.lens[seq]
        slots = self.grow(seq, n)
        self._write_table()
        return self.forward(x, i32(range(first, first + n)), i32(slots), self.table[seq:seq + 1],
                            i32([self.lens[seq]]), starts=i32([0, n]), max_q=n, max_kv=self.lens[seq])[-1]


class Decoder:
    """A captured step of several sequences: one token each, every buffer kept."""

    def __init__(self, server, seqs):
        self.server, self.seqs = server, seqs
        n, i32 = len(seqs), lambda: torch.zeros(len(seqs), dtype=torch.int32, device="cuda")  # noqa: E731
        self.x = torch.zeros((n, WIDTH), device="cuda")
        self.pos, self.slots, self.lens = i32(), i32() - 1, i32()
        self.table = torch.full((n, server.table.shape[1]), -1, dtype=torch.int32, device="cuda")
        self._run()  # once before the capture
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.y = self._run()

    def _run(self):
        return self.server.forward(self.x, self.pos, self.slots, self.table, self.lens)

    def step(self, x):
        s = self.server
        slots = [s.grow(q, 1)[0] for q in self.seqs]
        s._write_table()
        self.x.copy_(x)
        self.pos.copy_(torch.tensor([s.lens[q] - 1 for q in self.seqs], dtype=torch.int32))
        self.lens.copy_(torch.tensor([s.lens[q] for q in self.seqs], dtype=torch.int32))
        self.slots.copy_(torch.tensor(slots, dtype=torch.int32))
        self.table.copy_(s.table[self.seqs])
        self.graph.replay()
        return self.y


def main(prompt_tokens=333, steps=40, seed=2, **kw):
    """Returns the inputs, by sequence, and every sequence's last result."""
    gen = torch.Generator("cuda").manual_seed(seed)
    rand = lambda n: torch.randn((n, WIDTH), generator=gen, device="cuda")  # noqa: E731
    s = Server(**kw)
    x = rand(prompt_tokens)
    t = time.perf_counter()
    s.prompt(0, x)
    torch.cuda.synchronize()
    print(f"prompt of {prompt_tokens} tokens: {(time.perf_counter() - t) * 1e3:.2f} ms, first call")
    for child in (1, 2):
        s.fork(0, child)
    seen = {q: [x] for q in (0, 1, 2)}
    last = {}

    def decode(seqs, n):
        d = Decoder(s, seqs)
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            new = rand(len(seqs))
            y = d.step(new)
            for i, q in enumerate(seqs):
                seen[q].append(new[i:i + 1])
        torch.cuda.synchronize()
        print(f"{n} steps of sequences {seqs}: {(time.perf_counter() - t) / n * 1e6:.0f} us a step")
        for i, q in enumerate(seqs):
            last[q] = y[i].clone()

    decode([0, 1, 2], steps)
    s.release(1)
    live = s.compact()
    print(f"sequence 1 freed, {live} pages in use, together at the front")
    decode([0, 2], steps)
    return s, {q: torch.cat(v) for q, v in seen.items()}, last


if __name__ == "__main__":
    main()
