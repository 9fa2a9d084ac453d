"""Draft trees for several sequences at once over the 4-bit paged cache.

A small seeded transformer without MLPs, its projections Q8_0 matrices run by
spec_qmatmul, serves a batch of prompts greedily in two ways: a token a step,
and with draft trees (the root and two guesses a level, some of them wrong).  Each
step is one plan, and per layer one append (rotation, 4-bit rows into the
pages) and one attention; after a tree is verified its accepted path is
committed by appending those rows again, alone.  Both ways give the same tokens.

    python examples/kv4_tree_decoding.py
"""

import importlib
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
pkg = importlib.import_module("abyo-speculate_b200")
synth = importlib.import_module("abyo-speculate_b200.gguf_synth")

Q8_0 = 8
LAYERS, HIDDEN, HEADS, KV_HEADS, DIM, VOCAB, PAGE = 2, 512, 8, 2, 64, 997, 32


class Server:
    """Weights, the page pool and one batch handle; sequences are lists of tokens."""

    def __init__(self, n_pages: int = 64, seed: int = 0):
        import torch
        self.torch = torch
        rng = np.random.default_rng(seed)

        def weight(rows, cols, sigma):
            w = (rng.standard_normal((rows, cols)) * sigma).astype(np.float32)
            return pkg.QWeight(Q8_0, synth.quantize(w, Q8_0), rows, cols)

        wide = (HEADS + 2 * KV_HEADS) * DIM
        self.qkv = [weight(wide, HIDDEN, 2.0 / HIDDEN ** 0.5) for _ in range(LAYERS)]
        self.o = [weight(HIDDEN, HEADS * DIM, 1.5 / HIDDEN ** 0.5) for _ in range(LAYERS)]
        self.embed = torch.from_numpy(rng.standard_normal((VOCAB, HIDDEN)).astype(np.float32)).cuda()
        size = pkg.KV4Cache.pool_bytes(n_layers=LAYERS, n_kv_heads=KV_HEADS, head_dim=DIM, page_tokens=PAGE,
                                       n_pages=n_pages)
        self.pool = torch.empty(size, dtype=torch.uint8, device="cuda")
        self.cache = pkg.KV4Cache(self.pool, n_layers=LAYERS, n_heads=HEADS, n_kv_heads=KV_HEADS, head_dim=DIM,
                                  page_tokens=PAGE, n_pages=n_pages, rope=pkg.rope_tables(DIM, 1024, 1e4))
        self.step = pkg.KV4Batch(self.cache)
        self.free = list(range(n_pages))
        self.stream = torch.cuda.Stream()

    def pages_for(self, table, tokens: int):
        while len(table) * PAGE < tokens:
            table.append(self.free.pop())

    def project(self, w, x):
        """x [rows, cols] f32 -> x . W^T, 64 rows a call."""
        y = self.torch.empty(x.shape[0], w.n_rows, device="cuda")
        for a in range(0, x.shape[0], 64):
            part = x[a:a + 64].contiguous()
            w.matmul(part.data_ptr(), part.shape[0], y[a:].data_ptr(), self.stream.cuda_stream)
        return y

    def forward(self, tables, kv_len, tokens, positions=None, masks=None):
        """Rows of new tokens of every sequence: their next-token argmax, and the layers' k and v rows."""
        torch = self.torch
        rows = [len(t) for t in tokens]
        for t, n, m in zip(tables, kv_len, rows):
            self.pages_for(t, n + m)
        with torch.cuda.stream(self.stream):
            self.step.plan(kv_len, rows, tables, positions=positions, masks=masks)
            x = self.embed[torch.tensor([t for s in tokens for t in s], device="cuda")]
            kept = []
            for layer in range(LAYERS):
                y = self.project(self.qkv[layer], torch.nn.functional.rms_norm(x, (HIDDEN,)))
                y = y.view(len(x), HEADS + 2 * KV_HEADS, DIM)  # f32 rows as the product leaves them
                k, v = y[:, HEADS:HEADS + KV_HEADS], y[:, HEADS + KV_HEADS:]
                q = torch.empty(len(x), HEADS, DIM, dtype=torch.bfloat16, device="cuda")
                self.step.append(layer, y[:, :HEADS], k, v, q_out=q)
                o = torch.empty(len(x), HEADS, DIM, device="cuda")
                self.step.attend(layer, q, out=o)
                x = x + self.project(self.o[layer], o.view(len(x), -1))
                kept.append((k, v))
            best = (torch.nn.functional.rms_norm(x, (HIDDEN,)) @ self.embed.T).argmax(-1)
        self.step.status()
        best, out, at = best.tolist(), [], 0
        for m in rows:
            out.append(best[at:at + m])
            at += m
        return out, kept

    def commit(self, tables, kv_len, accepted, rows, kept):
        """Stores the accepted rows of every tree at their final slots."""
        src, at = [], 0
        for a, m in zip(accepted, rows):
            src += [at + i for i in a]
            at += m
        with self.torch.cuda.stream(self.stream):
            self.step.plan(kv_len, [len(a) for a in accepted], tables, src_rows=src)
            for layer, (k, v) in enumerate(kept):
                self.step.append(layer, None, k, v)


def plain(server: Server, prompts, n_new: int):
    tables = [[] for _ in prompts]
    seqs = [list(p) for p in prompts]
    out, _ = server.forward(tables, [0] * len(seqs), seqs)
    for s, o in zip(seqs, out):
        s.append(o[-1])
    for _ in range(n_new - 1):
        out, _ = server.forward(tables, [len(s) - 1 for s in seqs], [[s[-1]] for s in seqs])
        for s, o in zip(seqs, out):
            s.append(o[0])
    return seqs


def with_trees(server: Server, prompts, n_new: int, guess):
    """guess(sequence number, tokens so far, depth) -> two candidates a level."""
    tables = [[] for _ in prompts]
    seqs = [list(p) for p in prompts]
    out, _ = server.forward(tables, [0] * len(seqs), seqs)
    for s, o in zip(seqs, out):
        s.append(o[-1])
    steps = 0
    while min(len(s) - len(p) for s, p in zip(seqs, prompts)) < n_new:
        trees = []
        for b, s in enumerate(seqs):
            tok, par, parent = [s[-1]], [0], 0
            for depth in range(3):
                pair = guess(b, s, depth)
                par += [parent, parent]
                tok += pair
                parent = len(tok) - 2
            trees.append(pkg.DraftTree(tok, par))
        kv = [len(s) - 1 for s in seqs]
        out, kept = server.forward(tables, kv, [t.tokens() for t in trees],
                                   positions=[p for t, n in zip(trees, kv) for p in t.position_ids(n)],
                                   masks=[m for t in trees for m in t.ancestor_bits()])
        accepted = []
        for s, t, o in zip(seqs, trees, out):
            node, path = 0, [0]
            while True:
                nxt = [i for i in range(1, len(t)) if t.parent_of(i) == node and t.token_at(i) == o[node]]
                if not nxt:
                    break
                node = nxt[0]
                path.append(node)
            s += [t.token_at(i) for i in path[1:]] + [o[node]]
            accepted.append(path)
        server.commit(tables, kv, accepted, [len(t) for t in trees], kept)
        steps += 1
    return seqs, steps


def run(n_new: int = 24):
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (5, 40, 17, 70)]
    want = plain(Server(), prompts, n_new + 4)

    def guess(b, s, depth):  # the right token two times out of three, in first or second place
        at = len(s) + depth
        right = want[b][at] if at < len(want[b]) else 0
        wrong = int(rng.integers(0, VOCAB))
        return [[right, wrong], [wrong, right], [wrong, (wrong + 1) % VOCAB]][int(rng.integers(0, 3))]

    got, steps = with_trees(Server(), prompts, n_new, guess)
    same = all(g[:len(p) + n_new] == w[:len(p) + n_new] for g, w, p in zip(got, want, prompts))
    return same, steps, sum(len(g) - len(p) for g, p in zip(got, prompts)) / len(prompts)


if __name__ == "__main__":
    same, steps, tokens = run()
    print(f"{tokens:.1f} tokens a sequence in {steps} steps; equal to one token a step: {same}")
    sys.exit(0 if same else 1)
