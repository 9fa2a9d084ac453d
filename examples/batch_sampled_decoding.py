"""Sampled speculative decoding of several requests at once, each with its own adapter.

A small seeded model of the last token (an embedding, one Q8_0 projection with
low-rank adapters beside it, a Q8_0 head) serves a batch of requests; its draft
model is the same without the adapters.  A round draws a few tokens a request
from the draft (sample_rows, which keeps the rows they were drawn from), runs the
target over all of them (spec_qmatmul and LoraBank.apply) and accepts them
(verify_drafts).  With trees, the draft's two likeliest tokens a level are picked
instead and verify_trees walks them.  Decisions stay on the device; the host
reads each round's tokens.

    python examples/batch_sampled_decoding.py
"""

import importlib
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
pkg = importlib.import_module("abyo-speculate_b200")
synth = importlib.import_module("abyo-speculate_b200.gguf_synth")

Q8_0 = 8
HIDDEN, WIDE, VOCAB, RANK, ADAPTERS, DRAFTS, LEVELS = 256, 768, 1024, 16, 4, 4, 3


class Server:
    def __init__(self, adapters, seed: int = 0):
        """adapters: the request's adapter, -1 for none, by request."""
        import torch
        self.torch = torch
        rng = np.random.default_rng(seed)

        def weight(rows, cols, sigma):
            w = (rng.standard_normal((rows, cols)) * sigma).astype(np.float32)
            return pkg.QWeight(Q8_0, synth.quantize(w, Q8_0), rows, cols)

        def normal(*shape):
            return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda()

        self.up, self.head = weight(WIDE, HIDDEN, HIDDEN ** -0.5), weight(VOCAB, WIDE, 2.5 * WIDE ** -0.5)
        self.embed = normal(VOCAB, HIDDEN)
        self.bank = pkg.LoraBank((normal(ADAPTERS, RANK, HIDDEN) * HIDDEN ** -0.5).bfloat16(),
                                 (normal(ADAPTERS, WIDE, RANK) * 0.5 * RANK ** -0.5).bfloat16(),
                                 scales=rng.uniform(0.3, 0.9, ADAPTERS))
        self.adapters, self.n = list(adapters), len(adapters)
        self.plans = {}  # by rows a request
        self.uniforms = torch.Generator(device="cuda").manual_seed(seed + 1)
        self.stream = torch.cuda.Stream()
        torch.cuda.synchronize()

    def project(self, w, x):
        """x [rows, cols] f32 -> x . W^T, 64 rows a call."""
        y = self.torch.empty(x.shape[0], w.n_rows, device="cuda")
        for a in range(0, x.shape[0], 64):
            part = x[a:a + 64]
            w.matmul(part.data_ptr(), part.shape[0], y[a:].data_ptr(), self.stream.cuda_stream)
        return y

    def draft(self, tokens):
        return self.project(self.head, self.project(self.up, self.embed[tokens]))

    def target(self, tokens):
        """Logits of tokens [requests, rows], by rows; and the projection with the adapters, for a test."""
        per = tokens.shape[1]
        if per not in self.plans:
            self.plans[per] = pkg.LoraPlan([a for a in self.adapters for _ in range(per)], ADAPTERS)
        x = self.embed[tokens.reshape(-1)]
        y = self.bank.apply(self.plans[per], x, self.project(self.up, x))
        return self.project(self.head, y), y

    def rand(self, *shape):
        return self.torch.rand(*shape, device="cuda", generator=self.uniforms)

    def starts(self, per: int):
        return self.torch.arange(0, self.n * per + 1, per, dtype=self.torch.int32, device="cuda")

    def chain_round(self, last, temperature):
        """One round from tokens `last` [requests]: what verify_drafts took and gave."""
        torch, per = self.torch, DRAFTS + 1
        rows = torch.empty(self.n, per, dtype=torch.int32, device="cuda")  # a request's last token and its drafts
        rows[:, 0] = last
        q = torch.empty(self.n, per, VOCAB, device="cuda")
        for i in range(DRAFTS):
            rows[:, i + 1] = pkg.sample_rows(self.draft(rows[:, i]), self.rand(self.n), temperature, probs_out=q[:, i])
        drafts = torch.full_like(rows, -1)
        drafts[:, :-1] = rows[:, 1:]
        logits, wide = self.target(rows)
        u = self.rand(self.n * per)
        n, token = pkg.verify_drafts(logits, drafts.view(-1), q.view(-1, VOCAB), u, self.starts(per), temperature)
        return {"rows": rows, "drafts": drafts, "q": q, "logits": logits, "wide": wide, "u": u, "n": n, "token": token}

    def tree_round(self, last, temperature):
        """The same with trees: two candidates a level, the first of which has children."""
        torch, per = self.torch, 2 * LEVELS + 1
        rows = torch.empty(self.n, per, dtype=torch.int32, device="cuda")
        rows[:, 0] = last
        parents = [0]
        for level in range(LEVELS):
            up = max(2 * level - 1, 0)
            rows[:, 2 * level + 1:2 * level + 3] = self.draft(rows[:, up]).topk(2).indices
            parents += [up, up]
        parents = torch.tensor(parents * self.n, dtype=torch.int32, device="cuda")
        logits, wide = self.target(rows)
        u = self.rand(self.n * per)
        path, n, token = pkg.verify_trees(logits, rows.view(-1), parents, u, self.starts(per), temperature)
        return {"rows": rows, "parents": parents, "logits": logits, "wide": wide, "u": u, "path": path, "n": n, "token": token}


def run(n_new: int = 24, requests: int = 12, temperature: float = 0.8, trees: bool = False, seed: int = 0):
    """Tokens of every request, and the rounds they took."""
    server = Server([i % (ADAPTERS + 1) - 1 for i in range(requests)], seed)
    torch = server.torch
    with torch.cuda.stream(server.stream):
        last = torch.arange(requests, device="cuda", dtype=torch.int32)
        seqs, rounds = [[i] for i in range(requests)], 0
        while min(len(s) for s in seqs) <= n_new:
            rounds += 1
            r = server.tree_round(last, temperature) if trees else server.chain_round(last, temperature)
            last, rows = r["token"], r["rows"].tolist()
            per = len(rows[0])
            path = r["path"].view(-1, per).tolist() if trees else None
            for b, (s, n, t) in enumerate(zip(seqs, r["n"].tolist(), r["token"].tolist())):
                s += ([rows[b][i] for i in path[b][1:n]] if trees else rows[b][1:n + 1]) + [t]
        for plan in server.plans.values():
            plan.status()
    return seqs, rounds


def main():
    for trees in (False, True):
        seqs, rounds = run(trees=trees)
        new = sum(len(s) - 1 for s in seqs)
        print(f"{'trees' if trees else 'chains'}: {new} tokens of {len(seqs)} requests in {rounds} rounds")


if __name__ == "__main__":
    main()
