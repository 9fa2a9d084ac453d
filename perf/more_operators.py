"""Timed cases of a serving batch's operators around the verify step.

  sample   a token per row of logits from softmax(logits / temperature) and a
           given uniform number, with the row's probabilities where the next
           verification needs them (a draft step, or plain sampling)
  chain    drafted tokens of several sequences against the target's rows:
           accept draft i while u q_i <= p_i, then draw from max(p - q, 0) or
           from p behind the last draft
  tree     draft trees of several sequences whose candidates were picked, not
           drawn: the token drawn at a node leads to the child that holds it
  lora     low-rank adapters of many requests beside a shared projection's
           output: y + scale (x A^T) B^T with each row's own A and B

``run`` computes an operator in plain torch operations, or through the
package's entry points when ``own`` is true.  The probabilities, their sums
and every comparison with a uniform number are taken in 64 bits in the plain
form: a token is the first whose cumulative weight passes u times the row's,
and next to such a border 32 bits pick the neighbour.  Vocabularies and widths
are the repository's benchmark shapes (Llama-3-8B, Qwen2.5-7B and -0.5B).
"""

import importlib
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _rows_case(name, kind, vocab, dtype, seqs, rows, probs=False, greedy=0.0, pad=0, spread=2.0, shape=1):
    """Logits rows: seqs sequences of rows[0]..rows[1] rows; `greedy` of them at temperature 0; `pad` columns behind
    the vocabulary in each stored row; `spread`: standard deviation of the ordinary tokens' logits."""
    c = {"kind": kind, "vocab": vocab, "dtype": dtype, "seqs": seqs, "rows_min": rows[0], "rows_max": rows[1],
         "probs": probs, "greedy": greedy, "pad": pad, "spread": spread, "shape": shape}
    return {"name": name, **c} if name else c


def _lora_case(name, k, n, dtype, rank, bank, seqs, rows, x_f32=False, y_f32=False, mixed=False, none=0.0, shape=1):
    """seqs requests of rows[0]..rows[1] rows with adapters drawn from a bank of `bank` of rank `rank` (`mixed`: of
    ranks from 1 to `rank`); `none` of the requests have no adapter."""
    c = {"kind": "lora", "in": k, "out": n, "dtype": dtype, "rank": rank, "bank": bank, "seqs": seqs,
         "rows_min": rows[0], "rows_max": rows[1], "x_f32": x_f32, "y_f32": y_f32, "mixed": mixed, "none": none,
         "shape": shape}
    return {"name": name, **c} if name else c


def listed():
    return [
        # The next token of one sequence from the f32 row that the model returns: launch latency.
        _rows_case("sample_1", "sample", 128256, "f32", 1, (1, 1)),
        # One draft step of 64 sequences: tokens, and the rows q that their verification will need.
        _rows_case("sample_64_probs", "sample", 128256, "bf16", 64, (1, 1), probs=True, greedy=0.1),
        # Plain sampling of 192 requests over a vocabulary of odd size, rows behind one another.
        _rows_case("sample_192_odd", "sample", 151937, "f16", 192, (1, 1), spread=3.0),
        # The framework's headline step: k = 4 drafts of one sequence.
        _rows_case("chain_1x5", "chain", 128256, "f32", 1, (5, 5)),
        # k = 8 drafts at most of 24 sequences, some with fewer, stored rows padded.
        _rows_case("chain_24x9", "chain", 151936, "f32", 24, (2, 9), greedy=0.1, pad=128),
        # A full serving batch, k = 4.
        _rows_case("chain_64x5", "chain", 128256, "bf16", 64, (5, 5)),
        # The 60-node draft tree.
        _rows_case("tree_1x60", "tree", 128256, "f32", 1, (60, 60)),
        # Trees of 16 sequences in a batch.
        _rows_case("tree_16x31", "tree", 152064, "bf16", 16, (8, 31), greedy=0.2),
        # One token of one request beside the attention's output projection.
        _lora_case("lora_1", 4096, 4096, "bf16", 16, 8, 1, (1, 1)),
        # One token each of 64 requests, adapters of mixed ranks, beside the gate projection (Qwen2.5-7B).
        _lora_case("lora_64x1", 3584, 18944, "f16", 32, 64, 64, (1, 1), y_f32=True, mixed=True, none=0.1),
        # Verify rows of 24 requests in f32, as the quantized matmul takes and returns them, and trees of 60 among them.
        _lora_case("lora_24_verify", 4096, 14336, "bf16", 16, 20, 24, (5, 60), x_f32=True, y_f32=True),
        # Prompt rows of three requests of rank 64 beside the down projection.
        _lora_case("lora_8192", 14336, 4096, "bf16", 64, 4, 3, (2500, 2900)),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["sample", "chain", "tree", "lora", "lora"])
    shape = rng.randrange(1, 1 << 20)
    dtype = rng.choice(["bf16", "f16", "f32"])
    if kind == "lora":
        k, n = rng.choice([(4096, 4096), (4096, 14336), (14336, 4096), (3584, 18944), (896, 4864), (2048, 8192),
                           (log_int(100, 5000), log_int(100, 5000))])
        form = rng.choice(["token", "verify", "chunk"])
        if form == "token":
            seqs, rows = log_int(1, 128), (1, 1)
        elif form == "verify":
            r0 = rng.randrange(2, 10)
            seqs, rows = log_int(1, 48), (r0, r0 + rng.choice([0, 3, 50]))
        else:
            r0 = log_int(70, 2000)
            seqs, rows = rng.randrange(1, 4), (r0, r0 + rng.randrange(0, 500))
        return _lora_case(None, k, n, rng.choice(["bf16", "f16"]), rng.choice([4, 8, 16, 24, 32, 64]),
                          rng.randrange(1, 65), seqs, rows, rng.random() < 0.4, rng.random() < 0.4,
                          rng.random() < 0.4, rng.choice([0.0, 0.2]), shape)
    vocab = rng.choice([128256, 151936, 152064, log_int(1000, 152000)])
    if kind == "sample":
        seqs, rows = log_int(1, 192), (1, 1)
    elif kind == "chain":
        r1 = rng.randrange(2, 10)
        seqs, rows = log_int(1, 32), (rng.randrange(1, r1 + 1), r1)
    else:
        r1 = rng.randrange(3, 61)
        seqs, rows = max(1, log_int(1, 480) // r1), (rng.randrange(2, r1 + 1), r1)
    return _rows_case(None, kind, vocab, dtype, seqs, rows, kind == "sample" and rng.random() < 0.5,
                      rng.choice([0.0, 0.3]), rng.choice([0, 0, 64, 1]), rng.uniform(1.0, 3.0), shape)


def _shape(c):
    """Rows of each sequence (the same for every seed)."""
    r = random.Random(c["shape"] * 7919 + 13)
    rows = [r.randint(c["rows_min"], c["rows_max"]) for _ in range(c["seqs"])]
    if c["kind"] == "lora":
        most = c["bank"]
        adapters = [-1 if r.random() < c["none"] else r.randrange(most) for _ in rows]
        ranks = [r.randint(1, c["rank"]) if c["mixed"] else c["rank"] for _ in range(most)]
        return rows, adapters, ranks
    parents = []
    for m in rows:
        parents.append([0] + [r.randrange(max(0, i - 10), i) for i in range(1, m)])  # BFS order, at most 10 candidates
    return rows, parents


def work(c):
    if c["kind"] == "lora":
        rows, adapters, ranks = _shape(c)
        size = 2
        b = f = 0
        for a in {a for a in adapters if a >= 0}:
            b += ranks[a] * (c["in"] + c["out"]) * size
        for m, a in zip(rows, adapters):
            b += 2 * m * c["out"] * (4 if c["y_f32"] else 2)  # y in and out
            if a >= 0:
                b += m * c["in"] * (4 if c["x_f32"] else 2)
                f += 2 * m * ranks[a] * (c["in"] + c["out"])
        return {"bytes": b, "flops": f}
    rows, _ = _shape(c)
    v, size = c["vocab"], 4 if c["dtype"] == "f32" else 2
    b = sum(rows) * v * size
    if c["probs"]:
        b += sum(rows) * v * 4
    if c["kind"] == "chain":
        b += len(rows) * v * 4  # the draft's row at the first rejection
    return {"bytes": b, "flops": sum(rows) * v * 4}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _prepare_lora(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rows, adapters, ranks = _shape(c)
    k, n, r, dt = c["in"], c["out"], c["rank"], DTYPES[c["dtype"]]
    total = sum(rows)

    def normal(*size):
        return torch.randn(*size, device=DEV, generator=gen)

    ids = [a for m, a in zip(rows, adapters) for _ in range(m)]
    st = {"case": c, "ids": torch.tensor(ids, device=DEV), "bank": c["bank"], "ranks": torch.tensor(ranks, device=DEV)}
    st["a"] = (normal(c["bank"], r, k) / math.sqrt(k)).to(dt)
    st["b"] = (normal(c["bank"], n, r) * 0.3 / math.sqrt(r)).to(dt)
    st["scales"] = 0.5 + 1.5 * torch.rand(c["bank"], device=DEV, generator=gen)
    # Activations: normal, with a few strong channels.
    x = normal(total, k) * (1 + 8 * (torch.rand(1, k, device=DEV, generator=gen) < 0.01))
    st["x"] = x.to(torch.float32 if c["x_f32"] else dt)
    st["y"] = normal(total, n).to(torch.float32 if c["y_f32"] else dt)
    if own:
        pkg = importlib.import_module("abyo-speculate_b200")
        st["bank_own"] = pkg.LoraBank(st["a"], st["b"], ranks=ranks, scales=st["scales"])
        st["plan"] = pkg.LoraPlan(ids, c["bank"], device=DEV)
        st["out"] = torch.empty_like(st["y"])
    return st


def prepare(c, seed):
    if c["kind"] == "lora":
        return _prepare_lora(c, seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rows, parents = _shape(c)
    total, v, dt = sum(rows), c["vocab"], DTYPES[c["dtype"]]

    def rand(*size):
        return torch.rand(*size, device=DEV, generator=gen)

    # Logits as a language model's: most tokens normal, a few of them far above (most of the mass).
    x = c["spread"] * torch.randn(total, v, device=DEV, generator=gen)
    x.scatter_add_(1, torch.randint(0, v, (total, 24), device=DEV, generator=gen), 4 * c["spread"] + 4 + 5 * rand(total, 24))
    store = torch.empty(total, v + c["pad"], dtype=dt, device=DEV)
    store[:, v:] = 50.0  # what lies behind the vocabulary is no token
    logits = store[:, :v]
    logits.copy_(x)
    temp = 0.6 + 0.6 * rand(len(rows))
    temp[rand(len(rows)) < c["greedy"]] = 0.0
    seq = torch.tensor([b for b, m in enumerate(rows) for _ in range(m)], device=DEV)
    idx = torch.tensor([i for m in rows for i in range(m)], device=DEV)
    start = [0]
    for m in rows:
        start.append(start[-1] + m)
    st = {"case": c, "logits": logits, "temp": temp[seq].contiguous(), "u": (rand(total) * (1 << 24)).floor() / (1 << 24),
          "seq": seq, "idx": idx, "max_rows": max(rows), "rows": torch.tensor(rows, device=DEV),
          "start": torch.tensor(start, dtype=torch.int32, device=DEV)}
    if c["kind"] == "chain":
        # A draft model that mostly agrees: its logits are the target's and some noise (greedy rows: all on one token).
        noise = 0.7 * torch.randn(total, v, device=DEV, generator=gen)
        t = torch.where(st["temp"] > 0, st["temp"], 1e-4)[:, None]
        st["q"] = torch.softmax((x + noise) / t, -1)
        race = st["q"] / -torch.log(rand(total, v).clamp_min(1e-30))
        st["drafts"] = race.argmax(-1).to(torch.int32)
    if c["kind"] == "tree":
        # The candidates under a node are its row's best tokens in order.
        best = x.topk(12, -1).indices
        tokens, at = [], 0
        for m, ps in zip(rows, parents):
            seen = [0] * m
            tokens.append((at, 0))
            for p in ps[1:]:
                tokens.append((at + p, seen[p]))
                seen[p] += 1
            at += m
        tokens = torch.tensor(tokens, device=DEV)
        st["tokens"] = best[tokens[:, 0], tokens[:, 1]].to(torch.int32)
        st["parents"] = torch.tensor([p for ps in parents for p in ps], dtype=torch.int32, device=DEV)
    if own:
        st["pkg"] = importlib.import_module("abyo-speculate_b200")
        st["probs_out"] = torch.empty(total, v, device=DEV) if c["probs"] else None
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _weights(logits, temp):
    """Unnormalised probabilities in 64 bits; temperature 0: the first largest logit alone."""
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    t = temp.double()[:, None]
    w = torch.exp((x - top) / torch.where(t > 0, t, 1.0))
    at = torch.arange(x.shape[1], device=DEV)
    first = torch.where(x == top, at, x.shape[1]).amin(-1, keepdim=True)
    return torch.where(t > 0, w, (at == first).double())


def _draw(w, u):
    """The first token whose cumulative weight passes u times the row's."""
    c = w.cumsum(-1)
    pick = (c <= u.double()[:, None] * c[:, -1:]).sum(-1)
    at = torch.arange(w.shape[1], device=DEV)
    return torch.minimum(pick, torch.where(w > 0, at, -1).amax(-1)).to(torch.int32)


def _plain_sample(st):
    w = _weights(st["logits"], st["temp"])
    token = _draw(w, st["u"])
    return [token, (w / w.sum(-1, keepdim=True)).float()] if st["case"]["probs"] else [token]


def _plain_chain(st):
    rows, start = st["rows"], st["start"][:-1].long()
    w = _weights(st["logits"], st["temp"])
    p = w / w.sum(-1, keepdim=True)
    d = st["drafts"].long()[:, None]
    ok = st["u"].double() * st["q"].gather(1, d)[:, 0].double() <= p.gather(1, d)[:, 0]
    grid = torch.zeros(len(rows), st["max_rows"], dtype=torch.long, device=DEV)
    grid[st["seq"], st["idx"]] = (ok & (st["idx"] < rows[st["seq"]] - 1)).long()
    n = grid.cumprod(-1).sum(-1)
    last = start + n
    rejected = n < rows - 1
    rest = (p[last] - st["q"][last].double()).clamp_min(0.0)
    rest = torch.where((rejected & (rest.sum(-1) > 0))[:, None], rest, p[last])
    return [n.to(torch.int32), _draw(rest, st["u"][last + rejected])]


def _plain_tree(st):
    rows, m = st["rows"], st["max_rows"]
    drawn = _draw(_weights(st["logits"], st["temp"]), st["u"])

    def grid(x, fill):
        g = torch.full((len(rows), m), fill, dtype=torch.long, device=DEV)
        g[st["seq"], st["idx"]] = x.long()
        return g

    token, parent, pick = grid(st["tokens"], -1), grid(st["parents"], 0), grid(drawn, -2)
    i = torch.arange(m, device=DEV)
    twin = (token[:, :, None] == token[:, None]) & (parent[:, :, None] == parent[:, None]) & (i[:, None] > i) & (i > 0)
    hit = (token == pick.gather(1, parent)) & ~twin.any(-1)
    hit[:, 0] = True
    # Taken: a node that is hit, with all its ancestors.  hop doubles the reach of each step towards the root.
    hop, taken = parent, hit
    for _ in range(max(1, (m - 1).bit_length())):
        taken = taken & taken.gather(1, hop)
        hop = hop.gather(1, hop)
    n = taken.sum(-1)
    order = torch.where(taken, i, m).sort(-1).values
    path = torch.where(order < m, order, -1)
    deepest = order.gather(1, n[:, None] - 1)
    return [path[st["seq"], st["idx"]].to(torch.int32), n.to(torch.int32), pick.gather(1, deepest)[:, 0].to(torch.int32)]


def _plain_lora(st):
    bank, r = st["bank"], st["case"]["rank"]
    # Every row against every adapter; the others' ranks count nothing.
    t = (st["x"].float() @ st["a"].float().flatten(0, 1).T).view(-1, bank, r)
    live = (torch.arange(bank, device=DEV) == st["ids"][:, None])[..., None] & \
        (torch.arange(r, device=DEV) < st["ranks"][:, None])
    t = torch.where(live, t * st["scales"][:, None], 0.0)
    y = st["y"].float() + t.flatten(1) @ st["b"].float().transpose(0, 1).flatten(1).T
    return y.to(st["y"].dtype)


def run(st):
    kind = st["case"]["kind"]
    if not own:
        return {"sample": _plain_sample, "chain": _plain_chain, "tree": _plain_tree, "lora": _plain_lora}[kind](st)
    if kind == "lora":
        return st["bank_own"].apply(st["plan"], st["x"], st["y"], out=st["out"])
    pkg = st["pkg"]
    if kind == "sample":
        token = pkg.sample_rows(st["logits"], st["u"], st["temp"], probs_out=st["probs_out"])
        return [token, st["probs_out"]] if st["probs_out"] is not None else [token]
    if kind == "chain":
        return list(pkg.verify_drafts(st["logits"], st["drafts"], st["q"], st["u"], st["start"], st["temp"]))
    return list(pkg.verify_trees(st["logits"], st["tokens"], st["parents"], st["u"], st["start"], st["temp"]))


# ---------------------------------------------------------------------------
# The definitions in 64 bits, row by row
# ---------------------------------------------------------------------------
def _row_probs(st, r):
    x, t = st["logits"][r].double(), float(st["temp"][r])
    if t == 0.0:
        p = torch.zeros_like(x)
        p[int((x == x.max()).nonzero()[0])] = 1.0
        return p
    x = x / t
    return torch.exp(x - torch.logsumexp(x, 0))


def _row_token(p, u):
    c = torch.cumsum(p, 0)
    at = int(torch.searchsorted(c, float(u) * float(c[-1]), right=True))
    return min(at, int(p.nonzero()[-1]))


def _exact_chain(st):
    ns, tokens = [], []
    start, u = st["start"].tolist(), st["u"].tolist()
    for a, b in zip(start[:-1], start[1:]):
        n = 0
        while True:
            p = _row_probs(st, a + n)
            if n == b - a - 1:
                tokens.append(_row_token(p, u[a + n]))
                break
            q, d = st["q"][a + n].double(), int(st["drafts"][a + n])
            if float(q[d]) <= 0 or u[a + n] <= float(p[d] / q[d]):
                n += 1
                continue
            rest = torch.relu(p - q)
            tokens.append(_row_token(rest if float(rest.sum()) > 0 else p, u[a + n + 1]))
            break
        ns.append(n)
    return [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (ns, tokens)]


def _exact_tree(st):
    start, u = st["start"].tolist(), st["u"].tolist()
    token, parent = st["tokens"].tolist(), st["parents"].tolist()
    path, ns, last = [], [], []
    for a, b in zip(start[:-1], start[1:]):
        way = [0]
        while True:
            drawn = _row_token(_row_probs(st, a + way[-1]), u[a + way[-1]])
            below = [i for i in range(1, b - a) if parent[a + i] == way[-1] and token[a + i] == drawn]
            if not below:
                break
            way.append(below[0])
        path += way + [-1] * (b - a - len(way))
        ns.append(len(way))
        last.append(drawn)
    return [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (path, ns, last)]


def _exact_lora(st):
    y = st["y"].double()
    for i in st["ids"].unique().tolist():
        if i < 0:
            continue
        at = (st["ids"] == i).nonzero()[:, 0]
        r = int(st["ranks"][i])
        a, b = st["a"][i, :r].double(), st["b"][i, :, :r].double()
        y[at] += float(st["scales"][i]) * ((st["x"][at].double() @ a.T) @ b.T)
    return y


def exact(c, seed):
    st = prepare(c, seed)
    if c["kind"] == "lora":
        return _exact_lora(st)
    if c["kind"] == "chain":
        return _exact_chain(st)
    if c["kind"] == "tree":
        return _exact_tree(st)
    probs = [_row_probs(st, r) for r in range(st["logits"].shape[0])]
    token = torch.tensor([_row_token(p, u) for p, u in zip(probs, st["u"].tolist())], dtype=torch.int32, device=DEV)
    return [token, torch.stack(probs)] if c["probs"] else [token]
