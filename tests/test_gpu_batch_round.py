"""A round of a batch as it is used: shared projection, adapters, draft sampling, verification, against float64.

The projection with its adapters is compared by the bound that tests/test_gpu_lora.py
derives, from the projection's own f32 result; decisions are equal to
those of tests/batch_ref.py on the logits that the round computed."""

import importlib.util
import os

import numpy as np
import pytest

import batch_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "batch_sampled_decoding.py")
    spec = importlib.util.spec_from_file_location("batch_sampled_decoding", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def server(example, requests=9, seed=3):
    return example.Server([i % (example.ADAPTERS + 1) - 1 for i in range(requests)], seed)


def f64(t):
    return t.double().cpu().numpy()


def check_adapters(s, example, r):
    """r["wide"] against the shared projection's f32 result plus the adapters in float64."""
    per = r["rows"].shape[1]
    x = s.embed[r["rows"].reshape(-1)]
    y = s.project(s.up, x)
    s.stream.synchronize()
    a, b = f64(s.bank._keep[0]), f64(s.bank._keep[1])
    scales, x, y, got = f64(s.bank._keep[3]), f64(x), f64(y), f64(r["wide"])
    for row in range(len(x)):
        i = s.adapters[row // per]
        if i < 0:
            assert (got[row] == y[row]).all()
            continue
        t = scales[i] * (a[i] @ x[row])
        want = y[row] + b[i] @ t
        k, rank = a.shape[2], a.shape[1]
        dt = scales[i] * (np.abs(a[i]) @ np.abs(x[row])) * (2.0 ** -23 * (k / 8 + 32) + 2.0 ** -23) + np.abs(t) * (2.0 ** -22 + 2.0 ** -23)
        bound = np.abs(b[i]) @ dt + 2.0 ** -23 * (rank / 8 + 16) * (np.abs(b[i]) @ np.abs(t))
        assert (np.abs(got[row] - want) <= bound + 2.0 ** -24 * (np.abs(want) + bound)).all()


@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.3])
def test_chain_rounds(example, temperature):
    s = server(example)
    torch = s.torch
    with torch.cuda.stream(s.stream):
        last = torch.arange(s.n, device="cuda", dtype=torch.int32) * 7
        for _ in range(3):
            r = s.chain_round(last, temperature)
            check_adapters(s, example, r)
            per = example.DRAFTS + 1
            logits, q, drafts, u = f64(r["logits"]), r["q"].cpu().numpy().reshape(-1, example.VOCAB), r["drafts"].view(-1).tolist(), r["u"].tolist()
            want = [ref.chain(logits, drafts, q, u, [temperature] * len(u), b * per, (b + 1) * per, len(u)) for b in range(s.n)]
            assert list(zip(r["n"].tolist(), r["token"].tolist())) == want
            last = r["token"]


@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.3])
def test_tree_rounds(example, temperature):
    s = server(example)
    torch = s.torch
    with torch.cuda.stream(s.stream):
        last = torch.arange(s.n, device="cuda", dtype=torch.int32) * 5
        for _ in range(3):
            r = s.tree_round(last, temperature)
            check_adapters(s, example, r)
            per = 2 * example.LEVELS + 1
            logits, tokens, parents, u = f64(r["logits"]), r["rows"].view(-1).tolist(), r["parents"].tolist(), r["u"].tolist()
            path = r["path"].view(-1, per).tolist()
            for b, (n, t) in enumerate(zip(r["n"].tolist(), r["token"].tolist())):
                want, token = ref.tree(logits, tokens, parents, u, [temperature] * len(u), b * per, (b + 1) * per, len(u))
                assert path[b] == want + [-1] * (per - len(want)) and (n, t) == (len(want), token)
            last = r["token"]


@pytest.mark.parametrize("trees", [False, True])
def test_example_runs(example, trees):
    seqs, rounds = example.run(n_new=8, requests=5, trees=trees)
    assert rounds <= 8 and all(len(s) > 8 and all(0 <= t < example.VOCAB for t in s) for s in seqs)


def test_first_level_is_replayed_from_a_graph(example):
    """Draft step, adapters and verification captured once, replayed on new tokens and uniforms."""
    s = server(example)
    torch, per = s.torch, 3
    with torch.cuda.stream(s.stream):
        tokens = torch.zeros(s.n * per, dtype=torch.int32, device="cuda")
        u, u0 = s.rand(s.n * per), s.rand(s.n * per)
        base, x = torch.empty(s.n * per, example.VOCAB, device="cuda"), torch.empty(s.n * per, example.HIDDEN, device="cuda")
        wide, logits, q = torch.empty(s.n * per, example.WIDE, device="cuda"), torch.empty(s.n * per, example.VOCAB, device="cuda"), torch.empty(s.n * per, example.VOCAB, device="cuda")
        plan, start = pkg_of(example).LoraPlan([a for a in s.adapters for _ in range(per)], example.ADAPTERS), s.starts(per)
        out = torch.empty_like(wide)

        def device_part():
            drafts = pkg_of(example).sample_rows(base, u0, 0.9, probs_out=q)
            s.bank.apply(plan, x, wide, out=out)
            return drafts, pkg_of(example).verify_drafts(logits, drafts, q, u, start, 0.9)

        def inputs(seed):
            g = torch.Generator(device="cuda").manual_seed(seed)
            tokens.copy_(torch.randint(0, example.VOCAB, tokens.shape, device="cuda", generator=g, dtype=torch.int32))
            u.copy_(torch.rand(u.shape, device="cuda", generator=g))
            u0.copy_(torch.rand(u.shape, device="cuda", generator=g))
            x.copy_(s.embed[tokens])
            wide.copy_(s.project(s.up, x))
            base.copy_(s.draft(tokens))
            logits.copy_(base + 0.5 * torch.randn(base.shape, device="cuda", generator=g))

        inputs(0)
        device_part()
        s.stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s.stream):
            drafts, (n, token) = device_part()
        for seed in (1, 2):
            inputs(seed)
            graph.replay()
            s.stream.synchronize()
            got, kept = (drafts.tolist(), n.tolist(), token.tolist()), out.clone()
            want, (wn, wt) = device_part()
            assert got == (want.tolist(), wn.tolist(), wt.tolist()) and torch.equal(kept, out)
            lg, qn, un = f64(logits), q.cpu().numpy(), u.tolist()
            assert list(zip(got[1], got[2])) == [ref.chain(lg, got[0], qn, un, [0.9] * len(un), b * per, (b + 1) * per, len(un)) for b in range(s.n)]


def pkg_of(example):
    return example.pkg
