"""Verification of drafted tokens against its definition in 64 bits (draft_reference.py)."""
import numpy as np
import pytest

import draft_reference as ref
from test_gpu_fp4_cache import dev

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24  # the probability is rounded to f32 once


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def inputs(rng, nodes, vocab, mode, temperature, spread=2.5, liked=True):
    """Logits, tokens, parents, u and draft probabilities of a batch of trees whose drafts are good ones."""
    trees = [ref.grown(rng, n) for n in nodes]
    t = sum(nodes)
    logits = (rng.standard_normal((t, vocab)) * spread).astype(np.float32)
    if liked:
        for r in range(t):
            logits[r, rng.integers(0, vocab, 3)] += np.float32(12) + rng.standard_normal(3).astype(np.float32)
    heat = np.repeat(np.maximum(temperature, 0.3), nodes)[:, None]
    draft = softmax((logits + rng.standard_normal((t, vocab)) * 0.7) / heat).astype(np.float32)
    tokens, parents, at = np.zeros(t, np.int32), np.zeros(t, np.int32), 0
    for tree in trees:
        drawn = {}
        for i, p in enumerate(tree):
            parents[at + i] = p
            if p >= 0:
                if p not in drawn:
                    kids = tree.count(p)
                    q = draft[at + p].astype(np.float64)
                    if mode == "drawn":
                        drawn[p] = list(rng.choice(vocab, kids, p=q / q.sum()))
                    elif mode == "distinct" and np.count_nonzero(q) >= kids:
                        drawn[p] = list(rng.choice(vocab, kids, replace=False, p=q / q.sum()))
                    else:
                        drawn[p] = list(np.argsort(-q, kind="stable")[:kids]) + [0] * max(0, kids - vocab)
                tokens[at + i] = drawn[p].pop(0)
        at += len(tree)
    return dict(logits=logits, tokens=tokens, parents=parents, accept=rng.random(t).astype(np.float32),
                pick=rng.random(len(nodes)).astype(np.float32), probs=None if mode == "given" else draft)


def run(ctx, s, nodes, temperature, distinct=False, max_path=None, most=None, logits=None, probs=None):
    import torch

    n = len(nodes)
    max_path = max(max(nodes) - 1, 0) if max_path is None else max_path
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    out = [torch.full((n, max_path + 1), -9, dtype=torch.int32, device="cuda"),
           torch.full((n, max_path), -9, dtype=torch.int32, device="cuda"),
           torch.full((n,), -9, dtype=torch.int32, device="cuda"), torch.full((n,), -9.0, device="cuda")]
    ctx.verify_drafts(dev(s["logits"]) if logits is None else logits, dev(s["tokens"]), dev(s["parents"]), dev(cu),
                      max(max(nodes), 0) if most is None else most, dev(np.asarray(temperature, np.float32)), dev(s["accept"]),
                      dev(s["pick"]), (None if s["probs"] is None else dev(s["probs"])) if probs is None else probs, distinct, *out)
    return out


def check(out, s, nodes, temperature, distinct=False, max_path=None, what=""):
    tokens, path, count, prob = (x.cpu().numpy() for x in out)
    at = 0
    for b, n in enumerate(nodes):
        r = slice(at, at + n)
        want = ref.verify(s["logits"][r], s["tokens"][r], list(s["parents"][r]), temperature[b], s["accept"][r], s["pick"][b],
                          None if s["probs"] is None else s["probs"][r], distinct, max_path)
        got = tokens[b][tokens[b] >= 0].tolist(), path[b][path[b] >= 0].tolist()
        assert (got[0], got[1]) == (want[0], want[1]), (what, b, got, want[:2])
        assert count[b] == len(want[1]), (what, b)
        k = len(want[0])
        assert (tokens[b][k:] == -1).all() and (path[b][len(want[1]):] == -1).all(), (what, b)
        # rounded once, from sums that are exact to 1e-13
        assert abs(float(prob[b]) - want[2]) <= (HALF + 1e-11) * max(want[2], 1e-30), (what, b, prob[b], want[2])
        at += n


@pytest.mark.parametrize("mode", ["given", "drawn", "distinct"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 257, 4096, 4097, 8193, 32000, 128256])
def test_verify(gpu_ctx, mode, vocab):
    rng = np.random.default_rng(vocab + len(mode))
    nodes = [1, 8, 2, 5, 0, 13, 3, 6] if vocab > 10000 else [1, 8, 2, 5, 0, 33, 3, 70, 2, 9, 21, 4]
    temperature = rng.choice([0.0, 0.3, 0.7, 1.0, 1.5, -1.0], len(nodes))
    print(f"verify {mode} {vocab} {nodes}", flush=True)
    s = inputs(rng, nodes, vocab, mode, temperature)
    out = run(gpu_ctx, s, nodes, temperature, mode == "distinct")
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    check(out, s, nodes, temperature, mode == "distinct")
    again = run(gpu_ctx, s, nodes, temperature, mode == "distinct")
    assert all(bool((x == y).all()) for x, y in zip(out, again))


@pytest.mark.parametrize("mode", ["given", "drawn", "distinct"])
def test_flat_rows(gpu_ctx, mode):
    """Borders between tokens that lie 1e-5 and less apart, where sums of f32 weights would pick others."""
    rng = np.random.default_rng(31)
    nodes = [4] * 40
    temperature = np.full(40, 1.0)
    s = inputs(rng, nodes, 50000, mode, temperature, spread=0.5, liked=False)
    out = run(gpu_ctx, s, nodes, temperature, mode == "distinct")
    gpu_ctx.sync()
    check(out, s, nodes, temperature, mode == "distinct")


@pytest.mark.parametrize("mode", ["given", "drawn", "distinct"])
def test_wide_trees(gpu_ctx, mode):
    """Many children a node, tried one after the other, the largest tree among them."""
    rng = np.random.default_rng(8)
    nodes = [1024, 200, 65, 64]
    temperature = np.array([1.0, 0.7, 1.3, 1.0])
    s = inputs(rng, nodes, 500, mode, temperature, spread=1.0, liked=False)
    at = 0
    for n in nodes:  # half of the nodes behind the root
        for i in range(1, n):
            if i % 2:
                s["parents"][at + i] = 0
                s["tokens"][at + i] = rng.integers(0, 500)
        at += n
    out = run(gpu_ctx, s, nodes, temperature, mode == "distinct")
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    check(out, s, nodes, temperature, mode == "distinct")


@pytest.mark.parametrize("u", [0.0, 1e-7, 0.5, 1 - 2.0 ** -24, 1.0, np.nan])
@pytest.mark.parametrize("mode", ["given", "drawn"])
def test_ends_of_the_random_numbers(gpu_ctx, mode, u):
    rng = np.random.default_rng(12)
    nodes, temperature = [6, 6, 1, 4], np.array([1.0, 0.0, 0.5, 2.0])
    s = inputs(rng, nodes, 999, mode, temperature)
    s["accept"][:] = u
    s["pick"][:] = u
    out = run(gpu_ctx, s, nodes, temperature)
    gpu_ctx.sync()
    check(out, s, nodes, temperature)


def test_the_drafts_own_distribution_is_accepted(gpu_ctx):
    """q = p up to its rounding to f32: u below 1 - 1e-6 accepts, and a draft that never proposes what the
    model would say is rejected."""
    rng = np.random.default_rng(13)
    nodes, vocab = [5] * 8, 3000
    s = inputs(rng, nodes, vocab, "drawn", np.ones(8))
    s["probs"] = softmax(s["logits"].astype(np.float64)).astype(np.float32)
    s["accept"][:] = np.minimum(s["accept"], 1 - 1e-6)
    for i in range(1, 5):  # a path of drawn tokens
        s["parents"][i::5] = i - 1
        s["tokens"][i::5] = [rng.choice(vocab, p=p / p.sum()) for p in s["probs"][i - 1::5].astype(np.float64)]
    out = run(gpu_ctx, s, nodes, np.ones(8))
    gpu_ctx.sync()
    assert (out[2].cpu().numpy() == 4).all()
    check(out, s, nodes, np.ones(8))


@pytest.mark.parametrize("mode", ["given", "drawn", "distinct"])
def test_masked_and_far_logits(gpu_ctx, mode):
    """Logits of -inf (a top-k or top-p set), rows whose first thousands are masked, magnitudes at which weights leave f32
    and 64 bits, a vocabulary row that is all but one masked."""
    rng = np.random.default_rng(14)
    nodes, vocab = [5] * 8, 20000
    temperature = np.array([1.0, 1.0, 1.0, 0.01, 1.0, 0.0, 1e-9, 1.0])
    s = inputs(rng, nodes, vocab, mode, temperature)
    x = s["logits"].reshape(8, 5, vocab)
    keep = np.argsort(-x, -1)[..., :20]
    masked = np.full_like(x, -np.inf)
    np.put_along_axis(masked, keep, np.take_along_axis(x, keep, -1), -1)
    x[0] = masked[0]
    x[1, :, :vocab - 50] = -np.inf
    x[2] *= 40  # some hundred apart
    x[4] = x[4] * 1e4 - 3e5
    x[5] = masked[5]
    x[7] = -np.inf
    x[7, :, 12345] = -8.0
    s["tokens"].reshape(8, 5)[1, 1:] = vocab - 1 - np.arange(4)
    out = run(gpu_ctx, s, nodes, temperature, mode == "distinct")
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    check(out, s, nodes, temperature, mode == "distinct")


def test_rows_without_a_distribution(gpu_ctx):
    from ferrisinfer_amd import FerrisError

    rng = np.random.default_rng(15)
    nodes, vocab, temperature = [3] * 6, 600, np.array([1.0, 1.0, 1.0, 1.0, 0.0, 1.0])
    s = inputs(rng, nodes, vocab, "given", temperature)
    s["accept"][:] = 0.0  # every draft with any probability is accepted
    for i in (1, 2):
        s["parents"][i::3] = i - 1
        s["tokens"][i::3] = 5
    x = s["logits"].reshape(6, 3, vocab)
    x[:, :2, 5] = 30.0
    x[0, 0, 7] = np.nan
    x[1, 2, 7] = np.inf
    x[2, 1] = -np.inf
    x[3, 2, 599] = np.nan
    x[4, 2] = -np.inf
    out = run(gpu_ctx, s, nodes, temperature)
    with pytest.raises(FerrisError) as e:
        gpu_ctx.check_faults()
    assert e.value.kind == "Runtime" and "finite" in e.value.message
    tokens, path, count, prob = (o.cpu().numpy() for o in out)
    assert tokens.tolist()[:5] == [[-1, -1, -1], [5, 5, -1], [5, -1, -1], [5, 5, -1], [5, 5, -1]]
    assert count.tolist()[:5] == [0, 2, 1, 2, 2] and (prob[:5] == 0).all() and prob[5] > 0 and tokens[5, 2] >= 0
    gpu_ctx.check_faults()


def test_bad_drafts_are_reported(gpu_ctx):
    from ferrisinfer_amd import FerrisError

    rng = np.random.default_rng(16)
    nodes, vocab, temperature = [4, 4], 100, np.ones(2)
    for mode in ("given", "drawn"):
        s = inputs(rng, nodes, vocab, mode, temperature)
        s["parents"][:] = [-1, 0, 0, 0] * 2
        s["tokens"][1], s["tokens"][2] = vocab, -3  # passed over
        out = run(gpu_ctx, s, nodes, temperature)
        with pytest.raises(FerrisError) as e:
            gpu_ctx.check_faults()
        assert "token id" in e.value.message
        check(out, s, nodes, temperature)
    # parents that are not before their nodes: nodes of no one
    s["tokens"][1:3] = 0
    for bad in (2, 3, 1000, -2, -2 ** 31):
        s["parents"][2] = bad
        out = run(gpu_ctx, s, nodes, temperature)
        with pytest.raises(FerrisError) as e:
            gpu_ctx.check_faults()
        assert "parent" in e.value.message
        check(out, dict(s, parents=np.where(np.arange(8) == 2, -1, s["parents"])), nodes, temperature)
    # more nodes than max_query_len: the first ones
    s = inputs(rng, [6, 4], vocab, "given", temperature)
    out = run(gpu_ctx, s, [6, 4], temperature, most=4)
    with pytest.raises(FerrisError) as e:
        gpu_ctx.check_faults()
    assert "query" in e.value.message
    cut = {k: v if v is None or k == "pick" else np.concatenate([v[:4], v[6:]]) for k, v in s.items()}
    check(out, cut, [4, 4], temperature)


def test_paths_end_at_max_path(gpu_ctx):
    rng = np.random.default_rng(17)
    nodes, temperature = [6, 6, 6], np.array([1.0, 0.5, 0.0])
    s = inputs(rng, nodes, 700, "drawn", temperature)
    for i in range(1, 6):
        s["parents"][i::6] = i - 1
        s["tokens"][i::6] = s["logits"][i - 1::6].argmax(-1)
    s["accept"][:] = 0.0
    for longest in (0, 1, 3, 5, 9):
        out = run(gpu_ctx, s, nodes, temperature, max_path=longest)
        gpu_ctx.sync()
        assert out[2].tolist() == [min(longest, 5)] * 3
        check(out, s, nodes, temperature, max_path=longest)


def test_strides_and_alignment(gpu_ctx):
    import torch

    rng = np.random.default_rng(18)
    nodes, temperature = [5, 3, 7], np.array([1.0, 0.0, 0.7])
    for vocab, width, at in [(1000, 1024, 0), (1000, 1003, 0), (1000, 1024, 1), (997, 997, 0), (997, 1000, 3)]:
        for mode in ("given", "drawn"):
            s = inputs(rng, nodes, vocab, mode, temperature)
            views = []
            for x in (s["logits"], s["probs"]):
                if x is None:
                    views.append(None)
                    continue
                flat = torch.full((15 * width + 8,), float("nan"), device="cuda")
                view = torch.as_strided(flat, (15, vocab), (width, 1), at)
                view.copy_(dev(x))
                views.append(view)
            out = run(gpu_ctx, s, nodes, temperature, logits=views[0], probs=views[1])
            gpu_ctx.sync()
            gpu_ctx.check_faults()
            check(out, s, nodes, temperature, what=(vocab, width, at, mode))


def test_the_first_token_is_the_models(gpu_ctx):
    """20000 sequences of one launch: the first token's counts are the model's distribution's, whatever was drafted."""
    rng = np.random.default_rng(19)
    vocab, n = 6, 20000
    logits = rng.standard_normal(vocab)
    p, q = softmax(logits / 0.8), softmax(rng.standard_normal(vocab))
    for mode, kids in [("given", 2), ("drawn", 3), ("distinct", 3)]:
        if mode == "given":
            drafts = np.tile(np.arange(kids), (n, 1))
        elif mode == "drawn":
            drafts = rng.choice(vocab, (n, kids), p=q)
        else:
            drafts = np.stack([rng.choice(vocab, kids, replace=False, p=q) for _ in range(n)])
        size = kids + 1
        s = dict(logits=np.tile(logits.astype(np.float32), (n * size, 1)), tokens=np.insert(drafts, 0, 0, 1).reshape(-1).astype(np.int32),
                 parents=np.tile([-1] + [0] * kids, n).astype(np.int32), accept=rng.random(n * size).astype(np.float32),
                 pick=rng.random(n).astype(np.float32), probs=None if mode == "given" else np.tile(q.astype(np.float32), (n * size, 1)))
        out = run(gpu_ctx, s, [size] * n, np.full(n, 0.8), mode == "distinct", max_path=kids)
        gpu_ctx.sync()
        seen = np.bincount(out[0][:, 0].cpu().numpy(), minlength=vocab)
        # five standard deviations of a count hold in all but one of 10^6 runs
        assert (np.abs(seen - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all(), (mode, seen / n, p)


def test_empty_calls(gpu_ctx):
    import torch

    s = dict(logits=np.zeros((0, 9), np.float32), tokens=np.zeros(0, np.int32), parents=np.zeros(0, np.int32),
             accept=np.zeros(0, np.float32), pick=np.zeros(2, np.float32), probs=None)
    out = run(gpu_ctx, dict(s, logits=np.zeros((1, 9), np.float32), tokens=np.zeros(1, np.int32), parents=np.zeros(1, np.int32),
                            accept=np.zeros(1, np.float32)), [0, 0], np.ones(2), max_path=2)
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    assert out[0].tolist() == [[-1] * 3] * 2 and out[2].tolist() == [0, 0] and out[3].tolist() == [0.0, 0.0]


def test_refusals(gpu_ctx):
    import torch

    from ferrisinfer_amd import FerrisError

    i = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    f = lambda *n: torch.zeros(n, device="cuda")  # noqa: E731
    base = dict(logits=f(6, 40), tokens=i(6), parents=i(6) - 1, cu_seqlens=i(3), max_query_len=3, temperature=f(2), accept_u=f(6),
                pick_u=f(2), draft_probs=None, distinct=False, tokens_out=i(2, 4), path_out=i(2, 3), count_out=i(2), prob_out=f(2))
    gpu_ctx.verify_drafts(**base)
    for change, kind in [
        (dict(logits=f(6, 0)), "InvalidShape"), (dict(logits=f(40, 6).T), "InvalidLayout"), (dict(logits=f(6, 40).half()), "InvalidType"),
        (dict(logits=f(1, 1 << 21)[:, :(1 << 20) + 4], tokens=i(1), parents=i(1), accept_u=f(1)), "Unsupported"),
        (dict(max_query_len=1025), "Unsupported"), (dict(max_query_len=-1), "InvalidShape"), (dict(tokens=i(5)), "InvalidShape"),
        (dict(parents=i(6).long()), "InvalidType"), (dict(cu_seqlens=i(2)), "InvalidShape"), (dict(accept_u=f(5)), "InvalidShape"),
        (dict(pick_u=f(1)), "InvalidShape"), (dict(pick_u=f(2).double()), "InvalidType"), (dict(draft_probs=f(6, 39)), "InvalidShape"),
        (dict(draft_probs=f(5, 40)), "InvalidShape"), (dict(tokens_out=i(2, 3)), "InvalidShape"), (dict(path_out=i(1, 3)), "InvalidShape"),
        (dict(count_out=i(1)), "InvalidShape"), (dict(prob_out=f(1)), "InvalidShape"), (dict(tokens_out=i(4, 2).T), "InvalidLayout"),
        (dict(tokens_out=i(2, 1025), path_out=i(2, 1024)), "InvalidShape"), (dict(logits=f(6, 39).as_strided((6, 39), (20, 1))), "InvalidShape"),
    ]:
        with pytest.raises(FerrisError) as e:
            gpu_ctx.verify_drafts(**dict(base, **change))
        assert e.value.kind == kind, (change.keys(), e.value)
    gpu_ctx.check_faults()


def test_graph_replays_and_another_stream(gpu_ctx):
    import torch

    from ferrisinfer_amd import Context

    rng = np.random.default_rng(20)
    nodes, vocab, temperature = [5, 7, 2, 6], 9000, np.array([1.0, 0.7, 0.0, 1.2])
    s = inputs(rng, nodes, vocab, "drawn", temperature)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ctx = Context(0)
        held = {k: dev(v) for k, v in s.items()}
        cu, heat = dev(np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)), dev(temperature.astype(np.float32))
        i = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        out = [i(4, 7), i(4, 6), i(4), torch.zeros(4, device="cuda")]

        def call(out):
            ctx.verify_drafts(held["logits"], held["tokens"], held["parents"], cu, 7, heat, held["accept"], held["pick"], held["probs"],
                              False, *out)

        call(out)
        stream.synchronize()
        check(out, s, nodes, temperature)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(out)
        for k in range(4):
            new = rng.random(len(s["accept"])).astype(np.float32), rng.random(4).astype(np.float32)
            held["accept"].copy_(dev(new[0]))
            held["pick"].copy_(dev(new[1]))
            eager = [torch.empty_like(x) for x in out]
            call(eager)
            stream.synchronize()
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, eager)), k
            check(out, dict(s, accept=new[0], pick=new[1]), nodes, temperature)
        ctx.check_faults()
        ctx.close()
