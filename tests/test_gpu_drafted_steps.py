"""The drafted step as a decoder runs it (plan, append, attend, verify, keep), and the launches that verification and tree
attention take for sizes that no other test has."""
from fractions import Fraction

import numpy as np
import pytest

import draft_reference as ref
import fp4_reference as fp4
from test_gpu_fp4_cache import dev, tables_of
from test_gpu_tree_attention import PIECES, attend, checked, dtype_of, pool_of, trees_of
from test_gpu_verify_drafts import check, inputs, run

pytestmark = pytest.mark.gpu

HQ, HKV, D, BS, LAYERS, VOCAB, LONGEST = 4, 2, 32, 16, 2, 97, 160


class Decoder:
    """Two layers of random weights without an MLP; the projections are taken in 64 bits, so that a row's do not
    depend on how many rows a step has."""

    def __init__(self, ctx, seqs, kind, seed):
        import torch

        rng = np.random.default_rng(seed)
        w = lambda *n: dev(rng.standard_normal(n) / np.sqrt(n[0]))  # noqa: E731
        self.ctx, self.kind, self.hidden = ctx, kind, HQ * D
        self.embed, self.head = dev(rng.standard_normal((VOCAB, self.hidden))), w(self.hidden, VOCAB) * 4
        self.qkv = [w(self.hidden, (HQ + 2 * HKV) * D) for _ in range(LAYERS)]
        self.out = [w(HQ * D, self.hidden) for _ in range(LAYERS)]
        self.cos, self.sin = (torch.empty(LONGEST, D // 2, device="cuda") for _ in range(2))
        ctx.rope_table(LONGEST, D, D, 10000.0, self.cos, self.sin)
        self.nb = seqs * (LONGEST // BS) + 2
        pools = [pool_of(rng, kind, self.nb, HKV, BS, D)[0] for _ in range(2 * LAYERS)]
        self.k, self.v = pools[::2], pools[1::2]
        self.host_tables = tables_of(rng, [LONGEST] * seqs, BS, self.nb)
        self.tables = dev(self.host_tables)

    def slots(self, lens, nodes):
        """The slots of each sequence's last `nodes` positions."""
        at = [np.arange(x - n, x) for x, n in zip(lens, nodes)]
        return np.concatenate([self.host_tables[b, p // BS].astype(np.int64) * BS + p % BS for b, p in enumerate(at)])

    def forward(self, tokens, positions, slots, attention):
        import torch

        t = tokens.shape[0]
        x = self.embed[tokens.long()]
        for layer in range(LAYERS):
            normed = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
            parts = (normed @ self.qkv[layer]).float()
            q = torch.empty(t, HQ, D, device="cuda")
            self.ctx.qkv_rope_append(parts, 1, None, positions, self.cos, self.sin, D, LONGEST, slots, self.k[layer], self.v[layer],
                                     dtype_of(self.kind), self.nb, BS, HQ, HKV, D, q)
            got = torch.empty_like(q)
            attention(layer, q, got)
            x = x + got.reshape(t, -1).double() @ self.out[layer]
        return (x @ self.head).float()

    def decode(self, prompts, steps):
        """Each sequence's next tokens, one a step."""
        import torch

        tokens, told = [list(p) for p in prompts], []
        for i in range(max(len(p) for p in prompts) + steps - 1):
            live = [b for b, p in enumerate(prompts) if i < len(p) + steps - 1]
            lens = dev(np.full(len(live), i + 1, np.int32))
            tables = dev(self.host_tables[live])
            slots = dev(np.array([self.host_tables[b, i // BS].astype(np.int64) * BS + i % BS for b in live]))
            logits = self.forward(dev(np.array([tokens[b][i] for b in live], np.int32)), lens - 1, slots,
                                  lambda layer, q, got: self.ctx.attn_decode_paged(q, self.k[layer], self.v[layer], dtype_of(self.kind),
                                                                                   tables, lens, i + 1, HKV, BS, self.nb, D ** -0.5, got))
            for b, x in zip(live, logits.argmax(-1).tolist()):
                if i + 1 == len(tokens[b]):
                    tokens[b].append(x)
        torch.cuda.synchronize()
        self.ctx.check_faults()
        return tokens


class Step:
    """A drafted step over buffers that stay, so that it can be captured."""

    def __init__(self, dec, nodes, longest_path):
        import torch

        i = lambda *n, t=torch.int32: torch.zeros(n, dtype=t, device="cuda")  # noqa: E731
        rows, seqs = sum(nodes), len(nodes)
        self.dec, self.most, self.path_len = dec, max(nodes), longest_path
        self.tokens, self.parents, self.slots = i(rows), i(rows), i(rows, t=torch.int64)
        self.cu, self.lens = dev(np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)), i(seqs)
        self.mask, self.positions = i(rows, 1, t=torch.int64), i(rows)
        self.heat, self.u, self.pick = torch.zeros(seqs, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros(seqs, device="cuda")
        self.out, self.path, self.count, self.prob = i(seqs, longest_path + 1), i(seqs, longest_path), i(seqs), torch.zeros(seqs, device="cuda")

    def run(self):
        d, c = self.dec, self.dec.ctx
        c.tree_plan(self.parents, self.cu, self.lens, self.most, self.mask, self.positions)
        logits = d.forward(self.tokens, self.positions, self.slots,
                           lambda layer, q, got: c.attn_tree_paged(q, d.k[layer], d.v[layer], dtype_of(d.kind), d.tables, self.cu, self.lens,
                                                                   self.mask, self.most, LONGEST, HKV, BS, d.nb, D ** -0.5, got))
        c.verify_drafts(logits, self.tokens, self.parents, self.cu, self.most, self.heat, self.u, self.pick, None, False, self.out,
                        self.path, self.count, self.prob)
        c.kv_keep_path(d.k, d.v, dtype_of(d.kind), d.tables, self.cu, self.lens, self.path, d.nb, BS, HKV, D)


def drafted(rng, known, at, n):
    """A tree of n nodes on the sequence's token `at`: right continuations of it among wrong ones, in any order."""
    tokens, parents, right = [known[at]], [-1], [0]
    while len(tokens) < n:
        kind = rng.random()
        if kind < 0.5 and at + len(right) < len(known):
            parents.append(right[-1])
            tokens.append(known[at + len(right)])
            right.append(len(tokens) - 1)
        else:
            p = int(rng.integers(0, len(tokens)))
            parents.append(p)
            tokens.append(int(rng.integers(0, VOCAB)))
            if p in right and right.index(p) + 1 == len(right) and at + len(right) < len(known) and tokens[-1] == known[at + len(right)]:
                right.append(len(tokens) - 1)
    return tokens, parents


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
def test_drafted_steps_decode_what_single_tokens_do(gpu_ctx, kind, captured):
    """Greedy decoding in drafted steps, good and bad drafts mixed, gives the tokens of decoding one by one."""
    import torch

    from ferrisinfer_amd import Context

    rng = np.random.default_rng(40)
    steps, prompts = 40, [rng.integers(0, VOCAB, n).tolist() for n in (3, 30, 17, 1)]
    want = Decoder(gpu_ctx, 4, kind, 1).decode(prompts, steps + 12)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ctx = Context(0)
        dec = Decoder(ctx, 4, kind, 1)
        # the prompts, as one more known stretch of single tokens
        known = [list(t) for t in dec.decode(prompts, 1)]
        assert [k[:len(w)] for k, w in zip(known, want)] == [w[:len(k)] for k, w in zip(known, want)]
        nodes = [5, 9, 1, 7]
        step, graph, accepted = Step(dec, nodes, 8), None, 0
        for it in range(100):
            if min(len(k) - len(p) for k, p in zip(known, prompts)) >= steps:
                break
            if not captured:  # other trees each time; sequences that are done have none
                nodes = [0 if len(k) - len(p) >= steps else int(rng.integers(1, 10)) for k, p in zip(known, prompts)]
                step = Step(dec, nodes, 8)
            elif len(known[0]) - len(prompts[0]) >= steps + 1 or max(len(k) - len(p) for k, p in zip(known, prompts)) >= steps + 2:
                break
            trees = [drafted(rng, w, len(k) - 1, n) if n else ([], []) for w, k, n in zip(want, known, nodes)]
            lens = [len(k) - 1 + n for k, n in zip(known, nodes)]
            for to, x in [(step.tokens, np.concatenate([t[0] for t in trees])), (step.parents, np.concatenate([t[1] for t in trees])),
                          (step.lens, lens), (step.slots, dec.slots(lens, nodes))]:
                to.copy_(dev(np.asarray(x)))
            if captured and graph is None:
                step.run()  # sizes the workspace; every row that it wrote is written again
                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    step.run()
            if captured:
                graph.replay()
            else:
                step.run()
            stream.synchronize()
            ctx.check_faults()
            for b, (k, n) in enumerate(zip(known, nodes)):
                count = int(step.count[b])
                k += [x for x in step.out[b].tolist() if x >= 0]
                assert len(k) == lens[b] - n + 1 + (count + 1 if n else 0)
                assert k == want[b][:len(k)], (it, b, k[-8:], want[b][:len(k)][-8:])
                accepted += count
        assert it > 3 and accepted > 20
        # the rows that were moved are those of single tokens
        if kind == "f32":
            whole = Decoder(ctx, 4, kind, 1)
            whole.decode([k[:-1] for k in known], 1)
            for pools, other in ((dec.k, whole.k), (dec.v, whole.v)):
                for x, y in zip(pools, other):
                    for b, k in enumerate(known):
                        p = np.arange(len(k) - 1)
                        at = dev(dec.host_tables[b, p // BS].astype(np.int64)), dev(p % BS)
                        assert torch.allclose(x[at[0], :, at[1]], y[at[0], :, at[1]], rtol=0, atol=1e-4)
        ctx.close()


@pytest.mark.parametrize("mode", ["given", "drawn", "distinct"])
def test_verify_of_many_rows(gpu_ctx, mode):
    """More logits than are all summed in the first launch: launches a row, more rejections than have one, what is left."""
    rng = np.random.default_rng(50)
    nodes, vocab = [24, 9, 24, 1, 16, 24, 0, 24], 110000
    assert len(nodes) * max(nodes) * vocab > 20000000
    temperature = np.array([1.0, 0.7, 0.0, 1.0, 1.5, 1.0, 1.0, 0.9])
    s = inputs(rng, nodes, vocab, mode, temperature)
    at = 0
    for b, n in enumerate(nodes):
        if b in (0, 5):  # many unlikely children of one node
            s["parents"][at + 1:at + n] = 0
            s["tokens"][at + 1:at + n] = rng.choice(vocab, n - 1, replace=False)
        at += n
    out = run(gpu_ctx, s, nodes, temperature, mode == "distinct", max_path=6)
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    check(out, s, nodes, temperature, mode == "distinct", max_path=6)
    # the same walks where every row is summed at once, sequence by sequence
    at = 0
    for b, n in enumerate(nodes):
        r = slice(at, at + n)
        one = {k: v if v is None else v[b:b + 1] if k == "pick" else v[r] for k, v in s.items()}
        at += n
        if n == 0:
            continue
        alone = run(gpu_ctx, one, [n], temperature[b:b + 1], mode == "distinct", max_path=6)
        assert all(bool((x[b] == y[0]).all()) for x, y in zip(out, alone)), b


@pytest.mark.parametrize("mode", ["given", "drawn", "distinct"])
def test_verify_of_long_paths(gpu_ctx, mode):
    """Paths of more tokens than have a launch each: sequences that end before, there, and behind."""
    rng = np.random.default_rng(51)
    nodes, vocab = [40, 40, 23, 40], 130000
    assert len(nodes) * max(nodes) * vocab > 20000000
    temperature = np.array([1.0, 0.0, 0.8, 0.7])
    s = inputs(rng, nodes, vocab, mode, temperature)
    at = 0
    for b, n in enumerate(nodes):  # chains of the likeliest tokens, accepted whatever u
        for i in range(1, n):
            s["parents"][at + i] = i - 1
            s["tokens"][at + i] = s["logits"][at + i - 1].argmax()
        s["accept"][at:at + n] = 0.0
        at += n
    s["tokens"][80 + 23 + 9] = (s["tokens"][80 + 23 + 9] + 1) % vocab  # the last one's ninth is not, mostly
    s["accept"][80 + 23 + 9] = 0.999
    for longest in (39, 18, 3):
        out = run(gpu_ctx, s, nodes, temperature, mode == "distinct", max_path=longest)
        gpu_ctx.sync()
        gpu_ctx.check_faults()
        assert out[2].tolist()[:2] == [longest] * 2
        check(out, s, nodes, temperature, mode == "distinct", max_path=longest, what=longest)


def test_verify_of_many_rows_captured(gpu_ctx):
    """All of the launches in a graph: rows, rejections, what is left; replayed with other random numbers."""
    import torch

    from ferrisinfer_amd import Context

    rng = np.random.default_rng(54)
    nodes, vocab, temperature = [40, 12, 33, 25], 130000, np.array([1.0, 0.7, 0.0, 1.3])
    assert len(nodes) * max(nodes) * vocab > 20000000
    s = inputs(rng, nodes, vocab, "drawn", temperature)
    s["parents"][1:40] = 0  # a root of many children
    s["tokens"][1:40] = rng.choice(vocab, 39, replace=False)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ctx = Context(0)
        held = {k: dev(v) for k, v in s.items()}
        cu, heat = dev(np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)), dev(temperature.astype(np.float32))
        i = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731

        def call(out):
            ctx.verify_drafts(held["logits"], held["tokens"], held["parents"], cu, 40, heat, held["accept"], held["pick"], held["probs"],
                              False, *out)

        out, eager = ([i(4, 21), i(4, 20), i(4), torch.zeros(4, device="cuda")] for _ in range(2))
        call(out)
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            call(out)
        for k in range(4):
            new = rng.random(sum(nodes)).astype(np.float32), rng.random(4).astype(np.float32)
            if k == 1:
                new[0][:] = 0.0  # the longest paths
            held["accept"].copy_(dev(new[0]))
            held["pick"].copy_(dev(new[1]))
            call(eager)
            stream.synchronize()
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, eager)), k
            check(out, dict(s, accept=new[0], pick=new[1]), nodes, temperature, max_path=20, what=k)
        ctx.check_faults()
        ctx.close()


@pytest.mark.parametrize("mode", ["given", "drawn"])
@pytest.mark.parametrize("vocab", [262144, 262145, 600004, 1048576])
def test_verify_of_wide_vocabularies(gpu_ctx, mode, vocab):
    """A lane of the last workgroup has one, two, three and four segments."""
    rng = np.random.default_rng(vocab)
    nodes, temperature = [4, 2, 3], np.array([1.0, 0.0, 1.3])
    s = inputs(rng, nodes, vocab, mode, temperature)
    for pick in (0.1, 0.5, 0.999999):
        s["pick"][:] = pick
        out = run(gpu_ctx, s, nodes, temperature)
        gpu_ctx.sync()
        check(out, s, nodes, temperature, what=pick)
    # flat rows, where any segment may be drawn from
    s["logits"][:] = 0.0
    for pick in (0.1, 0.5, 0.999999):
        s["pick"][:] = pick
        out = run(gpu_ctx, s, nodes, temperature)
        gpu_ctx.sync()
        if mode == "drawn":
            check(out, s, nodes, temperature, what=pick)
            continue
        # Half of 262144 tokens is a border between two, which sums of a rounded 1 / 262145 do not find: in whole
        # numbers, the token behind pick * (those left).
        tokens, path, count, prob = (x.cpu().numpy() for x in out)
        at = 0
        for b, n in enumerate(nodes):
            r = slice(at, at + n)
            assert path[b][:count[b]].tolist() == ref.verify(s["logits"][r], s["tokens"][r], list(s["parents"][r]), temperature[b],
                                                             s["accept"][r], s["pick"][b])[1]
            node = path[b][count[b] - 1] if count[b] else 0
            tried = {int(s["tokens"][at + j]) for j in range(n) if s["parents"][at + j] == node and temperature[b] > 0}
            left = [x for x in range(vocab) if x not in tried]
            last = left[int(Fraction(float(s["pick"][b])) * len(left))] if temperature[b] > 0 else 0
            assert tokens[b][count[b]] == last, (b, pick, tokens[b], last)
            assert abs(float(prob[b]) * len(left) - 1) <= 2.0 ** -24 + 1e-11
            at += n


def test_verify_of_many_sequences(gpu_ctx):
    rng = np.random.default_rng(52)
    nodes, vocab = [int(n) for n in rng.integers(0, 4, 5000)], 20
    temperature = rng.choice([0.0, 1.0], 5000)
    for mode in ("given", "drawn"):
        s = inputs(rng, nodes, vocab, mode, temperature)
        for k in range(2):
            out = run(gpu_ctx, s, nodes, temperature)
            gpu_ctx.sync()
            check(out, s, nodes, temperature)


def test_two_contexts_at_once(gpu_ctx):
    """Each has a workspace, counters and a stream of its own."""
    import torch

    from ferrisinfer_amd import Context

    rng = np.random.default_rng(53)
    jobs = []
    for k in range(2):
        nodes, temperature = [6, 8, 3], np.array([1.0, 0.8, 0.0])
        s = inputs(rng, nodes, 40000, "drawn", temperature)
        jobs.append((s, nodes, temperature, run(gpu_ctx, s, nodes, temperature)))
    kind, seqs = "bf16", [(900, 9), (300, 5), (1500, 12)]
    nodes, lens = [n for _, n in seqs], [p + n for p, n in seqs]
    nb = sum(-(-n // BS) for n in lens)
    pools = [pool_of(rng, kind, nb, 2, BS, 64)[0] for _ in range(2)]
    tables, (_, mask) = tables_of(rng, lens, BS, nb), trees_of(rng, nodes)
    q = rng.standard_normal((sum(nodes), 8, 64)).astype(np.float32)
    args = (kind, q, pools, tables, nodes, lens, mask, 2, BS, nb, 0.125)
    want = checked(gpu_ctx, attend(gpu_ctx, *args))
    streams = [torch.cuda.Stream() for _ in range(2)]
    contexts = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            contexts.append(Context(0))
    outs = [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                s, n, t, _ = jobs[k]
                outs[k].append((run(contexts[k], s, n, t), attend(contexts[k], *args)))
    for k in range(2):
        streams[k].synchronize()
        contexts[k].check_faults()
        for got, att in outs[k]:
            assert all(torch.equal(x, y) for x, y in zip(got, jobs[k][3]))
            assert np.array_equal(att.cpu().numpy(), want)
        contexts[k].close()


# (sequences of cached rows and nodes), hq, hkv, d: how a launch lays its pieces out
LAYOUTS = {
    "more sequences than a plan holds": ([(int(p), int(n)) for p, n in zip(range(0, 300), [1, 2, 0, 5] * 75)], 2, 1, 32),
    "as many as it holds": ([(3 * i, 1 + i % 3) for i in range(256)], 2, 1, 32),
    "one long among short ones": ([(6000, 4)] + [(20, 3)] * 40, 4, 2, 32),
    "a long one, and empty ones": ([(0, 0), (0, 0), (4000, 7), (9, 0), (0, 0)], 4, 2, 64),
    "nothing but empty ones": ([(0, 0)] * 3, 4, 2, 32),
    "joined in the launch": ([(1900, 3), (1800, 70), (0, 2)], 8, 2, 64),
    "joined by a launch": ([(2100, 3), (1800, 70), (0, 2)], 8, 2, 64),
    "joined by a launch of many tiles": ([(6000, 4)] + [(20, 3)] * 40, 8, 4, 32),
    "joined in a launch of many tiles": ([(1900, 9)] + [(20, 3)] * 70, 8, 4, 32),
    "several tiles a sequence": ([(1000, 200), (30, 140)], 8, 2, 32),
}


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_launch_layouts(gpu_ctx, layout, kind):
    seqs, hq, hkv, d = LAYOUTS[layout]
    print(f"tree attention {kind} {layout}", flush=True)
    rng = np.random.default_rng(len(layout))
    nodes, lens = [n for _, n in seqs], [p + n for p, n in seqs]
    nb = sum(-(-n // BS) for n in lens) + 1
    (kd, kv), (vd, vv) = pool_of(rng, kind, nb, hkv, BS, d), pool_of(rng, kind, nb, hkv, BS, d)
    tables = tables_of(rng, lens, BS, nb)
    trees, mask = trees_of(rng, nodes)
    rows = sum(nodes)
    if rows == 0:
        mask = np.zeros((1, 1), np.int64)
    q = rng.standard_normal((max(rows, 1), hq, d)).astype(np.float32)
    for k in range(2):  # and again: whatever the first left in counters and workspace
        got = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, nodes, lens, mask, hkv, BS, nb, d ** -0.5))
        assert rows or (got == -7).all()
        at = 0
        for b, (p, n) in enumerate(seqs):
            if n:
                keys, values = (fp4.rows_of(x, tables[b], p + n, BS) for x in (kv, vv))
                shown = ref.visible(ref.ancestors(trees[b]), p, p + n)
                ref.check_attention(got[at:at + n], q[at:at + n], keys, values, shown, d ** -0.5, PIECES[kind], (b, kind, layout))
                at += n


# what the scales of a 4-bit pool's groups are, as (K, V) of a group (block, head, row, group) of a context of 500 rows
SCALES = {
    "the least that f16 holds": lambda rng, n: (rng.integers(104, 108, n), rng.integers(104, 108, n)),
    "the largest": lambda rng, n: (rng.integers(137, 141, n), rng.integers(137, 141, n)),
    "all that it holds": lambda rng, n: (rng.integers(104, 141, n), rng.integers(104, 141, n)),
    "the least that is normal": lambda rng, n: (rng.integers(109, 112, n), rng.integers(109, 112, n)),
    "the largest of those": lambda rng, n: (rng.integers(133, 136, n), rng.integers(133, 136, n)),
    "all of those": lambda rng, n: (rng.integers(109, 136, n), rng.integers(109, 136, n)),
    "less": lambda rng, n: (rng.integers(80, 104, n), rng.integers(1, 104, n)),
    "more": lambda rng, n: (rng.integers(141, 160, n), rng.integers(141, 200, n)),
    "one K group beyond": lambda rng, n: (np.where(np.arange(n) == n // 2, 150, 127), np.full(n, 127)),
    "one V group below": lambda rng, n: (np.full(n, 127), np.where(np.arange(n) == n // 3, 90, 127)),
    "any": lambda rng, n: (rng.integers(60, 150, n), rng.integers(1, 220, n)),
}


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("scale,size", [(1e-8, 1e-36), (1e-12, 1e-30), (1e20, 1e-20), (1e-20, 1e20), (1e-30, 1e-38), (0.125, 1e-42)])
def test_small_and_large_scales_and_queries(gpu_ctx, kind, scale, size):
    """The scale and Q's sizes make up for each other, or leave scores of nothing: every key that is seen weighs the same."""
    rng = np.random.default_rng(61)
    hq, hkv, d, prefix, n = 4, 2, 64, 90, 21
    keys, nb = prefix + n, 9
    (kd, kv), (vd, vv) = pool_of(rng, kind, nb, hkv, BS, d), pool_of(rng, kind, nb, hkv, BS, d)
    tables = tables_of(rng, [keys], BS, nb)
    trees, mask = trees_of(rng, [n])
    q = (rng.standard_normal((n, hq, d)) * size).astype(np.float32)
    q[4] = 0.0
    got = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, [n], [keys], mask, hkv, BS, nb, scale))
    k, v = (fp4.rows_of(x, tables[0], keys, BS) for x in (kv, vv))
    shown = ref.visible(ref.ancestors(trees[0]), prefix, keys)
    ref.check_attention(got, q, k, v, shown, float(np.float32(scale)), PIECES[kind], (scale, size))


@pytest.mark.parametrize("d,prefix", [(32, 500), (64, 490), (128, 497), (128, 5000)])
@pytest.mark.parametrize("scales", list(SCALES))
def test_scales_of_four_bit_groups(gpu_ctx, scales, d, prefix):
    rng = np.random.default_rng(d + prefix)
    hq, hkv, n = 8, 2, 11
    keys = prefix + n
    nb = -(-keys // BS) + 1
    tables = tables_of(rng, [keys], BS, nb)
    pools, values = [], []
    for which in range(2):
        raw, value = pool_of(rng, "mxfp4", nb, hkv, BS, d)
        at = nb * hkv * BS * (d // 2)
        old = raw[at:].cpu().numpy().astype(np.int64)
        new = np.asarray(SCALES[scales](rng, old.size)[which], np.int64)
        if "one" in scales:  # in a row that is seen
            seen = np.zeros((nb, hkv, BS, d // 32), bool)
            seen[tables[0, 7], 1, 3, 0] = True
            new = np.where(seen.reshape(-1), np.unique(new)[np.argmax(np.abs(np.unique(new) - 127))], 127)
        raw[at:] = dev(new.astype(np.uint8))
        pools.append(raw)
        values.append((value.reshape(-1, 32) * np.exp2((new - old).astype(np.float64))[:, None]).reshape(value.shape))
    trees, mask = trees_of(rng, [n])
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    k, v = (fp4.rows_of(x, tables[0], keys, BS) for x in values)
    # scores of a few units, whatever K's scales: rows of Q of very different sizes
    q /= np.float32(np.sqrt((k * k).mean()))
    q[3] = 0.0
    q[5] *= np.float32(1e-9)
    q[6] *= 3
    got = checked(gpu_ctx, attend(gpu_ctx, "mxfp4", q, pools, tables, [n], [keys], mask, hkv, BS, nb, d ** -0.5))
    shown = ref.visible(ref.ancestors(trees[0]), prefix, keys)
    ref.check_attention(got, q, k, v, shown, d ** -0.5, PIECES["mxfp4"], scales)
