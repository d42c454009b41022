"""Serving with drafted tokens, as operators that can be timed and compared.

A cheap draft proposes a tree of tokens behind each sequence's last one, and one forward step of the
model scores every node of every tree.  Node 0 of a sequence's tree is the token it already has; every
other node is a drafted token whose parent comes before it.  The step's rows are packed by cu_seqlens,
appended to the paged pool in the order of the nodes, and:

  plan    the parents of the nodes become their masks (one bit for each ancestor) and positions
  attend  the rows attend the cached prefix and their own ancestors in the pool
  verify  the drafted tokens are accepted or not against the model's logits, so that the tokens are
          distributed as the model's own are, and one more token is drawn where the path ends
  keep    the K/V rows of the accepted path move to the places behind the prefix, in every layer

``run`` makes the framework's calls where ``own`` is true and computes the plain forms elsewhere.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 16
GROUP = 32  # elements that share a scale in a 4-bit pool
EPSILON = 2.0 ** -23  # the least temperature that is divided by

# query heads, kv heads, head dimension and vocabulary of the decoders this repository is configured for
MODELS = {"tiny": (8, 2, 32, 32000), "qwen2": (14, 2, 64, 151936), "llama3": (32, 8, 128, 128256)}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one chat user's tree
        dict(name="plan-1", op="plan", seqs=1, min_nodes=8, max_nodes=8, depth=4),
        # a full server, trees of mixed sizes wider than a word
        dict(name="plan-256", op="plan", seqs=256, min_nodes=17, max_nodes=100, depth=8),
        # one chat user, a short history, f32 pool: pure latency
        dict(name="attend-1", op="attend", model="qwen2", pool="f32", seqs=1, min_nodes=8, max_nodes=8, depth=4, min_ctx=700,
             max_ctx=700),
        # a batch of 64 users, trees of mixed sizes, histories between 128 and 2048 tokens
        dict(name="attend-64", op="attend", model="llama3", pool="bf16", seqs=64, min_nodes=5, max_nodes=16, depth=5,
             min_ctx=128, max_ctx=2048),
        # two users with very long histories, 4-bit pool: few rows, a long axis
        dict(name="attend-long", op="attend", model="llama3", pool="mxfp4", seqs=2, min_nodes=24, max_nodes=32, depth=6,
             min_ctx=60001, max_ctx=100003),
        # wide trees behind long histories: the most arithmetic
        dict(name="attend-wide", op="attend", model="llama3", pool="bf16", seqs=32, min_nodes=64, max_nodes=64, depth=8,
             min_ctx=512, max_ctx=8192),
        # one chat user, drafts looked up rather than drawn (no draft probabilities)
        dict(name="verify-1", op="verify", model="qwen2", seqs=1, min_nodes=8, max_nodes=8, depth=4, drafts="given",
             temperature=0.7, greedy=0),
        # a batch of 64 users, four tokens in a row drawn from a draft model; every fourth user is greedy
        dict(name="verify-64", op="verify", model="llama3", seqs=64, min_nodes=5, max_nodes=5, depth=4, drafts="drawn",
             temperature=1.0, greedy=4),
        # trees of several children a node, drawn without repetition
        dict(name="verify-tree-16", op="verify", model="llama3", seqs=16, min_nodes=24, max_nodes=32, depth=6,
             drafts="distinct", temperature=0.8, greedy=0),
        # a greedy batch with wide looked-up trees
        dict(name="verify-greedy-32", op="verify", model="qwen2", seqs=32, min_nodes=9, max_nodes=33, depth=5, drafts="given",
             temperature=0.0, greedy=0),
        # one chat user: the two rows of a side branch, in 24 layers
        dict(name="keep-1", op="keep", model="qwen2", pool="f32", layers=24, seqs=1, depth=4, side=2),
        # a batch of 32 users in 32 layers
        dict(name="keep-32", op="keep", model="llama3", pool="bf16", layers=32, seqs=32, depth=6, side=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "attend", "attend", "attend", "verify", "verify", "keep"])
    model = rng.choice(sorted(MODELS))
    hq, hkv, d, vocab = MODELS[model]
    if op == "plan":
        seqs, nodes = _log(rng, 1, 256), _log(rng, 1, 100)
        return dict(op=op, seqs=seqs, max_nodes=nodes, min_nodes=max(1, int(nodes * rng.uniform(0.1, 1.0))), depth=rng.randint(1, 8))
    if op == "attend":
        seqs, nodes = _log(rng, 1, 64), _log(rng, 1, 64)
        longest = _log(rng, 1, 100003) if rng.random() < 0.9 else 0
        # rows of the caches and (query, key) pairs of all heads at most as in the largest listed case
        longest = min(longest, 32 * 8192 * 1024 // (seqs * hkv * d), 32 * 8192 * 64 * 32 // (2 * seqs * nodes * hq))
        return dict(op=op, model=model, pool=rng.choice(["f32", "bf16", "mxfp4"]), seqs=seqs, max_nodes=nodes,
                    min_nodes=max(1, int(nodes * rng.uniform(0.1, 1.0))), depth=rng.randint(1, 8), max_ctx=longest,
                    min_ctx=int(longest * rng.uniform(0.05, 1.0)))
    if op == "verify":
        seqs = _log(rng, 1, 64)
        nodes = _log(rng, 1, max(1, min(33, 320 // seqs)))
        return dict(op=op, model=model, seqs=seqs, max_nodes=nodes, min_nodes=max(1, int(nodes * rng.uniform(0.1, 1.0))),
                    depth=rng.randint(1, 6), drafts=rng.choice(["given", "drawn", "distinct"]),
                    temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.3]), greedy=rng.choice([0, 0, 2, 4]))
    depth = rng.randint(1, 6)
    seqs = _log(rng, 1, 32)
    return dict(op=op, model=model, pool=rng.choice(["f32", "bf16"]), layers=_log(rng, 1, 1 + 31 // (1 + (seqs * hkv * d) // 16384)),
                seqs=seqs, depth=depth, side=rng.randint(0, depth))


# ---------------------------------------------------------------- sizes of a case

def _spread(n, lo, hi):
    """n ragged lengths in [lo, hi], the ends among them, in a fixed mixed order."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * 7919) % n) // (n - 1) for i in range(n)]  # 7919: a prime above any n


def _sequences(case):
    """(cached rows, nodes) of every sequence."""
    if case["op"] == "keep":  # into the middle of a block
        return [((i * 5) % 40, 1 + case["depth"] + case["side"]) for i in range(case["seqs"])]
    nodes = _spread(case["seqs"], case["min_nodes"], case["max_nodes"])
    if case["op"] == "attend":
        return list(zip(_spread(case["seqs"], case["min_ctx"], case["max_ctx"])[::-1], nodes))
    return [(0, n) for n in nodes]


def _row_bytes(case):
    """Bytes of one token's K (or V) row."""
    _, hkv, d, _ = MODELS[case["model"]]
    return hkv * {"f32": 4 * d, "bf16": 2 * d, "mxfp4": d // 2 + d // GROUP}[case["pool"]]


def work(case):
    seqs = _sequences(case)
    nodes = sum(n for _, n in seqs)
    if case["op"] == "plan":
        words = -(-case["max_nodes"] // 64)
        return {"bytes": nodes * (4 + 8 * words + 4) + 8 * len(seqs), "flops": nodes * min(case["depth"], case["max_nodes"])}
    hq, hkv, d, vocab = MODELS[case["model"]]
    if case["op"] == "attend":
        keys = sum(p + n for p, n in seqs)
        pairs = sum(n * p + n * (1 + min(case["depth"], n - 1) / 2) for p, n in seqs)
        return {"bytes": 2 * keys * _row_bytes(case) + 8 * nodes * hq * d, "flops": 4 * pairs * hq * d}
    if case["op"] == "verify":
        # a sequence's rows: the nodes of its path, as long as tokens are accepted six times in ten
        # (where there is a choice of several, eight in ten), and the draft's row where the path ends
        rows = 0.0
        for _, n in seqs:
            share = 0.6 if n - 1 <= case["depth"] else 0.8
            rows += sum(share ** i for i in range(min(case["depth"], n - 1) + 1))
            rows += 0 if case["drafts"] == "given" or case["temperature"] <= 0 else 1
        return {"bytes": 4 * rows * vocab, "flops": 4 * rows * vocab}
    moved = case["seqs"] * case["side"] * case["layers"] * 2
    return {"bytes": 2 * moved * _row_bytes(case) + 64 * case["seqs"], "flops": moved}


# ---------------------------------------------------------------- the 4-bit format (values only)

#: the values of the eight codes without a sign
LADDER = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pool_parts(pool, case, blocks):
    """A 4-bit pool's codes [blocks, Hkv, BLOCK, D / 2] (element 2 i in the low half of byte i) and, behind
    them, its scales [blocks, Hkv, BLOCK, D / GROUP] (the scale's exponent + 127)."""
    _, hkv, d, _ = MODELS[case["model"]]
    n = blocks * hkv * BLOCK * (d // 2)
    return pool[:n].view(blocks, hkv, BLOCK, d // 2), pool[n:].view(blocks, hkv, BLOCK, d // GROUP)


def _four_bit_values(codes, scales):
    one = torch.tensor(LADDER + tuple(-v for v in LADDER), device=codes.device)
    byte = torch.arange(256, device=codes.device)
    v = torch.stack([one[byte & 15], one[byte >> 4]], -1)[codes.int()].flatten(-2).unflatten(-1, (-1, GROUP))
    return (v * (scales.int() << 23).view(torch.float32).unsqueeze(-1)).flatten(-2)


# ---------------------------------------------------------------- inputs

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _device(a, kind):
    return torch.from_numpy(np.ascontiguousarray(a, kind)).cuda()


def _grown(n, depth, r):
    """The parents of a tree of n nodes: the draft's best guesses in a row, then branches behind any node."""
    parents, deep = [-1], [0]
    for i in range(1, n):
        p = i - 1 if i <= depth else int(r.randint(0, i))
        while deep[p] >= depth:
            p = parents[p]
        parents.append(p)
        deep.append(deep[p] + 1)
    return parents


def _trees(case, seed):
    """The parents of every sequence's nodes."""
    r = np.random.RandomState(seed % (1 << 31))
    if case["op"] == "keep":  # a side branch of `side` nodes behind some node of the main path
        from_ = [int(r.randint(0, case["depth"] - case["side"] + 1)) for _ in range(case["seqs"])]
        main = list(range(-1, case["depth"]))
        return [main + ([f] + list(range(len(main), len(main) + case["side"] - 1)) if case["side"] else []) for f in from_], from_
    return [_grown(n, case["depth"], r) for _, n in _sequences(case)]


def _histories(case, seed):
    """Cached rows of the sequences of a plan, which no pool bounds."""
    return np.random.RandomState(seed % (1 << 31) + 1).randint(0, 8192, case["seqs"])


def _packed(case):
    """cu_seqlens, lengths with the tree's rows, and where a packed row lies in a padded batch."""
    seqs = _sequences(case)
    cu = np.concatenate([[0], np.cumsum([n for _, n in seqs])])
    widest = max(n for _, n in seqs)
    flat = np.concatenate([i * widest + np.arange(n) for i, (_, n) in enumerate(seqs)])
    padded = np.stack([cu[i] + np.minimum(np.arange(widest), n - 1) for i, (_, n) in enumerate(seqs)])
    return dict(case=dict(case), cu=_device(cu, np.int32), lens=_device([p + n for p, n in seqs], np.int32),
                flat=_device(flat, np.int64), padded=_device(padded, np.int64), widest=widest, rows=int(cu[-1]),
                longest=max(p + n for p, n in seqs))


def _paged(case, seed):
    """Block tables over a pool handed out in a random order, as a paged server's are after a while."""
    lens = [p + n for p, n in _sequences(case)]
    blocks = [-(-x // BLOCK) for x in lens]
    pool = sum(blocks) + 8
    perm = np.random.RandomState(seed % (1 << 31)).permutation(pool)
    tables = np.zeros((len(lens), max(blocks)), np.int32)
    at = 0
    for i, k in enumerate(blocks):
        tables[i, :k] = perm[at:at + k]
        at += k
    return dict(tables=_device(tables, np.int32), pool=pool)


def _filled_pool(case, blocks, g, spread, layers=()):
    """A pool whose rows were written before: normal values, their size varying by channel as keys' do."""
    _, hkv, d, _ = MODELS[case["model"]]
    if case["pool"] == "mxfp4":
        n = blocks * hkv * BLOCK * d
        pool = torch.empty(n // 2 + n // GROUP, dtype=torch.uint8, device="cuda")
        pool[:n // 2] = torch.randint(0, 256, (n // 2,), dtype=torch.uint8, generator=g, device="cuda")
        around = 124 + torch.round(2 * spread * _normal(g, hkv, 1, d // GROUP))
        _pool_parts(pool, case, blocks)[1][:] = around.to(torch.uint8)
        return pool
    pool = torch.empty(*layers, blocks, hkv, BLOCK, d, dtype=torch.float32 if case["pool"] == "f32" else torch.bfloat16, device="cuda")
    size = torch.exp(spread * _normal(g, hkv, 1, d))
    flat = pool.view(-1, hkv, BLOCK, d)
    for i in range(0, flat.shape[0], 4096):
        n = min(4096, flat.shape[0] - i)
        flat[i:i + n] = _normal(g, n, hkv, BLOCK, d) * size
    return pool


def _masks(trees, words):
    """The ancestors of every node and itself, as bits of its sequence's nodes."""
    rows = []
    for parents in trees:
        bits = []
        for i, p in enumerate(parents):
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        rows += [[(b >> 64 * w) & (2 ** 64 - 1) for w in range(words)] for b in bits]
    return torch.from_numpy(np.array(rows, np.uint64).view(np.int64)).cuda()


def _verify_inputs(case, seed, g):
    """Logits of a model that is sure of few tokens and leaves a tail to the others; a draft that is nearly
    of its opinion; the children of a node are the draft's best tokens, or drawn from it."""
    vocab = MODELS[case["model"]][3]
    m = _packed(case)
    trees = _trees(case, seed)
    t = m["rows"]
    first = np.repeat(m["cu"].cpu().numpy()[:-1], [len(p) for p in trees])
    parents = np.concatenate(trees)
    rank = np.concatenate([[sum(q == p for q in ps[:i]) for i, p in enumerate(ps)] for ps in trees])
    rank[parents < 0] = 0
    best = 4
    logits = 2.5 * _normal(g, t, vocab)
    liked = torch.randint(0, vocab, (t, best), generator=g, device="cuda")
    logits.scatter_(1, liked, 13 + 2 * _normal(g, t, best))
    temperature = torch.full((case["seqs"],), float(case["temperature"]), device="cuda")
    if case["greedy"]:
        temperature[::case["greedy"]] = 0.0
    # the draft's opinion, at the temperature it is asked for
    opinion = logits + 0.7 * _normal(g, t, vocab)
    most = int(rank.max()) + 1
    probs = None
    if case["drafts"] == "given":
        chosen = torch.topk(opinion, most, -1).indices
    else:
        by_row = temperature.clamp(min=0.3).repeat_interleave(m["cu"].diff().long())
        probs = torch.softmax(opinion / by_row[:, None], -1)
        chosen = torch.multinomial(probs, most, replacement=case["drafts"] == "drawn", generator=g)
    at = torch.from_numpy(np.maximum(first + parents, 0)).cuda()
    tokens = chosen[at, torch.from_numpy(rank).cuda()].int()
    deep = [0] * t
    for i in range(t):
        deep[i] = 0 if parents[i] < 0 else deep[first[i] + parents[i]] + 1
    return dict(m, logits=logits, tokens=tokens, parents=_device(parents, np.int32), temperature=temperature, probs=probs,
                accept=torch.rand(t, generator=g, device="cuda"), pick=torch.rand(case["seqs"], generator=g, device="cuda"),
                deepest=max(max(deep), 1), most=most)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "verify":
        s = _verify_inputs(case, seed, g)
        n, kind = case["seqs"], dict(dtype=torch.int32, device="cuda")
        return dict(s, out_tokens=torch.empty(n, s["deepest"] + 1, **kind), path=torch.empty(n, s["deepest"], **kind),
                    count=torch.empty(n, **kind), prob=torch.empty(n, device="cuda"))
    s = _packed(case)
    words = -(-s["widest"] // 64)
    if case["op"] == "plan":
        s["lens"] += _device(_histories(case, seed), np.int32)
        return dict(s, parents=_device(np.concatenate(_trees(case, seed)), np.int32), words=words,
                    mask=torch.empty(s["rows"], words, dtype=torch.int64, device="cuda"),
                    positions=torch.empty(s["rows"], dtype=torch.int32, device="cuda"))
    s |= _paged(case, seed)
    if case["op"] == "keep":
        trees, from_ = _trees(case, seed)
        path = np.full((case["seqs"], case["depth"]), -1)
        for b, f in enumerate(from_):  # the main path up to the branch, then the branch
            path[b, :f] = np.arange(1, f + 1)
            path[b, f:f + case["side"]] = case["depth"] + 1 + np.arange(case["side"])
        layers = (case["layers"],)
        return dict(s, path=_device(path, np.int32), k=_filled_pool(case, s["pool"], g, 0.5, layers),
                    v=_filled_pool(case, s["pool"], g, 0.1, layers))
    hq, hkv, d, _ = MODELS[case["model"]]
    return dict(s, k=_filled_pool(case, s["pool"], g, 0.5), v=_filled_pool(case, s["pool"], g, 0.1),
                q=_normal(g, s["rows"], hq, d), out=torch.empty(s["rows"], hq, d, device="cuda"),
                mask=_masks(_trees(case, seed), words))


# ---------------------------------------------------------------- one pass: the framework's calls

_CONTEXT = None


def _ctx():
    """A program keeps one context per GPU."""
    global _CONTEXT
    if _CONTEXT is None:
        from ferrisinfer_amd import Context

        _CONTEXT = Context(0)
    return _CONTEXT


def _kind(case):
    from ferrisinfer_amd import DTYPE_BF16, DTYPE_F32, DTYPE_MXFP4

    return {"f32": DTYPE_F32, "bf16": DTYPE_BF16, "mxfp4": DTYPE_MXFP4}[case["pool"]]


def _own_plan(s):
    _ctx().tree_plan(s["parents"], s["cu"], s["lens"], s["widest"], s["mask"], s["positions"])
    return s["mask"], s["positions"]


def _own_attend(s):
    _, hkv, d, _ = MODELS[s["case"]["model"]]
    _ctx().attn_tree_paged(s["q"], s["k"], s["v"], _kind(s["case"]), s["tables"], s["cu"], s["lens"], s["mask"], s["widest"],
                           s["longest"], hkv, BLOCK, s["pool"], d ** -0.5, s["out"])
    return s["out"]


def _own_verify(s):
    _ctx().verify_drafts(s["logits"], s["tokens"], s["parents"], s["cu"], s["widest"], s["temperature"], s["accept"], s["pick"],
                         s["probs"], s["case"]["drafts"] == "distinct", s["out_tokens"], s["path"], s["count"], s["prob"])
    return dict(tokens=s["out_tokens"], path=s["path"], count=s["count"], prob=s["prob"])


def _own_keep(s):
    _, hkv, d, _ = MODELS[s["case"]["model"]]
    _ctx().kv_keep_path(list(s["k"]), list(s["v"]), _kind(s["case"]), s["tables"], s["cu"], s["lens"], s["path"], s["pool"], BLOCK,
                        hkv, d)
    return s["k"], s["v"]


# ---------------------------------------------------------------- one pass: the plain forms

def _batched(s, packed, pad):
    """Packed rows [T] as a padded batch [B, widest]."""
    n = (s["cu"][1:] - s["cu"][:-1])[:, None]
    real = torch.arange(s["widest"], device=packed.device) < n
    return torch.where(real, packed[s["padded"]], torch.full((), pad, dtype=packed.dtype, device=packed.device))


def _plain_plan(s):
    parents = _batched(s, s["parents"], -1).long()  # [B, N]
    n, nodes = parents.shape[1], torch.arange(parents.shape[1], device=parents.device)
    # ancestors by steps upwards: column n stands for "none"
    up = torch.where(parents < 0, torch.full_like(parents, n), parents)
    up = torch.cat([up, torch.full_like(up[:, :1], n)], 1)
    at = nodes.expand_as(parents)
    seen = torch.zeros(*parents.shape, n + 1, dtype=torch.int64, device=parents.device)
    for _ in range(min(s["case"]["depth"], n) + 1):
        seen.scatter_(2, at[..., None], 1)
        at = up.gather(1, at)
    seen = seen[..., :n]
    bits = torch.nn.functional.pad(seen, (0, 64 * s["words"] - n)).unflatten(-1, (s["words"], 64))
    mask = (bits << torch.arange(64, device=parents.device)).sum(-1)
    prefix = s["lens"] - (s["cu"][1:] - s["cu"][:-1])
    positions = prefix[:, None] + seen.sum(-1) - 1
    return mask.flatten(0, 1)[s["flat"]], positions.flatten()[s["flat"]].int()


def _history(s, pool):
    """The f32 rows [B, Hkv, keys, D] that the block tables name."""
    at = s["tables"].long()
    if s["case"]["pool"] == "mxfp4":
        codes, scales = _pool_parts(pool, s["case"], s["pool"])
        return _four_bit_values(codes[at], scales[at]).transpose(1, 2).flatten(2, 3)
    return pool[at].float().transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    hq, hkv, d, _ = MODELS[s["case"]["model"]]
    k = _history(s, s["k"])
    q = s["q"][s["padded"]].unflatten(2, (hkv, -1)).permute(0, 2, 3, 1, 4)  # [B, Hkv, G, Q, D]
    g, n = q.shape[2:4]
    x = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)) * d ** -0.5  # [B, Hkv, G Q, keys]
    # key p of a sequence: the prefix's, or node p - prefix of its tree
    prefix = (s["lens"] - (s["cu"][1:] - s["cu"][:-1])).long()[:, None]
    node = torch.arange(k.shape[2], device=k.device) - prefix  # [B, keys]
    tree = (node >= 0) & (node < (s["cu"][1:] - s["cu"][:-1])[:, None])
    words = s["mask"][s["padded"]]  # [B, Q, words]
    word = words.gather(2, (node.clamp(0, s["widest"] - 1) // 64)[:, None].expand(-1, n, -1))
    seen = (node < 0)[:, None] | (tree[:, None] & ((word >> (node.clamp(min=0) % 64)[:, None]) & 1).bool())
    x = x.unflatten(2, (g, n)).masked_fill(~seen[:, None, None], -math.inf).flatten(2, 3)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    x = torch.matmul(e / e.sum(-1, keepdim=True), _history(s, s["v"]))
    return x.unflatten(2, (g, n)).permute(0, 3, 1, 2, 4).reshape(-1, hq, d)[s["flat"]]


def _children(s):
    """The children of every node [B, N, most], in order; -1 behind the last."""
    parents = _batched(s, s["parents"], -1).long()
    n = parents.shape[1]
    order = torch.arange(n, device=parents.device)
    rank = ((parents[:, :, None] == parents[:, None, :]) & (order[:, None] > order)).sum(-1)
    # those without a parent go to a row of their own
    kids = torch.full((parents.shape[0], (n + 1) * s["most"]), -1, dtype=torch.int64, device=parents.device)
    at = torch.where(parents < 0, torch.full_like(parents, n), parents) * s["most"] + rank.clamp(max=s["most"] - 1)
    return kids.scatter_(1, at, order.expand_as(at)).view(-1, n + 1, s["most"])[:, :n]


def _plain_verify(s):
    case = s["case"]
    first, kids, nodes = s["cu"][:-1].long(), _children(s), s["cu"][1:] - s["cu"][:-1]
    batch = torch.arange(first.numel(), device=first.device)
    index = torch.arange(s["logits"].shape[1], device=first.device)
    greedy, u = (s["temperature"] <= 0)[:, None], s["accept"].double()
    heat = s["temperature"].double().clamp(min=EPSILON)[:, None]
    path = torch.full_like(s["path"], -1)
    tokens, prob = torch.full_like(s["out_tokens"], -1), torch.zeros_like(s["prob"], dtype=torch.float64)
    at, count, alive = torch.zeros_like(first), torch.zeros_like(first), nodes > 0
    for step in range(s["deepest"] + 1):
        # the model's distribution at the node: where greedy, all on the first of the largest
        x = s["logits"][first + at].double()
        top = x.amax(-1, keepdim=True)
        best = torch.where(x == top, index, index.numel()).amin(-1, keepdim=True)
        w = torch.exp((x - top) / heat)
        sure = 1 / torch.exp(x - top).sum(-1)
        p = torch.where(greedy, (index == best).double(), w / w.sum(-1, keepdim=True))
        left, mass, moved, to = p, torch.ones_like(prob), torch.zeros_like(alive), at
        part, taken = torch.zeros_like(prob), torch.zeros_like(prob)
        q = None if s["probs"] is None else torch.where(greedy, 0.0, s["probs"][first + at].double())
        for r in range(s["most"] if step < s["deepest"] else 0):
            kid = kids[batch, at, r]
            row = first + kid.clamp(min=0)
            drafted = s["tokens"][row].long()[:, None]
            can = alive & ~moved & (kid >= 0) & (taken < 1)
            if q is None:  # a given token: accepted with its probability, otherwise out of the distribution
                weight, sized = torch.ones_like(prob), mass
            else:  # drawn from q: accepted with min(1, p / q), otherwise q is taken off p
                weight, sized = torch.where(greedy[:, 0], 1.0, q.gather(1, drafted)[:, 0]), mass / (1 - taken)
            yes = can & (u[row] * sized * weight < left.gather(1, drafted)[:, 0])
            no = can & ~yes
            if q is None:
                left = left.masked_fill(no[:, None] & (index == drafted), 0)
            else:
                part = part + torch.where(no, sized, 0.0)
                left = torch.where(no[:, None], (p - part[:, None] * q).clamp(min=0), left)
                taken = taken + (torch.where(no, q.gather(1, drafted)[:, 0], 0.0) if case["drafts"] == "distinct" else 0)
            mass = left.sum(-1)
            moved, to = moved | yes, torch.where(yes, kid, to)
        # where the path ends: the first token at which the sum passes the given share
        left = torch.where((mass > 0)[:, None], left, p)
        total = left.cumsum(-1)
        pick = (total <= s["pick"].double()[:, None] * total[:, -1:]).sum(-1)
        pick = torch.minimum(pick, torch.where(left > 0, index, -1).amax(-1))
        ended, at_count = alive & ~moved, count[:, None]
        chosen = torch.where(moved, s["tokens"][first + to].long(), pick)
        here = torch.arange(tokens.shape[1], device=first.device) == at_count
        tokens = torch.where(here & alive[:, None], chosen[:, None].int(), tokens)
        path = torch.where(here[:, :-1] & moved[:, None], to[:, None].int(), path)
        odds = torch.where(greedy[:, 0], sure, left.gather(1, pick[:, None])[:, 0] / total[:, -1])
        prob = torch.where(ended, odds, prob)
        count, at, alive = count + moved.long(), to, alive & moved
    return dict(tokens=tokens, path=path, count=count.int(), prob=prob.float())


def _plain_keep(s):
    path = s["path"].long()
    prefix = (s["lens"] - (s["cu"][1:] - s["cu"][:-1])).long()[:, None]
    to = 1 + torch.arange(path.shape[1], device=path.device)
    # places behind the path's end move node 0 onto itself
    src, dst = prefix + path.clamp(min=0), prefix + torch.where(path < 0, 0, to)
    src_block, dst_block = (s["tables"].long().gather(1, x // BLOCK).flatten() for x in (src, dst))
    src_row, dst_row = (src % BLOCK).flatten(), (dst % BLOCK).flatten()
    for pool in (s["k"], s["v"]):
        pool[:, dst_block, :, dst_row] = pool[:, src_block, :, src_row]
    return s["k"], s["v"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "attend": _own_attend, "verify": _own_verify, "keep": _own_keep}[op](state)
    return {"plan": _plain_plan, "attend": _plain_attend, "verify": _plain_verify, "keep": _plain_keep}[op](state)


# ---------------------------------------------------------------- the definition, in 64 bits

def _defined_rows(s, pool, b, n):
    """Rows [n, Hkv, D] of sequence b."""
    _, hkv, d, _ = MODELS[s["case"]["model"]]
    at = s["tables"][b, :-(-n // BLOCK)].long()
    if s["case"]["pool"] != "mxfp4":
        return pool[at].double().transpose(1, 2).reshape(-1, hkv, d)[:n]
    codes, scales = (x[at] for x in _pool_parts(pool, s["case"], s["pool"]))
    nibble = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    value = torch.where(nibble >= 8, -1.0, 1.0) * torch.tensor(LADDER, dtype=torch.float64, device=codes.device)[nibble % 8]
    value = value * torch.pow(2.0, scales.double() - 127).repeat_interleave(GROUP, -1)
    return value.transpose(1, 2).reshape(-1, hkv, d)[:n]


def _defined_softmax(x):
    """By exp: softmax itself is off by 1e-7 in 64 bits on the GPU."""
    e = torch.exp(x - x.max(-1, keepdim=True).values)
    return e / e.sum(-1, keepdim=True)


def _defined_attend(case, seed, s):
    hq, hkv, d, _ = MODELS[case["model"]]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    cu = s["cu"].tolist()
    for b, (parents, n) in enumerate(zip(_trees(case, seed), s["lens"].tolist())):
        k, v = _defined_rows(s, s["k"], b, n), _defined_rows(s, s["v"], b, n)
        prefix = n - len(parents)
        hidden = np.zeros((len(parents), n), bool)
        hidden[:, prefix:] = True
        for i in range(len(parents)):
            j = i
            while j >= 0:
                hidden[i, prefix + j] = False
                j = parents[j]
        hidden = torch.from_numpy(hidden).cuda()
        for h in range(hq):
            x = s["q"][cu[b]:cu[b + 1], h].double() @ k[:, h // (hq // hkv)].T.contiguous() / math.sqrt(d)
            x[hidden] = -math.inf
            out[cu[b]:cu[b + 1], h] = _defined_softmax(x) @ v[:, h // (hq // hkv)].contiguous()
    return out


def _defined_distribution(logits, temperature):
    if temperature <= 0:
        first = int((logits == logits.max()).nonzero()[0, 0])
        p = torch.zeros_like(logits)
        p[first] = 1
        return p, float(_defined_softmax(logits)[first])
    return _defined_softmax(logits / max(temperature, EPSILON)), None


def _defined_verify(case, seed, s):
    out = dict(tokens=torch.full_like(s["out_tokens"], -1), path=torch.full_like(s["path"], -1),
               count=torch.zeros_like(s["count"]), prob=torch.zeros_like(s["prob"], dtype=torch.float64))
    cu, tokens, heat = s["cu"].tolist(), s["tokens"].tolist(), s["temperature"].tolist()
    u, last = s["accept"].tolist(), s["pick"].tolist()
    for b, parents in enumerate(_trees(case, seed)):
        node, steps = 0, 0
        while True:
            p, sure = _defined_distribution(s["logits"][cu[b] + node].double(), heat[b])
            q = None if s["probs"] is None or heat[b] <= 0 else s["probs"][cu[b] + node].double()
            rest, drafted, found, taken = p, q, None, []
            for kid in [i for i, parent in enumerate(parents) if parent == node]:
                x = tokens[cu[b] + kid]
                odds = float(rest[x]) if q is None else float(rest[x] / drafted[x]) if drafted[x] > 0 else math.inf
                if u[cu[b] + kid] < odds:
                    found = kid
                    break
                rest = rest.clone()
                if q is None:
                    rest[x] = 0
                else:
                    rest = (rest - drafted).clamp(min=0)
                    if case["drafts"] == "distinct":
                        taken.append(x)
                        drafted = q / (1 - float(q[taken].sum()))
                        drafted[taken] = 0
                rest = rest / rest.sum()
            if found is None:
                total = rest.cumsum(-1)
                x = int((total > last[b] * total[-1]).nonzero()[0, 0])
                out["tokens"][b, steps], out["prob"][b] = x, float(rest[x]) if sure is None else sure
                out["count"][b] = steps
                break
            out["path"][b, steps], out["tokens"][b, steps] = found, tokens[cu[b] + found]
            node, steps = found, steps + 1
    return out


def exact(case, seed):
    if case["op"] == "plan":
        trees = _trees(case, seed)
        deep = []
        for prefix, parents in zip(_histories(case, seed).tolist(), trees):
            here = []
            for p in parents:
                here.append(prefix if p < 0 else here[p] + 1)
            deep += here
        return _masks(trees, -(-max(map(len, trees)) // 64)), _device(deep, np.int32)
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _defined_attend(case, seed, s)
    if case["op"] == "verify":
        return _defined_verify(case, seed, s)
    pools = []
    cu, path, lens, tables = (s[x].tolist() for x in ("cu", "path", "lens", "tables"))
    for pool in (s["k"], s["v"]):
        new = pool.double()
        for b in range(len(lens)):
            prefix = lens[b] - (cu[b + 1] - cu[b])
            for i, node in enumerate(x for x in path[b] if x >= 0):
                src, dst = prefix + node, prefix + 1 + i
                new[:, tables[b][dst // BLOCK], :, dst % BLOCK] = pool[:, tables[b][src // BLOCK], :, src % BLOCK].double()
        pools.append(new)
    return tuple(pools)
