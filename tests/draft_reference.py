"""Trees of drafted tokens in numpy, 64 bits: masks, attention over them with the size of an f32 error, and
the verification's definition, one child after the other."""
import math

import numpy as np

U = 2.0 ** -24  # half a step of f32, relative
TENSOR, ROW = 3.0, 6.0  # how many times its size the error may be, over a sequence and in one row


def grown(rng, nodes, width=3):
    """Parents of a random tree: each node behind one of the last `width` or any before it."""
    return ([-1] + [int(rng.integers(max(0, i - width), i)) if rng.random() < 0.7 else int(rng.integers(0, i))
                    for i in range(1, nodes)])[:nodes]


def ancestors(parents):
    """bool [n, n]: node i's ancestors and itself."""
    seen = np.zeros((len(parents),) * 2, bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def words_of(seen, words):
    """int64 [n, words] of bool [n, nodes]."""
    bits = np.zeros((seen.shape[0], 64 * words), np.uint64)
    bits[:, :seen.shape[1]] = seen
    return (bits.reshape(-1, words, 64) << np.arange(64, dtype=np.uint64)).sum(-1, dtype=np.uint64).view(np.int64)


def visible(seen, prefix, keys):
    """bool [n, keys]: what each node attends, of positions 0 .. keys - 1."""
    out = np.zeros((seen.shape[0], keys), bool)
    out[:, :max(prefix, 0)] = True
    for j in range(seen.shape[1]):
        if 0 <= prefix + j < keys:
            out[:, prefix + j] = seen[:, j]
    return out


def expected(q, k, v, shown, scale, additions, pieces):
    """(o, r): the 64-bit output [n, Hq, D] of q [n, Hq, D] over the keys of k, v [keys, Hkv, D] that shown
    [n, keys] has set (zero where there is none), and the size [n, Hq] of the f32 error's 2-norm.

    Each rounding is off by up to half a step U of its result, U / sqrt(3) in the mean square, and roundings add in
    squares.  A score is added up in `pieces` products for each 32 elements, two roundings each, at sums of
    about a = sqrt(sum (q k scale)^2) and |s|, then scaled; the exponent's argument and the constant it is scaled
    by round at |s - max|; the exponential is within 2 U.  A weight's relative error e moves the output by
    p e (v - o).  `additions` roundings of the weighted sum and of the weights' sum fall on running sums whose mean
    square is half of the last one's, |o|^2 + sum p^2 |v|^2, and six more join, invert and scale.  Where K and V
    are split too (six pieces), three cross products below 2^-24 of q k (of p v) are left out: half of one
    rounding each at a, three at the weighted sum."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    out, err = np.zeros(q.shape), np.full((n, hq), 1e-300)
    q = q.astype(np.float64)
    some = shown.any(1)
    split = 3 if pieces > 3 else 0
    for h in range(hq):
        kh, vh = k[:, h // group], v[:, h // group]
        with np.errstate(invalid="ignore"):
            s = np.where(shown, q[:, h] @ kh.T * scale, -np.inf)[some]
        a2 = (q[some, h] ** 2) @ (kh ** 2).T * scale ** 2
        x = s - s.max(1, keepdims=True, initial=-np.inf)
        p = np.exp(x)
        p /= p.sum(1, keepdims=True)
        o = p @ vh
        x, s = np.where(shown[some], x, 0.0), np.where(shown[some], s, 0.0)
        e2 = (2 * pieces * d / 32) * (a2 + s * s) + split * a2 + s * s + 2 * x * x + 12
        o2, v2 = (o * o).sum(1), (vh * vh).sum(1)
        apart = np.maximum(v2[None] - 2 * o @ vh.T + o2[:, None], 0)
        p2 = p * p
        err[some, h] += np.sqrt((p2 * e2 * apart).sum(1) + (additions / 2 + 6 + split) * (o2 + p2 @ v2)) * U / np.sqrt(3)
        out[some, h] = o
    return out, err


def additions(keys, pieces):
    """`pieces` products for each 32 keys, and parts of four chunks and more joined."""
    return 2 * pieces * (keys / 64 + 1)


def check_attention(got, q, k, v, shown, scale, pieces, what=""):
    want, err = expected(q, k, v, shown, scale, additions(shown.shape[1], pieces), pieces)
    off = np.sqrt(((got.astype(np.float64) - want) ** 2).sum(-1))
    total, size = np.sqrt((off ** 2).sum()), np.sqrt((err ** 2).sum())
    assert total <= TENSOR * size, (what, "sequence", total / size, total / np.sqrt((want ** 2).sum()))
    assert (off / err).max() <= ROW, (what, "row", (off / err).max())


# ---------------------------------------------------------------- verification

def distribution(logits, temperature):
    """p of a row, or None where there is none."""
    x = np.asarray(logits, np.float64)
    if temperature <= 0:
        p = np.zeros(x.size)
        best = np.nanargmax(np.where(np.isnan(x), -np.inf, x))
        if x[best] == -np.inf:
            return None
        p[best] = 1.0
        return p
    if not (x < np.inf).all() or x.max() == -np.inf:
        return None
    e = np.exp((x - x.max()) / max(float(temperature), 2.0 ** -23))
    return e / e.sum()


def verify(logits, tokens, parents, temperature, accept, pick, probs=None, distinct=False, max_path=None):
    """(tokens, path, probability) of one sequence: the accepted tokens and the last one (absent where a
    distribution fails), the accepted nodes, the last token's probability."""
    out, path, node = [], [], 0
    limit = len(tokens) if max_path is None else max_path
    temperature = np.float32(temperature)
    if len(tokens) == 0:
        return out, path, 0.0
    while True:
        p = distribution(logits[node], temperature)
        kids = [i for i, parent in enumerate(parents) if parent == node] if len(path) < limit else []
        if p is None:
            return out, path, 0.0
        q = None if probs is None or temperature <= 0 else np.asarray(probs[node], np.float64)
        rest, gone, found = p, [], None
        for kid in kids:
            x = int(tokens[kid])
            if not 0 <= x < p.size:
                continue
            u = float(accept[kid])
            if q is None:  # greedy: the random numbers do not count
                if rest[x] > 0 if temperature <= 0 else u * rest.sum() < rest[x]:
                    found = kid
                    break
                rest = rest.copy()
                rest[x] = 0.0
                continue
            now = q
            if distinct:
                spent = math.fsum(q[y] for y in gone)
                if spent >= 1:
                    continue
                now = q / (1 - spent)
                now[list(set(gone))] = 0.0
            share = rest / rest.sum()
            if u * now[x] < share[x]:
                found = kid
                break
            rest = np.maximum(share - now, 0.0)
            gone.append(x)
            if not rest.sum() > 0:
                rest = np.zeros(p.size)
                rest[0] = 0.0
                break
        if found is None:
            if not rest.sum() > 0:
                rest = p
            total = np.cumsum(rest)
            over = np.nonzero(total > float(pick) * total[-1])[0]
            last = int(over[0]) if over.size else int(np.nonzero(rest > 0)[0][-1])
            out.append(last)
            if temperature <= 0:
                x = np.asarray(logits[node], np.float64)
                return out, path, 1.0 / np.exp(x - x[last]).sum()
            return out, path, rest[last] / total[-1]
        out.append(int(tokens[found]))
        path.append(found)
        node = found
