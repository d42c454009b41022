"""How far f32 attention over a 4-bit pool is from the 64-bit one, as a size to be expected and not
as a worst case: a kernel that keeps fewer than three bf16 pieces of its queries or probabilities, or
leaves out a key, is farther off (test_fp4_accuracy.py holds that against simulations of such kernels).

Each rounding is off by up to half a step u = 2^-24 of its result, evenly either way: u / sqrt(3) in
the mean square, and roundings add in squares.  For a row with weights p_j over values v_j, o = sum p_j v_j:

  * the score s_j is added up in steps of 32 products (three a product where the pieces are products of
    their own), each of which may round twice, at sums of about size a_j = sqrt(sum (q k scale)^2) and
    |s_j|, then scaled (|s_j|); the exponent's argument and the constant it is scaled by round at
    |s_j - max|; the exponential is within 2 u.  A weight's relative error e_j moves the output by
    p_j e_j (v_j - o).
  * `additions` roundings of the weighted sum and of the weights' sum, at running sums whose mean square
    is half of the last one's (|o|^2 + sum p_j^2 |v_j|^2), and six more to join, invert and scale.
"""
import numpy as np

U = 2.0 ** -24
TENSOR, ROW = 3.0, 6.0  # how many times its size the error may be, over a sequence and in one row


def expected(q, k, v, first, scale, additions):
    """(o, r): the 64-bit output [n, Hq, D] of q [n, Hq, D] at positions first .. over k, v [keys, Hkv, D], and
    the size [n, Hq] of the f32 error's 2-norm."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    out, err = np.empty(q.shape), np.empty((n, hq))
    q = q.astype(np.float64)
    hidden = np.arange(k.shape[0])[None] > first + np.arange(n)[:, None]
    for h in range(hq):
        kh, vh = k[:, h // group], v[:, h // group]
        s = q[:, h] @ kh.T * scale
        a2 = (q[:, h] ** 2) @ (kh ** 2).T * scale ** 2
        x = np.where(hidden, -np.inf, s)
        x = x - x.max(1, keepdims=True)
        p = np.exp(x)
        p /= p.sum(1, keepdims=True)
        o = p @ vh
        x = np.where(hidden, 0.0, x)
        steps = 2 * 3 * d / 32
        e2 = steps * (a2 + s * s) + s * s + 2 * x * x + 12
        o2, v2 = (o * o).sum(1), (vh * vh).sum(1)
        apart = np.maximum(v2[None] - 2 * o @ vh.T + o2[:, None], 0)
        p2 = p * p
        err[:, h] = np.sqrt((p2 * e2 * apart).sum(1) + (additions / 2 + 6) * (o2 + p2 @ v2)) * U / np.sqrt(3)
        out[:, h] = o
    return out, err


def decode_additions(keys):
    """A wave adds at most 8 times, pieces 2 and waves 4 times, the partitions (512 or 256 keys) in four strands."""
    return 20 + keys / 1024


def prefill_additions(keys):
    """Three products for each 32 keys; ranges of keys are joined by fewer additions than they save."""
    return 6 * (keys / 64 + 1)


def check(got, q, k, v, first, scale, additions, what=""):
    want, err = expected(q, k, v, first, scale, additions)
    off = np.sqrt(((got.astype(np.float64) - want) ** 2).sum(-1))
    total, size = np.sqrt((off ** 2).sum()), np.sqrt((err ** 2).sum())
    assert total <= TENSOR * size, (what, "sequence", total / size, total / np.sqrt((want ** 2).sum()))
    worst = (off / err).max()
    assert worst <= ROW, (what, "row", worst)
