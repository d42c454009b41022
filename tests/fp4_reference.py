"""4-bit KV pools in numpy: the format of FI_DTYPE_MXFP4 and attention over it, in 64 bits."""
import numpy as np

LADDER = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
GROUP = 32
HALF = 2.0 ** -24  # half a step of f32, relative


def quantise(x):
    """f32 [..., D] -> (codes uint8 [..., D / 2], scales uint8 [..., D / 32])."""
    g = np.asarray(x, np.float32).astype(np.float64).reshape(*x.shape[:-1], -1, GROUP)
    fine = np.isfinite(g).all(-1, keepdims=True)
    top = np.abs(np.where(fine, g, 0.0)).max(-1, keepdims=True)
    mantissa, e = np.frexp(top)  # top = mantissa * 2^e, mantissa in [0.5, 1)
    e = np.where(top == 0, -200, e - 1 - 2 + (mantissa >= 0.875))  # 2^e: the smallest scale with top < 7 * 2^e
    e = np.clip(e, -125, 125)
    a = np.abs(np.where(fine, g, 0.0)) / np.exp2(e.astype(np.float64))
    code = np.zeros(a.shape, np.uint8)
    for i, (lo, hi) in enumerate(zip(LADDER[:-1], LADDER[1:])):
        middle = (lo + hi) / 2
        code += (a > middle) | ((a == middle) & (i % 2 == 1))  # ties to the even code
    code |= (np.signbit(g) & fine).astype(np.uint8) << 3
    code = code.reshape(*x.shape)
    scales = np.where(fine, e + 127, 255).astype(np.uint8)[..., 0]
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def values(codes, scales):
    """The values of codes and scales, in f64."""
    nibble = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = LADDER[nibble & 7] * np.where(nibble & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(s, GROUP, -1)


def pool_bytes(codes, scales):
    """A pool array's bytes from codes [nb, hkv, bs, d / 2] and scales [nb, hkv, bs, d / 32]."""
    return np.concatenate([codes.reshape(-1), scales.reshape(-1)])


def split_pool(pool, nb, hkv, bs, d):
    """(codes, scales) views of a pool array's bytes."""
    n = nb * hkv * bs * (d // 2)
    return pool[:n].reshape(nb, hkv, bs, d // 2), pool[n:].reshape(nb, hkv, bs, d // GROUP)


def rows_of(pool_values, table, length, bs):
    """[length, Hkv, D] of one sequence from pool values [nb, hkv, bs, d]."""
    t = np.arange(length)
    return pool_values[np.asarray(table)[t // bs], :, t % bs]


def attention(q, k, v, first, scale):
    """q [n, Hq, D] at positions first .. over k, v [keys, Hkv, D]; query i sees keys <= first + i."""
    n, hq, _ = q.shape
    group = hq // k.shape[1]
    out = np.empty(q.shape)
    q = q.astype(np.float64)
    for h in range(hq):
        s = (q[:, h] @ k[:, h // group].T) * scale
        for i in range(n):
            keys = min(first + i + 1, k.shape[0])
            x = s[i, :keys]
            p = np.exp(x - x.max()) if keys else x
            out[i, h] = (p @ v[:keys, h // group]) / p.sum() if keys else 0.0
    return out


def attention_tolerance(q, k, v, scale, keys):
    """How far an f32 attention may be from the 64-bit one, absolutely.  A score is a sum of D
    products kept in f32: off by at most (D + 4) half steps of sum |q k|, which moves every weight
    by that much relative to itself, in numerator and denominator; the exponentials of scores below
    their maximum are off by 4 steps and, through the rounding of an argument of size x, x half steps
    more; the weighted sum and the weights' sum over n keys are each off by a half step per level of
    the pieces they are added in (at most n).  All of it times the largest |V|."""
    d = q.shape[-1]
    big = max(float(np.abs(k[..., h, :]).max(initial=0.0)) for h in range(k.shape[-2]))
    s = float(np.abs(q).sum(-1).max()) * big * scale
    relative = 2 * ((d + 4) * s + 2 * s + 8) + 2 * min(keys, 256) + 2 * keys / 64
    return relative * HALF * float(np.abs(v).max(initial=0.0)) + 1e-30
