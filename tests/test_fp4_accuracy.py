"""That the tolerance of fp4_accuracy.py tells f32 attention over a 4-bit pool from attention with fewer
pieces or fewer keys: both simulated in numpy, with the kernels' products and the order of their sums."""
import numpy as np
import pytest

import fp4_accuracy as acc
import fp4_reference as fp4


def bf16(x):
    bits = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)


def pieces(x, count):
    x, out = np.asarray(x, np.float32), []
    for _ in range(count):
        out.append(bf16(x))
        x = x - out[-1]
    return out[::-1]  # smallest first


def simulate(q, k, v, first, scale, q_pieces=3, p_pieces=3, wave=128):
    """f32 attention of q [n, Hq, D]: products of pieces in steps of 32, f32 sums, waves of `wave` keys joined
    by their maxima."""
    n, hq, d = q.shape
    f32 = np.float32
    out = np.empty(q.shape, f32)
    hidden = np.arange(k.shape[0])[None] > first + np.arange(n)[:, None]
    for h in range(hq):
        kh, vh = (x[:, h * k.shape[1] // hq].astype(f32) for x in (k, v))
        s = np.zeros((n, len(kh)), f32)
        for c in range(0, d, 32):
            for piece in pieces(q[:, h, c:c + 32], q_pieces):
                s += (piece.astype(np.float64) @ kh[:, c:c + 32].T.astype(np.float64)).astype(f32)
        s = np.where(hidden, f32(-np.inf), s * f32(scale * 1.4426950408889634))
        point = s.max(1, keepdims=True)
        p = np.exp2((s - point).astype(np.float64)).astype(f32)
        total, weight = np.zeros((n, d), f32), np.zeros(n, f32)
        for w in range(0, len(kh), wave):
            o = np.zeros((n, d), f32)
            for c in range(w, min(w + wave, len(kh)), 32):
                for piece in pieces(p[:, c:min(c + 32, w + wave)], p_pieces):
                    o += (piece.astype(np.float64) @ vh[c:min(c + 32, w + wave)].astype(np.float64)).astype(f32)
            total += o
            weight += p[:, w:w + wave].sum(1, dtype=f32)
        out[:, h] = total * (f32(1) / weight)[:, None]
    return out


def refused(*args):
    try:
        acc.check(*args)
    except AssertionError:
        return True
    return False


DECODE = [(33, 2, 2, 32), (65, 14, 2, 64), (129, 14, 2, 64), (257, 14, 2, 64), (700, 14, 2, 64), (1025, 32, 8, 128),
          (300, 8, 1, 128), (90, 5, 1, 64), (333, 6, 2, 128), (77, 3, 1, 32), (2050, 16, 4, 128), (4000, 7, 1, 32),
          (16384, 7, 1, 64)]
PREFILL = [(0, 65, 2, 2, 32), (29, 61, 14, 2, 64), (100, 20, 14, 2, 64), (511, 130, 8, 2, 128), (0, 200, 8, 1, 128),
           (40, 77, 5, 1, 64), (1, 300, 6, 2, 128), (300, 257, 4, 1, 128)]


def inputs(keys, rows, hq, hkv, d):
    rng = np.random.default_rng(keys + d)
    k, v = (fp4.values(*fp4.quantise(rng.standard_normal((keys, hkv, d)).astype(np.float32))) for _ in range(2))
    return rng.standard_normal((rows, hq, d)).astype(np.float32), k, v


@pytest.mark.parametrize("shape", DECODE + PREFILL, ids=str)
def test_tolerance_refuses_fewer_pieces_and_keys(shape):
    cached, rows, (hq, hkv, d) = (shape[0] - 1, 1, shape[1:]) if len(shape) == 4 else (shape[0], shape[1], shape[2:])
    keys, scale = cached + rows, d ** -0.5
    q, k, v = inputs(keys, rows, hq, hkv, d)
    additions = (acc.decode_additions if len(shape) == 4 else acc.prefill_additions)(keys)
    tail = (q, k, v, cached, scale, additions)
    wave = 128 if len(shape) == 4 else keys
    acc.check(simulate(q, k, v, cached, scale, wave=wave), *tail)
    for fewer in ((2, 3), (3, 2), (1, 3), (3, 1)):
        assert refused(simulate(q, k, v, cached, scale, *fewer, wave=wave), *tail), fewer
    # without the last key of the last row, and without one in the middle
    assert refused(np.concatenate([simulate(q[:-1], k, v, cached, scale, wave=wave), simulate(
        q[-1:], k[:-1], v[:-1], keys, scale, wave=wave)]) if rows > 1 else simulate(q, k[:-1], v[:-1], keys, scale), *tail)
    half = keys // 2
    less_k, less_v = (np.delete(x, half, 0) for x in (k, v))
    assert refused(simulate(q, less_k, less_v, max(cached - 1, 0), scale, wave=wave), *tail)


@pytest.mark.parametrize("size", [3.0, 20.0])
def test_tolerance_holds_for_large_scores(size):
    q, k, v = inputs(513, 1, 8, 2, 128)
    k = fp4.values(*fp4.quantise((k * size).astype(np.float32)))
    tail = (q, k, v, 512, 128 ** -0.5, acc.decode_additions(513))
    acc.check(simulate(q, k, v, 512, 128 ** -0.5), *tail)
    assert refused(simulate(q, k, v, 512, 128 ** -0.5, 2, 3), *tail)
