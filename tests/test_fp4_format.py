"""The 4-bit KV format without a GPU: the reference's own rounding against a search over every
code, pool sizes, and the refusals that are made before a device is looked at."""
import ctypes as C

import numpy as np
import pytest

import fp4_reference as fp4


def test_rounding_is_the_nearest_value_of_the_smallest_fitting_scale():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((400, 64)) * np.exp(rng.standard_normal((400, 1)) * 15)).astype(np.float32)
    codes, scales = fp4.quantise(x)
    v = fp4.values(codes, scales).reshape(400, 2, 32)
    g = x.astype(np.float64).reshape(400, 2, 32)
    s = np.exp2(scales.astype(np.float64) - 127)[..., None]
    top = np.abs(g).max(-1, keepdims=True)
    assert (top < 7 * s).all() and (top >= 3.5 * s).all()  # the smallest power of two with top < 7 s
    every = np.concatenate([fp4.LADDER, -fp4.LADDER]) * s[..., None]
    assert np.array_equal(np.abs(g - v), np.abs(g[..., None] - every).min(-1))
    step = np.where(np.abs(v) < 2 * s, 0.5, np.where(np.abs(v) < 4 * s, 1.0, 2.0)) * s
    assert (np.abs(g - v) <= step / 2 + 1e-300).all()


def test_rounding_at_ties_and_ends():
    x = np.zeros((1, 32), np.float32)
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.9]
    x[0, 31] = -0.0
    codes, scales = fp4.quantise(x)
    assert scales[0, 0] == 127
    assert fp4.values(codes, scales)[0, :8].tolist() == [0, 1, 1, 2, 2, 4, 4, 6]
    assert codes[0, 15] == 0x80  # the sign of zero is kept
    for value, scale, read in [(0.0, 2, 0.0), (1e-45, 2, 0.0), (3.4e38, 252, 6.0 * 2.0 ** 125), (np.inf, 255, np.nan),
                               (np.nan, 255, np.nan), (7.0, 128, 8.0), (6.999999, 127, 6.0)]:
        y = np.zeros((1, 32), np.float32)
        y[0, 3] = value
        codes, scales = fp4.quantise(y)
        got = fp4.values(codes, scales)[0, 3]
        assert scales[0, 0] == scale and (got == read or np.isnan(read) and np.isnan(got)), (value, scales, got)


def test_pool_sizes():
    from ferrisinfer_amd import DTYPE_BF16, DTYPE_F16, DTYPE_F32, DTYPE_MXFP4, FerrisError, kv_pool_bytes

    assert kv_pool_bytes(DTYPE_MXFP4, 7, 16, 8, 128) == 7 * 16 * 8 * (64 + 4)
    assert kv_pool_bytes(DTYPE_MXFP4, 3, 5, 2, 32) == 3 * 5 * 2 * 17
    assert kv_pool_bytes(DTYPE_MXFP4, 1 << 20, 16, 8, 128) == (1 << 27) * 68  # past 32 bits
    assert kv_pool_bytes(DTYPE_F32, 3, 5, 2, 32) == 3 * 5 * 2 * 128
    assert kv_pool_bytes(DTYPE_BF16, 3, 5, 2, 40) == 3 * 5 * 2 * 80
    for args, kind in [((DTYPE_F16, 3, 5, 2, 32), "InvalidType"), ((4, 3, 5, 2, 32), "InvalidType"),
                       ((DTYPE_MXFP4, 3, 5, 2, 48), "Unsupported"), ((DTYPE_MXFP4, 3, 5, 2, 256), "Unsupported"),
                       ((DTYPE_MXFP4, 0, 5, 2, 32), "InvalidConfig"), ((DTYPE_F32, 3, -1, 2, 32), "InvalidConfig")]:
        with pytest.raises(FerrisError) as e:
            kv_pool_bytes(*args)
        assert e.value.kind == kind, args


def _consume(**change):
    """fi_qkv_norm_rope_append without a context: its refusal, by the checks made before a device."""
    from ferrisinfer_amd import kernel

    a = dict(splits=1, eps=1e-6, axes=1, pair_axes=None, rotary=64, pool=2, dtype=0, blocks=4, bs=16, tokens=3, hq=4,
             hkv=2, d=64, weight=None)
    a.update(change)
    named = None if a["pair_axes"] is None else (C.c_int32 * len(a["pair_axes"]))(*a["pair_axes"])
    with pytest.raises(kernel.FerrisError) as e:
        kernel.check(kernel.load().fi_qkv_norm_rope_append(
            None, None, a["splits"], None, None, None, a["weight"], None, a["eps"], None, a["axes"], named, None, None,
            a["rotary"], 64, None, None, None, a["dtype"], a["blocks"], a["bs"], a["tokens"], a["hq"], a["hkv"], a["d"],
            None))
    return e.value.kind, e.value.message


@pytest.mark.parametrize("change,kind,words", [
    (dict(splits=0), "InvalidShape", "bad shape"),
    (dict(tokens=-1), "InvalidShape", "bad shape"),
    (dict(hq=5), "InvalidShape", "divisible"),
    (dict(hkv=0), "InvalidShape", "divisible"),
    (dict(d=48, rotary=48), "Unsupported", "head_dim"),
    (dict(d=256), "Unsupported", "head_dim"),
    (dict(rotary=66), "InvalidConfig", "rotary_dims"),
    (dict(rotary=7), "InvalidConfig", "rotary_dims"),
    (dict(rotary=-8), "InvalidConfig", "rotary_dims"),
    (dict(rotary=12), "Unsupported", "multiple of 4"),
    (dict(blocks=0), "InvalidConfig", "pool"),
    (dict(bs=0), "InvalidConfig", "pool"),
    (dict(dtype=2), "InvalidType", "KV dtype"),
    (dict(dtype=4), "InvalidType", "KV dtype"),
    (dict(axes=0), "InvalidConfig", "axes"),
    (dict(axes=5, pair_axes=[0] * 32), "InvalidConfig", "axes"),
    (dict(axes=2), "InvalidConfig", "each pair's axis"),
    (dict(axes=2, pair_axes=[0] * 31 + [2]), "InvalidConfig", "pair 31"),
    (dict(axes=3, pair_axes=[0] * 5 + [-1] + [0] * 26), "InvalidConfig", "pair 5"),
    (dict(weight=16, eps=-1e-6), "InvalidConfig", "eps"),
    (dict(weight=16, eps=float("nan")), "InvalidConfig", "eps"),
    (dict(weight=16, eps=float("inf")), "InvalidConfig", "eps"),
    (dict(tokens=2 ** 31 - 1, hq=64, hkv=64, d=128, rotary=128), "InvalidShape", "too many tokens"),
    (dict(tokens=1, hq=2 ** 24, hkv=2 ** 24, d=128, rotary=128), "InvalidShape", "too wide"),
])
def test_consumer_refusals(change, kind, words):
    got, message = _consume(**change)
    assert got == kind and words in message, (got, message)


def test_consumer_of_a_four_bit_pool_keeps_its_name_in_refusals():
    from ferrisinfer_amd import DTYPE_MXFP4, kernel

    with pytest.raises(kernel.FerrisError) as e:
        kernel.check(kernel.load().fi_qkv_rope_append(None, None, 1, None, None, None, None, None, None, 12, 64, None,
                                                      None, None, DTYPE_MXFP4, 4, 16, 3, 4, 2, 64, None))
    assert e.value.kind == "Unsupported" and e.value.message.startswith("fi_qkv_rope_append")
