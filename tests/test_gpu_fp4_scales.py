"""Every scale byte of the 4-bit KV format on the GPU: what appending writes and what reading gives."""
import numpy as np
import pytest

import fp4_reference as fp4
from test_gpu_fp4_cache import dev

pytestmark = pytest.mark.gpu

TIES = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)


def groups_of_every_scale():
    """f32 [N, 32]: for each scale 2^(E - 127), E from 2 to 252, groups that have it: every tie and its
    neighbours on both sides, of either sign, under largest values from 3.5 scales to just below 7; at the
    ends also subnormal groups and values up to the largest f32."""
    rng = np.random.default_rng(70)
    rows = []
    largest = np.finfo(np.float32).max
    for e in range(2, 253):
        s = np.float32(2.0 ** (e - 127))
        ties = TIES * s
        near = np.concatenate([ties, np.nextafter(ties, np.float32(0)), np.nextafter(ties, np.float32(np.inf))])
        tops = [3.5 * s, 4 * s, 6 * s, 6.5 * s, np.nextafter(np.float32(7 * s), np.float32(0))]
        if e == 2:  # below: the scale stays
            tops += [0.0, 2.0 ** -149, 2.0 ** -127, 2.0 ** -126, 3 * s]
        if e == 252:  # above: cut off
            tops += [7 * s, largest]
        for top in tops:
            row = np.zeros(32, np.float32)
            row[:21] = near
            row[21:31] = rng.uniform(0, 1, 10) * top
            row[np.abs(row) > top] = 0
            row[31] = top
            row *= rng.choice(np.array([-1, 1], np.float32), 32)
            rows.append(rng.permutation(row))
    return np.stack(rows)


@pytest.mark.parametrize("d", [32, 128])
@pytest.mark.parametrize("entry", ["append", "consumer"])
def test_appending_at_every_scale(gpu_ctx, entry, d):
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, kv_pool_bytes

    groups = groups_of_every_scale()
    groups = groups[:len(groups) // (d // 32) * (d // 32)]
    rows = groups.reshape(-1, 1, d)
    t, bs = len(rows), 16
    codes, scales = fp4.quantise(rows)
    assert set(range(2, 253)) <= set(scales.reshape(-1).tolist())
    nb = -(-t // bs)
    pools = [torch.zeros(kv_pool_bytes(DTYPE_MXFP4, nb, bs, 1, d), dtype=torch.uint8, device="cuda") for _ in range(2)]
    slots = np.arange(t, dtype=np.int64)
    value = rows[::-1].copy()
    if entry == "append":
        gpu_ctx.kv_append(dev(rows), dev(value), dev(slots), *pools, DTYPE_MXFP4, nb, bs, 1, d)
    else:  # no norm, no rotation: the rows themselves
        q = torch.empty(t, 1, d, device="cuda")
        parts = np.concatenate([rows, rows, value], -1).reshape(1, t, 3 * d)
        gpu_ctx.qkv_norm_rope_append(dev(parts), 1, None, None, 0.0, dev(np.zeros(t, np.int32)), None, None, None, 0, 0,
                                     dev(slots), *pools, DTYPE_MXFP4, nb, bs, 1, 1, d, q)
        assert np.array_equal(q.cpu().numpy(), rows)
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    for pool, c, s in ((pools[0], codes, scales), (pools[1], codes[::-1], scales[::-1])):
        got_c, got_s = fp4.split_pool(pool.cpu().numpy(), nb, 1, bs, d)
        got_c, got_s = got_c.reshape(nb * bs, -1)[:t], got_s.reshape(nb * bs, -1)[:t]
        bad = np.nonzero((got_s != s.reshape(t, -1)).any(1) | (got_c != c.reshape(t, -1)).any(1))[0]
        assert bad.size == 0, (bad[:8], s.reshape(t, -1)[bad[:8]])


def test_reading_every_scale(gpu_ctx):
    """All sixteen codes at every scale byte that a pool may hold (0 to 252, and 255: NaN)."""
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4

    kept = np.array([*range(253), 255], np.uint8)
    nb, bs, d = len(kept), 1, 32
    codes = np.tile(np.arange(16, dtype=np.uint8) * 16 + np.arange(16, dtype=np.uint8)[::-1], (nb, 1)).reshape(nb, 1, bs, d // 2)
    pool = dev(fp4.pool_bytes(codes, kept.reshape(nb, 1, bs, 1)))
    outs = [torch.empty(nb, 1, d, device="cuda") for _ in range(2)]
    gpu_ctx.kv_gather(pool, pool, DTYPE_MXFP4, dev(np.arange(nb, dtype=np.int32)), nb, nb, bs, 1, d, *outs)
    gpu_ctx.sync()
    want = fp4.values(codes, kept.reshape(nb, 1, bs, 1)).reshape(nb, 1, d)
    for out in outs:
        got = out.cpu().numpy().astype(np.float64)
        bad = np.nonzero(~((got == want) | (np.isnan(got) & np.isnan(want))).all((1, 2)))[0]
        assert bad.size == 0, kept[bad]


@pytest.mark.parametrize("e", [2, 3, 126, 250, 252])
def test_attention_at_the_scales_ends(gpu_ctx, e):
    """One key a row: the softmax is 1 and the output is the value row, whatever its scale.  Decode's weight is
    exactly 1; prefill's is 2^x for the rounding error x of the score's scaling, and its three-piece product
    with the value (two roundings), the reciprocal of the weights' sum and the product with it are off by half
    a step each."""
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4

    rng = np.random.default_rng(71)
    hkv, d, bs, nb = 2, 64, 4, 5
    codes = rng.integers(0, 256, (nb, hkv, bs, d // 2), dtype=np.uint8)
    value = dev(fp4.pool_bytes(codes, np.full((nb, hkv, bs, d // 32), e, np.uint8)))
    key = dev(fp4.pool_bytes(codes, np.full((nb, hkv, bs, d // 32), min(e, 127), np.uint8)))
    tables = rng.permutation(nb).astype(np.int32)[:, None]
    want = fp4.values(codes, np.full((nb, hkv, bs, d // 32), e, np.uint8))[tables[:, 0], :, 0]  # [nb, hkv, d]
    q = dev(rng.standard_normal((nb, 2 * hkv, d)).astype(np.float32))
    lens = dev(np.ones(nb, np.int32))
    for prefill in (False, True):
        out = torch.empty_like(q)
        if prefill:
            gpu_ctx.attn_prefill_paged(q, key, value, DTYPE_MXFP4, dev(tables), dev(np.arange(nb + 1, dtype=np.int32)), lens, 1,
                                       hkv, bs, nb, 0.125, out)
        else:
            gpu_ctx.attn_decode_paged(q, key, value, DTYPE_MXFP4, dev(tables), lens, 1, hkv, bs, nb, 0.125, out)
        gpu_ctx.sync()
        gpu_ctx.check_faults()
        off = np.abs(out.cpu().numpy().reshape(nb, hkv, 2, d) - want[:, :, None])
        assert (off <= (4 * 2.0 ** -24 * np.abs(want[:, :, None]) if prefill else 0)).all(), prefill
