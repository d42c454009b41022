"""Calls over a 4-bit KV pool with nothing to do: they succeed, as over the other pools, and write nothing."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
def test_calls_without_rows(gpu_ctx, kind):
    import torch

    from ferrisinfer_amd import DTYPE_BF16, DTYPE_F32, DTYPE_MXFP4, kv_pool_bytes

    dtype = {"f32": DTYPE_F32, "bf16": DTYPE_BF16, "mxfp4": DTYPE_MXFP4}[kind]
    nb, bs, hq, hkv, d = 4, 16, 4, 2, 32
    pools = [torch.full((kv_pool_bytes(dtype, nb, bs, hkv, d),), 7, dtype=torch.uint8, device="cuda") for _ in range(2)]
    f32 = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    table, slots, parts = f32(8, d // 2), torch.zeros(0, dtype=torch.int64, device="cuda"), f32(1, 0, (hq + 2 * hkv) * d)
    rope = (ints(0), table, table, d, 8, slots, *pools, dtype)
    gpu_ctx.kv_append(f32(0, hkv, d), f32(0, hkv, d), slots, *pools, dtype, nb, bs, hkv, d)
    gpu_ctx.kv_copy_blocks(*pools, dtype, ints(0), ints(0), ints(0), nb, bs, hkv, d)
    gpu_ctx.kv_gather(*pools, dtype, ints(0), 0, nb, bs, hkv, d, f32(1), f32(1))
    gpu_ctx.qkv_rope_append(parts, 1, None, *rope, nb, bs, hq, hkv, d, f32(0, hq, d))
    gpu_ctx.qkv_norm_rope_append(parts, 1, None, None, 0.0, rope[0], None, *rope[1:], nb, bs, hq, hkv, d, f32(0, hq, d))
    for longest in (0, 16):
        gpu_ctx.attn_decode_paged(f32(0, hq, d), *pools, dtype, ints(0, 1), ints(0), longest, hkv, bs, nb, 1.0, f32(0, hq, d))
        gpu_ctx.attn_decode_paged_noalloc(f32(0, hq, d), *pools, dtype, ints(0, 1), ints(0), longest, hkv, bs, nb, 1.0,
                                          f32(0, hq, d))
        # no query buffer either: there are no rows for it
        gpu_ctx.attn_decode_paged_qkv(parts, 1, None, *rope, ints(0, 1), ints(0), longest, hq, hkv, d, bs, nb, 1.0,
                                      f32(0, hq, d))
    gpu_ctx.attn_prefill_paged(f32(0, hq, d), *pools, dtype, ints(0, 1), ints(1), ints(0), 0, hkv, bs, nb, 1.0, f32(0, hq, d))
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    assert all(bool((p == 7).all()) for p in pools)


def test_negative_and_zero_scales_of_decode(gpu_ctx):
    """Decode takes any finite scale: the largest score is taken after scaling."""
    import numpy as np

    import fp4_accuracy as acc
    import fp4_reference as fp4
    from test_gpu_fp4_cache import decode, dev, random_pool, tables_of

    rng = np.random.default_rng(110)
    lens, hq, hkv, d, bs, nb = [700, 40], 8, 2, 64, 16, 50
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((2, hq, d)).astype(np.float32)
    for scale in (-0.5, 0.0):
        got = decode(gpu_ctx, q, (dev(kb), dev(vb)), tables, lens, hkv, bs, nb, scale)
        for b, n in enumerate(lens):
            k, v = (fp4.rows_of(x, tables[b], n, bs) for x in (kv, vv))
            acc.check(got[b:b + 1], q[b:b + 1], k, v, n - 1, scale, acc.decode_additions(n), (scale, b))
