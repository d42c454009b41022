"""Decode attention over a 4-bit pool at the longest contexts, where narrow rows make up to 512 partitions."""
import numpy as np
import pytest

import fp4_accuracy as acc
import fp4_reference as fp4
from test_gpu_fp4_cache import decode, dev, random_pool, tables_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,hq,hkv,d,bs", [
    ([100003, 700, 65537], 8, 2, 32, 16),
    ([131072, 1], 14, 2, 64, 16),
    ([67195], 2, 1, 128, 64),
    ([65536 + 255, 16385, 16384], 3, 1, 64, 5),   # a last partition of 255 tokens, 65 and 64 partitions beside it
    ([131072], 4, 4, 128, 16),                     # wide rows: 256 partitions
])
def test_decode_of_long_contexts(gpu_ctx, lens, hq, hkv, d, bs):
    print(f"decode {lens} {hq} {hkv} {d}", flush=True)
    rng = np.random.default_rng(sum(lens))
    nb = sum(-(-n // bs) for n in lens) + 1
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((len(lens), hq, d)).astype(np.float32)
    pools, scale = (dev(kb), dev(vb)), d ** -0.5
    got = decode(gpu_ctx, q, pools, tables, lens, hkv, bs, nb, scale)
    for b, n in enumerate(lens):
        k, v = (fp4.rows_of(x, tables[b], n, bs) for x in (kv, vv))
        acc.check(got[b:b + 1], q[b:b + 1], k, v, n - 1, scale, acc.decode_additions(n), (b, n))
    assert np.array_equal(got, decode(gpu_ctx, q, pools, tables, lens, hkv, bs, nb, scale, entry="attn_decode_paged_noalloc"))
    for b, n in enumerate(lens):  # alone: as many partitions as it has itself
        width = -(-n // bs)
        one = decode(gpu_ctx, q[b:b + 1], pools, tables[b:b + 1, :width], [n], hkv, bs, nb, scale)
        assert np.array_equal(one[0], got[b]), n


def test_nan_and_large_scores_past_256_partitions(gpu_ctx):
    """A key that takes nearly all the weight, and a NaN group, in a late partition."""
    rng = np.random.default_rng(91)
    hq, hkv, d, bs, n = 2, 1, 32, 16, 100003
    nb = -(-n // bs)
    (kb, _), (vb, _) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, [n], bs, nb)
    q = rng.standard_normal((1, hq, d)).astype(np.float32)
    at = 90001
    codes, scales = fp4.split_pool(kb, nb, hkv, bs, d)
    code, scale = fp4.quantise((40 * q[0, 0] / np.abs(q[0, 0]).max())[None].astype(np.float32))
    codes[tables[0, at // bs], 0, at % bs], scales[tables[0, at // bs], 0, at % bs] = code[0], scale[0]
    kv, vv = (fp4.values(*fp4.split_pool(x, nb, hkv, bs, d)) for x in (kb, vb))
    k, v = (fp4.rows_of(x, tables[0], n, bs) for x in (kv, vv))
    got = decode(gpu_ctx, q, (dev(kb), dev(vb)), tables, [n], hkv, bs, nb, d ** -0.5)
    acc.check(got, q, k, v, n - 1, d ** -0.5, acc.decode_additions(n))
    fp4.split_pool(vb, nb, hkv, bs, d)[1][tables[0, 80000 // bs], 0, 0, 0] = 255
    assert np.isnan(decode(gpu_ctx, q, (dev(kb), dev(vb)), tables, [n], hkv, bs, nb, d ** -0.5)).all()


def test_longer_contexts_are_refused(gpu_ctx):
    import torch

    from ferrisinfer_amd import DTYPE_BF16, DTYPE_MXFP4, FerrisError

    pool = torch.zeros(1 << 12, dtype=torch.uint8, device="cuda")
    table = torch.zeros(1, 9000, dtype=torch.int32, device="cuda")
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 2, 32, device="cuda")
    for dtype, longest in ((DTYPE_MXFP4, 131072), (DTYPE_BF16, 65536)):
        gpu_ctx.attn_decode_paged(q, pool, pool, dtype, table, lens, longest, 1, 16, 2, 1.0, q.clone())
        with pytest.raises(FerrisError) as e:
            gpu_ctx.attn_decode_paged(q, pool, pool, dtype, table, lens, longest + 1, 1, 16, 2, 1.0, q.clone())
        assert e.value.kind == "Unsupported" and str(longest) in e.value.message
    gpu_ctx.check_faults()
