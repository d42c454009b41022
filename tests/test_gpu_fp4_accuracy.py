"""f32 accuracy of decode and prefill attention over a 4-bit KV pool: the error against 64 bits is of the
size that f32 roundings give, which no kernel with fewer bf16 pieces or a key less reaches
(fp4_accuracy.py, test_fp4_accuracy.py)."""
import numpy as np
import pytest

import fp4_accuracy as acc
import fp4_reference as fp4
from test_gpu_fp4_cache import CASES as DECODE, decode, dev, random_pool, tables_of
from test_gpu_fp4_prefill import CASES as PREFILL, prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("entry", ["attn_decode_paged", "attn_decode_paged_noalloc"])
@pytest.mark.parametrize("case", DECODE + [
    ([700] * 40, 14, 2, 64, 16),               # a launch that merges its partitions by itself
    ([5000, 100], 32, 8, 128, 16),             # and one of more
    ([17000, 300, 65536], 2, 1, 32, 16),       # past 64 partitions, and 256 of them
    ([40000], 8, 4, 128, 16),
], ids=lambda c: f"{c[1]}-{c[2]}-{c[3]}-bs{c[4]}-{len(c[0])}x{max(c[0])}")
def test_decode_is_f32_accurate(gpu_ctx, case, entry):
    lens, hq, hkv, d, bs = case
    print(f"decode accuracy {hq} {hkv} {d} {bs} {max(lens)} {entry}", flush=True)
    rng = np.random.default_rng(sum(lens) + d + 1)
    nb = sum(-(-n // bs) for n in lens) + 3
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((len(lens), hq, d)).astype(np.float32)
    scale = d ** -0.5
    got = decode(gpu_ctx, q, (dev(kb), dev(vb)), tables, lens, hkv, bs, nb, scale, entry=entry)
    for b, n in enumerate(lens):
        if n:
            k, v = (fp4.rows_of(x, tables[b], n, bs) for x in (kv, vv))
            acc.check(got[b:b + 1], q[b:b + 1], k, v, n - 1, scale, acc.decode_additions(n), (b, n))


@pytest.mark.parametrize("size", [3.0, 20.0])
def test_decode_of_large_scores_is_f32_accurate(gpu_ctx, size):
    rng = np.random.default_rng(80)
    lens, hq, hkv, d, bs, nb = [513, 40], 8, 2, 128, 16, 40
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d, size), random_pool(rng, nb, hkv, bs, d, 1e30)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((2, hq, d)).astype(np.float32)
    got = decode(gpu_ctx, q, (dev(kb), dev(vb)), tables, lens, hkv, bs, nb, d ** -0.5)
    for b, n in enumerate(lens):
        k, v = (fp4.rows_of(x, tables[b], n, bs) for x in (kv, vv))
        acc.check(got[b:b + 1], q[b:b + 1], k, v, n - 1, d ** -0.5, acc.decode_additions(n), (b, n))


@pytest.mark.parametrize("case", PREFILL + [
    ([(8 * i % 90, 120 + i) for i in range(20)], 32, 8, 128, 16),      # a planned launch
    ([(16000, 5)], 32, 8, 128, 16),                                    # ranges of keys
    ([(3000, 40), (0, 3), (255, 1), (511, 2)], 14, 2, 64, 16),         # cut and whole tiles beside each other
    ([(1500, 70), (100, 257)], 6, 2, 128, 5),
    ([(5000, 6)], 1, 1, 32, 1),
], ids=lambda c: f"{c[1]}-{c[2]}-{c[3]}-bs{c[4]}-{len(c[0])}x{max(n for _, n in c[0])}-{max(p for p, _ in c[0])}")
def test_prefill_is_f32_accurate(gpu_ctx, case):
    seqs, hq, hkv, d, bs = case
    print(f"prefill accuracy {hq} {hkv} {d} {bs} {seqs[:3]}", flush=True)
    new, lens = [n for _, n in seqs], [p + n for p, n in seqs]
    rng = np.random.default_rng(sum(lens) + d + 1)
    nb = sum(-(-n // bs) for n in lens) + 3
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((sum(new), hq, d)).astype(np.float32)
    got = prefill(gpu_ctx, q, (dev(kb), dev(vb)), tables, new, lens, hkv, bs, nb, d ** -0.5)
    at = 0
    for b, (p, n) in enumerate(seqs):
        if n:
            k, v = (fp4.rows_of(x, tables[b], p + n, bs) for x in (kv, vv))
            acc.check(got[at:at + n], q[at:at + n], k, v, p, d ** -0.5, acc.prefill_additions(p + n), (b, p, n))
        at += n


@pytest.mark.parametrize("size", [3.0, 20.0])
def test_prefill_of_large_scores_is_f32_accurate(gpu_ctx, size):
    rng = np.random.default_rng(81)
    hq, hkv, d, bs, n, nb = 8, 2, 128, 16, 150, 12
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d, size), random_pool(rng, nb, hkv, bs, d, 1e-20)
    tables = tables_of(rng, [n], bs, nb)
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    got = prefill(gpu_ctx, q, (dev(kb), dev(vb)), tables, [n], [n], hkv, bs, nb, d ** -0.5)
    k, v = (fp4.rows_of(x, tables[0], n, bs) for x in (kv, vv))
    acc.check(got, q, k, v, 0, d ** -0.5, acc.prefill_additions(n))
