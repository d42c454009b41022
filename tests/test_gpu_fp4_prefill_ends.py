"""Prefill attention over a 4-bit KV pool where keys end: at the block table's width,
before a row's position, and at scales that appending never writes."""
import numpy as np
import pytest

import fp4_accuracy as acc
import fp4_reference as fp4
from test_gpu_fp4_cache import dev, random_pool, tables_of
from test_gpu_fp4_prefill import prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,seen,bs,blocks", [
    (5, 1000, 16, 19),        # 304 keys: the last chunk of 64 is not full
    (200, 310, 16, 19),       # rows before, at and past the table's last key
    (7, 2 ** 31 - 1, 5, 13),  # 65 keys
    (70, 66, 1, 3),
    (6, 9000, 8, 1025),       # 8200 keys in ranges
])
def test_keys_end_with_the_block_table(gpu_ctx, n, seen, bs, blocks):
    """A context length past the table's width is reported, and the keys of the table are what counts."""
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, FerrisError

    print(f"prefill past the table {n} {seen} {bs} {blocks}", flush=True)
    rng = np.random.default_rng(52)
    hq, hkv, d = 8, 2, 64
    (kb, kv), (vb, vv) = random_pool(rng, blocks, hkv, bs, d), random_pool(rng, blocks, hkv, bs, d)
    tables = rng.permutation(blocks).astype(np.int32)[None]
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    out = torch.full(q.shape, -7.0, device="cuda")
    gpu_ctx.attn_prefill_paged(dev(q), dev(kb), dev(vb), DTYPE_MXFP4, dev(tables), dev(np.array([0, n], np.int32)),
                               dev(np.array([seen], np.int32)), n, hkv, bs, blocks, d ** -0.5, out)
    gpu_ctx.sync()
    with pytest.raises(FerrisError) as e:
        gpu_ctx.check_faults()
    assert e.value.kind == "Runtime"
    k, v = (fp4.rows_of(x, tables[0], blocks * bs, bs) for x in (kv, vv))
    first = seen - n
    got, skip = out.cpu().numpy(), max(0, -first)
    assert (got[:skip] == 0).all()
    acc.check(got[skip:], q[skip:], k, v, first + skip, d ** -0.5, acc.prefill_additions(blocks * bs))


@pytest.mark.parametrize("long", [0, 3000])
@pytest.mark.parametrize("seen", [0, -5, -2 ** 31])
def test_a_sequence_without_keys_names_no_block(gpu_ctx, seen, long):
    """New rows at negative positions get zeros, whatever their row of the block table holds; in a launch
    whose other sequence is cut into ranges of keys, too."""
    rng = np.random.default_rng(53)
    hq, hkv, d, bs = 4, 1, 128, 16
    new, lens = [20, 40], [seen, long + 40]
    nb = -(-lens[1] // bs) + 2
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, [0, lens[1]], bs, nb)
    assert (tables[0] == -1).all()
    q = rng.standard_normal((60, hq, d)).astype(np.float32)
    got = prefill(gpu_ctx, q, (dev(kb), dev(vb)), tables, new, lens, hkv, bs, nb, d ** -0.5)
    assert (got[:20] == 0).all()
    k, v = (fp4.rows_of(x, tables[1], lens[1], bs) for x in (kv, vv))
    acc.check(got[20:], q[20:], k, v, long, d ** -0.5, acc.prefill_additions(lens[1]))


@pytest.mark.parametrize("cached,n", [(0, 12), (0, 70), (1300, 6)])
def test_a_block_out_of_range_is_still_reported(gpu_ctx, cached, n):
    """At the sequence's first key, and at its last, in a chunk that is not full."""
    from ferrisinfer_amd import FerrisError

    rng = np.random.default_rng(54)
    hq, hkv, d, bs = 4, 1, 64, 16
    nb = -(-(cached + n) // bs)
    pools = tuple(dev(random_pool(rng, nb, hkv, bs, d)[0]) for _ in range(2))
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    for at in (0, -1):
        for bad in (nb, -1):
            tables = tables_of(rng, [cached + n], bs, nb)
            tables[0, at] = bad
            with pytest.raises(FerrisError) as e:
                prefill(gpu_ctx, q, pools, tables, [n], [cached + n], hkv, bs, nb, 1.0)
            assert e.value.kind == "Runtime"


@pytest.mark.parametrize("e", [253, 254, 255])
def test_scales_past_the_formats_reach_only_rows_that_see_them(gpu_ctx, e):
    """Appending writes no scale above 252 but 255; a pool that holds one, from elsewhere, harms the rows that
    see its key and no others."""
    rng = np.random.default_rng(55)
    n, hq, hkv, d, bs = 90, 8, 2, 64, 16
    nb = -(-n // bs) + 1
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, [n], bs, nb)
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    k, v = (fp4.rows_of(x, tables[0], n, bs) for x in (kv, vv))
    for at_k, at_v in ((41, n), (n, 41), (70, 30)):
        ks, vs = kb.copy(), vb.copy()
        for pool, at in ((ks, at_k), (vs, at_v)):
            if at < n:
                codes, scales = fp4.split_pool(pool, nb, hkv, bs, d)
                codes[tables[0, at // bs], :, at % bs] |= 0x77  # magnitudes of 6 scales
                scales[tables[0, at // bs], :, at % bs] = e
        got = prefill(gpu_ctx, q, (dev(ks), dev(vs)), tables, [n], [n], hkv, bs, nb, d ** -0.5)
        clean = min(at_k, at_v)
        acc.check(got[:clean], q[:clean], k, v, 0, d ** -0.5, acc.prefill_additions(n))
