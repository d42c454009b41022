"""Prefill attention over a 4-bit KV pool against 64-bit arithmetic."""
import numpy as np
import pytest

import fp4_reference as fp4
from test_gpu_fp4_cache import dev, random_pool, tables_of

pytestmark = pytest.mark.gpu


def prefill(ctx, q, pools, tables, new, lens, hkv, bs, nb, scale, longest=None, out=None):
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4

    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    out = torch.full(q.shape, -7.0, device="cuda") if out is None else out
    ctx.attn_prefill_paged(q if not isinstance(q, np.ndarray) else dev(q), *pools, DTYPE_MXFP4, dev(tables), dev(cu),
                           dev(np.asarray(lens, np.int32)), max(new) if longest is None else longest, hkv, bs, nb, scale, out)
    ctx.sync()
    ctx.check_faults()
    return out.cpu().numpy()


def attention64(q, k, v, first, scale):
    """fp4_reference.attention by torch in f64 (no NaN among the keys)."""
    import torch

    q, k, v = (torch.from_numpy(np.ascontiguousarray(x, np.float64)).cuda() for x in (q, k, v))
    n, hq, _ = q.shape
    out = torch.empty_like(q)
    hidden = torch.arange(k.shape[0], device="cuda")[None] > first + torch.arange(n, device="cuda")[:, None]
    for h in range(hq):
        s = (q[:, h].contiguous() @ k[:, h * k.shape[1] // hq].T.contiguous()) * scale
        out[:, h] = torch.softmax(s.masked_fill(hidden, -float("inf")), -1) @ v[:, h * k.shape[1] // hq].contiguous()
    return out.cpu().numpy()


CASES = [
    # (cached, new) of each sequence, hq, hkv, d, block size
    ([(0, 1)], 1, 1, 32, 16),
    ([(0, 1), (5, 1), (63, 2), (64, 1), (0, 64), (0, 65)], 2, 2, 32, 16),
    ([(3, 17), (29, 61), (0, 33)], 14, 2, 64, 16),
    ([(100, 20), (0, 0), (7, 3)], 14, 2, 64, 5),        # a sequence without new rows, odd blocks
    ([(511, 130), (0, 90)], 32, 8, 128, 16),
    ([(0, 200)], 8, 1, 128, 64),
    ([(40, 77)], 5, 1, 64, 1),                          # blocks of one row
    ([(1, 300), (2, 31)], 6, 2, 128, 128),              # a block wider than a chunk
    ([(2000, 5)], 4, 4, 32, 16),
    ([(0, 700)], 14, 2, 64, 16),                        # key splits
    ([(300, 600), (11, 257)], 4, 1, 128, 16),           # key splits, rows that a later split does not see
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[1]}-{c[2]}-{c[3]}-bs{c[4]}-{len(c[0])}x{max(n for _, n in c[0])}")
def test_prefill(gpu_ctx, case):
    seqs, hq, hkv, d, bs = case
    print(f"prefill {case}", flush=True)
    new, lens = [n for _, n in seqs], [p + n for p, n in seqs]
    rng = np.random.default_rng(sum(lens) + d)
    nb = sum(-(-n // bs) for n in lens) + 3
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((sum(new), hq, d)).astype(np.float32)
    pools = dev(kb), dev(vb)
    scale = d ** -0.5
    got = prefill(gpu_ctx, q, pools, tables, new, lens, hkv, bs, nb, scale)
    at = 0
    for b, (p, n) in enumerate(seqs):
        if n == 0:
            continue
        k, v = (fp4.rows_of(x, tables[b], p + n, bs) for x in (kv, vv))
        want = attention64(q[at:at + n], k, v, p, scale)
        tol = fp4.attention_tolerance(q[at:at + n], k, v, scale, p + n)
        worst = np.abs(got[at:at + n] - want).max()
        assert worst <= tol, (b, worst, tol)
        at += n
    # the same call again, and with a looser bound of the query lengths
    assert np.array_equal(got, prefill(gpu_ctx, q, pools, tables, new, lens, hkv, bs, nb, scale))
    loose = prefill(gpu_ctx, q, pools, tables, new, lens, hkv, bs, nb, scale, longest=max(new) + 1)
    assert np.abs(loose - got).max() <= 2 * max(fp4.attention_tolerance(q, kv.reshape(-1, hkv, d), vv, scale, max(lens)), 0)


@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 32), (32, 8, 128), (14, 2, 64)])
def test_prefill_two_row_groups(gpu_ctx, hq, hkv, d):
    """Launches large enough for two row groups a wave: many sequences, planned tiles."""
    rng = np.random.default_rng(d)
    g = {8: 8, 7: 8, 4: 4}[hq // hkv]
    rows = 128 // g
    n_seqs = 2 * 256 // hkv // 8 + 1
    new = [8 * rows - (i * 5) % 9 for i in range(n_seqs)]
    cached = [(i * 37) % 90 for i in range(n_seqs)]
    lens = [p + n for p, n in zip(cached, new)]
    bs = 16
    nb = sum(-(-n // bs) for n in lens) + 3
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((sum(new), hq, d)).astype(np.float32)
    got = prefill(gpu_ctx, q, (dev(kb), dev(vb)), tables, new, lens, hkv, bs, nb, d ** -0.5)
    at = 0
    for b, (p, n) in enumerate(zip(cached, new)):
        k, v = (fp4.rows_of(x, tables[b], p + n, bs) for x in (kv, vv))
        want = attention64(q[at:at + n], k, v, p, d ** -0.5)
        assert np.abs(got[at:at + n] - want).max() <= fp4.attention_tolerance(q[at:at + n], k, v, d ** -0.5, p + n)
        at += n


def test_prefill_of_one_row_is_decode(gpu_ctx):
    """The last row of a prompt and a decode of it see the same keys."""
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4

    rng = np.random.default_rng(21)
    hq, hkv, d, bs, nb = 14, 2, 64, 16, 30
    lens = [1, 90, 257]
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((3, hq, d)).astype(np.float32)
    pools = dev(kb), dev(vb)
    got = prefill(gpu_ctx, q, pools, tables, [1, 1, 1], lens, hkv, bs, nb, 0.125)
    out = torch.empty(3, hq, d, device="cuda")
    gpu_ctx.attn_decode_paged(dev(q), *pools, DTYPE_MXFP4, dev(tables), dev(np.asarray(lens, np.int32)), 257, hkv, bs, nb,
                              0.125, out)
    tol = max(fp4.attention_tolerance(q[b], *(fp4.rows_of(x, tables[b], n, bs) for x in (kv, vv)), 0.125, n)
              for b, n in enumerate(lens))
    assert np.abs(out.cpu().numpy() - got).max() <= 2 * tol


@pytest.mark.parametrize("n,hq,hkv,d", [(100, 8, 2, 64), (500, 4, 1, 128), (70, 2, 2, 32)])
def test_prefill_nan_reaches_only_rows_that_see_it(gpu_ctx, n, hq, hkv, d):
    """A NaN group of K makes the rows at and after its key NaN, one of V their 32 dims; earlier rows
    in the same chunk, other heads, and rows past the end stay exact.  (500 rows of one kv head: key
    splits; keys 0 to 3 NaN: rows whose first split sees nothing else.)"""
    rng = np.random.default_rng(n)
    bs = 16
    nb = -(-n // bs) + 2
    (kb, _), (vb, _) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, [n], bs, nb)
    ks, vs = fp4.split_pool(kb, nb, hkv, bs, d)[1], fp4.split_pool(vb, nb, hkv, bs, d)[1]
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    row = lambda t: (tables[0, t // bs], t % bs)  # noqa: E731
    for blk, off in [row(t) for t in range(n, -(-n // bs) * bs)]:
        ks[blk, :, off] = vs[blk, :, off] = 255
    clean_k, clean_v = kb.copy(), vb.copy()
    at_k, at_v, dim_group = n - 9, n // 2, d // 32 - 1
    ks[row(at_k)[0], 0, row(at_k)[1], 0] = 255
    vs[row(at_v)[0], hkv - 1, row(at_v)[1], dim_group] = 255
    got = prefill(gpu_ctx, q, (dev(kb), dev(vb)), tables, [n], [n], hkv, bs, nb, d ** -0.5)
    want = np.zeros((n, hkv, hq // hkv, d), bool)
    want[at_k:, 0] = True
    want[at_v:, hkv - 1, :, 32 * dim_group:32 * dim_group + 32] = True
    want = want.reshape(n, hq, d)
    assert np.array_equal(np.isnan(got), want)
    kv, vv = (fp4.rows_of(fp4.values(*fp4.split_pool(x, nb, hkv, bs, d)), tables[0], n, bs) for x in (clean_k, clean_v))
    ref = attention64(q, kv, vv, 0, d ** -0.5)
    assert np.abs(got - ref)[~want].max() <= fp4.attention_tolerance(q, kv, vv, d ** -0.5, n)
    ks, vs = fp4.split_pool(clean_k, nb, hkv, bs, d)[1], fp4.split_pool(clean_v, nb, hkv, bs, d)[1]
    for t in range(4):
        ks[row(t)[0], 0, row(t)[1], 0] = 255
    got = prefill(gpu_ctx, q, (dev(clean_k), dev(vb)), tables, [n], [n], hkv, bs, nb, d ** -0.5)
    assert np.isnan(got[:, :hq // hkv]).all()


def test_prefill_large_scores_and_far_values(gpu_ctx):
    rng = np.random.default_rng(30)
    hq, hkv, d, bs, n = 8, 2, 128, 16, 150
    nb = 12
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d, 30.0), random_pool(rng, nb, hkv, bs, d, 1e-30)
    tables = tables_of(rng, [n], bs, nb)
    q = (3 * rng.standard_normal((n, hq, d))).astype(np.float32)
    got = prefill(gpu_ctx, q, (dev(kb), dev(vb)), tables, [n], [n], hkv, bs, nb, d ** -0.5)
    k, v = (fp4.rows_of(x, tables[0], n, bs) for x in (kv, vv))
    assert np.abs(got - attention64(q, k, v, 0, d ** -0.5)).max() <= fp4.attention_tolerance(q, k, v, d ** -0.5, n)


def test_prefill_rows_without_keys_and_bad_inputs(gpu_ctx):
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, FerrisError

    rng = np.random.default_rng(31)
    hq, hkv, d, bs, nb = 4, 1, 128, 16, 40
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    pools = dev(kb), dev(vb)
    for n, seen in ((20, 12), (300, 290), (300, 0)):  # one launch, and key splits
        q = rng.standard_normal((n, hq, d)).astype(np.float32)
        tables = tables_of(rng, [n], bs, nb)
        got = prefill(gpu_ctx, q, pools, tables, [n], [seen], hkv, bs, nb, d ** -0.5)
        assert (got[:n - seen] == 0).all()
        if seen:
            k, v = (fp4.rows_of(x, tables[0], seen, bs) for x in (kv, vv))
            want = attention64(q[n - seen:], k, v, 0, d ** -0.5)
            assert np.abs(got[n - seen:] - want).max() <= fp4.attention_tolerance(q, k, v, d ** -0.5, seen)
    q = rng.standard_normal((20, hq, d)).astype(np.float32)
    tables = tables_of(rng, [20], bs, nb)
    for bad in (nb, -1):
        t = tables.copy()
        t[0, 1] = bad
        with pytest.raises(FerrisError) as e:
            prefill(gpu_ctx, q, pools, t, [20], [20], hkv, bs, nb, 1.0)
        assert e.value.kind == "Runtime"
    out = torch.full((100, hq, d), -7.0, device="cuda")
    q = rng.standard_normal((100, hq, d)).astype(np.float32)
    with pytest.raises(FerrisError):  # more rows than max_query_len sized tiles for
        prefill(gpu_ctx, q, pools, tables_of(rng, [100], bs, nb), [100], [100], hkv, bs, nb, 1.0, longest=16, out=out)
    assert (out.cpu().numpy()[-1] == -7.0).all()
    for kind, change in (("InvalidConfig", dict(scale=0.0)), ("InvalidConfig", dict(scale=-1.0)),
                         ("InvalidConfig", dict(scale=float("nan"))), ("Unsupported", dict(d=96)), ("Unsupported", dict(hq=9))):
        qd = torch.zeros(4, change.get("hq", hq), change.get("d", d), device="cuda")
        with pytest.raises(FerrisError) as e:
            gpu_ctx.attn_prefill_paged(qd, *pools, DTYPE_MXFP4, dev(tables), dev(np.array([0, 4], np.int32)),
                                       dev(np.array([4], np.int32)), 4, hkv, bs, nb, change.get("scale", 1.0), qd.clone())
        assert e.value.kind == kind, (change, e.value)


@pytest.mark.parametrize("seqs,hq,hkv,d", [([(0, 90), (30, 41)], 14, 2, 64), ([(100, 400)], 4, 1, 128),
                                           ([(0, 130)] * 40, 32, 8, 128)])
def test_prefill_replayed(gpu_ctx, seqs, hq, hkv, d):
    """A captured prefill (planned tiles, key splits) equals the eager one on every replay."""
    import ctypes

    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, Context, kernel

    rng = np.random.default_rng(33)
    bs = 16
    new, lens = [n for _, n in seqs], [p + n for p, n in seqs]
    nb = sum(-(-n // bs) for n in lens) + 3
    pools = tuple(dev(random_pool(rng, nb, hkv, bs, d)[0]) for _ in range(2))
    tables = dev(tables_of(rng, lens, bs, nb))
    cu, lens_d = dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)), dev(np.asarray(lens, np.int32))
    qs = [dev(rng.standard_normal((sum(new), hq, d)).astype(np.float32)) for _ in range(3)]
    tail = (pools[0], pools[1], DTYPE_MXFP4, tables, cu, lens_d, max(new), hkv, bs, nb, d ** -0.5)
    want = [torch.empty_like(q) for q in qs]
    for q, w in zip(qs, want):
        gpu_ctx.attn_prefill_paged(q, *tail, w)
    torch.cuda.synchronize()
    own = Context(0, use_torch_stream=False)
    lib = own.lib
    q, out = qs[0].clone(), torch.empty_like(qs[0])
    torch.cuda.synchronize()
    own.attn_prefill_paged(q, *tail, out)
    own.sync()
    lib.fi_graph_begin.argtypes = [ctypes.c_void_p]
    lib.fi_graph_end.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]
    lib.fi_graph_launch.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    lib.fi_graph_destroy.argtypes = [ctypes.c_void_p]
    kernel.check(lib.fi_graph_begin(own.handle))
    own.attn_prefill_paged(q, *tail, out)
    graph = ctypes.c_void_p()
    kernel.check(lib.fi_graph_end(own.handle, ctypes.byref(graph)))
    for i in (0, 1, 2, 1):
        q.copy_(qs[i])
        out.fill_(-1)
        torch.cuda.synchronize()
        kernel.check(lib.fi_graph_launch(own.handle, graph))
        own.sync()
        assert torch.equal(out, want[i]), i
        other = torch.empty_like(out)
        gpu_ctx.attn_prefill_paged(qs[2], *tail, other)
        torch.cuda.synchronize()
        assert torch.equal(other, want[2])
    own.check_faults()
    kernel.check(lib.fi_graph_destroy(graph))
    own.close()


@pytest.mark.parametrize("seqs,hq,hkv,d,bs", [
    ([(16000, 5)], 32, 8, 128, 16),                         # 24 ranges of one tile's keys
    ([(20000, 1)], 1, 1, 32, 16),                           # 32 ranges, as many as a tile is cut into
    ([(3000, 40), (0, 3), (255, 1), (256, 1), (511, 2), (0, 0)], 14, 2, 64, 16),  # cut, whole and absent beside each other
    ([(1500, 70), (100, 257)], 6, 2, 128, 5),               # tiles of 1, 2, .. ranges
    ([(9000, 300)], 14, 2, 64, 64),                         # more tiles: longer ranges
])
def test_prefill_of_few_rows_over_long_prefixes(gpu_ctx, seqs, hq, hkv, d, bs):
    print(f"prefill over prefixes {seqs}", flush=True)
    new, lens = [n for _, n in seqs], [p + n for p, n in seqs]
    rng = np.random.default_rng(sum(lens) + d)
    nb = sum(-(-n // bs) for n in lens) + 3
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    wide = np.concatenate([tables, np.full((len(lens), 40000 // bs), -1, np.int32)], 1)  # far wider than its sequences
    q = rng.standard_normal((sum(new), hq, d)).astype(np.float32)
    scale = d ** -0.5
    for table in (tables, wide):
        got = prefill(gpu_ctx, q, (dev(kb), dev(vb)), table, new, lens, hkv, bs, nb, scale)
        at = 0
        for b, (p, n) in enumerate(seqs):
            if n == 0:
                continue
            k, v = (fp4.rows_of(x, tables[b], p + n, bs) for x in (kv, vv))
            want = attention64(q[at:at + n], k, v, p, scale)
            assert np.abs(got[at:at + n] - want).max() <= fp4.attention_tolerance(q[at:at + n], k, v, scale, p + n), b
            at += n


def test_prefill_nan_in_one_range_of_a_long_prefix(gpu_ctx):
    """Ranges of keys of which one holds a NaN group of V, and one of K in another kv head."""
    rng = np.random.default_rng(50)
    hq, hkv, d, bs, n, p = 8, 2, 64, 16, 6, 2500
    nb = -(-(n + p) // bs) + 1
    (kb, _), (vb, _) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, [n + p], bs, nb)
    fp4.split_pool(kb, nb, hkv, bs, d)[1][tables[0, 70], 0, 3, 1] = 255
    fp4.split_pool(vb, nb, hkv, bs, d)[1][tables[0, 20], 1, 9, 0] = 255
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    got = prefill(gpu_ctx, q, (dev(kb), dev(vb)), tables, [n], [n + p], hkv, bs, nb, d ** -0.5)
    want = np.zeros((n, hkv, hq // hkv, d), bool)
    want[:, 0] = True
    want[:, 1, :, :32] = True
    assert np.array_equal(np.isnan(got), want.reshape(n, hq, d))


@pytest.mark.parametrize("n,seen", [(5, 1000), (5, 2 ** 31 - 1), (200, 2 ** 30), (5, -2 ** 31 + 64)])
def test_prefill_context_beyond_the_block_table(gpu_ctx, n, seen):
    """Keys end with the table, whatever the context length says: the call ends and reports it."""
    from ferrisinfer_amd import FerrisError

    rng = np.random.default_rng(51)
    hq, hkv, d, bs, nb = 4, 2, 64, 16, 20
    pools = tuple(dev(random_pool(rng, nb, hkv, bs, d)[0]) for _ in range(2))
    tables = np.arange(nb, dtype=np.int32)[None]
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    if seen < 0:  # rows without keys
        assert (prefill(gpu_ctx, q, pools, tables, [n], [seen], hkv, bs, nb, d ** -0.5) == 0).all()
        return
    with pytest.raises(FerrisError) as e:
        prefill(gpu_ctx, q, pools, tables, [n], [seen], hkv, bs, nb, d ** -0.5)
    assert e.value.kind == "Runtime"
    prefill(gpu_ctx, q, pools, tables, [n], [nb * bs], hkv, bs, nb, d ** -0.5)  # the whole table is served
