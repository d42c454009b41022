"""4-bit KV pools on the GPU: append, copy, gather and decode attention against 64-bit numpy."""
import numpy as np
import pytest

import fp4_reference as fp4

pytestmark = pytest.mark.gpu


def dev(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def random_pool(rng, nb, hkv, bs, d, size=1.0):
    """(bytes, values) of a pool array whose rows were appended from normal values."""
    x = (rng.standard_normal((nb, hkv, bs, d)) * size).astype(np.float32)
    codes, scales = fp4.quantise(x)
    return fp4.pool_bytes(codes, scales), fp4.values(codes, scales)


def tables_of(rng, lens, bs, nb):
    """Block tables of sequences of these lengths over a shuffled pool, unused entries -1."""
    need = [-(-n // bs) for n in lens]
    assert sum(need) <= nb
    perm = rng.permutation(nb).astype(np.int32)
    tables = np.full((len(lens), max(max(need), 1)), -1, np.int32)
    at = 0
    for i, k in enumerate(need):
        tables[i, :k] = perm[at:at + k]
        at += k
    return tables


# ---------------------------------------------------------------- append, copy, gather

@pytest.mark.parametrize("t,hkv,d,bs,nb", [(1, 1, 32, 1, 3), (1, 8, 128, 16, 9), (37, 2, 64, 16, 8), (70, 3, 32, 5, 20),
                                           (300, 8, 128, 16, 24), (129, 5, 64, 7, 33)])
def test_append_writes_the_formats_bytes(gpu_ctx, t, hkv, d, bs, nb):
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, kv_pool_bytes

    print(f"append {t} {hkv} {d} {bs}", flush=True)
    rng = np.random.default_rng(t * 1000 + d)
    size = np.exp(rng.standard_normal((t, hkv, 1)) * 6)
    rows = [(rng.standard_normal((t, hkv, d)) * size).astype(np.float32) for _ in range(2)]
    rows[0][0, 0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5]  # ties, where the group's scale is 1
    rows[0][0, 0, 8:32] = 0
    rows[1][t // 2, hkv - 1, 3] = np.inf
    rows[1][t - 1, 0, d - 1] = np.nan
    rows[0][t - 1, hkv - 1] = 0  # a group of zeros
    slots = rng.permutation(nb * bs)[:t].astype(np.int64)
    if t > 2:
        slots[1] = -1  # skipped
    before = [rng.integers(0, 256, kv_pool_bytes(DTYPE_MXFP4, nb, bs, hkv, d), dtype=np.uint8) for _ in range(2)]
    pools = [dev(b) for b in before]
    for shift in (0, 1):  # 16-byte aligned rows, and rows one float off
        src = []
        for r in rows:
            flat = torch.zeros(r.size + 4, device="cuda")
            flat[shift:shift + r.size] = dev(r).reshape(-1)
            src.append(flat[shift:shift + r.size].view(t, hkv, d))
        got = [p.clone() for p in pools]
        gpu_ctx.kv_append(*src, dev(slots), *got, DTYPE_MXFP4, nb, bs, hkv, d)
        gpu_ctx.sync()
        gpu_ctx.check_faults()
        for g, b, r in zip(got, before, rows):
            want = b.copy()
            codes, scales = fp4.split_pool(want, nb, hkv, bs, d)
            c, s = fp4.quantise(r)
            for i, slot in enumerate(slots):
                if slot >= 0:
                    codes[slot // bs, :, slot % bs], scales[slot // bs, :, slot % bs] = c[i], s[i]
            assert np.array_equal(g.cpu().numpy(), want)


def test_append_reports_a_slot_beyond_the_pool(gpu_ctx):
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, FerrisError, kv_pool_bytes

    nb, bs, hkv, d = 3, 4, 2, 32
    pool = [torch.full((kv_pool_bytes(DTYPE_MXFP4, nb, bs, hkv, d),), 7, dtype=torch.uint8, device="cuda") for _ in range(2)]
    x = torch.ones(2, hkv, d, device="cuda")
    gpu_ctx.kv_append(x, x, dev(np.array([nb * bs, -5], np.int64)), *pool, DTYPE_MXFP4, nb, bs, hkv, d)
    with pytest.raises(FerrisError) as e:
        gpu_ctx.check_faults()
    assert e.value.kind == "Runtime"
    assert all(bool((p == 7).all()) for p in pool)


@pytest.mark.parametrize("length,hkv,d,bs", [(0, 2, 32, 16), (1, 1, 32, 1), (33, 2, 64, 16), (50, 8, 128, 16), (17, 3, 64, 5)])
def test_gather_reads_the_values(gpu_ctx, length, hkv, d, bs):
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, FerrisError

    rng = np.random.default_rng(length + d)
    nb = 12
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d, 1e-20)
    fp4.split_pool(kb, nb, hkv, bs, d)[1][2, 0, 0, 0] = 255  # a group of NaN
    kv = fp4.values(*fp4.split_pool(kb, nb, hkv, bs, d))
    table = np.concatenate([[2], rng.permutation(np.setdiff1d(np.arange(nb), [2]))]).astype(np.int32)[:max(1, -(-length // bs))]
    k_out, v_out = (torch.full((length + 2, hkv, d), -3.0, device="cuda") for _ in range(2))
    gpu_ctx.kv_gather(dev(kb), dev(vb), DTYPE_MXFP4, dev(table), length, nb, bs, hkv, d, k_out, v_out)
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    for out, want in ((k_out, kv), (v_out, vv)):
        got = out.cpu().numpy()
        assert (got[length:] == -3.0).all()  # rows behind the last are left as they were
        assert np.array_equal(got[:length].astype(np.float64), fp4.rows_of(want, table, length, bs), equal_nan=True)
    if length:
        bad = table.copy()
        bad[-1] = nb
        gpu_ctx.kv_gather(dev(kb), dev(vb), DTYPE_MXFP4, dev(bad), length, nb, bs, hkv, d, k_out, v_out)
        with pytest.raises(FerrisError):
            gpu_ctx.check_faults()
        assert (k_out.cpu().numpy()[(len(bad) - 1) * bs:length] == 0).all()


def test_copy_blocks_copies_whole_rows(gpu_ctx):
    from ferrisinfer_amd import DTYPE_MXFP4

    rng = np.random.default_rng(5)
    for nb, bs, hkv, d in ((9, 16, 8, 128), (7, 5, 2, 32), (6, 3, 3, 64)):
        before = [rng.integers(0, 256, nb * bs * hkv * d * 17 // 32, dtype=np.uint8) for _ in range(2)]
        pools = [dev(b) for b in before]
        src, dst, counts = np.array([0, 1, 2], np.int32), np.array([4, 5, 3], np.int32), np.array([bs, 1, 0], np.int32)
        gpu_ctx.kv_copy_blocks(*pools, DTYPE_MXFP4, dev(src), dev(dst), dev(counts), nb, bs, hkv, d)
        gpu_ctx.sync()
        gpu_ctx.check_faults()
        for p, b in zip(pools, before):
            want = b.copy()
            for part in fp4.split_pool(want, nb, hkv, bs, d):
                for s, t, n in zip(src, dst, counts):
                    part[t, :, :n] = part[s, :, :n]
            assert np.array_equal(p.cpu().numpy(), want)


# ---------------------------------------------------------------- decode attention

def decode(ctx, q, pools, tables, lens, hkv, bs, nb, scale, longest=None, entry="attn_decode_paged"):
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4

    out = torch.full(q.shape, -7.0, device="cuda")
    longest = max(int(max(lens)), 0) if longest is None else longest
    getattr(ctx, entry)(dev(q), pools[0], pools[1], DTYPE_MXFP4, dev(tables), dev(np.asarray(lens, np.int32)), longest,
                        hkv, bs, nb, scale, out)
    ctx.sync()
    ctx.check_faults()
    return out.cpu().numpy()


CASES = [
    # lengths, hq, hkv, d, block size
    ([1], 1, 1, 32, 16),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33], 2, 2, 32, 16),     # no keys, one, the edges of a step
    ([5, 63, 64, 65, 127, 128, 129, 255, 256, 257], 14, 2, 64, 16),  # narrow rows: waves of 64, partitions of 256
    ([127, 128, 129, 511, 512, 513, 1025], 32, 8, 128, 16),  # wide rows: waves of 128, partitions of 512
    ([700], 14, 2, 64, 16),
    ([300, 40], 8, 1, 128, 16),    # eight heads
    ([90, 1000], 5, 1, 64, 16),    # five heads: a second tile with one
    ([90, 333], 6, 2, 128, 7),     # odd block size
    ([77, 10], 3, 1, 32, 1),       # blocks of one row
    ([2050, 1], 16, 4, 128, 32),
    ([4000, 3], 7, 1, 32, 64),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[1]}-{c[2]}-{c[3]}-bs{c[4]}-max{max(c[0])}")
def test_decode(gpu_ctx, case):
    lens, hq, hkv, d, bs = case
    print(f"decode {case}", flush=True)
    rng = np.random.default_rng(sum(lens) + d)
    nb = sum(-(-n // bs) for n in lens) + 3
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((len(lens), hq, d)).astype(np.float32)
    scale = d ** -0.5
    pools = dev(kb), dev(vb)
    got = decode(gpu_ctx, q, pools, tables, lens, hkv, bs, nb, scale)
    for b, n in enumerate(lens):
        k, v = (fp4.rows_of(x, tables[b], n, bs) for x in (kv, vv))
        want = fp4.attention(q[b:b + 1], k, v, n - 1, scale)[0]
        worst = np.abs(got[b] - want).max()
        assert worst <= fp4.attention_tolerance(q[b], k, v, scale, n), (b, n, worst)
    again = decode(gpu_ctx, q, pools, tables, lens, hkv, bs, nb, scale)
    assert np.array_equal(got, again)  # every summation order is fixed
    assert np.array_equal(got, decode(gpu_ctx, q, pools, tables, lens, hkv, bs, nb, scale, entry="attn_decode_paged_noalloc"))
    for b in range(len(lens)):  # and does not depend on the batch
        one = decode(gpu_ctx, q[b:b + 1], pools, tables[b:b + 1], lens[b:b + 1], hkv, bs, nb, scale)
        assert np.array_equal(one[0], got[b])


def test_decode_large_scores_and_far_values(gpu_ctx):
    """Scores in the hundreds (one key takes nearly all the weight) and V scales near the format's ends."""
    rng = np.random.default_rng(8)
    lens, hq, hkv, d, bs = [513, 40], 8, 2, 128, 16
    nb = 40
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d, 20.0), random_pool(rng, nb, hkv, bs, d, 1e30)
    tables = tables_of(rng, lens, bs, nb)
    q = (3 * rng.standard_normal((2, hq, d))).astype(np.float32)
    got = decode(gpu_ctx, q, (dev(kb), dev(vb)), tables, lens, hkv, bs, nb, d ** -0.5)
    for b, n in enumerate(lens):
        k, v = (fp4.rows_of(x, tables[b], n, bs) for x in (kv, vv))
        want = fp4.attention(q[b:b + 1], k, v, n - 1, d ** -0.5)[0]
        assert np.abs(got[b] - want).max() <= fp4.attention_tolerance(q[b], k, v, d ** -0.5, n)


def test_decode_nan_stays_in_its_sequence_and_dims(gpu_ctx):
    """A NaN group of K makes its head's whole output NaN, one of V the group's 32 dims; rows past a
    sequence's end, other sequences and other kv heads do not see either."""
    rng = np.random.default_rng(9)
    lens, hq, hkv, d, bs = [40, 50, 20], 8, 2, 64, 16
    nb = 12
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    ks, vs = fp4.split_pool(kb, nb, hkv, bs, d)[1], fp4.split_pool(vb, nb, hkv, bs, d)[1]
    ks[tables[0, 1], 0, 3, 1] = 255
    vs[tables[1, 2], 1, 0, 1] = 255
    ks[tables[2, 1], :, 4:] = 255  # rows 20 and up of the last sequence's second block: past its end
    vs[tables[2, 1], :, 4:] = 255
    kv, vv = fp4.values(*fp4.split_pool(kb, nb, hkv, bs, d)), fp4.values(*fp4.split_pool(vb, nb, hkv, bs, d))
    q = rng.standard_normal((3, hq, d)).astype(np.float32)
    got = decode(gpu_ctx, q, (dev(kb), dev(vb)), tables, lens, hkv, bs, nb, 0.125)
    nan = np.isnan(got)
    want = np.zeros_like(nan)
    want[0, :4] = True
    want[1, 4:, 32:] = True
    assert np.array_equal(nan, want)
    for b, n in enumerate(lens):
        k, v = (fp4.rows_of(x, tables[b], n, bs) for x in (kv, vv))
        ref = fp4.attention(q[b:b + 1], k, v, n - 1, 0.125)[0]
        fine = ~want[b]
        tol = fp4.attention_tolerance(q[b], np.nan_to_num(k), np.nan_to_num(v), 0.125, n)
        assert np.abs(got[b] - ref)[fine].max(initial=0) <= tol


def test_decode_bad_block_and_context_are_reported(gpu_ctx):
    from ferrisinfer_amd import FerrisError

    rng = np.random.default_rng(10)
    hq, hkv, d, bs, nb = 4, 2, 32, 16, 6
    pools = tuple(dev(random_pool(rng, nb, hkv, bs, d)[0]) for _ in range(2))
    q = rng.standard_normal((2, hq, d)).astype(np.float32)
    for tables in ([[0, nb], [1, 2]], [[0, -1], [1, 2]]):
        with pytest.raises(FerrisError) as e:
            decode(gpu_ctx, q, pools, np.array(tables, np.int32), [20, 20], hkv, bs, nb, 1.0)
        assert e.value.kind == "Runtime"
    wide = np.zeros((2, 40), np.int32)
    with pytest.raises(FerrisError):  # longer than the partitions that max_context_len sized
        decode(gpu_ctx, q, pools, wide, [400, 20], hkv, bs, nb, 1.0, longest=200)
    decode(gpu_ctx, q, pools, wide, [-3, 20], hkv, bs, nb, 1.0)


def test_decode_pool_offsets_past_32_bits(gpu_ctx):
    """Blocks whose codes and scales lie past 4 GiB of their array."""
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, kv_pool_bytes

    rng = np.random.default_rng(11)
    hq, hkv, d, bs = 32, 8, 128, 16
    nb = (1 << 32) // (hkv * bs * 64) + 300
    size = kv_pool_bytes(DTYPE_MXFP4, nb, bs, hkv, d)
    pools = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    n = 700
    table = (nb - 1 - rng.permutation(60)[:44]).astype(np.int32)[None]
    slots = (table[0].astype(np.int64)[np.arange(n) // bs] * bs + np.arange(n) % bs)
    k, v = (rng.standard_normal((n, hkv, d)).astype(np.float32) for _ in range(2))
    gpu_ctx.kv_append(dev(k), dev(v), dev(slots), *pools, DTYPE_MXFP4, nb, bs, hkv, d)
    kq, vq = fp4.values(*fp4.quantise(k)), fp4.values(*fp4.quantise(v))
    k_out, v_out = (torch.empty(n, hkv, d, device="cuda") for _ in range(2))
    gpu_ctx.kv_gather(*pools, DTYPE_MXFP4, dev(table[0]), n, nb, bs, hkv, d, k_out, v_out)
    assert np.array_equal(k_out.cpu().numpy(), kq) and np.array_equal(v_out.cpu().numpy(), vq)
    q = rng.standard_normal((1, hq, d)).astype(np.float32)
    got = decode(gpu_ctx, q, pools, table, [n], hkv, bs, nb, d ** -0.5)
    want = fp4.attention(q, kq, vq, n - 1, d ** -0.5)
    assert np.abs(got - want).max() <= fp4.attention_tolerance(q, kq, vq, d ** -0.5, n)


def test_pool_refusals(gpu_ctx):
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, FerrisError

    pool = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    odd = pool[4:]
    x = torch.zeros(2, 2, 32, device="cuda")
    slots = torch.zeros(2, dtype=torch.int64, device="cuda")
    ints = torch.zeros(2, dtype=torch.int32, device="cuda")
    bt = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    q = torch.zeros(65, device="cuda")
    calls = [
        ("Unsupported", lambda: gpu_ctx.kv_append(x, x, slots, pool, pool, DTYPE_MXFP4, 4, 4, 2, 48)),
        ("InvalidLayout", lambda: gpu_ctx.kv_append(x, x, slots, pool, odd, DTYPE_MXFP4, 4, 4, 2, 32)),
        ("Unsupported", lambda: gpu_ctx.kv_copy_blocks(pool, pool, DTYPE_MXFP4, ints, ints, ints, 4, 4, 2, 16)),
        ("InvalidLayout", lambda: gpu_ctx.kv_copy_blocks(odd, pool, DTYPE_MXFP4, ints, ints, ints, 4, 4, 2, 32)),
        ("Unsupported", lambda: gpu_ctx.kv_gather(pool, pool, DTYPE_MXFP4, ints, 2, 4, 4, 2, 36, x, x)),
        ("Unsupported", lambda: gpu_ctx.attn_decode_paged(torch.zeros(1, 2, 96, device="cuda"), pool, pool, DTYPE_MXFP4, bt,
                                                          ints, 4, 2, 4, 4, 1.0, x)),
        ("Unsupported", lambda: gpu_ctx.attn_decode_paged(torch.zeros(1, 9, 32, device="cuda"), pool, pool, DTYPE_MXFP4, bt,
                                                          ints, 4, 1, 4, 4, 1.0, x)),
        ("InvalidLayout", lambda: gpu_ctx.attn_decode_paged(x[:1], odd, pool, DTYPE_MXFP4, bt, ints, 4, 2, 4, 4, 1.0, x)),
        ("InvalidLayout", lambda: gpu_ctx.attn_decode_paged(q[1:].view(1, 2, 32), pool, pool, DTYPE_MXFP4, bt, ints, 4, 2,
                                                            4, 4, 1.0, x)),
        ("InvalidShape", lambda: gpu_ctx.attn_decode_paged(x[:1], pool, pool, DTYPE_MXFP4, bt, ints, 17, 2, 4, 4, 1.0, x)),
    ]
    for i, (kind, call) in enumerate(calls):
        with pytest.raises(FerrisError) as e:
            call()
        assert e.value.kind == kind, (i, e.value)


@pytest.mark.parametrize("lens,hq,hkv,d", [([700, 30], 14, 2, 64), ([1400, 600, 9], 32, 8, 128)])
def test_decode_replayed_and_on_another_stream(gpu_ctx, lens, hq, hkv, d):
    """A captured decode equals the eager one on every replay, with eager work between the replays,
    and follows metadata that changes between them."""
    import ctypes

    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, Context, kernel

    rng = np.random.default_rng(12)
    bs = 16
    nb = sum(-(-n // bs) for n in lens) + 3
    pools = tuple(dev(random_pool(rng, nb, hkv, bs, d)[0]) for _ in range(2))
    tables = dev(tables_of(rng, lens, bs, nb))
    qs = [dev(rng.standard_normal((len(lens), hq, d)).astype(np.float32)) for _ in range(4)]
    cut = [np.asarray([max(1, n - 13 * i) for n in lens], np.int32) for i in range(4)]
    want = []
    for q, c in zip(qs, cut):
        out = torch.empty_like(q)
        gpu_ctx.attn_decode_paged(q, *pools, DTYPE_MXFP4, tables, dev(c), max(lens), hkv, bs, nb, d ** -0.5, out)
        want.append(out)
    torch.cuda.synchronize()
    own = Context(0, use_torch_stream=False)  # its own stream
    lib = own.lib
    q, lens_d, out = torch.empty_like(qs[0]), dev(cut[0]), torch.empty_like(qs[0])
    call = lambda: own.attn_decode_paged(q, *pools, DTYPE_MXFP4, tables, lens_d, max(lens), hkv, bs, nb, d ** -0.5, out)  # noqa: E731
    q.copy_(qs[0])
    torch.cuda.synchronize()
    call()  # sizes the workspace
    own.sync()
    lib.fi_graph_begin.argtypes = [ctypes.c_void_p]
    lib.fi_graph_end.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]
    lib.fi_graph_launch.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    lib.fi_graph_destroy.argtypes = [ctypes.c_void_p]
    kernel.check(lib.fi_graph_begin(own.handle))
    call()
    graph = ctypes.c_void_p()
    kernel.check(lib.fi_graph_end(own.handle, ctypes.byref(graph)))
    for i in (0, 1, 2, 3, 1):
        q.copy_(qs[i])
        lens_d.copy_(dev(cut[i]))
        out.fill_(-1)
        torch.cuda.synchronize()
        kernel.check(lib.fi_graph_launch(own.handle, graph))
        own.sync()
        own.check_faults()
        assert torch.equal(out, want[i]), i
        other = torch.empty_like(out)
        gpu_ctx.attn_decode_paged(qs[2], *pools, DTYPE_MXFP4, tables, dev(cut[2]), max(lens), hkv, bs, nb, d ** -0.5, other)
        torch.cuda.synchronize()
        assert torch.equal(other, want[2])
    kernel.check(lib.fi_graph_destroy(graph))
    own.close()


def test_launch_limits_and_refusals_before_rows_are_written(gpu_ctx):
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, FerrisError

    pool = torch.full((1 << 16,), 7, dtype=torch.uint8, device="cuda")
    x = torch.zeros(1, 2, 32, device="cuda")
    slots = torch.zeros(1, dtype=torch.int64, device="cuda")
    bt = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    ints = torch.zeros(1, dtype=torch.int32, device="cuda")
    many = torch.empty(1 << 23, 2, 32, device="cuda")
    calls = [  # sizes that the checks refuse before anything is read
        ("2^24", lambda: gpu_ctx.attn_decode_paged(many, pool, pool, DTYPE_MXFP4, bt, ints, 4, 2, 4, 4, 1.0, x)),
        ("2^32", lambda: gpu_ctx.attn_decode_paged(x, pool, pool, DTYPE_MXFP4, bt, ints, 4, 2, 1 << 12, 1 << 20, 1.0, x)),
    ]
    for words, call in calls:
        with pytest.raises(FerrisError) as e:
            call()
        assert e.value.kind == "Unsupported" and words in e.value.message
    table = torch.ones(64, 16, device="cuda")
    before = pool.clone()
    for hq, longest, kind in ((9, 4, "Unsupported"), (4, 17, "InvalidShape")):  # too many heads a kv head, too short a table
        parts, q = torch.ones(1, (hq + 2) * 32, device="cuda"), torch.zeros(1, hq, 32, device="cuda")
        with pytest.raises(FerrisError) as e:
            gpu_ctx.attn_decode_paged_qkv(parts, 1, None, ints, table, table, 32, 64, slots, pool, pool, DTYPE_MXFP4, bt, ints,
                                          longest, hq, 1, 32, 4, 4, 1.0, q.clone(), q)
        assert e.value.kind == kind
    gpu_ctx.sync()
    assert torch.equal(pool, before)


def test_two_contexts_decode_at_once(gpu_ctx):
    """Calls of two contexts on streams of their own, each merging its partitions by itself."""
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, Context

    rng = np.random.default_rng(60)
    hq, hkv, d, bs, lens = 8, 2, 128, 16, [2000, 900, 1500]
    nb = sum(-(-n // bs) for n in lens) + 1
    pools = [tuple(dev(random_pool(rng, nb, hkv, bs, d)[0]) for _ in range(2)) for _ in range(2)]
    tables = dev(tables_of(rng, lens, bs, nb))
    q = dev(rng.standard_normal((3, hq, d)).astype(np.float32))
    ints = dev(np.array(lens, np.int32))
    other = Context(0, use_torch_stream=False)
    want = []
    for k, v in pools:
        want.append(torch.empty_like(q))
        gpu_ctx.attn_decode_paged(q, k, v, DTYPE_MXFP4, tables, ints, 2000, hkv, bs, nb, d ** -0.5, want[-1])
    gpu_ctx.sync()
    outs = [[torch.empty_like(q) for _ in range(20)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(20):
        for ctx, (k, v), out in zip((gpu_ctx, other), pools, outs):
            ctx.attn_decode_paged(q, k, v, DTYPE_MXFP4, tables, ints, 2000, hkv, bs, nb, d ** -0.5, out[i])
    gpu_ctx.sync()
    other.sync()
    other.close()
    assert all(torch.equal(o, w) for out, w in zip(outs, want) for o in out)


@pytest.mark.parametrize("lens,hq,hkv,d", [([17000, 300, 65536], 2, 1, 32), ([40000], 8, 4, 128), ([16384], 7, 1, 64)])
def test_decode_of_many_partitions(gpu_ctx, lens, hq, hkv, d):
    """64 partitions, more, and as many as a launch takes (65536 tokens of narrow rows)."""
    print(f"decode {lens} {hq} {hkv} {d}", flush=True)
    rng = np.random.default_rng(sum(lens))
    bs = 16
    nb = sum(-(-n // bs) for n in lens) + 1
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((len(lens), hq, d)).astype(np.float32)
    scale = d ** -0.5
    got = decode(gpu_ctx, q, (dev(kb), dev(vb)), tables, lens, hkv, bs, nb, scale)
    for b, n in enumerate(lens):
        k, v = (fp4.rows_of(x, tables[b], n, bs) for x in (kv, vv))
        want = fp4.attention(q[b:b + 1], k, v, n - 1, scale)
        assert np.abs(got[b] - want[0]).max() <= fp4.attention_tolerance(q[b:b + 1], k, v, scale, n), b
    alone = decode(gpu_ctx, q[:1], (dev(kb), dev(vb)), tables[:1], lens[:1], hkv, bs, nb, scale)
    assert np.array_equal(alone[0], got[0])  # whatever the launch's other sequences are
