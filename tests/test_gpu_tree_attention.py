"""Attention of drafted trees over paged pools against 64-bit numpy (draft_reference.py)."""
import numpy as np
import pytest

import draft_reference as ref
import fp4_reference as fp4
from test_gpu_fp4_cache import dev, random_pool, tables_of

pytestmark = pytest.mark.gpu

PIECES = {"f32": 6, "bf16": 3, "mxfp4": 3}


def dtype_of(pool):
    from ferrisinfer_amd import DTYPE_BF16, DTYPE_F32, DTYPE_MXFP4

    return {"f32": DTYPE_F32, "bf16": DTYPE_BF16, "mxfp4": DTYPE_MXFP4}[pool]


def pool_of(rng, kind, nb, hkv, bs, d, size=1.0):
    """(device array, values [nb, hkv, bs, d] in f64)."""
    import torch

    if kind == "mxfp4":
        raw, values = random_pool(rng, nb, hkv, bs, d, size)
        return dev(raw), values
    x = (rng.standard_normal((nb, hkv, bs, d)) * size).astype(np.float32)
    t = dev(x)
    if kind == "bf16":
        t = t.to(torch.bfloat16)
    return t, t.double().cpu().numpy()


def attend(ctx, kind, q, pools, tables, nodes, lens, mask, hkv, bs, nb, scale, longest=None, most=None, out=None):
    import torch

    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    out = torch.full(q.shape, -7.0, device="cuda") if out is None else out
    ctx.attn_tree_paged(dev(q), *pools, dtype_of(kind), dev(tables), dev(cu), dev(np.asarray(lens, np.int32)), dev(mask),
                        max(nodes) if most is None else most, max(max(lens), 0) if longest is None else longest, hkv, bs, nb,
                        scale, out)
    return out


def checked(ctx, out):
    ctx.sync()
    ctx.check_faults()
    return out.cpu().numpy()


def trees_of(rng, nodes, words=None):
    trees = [ref.grown(rng, n) for n in nodes]
    words = -(-max(max(nodes), 1) // 64) if words is None else words
    mask = [ref.words_of(ref.ancestors(p), words) for p in trees if p]
    return trees, np.concatenate(mask) if mask else np.zeros((0, words), np.int64)


CASES = [
    # (cached, nodes) of each sequence, hq, hkv, d, block size
    ([(0, 1)], 1, 1, 32, 16),
    ([(0, 1), (5, 1), (31, 2), (32, 1), (33, 31), (0, 64), (0, 65)], 2, 2, 32, 16),
    ([(63, 1), (64, 1), (62, 3), (1, 63), (127, 2), (128, 33)], 4, 2, 64, 16),
    ([(700, 8)], 14, 2, 64, 16),
    ([(100, 20), (7, 0), (7, 3)], 14, 2, 64, 5),             # a sequence without rows, odd blocks
    ([(511, 16), (0, 9), (300, 13)], 32, 8, 128, 16),
    ([(40, 77)], 5, 1, 64, 1),                               # blocks of one row, trees wider than a word
    ([(1, 130), (2, 31)], 6, 2, 128, 128),                   # blocks wider than a chunk
    ([(0, 300)], 3, 3, 32, 16),                              # a tree over several parts
    ([(900, 4)], 12, 1, 64, 16),                             # more than 8 query heads a KV head
    ([(2500, 5), (3, 2), (1300, 17)], 8, 2, 32, 16),         # parts
    ([(5000, 33)], 32, 8, 128, 16),
]


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[1]}-{c[2]}-{c[3]}-bs{c[4]}-{len(c[0])}x{max(n for _, n in c[0])}")
def test_attends_prefix_and_ancestors(gpu_ctx, case, kind):
    seqs, hq, hkv, d, bs = case
    print(f"tree attention {kind} {case}", flush=True)
    rng = np.random.default_rng(sum(p + n for p, n in seqs) + d)
    nodes, lens = [n for _, n in seqs], [p + n for p, n in seqs]
    nb = sum(-(-n // bs) for n in lens) + 3
    (kd, kv), (vd, vv) = pool_of(rng, kind, nb, hkv, bs, d), pool_of(rng, kind, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    trees, mask = trees_of(rng, nodes)
    q = rng.standard_normal((sum(nodes), hq, d)).astype(np.float32)
    scale = d ** -0.5
    got = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, nodes, lens, mask, hkv, bs, nb, scale))
    at = 0
    for b, (p, n) in enumerate(seqs):
        if n == 0:
            continue
        k, v = (fp4.rows_of(x, tables[b], p + n, bs) for x in (kv, vv))
        shown = ref.visible(ref.ancestors(trees[b]), p, p + n)
        ref.check_attention(got[at:at + n], q[at:at + n], k, v, shown, scale, PIECES[kind], (b, kind))
        at += n
    again = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, nodes, lens, mask, hkv, bs, nb, scale))
    assert np.array_equal(got, again)
    # looser bounds of lengths and nodes, a mask with a word to spare
    wide = np.concatenate([mask, rng.integers(-2 ** 63, 2 ** 63, (mask.shape[0], 1))], 1)
    width = tables.shape[1] * bs
    loose = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, nodes, lens, wide, hkv, bs, nb, scale, longest=width,
                                    most=max(nodes) + 5))
    at = 0
    for b, (p, n) in enumerate(seqs):
        if n:
            k, v = (fp4.rows_of(x, tables[b], p + n, bs) for x in (kv, vv))
            shown = ref.visible(ref.ancestors(trees[b]), p, p + n)
            ref.check_attention(loose[at:at + n], q[at:at + n], k, v, shown, scale, PIECES[kind], (b, kind, "loose"))
        at += n


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("prefix,n", [(0, 70), (3, 40), (61, 66), (500, 7)])
def test_any_mask(gpu_ctx, kind, prefix, n):
    """Masks that no tree gives: bits at random, rows that see nothing of the tree, bits behind it."""
    rng = np.random.default_rng(prefix + n)
    hq, hkv, d, bs = 6, 2, 64, 16
    keys, nb = prefix + n, -(-(prefix + n) // bs) + 2
    (kd, kv), (vd, vv) = pool_of(rng, kind, nb, hkv, bs, d), pool_of(rng, kind, nb, hkv, bs, d)
    tables = tables_of(rng, [keys], bs, nb)
    seen = rng.random((n, n)) < 0.3
    seen[n // 2] = False
    seen[0] = False
    seen[n - 1] = True
    words = np.concatenate([seen, rng.random((n, 64 * 3 - n)) < 0.5], 1)  # bits of nodes that are not there
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    got = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, [n], [keys], ref.words_of(words, 3), hkv, bs, nb, d ** -0.5))
    k, v = (fp4.rows_of(x, tables[0], keys, bs) for x in (kv, vv))
    shown = ref.visible(seen, prefix, keys)
    ref.check_attention(got, q, k, v, shown, d ** -0.5, PIECES[kind])
    if prefix == 0:
        assert (got[0] == 0).all() and (got[n // 2] == 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3.0e38])
@pytest.mark.parametrize("prefix", [0, 60, 330])
def test_what_a_row_does_not_see_does_not_reach_it(gpu_ctx, kind, bad, prefix):
    """K and V of one node hold what is not a number: its descendants get it, every other row is as without."""
    import torch

    if kind == "mxfp4" and not np.isnan(bad):
        pytest.skip("a 4-bit group holds numbers or NaN")
    rng = np.random.default_rng(prefix)
    hq, hkv, d, bs, n = 4, 2, 64, 16, 21
    keys, nb = prefix + n, -(-(prefix + n) // bs) + 2
    (kd, kv), (vd, vv) = pool_of(rng, kind, nb, hkv, bs, d), pool_of(rng, kind, nb, hkv, bs, d)
    tables = tables_of(rng, [keys], bs, nb)
    trees, mask = trees_of(rng, [n])
    seen = ref.ancestors(trees[0])
    hidden = 7
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    before = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, [n], [keys], mask, hkv, bs, nb, d ** -0.5))
    block, row = tables[0][(prefix + hidden) // bs], (prefix + hidden) % bs
    if kind == "mxfp4":
        for pool in (kd, vd):  # the scales of both KV heads' rows, all groups of head 0, the second of head 1
            scales = pool[nb * hkv * bs * (d // 2):].view(nb, hkv, bs, d // 32)
            scales[block, 0, row] = 255
            scales[block, 1, row, 1] = 255
    else:
        kd[block, :, row, 5] = bad
        vd[block, 0, row, 9] = bad
        vd[block, 1, row, 40] = bad
    got = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, [n], [keys], mask, hkv, bs, nb, d ** -0.5))
    blind = ~seen[:, hidden]
    assert blind.sum() > 3 and (~blind).sum() > 1
    assert np.array_equal(got[blind], before[blind])
    if np.isnan(bad):
        assert np.isnan(got[~blind, 0]).all() and np.isnan(got[~blind, 3]).all()
    # V alone: only the columns that hold it
    if kind != "mxfp4":
        kd[block, :, row, 5] = 0.5
        got = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, [n], [keys], mask, hkv, bs, nb, d ** -0.5))
        assert np.array_equal(got[blind], before[blind])
        cols = np.ones((hq, d), bool)
        cols[:2, 9] = cols[2:, 40] = False
        assert np.isfinite(got[:, cols]).all()
        if not np.isfinite(bad):
            at = got[~blind][:, ~cols]
            assert np.isnan(at).all() if np.isnan(bad) else (at == bad).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
def test_large_and_equal_scores(gpu_ctx, kind):
    """Scores of hundreds (one key holds nearly all weight), and rows whose scores are all equal."""
    rng = np.random.default_rng(5)
    hq, hkv, d, bs, prefix, n = 8, 2, 128, 16, 700, 9
    keys, nb = prefix + n, -(-(prefix + n) // bs) + 2
    (kd, kv), (vd, vv) = pool_of(rng, kind, nb, hkv, bs, d, 20.0), pool_of(rng, kind, nb, hkv, bs, d)
    tables = tables_of(rng, [keys], bs, nb)
    trees, mask = trees_of(rng, [n])
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    q[3] = 0.0
    got = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, [n], [keys], mask, hkv, bs, nb, d ** -0.5))
    k, v = (fp4.rows_of(x, tables[0], keys, bs) for x in (kv, vv))
    ref.check_attention(got, q, k, v, ref.visible(ref.ancestors(trees[0]), prefix, keys), d ** -0.5, PIECES[kind])


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
def test_one_node_is_a_decode_step(gpu_ctx, kind):
    import torch

    rng = np.random.default_rng(9)
    hq, hkv, d, bs, lens = 32, 8, 128, 16, [1, 300, 64, 2049]
    nb = sum(-(-n // bs) for n in lens) + 1
    (kd, kv), (vd, vv) = pool_of(rng, kind, nb, hkv, bs, d), pool_of(rng, kind, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((len(lens), hq, d)).astype(np.float32)
    got = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, [1] * 4, lens, np.ones((4, 1), np.int64), hkv, bs, nb, d ** -0.5))
    want = torch.empty(q.shape, device="cuda")
    gpu_ctx.attn_decode_paged(dev(q), kd, vd, dtype_of(kind), dev(tables), dev(np.asarray(lens, np.int32)), max(lens), hkv, bs, nb,
                              d ** -0.5, want)
    want = checked(gpu_ctx, want)
    for b, n in enumerate(lens):
        k, v = (fp4.rows_of(x, tables[b], n, bs) for x in (kv, vv))
        _, err = ref.expected(q[b:b + 1], k, v, np.ones((1, n), bool), d ** -0.5, ref.additions(n, 6), 6)
        off = np.sqrt(((got[b] - want[b]).astype(np.float64) ** 2).sum(-1))
        assert (off <= 2 * ref.ROW * err[0]).all(), b  # each within ROW times its size


def test_a_long_cache_past_32_bit_offsets(gpu_ctx):
    """Rows that lie more than 2^32 bytes into an f32 pool, and more than 2^31 elements."""
    import torch

    hq, hkv, d, bs, nb = 2, 1, 128, 16, 1 << 20  # 8 GiB an array
    rng = np.random.default_rng(4)
    k, v = (torch.zeros(nb, hkv, bs, d, device="cuda") for _ in range(2))
    lens, nodes = [100, 40], [5, 3]
    tables = np.stack([nb - 1 - np.arange(7), nb // 2 + 7 - np.arange(7)]).astype(np.int32)
    rows = [rng.standard_normal((7, hkv, bs, d)).astype(np.float32) for _ in range(4)]
    for pool, a, b in ((k, rows[0], rows[1]), (v, rows[2], rows[3])):
        pool[torch.from_numpy(tables[0]).long().cuda()] = dev(a)
        pool[torch.from_numpy(tables[1]).long().cuda()] = dev(b)
    trees, mask = trees_of(rng, nodes)
    q = rng.standard_normal((8, hq, d)).astype(np.float32)
    got = checked(gpu_ctx, attend(gpu_ctx, "f32", q, (k, v), tables, nodes, lens, mask, hkv, bs, nb, d ** -0.5))
    for b, at in ((0, slice(0, 5)), (1, slice(5, 8))):
        kk, vv = (x.transpose(0, 2, 1, 3).reshape(-1, hkv, d)[:lens[b]].astype(np.float64) for x in (rows[b], rows[2 + b]))
        shown = ref.visible(ref.ancestors(trees[b]), lens[b] - nodes[b], lens[b])
        ref.check_attention(got[at], q[at], kk, vv, shown, d ** -0.5, 6, b)


def small(rng, kind="bf16", lens=(50, 90), nodes=(4, 7), hq=4, hkv=2, d=64, bs=16):
    nb = sum(-(-n // bs) for n in lens) + 2
    pools = [pool_of(rng, kind, nb, hkv, bs, d) for _ in range(2)]
    trees, mask = trees_of(rng, list(nodes))
    q = rng.standard_normal((sum(nodes), hq, d)).astype(np.float32)
    return dict(kind=kind, q=q, pools=(pools[0][0], pools[1][0]), tables=tables_of(rng, list(lens), bs, nb), nodes=list(nodes),
                lens=list(lens), mask=mask, hkv=hkv, bs=bs, nb=nb, scale=d ** -0.5)


def test_rows_behind_the_last_sequence_are_left(gpu_ctx):
    import torch

    s = small(np.random.default_rng(1))
    want = checked(gpu_ctx, attend(gpu_ctx, **s))
    n = s["q"].shape[0]
    q = np.concatenate([s["q"], s["q"][:3]])
    mask = np.concatenate([s["mask"], s["mask"][:3]])
    out = torch.full((n + 3,) + s["q"].shape[1:], 3.25, device="cuda")
    got = checked(gpu_ctx, attend(gpu_ctx, **dict(s, q=q, mask=mask), out=out))
    assert np.array_equal(got[:n], want) and (got[n:] == 3.25).all()


def test_bad_metadata_is_reported(gpu_ctx):
    from ferrisinfer_amd import FerrisError

    rng = np.random.default_rng(2)
    s = small(rng)
    good = checked(gpu_ctx, attend(gpu_ctx, **s))
    # a block outside the pool, in the first sequence: the second is as it was
    tables = s["tables"].copy()
    tables[0, 1] = s["nb"]
    out = attend(gpu_ctx, **dict(s, tables=tables))
    with pytest.raises(FerrisError) as e:
        gpu_ctx.check_faults()
    assert "block" in e.value.message and np.array_equal(out.cpu().numpy()[4:], good[4:])
    # a length past max_context_len, and a tree of more nodes than max_query_len
    out = attend(gpu_ctx, **s, longest=60)
    with pytest.raises(FerrisError) as e:
        gpu_ctx.check_faults()
    assert "context" in e.value.message and np.array_equal(out.cpu().numpy()[:4], good[:4])
    out = attend(gpu_ctx, **s, most=5)
    with pytest.raises(FerrisError) as e:
        gpu_ctx.check_faults()
    got = out.cpu().numpy()
    assert "query" in e.value.message and (got[9:] == -7.0).all()
    assert np.abs(got[:9] - good[:9]).max() < 1e-5  # of values below 4, sums of f32 parts
    # lengths shorter than the tree: nodes without a cached row, rows that see none of the others
    short = checked(gpu_ctx, attend(gpu_ctx, **dict(s, lens=[2, -5]), longest=90))
    assert (short[4:] == 0).all() and np.isfinite(short).all() and (short[:2] == 0).all()


def test_refusals(gpu_ctx):
    import torch

    from ferrisinfer_amd import FerrisError

    s = small(np.random.default_rng(3))
    cu, lens = dev(np.array([0, 4, 11], np.int32)), dev(np.array([50, 90], np.int32))
    q, out, mask, tables = dev(s["q"]), torch.empty(s["q"].shape, device="cuda"), dev(s["mask"]), dev(s["tables"])
    base = dict(q=q, k_cache=s["pools"][0], v_cache=s["pools"][1], kv_dtype=1, block_tables=tables, cu_seqlens=cu,
                context_lens=lens, tree_mask=mask, max_query_len=7, max_context_len=90, num_kv_heads=2, block_size=16,
                num_blocks=s["nb"], scale=0.125, out=out)
    gpu_ctx.attn_tree_paged(**base)
    for change, kind in [
        (dict(kv_dtype=2), "InvalidType"), (dict(max_query_len=-1), "InvalidShape"), (dict(max_context_len=-1), "InvalidShape"),
        (dict(max_context_len=97), "InvalidShape"), (dict(num_kv_heads=3), "InvalidShape"), (dict(block_size=0), "InvalidConfig"),
        (dict(num_blocks=0), "InvalidConfig"), (dict(scale=0.0), "InvalidConfig"), (dict(scale=float("nan")), "InvalidConfig"),
        (dict(scale=float("inf")), "InvalidConfig"), (dict(max_query_len=65), "InvalidShape"),
        (dict(max_query_len=1025), "Unsupported"), (dict(k_cache=s["pools"][0].data_ptr() + 8), "InvalidLayout"),
        (dict(v_cache=None), "InvalidConfig"), (dict(q=q[:, :, :32].contiguous(), out=out[:, :, :16].contiguous()), "InvalidShape"),
        (dict(q=q.transpose(0, 1)), "InvalidLayout"), (dict(q=q.double()), "InvalidType"), (dict(tree_mask=mask.int()), "InvalidType"),
        (dict(tree_mask=mask[:10]), "InvalidShape"), (dict(out=out[:10]), "InvalidShape"), (dict(cu_seqlens=cu[:2]), "InvalidShape"),
        (dict(cu_seqlens=cu.long()), "InvalidType"), (dict(block_tables=tables[:1]), "InvalidShape"),
        (dict(block_tables=torch.cat([tables, tables], 1)[:, ::2]), "InvalidLayout"),
        (dict(q=torch.empty(11, 4, 48, device="cuda"), out=torch.empty(11, 4, 48, device="cuda")), "Unsupported"),
    ]:
        with pytest.raises(FerrisError) as e:
            gpu_ctx.attn_tree_paged(**dict(base, **change))
        assert e.value.kind == kind, (change.keys(), e.value)
    gpu_ctx.check_faults()


def test_graph_replays_and_another_stream(gpu_ctx):
    import torch

    from ferrisinfer_amd import Context

    rng = np.random.default_rng(6)
    s = small(rng, lens=(1500, 700), nodes=(9, 20))  # parts, joined through the workspace
    want = checked(gpu_ctx, attend(gpu_ctx, **s))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ctx = Context(0)
        assert ctx.stream == stream.cuda_stream
        q, out = dev(s["q"]), torch.empty(s["q"].shape, device="cuda")
        args = (q, *s["pools"], dtype_of("bf16"), dev(s["tables"]), dev(np.array([0, 9, 29], np.int32)),
                dev(np.array(s["lens"], np.int32)), dev(s["mask"]), 20, 1500, 2, 16, s["nb"], s["scale"], out)
        ctx.attn_tree_paged(*args)  # sizes the workspace
        stream.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ctx.attn_tree_paged(*args)
        for i in range(4):
            out.fill_(i)
            q.copy_(dev(s["q"] * (1 + i)))
            eager = torch.empty_like(out)
            ctx.attn_tree_paged(*args[:-1], eager)
            stream.synchronize()
            graph.replay()
            stream.synchronize()
            assert torch.equal(out, eager), i
        ctx.check_faults()
        ctx.close()
