"""Masks and positions of drafted trees, and the accepted path's rows moved in the pools."""
import numpy as np
import pytest

import draft_reference as ref
from test_gpu_fp4_cache import dev, tables_of
from test_gpu_tree_attention import dtype_of, pool_of

pytestmark = pytest.mark.gpu


def plan(ctx, trees, lens, words, most=None, rows=0, fill=-7):
    import torch

    nodes = [len(p) for p in trees]
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    t = sum(nodes) + rows
    mask = torch.full((t, words), fill, dtype=torch.int64, device="cuda")
    positions = torch.full((t,), fill, dtype=torch.int32, device="cuda")
    parents = np.concatenate([np.asarray(p, np.int32) for p in trees] + [np.zeros(rows, np.int32)])
    ctx.tree_plan(dev(parents), dev(cu), dev(np.asarray(lens, np.int32)), max(nodes) if most is None else most, mask, positions)
    ctx.sync()
    return mask.cpu().numpy(), positions.cpu().numpy()


@pytest.mark.parametrize("nodes,words", [([1], 1), ([8], 1), ([1, 0, 5, 64, 63, 2], 1), ([65, 128, 1, 0, 129], 3), ([100, 17], 5),
                                         ([1024, 3, 500], 16), ([300, 1, 1000], 17)])
def test_plan(gpu_ctx, nodes, words):
    rng = np.random.default_rng(sum(nodes))
    trees = [ref.grown(rng, n, 2 if b % 2 else 40) for b, n in enumerate(nodes)]
    lens = [n + int(rng.integers(0, 5000)) for n in nodes]
    lens[0] = nodes[0]  # no prefix
    mask, positions = plan(gpu_ctx, trees, lens, words, rows=2)
    gpu_ctx.check_faults()
    at = 0
    for p, n in zip(trees, lens):
        seen = ref.ancestors(p)
        if p:
            assert np.array_equal(mask[at:at + len(p)], ref.words_of(seen, words))
        assert np.array_equal(positions[at:at + len(p)], n - len(p) + seen.sum(1) - 1)
        at += len(p)
    assert (mask[at:] == -7).all() and (positions[at:] == -7).all()  # rows behind the last tree


def test_plan_reports(gpu_ctx):
    from ferrisinfer_amd import FerrisError

    good = [-1, 0, 1, 1, 3]
    for bad in (3, 4, 70, -2, 2 ** 31 - 1, -2 ** 31):
        tree = list(good)
        tree[3] = bad
        mask, positions = plan(gpu_ctx, [good, tree], [30, 40], 1)
        with pytest.raises(FerrisError) as e:
            gpu_ctx.check_faults()
        assert "parent" in e.value.message
        seen = ref.ancestors([-1, 0, 1, -1, 3])
        assert np.array_equal(mask[5:], ref.words_of(seen, 1)) and np.array_equal(positions[5:], 35 + seen.sum(1) - 1)
    mask, positions = plan(gpu_ctx, [good, [-1, 0]], [30, 20], 1, most=3)
    with pytest.raises(FerrisError) as e:
        gpu_ctx.check_faults()
    assert "query" in e.value.message
    assert (positions == [25, 26, 27, -7, -7, 18, 19]).all() and (mask[3:5] == -7).all()
    _, positions = plan(gpu_ctx, [good], [-2 ** 31], 1)  # a length below 0 counts as 0
    assert positions.tolist() == [-5, -4, -3, -3, -2]


def test_plan_refusals(gpu_ctx):
    import torch

    from ferrisinfer_amd import FerrisError

    i = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    base = dict(parents=i(6) - 1, cu_seqlens=i(3), context_lens=i(2), max_query_len=3, mask_out=i(6, 1).long(), positions_out=i(6))
    gpu_ctx.tree_plan(**base)
    for change, kind in [(dict(max_query_len=-1), "InvalidShape"), (dict(max_query_len=65), "InvalidShape"),
                         (dict(max_query_len=1025, mask_out=i(6, 20).long()), "Unsupported"), (dict(mask_out=i(5, 1).long()), "InvalidShape"),
                         (dict(mask_out=i(6, 1)), "InvalidType"), (dict(mask_out=i(6, 4).long()[:, ::2]), "InvalidLayout"),
                         (dict(positions_out=i(5)), "InvalidShape"), (dict(parents=i(6).float()), "InvalidType"),
                         (dict(cu_seqlens=i(2)), "InvalidShape"), (dict(mask_out=i(6, 0).long()), "InvalidShape")]:
        with pytest.raises(FerrisError) as e:
            gpu_ctx.tree_plan(**dict(base, **change))
        assert e.value.kind == kind, change.keys()
    gpu_ctx.check_faults()


# ---------------------------------------------------------------- the accepted rows

def rows(raw, kind, nb, hkv, bs, d):
    """A pool array's head rows as bytes [nb, hkv, bs, x]."""
    import torch

    if kind != "mxfp4":
        return raw.view(torch.uint8).cpu().numpy().reshape(nb, hkv, bs, -1)
    b = raw.cpu().numpy()
    n = nb * hkv * bs * (d // 2)
    return np.concatenate([b[:n].reshape(nb, hkv, bs, -1), b[n:].reshape(nb, hkv, bs, -1)], -1)


def moved(before, table, prefix, path, bs):
    after = before.copy()
    for i, node in enumerate(path):
        src, dst = prefix + node, prefix + 1 + i
        after[table[dst // bs], :, dst % bs] = before[table[src // bs], :, src % bs]
    return after


PATHS = [[], [1], [2], [1, 2, 3], [2, 3], [1, 3, 4, 8], [3, 4, 5, 6, 7, 8], [9], list(range(4, 24)), [1, 2, 9, 10, 30, 31]]


@pytest.mark.parametrize("kind,hkv,d,bs", [("f32", 2, 64, 16), ("f32", 3, 5, 4), ("f32", 8, 128, 1), ("bf16", 8, 128, 16),
                                           ("bf16", 1, 3, 5), ("bf16", 2, 32, 64), ("mxfp4", 8, 128, 16), ("mxfp4", 2, 64, 3),
                                           ("mxfp4", 3, 32, 16)])
@pytest.mark.parametrize("layers", [1, 3])
def test_keep(gpu_ctx, kind, hkv, d, bs, layers):
    rng = np.random.default_rng(d + bs)
    nodes = [40] * len(PATHS)
    prefix = [int(rng.integers(0, 70)) for _ in PATHS]
    lens = [p + n for p, n in zip(prefix, nodes)]
    nb = sum(-(-n // bs) for n in lens) + 2
    tables = tables_of(rng, lens, bs, nb)
    k, v = ([pool_of(rng, kind, nb, hkv, bs, d)[0] for _ in range(layers)] for _ in range(2))
    before = [rows(x, kind, nb, hkv, bs, d) for x in k + v]
    longest = max(len(p) for p in PATHS)
    path = np.array([p + [-1] * (longest - len(p)) for p in PATHS], np.int32)
    cu = np.arange(len(PATHS) + 1, dtype=np.int32) * 40
    gpu_ctx.kv_keep_path(k, v, dtype_of(kind), dev(tables), dev(cu), dev(np.asarray(lens, np.int32)), dev(path), nb, bs, hkv, d)
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    for x, old in zip(k + v, before):
        want = old
        for b, p in enumerate(PATHS):
            want = moved(want, tables[b], prefix[b], p, bs)
        assert np.array_equal(rows(x, kind, nb, hkv, bs, d), want)


def test_keep_many_layers(gpu_ctx):
    """More layers than one launch holds."""
    rng = np.random.default_rng(3)
    nb, hkv, bs, d = 3, 1, 16, 32
    k, v = ([pool_of(rng, "bf16", nb, hkv, bs, d)[0] for _ in range(130)] for _ in range(2))
    before = [rows(x, "bf16", nb, hkv, bs, d) for x in k + v]
    table = np.array([[2, 0]], np.int32)
    gpu_ctx.kv_keep_path(k, v, 1, dev(table), dev(np.array([0, 9], np.int32)), dev(np.array([21], np.int32)),
                         dev(np.array([[2, 5, 8]], np.int32)), nb, bs, hkv, d)
    gpu_ctx.sync()
    for x, old in zip(k + v, before):
        assert np.array_equal(rows(x, "bf16", nb, hkv, bs, d), moved(old, table[0], 12, [2, 5, 8], bs))


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
def test_keep_reports(gpu_ctx, kind):
    from ferrisinfer_amd import FerrisError

    rng = np.random.default_rng(4)
    nb, hkv, bs, d = 6, 2, 16, 64
    table = np.array([[2, 0, 4]], np.int32)

    def call(path, tables=table, lens=(40,), nodes=10):
        k, v = (pool_of(rng, kind, nb, hkv, bs, d)[0] for _ in range(2))
        before = [rows(x, kind, nb, hkv, bs, d) for x in (k, v)]
        gpu_ctx.kv_keep_path([k], [v], dtype_of(kind), dev(tables), dev(np.array([0, nodes], np.int32)), dev(np.array(lens, np.int32)),
                             dev(np.array([path], np.int32)), nb, bs, hkv, d)
        return (k, v), before

    # entries that end a path early: not rising, no node of the tree
    for path, taken in [([2, 2, 5], [2]), ([3, 1], [3]), ([2, 10], [2]), ([0, 4], []), ([2, 7, 2 ** 31 - 1], [2, 7])]:
        pools, before = call(path)
        with pytest.raises(FerrisError) as e:
            gpu_ctx.check_faults()
        assert "path" in e.value.message
        for x, old in zip(pools, before):
            assert np.array_equal(rows(x, kind, nb, hkv, bs, d), moved(old, table[0], 30, taken, bs))
    # what a path ends with is not looked at
    pools, before = call([2, -1, 1])
    gpu_ctx.check_faults()
    assert np.array_equal(rows(pools[0], kind, nb, hkv, bs, d), moved(before[0], table[0], 30, [2], bs))
    # blocks outside the pool, positions behind the table and before the sequence: rows that stay
    for tables, lens in [(np.array([[2, nb, 4]], np.int32), (40,)), (np.array([[2, -1, 4]], np.int32), (40,)), (table, (100,)), (table, (3,))]:
        pools, before = call([2, 5], tables, lens)
        with pytest.raises(FerrisError) as e:
            gpu_ctx.check_faults()
        assert "block" in e.value.message
        if lens[0] != 40:
            assert np.array_equal(rows(pools[0], kind, nb, hkv, bs, d), before[0])


def test_keep_refusals(gpu_ctx):
    import torch

    from ferrisinfer_amd import FerrisError

    i = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = lambda: torch.zeros(4, 2, 16, 64, device="cuda")  # noqa: E731
    base = dict(k_caches=[pool()], v_caches=[pool()], kv_dtype=0, block_tables=i(2, 2), cu_seqlens=i(3), context_lens=i(2), path=i(2, 3) - 1,
                num_blocks=4, block_size=16, num_kv_heads=2, head_dim=64)
    gpu_ctx.kv_keep_path(**base)
    gpu_ctx.kv_keep_path(**dict(base, k_caches=[], v_caches=[]))
    gpu_ctx.kv_keep_path(**dict(base, path=i(2, 0)))
    for change, kind in [(dict(kv_dtype=2), "InvalidType"), (dict(v_caches=[]), "InvalidShape"), (dict(num_blocks=0), "InvalidConfig"),
                         (dict(head_dim=0), "InvalidConfig"), (dict(k_caches=[None]), "InvalidConfig"), (dict(path=i(2, 3).long()), "InvalidType"),
                         (dict(path=i(3, 2).T), "InvalidLayout"), (dict(cu_seqlens=i(2)), "InvalidShape"),
                         (dict(block_tables=i(1, 2)), "InvalidShape"), (dict(context_lens=i(1)), "InvalidShape"),
                         (dict(kv_dtype=3, head_dim=48), "Unsupported"),
                         (dict(kv_dtype=3, k_caches=[base["k_caches"][0].data_ptr() + 8]), "InvalidLayout")]:
        with pytest.raises(FerrisError) as e:
            gpu_ctx.kv_keep_path(**dict(base, **change))
        assert e.value.kind == kind, change.keys()
    gpu_ctx.check_faults()


def test_graph_replays(gpu_ctx):
    import torch

    from ferrisinfer_amd import Context

    rng = np.random.default_rng(5)
    nb, hkv, bs, d = 8, 2, 16, 64
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ctx = Context(0)
        k, v = (pool_of(rng, "bf16", nb, hkv, bs, d)[0] for _ in range(2))
        table = np.array([[2, 0, 4], [1, 7, 3]], np.int32)
        path, parents = dev(np.zeros((2, 3), np.int32)), dev(np.zeros(20, np.int32))
        cu, lens = dev(np.array([0, 10, 20], np.int32)), dev(np.array([40, 33], np.int32))
        mask, positions = torch.zeros(20, 1, dtype=torch.int64, device="cuda"), torch.zeros(20, dtype=torch.int32, device="cuda")
        tables = dev(table)

        def call():
            ctx.tree_plan(parents, cu, lens, 10, mask, positions)
            ctx.kv_keep_path([k], [v], 1, tables, cu, lens, path, nb, bs, hkv, d)

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for paths in ([[2, 3, 9], [1, 4, -1]], [[-1, 0, 0], [5, 6, 7]], [[1, 2, 3], [9, -1, -1]]):
            trees = [ref.grown(rng, 10) for _ in range(2)]
            parents.copy_(dev(np.concatenate(trees).astype(np.int32)))
            path.copy_(dev(np.array(paths, np.int32)))
            before = [rows(x, "bf16", nb, hkv, bs, d) for x in (k, v)]
            graph.replay()
            stream.synchronize()
            for x, old in zip((k, v), before):
                for b, prefix in enumerate((30, 23)):
                    p = paths[b]
                    p = p[:p.index(-1)] if -1 in p else p
                    old = moved(old, table[b], prefix, p, bs)
                assert np.array_equal(rows(x, "bf16", nb, hkv, bs, d), old)
            want = np.concatenate([ref.words_of(ref.ancestors(p), 1) for p in trees])
            assert np.array_equal(mask.cpu().numpy(), want)
        ctx.check_faults()
        ctx.close()
