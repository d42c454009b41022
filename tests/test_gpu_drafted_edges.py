"""Steps over drafted tokens where a draft, a mask or a length is at the end of what is allowed."""
import numpy as np
import pytest

import draft_reference as ref
import fp4_reference as fp4
from test_gpu_fp4_cache import dev, tables_of
from test_gpu_tree_attention import PIECES, attend, checked, pool_of, trees_of
from test_gpu_tree_rows import moved, rows
from test_gpu_verify_drafts import check, inputs, run

pytestmark = pytest.mark.gpu


FAR = [np.finfo(np.float32).min, np.float32(-1e30), np.float32(-1e20), np.float32(-1e9)]


@pytest.mark.parametrize("mode", ["given", "drawn", "distinct"])
@pytest.mark.parametrize("far", FAR, ids=lambda x: f"{x:.0e}")
@pytest.mark.parametrize("seqs,vocab", [(16, 20000), (16, 128256)])
def test_finite_masks(gpu_ctx, mode, far, seqs, vocab):
    """Tokens that are masked by a finite number: most segments of a row hold nothing else, and some rows.  The
    temperatures are those at which such a number's product with 1 / temperature is rounded, up and down."""
    rng = np.random.default_rng(31)
    nodes = [11] * seqs  # 23 million logits are summed a row a launch, 3.5 million all at once
    temperature = np.resize([0.0, 0.3, 0.6, 0.7, 0.8, 1.0, 1.3, 1e-9], seqs)
    s = inputs(rng, nodes, vocab, mode, temperature)
    x = s["logits"].reshape(seqs, 11, vocab)
    kept = np.argsort(-x, -1)[..., :50]
    masked = np.full_like(x, far)
    np.put_along_axis(masked, kept, np.take_along_axis(x, kept, -1), -1)
    x[:] = masked
    x[3, :, 5000:] = far                # all but the first tokens, some of them masked as well
    x[4] = far                          # rows of nothing else: all alike
    x[6, :, :vocab - 40] = far
    x[6, :, vocab - 40:] = -7.5
    x[7, :, :9000] = np.float32(-np.inf)  # both kinds
    x[9, 0] = -far                      # and the other end
    x[10, :, 17] = -far
    out = run(gpu_ctx, s, nodes, temperature, mode == "distinct")
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    check(out, s, nodes, temperature, mode == "distinct")


@pytest.mark.parametrize("mode", ["given", "drawn"])
def test_large_logits(gpu_ctx, mode):
    """Logits of any size that f32 has: only the largest ones weigh anything where f32's steps are wide."""
    rng = np.random.default_rng(32)
    sizes = [1e4, 1e7, 1e9, 1e11, 1e13, 1e15, 1e20, 1e30, 3e38]
    seqs, vocab = 2 * len(sizes), 9000
    nodes, temperature = [4] * seqs, np.resize([1.0, 0.37], seqs)
    s = inputs(rng, nodes, vocab, mode, temperature, liked=False)
    x = s["logits"].reshape(seqs, 4, vocab)
    for b in range(seqs):
        x[b] = (rng.integers(-40, 1, (4, vocab)) * 2.0 ** -6 + rng.choice([-1, 1])) * sizes[b // 2]
        s["tokens"].reshape(seqs, 4)[b, 1:] = x[b].argmax(-1)[s["parents"].reshape(seqs, 4)[b, 1:]]
    x[np.isinf(x)] = np.finfo(np.float32).max
    out = run(gpu_ctx, s, nodes, temperature)
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    check(out, s, nodes, temperature)


@pytest.mark.parametrize("vocab", [4096, 20000, 128256])
def test_greedy_rows_take_the_first_of_the_largest(gpu_ctx, vocab):
    """Equal maxima in a segment's waves and quads, in other segments, many of them; drafts on the first and on a later one."""
    rng = np.random.default_rng(vocab)
    places = [(300, 1030), (1030, 300, 4000), (255, 256), (256, 1024), (0, 4095), (4095, 1279, 1280), (1535, 1024, 770), (3, 1027, 2051, 3075),
              (vocab - 1, 512), (vocab - 1, vocab - 2), (511, 1023, 2047), (1100, 900)]
    nodes, temperature = [3] * (len(places) + 4), np.zeros(len(places) + 4)
    s = inputs(rng, nodes, vocab, "given", temperature, liked=False)
    x = s["logits"].reshape(-1, 3, vocab)
    s["parents"][:] = [-1, 0, 0] * len(nodes)
    tokens = s["tokens"].reshape(-1, 3)
    for b, at in enumerate(places):
        x[b, :, list(at)] = 40.0
        tokens[b, 1:] = (at[0], min(at)) if b % 2 else (max(at), at[0])
    for b in range(len(places), len(nodes)):  # logits of eight bits: hundreds of equal maxima
        x[b] = np.round(np.clip(x[b], -4, 4) * 2) / 2
        tokens[b, 1:] = rng.choice(np.nonzero(x[b, 0] == x[b, 0].max())[0], 2)
    x[-1] = 0.0
    tokens[-1, 1:] = 1, 0
    out = run(gpu_ctx, s, nodes, temperature)
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    check(out, s, nodes, temperature)


@pytest.mark.parametrize("seqs,ahead,vocab", [(24, 0, 5000), (16, 0, 140000), (8, 22, 100000)], ids=["rows at once", "a row a launch", "far down"])
def test_given_drafts_that_leave_little(gpu_ctx, seqs, ahead, vocab):
    """A draft that the model all but wants, rejected by a random number next to 1: it leaves 1e-7 of the row, and the next
    ones are held against that, which is within 2^-46 of the row."""
    rng = np.random.default_rng(33)
    size, n = 8, 8 + ahead
    nodes, temperature = [n] * seqs, np.ones(seqs)
    parents = list(range(-1, ahead)) + [ahead] * (size - 1)  # (`ahead` accepted ones in front)
    s = dict(logits=np.full((seqs * n, vocab), -200.0, np.float32), tokens=np.zeros(seqs * n, np.int32),
             parents=np.tile(parents, seqs).astype(np.int32), accept=rng.random(seqs * n).astype(np.float32),
             pick=rng.random(seqs).astype(np.float32), probs=None)
    x, tokens, u = s["logits"].reshape(seqs, n, vocab), s["tokens"].reshape(seqs, n), s["accept"].reshape(seqs, n)
    for b in range(seqs):
        liked = rng.choice(vocab, 9, replace=False)
        x[b, :, liked[0]] = 30.0
        tokens[b, :ahead + 1] = liked[0]
        u[b, :ahead + 1] = 0.0
        x[b, ahead, liked[1:]] = 30.0 - 15.9 - 2.08 + rng.random(8).astype(np.float32) / 64  # eight that have 1.2e-7 in all
        tokens[b, ahead + 1:] = [liked[0], liked[1], liked[0], liked[2], liked[1], liked[3], int(rng.integers(vocab))]
        u[b, ahead + 1] = 1 - 2.0 ** -24
    out = run(gpu_ctx, s, nodes, temperature)
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    check(out, s, nodes, temperature)


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("bs", [1, 5, 16])
@pytest.mark.parametrize("keys", [65, 64, 129, 3, 160])
def test_a_last_node_that_holds_no_numbers(gpu_ctx, kind, bs, keys):
    """The last node's V, which fills the rest of a chunk, in block tables just as wide as the keys: the rows that see the node
    get it, the others are as without."""
    rng = np.random.default_rng(keys + bs)
    hq, hkv, d, n = 4, 2, 64, 3
    tables = tables_of(rng, [keys, keys], bs, 2 * keys + 2)
    assert tables.shape == (2, -(-keys // bs))
    nb = 2 * keys + 2
    (kd, _), (vd, _) = pool_of(rng, kind, nb, hkv, bs, d), pool_of(rng, kind, nb, hkv, bs, d)
    seen = ref.ancestors([-1, 0, 0])  # the last node is seen by itself alone
    mask = np.concatenate([ref.words_of(seen, 1)] * 2)
    q = rng.standard_normal((2 * n, hq, d)).astype(np.float32)
    args = (gpu_ctx, kind, q, (kd, vd), tables, [n, n], [keys, keys], mask, hkv, bs, nb, d ** -0.5)
    before = checked(gpu_ctx, attend(*args))
    assert np.isfinite(before).all()
    for b in range(2):
        block, row = tables[b][(keys - 1) // bs], (keys - 1) % bs
        if kind == "mxfp4":
            vd[nb * hkv * bs * (d // 2):].view(nb, hkv, bs, d // 32)[block, 1, row, 0] = 255
        else:
            vd[block, 1, row, 3] = float("nan")
    got = checked(gpu_ctx, attend(*args))
    blind = np.tile([True, True, False], 2)
    assert np.array_equal(got[blind], before[blind])
    assert np.isnan(got[~blind][:, 2:, 3]).all() and np.array_equal(got[~blind][:, :2], before[~blind][:, :2])
    # (four bits: of the group's columns; the others have theirs)
    assert np.array_equal(got[~blind][:, :, 32:], before[~blind][:, :, 32:])


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("d,prefix", [(64, 490), (128, 497), (128, 5000)])
def test_channels_of_very_different_sizes(gpu_ctx, kind, d, prefix):
    """K's channels are 2^20 apart in size and Q's the other way round, by powers of two: the scores, and what an f32 product
    of them rounds, are as without."""
    rng = np.random.default_rng(d + prefix)
    hq, hkv, n, bs = 8, 2, 11, 16
    keys = prefix + n
    nb = -(-keys // bs) + 1
    tables = tables_of(rng, [keys], bs, nb)
    (kd, kv), (vd, vv) = pool_of(rng, kind, nb, hkv, bs, d), pool_of(rng, kind, nb, hkv, bs, d)
    by = np.where(np.arange(d // 32) % 2, -12, 8)
    each = np.repeat(np.exp2(by), 32)
    if kind == "mxfp4":
        scales = kd[nb * hkv * bs * (d // 2):].view(-1, d // 32)
        scales.copy_(dev((scales.cpu().numpy().astype(np.int64) + by).astype(np.uint8)))
    else:
        kd *= dev(each.astype(np.float32)).to(kd.dtype)
    kv = kv * each
    trees, mask = trees_of(rng, [n])
    q = (rng.standard_normal((n, hq, d)) / each).astype(np.float32)
    got = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, [n], [keys], mask, hkv, bs, nb, d ** -0.5))
    k, v = (fp4.rows_of(x, tables[0], keys, bs) for x in (kv, vv))
    ref.check_attention(got, q, k, v, ref.visible(ref.ancestors(trees[0]), prefix, keys), d ** -0.5, PIECES[kind])


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("prefix", [400, 3000])
@pytest.mark.parametrize("ahead", [8.0, 14.0, 20.0, 30.0, 45.0])
def test_a_key_that_takes_the_weight_and_gives_nothing(gpu_ctx, kind, prefix, ahead):
    """The first key's score is far above the others' and its V is zero: what is left are weights of 2^-12 to 2^-65."""
    rng = np.random.default_rng(prefix)
    hq, hkv, d, n, bs = 8, 2, 64, 9, 16
    keys = prefix + n
    nb = -(-keys // bs) + 1
    tables = tables_of(rng, [keys], bs, nb)
    (kd, kv), (vd, vv) = pool_of(rng, kind, nb, hkv, bs, d), pool_of(rng, kind, nb, hkv, bs, d)
    first = tables[0, 0]
    if kind == "mxfp4":
        for pool, code in ((kd, 0x22), (vd, 0)):  # codes of 1, of 0; scales of 1
            pool[:nb * hkv * bs * (d // 2)].view(nb, hkv, bs, d // 2)[first, :, 0] = code
            pool[nb * hkv * bs * (d // 2):].view(nb, hkv, bs, d // 32)[first, :, 0] = 127
    else:
        kd[first, :, 0] = 1.0
        vd[first, :, 0] = 0.0
    kv[first, :, 0], vv[first, :, 0] = 1.0, 0.0
    trees, mask = trees_of(rng, [n])
    q = rng.standard_normal((n, hq, d)).astype(np.float32) * np.float32(0.1)
    q += np.float32(ahead / np.sqrt(d))  # the first key's score: `ahead` and a little
    got = checked(gpu_ctx, attend(gpu_ctx, kind, q, (kd, vd), tables, [n], [keys], mask, hkv, bs, nb, d ** -0.5))
    k, v = (fp4.rows_of(x, tables[0], keys, bs) for x in (kv, vv))
    ref.check_attention(got, q, k, v, ref.visible(ref.ancestors(trees[0]), prefix, keys), d ** -0.5, PIECES[kind])


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
def test_lengths_past_a_bound_of_nothing(gpu_ctx, kind):
    """max_context_len 0: no row sees a key, whatever the lengths are, and those are reported."""
    from ferrisinfer_amd import FerrisError

    rng = np.random.default_rng(34)
    hkv, d, bs, nb, nodes = 2, 64, 16, 8, [3, 5, 2]
    pools = [pool_of(rng, kind, nb, hkv, bs, d)[0] for _ in range(2)]
    _, mask = trees_of(rng, nodes)
    q = rng.standard_normal((10, 4, d)).astype(np.float32)
    for lens in ([20, 30, 2], [20, 0, 2]):
        out = attend(gpu_ctx, kind, q, pools, tables_of(rng, lens, bs, nb), nodes, lens, mask, hkv, bs, nb, 0.1, longest=0)
        with pytest.raises(FerrisError) as e:
            gpu_ctx.check_faults()
        assert "context" in e.value.message and bool((out == 0).all())


@pytest.mark.parametrize("seqs", [1, 3])
def test_steps_without_rows(gpu_ctx, seqs):
    """No sequence has a node, and the arrays of rows none: an empty tensor has no address."""
    import torch

    i = lambda *n: torch.full(n, 5, dtype=torch.int32, device="cuda")  # noqa: E731
    f = lambda *n: torch.full(n, 5.0, device="cuda")  # noqa: E731
    mask, cu, lens = torch.zeros((0, 1), dtype=torch.int64, device="cuda"), i(seqs + 1) * 0, i(seqs)
    gpu_ctx.tree_plan(i(0), cu, lens, 4, mask, i(0))
    pools = [torch.zeros(4, 2, 16, 64, device="cuda") for _ in range(2)]
    gpu_ctx.attn_tree_paged(f(0, 4, 64), *pools, 0, i(seqs, 1) * 0, cu, lens, mask, 4, 16, 2, 16, 4, 0.1, f(0, 4, 64))
    for probs in (None, f(0, 50)):
        tokens, path, count, prob = i(seqs, 4), i(seqs, 3), i(seqs), f(seqs)
        gpu_ctx.verify_drafts(f(0, 50), i(0), i(0), cu, 4, f(seqs), f(0), f(seqs), probs, False, tokens, path, count, prob)
        gpu_ctx.sync()
        assert bool((tokens == -1).all()) and bool((path == -1).all()) and bool((count == 0).all()) and bool((prob == 0).all())
    gpu_ctx.kv_keep_path([pools[0]], [pools[1]], 0, i(seqs, 1) * 0, cu, lens, path, 4, 16, 2, 64)
    gpu_ctx.check_faults()
    # lengths that say otherwise are reported: rows that are not there are not read
    cu[-1] = 2
    gpu_ctx.verify_drafts(f(0, 50), i(0), i(0), cu, 4, f(seqs), f(0), f(seqs), None, False, tokens, path, count, prob)
    from ferrisinfer_amd import FerrisError

    with pytest.raises(FerrisError) as e:
        gpu_ctx.check_faults()
    assert "query" in e.value.message and bool((tokens == -1).all())


@pytest.mark.parametrize("layers", [1, 3, 70])
def test_pools_that_are_listed_more_than_once(gpu_ctx, layers):
    """Layers that share a cache, and K and V in one array: the rows move once."""
    rng = np.random.default_rng(35)
    nb, hkv, bs, d, paths = 6, 2, 16, 32, [[2, 3, 5, 8], [1, 4, 5, 9]]
    pools = [pool_of(rng, "bf16", nb, hkv, bs, d)[0] for _ in range(2)]
    table = np.array([[2, 0, 4], [1, 5, 3]], np.int32)
    for k, v in [([pools[0]], [pools[0]]), ([pools[0]] * 2, [pools[1]] * 2), ([pools[0], pools[1]], [pools[1], pools[0]])]:
        before = [rows(x, "bf16", nb, hkv, bs, d) for x in pools]
        gpu_ctx.kv_keep_path(k * layers, v * layers, 1, dev(table), dev(np.array([0, 10, 20], np.int32)), dev(np.array([40, 33], np.int32)),
                             dev(np.array(paths, np.int32)), nb, bs, hkv, d)
        gpu_ctx.sync()
        gpu_ctx.check_faults()
        for x, old in zip(pools, before):
            if x is pools[0] or len(k) > 1:
                for b, prefix in enumerate((30, 23)):
                    old = moved(old, table[b], prefix, paths[b], bs)
            assert np.array_equal(rows(x, "bf16", nb, hkv, bs, d), old)
