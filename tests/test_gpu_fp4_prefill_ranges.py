"""Prefill attention over a 4-bit KV pool in ranges of keys (few new rows over a long prefix): launches that
are shown to run that way, by bits that differ from those of a launch too full for it."""
import ctypes

import numpy as np
import pytest

import fp4_accuracy as acc
import fp4_reference as fp4
from test_gpu_fp4_cache import dev, random_pool, tables_of
from test_gpu_fp4_prefill import prefill

pytestmark = pytest.mark.gpu

SHAPES = [  # cached, new, hq, hkv, d, block size
    (2500, 6, 8, 2, 64, 16),
    (3000, 40, 14, 2, 64, 16),
    (2100, 9, 4, 1, 128, 5),
    (4000, 3, 2, 2, 32, 16),
]
COPIES = 800  # of a sequence: more workgroups than run at a time


def one_sequence(shape, seed):
    cached, n, hq, hkv, d, bs = shape
    rng = np.random.default_rng(seed)
    nb = -(-(cached + n) // bs) + 2
    (kb, _), (vb, _) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, [cached + n], bs, nb)
    return rng, nb, kb, vb, tables, rng.standard_normal((n, hq, d)).astype(np.float32)


def whole(ctx, shape, q, pools, tables, nb):
    """The sequence's rows from a launch of many copies of it, whose tiles are not cut."""
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4

    cached, n, hq, hkv, d, bs = shape
    many = dev(q).repeat(COPIES, 1, 1)
    out = torch.empty_like(many)
    ctx.attn_prefill_paged(many, *pools, DTYPE_MXFP4, dev(tables).repeat(COPIES, 1),
                           dev(np.arange(0, COPIES * n + 1, n, dtype=np.int32)), dev(np.full(COPIES, cached + n, np.int32)), n,
                           hkv, bs, nb, d ** -0.5, out)
    ctx.sync()
    ctx.check_faults()
    assert torch.equal(out[:n], out[-n:])
    return out[:n].cpu().numpy()


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_ranges_and_whole_tiles_are_f32_accurate(gpu_ctx, shape):
    print(f"ranges {shape}", flush=True)
    cached, n, hq, hkv, d, bs = shape
    rng, nb, kb, vb, tables, q = one_sequence(shape, 100)
    pools = dev(kb), dev(vb)
    cut = prefill(gpu_ctx, q, pools, tables, [n], [cached + n], hkv, bs, nb, d ** -0.5)
    full = whole(gpu_ctx, shape, q, pools, tables, nb)
    assert not np.array_equal(cut, full)  # the sequence alone does run in ranges
    k, v = (fp4.rows_of(fp4.values(*fp4.split_pool(x, nb, hkv, bs, d)), tables[0], cached + n, bs) for x in (kb, vb))
    for got in (cut, full):
        acc.check(got, q, k, v, cached, d ** -0.5, acc.prefill_additions(cached + n))
    assert np.array_equal(cut, prefill(gpu_ctx, q, pools, tables, [n], [cached + n], hkv, bs, nb, d ** -0.5))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_a_range_of_nothing_but_nan(gpu_ctx, shape, where):
    """The keys of whole ranges are NaN in one kv head: its rows are NaN, whichever ranges those are, the other
    heads' and a sequence's beside it are not touched."""
    cached, n, hq, hkv, d, bs = shape
    rng, nb, kb, vb, tables, q = one_sequence(shape, 101)
    clean = prefill(gpu_ctx, q, (dev(kb), dev(vb)), tables, [n], [cached + n], hkv, bs, nb, d ** -0.5)
    scales = fp4.split_pool(kb, nb, hkv, bs, d)[1]
    at = {"first": 0, "middle": cached // 2, "last": cached - 700}[where]
    for t in range(at, at + 700):
        scales[tables[0, t // bs], 0, t % bs, 0] = 255
    got = prefill(gpu_ctx, q, (dev(kb), dev(vb)), tables, [n], [cached + n], hkv, bs, nb, d ** -0.5)
    group = hq // hkv
    assert np.isnan(got[:, :group]).all() and np.array_equal(got[:, group:], clean[:, group:])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_captured_and_replayed(gpu_ctx, shape):
    """A captured launch in ranges equals the eager one on every replay, with eager work between them."""
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, Context, kernel

    cached, n, hq, hkv, d, bs = shape
    rng, nb, kb, vb, tables, q0 = one_sequence(shape, 102)
    pools = dev(kb), dev(vb)
    qs = [dev(q0), *(dev(rng.standard_normal(q0.shape).astype(np.float32)) for _ in range(2))]
    lens = [cached + n, cached + n - 700, cached + n]
    cu, table, lens_d = dev(np.array([0, n], np.int32)), dev(tables), dev(np.array(lens[:1], np.int32))
    tail = (*pools, DTYPE_MXFP4, table, cu, lens_d, n, hkv, bs, nb, d ** -0.5)
    want = []
    for q, length in zip(qs, lens):
        lens_d.fill_(length)
        want.append(torch.empty_like(q))
        gpu_ctx.attn_prefill_paged(q, *tail, want[-1])
    torch.cuda.synchronize()
    assert not np.array_equal(want[0].cpu().numpy(), whole(gpu_ctx, shape, q0, pools, tables, nb))
    own = Context(0, use_torch_stream=False)
    q, out = qs[0].clone(), torch.empty_like(qs[0])
    lens_d.fill_(lens[0])
    torch.cuda.synchronize()
    own.attn_prefill_paged(q, *tail, out)  # sizes the workspace
    own.sync()
    lib = own.lib
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
        lens_d.fill_(lens[i])
        out.fill_(-1)
        torch.cuda.synchronize()
        kernel.check(lib.fi_graph_launch(own.handle, graph))
        own.sync()
        assert torch.equal(out, want[i]), i
        other = torch.empty_like(out)
        lens_d.fill_(lens[2])
        gpu_ctx.attn_prefill_paged(qs[2], *tail, other)
        torch.cuda.synchronize()
        assert torch.equal(other, want[2])
    own.check_faults()
    kernel.check(lib.fi_graph_destroy(graph))
    own.close()


def test_rows_without_keys_beside_ranges(gpu_ctx):
    """Rows that see no key, rows of a short sequence and rows over a long prefix in one launch of ranges."""
    rng = np.random.default_rng(103)
    hq, hkv, d, bs = 8, 2, 64, 16
    new, lens = [20, 300, 5, 33], [12, 290, 5, 3033]
    nb = sum(-(-n // bs) for n in lens) + 2
    (kb, kv), (vb, vv) = random_pool(rng, nb, hkv, bs, d), random_pool(rng, nb, hkv, bs, d)
    tables = tables_of(rng, lens, bs, nb)
    q = rng.standard_normal((sum(new), hq, d)).astype(np.float32)
    pools = dev(kb), dev(vb)
    got = prefill(gpu_ctx, q, pools, tables, new, lens, hkv, bs, nb, d ** -0.5)
    full = whole(gpu_ctx, (3000, 33, hq, hkv, d, bs), q[-33:], pools, tables[3:], nb)
    assert not np.array_equal(got[-33:], full)
    at = 0
    for b, (n, length) in enumerate(zip(new, lens)):
        mine, skip = slice(at, at + n), max(0, n - length)
        assert (got[mine][:skip] == 0).all()
        k, v = (fp4.rows_of(x, tables[b], length, bs) for x in (kv, vv))
        acc.check(got[mine][skip:], q[mine][skip:], k, v, length - n + skip, d ** -0.5, acc.prefill_additions(length), b)
        at += n
