"""The q|k|v consumer with head norms and position axes against 64-bit numpy, over f32, bf16 and
4-bit pools."""
import numpy as np
import pytest

import fp4_reference as fp4

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24


def dev(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def inputs(rng, t, hq, hkv, d, splits, axes, rotary, bias, norm, bs, far=96, kind="f32", size=1.0):
    w = (hq + 2 * hkv) * d
    half = rotary // 2
    nb = -(-t // bs) + 2
    angle = rng.uniform(0, 6.28, (far, half))
    return dict(parts=(size * rng.standard_normal((splits, t, w))).astype(np.float32),
                bias=[rng.standard_normal(n).astype(np.float32) for n in (hq * d, hkv * d, hkv * d)] if bias else None,
                norms=[(1 + 0.3 * rng.standard_normal(d)).astype(np.float32) for _ in range(2)] if norm else None,
                positions=rng.integers(0, far, (axes, t)).astype(np.int32),
                pair_axes=rng.integers(0, axes, half).tolist(), far=far, nb=nb,
                cos=np.cos(angle).astype(np.float32), sin=np.sin(angle).astype(np.float32),
                slots=rng.permutation(nb * bs)[:t].astype(np.int64))


def reference(x, hq, hkv, d, rotary, eps):
    """(q, k, v) [T, heads, D] in 64 bits, and how far each may be off in f32, absolutely."""
    parts = x["parts"].astype(np.float64)
    y = parts.sum(0)
    splits = parts.shape[0]
    off = np.abs(parts).sum(0) * splits  # half steps: every partial sum rounds once
    if x["bias"]:
        b = np.concatenate(x["bias"]).astype(np.float64)
        y, off = y + b, off + np.abs(y + b)
    y, off = y.reshape(-1, hq + 2 * hkv, d), off.reshape(-1, hq + 2 * hkv, d)
    outs, offs = [], []
    half = rotary // 2
    at = x["positions"][x["pair_axes"], :].T if half else None  # [T, half]
    for i, part in enumerate((slice(0, hq), slice(hq, hq + hkv), slice(hq + hkv, None))):
        z, o = y[:, part].copy(), off[:, part].copy()
        if i < 2 and x["norms"]:
            w = x["norms"][i].astype(np.float64)
            r = 1 / np.sqrt((z * z).mean(-1, keepdims=True) + eps)
            # the inputs' own errors, through the element and through the mean; the mean's D additions and
            # squares, halved by the root; the root, the quotient and the two products
            moved = (np.abs(z) * o).mean(-1, keepdims=True) * r * r
            o = (o + np.abs(z) * moved) * np.abs(w) * r + np.abs(z * w) * r * (d / 2 + 6)
            z = z * r * w
        if i < 2 and half:
            c, s = (m[at, np.arange(half)].astype(np.float64)[:, None] for m in (x["cos"], x["sin"]))
            lo, hi, ol, oh = z[..., :half].copy(), z[..., half:rotary].copy(), o[..., :half].copy(), o[..., half:rotary].copy()
            z[..., :half], z[..., half:rotary] = lo * c - hi * s, hi * c + lo * s
            o[..., :half] = ol * np.abs(c) + oh * np.abs(s) + 2 * (np.abs(lo * c) + np.abs(hi * s))
            o[..., half:rotary] = oh * np.abs(c) + ol * np.abs(s) + 2 * (np.abs(hi * c) + np.abs(lo * s))
        outs.append(z)
        offs.append(o * HALF * 1.01 + 1e-30)  # 1.01: errors of errors
    return outs, offs


CASES = [
    # tokens, hq, hkv, d, splits, axes, rotary, bias, norm, block size
    (1, 14, 2, 64, 7, 1, 64, True, True, 16),
    (1, 1, 1, 32, 1, 1, 32, False, True, 16),
    (5, 8, 2, 32, 3, 3, 32, True, True, 5),
    (33, 32, 8, 128, 4, 1, 128, False, True, 16),
    (70, 14, 2, 64, 1, 3, 64, True, True, 16),
    (19, 6, 2, 128, 9, 4, 64, True, True, 16),     # half the dims rotary, more than one batch of splits
    (7, 4, 4, 64, 2, 2, 16, False, False, 1),      # no norm, a few rotary pairs
    (7, 4, 1, 128, 2, 1, 0, True, True, 16),       # no rotation
    (301, 5, 1, 32, 2, 2, 24, True, True, 7),
]


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("case", CASES)
def test_consumer(gpu_ctx, case, kind):
    import torch

    from ferrisinfer_amd import DTYPE_BF16, DTYPE_F32, DTYPE_MXFP4, kv_pool_bytes

    t, hq, hkv, d, splits, axes, rotary, bias, norm, bs = case
    print(f"consumer {case} {kind}", flush=True)
    rng = np.random.default_rng(t * 7 + d + splits)
    x = inputs(rng, t, hq, hkv, d, splits, axes, rotary, bias, norm, bs)
    if t > 4:
        x["slots"][2] = -1  # not appended; its query row still is
    dtype = {"f32": DTYPE_F32, "bf16": DTYPE_BF16, "mxfp4": DTYPE_MXFP4}[kind]
    before = [rng.integers(0, 100, kv_pool_bytes(dtype, x["nb"], bs, hkv, d), dtype=np.uint8) for _ in range(2)]
    pools = [dev(b) for b in before]
    q = torch.full((t + 1, hq, d), -9.0, device="cuda")
    put = lambda v: None if v is None else [dev(y) for y in v]  # noqa: E731
    gpu_ctx.qkv_norm_rope_append(dev(x["parts"]), splits, put(x["bias"]), put(x["norms"]), 1e-6, dev(x["positions"]),
                                 x["pair_axes"], dev(x["cos"]), dev(x["sin"]), rotary, x["far"], dev(x["slots"]), *pools,
                                 dtype, x["nb"], bs, hq, hkv, d, q[:t])
    gpu_ctx.sync()
    gpu_ctx.check_faults()
    outs, offs = reference(x, hq, hkv, d, rotary, 1e-6)
    got = q.cpu().numpy()
    assert (got[t] == -9.0).all()
    assert (np.abs(got[:t] - outs[0]) <= offs[0]).all()
    for pool, b, want, off in zip(pools, before, outs[1:], offs[1:]):
        raw = pool.cpu().numpy()
        live = [i for i in range(t) if x["slots"][i] >= 0]
        slots = x["slots"][live]
        if kind == "mxfp4":
            codes, scales = fp4.split_pool(raw.copy(), x["nb"], hkv, bs, d)
            rows = fp4.values(codes, scales)[slots // bs, :, slots % bs]
            # a value within its error of a border may take either side: between the codes of the ends
            lo, hi = want[live] - off[live], want[live] + off[live]
            scale = np.repeat(np.exp2(scales[slots // bs, :, slots % bs].astype(np.float64) - 127), 32, -1)
            mag = np.abs(rows) / scale
            half = np.where(mag < 2, 0.25, np.where(mag < 4, 0.5, 1.0)) * scale
            assert (rows - half <= hi).all() and (rows + half >= lo).all()
            top = np.abs(want[live]).reshape(len(live), hkv, -1, 32).max(-1)
            err = off[live].reshape(len(live), hkv, -1, 32).max(-1)
            s = np.exp2(scales[slots // bs, :, slots % bs].astype(np.float64) - 127)
            assert (top - err < 7 * s).all() and (top + err >= 3.5 * s).all()
            codes[slots // bs, :, slots % bs] = 0
            scales[slots // bs, :, slots % bs] = 0
            c0, s0 = fp4.split_pool(b.copy(), x["nb"], hkv, bs, d)
            c0[slots // bs, :, slots % bs] = 0
            s0[slots // bs, :, slots % bs] = 0
            assert np.array_equal(codes, c0) and np.array_equal(scales, s0)  # other rows are left
        else:
            cell = np.float32 if kind == "f32" else np.uint16
            grid = raw.view(cell).reshape(x["nb"], hkv, bs, d)
            rows = grid[slots // bs, :, slots % bs]
            if kind == "bf16":
                rows = (rows.astype(np.uint32) << 16).view(np.float32)
                off = off + (np.abs(want) + off) * 2.0 ** -8  # one more rounding
            assert (np.abs(rows - want[live]) <= off[live]).all()
            rest, rest0 = grid.copy(), b.view(cell).reshape(grid.shape).copy()
            rest[slots // bs, :, slots % bs] = 0
            rest0[slots // bs, :, slots % bs] = 0
            assert np.array_equal(rest, rest0, equal_nan=kind == "f32")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,rotary", [(14, 2, 64, 64), (32, 8, 128, 64), (8, 2, 32, 32)])
def test_without_norms_it_is_the_plain_consumer(gpu_ctx, kind, hq, hkv, d, rotary):
    import torch

    from ferrisinfer_amd import DTYPE_BF16, DTYPE_F32

    rng = np.random.default_rng(3)
    t, bs = 45, 16
    x = inputs(rng, t, hq, hkv, d, 5, 1, rotary, True, False, bs)
    dtype, cell = (DTYPE_F32, torch.float32) if kind == "f32" else (DTYPE_BF16, torch.bfloat16)
    got = []
    for norm_entry in (False, True):
        pools = [torch.zeros(x["nb"], hkv, bs, d, dtype=cell, device="cuda") for _ in range(2)]
        q = torch.zeros(t, hq, d, device="cuda")
        tail = (dev(x["cos"]), dev(x["sin"]), rotary, x["far"], dev(x["slots"]), *pools, dtype, x["nb"], bs, hq, hkv, d, q)
        parts, bias, pos = dev(x["parts"]), [dev(b) for b in x["bias"]], dev(x["positions"][0])
        if norm_entry:
            gpu_ctx.qkv_norm_rope_append(parts, 5, bias, None, 0.0, pos, None, *tail)
        else:
            gpu_ctx.qkv_rope_append(parts, 5, bias, pos, *tail)
        gpu_ctx.check_faults()
        got.append((q, *pools))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_four_bit_pool_through_the_plain_consumer_and_the_decode_entry(gpu_ctx):
    """fi_qkv_rope_append over a 4-bit pool equals the f32 consumer followed by fi_kv_append, and
    fi_attn_decode_paged_qkv the consumer followed by fi_attn_decode_paged."""
    import torch

    from ferrisinfer_amd import DTYPE_F32, DTYPE_MXFP4, FerrisError, kv_pool_bytes

    rng = np.random.default_rng(4)
    t, hq, hkv, d, bs = 9, 14, 2, 64, 16
    x = inputs(rng, t, hq, hkv, d, 3, 1, d, True, False, bs)
    parts, bias, pos = dev(x["parts"]), [dev(b) for b in x["bias"]], dev(x["positions"][0])
    nb = t
    table = np.arange(nb, dtype=np.int32)[:, None]
    lens = rng.integers(1, bs, t).astype(np.int32)
    slots = dev(np.arange(nb, dtype=np.int64) * bs + lens - 1)
    head = (dev(x["cos"]), dev(x["sin"]), d, x["far"], slots)
    f32 = [torch.zeros(nb, hkv, bs, d, device="cuda") for _ in range(2)]
    start = [torch.randint(0, 120, (kv_pool_bytes(DTYPE_MXFP4, nb, bs, hkv, d),), dtype=torch.uint8, device="cuda")
             for _ in range(2)]
    a, b, c = ([p.clone() for p in start] for _ in range(3))
    q, q2, q3 = (torch.zeros(t, hq, d, device="cuda") for _ in range(3))
    gpu_ctx.qkv_rope_append(parts, 3, bias, pos, *head, *f32, DTYPE_F32, nb, bs, hq, hkv, d, q)
    rows = [p.transpose(1, 2).reshape(-1, hkv, d)[slots].contiguous() for p in f32]
    gpu_ctx.kv_append(*rows, slots, *a, DTYPE_MXFP4, nb, bs, hkv, d)
    gpu_ctx.qkv_rope_append(parts, 3, bias, pos, *head, *b, DTYPE_MXFP4, nb, bs, hq, hkv, d, q2)
    assert torch.equal(q, q2) and all(torch.equal(m, n) for m, n in zip(a, b))
    out, out2 = torch.zeros_like(q), torch.zeros_like(q)
    gpu_ctx.attn_decode_paged(q, *a, DTYPE_MXFP4, dev(table), dev(lens), bs, hkv, bs, nb, 0.125, out)
    gpu_ctx.attn_decode_paged_qkv(parts, 3, bias, pos, *head, *c, DTYPE_MXFP4, dev(table), dev(lens), bs, hq, hkv, d, bs,
                                  nb, 0.125, out2, q_out=q3)
    gpu_ctx.check_faults()
    assert torch.equal(out, out2) and torch.equal(q, q3) and all(torch.equal(m, n) for m, n in zip(a, c))
    with pytest.raises(FerrisError) as e:
        gpu_ctx.attn_decode_paged_qkv(parts, 3, bias, pos, *head, *c, DTYPE_MXFP4, dev(table), dev(lens), bs, hq, hkv, d,
                                      bs, nb, 0.125, out2)
    assert e.value.kind == "InvalidConfig"


def test_bad_slots_positions_and_layouts(gpu_ctx):
    import torch

    from ferrisinfer_amd import DTYPE_F32, FerrisError

    rng = np.random.default_rng(6)
    t, hq, hkv, d, bs = 3, 2, 1, 32, 16
    x = inputs(rng, t, hq, hkv, d, 1, 2, d, False, True, bs)
    pools = [torch.zeros(x["nb"], hkv, bs, d, device="cuda") for _ in range(2)]
    q = torch.zeros(t, hq, d, device="cuda")

    def call(positions=x["positions"], slots=x["slots"], parts=dev(x["parts"]), axes=x["pair_axes"]):
        gpu_ctx.qkv_norm_rope_append(parts, 1, None, [dev(n) for n in x["norms"]], 1e-6, dev(positions), axes,
                                     dev(x["cos"]), dev(x["sin"]), d, x["far"], dev(slots), *pools, DTYPE_F32, x["nb"], bs,
                                     hq, hkv, d, q)
        gpu_ctx.check_faults()

    call()
    for bad in (x["far"], -1):
        p = x["positions"].copy()
        p[x["pair_axes"][0], 1] = bad
        with pytest.raises(FerrisError) as e:
            call(positions=p)
        assert e.value.kind == "Runtime"
    s = x["slots"].copy()
    s[1] = x["nb"] * bs
    with pytest.raises(FerrisError) as e:
        call(slots=s)
    assert e.value.kind == "Runtime"
    flat = torch.zeros(x["parts"].size + 1, device="cuda")
    with pytest.raises(FerrisError) as e:
        call(parts=flat[1:])
    assert e.value.kind == "InvalidLayout"
    with pytest.raises(FerrisError) as e:
        call(axes=x["pair_axes"][:-1])
    assert e.value.kind == "InvalidShape"
    call()


@pytest.mark.parametrize("kind", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("case", [
    # head rows past what one row a thread keeps resident: two, three, four, five and six rows a thread
    (1101, 8, 4, 128, 1, 3, 128, True, True, 16),
    (1101, 8, 4, 128, 2, 1, 64, False, True, 16),
    (701, 12, 6, 128, 1, 1, 128, True, True, 16),
    (520, 16, 8, 128, 2, 4, 128, True, False, 5),
    (430, 24, 8, 128, 1, 2, 128, False, True, 16),
    (350, 32, 8, 128, 1, 3, 128, True, True, 16),
    (1900, 14, 2, 64, 1, 3, 64, True, True, 16),     # two rows a thread, heads that do not fill the second
    (2100, 30, 2, 32, 1, 1, 32, True, True, 16),
])
def test_consumer_of_many_tokens(gpu_ctx, case, kind):
    test_consumer(gpu_ctx, case, kind)
