"""A model served over 4-bit KV pools, by the runtime and by the bf16-weight decoder, against a
64-bit forward pass that keeps K and V in the same 4-bit format."""
from dataclasses import replace

import numpy as np
import pytest

import fp4_reference as fp4
from test_gpu_fp4_cache import dev
from test_gpu_model import PACK_KEYS, build_pair, drive
from test_gpu_qkv_norm import reference as consumer64

pytestmark = pytest.mark.gpu


def logits64(cfg, w, ids):
    """Logits [len(ids), vocab] of the decoder (reference.rs:163-370) in f64, K and V read in 4 bits.
    Every key is read from the pool, the row's own among them, so one causal pass over a sequence gives
    every step's logits however its rows were chunked."""
    h, hq, hkv, eps = cfg["hidden"], cfg["heads"], cfg["kv_heads"], cfg["eps"]
    d, n = h // hq, len(ids)
    w = {k: v.astype(np.float64) for k, v in w.items()}
    norm = lambda x, g: x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * g  # noqa: E731
    angle = np.arange(n)[:, None] * cfg["theta"] ** (-2.0 * np.arange(d // 2) / d)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]

    def rope(x):
        lo, hi = x[..., :d // 2], x[..., d // 2:]
        return np.concatenate([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    def stored(x):
        return fp4.values(*fp4.quantise(x.astype(np.float32)))

    x = w["tok_embeddings.weight"][np.asarray(ids, np.int64)]
    for layer in range(cfg["layers"]):
        p = f"layers.{layer}."
        a = norm(x, w[p + "attention_norm.weight"])
        q = rope((a @ w[p + "attention.wq.weight"]).reshape(n, hq, d))
        k = stored(rope((a @ w[p + "attention.wk.weight"]).reshape(n, hkv, d)))
        v = stored((a @ w[p + "attention.wv.weight"]).reshape(n, hkv, d))
        x = x + fp4.attention(q, k, v, 0, d ** -0.5).reshape(n, h) @ w[p + "attention.wo.weight"]
        a = norm(x, w[p + "ffn_norm.weight"])
        gate = a @ w[p + "feed_forward.w3.weight"]
        x = x + (a @ w[p + "feed_forward.w1.weight"] * gate / (1 + np.exp(-gate))) @ w[p + "feed_forward.w2.weight"]
    return norm(x, w["norm.weight"]) @ w["output.weight"].T


@pytest.mark.parametrize("sharing", [False, True])
def test_runtime_over_a_four_bit_pool(orc, sharing):
    """Ticks and packing equal the reference scheduler's.  Every greedy token is the 64-bit pass's over
    the same history, but where that pass's two best logits are within 2e-2 of their size: a K or V
    element that f32 leaves at the other side of a rounding boundary takes the neighbouring code.
    Replayed decode ticks equal eager ones bit for bit."""
    from ferrisinfer_amd.workloads import TINY_LLAMA_C1, c1_requests, random_weights

    from test_gpu_graph import assert_same_run, make_runtime

    print(f"4-bit runtime, sharing {sharing}", flush=True)
    cfg = dict(TINY_LLAMA_C1, layers=2)
    weights = random_weights(cfg, seed=11)
    requests, kw = c1_requests(2), {}
    if sharing:  # prefixes shared inside a block (copied rows), chunked prefill, small batches
        rng = np.random.default_rng(7)
        base = rng.integers(0, cfg["vocab"], size=40).astype(np.uint32)
        requests = [(base.copy(), 6), (np.concatenate([base[:37], rng.integers(0, 4096, 9)]).astype(np.uint32), 5),
                    (np.concatenate([base[:32], rng.integers(0, 4096, 3)]).astype(np.uint32), 4), (base.copy(), 3)]
        kw = dict(max_batch=3, max_chunk=20, max_batch_tokens=50, min_share=16)
    _, ref, gpu = build_pair(orc, cfg, weights, kw, kv_dtype="mxfp4")
    rpacks, gpacks = [], []
    rid, rticks = drive(ref, requests, rpacks)
    gid, gticks = drive(gpu, requests, gpacks)
    assert rid == gid and [k for k, _ in rticks] == [k for k, _ in gticks]
    if sharing:
        assert any(u["reused"] > 0 for _, us in gticks for u in us)
        assert any(np.size(p["copy_count"]) and np.max(p["copy_count"]) > 0 for p in gpacks)
    else:  # with sharing, block ids depend on the tokens through what is released when
        for i, (a, b) in enumerate(zip(rpacks, gpacks)):
            for key in PACK_KEYS:
                assert np.array_equal(a[key], b[key]), (i, key)
    ties = 0
    for seq, (prompt, count) in zip(gid, requests):
        got = list(gpu.generated(seq))
        assert len(got) == count
        logits = logits64(cfg, weights, list(prompt) + got[:-1])[len(prompt) - 1:]
        for i, (token, row) in enumerate(zip(got, logits)):
            if token != int(row.argmax()):
                assert row.max() - row[token] <= 2e-2 * max(1.0, abs(row.max())), (seq, i, token, int(row.argmax()))
                ties += 1
    print(f"{ties} near ties", flush=True)
    assert ties <= 3
    assert gpu.pool_free_count() == 4096
    eager = make_runtime(cfg, weights, False, kw, kv_dtype="mxfp4")
    graph = make_runtime(cfg, weights, True, kw, kv_dtype="mxfp4")
    assert_same_run(eager, graph, requests)


def test_runtime_replays_decode_of_wide_groups_with_biases():
    """Head dim 64, 7 query heads to a K/V head and q/k/v biases: the runtime's ticks in 4 bits."""
    from ferrisinfer_amd.workloads import random_weights

    from test_gpu_graph import assert_same_run, make_runtime

    cfg = dict(hidden=896, intermediate=512, layers=1, heads=14, kv_heads=2, vocab=1024, max_pos=2048, eps=1e-6,
               theta=1000000.0, tie=False)
    weights = random_weights(cfg, seed=4, qkv_bias=True)
    rng = np.random.default_rng(3)
    requests = [(rng.integers(0, 1024, n).astype(np.uint32), 9) for n in (1, 15, 16, 300)]
    eager = make_runtime(cfg, weights, False, {}, kv_dtype="mxfp4")
    graph = make_runtime(cfg, weights, True, {}, kv_dtype="mxfp4")
    assert_same_run(eager, graph, requests)


@pytest.mark.parametrize("norms,axes", [(False, None), (True, None), (True, 3)])
def test_decoder_over_four_bit_pools(orc, norms, axes):
    """Two layers of the bf16-weight decoder over one mixed step: consumer, append, decode rows and a
    prefill chunk as they follow each other.  The last layer's consumer against 64 bits on the
    decoder's own q|k|v partials, its pool bytes against the format's rounding of them, its attention
    against 64 bits on its own queries and pools."""
    import torch

    from ferrisinfer_amd import DTYPE_MXFP4, Context
    from ferrisinfer_amd.bf16_decoder import Bf16Decoder, build_step_batch

    print(f"4-bit decoder, norms {norms}, axes {axes}", flush=True)
    h, f, hq, hkv, v, bs, eps = 1024, 1024, 8, 2, 2048, 16, 1e-6
    cfg = dict(hidden=h, intermediate=f, layers=2, heads=hq, kv_heads=hkv, vocab=v, max_pos=512, eps=eps, theta=500000.0,
               tie=False)
    d = h // hq
    rng = np.random.default_rng(9)
    decode_ctx, chunks = [37, 1, 300, 16], [(16, 19), (0, 50)]
    lens = decode_ctx + [p + n for p, n in chunks]
    nb = sum(-(-n // bs) for n in lens) + 3
    nd, t = len(decode_ctx), len(decode_ctx) + sum(n for _, n in chunks)
    wbits = lambda *s: dev(orc.f32_to_bf16((0.02 * rng.standard_normal(s)).astype(np.float32)).view(np.int16))  # noqa: E731
    near = lambda n: (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)  # noqa: E731
    ctx = Context(0)
    pair_axes = None if axes is None else [i % axes for i in range(d // 2)]
    dec = Bf16Decoder(ctx, cfg, nb, bs, max_tokens=t, max_last_rows=len(lens), kv_dtype=DTYPE_MXFP4, pair_axes=pair_axes)
    head_norms = [near(d), near(d)] if norms else None
    for _ in range(2):
        dec.set_layer(wbits(h, h), wbits(h, hkv * d), wbits(h, hkv * d), wbits(h, h), wbits(h, f), wbits(f, h), wbits(h, f),
                      dev(near(h)), dev(near(h)), *(map(dev, head_norms) if norms else ()))
    dec.set_head(dev(near(h)), wbits(v, h))
    for pool in dec.k_pools + dec.v_pools:
        codes, scales = fp4.quantise(rng.standard_normal((nb, hkv, bs, d)).astype(np.float32))
        pool.copy_(dev(fp4.pool_bytes(codes, scales)))
    batch, tables = build_step_batch(decode_ctx, chunks, bs, nb, seed=3)
    if axes:
        batch = replace(batch, positions=torch.stack([batch.positions, *(
            dev(rng.integers(0, 512, t).astype(np.int32)) for _ in range(axes - 1))]).contiguous())
    seen = {}
    name = "qkv_norm_rope_append" if norms or axes else "qkv_rope_append"
    call = getattr(ctx, name)

    def consume(parts, splits, *rest):
        seen.update(parts=parts.reshape(-1)[:splits * t * (hq + 2 * hkv) * d].clone().reshape(splits, t, -1))
        call(parts, splits, *rest)

    setattr(ctx, name, consume)
    x = dev((0.5 * rng.standard_normal((t, h))).astype(np.float32))
    out = dec.step(x, batch, head=False).clone()
    q, attn = dec.q[:t].cpu().numpy(), dec.attn[:t].cpu().numpy()
    pools = [p[-1].cpu().numpy() for p in (dec.k_pools, dec.v_pools)]
    setattr(ctx, name, call)
    again = dec.step(x, batch, head=False)  # the new rows are rewritten with the same bytes
    ctx.check_faults()
    assert torch.equal(out, again) and torch.isfinite(out).all()
    assert np.array_equal(pools[0], dec.k_pools[-1].cpu().numpy()) and np.array_equal(pools[1], dec.v_pools[-1].cpu().numpy())

    slots = batch.slot_mapping.cpu().numpy()
    positions = batch.positions.cpu().numpy().reshape(axes or 1, t)
    (rq, rk, rv), offs = consumer64(dict(parts=seen["parts"].cpu().numpy(), bias=None, norms=head_norms, positions=positions,
                                         pair_axes=pair_axes or [0] * (d // 2), cos=dec.cos.cpu().numpy(),
                                         sin=dec.sin.cpu().numpy()), hq, hkv, d, d, eps)
    assert (np.abs(q - rq) <= offs[0]).all()
    values = []
    for pool, want, off in zip(pools, (rk, rv), offs[1:]):
        codes, scales = fp4.split_pool(pool, nb, hkv, bs, d)
        values.append(fp4.values(codes, scales))
        got = values[-1][slots // bs, :, slots % bs]
        # a value within its f32 error of a rounding border may take either side
        scale = np.exp2(scales[slots // bs, :, slots % bs].astype(np.float64) - 127)
        top, err = (np.abs(z).reshape(t, hkv, -1, fp4.GROUP).max(-1) for z in (want, off))
        assert (top - err < 7 * scale).all() and (top + err >= 3.5 * scale).all()
        scale = np.repeat(scale, fp4.GROUP, -1)
        half = np.where(np.abs(got) < 2 * scale, 0.25, np.where(np.abs(got) < 4 * scale, 0.5, 1.0)) * scale
        assert (got - half <= want + off).all() and (got + half >= want - off).all()
    row = 0
    for s, length in enumerate(lens):
        count = 1 if s < nd else chunks[s - nd][1]
        k, vv = (fp4.rows_of(x, tables[s], length, bs) for x in values)
        mine = q[row:row + count]
        want = fp4.attention(mine, k, vv, length - count, d ** -0.5)
        off = fp4.attention_tolerance(mine, k, vv, d ** -0.5, length)
        assert np.abs(attn[row:row + count] - want).max() <= off, s
        row += count
    ctx.close()
