"""Serving from a KV cache held in 4 bits, as operators that can be timed and compared.

A paged pool may hold K and V as 4-bit floating point (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives) in groups of 32 consecutive elements of a head's row, each group with one power-of-two
scale: 17 bytes for 32 elements where bf16 takes 64.  The operators are the ones between a layer's
q|k|v projection and its output projection:

  consume   the q|k|v projection's partial sums: bias, RMS norm of every query and key head,
            rotation by one position or by several (time, height, width), append to the pool
  write     K/V rows appended to a 4-bit pool, and its blocks read back as values
  decode    one new token a sequence against a 4-bit pool
  prefill   prompt chunks against a 4-bit pool, causal, packed sequences

``run`` makes the framework's calls where ``own`` is true and computes the plain forms elsewhere.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 16
GROUP = 32  # elements that share a scale
EPS = 1e-6

# query heads, kv heads, head dimension of the decoders this repository is configured for
MODELS = {"tiny": (8, 2, 32), "qwen2": (14, 2, 64), "llama3": (32, 8, 128)}
THETA = {"tiny": 10000.0, "qwen2": 1000000.0, "llama3": 500000.0}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one chat user's next token over a small decoder's f32 pool: pure latency
        dict(name="consume-1", op="consume", model="qwen2", tokens=1, splits=7, pool="f32", axes=1, norm=True, bias=True,
             rotary=1.0),
        # the decode step of a 64-user batch, bf16 pool
        dict(name="consume-64", op="consume", model="llama3", tokens=64, splits=4, pool="bf16", axes=1, norm=True,
             bias=False, rotary=1.0),
        # a chunk of an image prompt: positions in time, height and width
        dict(name="consume-image-2k", op="consume", model="llama3", tokens=2048, splits=1, pool="bf16", axes=3, norm=True,
             bias=True, rotary=1.0),
        # the new rows of a 64-user batch
        dict(name="write-64", op="write", model="llama3", seqs=64, new=1),
        # a long prompt of odd length, taken in at once
        dict(name="write-prompt", op="write", model="llama3", seqs=1, new=6001),
        # one chat user, a short history
        dict(name="decode-1", op="decode", model="qwen2", seqs=1, min_ctx=700, max_ctx=700),
        # the standalone ragged batch: 64 users, histories between 128 and 2048 tokens
        dict(name="decode-64", op="decode", model="llama3", seqs=64, min_ctx=128, max_ctx=2048),
        # two users with very long histories: few rows, a long axis
        dict(name="decode-long", op="decode", model="llama3", seqs=2, min_ctx=60001, max_ctx=100003),
        # a full server, long histories
        dict(name="decode-128", op="decode", model="llama3", seqs=128, min_ctx=512, max_ctx=8192),
        # a few short prompts of odd lengths
        dict(name="prefill-3", op="prefill", model="qwen2", seqs=3, min_new=17, max_new=61, max_prefix=29),
        # prompts of mixed length arriving together, some behind a shared prefix
        dict(name="prefill-16", op="prefill", model="llama3", seqs=16, min_new=32, max_new=1024, max_prefix=512),
        # the second chunk of a long prompt
        dict(name="prefill-chunk", op="prefill", model="llama3", seqs=1, min_new=2048, max_new=2048, max_prefix=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["consume", "write", "decode", "decode", "prefill", "prefill"])
    model = rng.choice(sorted(MODELS))
    hq, hkv, d = MODELS[model]
    if op == "consume":
        return dict(op=op, model=model, tokens=_log(rng, 1, 2048), splits=rng.randint(1, 8) if rng.random() < 0.5 else 1,
                    pool=rng.choice(["f32", "bf16"]), axes=rng.choice([1, 1, 2, 3]), norm=rng.random() < 0.8,
                    bias=rng.random() < 0.5, rotary=rng.choice([1.0, 1.0, 0.5]))
    if op == "write":
        seqs = _log(rng, 1, 128)
        return dict(op=op, model=model, seqs=seqs, new=_log(rng, 1, 6001 // seqs))
    if op == "decode":
        seqs, longest = _log(rng, 1, 128), _log(rng, 1, 100003)
        longest = min(longest, max(1, 128 * 8192 * 1024 // (seqs * hkv * d)))
        return dict(op=op, model=model, seqs=seqs, max_ctx=longest, min_ctx=max(1, int(longest * rng.uniform(0.05, 1.0))))
    seqs = _log(rng, 1, 16)
    new = _log(rng, 1, 2048 // seqs)
    return dict(op=op, model=model, seqs=seqs, max_new=new, min_new=max(1, int(new * rng.uniform(0.1, 1.0))),
                max_prefix=rng.choice([0, _log(rng, 1, 2048)]))


# ---------------------------------------------------------------- sizes of a case

def _spread(n, lo, hi):
    """n ragged lengths in [lo, hi], the ends among them, in a fixed mixed order."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * 7919) % n) // (n - 1) for i in range(n)]  # 7919: a prime above any n


def _sequences(case):
    """(cached rows, new rows) of every sequence."""
    if case["op"] == "decode":
        return [(c - 1, 1) for c in _spread(case["seqs"], case["min_ctx"], case["max_ctx"])]
    if case["op"] == "write":  # into the middle of a history, so that blocks are shared with older rows
        return [((i * 5) % 40, case["new"]) for i in range(case["seqs"])]
    if case["op"] == "prefill":
        prefix = _spread(case["seqs"], 0, case["max_prefix"])
        return [(prefix[-1 - i], n) for i, n in enumerate(_spread(case["seqs"], case["min_new"], case["max_new"]))]
    return [((i * 5) % 40, n) for i, n in enumerate(_consume_chunks(case["tokens"]))]


def _consume_chunks(tokens):
    """The tokens of a step: up to 64 sequences."""
    n = min(tokens, 64)
    return [tokens // n + (i < tokens % n) for i in range(n)]


def work(case):
    hq, hkv, d = MODELS[case["model"]]
    seqs = _sequences(case)
    tokens = sum(n for _, n in seqs)
    row = hkv * (d // 2 + d // GROUP)  # bytes of one token's K (or V) row in 4 bits
    if case["op"] == "consume":
        w = (hq + 2 * hkv) * d
        cell = 4 if case["pool"] == "f32" else 2
        return {"bytes": tokens * (4 * case["splits"] * w + 4 * hq * d + 2 * cell * hkv * d), "flops": 12 * tokens * w}
    if case["op"] == "write":
        blocks = sum(-(-(p + n) // BLOCK) - p // BLOCK for p, n in seqs)
        read = blocks * BLOCK
        return {"bytes": tokens * 2 * (4 * hkv * d + row) + read * 2 * (4 * hkv * d + row), "flops": 4 * (tokens + read) * hkv * d}
    keys = sum(p + n for p, n in seqs)
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in seqs)  # (query, key) pairs that attend
    return {"bytes": 2 * keys * row + 8 * tokens * hq * d, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------- the 4-bit format

#: the values of the eight codes without a sign
LADDER = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(e):
    """2**e in f32 for whole e in [-126, 127], exactly."""
    return ((e + 127) << 23).view(torch.float32)


def _to_four_bits(x):
    """f32 [..., D] -> codes [..., D / 2] (element 2 i in the low half of byte i) and scales [..., D / 32]
    (the scale's exponent + 127).  The scale is the smallest power of two with no value at 7 scales or
    more, so every value is off by at most half a step, and between 2**-125 and 2**125; a group that
    holds an infinity or a NaN has scale 255 and reads as NaN."""
    g = x.float().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    bits = top.view(torch.int32)
    fine = torch.isfinite(top)
    e = ((bits >> 23) - 2 + ((bits & 0x7FFFFF) >= 0x600000).int()).clamp(2, 252)
    a = g.abs() * _power(127 - e).unsqueeze(-1)
    half = torch.where(a < 2, 2.0, torch.where(a < 4, 1.0, 0.5))  # 1 / step
    a = (torch.round(a * half) / half).clamp(max=6.0)  # ties to even
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4))
    code = torch.where(fine.unsqueeze(-1), code, torch.zeros_like(code)).to(torch.uint8)
    code = (code | (torch.signbit(g) & fine.unsqueeze(-1)).to(torch.uint8) << 3).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.where(fine, e, torch.full_like(e, 255)).to(torch.uint8)


def _pair_table(device):
    one = torch.tensor(LADDER + tuple(-v for v in LADDER), device=device)
    byte = torch.arange(256, device=device)
    return torch.stack([one[byte & 15], one[byte >> 4]], -1)


def _from_four_bits(codes, scales):
    """The f32 values of codes and scales."""
    v = _pair_table(codes.device)[codes.int()].flatten(-2).unflatten(-1, (-1, GROUP))
    s = torch.where(scales == 255, torch.full((), math.nan, device=codes.device), _power(scales.int() - 127))
    return (v * s.unsqueeze(-1)).flatten(-2)


def _pool_shapes(case, blocks):
    _, hkv, d = MODELS[case["model"]]
    return (blocks, hkv, BLOCK, d // 2), (blocks, hkv, BLOCK, d // GROUP)


def _parts_of(pool, case, blocks):
    """A 4-bit pool's codes [blocks, Hkv, BLOCK, D / 2] and, behind them, its scales [blocks, Hkv, BLOCK, D / 32]."""
    c, s = _pool_shapes(case, blocks)
    n = math.prod(c)
    return pool[:n].view(c), pool[n:].view(s)


# ---------------------------------------------------------------- inputs

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _metadata(case, seed):
    """Block tables, slots and lengths of the sequences over a pool handed out in a random order, as a
    paged server's are after a while; and, for the plain forms, where a packed row lies in a padded batch."""
    seqs = _sequences(case)
    lens = [p + n for p, n in seqs]
    blocks = [-(-x // BLOCK) for x in lens]
    pool = sum(blocks) + 8
    perm = np.random.RandomState(seed % (1 << 31)).permutation(pool)
    tables = np.zeros((len(seqs), max(blocks)), np.int32)
    widest = max(n for _, n in seqs)
    at, slots, cu, flat, padded, touched = 0, [], [0], [], [], []
    for i, ((prefix, new), k) in enumerate(zip(seqs, blocks)):
        tables[i, :k] = perm[at:at + k]
        at += k
        p = np.arange(prefix, prefix + new)
        slots.append(tables[i, p // BLOCK].astype(np.int64) * BLOCK + p % BLOCK)
        flat.append(i * widest + np.arange(new))
        padded.append(cu[-1] + np.minimum(np.arange(widest), new - 1))
        touched.append(tables[i, prefix // BLOCK:k])
        cu.append(cu[-1] + new)
    to = lambda a, t: torch.from_numpy(np.ascontiguousarray(a, t)).cuda()  # noqa: E731
    return dict(pool=pool, tables=to(tables, np.int32), lens=to(lens, np.int32), cu=to(cu, np.int32),
                slots=to(np.concatenate(slots), np.int64), flat=to(np.concatenate(flat), np.int64),
                padded=to(np.stack(padded), np.int64), touched=to(np.concatenate(touched), np.int32),
                max_ctx=max(lens), max_new=widest, rows=cu[-1])


def _filled_pool(case, blocks, g, spread):
    """A pool whose rows were written before: normal values, their size varying by channel as keys' do."""
    _, hkv, d = MODELS[case["model"]]
    size = torch.exp(spread * _normal(g, hkv, 1, d))
    pool = torch.empty(sum(math.prod(s) for s in _pool_shapes(case, blocks)), dtype=torch.uint8, device="cuda")
    codes, scales = _parts_of(pool, case, blocks)
    for i in range(0, blocks, 4096):
        n = min(4096, blocks - i)
        codes[i:i + n], scales[i:i + n] = _to_four_bits(_normal(g, n, hkv, BLOCK, d) * size)
    return pool


def _pair_axes(half, axes):
    """The axis whose position turns each rotary pair: about a quarter for time, the rest shared."""
    if axes == 1:
        return [0] * half
    first = half // 4 if axes == 3 else half // 2
    second = (half - first) // 2 if axes == 3 else half - first
    return [0] * first + [1] * second + [2] * (half - first - second)


def _consume_inputs(case, seed, g):
    hq, hkv, d = MODELS[case["model"]]
    t, w = case["tokens"], (hq + 2 * hkv) * d
    m = _metadata(case, seed)
    rotary = int(d * case["rotary"])
    r = np.random.RandomState(seed % (1 << 31))
    far = 4096
    positions = r.randint(0, far, (case["axes"], t)).astype(np.int32)
    inv = THETA[case["model"]] ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(far, dtype=torch.float64, device="cuda")[:, None] * inv
    kind = torch.float32 if case["pool"] == "f32" else torch.bfloat16
    return dict(m, parts=_normal(g, case["splits"], t, w) / math.sqrt(case["splits"]), rotary=rotary,
                bias=[_normal(g, n) * 0.1 for n in (hq * d, hkv * d, hkv * d)] if case["bias"] else None,
                norms=[1 + 0.2 * _normal(g, d) for _ in range(2)] if case["norm"] else None,
                positions=torch.from_numpy(positions).cuda(), pair_axes=_pair_axes(rotary // 2, case["axes"]),
                axis_rows=torch.tensor(_pair_axes(rotary // 2, case["axes"]), device="cuda"),
                cos=angle.cos().float(), sin=angle.sin().float(), far=far, q=torch.empty(t, hq, d, device="cuda"),
                k=_normal(g, m["pool"], hkv, BLOCK, d).to(kind), v=_normal(g, m["pool"], hkv, BLOCK, d).to(kind))


def prepare(case, seed):
    hq, hkv, d = MODELS[case["model"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "consume":
        return dict(_consume_inputs(case, seed, g), case=dict(case))
    m = _metadata(case, seed)
    s = dict(m, case=dict(case), k=_filled_pool(case, m["pool"], g, 0.5), v=_filled_pool(case, m["pool"], g, 0.1))
    if case["op"] == "write":
        n = int(m["touched"].numel()) * BLOCK
        size = torch.exp(0.5 * _normal(g, hkv, d))
        s["key"], s["value"] = _normal(g, m["rows"], hkv, d) * size, _normal(g, m["rows"], hkv, d)
        s["k_out"], s["v_out"] = (torch.empty(n, hkv, d, device="cuda") for _ in range(2))
    else:
        s["q"] = _normal(g, m["rows"], hq, d)
        s["out"] = torch.empty_like(s["q"])
    return s


# ---------------------------------------------------------------- one pass: the framework's calls

_CONTEXT = None


def _ctx():
    """A program keeps one context per GPU."""
    global _CONTEXT
    if _CONTEXT is None:
        from ferrisinfer_amd import Context

        _CONTEXT = Context(0)
    return _CONTEXT


def _own_consume(s):
    from ferrisinfer_amd import DTYPE_BF16, DTYPE_F32

    hq, hkv, d = MODELS[s["case"]["model"]]
    _ctx().qkv_norm_rope_append(s["parts"], s["case"]["splits"], s["bias"], s["norms"], EPS, s["positions"],
                                s["pair_axes"], s["cos"], s["sin"], s["rotary"], s["far"], s["slots"], s["k"], s["v"],
                                DTYPE_F32 if s["case"]["pool"] == "f32" else DTYPE_BF16, s["pool"], BLOCK, hq, hkv, d,
                                s["q"])
    return s["q"], s["k"], s["v"]


def _own_write(s):
    from ferrisinfer_amd import DTYPE_MXFP4

    _, hkv, d = MODELS[s["case"]["model"]]
    c = _ctx()
    c.kv_append(s["key"], s["value"], s["slots"], s["k"], s["v"], DTYPE_MXFP4, s["pool"], BLOCK, hkv, d)
    c.kv_gather(s["k"], s["v"], DTYPE_MXFP4, s["touched"], s["touched"].numel() * BLOCK, s["pool"], BLOCK, hkv, d,
                s["k_out"], s["v_out"])
    return s["k_out"], s["v_out"]


def _own_decode(s):
    from ferrisinfer_amd import DTYPE_MXFP4

    _, hkv, d = MODELS[s["case"]["model"]]
    _ctx().attn_decode_paged(s["q"], s["k"], s["v"], DTYPE_MXFP4, s["tables"], s["lens"], s["max_ctx"], hkv, BLOCK,
                             s["pool"], d ** -0.5, s["out"])
    return s["out"]


def _own_prefill(s):
    from ferrisinfer_amd import DTYPE_MXFP4

    _, hkv, d = MODELS[s["case"]["model"]]
    _ctx().attn_prefill_paged(s["q"], s["k"], s["v"], DTYPE_MXFP4, s["tables"], s["cu"], s["lens"], s["max_new"], hkv,
                              BLOCK, s["pool"], d ** -0.5, s["out"])
    return s["out"]


# ---------------------------------------------------------------- one pass: the plain forms

def _normed(x, weight):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _rotated(x, cos, sin):
    """x [T, heads, D] with its first 2 half elements turned by [T, half] cosines and sines."""
    half = cos.shape[-1]
    lo, hi = x[..., :half], x[..., half:2 * half]
    c, s = cos.unsqueeze(1), sin.unsqueeze(1)
    return torch.cat([lo * c - hi * s, hi * c + lo * s, x[..., 2 * half:]], -1)


def _plain_consume(s):
    hq, hkv, d = MODELS[s["case"]["model"]]
    x = s["parts"].sum(0)
    if s["bias"]:
        x = x + torch.cat(s["bias"])
    q, k, v = (y.unflatten(-1, (-1, d)) for y in x.split([hq * d, hkv * d, hkv * d], -1))
    if s["norms"]:
        q, k = _normed(q, s["norms"][0]), _normed(k, s["norms"][1])
    at = s["positions"].long()[s["axis_rows"]].T  # [T, half]
    pair = torch.arange(at.shape[1], device=at.device)
    cos, sin = s["cos"][at, pair], s["sin"][at, pair]
    q, k = _rotated(q, cos, sin), _rotated(k, cos, sin)
    block, row = s["slots"] // BLOCK, s["slots"] % BLOCK
    s["k"][block, :, row], s["v"][block, :, row] = k.to(s["k"].dtype), v.to(s["v"].dtype)
    return q, s["k"], s["v"]


def _plain_write(s):
    block, row = s["slots"] // BLOCK, s["slots"] % BLOCK
    return _written(s, s["k"], s["key"], block, row), _written(s, s["v"], s["value"], block, row)


def _written(s, pool, rows, block, row):
    codes, scales = _parts_of(pool, s["case"], s["pool"])
    codes[block, :, row], scales[block, :, row] = _to_four_bits(rows)
    at = s["touched"].long()
    return _from_four_bits(codes[at], scales[at]).transpose(1, 2).flatten(0, 1)


def _history(s, pool):
    """The f32 rows [B, Hkv, keys, D] that the block tables name."""
    codes, scales = _parts_of(pool, s["case"], s["pool"])
    at = s["tables"].long()
    return _from_four_bits(codes[at], scales[at]).transpose(1, 2).flatten(2, 3)


def _softmax(x):
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_decode(s):
    hq, hkv, d = MODELS[s["case"]["model"]]
    k = _history(s, s["k"])
    x = torch.matmul(s["q"].unflatten(1, (hkv, -1)), k.transpose(2, 3)) * d ** -0.5
    seen = torch.arange(k.shape[2], device=k.device) < s["lens"][:, None]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    return torch.matmul(_softmax(x), _history(s, s["v"])).flatten(1, 2)


def _plain_prefill(s):
    hq, hkv, d = MODELS[s["case"]["model"]]
    k, v = _history(s, s["k"]), _history(s, s["v"])
    q = s["q"][s["padded"]].unflatten(2, (hkv, -1)).permute(0, 2, 3, 1, 4)  # [B, Hkv, G, Q, D]
    x = torch.matmul(q, k.unsqueeze(2).transpose(3, 4)) * d ** -0.5
    new = s["cu"][1:] - s["cu"][:-1]
    at = (s["lens"] - new)[:, None] + torch.arange(s["max_new"], device=k.device)  # positions [B, Q]
    seen = torch.arange(k.shape[2], device=k.device) <= at[..., None]
    x = _softmax(x.masked_fill(~seen[:, None, None], -math.inf))
    return torch.matmul(x, v.unsqueeze(2)).permute(0, 3, 1, 2, 4).reshape(-1, hq, d)[s["flat"]]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"consume": _own_consume, "write": _own_write, "decode": _own_decode, "prefill": _own_prefill}[op](state)
    return {"consume": _plain_consume, "write": _plain_write, "decode": _plain_decode, "prefill": _plain_prefill}[op](state)


# ---------------------------------------------------------------- the definition, in 64 bits

def _defined_values(codes, scales):
    ladder = torch.tensor(LADDER, dtype=torch.float64, device=codes.device)
    nibble = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    value = torch.where(nibble >= 8, -1.0, 1.0) * ladder[nibble % 8]
    scale = torch.pow(2.0, scales.double() - 127)
    scale[scales == 255] = math.nan
    return value * scale.repeat_interleave(GROUP, -1)


def _defined_rounding(x):
    """The values 4 bits hold for x [..., D]: the scale's exponent from the group's largest value, then the
    nearest of the ladder's values, halfway ones to the even code."""
    g = x.double().reshape(*x.shape[:-1], -1, GROUP)
    top = g.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top))
    e = torch.where(torch.ldexp(torch.ones_like(e), e) > top, e - 1, e)  # log2 may round up to a whole number
    e = torch.where(torch.ldexp(torch.ones_like(e), e + 1) <= top, e + 1, e)
    e = torch.where(top / torch.exp2(e) >= 1.75, e + 1, e) - 2
    e = torch.where(top == 0, torch.full_like(e, -125), e).clamp(-125, 125)
    a = g.abs() / torch.exp2(e)
    code = torch.zeros_like(a)
    for i in range(7):
        middle = (LADDER[i] + LADDER[i + 1]) / 2
        code += (a > middle).double() + ((a == middle).double() if i % 2 else 0)
    ladder = torch.tensor(LADDER, dtype=torch.float64, device=x.device)
    return (torch.sign(g) * ladder[code.long()] * torch.exp2(e)).reshape(x.shape)


def _defined_attention(q, k, v, start):
    """q [n, Hq, D] at positions start .. start + n - 1 over k, v [keys, Hkv, D]."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    out = torch.empty_like(q)
    hidden = torch.arange(k.shape[0], device=q.device)[None] > start + torch.arange(n, device=q.device)[:, None]
    for h in range(hq):
        x = q[:, h] @ k[:, h // group].T.contiguous() / math.sqrt(d)
        x[hidden] = -math.inf
        out[:, h] = torch.softmax(x, -1) @ v[:, h // group]
    return out


def exact(case, seed):
    hq, hkv, d = MODELS[case["model"]]
    s = prepare(case, seed)
    if case["op"] == "consume":
        return _defined_consume(case, s)
    (kc, ks), (vc, vs) = (_parts_of(s[n], case, s["pool"]) for n in ("k", "v"))
    if case["op"] == "write":
        outs = []
        for codes, scales, rows in ((kc, ks, s["key"]), (vc, vs, s["value"])):
            values = _defined_values(codes, scales).transpose(1, 2).reshape(-1, hkv, d)
            values[s["slots"]] = _defined_rounding(rows)
            outs.append(values.reshape(-1, BLOCK, hkv, d)[s["touched"].long()].reshape(-1, hkv, d))
        return tuple(outs)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    cu = s["cu"].tolist()
    for b, n in enumerate(s["lens"].tolist()):
        at = s["tables"][b, :-(-n // BLOCK)].long()
        k, v = (_defined_values(c[at], z[at]).transpose(1, 2).reshape(-1, hkv, d)[:n] for c, z in ((kc, ks), (vc, vs)))
        if case["op"] == "decode":
            out[b:b + 1] = _defined_attention(s["q"][b:b + 1].double(), k, v, n - 1)
        else:
            rows = slice(cu[b], cu[b + 1])
            out[rows] = _defined_attention(s["q"][rows].double(), k, v, n - (cu[b + 1] - cu[b]))
    return out


def _defined_consume(case, s):
    hq, hkv, d = MODELS[case["model"]]
    x = s["parts"].double().sum(0)
    if s["bias"]:
        x += torch.cat(s["bias"]).double()
    x = x.reshape(-1, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if s["norms"]:
        q, k = (y * (y.pow(2).mean(-1, keepdim=True) + EPS).pow(-0.5) * w.double() for y, w in ((q, s["norms"][0]), (k, s["norms"][1])))
    half = s["rotary"] // 2
    outs = []
    for y in (q, k):
        z = y.clone()
        for i in range(half):
            at = s["positions"][s["pair_axes"][i]].long()
            c, sn = s["cos"][at, i].double()[:, None], s["sin"][at, i].double()[:, None]
            z[..., i] = y[..., i] * c - y[..., i + half] * sn
            z[..., i + half] = y[..., i + half] * c + y[..., i] * sn
        outs.append(z)
    pools = []
    for pool, rows in ((s["k"], outs[1]), (s["v"], v)):
        p = pool.double().transpose(1, 2).reshape(-1, hkv, d)
        p[s["slots"]] = rows
        pools.append(p.reshape(-1, BLOCK, hkv, d).transpose(1, 2).contiguous())
    return outs[0], pools[0], pools[1]
