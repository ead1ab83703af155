"""The steps around the selector that performance is measured on: what a serving process runs before a selection (norm and
rotation of queries and keys, the quantised key cache) and after it (attention over the selected tokens).

A case is one call, as a layer of such a process makes it. `op` names the entry point:

  norm_rope  qk_norm_rope       per-head norm and position rotation of q and k, same type in and out
  step       indexer_qk_write   the indexer's q (e4m3, its scale folded into the head weights) and k (normed, rotated, quantised
                                into the key cache as it is written)
  write      cache_write        keys and values quantised into their caches
  read       cache_read         rows of a quantised cache back in bf16
  attend     sparse_attention   attention of every query token over the cache rows its selection names

Where `own` is false the same results come from elementary torch operations in 32 bits.
"""
from __future__ import annotations

import functools
import math
import os
import sys
from types import SimpleNamespace

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
AMAX_FLOOR = 2.0 ** -96  # of a row's largest magnitude: keeps the scale of a row of zeros positive
EPS = 1e-6


def _rope(tokens, q_heads, kv_heads, dim, rotary, dtype="bf16", norm="rms", interleaved=False, fused_qkv=True):
    return {"op": "norm_rope", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "dtype": dtype, "norm": norm, "interleaved": interleaved, "fused_qkv": fused_qkv}


def _step(tokens, heads=64, dim=128, rotary=64, dtype="bf16", interleaved=False):
    return {"op": "step", "tokens": tokens, "q_heads": heads, "dim": dim, "rotary": rotary, "dtype": dtype,
            "interleaved": interleaved}


def _write(tokens, kv_heads, dim=128, dtype="bf16"):
    return {"op": "write", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def _read(rows, picks, kv_heads, dim=128):
    return {"op": "read", "tokens": rows, "topk": picks, "kv_heads": kv_heads, "dim": dim}


def _attend(tokens, q_heads, kv_heads, topk, context, dtype="bf16", cache="fp8", dim=128, shared=False):
    return {"op": "attend", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "topk": topk, "context": context,
            "dtype": dtype, "cache": cache, "dim": dim, "shared": shared}


def listed():
    return [
        # one token of one request: launch latency
        dict(name="norm_rope_t1", **_rope(1, 64, 8, 128, 128)),
        # a prefill chunk, q and k as slices of the fused projection's output: the stream
        dict(name="norm_rope_t16k", **_rope(16384, 64, 8, 128, 128)),
        # 32-bit activations, an odd number of tokens, a head size and a rotated part that fill no power of two
        dict(name="norm_rope_odd_fp32", **_rope(1021, 6, 3, 80, 48, dtype="fp32", norm="layer", interleaved=True)),
        # the indexer's q and k of a decode batch ...
        dict(name="index_step_t64", **_step(64)),
        # ... and of a prefill chunk
        dict(name="index_step_t8k", **_step(8192)),
        # keys and values of a prefill chunk into an fp8 cache
        dict(name="cache_write_t8k", **_write(8192, 8)),
        # the rows that one token has selected, and the context of several requests, back from the cache
        dict(name="cache_read_1x2k", **_read(1, 2048, 1)),
        dict(name="cache_read_64x2k", **_read(64, 2048, 2)),
        # one request's decode step: few rows, the work has to be split over the selection
        dict(name="attend_t1_fp8", **_attend(1, 64, 8, 2048, 131072)),
        # a decode batch, 16-bit cache
        dict(name="attend_t64_bf16", **_attend(64, 64, 8, 2048, 8192, cache="same")),
        # an odd batch of small heads, another k, fp16
        dict(name="attend_t61_odd", **_attend(61, 21, 3, 1000, 5001, dtype="fp16", dim=64)),
        # a prefill chunk of one request, all query heads on one key head: the largest, bound by arithmetic
        dict(name="attend_t1k_mqa", **_attend(1024, 128, 1, 2048, 65536, shared=True)),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm_rope", "step", "write", "read", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "norm_rope":
        dim = rng.choice([64, 64, 80, 96, 128, 128, 192, 256])
        kv = rng.choice([1, 2, 3, 4, 8])
        q_heads = kv * rng.choice([1, 2, 5, 8])
        size = (q_heads + kv) * dim * (2 if dtype == "fp32" else 1)
        return _rope(spread(1, min(16384, 16384 * 72 * 128 // size)), q_heads, kv, dim, rng.choice([16, 32, 48, 64, dim]), dtype,
                     rng.choice(["rms", "rms", "layer", "none"]), rng.random() < 0.4, rng.random() < 0.7)
    if op == "step":
        return _step(spread(1, 8192), rng.choice([8, 16, 32, 64]), 128, rng.choice([32, 64, 128]), dtype, rng.random() < 0.5)
    if op == "write":
        return _write(spread(1, 8192), rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 96, 128, 128, 256]), dtype)
    if op == "read":
        tokens, picks = spread(1, 64), rng.choice([spread(1, 4096), 2048])
        kv = rng.choice([1, 2, 4])
        return _read(tokens, max(1, min(picks, 64 * 2048 * 2 // (tokens * kv))), kv, rng.choice([64, 96, 128, 128, 256]))
    kv, group = rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 7, 8, 16, 32, 64, 128])
    kv = min(kv, max(1, 128 // group))
    topk = rng.choice([2048, 2048, spread(1, 4096), spread(64, 4096)])
    dim = rng.choice([64, 128, 128])
    shared = rng.random() < 0.4
    most = min(1024 * 2048 // (topk * kv), 1024 * 128 * 2048 // (kv * group * topk), 1024)
    tokens = spread(1, max(1, most if shared else min(most, 64)))
    context = spread(max(topk, 64), 65536 if shared else max(topk + 1, 65536 // max(kv * tokens // 8, 1)))
    return _attend(tokens, kv * group, kv, topk, context, rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["fp8", "fp8", "same"]), dim,
                   shared)


# ---- inputs --------------------------------------------------------------------------------------
def _randn(gen, dev, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device=dev) * scale


def _angles(positions, rotary):
    """A table of cosines | sines for positions 0..n-1, worked out in 64 bits."""
    f = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=positions.device) / rotary)
    a = positions.double().unsqueeze(1) * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def _activations(gen, dev, tokens, heads, dim, dtype):
    """Projection outputs: every head has a magnitude of its own, and a few channels stand out."""
    x = _randn(gen, dev, tokens, heads, dim) * (0.5 + torch.rand(heads, 1, generator=gen, device=dev))
    x[..., ::37] *= 4.0
    return x.to(dtype)


def _fp8_rows(gen, dev, rows, heads, dim):
    """A cache of e4m3 rows and their scales, in pieces (a long cache is quickly made and needs no room beside it)."""
    codes = torch.empty(rows, heads, dim, dtype=FP8, device=dev)
    step = max(1, (1 << 27) // (heads * dim))
    for at in range(0, rows, step):
        n = min(step, rows - at)
        codes[at:at + n] = _randn(gen, dev, n, heads, dim, scale=120.0).clamp_(-FP8_MAX, FP8_MAX).to(FP8)
    return codes, (0.5 + torch.rand(rows, heads, generator=gen, device=dev)) / 120.0


def _same_rows(gen, dev, rows, heads, dim, dtype):
    x = torch.empty(rows, heads, dim, dtype=dtype, device=dev)
    step = max(1, (1 << 27) // (heads * dim))
    for at in range(0, rows, step):
        n = min(step, rows - at)
        x[at:at + n] = _randn(gen, dev, n, heads, dim).to(dtype)
    return x


def _picks(gen, dev, rows, topk, context):
    """What a selection hands out: distinct indices of a row's keys in no order; rows of fewer keys than topk hold theirs in
    order, then -1. Returns them and the rows' lengths."""
    lengths = torch.randint(max(1, context // 2), context + 1, (rows,), generator=gen, device=dev)
    lengths[rows // 2] = max(1, min(context, topk // 2 + 1))
    out = torch.empty(rows, topk, dtype=torch.int32, device=dev)
    step = max(1, (1 << 25) // context)
    for at in range(0, rows, step):
        n = min(step, rows - at)
        ln = lengths[at:at + n].unsqueeze(1)
        r = torch.rand(n, context, generator=gen, device=dev)
        r.masked_fill_(torch.arange(context, device=dev).unsqueeze(0) >= ln, -1.0)
        i = torch.topk(r, min(topk, context), dim=1, sorted=False).indices
        if topk > context:
            i = torch.nn.functional.pad(i, (0, topk - context))
        j = torch.arange(topk, device=dev).unsqueeze(0)
        out[at:at + n] = torch.where(ln <= topk, torch.where(j < ln, j, -1), i).to(torch.int32)
    return out


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    c = SimpleNamespace(**case)
    s = SimpleNamespace(case=c)
    T, D, op = c.tokens, c.dim, c.op
    if op in ("norm_rope", "step"):
        dtype = DTYPES[c.dtype]
        limit = 2 * T + 4096
        s.cos_sin = _angles(torch.arange(limit, device=dev), c.rotary)
        first = int(torch.randint(0, limit - T + 1, (1,), generator=gen, device=dev))
        s.positions = torch.arange(first, first + T, device=dev, dtype=torch.int32)
    if op == "norm_rope":
        n = c.q_heads + c.kv_heads
        qkv = _activations(gen, dev, T, n + c.kv_heads, D, dtype)
        s.q, s.k = qkv[:, :c.q_heads], qkv[:, c.q_heads:n]
        if not c.fused_qkv:
            s.q, s.k = s.q.contiguous(), s.k.contiguous()
        s.norm = None if c.norm == "none" else c.norm
        s.qw = s.kw = s.qb = s.kb = None
        if s.norm:
            s.qw, s.kw = ((1.0 + _randn(gen, dev, D, scale=0.2)).to(dtype) for _ in range(2))
        if s.norm == "layer":
            s.qb, s.kb = (_randn(gen, dev, D, scale=0.1).to(dtype) for _ in range(2))
    elif op == "step":
        s.q = _activations(gen, dev, T, c.q_heads, D, dtype)
        s.k = _activations(gen, dev, T, 1, D, dtype)[:, 0]
        s.w = torch.rand(T, c.q_heads, generator=gen, device=dev)
        s.kw, s.kb = 1.0 + _randn(gen, dev, D, scale=0.2), _randn(gen, dev, D, scale=0.1)
        s.cache, s.scale = _fp8_rows(gen, dev, limit, 1, D)
        s.cache, s.scale = s.cache[:, 0], s.scale[:, 0].contiguous()
        # (a token's cache row is its position; the batch's last token is padding where there are several)
        s.slots = s.positions.clone()
        if T > 1:
            s.slots[-1] = -1
    elif op == "write":
        dtype = DTYPES[c.dtype]
        n = 2 * T + 64
        s.k, s.v = (_activations(gen, dev, T, c.kv_heads, D, dtype) for _ in range(2))
        s.k_cache, s.k_scale = _fp8_rows(gen, dev, n, c.kv_heads, D)
        s.v_cache, s.v_scale = _fp8_rows(gen, dev, n, c.kv_heads, D)
        s.slots = torch.randperm(n, generator=gen, device=dev)[:T].to(torch.int32)
        if T > 1:
            s.slots[T // 2] = -1
    elif op == "read":
        context = c.topk + c.topk // 2 + 1
        s.cache, s.scale = _fp8_rows(gen, dev, T * context, c.kv_heads, D)
        s.slots = _picks(gen, dev, T, c.topk, context)
        s.offsets = torch.arange(T, device=dev, dtype=torch.int32) * context
    else:
        dtype = DTYPES[c.dtype]
        rows = c.context if c.shared else T * c.context
        s.q = _randn(gen, dev, T, c.q_heads, D, scale=2.0).to(dtype)
        s.k_scale = s.v_scale = None
        if c.cache == "fp8":
            s.k_cache, s.k_scale = _fp8_rows(gen, dev, rows, c.kv_heads, D)
            s.v_cache, s.v_scale = _fp8_rows(gen, dev, rows, c.kv_heads, D)
        else:
            s.k_cache = _same_rows(gen, dev, rows, c.kv_heads, D, dtype)
            s.v_cache = _same_rows(gen, dev, rows, c.kv_heads, D, dtype)
        s.indices = _picks(gen, dev, T, c.topk, c.context)
        s.offsets = None if c.shared else torch.arange(T, device=dev, dtype=torch.int32) * c.context
    return s


# ---- one pass ------------------------------------------------------------------------------------
@functools.cache
def _framework():
    at = os.path.join(os.getcwd(), "flash-float-jit-kernels_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from jit_kernel.kv_cache import cache_read, cache_write
    from jit_kernel.norm_rope import indexer_qk_write, qk_norm_rope
    from jit_kernel.sparse_attention import sparse_attention
    return SimpleNamespace(qk_norm_rope=qk_norm_rope, indexer_qk_write=indexer_qk_write, cache_write=cache_write,
                           cache_read=cache_read, sparse_attention=sparse_attention)


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    f, c = _framework(), s.case
    if c.op == "norm_rope":
        return f.qk_norm_rope(s.q, s.k, s.positions, s.cos_sin, q_norm=s.norm, k_norm=s.norm, q_weight=s.qw, k_weight=s.kw,
                              q_bias=s.qb, k_bias=s.kb, eps=EPS, interleaved=c.interleaved)
    if c.op == "step":
        q8, w = f.indexer_qk_write(s.q, s.k, s.w, s.positions, s.cos_sin, s.slots, s.cache, s.scale, k_norm="layer",
                                   k_weight=s.kw, k_bias=s.kb, eps=EPS, interleaved=c.interleaved)
        return q8, w, s.cache, s.scale
    if c.op == "write":
        f.cache_write(s.k, s.slots, s.k_cache, s.k_scale, s.v, s.v_cache, s.v_scale)
        return s.k_cache, s.k_scale, s.v_cache, s.v_scale
    if c.op == "read":
        return f.cache_read(s.cache, s.scale, s.slots, offsets=s.offsets)
    return f.sparse_attention(s.q, s.k_cache, s.v_cache, s.indices, k_scale=s.k_scale, v_scale=s.v_scale, offsets=s.offsets,
                              return_lse=True)


def _plain_norm(x, norm, weight, bias):
    x = x.float()
    if norm is None:
        return x
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    return x if bias is None else x + bias.float()


def _plain_rotate(x, positions, cos_sin, interleaved):
    """x [T, H, D], its first R of D channels rotated: pairs (i, i + R/2), or (2i, 2i + 1)."""
    R = cos_sin.size(1)
    cos, sin = cos_sin[positions.long()].unsqueeze(1).split(R // 2, -1)
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([y, x[..., R:]], -1)


def _plain_quantise(y):
    """Rows of y as e4m3 and a scale each: a row's largest finite magnitude becomes 448."""
    amax = torch.where(y.isfinite(), y.abs(), 0.0).amax(-1, keepdim=True).clamp_min(AMAX_FLOOR)
    return (y * (FP8_MAX / amax)).clamp(-FP8_MAX, FP8_MAX).to(FP8), (amax / FP8_MAX).squeeze(-1)


def _plain_put(codes, scale, slots, cache, cache_scale):
    """Rows of padding tokens (slot -1) go nowhere."""
    keep = slots >= 0
    cache.view(torch.uint8)[slots[keep].long()] = codes.view(torch.uint8)[keep]
    cache_scale[slots[keep].long()] = scale[keep]


def _plain_rows(cache, scale, at):
    """Rows `at` of a cache, in 32 bits; zeros where `at` is negative."""
    i = at.clamp_min(0).long()
    if scale is None:
        x = cache[i].float()
    else:
        x = cache.view(torch.uint8)[i].view(FP8).float() * scale[i].unsqueeze(-1)
    return x * (at >= 0).unsqueeze(-1).unsqueeze(-1)


def _plain(s):
    c = s.case
    if c.op == "norm_rope":
        return tuple(_plain_rotate(_plain_norm(x, s.norm, w, b), s.positions, s.cos_sin, c.interleaved).to(x.dtype)
                     for x, w, b in ((s.q, s.qw, s.qb), (s.k, s.kw, s.kb)))
    if c.op == "step":
        q8, q_scale = _plain_quantise(_plain_rotate(s.q.float(), s.positions, s.cos_sin, c.interleaved))
        k = _plain_norm(s.k, "layer", s.kw, s.kb).unsqueeze(1)
        k8, k_scale = _plain_quantise(_plain_rotate(k, s.positions, s.cos_sin, c.interleaved))
        _plain_put(k8[:, 0], k_scale[:, 0], s.slots, s.cache, s.scale)
        return q8, s.w * q_scale, s.cache, s.scale
    if c.op == "write":
        _plain_put(*_plain_quantise(s.k.float()), s.slots, s.k_cache, s.k_scale)
        _plain_put(*_plain_quantise(s.v.float()), s.slots, s.v_cache, s.v_scale)
        return s.k_cache, s.k_scale, s.v_cache, s.v_scale
    at = s.slots if c.op == "read" else s.indices
    at = at if s.offsets is None else torch.where(at >= 0, at + s.offsets.unsqueeze(1), -1)
    if c.op == "read":
        return _plain_rows(s.cache, s.scale, at).to(torch.bfloat16)
    T, H, G = c.tokens, c.kv_heads, c.q_heads // c.kv_heads
    k, v = _plain_rows(s.k_cache, s.k_scale, at), _plain_rows(s.v_cache, s.v_scale, at)  # [T, K, H, D]
    x = (s.q.float() * c.dim ** -0.5).view(T, H, G, c.dim) @ k.permute(0, 2, 3, 1)
    del k
    x.masked_fill_((at < 0).view(T, 1, 1, -1), -math.inf)
    m = x.amax(-1, keepdim=True).clamp_min(-3e38)
    x.sub_(m).exp_()
    z = x.sum(-1, keepdim=True)
    o = (x @ v.transpose(1, 2)) / torch.where(z > 0, z, 1.0)
    return o.reshape(T, c.q_heads, c.dim).to(s.q.dtype), (m + z.log()).view(T, c.q_heads)


# ---- the same from the definitions, in 64 bits -----------------------------------------------------
def _exact_head_rows(x, norm, weight, bias, s):
    x = x.double()
    D = x.size(-1)
    if norm is not None:
        mean = x.sum(-1, keepdim=True) / D if norm == "layer" else torch.zeros_like(x[..., :1])
        x = weight.double() * (x - mean) / (((x - mean) ** 2).sum(-1, keepdim=True) / D + EPS).sqrt()
        if bias is not None:
            x = x + bias.double()
    R = s.cos_sin.size(1)
    turn = torch.complex(*s.cos_sin.double()[s.positions.long()].view(-1, 1, 2, R // 2).unbind(2))
    i = torch.arange(R // 2, device=x.device)
    re, im = (2 * i, 2 * i + 1) if s.case.interleaved else (i, i + R // 2)
    z = torch.complex(x[..., re], x[..., im]) * turn
    out = x.clone()
    out[..., re], out[..., im] = z.real, z.imag
    return out


def _exact_fp8(y):
    """The nearest of e4m3's values to 448 y / (largest of the row), ties to even: spacing 2^-9 below 2^-6, three bits above."""
    amax = y.abs().amax(-1, keepdim=True).clamp_min(AMAX_FLOOR)
    x = y / amax * FP8_MAX
    spacing = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / spacing) * spacing, (amax / FP8_MAX).squeeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    c = s.case
    if c.op == "norm_rope":
        return tuple(_exact_head_rows(x, s.norm, w, b, s) for x, w, b in ((s.q, s.qw, s.qb), (s.k, s.kw, s.kb)))
    if c.op in ("step", "write"):
        if c.op == "step":
            q8, q_scale = _exact_fp8(_exact_head_rows(s.q, None, None, None, s))
            rows = [(_exact_head_rows(s.k.unsqueeze(1), "layer", s.kw, s.kb, s)[:, 0], s.cache, s.scale)]
            out = [q8, s.w.double() * q_scale]
        else:
            rows, out = [(s.k.double(), s.k_cache, s.k_scale), (s.v.double(), s.v_cache, s.v_scale)], []
        to = s.slots.tolist()
        src = [t for t, slot in enumerate(to) if slot >= 0]
        dst = [to[t] for t in src]
        for y, cache, scale in rows:
            y8, y_scale = _exact_fp8(y)
            cache, scale = cache.double(), scale.double()
            cache[dst], scale[dst] = y8[src], y_scale[src]
            out += [cache, scale]
        return tuple(out)
    if c.op == "read":
        out = torch.zeros(c.tokens, c.topk, c.kv_heads, c.dim, dtype=torch.float64, device=s.cache.device)
        for t in range(c.tokens):
            n = int((s.slots[t] >= 0).sum())
            at = s.slots[t, :n].long() + t * (s.cache.size(0) // c.tokens)
            out[t, :n] = s.cache.view(torch.uint8)[at].view(FP8).double() * s.scale[at].double().unsqueeze(-1)
        return out
    # attention: softmax over the selected keys, token by token
    G = c.q_heads // c.kv_heads
    o = torch.zeros(c.tokens, c.q_heads, c.dim, dtype=torch.float64, device=s.q.device)
    lse = torch.full((c.tokens, c.q_heads), -math.inf, dtype=torch.float64, device=s.q.device)
    for t in range(c.tokens):
        at = s.indices[t][s.indices[t] >= 0].long() + (0 if s.offsets is None else t * c.context)
        if c.cache == "fp8":
            k, v = (x.view(torch.uint8)[at].view(FP8).double() * y[at].double().unsqueeze(-1)
                    for x, y in ((s.k_cache, s.k_scale), (s.v_cache, s.v_scale)))
        else:
            k, v = s.k_cache[at].double(), s.v_cache[at].double()
        x = torch.einsum("hgd,nhd->hgn", s.q[t].double().view(c.kv_heads, G, c.dim), k) / math.sqrt(c.dim)
        lse[t] = torch.logsumexp(x, -1).view(-1)
        o[t] = torch.einsum("hgn,nhd->hgd", torch.softmax(x, -1), v).reshape(c.q_heads, c.dim)
    return o, lse


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    c = SimpleNamespace(**case)
    T, D, op = c.tokens, c.dim, c.op
    if op == "norm_rope":
        n = T * (c.q_heads + c.kv_heads) * D
        return {"bytes": 2 * n * (4 if c.dtype == "fp32" else 2) + T * (4 + 4 * c.rotary), "flops": 8 * n}
    if op == "step":
        width = 4 if c.dtype == "fp32" else 2
        return {"bytes": T * (c.q_heads + 1) * (D * (width + 1) + 4) + T * (4 * c.q_heads + 8 + 4 * c.rotary),
                "flops": 8 * T * (c.q_heads + 1) * D}
    if op == "write":
        n = 2 * T * c.kv_heads
        return {"bytes": n * (D * ((4 if c.dtype == "fp32" else 2) + 1) + 4) + 4 * T, "flops": 3 * n * D}
    if op == "read":
        n = T * c.topk * c.kv_heads
        return {"bytes": n * (3 * D + 4) + 4 * T * c.topk, "flops": n * D}
    # keys that a row of the selection names: all of them, but for the shortest
    keys = T * min(c.topk, c.context)
    row = 2 * (D + 4) if c.cache == "fp8" else 4 * D
    once = min(keys, c.context) if c.shared else keys
    return {"bytes": once * c.kv_heads * row + 4 * T * c.topk + 4 * T * c.q_heads * D + 4 * T * c.q_heads,
            "flops": 4 * keys * c.q_heads * D}
