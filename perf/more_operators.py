"""Steps of a serving layer that attends to its whole context: what performance is measured on beside the steps around the selector.

A case is one call, as a layer of a serving process makes it. `op` names the entry point:

  attend  paged_attention   attention of every sequence's newest token over its pages of a cache of keys and values; with `weight`
                            the weights each cached row has had so far are brought up to date in the same call
  evict   cache_evict       of every sequence and key head the rows with the largest accumulated weight (and the first and the
                            last ones) move to other pages, the rest is dropped
  rotate  qk_norm_rope      per-head norm and rotation of q and k by positions with several axes (time, height, width)

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
EPS = 1e-6


def _attend(batch, context, q_heads, kv_heads, page, dtype="bf16", cache="same", dim=128, weight=False):
    return {"op": "attend", "batch": batch, "context": context, "q_heads": q_heads, "kv_heads": kv_heads, "page": page,
            "dtype": dtype, "cache": cache, "dim": dim, "weight": weight}


def _evict(batch, context, budget, kv_heads, page, recent, sinks, dtype="bf16", cache="same", dim=128):
    return {"op": "evict", "batch": batch, "context": context, "budget": budget, "kv_heads": kv_heads, "page": page,
            "recent": recent, "sinks": sinks, "dtype": dtype, "cache": cache, "dim": dim}


def _rotate(tokens, q_heads, kv_heads, dim, rotary, axes, mixed, dtype="bf16", norm="rms", interleaved=False):
    return {"op": "rotate", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "axes": axes, "mixed": mixed, "dtype": dtype, "norm": norm, "interleaved": interleaved}


def listed():
    return [
        # the first steps of one request: launch latency
        dict(name="attend_b1_100", **_attend(1, 100, 64, 8, 16)),
        # one request with a long context: the cache's length has to be split over the whole device
        dict(name="attend_b1_128k", **_attend(1, 131072, 64, 8, 64)),
        # a decode batch of ragged lengths, 16-bit cache: the stream
        dict(name="attend_b64_8k", **_attend(64, 8192, 64, 8, 64)),
        # twice the context in an fp8 cache
        dict(name="attend_b64_16k_fp8", **_attend(64, 16384, 64, 8, 64, cache="fp8")),
        # an odd batch, small heads in groups of seven, fp16, pages of five rows
        dict(name="attend_b37_odd", **_attend(37, 2999, 21, 3, 5, dtype="fp16", dim=64)),
        # the decode batch with the weights of its rows added up: 16 bits, and one request in fp8
        dict(name="weigh_b64_8k", **_attend(64, 8192, 64, 8, 64, weight=True)),
        dict(name="weigh_b1_8k_fp8", **_attend(1, 8192, 64, 8, 16, cache="fp8", weight=True)),
        # one request's cache that has grown by a few hundred rows beyond its budget
        dict(name="evict_b1_4k", **_evict(1, 4608, 4096, 8, 64, 512, 4)),
        # a batch thinned to a quarter, fp8 cache
        dict(name="evict_b32_8k_fp8", **_evict(32, 8192, 2048, 8, 64, 256, 4, cache="fp8")),
        # odd sizes, pages of 24 rows, no protected rows, small heads
        dict(name="evict_b13_odd", **_evict(13, 20011, 1001, 3, 24, 0, 0, dtype="fp16", dim=64)),
        # one token of one request with three axes
        dict(name="rotate_t1", **_rotate(1, 64, 8, 128, 128, 3, False)),
        # a prefill chunk of text, images and video, the axes' channels mixed
        dict(name="rotate_t16k", **_rotate(16384, 64, 8, 128, 128, 3, True)),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attend", "attend", "attend", "evict", "evict", "rotate"])
    dim = rng.choice([64, 128, 128])
    dtype, cache = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["same", "fp8"])
    page = rng.choice([1, 5, 16, 16, 24, 32, 64, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 8])
    row = kv * dim * (2 if cache == "same" else 1)
    if op == "attend":
        batch = spread(1, 64)
        context = spread(1, min(131072, 64 * 8192 * 8 * 128 * 2 // (batch * row)))
        return _attend(batch, context, kv * rng.choice([1, 2, 4, 5, 7, 8, 8, 16]), kv, page, dtype, cache, dim, rng.random() < 0.4)
    if op == "evict":
        batch = spread(1, 32)
        context = spread(2, min(65536, 32 * 8192 * 8 * 128 // (batch * row)))
        budget = max(1, min(context, int(context * rng.uniform(0.1, 1.05))))
        sinks = rng.choice([0, 0, 4, budget // 16])
        sinks = min(sinks, budget)
        return _evict(batch, context, budget, kv, page, rng.choice([0, budget // 8, (budget - sinks) // 2, budget - sinks]) % (budget - sinks + 1),
                      sinks, dtype, cache, dim)
    dim, dtype = rng.choice([64, 80, 96, 128, 128, 256]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    q_heads = kv * rng.choice([1, 2, 5, 8])
    size = (q_heads + kv) * dim * (2 if dtype == "fp32" else 1)
    return _rotate(spread(1, min(16384, 16384 * 72 * 128 // size)), q_heads, kv, dim, rng.choice([16, 32, 48, 64, dim]), rng.choice([2, 3, 3, 4]),
                   rng.random() < 0.5, dtype, rng.choice(["rms", "rms", "layer", "none"]), rng.random() < 0.3)


# ---- inputs --------------------------------------------------------------------------------------
def _randn(gen, dev, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device=dev) * scale


def _rows(gen, dev, rows, heads, dim, dtype, fp8):
    """A cache of rows, made in pieces; e4m3 codes with their scales, or (rows of `dtype`, None)."""
    x = torch.empty(rows, heads, dim, dtype=FP8 if fp8 else dtype, device=dev)
    step = max(1, (1 << 27) // (heads * dim))
    for at in range(0, rows, step):
        n = min(step, rows - at)
        y = _randn(gen, dev, n, heads, dim, scale=120.0 if fp8 else 1.0)
        x[at:at + n] = y.clamp_(-FP8_MAX, FP8_MAX).to(FP8) if fp8 else y.to(dtype)
    return x, (0.5 + torch.rand(rows, heads, generator=gen, device=dev)) / 120.0 if fp8 else None


def _lengths(gen, dev, batch, context):
    """Of a ragged batch: half the context to all of it, one sequence of the full length; of larger ones one has just begun and
    one is a padding row."""
    n = torch.randint(max(1, context // 2), context + 1, (batch,), generator=gen, device=dev, dtype=torch.int32)
    n[0] = context
    if batch > 8:
        n[batch // 2], n[batch - 1] = 1, 0
    return n


def _axes(rotary, axes, mixed):
    """The axis each pair of channels turns by: in blocks of about the same size, or in turn."""
    pairs = rotary // 2
    return tuple(i % axes if mixed else i * axes // pairs for i in range(pairs))


def _grid(gen, dev, tokens, axes):
    """Positions of text, whose axes run together, with an image or a clip of a few frames (frame, row, column) in every other
    stretch of about 300 tokens."""
    at = torch.arange(tokens, device=dev)
    part, inside = at // 300, at % 300
    base = at - inside + int(torch.randint(0, 1000, (1,), generator=gen, device=dev))
    frame = [inside // 150, inside % 150 // 15, inside % 15, inside % 7]
    return torch.stack([torch.where(part % 2 == 1, base + frame[a], base + inside) for a in range(axes)]).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    c = SimpleNamespace(**case)
    s = SimpleNamespace(case=c)
    dtype, D = DTYPES[c.dtype], c.dim
    if c.op == "rotate":
        T, n = c.tokens, c.q_heads + c.kv_heads
        # (q and k are slices of the fused projection's output; every head has a magnitude of its own)
        qkv = (_randn(gen, dev, T, n + c.kv_heads, D) * (0.5 + torch.rand(n + c.kv_heads, 1, generator=gen, device=dev))).to(dtype)
        s.q, s.k = qkv[:, :c.q_heads], qkv[:, c.q_heads:n]
        s.positions = _grid(gen, dev, T, c.axes)
        s.axes = _axes(c.rotary, c.axes, c.mixed)
        f = 10000.0 ** (-torch.arange(0, c.rotary, 2, dtype=torch.float64, device=dev) / c.rotary)
        a = torch.arange(T + 1600, dtype=torch.float64, device=dev).unsqueeze(1) * f
        s.cos_sin = torch.cat([a.cos(), a.sin()], 1).float()
        s.norm = None if c.norm == "none" else c.norm
        s.qw = s.kw = s.qb = s.kb = None
        if s.norm:
            s.qw, s.kw = ((1.0 + _randn(gen, dev, D, scale=0.2)).to(dtype) for _ in range(2))
        if s.norm == "layer":
            s.qb, s.kb = (_randn(gen, dev, D, scale=0.1).to(dtype) for _ in range(2))
        return s
    B, H, P = c.batch, c.kv_heads, c.page
    per = -(-c.context // P)
    more = -(-c.budget // P) if c.op == "evict" else 0
    pages = B * (per + more) + 3
    s.k_cache, s.k_scale = _rows(gen, dev, pages * P, H, D, dtype, c.cache == "fp8")
    s.v_cache, s.v_scale = _rows(gen, dev, pages * P, H, D, dtype, c.cache == "fp8")
    # (pages lie in no order; a sequence has as many as it needs)
    s.lengths = _lengths(gen, dev, B, c.context)
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    s.page_table = order[:B * per].view(B, per).clone()
    s.page_table[torch.arange(per, device=dev) * P >= s.lengths.unsqueeze(1)] = -1
    if c.op == "attend":
        s.q = _randn(gen, dev, B, c.q_heads, D, scale=1.5).to(dtype)
        s.weight = s.weight_out = None
        if c.weight:
            s.weight = torch.rand(B, H, per * P, generator=gen, device=dev)
            s.weight_out = torch.zeros_like(s.weight)
        return s
    s.to_table = order[B * per:B * (per + more)].view(B, more).clone()
    # accumulated weights: few rows have had most of it, and some none at all
    s.weight = torch.exp(_randn(gen, dev, B, H, per * P, scale=2.0) - 6.0)
    s.weight.masked_fill_(torch.rand(B, H, per * P, generator=gen, device=dev) < 0.1, 0.0)
    return s


# ---- one pass ------------------------------------------------------------------------------------
@functools.cache
def _framework():
    at = os.path.join(os.getcwd(), "flash-float-jit-kernels_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from jit_kernel.kv_cache import cache_evict
    from jit_kernel.norm_rope import qk_norm_rope
    from jit_kernel.paged_attention import paged_attention
    return SimpleNamespace(paged_attention=paged_attention, cache_evict=cache_evict, qk_norm_rope=qk_norm_rope)


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    f, c = _framework(), s.case
    if c.op == "attend":
        out, lse = f.paged_attention(s.q, s.k_cache, s.v_cache, s.page_table, s.lengths, page_size=c.page, k_scale=s.k_scale,
                                     v_scale=s.v_scale, weight=s.weight, weight_out=s.weight_out, return_lse=True)
        return (out, lse) if s.weight is None else (out, lse, s.weight_out)
    if c.op == "evict":
        kept, lengths, weight = f.cache_evict(s.k_cache, s.v_cache, s.weight, s.page_table, s.lengths, s.to_table, page_size=c.page,
                                              budget=c.budget, recent=c.recent, sinks=c.sinks, k_scale=s.k_scale, v_scale=s.v_scale)
        return (kept, lengths, weight, s.k_cache, s.v_cache) + (() if s.k_scale is None else (s.k_scale, s.v_scale))
    return f.qk_norm_rope(s.q, s.k, s.positions, s.cos_sin, axes=s.axes, q_norm=s.norm, k_norm=s.norm, q_weight=s.qw, k_weight=s.kw,
                          q_bias=s.qb, k_bias=s.kb, eps=EPS, interleaved=c.interleaved)


def _bytes(x):
    return x.view(torch.uint8) if x.dtype is FP8 else x


def _plain_attend(s):
    c = s.case
    B, H, G, D, P = c.batch, c.kv_heads, c.q_heads // c.kv_heads, c.dim, c.page
    L = s.page_table.size(1) * P
    out, lse = torch.empty_like(s.q), torch.empty(B, c.q_heads, device=s.q.device)
    j = torch.arange(L, device=s.q.device)
    step = max(1, (1 << 28) // (L * H * D))
    for at in range(0, B, step):
        b = slice(at, min(B, at + step))
        n = b.stop - at
        slots = (s.page_table[b].long().clamp_min(0) * P).repeat_interleave(P, 1) + j % P
        there = j < s.lengths[b].unsqueeze(1)
        k, v = _bytes(s.k_cache)[slots].view(s.k_cache.dtype).float(), _bytes(s.v_cache)[slots].view(s.v_cache.dtype).float()
        if s.k_scale is not None:
            k, v = k.mul_(s.k_scale[slots].unsqueeze(-1)), v.mul_(s.v_scale[slots].unsqueeze(-1))
        x = (s.q[b].float() * D ** -0.5).view(n, H, G, D) @ k.permute(0, 2, 3, 1)
        del k
        x.masked_fill_(~there.view(n, 1, 1, L), -math.inf)
        m = x.amax(-1, keepdim=True).clamp_min(-3e38)
        x.sub_(m).exp_()
        z = x.sum(-1, keepdim=True)
        x.div_(torch.where(z > 0, z, 1.0))
        out[b] = (x @ v.transpose(1, 2)).reshape(n, c.q_heads, D).to(out.dtype)
        lse[b] = (m + z.log()).view(n, c.q_heads)
        if s.weight is not None:
            new = s.weight[b] + x.sum(2)
            s.weight_out[b] = torch.where(there.unsqueeze(1), new, s.weight_out[b])
    return (out, lse) if s.weight is None else (out, lse, s.weight_out)


def _plain_evict(s):
    c = s.case
    B, H, P, K = c.batch, c.kv_heads, c.page, c.budget
    L, dev = s.weight.size(2), s.weight.device
    j = torch.arange(L, device=dev)
    n = s.lengths.unsqueeze(1)
    rank = torch.where((j < c.sinks) | (j >= n - c.recent), math.inf, s.weight.transpose(0, 1))  # [H, B, L]
    rank = torch.where(j < n, rank, -math.inf).transpose(0, 1)
    # (stable: of equal weights the lower positions stay; a sequence of up to K rows keeps all of them)
    best = torch.sort(rank, dim=2, descending=True, stable=True).indices[..., :K]
    best = torch.nn.functional.pad(best, (0, K - best.size(2)), value=L)
    left = torch.minimum(s.lengths, torch.full_like(s.lengths, K))
    at = torch.arange(K, device=dev)
    best = torch.where(at < left.view(B, 1, 1), best, L).sort(2).values
    kept = torch.where(best < L, best, -1)
    weight = torch.zeros_like(s.weight)
    take = min(K, L)
    weight[..., :take] = torch.where(kept >= 0, s.weight.gather(2, kept.clamp_min(0)), 0.0)[..., :take]
    b, h, i = (kept >= 0).nonzero(as_tuple=True)
    pos = kept[b, h, i]
    src = s.page_table[b, pos // P].long() * P + pos % P
    dst = s.to_table[b, i // P].long() * P + i % P
    for x in (s.k_cache, s.v_cache, s.k_scale, s.v_scale):
        if x is not None:
            _bytes(x)[dst, h] = _bytes(x)[src, h]
    return (kept.to(torch.int32), left, weight, s.k_cache, s.v_cache) + (() if s.k_scale is None else (s.k_scale, s.v_scale))


def _plain_rotate(x, s, weight, bias):
    c, R, T = s.case, s.cos_sin.size(1), x.size(0)
    x = x.float()
    if s.norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    if s.norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        x = x if bias is None else x + bias.float()
    i = torch.arange(R // 2, device=x.device)
    at = s.positions[torch.tensor(s.axes, device=x.device)].long()  # [R / 2, T]
    cos, sin = (s.cos_sin[at, (i + o).unsqueeze(1)].t().unsqueeze(1) for o in (0, R // 2))
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if c.interleaved else (x[..., :R // 2], x[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([a, b], -1).flatten(-2) if c.interleaved else torch.cat([a, b], -1)
    return torch.cat([y, x[..., R:]], -1)


def _plain(s):
    if s.case.op == "attend":
        return _plain_attend(s)
    if s.case.op == "evict":
        return _plain_evict(s)
    return tuple(_plain_rotate(x, s, w, b).to(x.dtype) for x, w, b in ((s.q, s.qw, s.qb), (s.k, s.kw, s.kb)))


# ---- the same from the definitions, in 64 bits -----------------------------------------------------
def _slots(table, page, n):
    """Cache rows of positions 0..n-1, from a row of a page table."""
    return torch.tensor([e * page + r for e in table[:-(-n // page)] for r in range(page)][:n], dtype=torch.long)


def _wide(cache, scale, at):
    x = _bytes(cache)[at].view(cache.dtype).double()
    return x if scale is None else x * scale[at].double().unsqueeze(-1)


def _exact_attend(s):
    c, dev = s.case, s.q.device
    G = c.q_heads // c.kv_heads
    o = torch.zeros(c.batch, c.q_heads, c.dim, dtype=torch.float64, device=dev)
    lse = torch.full((c.batch, c.q_heads), -math.inf, dtype=torch.float64, device=dev)
    weight = None if s.weight is None else s.weight_out.double()
    lengths, table = s.lengths.tolist(), s.page_table.tolist()
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        at = _slots(table[b], c.page, n).to(dev)
        k, v = _wide(s.k_cache, s.k_scale, at), _wide(s.v_cache, s.v_scale, at)
        for h in range(c.kv_heads):
            x = s.q[b, h * G:(h + 1) * G].double() @ k[:, h].t() / math.sqrt(c.dim)
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(x, 1)
            p = torch.softmax(x, 1)
            o[b, h * G:(h + 1) * G] = p @ v[:, h]
            if weight is not None:
                weight[b, h, :n] = s.weight[b, h, :n].double() + p.sum(0)
    return (o, lse) if weight is None else (o, lse, weight)


def _exact_evict(s):
    c = s.case
    lengths, table, to = s.lengths.tolist(), s.page_table.tolist(), s.to_table.tolist()
    kept = torch.full((c.batch, c.kv_heads, c.budget), -1, dtype=torch.int32)
    weight = torch.zeros(s.weight.shape, dtype=torch.float64)
    w = s.weight.double().cpu()
    moves = [[], [], []]
    for b, n in enumerate(lengths):
        m = min(n, c.budget)
        if m == 0:
            continue
        src, dst = _slots(table[b], c.page, n), _slots(to[b], c.page, m)
        first, last = min(c.sinks, n), max(min(c.sinks, n), n - c.recent)
        for h in range(c.kv_heads):
            if n <= c.budget:
                stay = torch.arange(n)
            else:
                middle = w[b, h, first:last]
                # (two orders of the same positions: by position, then, without changing that, by weight)
                order = torch.argsort(-middle, stable=True)[:c.budget - first - (n - last)] + first
                stay = torch.cat([torch.arange(first), order, torch.arange(last, n)]).sort().values
            kept[b, h, :m] = stay.to(torch.int32)
            weight[b, h, :m] = w[b, h, stay]
            moves[0].append(src[stay])
            moves[1].append(dst)
            moves[2].append(torch.full((m,), h))
    out = []
    src, dst, head = (torch.cat(x).to(s.weight.device) if x else torch.zeros(0, dtype=torch.long, device=s.weight.device) for x in moves)
    for x in (s.k_cache, s.v_cache, s.k_scale, s.v_scale):
        if x is not None:
            y = x.clone()
            _bytes(y)[dst, head] = _bytes(x)[src, head]
            out.append(y)
    return (kept, torch.tensor([min(n, c.budget) for n in lengths], dtype=torch.int32), weight, *out)


def _exact_rotate(x, s, weight, bias):
    x, R = x.double(), s.cos_sin.size(1)
    if s.norm is not None:
        mean = x.sum(-1, keepdim=True) / x.size(-1) if s.norm == "layer" else torch.zeros_like(x[..., :1])
        x = weight.double() * (x - mean) / (((x - mean) ** 2).sum(-1, keepdim=True) / x.size(-1) + EPS).sqrt()
        if bias is not None:
            x = x + bias.double()
    out = x.clone()
    table = s.cos_sin.double()
    for i, axis in enumerate(s.axes):
        row = table[s.positions[axis].long()]
        turn = torch.complex(row[:, i], row[:, R // 2 + i]).unsqueeze(1)
        a, b = (2 * i, 2 * i + 1) if s.case.interleaved else (i, i + R // 2)
        z = torch.complex(x[..., a], x[..., b]) * turn
        out[..., a], out[..., b] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s.case.op == "attend":
        return _exact_attend(s)
    if s.case.op == "evict":
        return _exact_evict(s)
    return tuple(_exact_rotate(x, s, w, b) for x, w, b in ((s.q, s.qw, s.qb), (s.k, s.kw, s.kb)))


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    c = SimpleNamespace(**case)
    D = c.dim
    if c.op == "rotate":
        n = c.tokens * (c.q_heads + c.kv_heads) * D
        return {"bytes": 2 * n * (4 if c.dtype == "fp32" else 2) + c.tokens * (4 * c.axes + 4 * c.rotary), "flops": 8 * n}
    row = 2 * (D + 4) if c.cache == "fp8" else 4 * D
    # (a sequence has three quarters of the context on average, the first one all of it)
    half = max(1, c.context // 2)
    full = c.batch - (3 if c.batch > 8 else 1)
    if c.op == "attend":
        keys = c.context + full * (half + c.context) / 2 + (1 if c.batch > 8 else 0)
        return {"bytes": keys * c.kv_heads * (row + (8 if c.weight else 0)) + 4 * c.batch * c.q_heads * (D + 1), "flops": 4 * keys * c.q_heads * D}
    keys = c.context + full * (half + c.context) / 2 + (1 if c.batch > 8 else 0)
    # (of lengths between half the context and all of it)
    if c.budget <= half:
        left = c.budget
    else:
        span = max(1, c.context - half)
        left = ((c.budget - half) * (half + c.budget) / 2 + (c.context - c.budget) * c.budget) / span
    rows = c.kv_heads * (min(c.budget, c.context) + full * min(left, c.context) + (1 if c.batch > 8 else 0))
    return {"bytes": 4 * keys * c.kv_heads + rows * (2 * row + 12) + 8 * c.batch, "flops": keys * c.kv_heads}
