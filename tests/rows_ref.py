"""Plain 64-bit statements of the head-row, cache and attention ops, with the error each of their roundings may make."""
from __future__ import annotations

import math

import torch

FP8 = torch.float8_e4m3fn
U32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def angles(n, rotary, device="cpu", base=10000.0):
    f = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    a = torch.arange(n, dtype=torch.float64).unsqueeze(1) * f
    return torch.cat([a.cos(), a.sin()], 1).float().to(device)


def head_rows(x, norm=None, weight=None, bias=None, eps=1e-6, positions=None, cos_sin=None, interleaved=False):
    """x [T, H, D] -> (y in 64 bits, bound of the error of y computed in 32 bits).

    The bound: a sum of D terms by lanes and shuffles carries at most 13 roundings, its root half of that, rsqrt 2 ulp, the
    products around it 3 roundings, mean and difference 14 more of the largest |x| (layer); the rotation doubles what its two
    operands carry and adds 3. Under 64 half steps of S, the size of a row's largest product, doubled where rotated."""
    x = x.double()
    D = x.size(-1)
    size = x.abs().amax(-1, keepdim=True)
    if norm is not None:
        m = x.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(size)
        r = 1.0 / (((x - m) ** 2).mean(-1, keepdim=True) + eps).sqrt()
        w = torch.ones(D, dtype=torch.float64, device=x.device) if weight is None else weight.double()
        x = (x - m) * r * w
        size = size * r * w.abs().max()
        if bias is not None:
            x = x + bias.double()
            size = size + bias.double().abs().max()
    if cos_sin is not None:
        R = cos_sin.size(1)
        cs = cos_sin.double()[positions.long()].unsqueeze(1)
        c, s = cs[..., :R // 2], cs[..., R // 2:]
        y = x.clone()
        if interleaved:
            a, b = x[..., 0:R:2], x[..., 1:R:2]
            y[..., 0:R:2], y[..., 1:R:2] = a * c - b * s, b * c + a * s
        else:
            a, b = x[..., :R // 2], x[..., R // 2:R]
            y[..., :R // 2], y[..., R // 2:R] = a * c - b * s, b * c + a * s
        x, size = y, size * 2
    return x, (64 * U32 * size).expand_as(x)


def check_dense(got, ref, bound, what=""):
    y, e = ref, bound
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    lim = e + half_step(got.dtype) * (y.abs() + e) + tiny
    bad = (got.double() - y).abs() > lim
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst {((got.double() - y).abs() / lim).max():.2f} x"


def check_quantised(codes, scale, ref, bound, what=""):
    """codes [.., D] e4m3 and scale [..] of rows ref [.., D]: the scale is amax / 448 to the error of amax and two roundings, a
    code is off by half a step of e4m3 (2^-4 of its value, 2^-10 below 2^-6) and the error of what was rounded."""
    amax = ref.abs().amax(-1).clamp_min(2.0 ** -96)
    s = scale.double()
    assert bool(((s * 448 - amax).abs() <= bound.amax(-1) + 4 * U32 * amax).all()), f"{what}: scales"
    got = codes.double() * s.unsqueeze(-1)
    z = (ref.abs() + bound) / s.unsqueeze(-1)
    lim = s.unsqueeze(-1) * torch.maximum(z * 2.0 ** -4, torch.full_like(z, 2.0 ** -10)) * (1 + 8 * U32) + bound * 2
    bad = (got - ref).abs() > lim
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} codes of {bad.numel()} beyond half a step"


def quantise(y):
    """Codes and scales from the definition, for making caches: y [.., D]."""
    y = y.float()
    amax = torch.where(y.isfinite(), y.abs(), 0.0).amax(-1, keepdim=True).clamp_min(2.0 ** -96)
    return (y * (448.0 / amax)).clamp(-448, 448).to(FP8), (amax / 448.0).squeeze(-1)


def cache_values(cache, scale):
    return cache.double() if scale is None else cache.double() * scale.double().unsqueeze(-1)


def attention(q, k, v, indices, offsets=None, softmax_scale=None, k_scale=None, v_scale=None):
    """Token by token in 64 bits. Returns (out, lse, bound of out's error before its last rounding, bound of lse's)."""
    T, Hq, D = q.shape
    Hk = k.size(1)
    G = Hq // Hk
    scale = D ** -0.5 if softmax_scale is None else softmax_scale
    o = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    eo, el = torch.zeros_like(o), torch.zeros_like(lse)
    fp8 = k_scale is not None
    for t in range(T):
        at = indices[t].long()
        off = 0 if offsets is None else int(offsets[t])
        at = torch.where(at >= 0, at + off, -1)
        at = at[(at >= 0) & (at < k.size(0))]
        if at.numel() == 0:
            continue
        kk = cache_values(k[at], None if not fp8 else k_scale[at])
        vv = cache_values(v[at], None if not fp8 else v_scale[at])
        qq = q[t].double().view(Hk, G, D)
        s = torch.einsum("hgd,nhd->hgn", qq, kk) * scale
        lse[t] = torch.logsumexp(s, -1).view(-1)
        p = torch.softmax(s, -1)
        o[t] = torch.einsum("hgn,nhd->hgd", p, vv).reshape(Hq, D)
        # a score: D products summed in 32 bits (four half steps each leave room for how the tensor cores align their terms)
        # and two products behind it; fp8: queries in fp16 lose 2^-25 of the head's largest per element
        d = 4 * (D + 4) * U32 * torch.einsum("hgd,nhd->hgn", qq.abs(), kk.abs()) * abs(scale)
        if fp8:
            d = d + D * 2.0 ** -24 * qq.abs().amax(-1, keepdim=True) * kk.abs().amax() * abs(scale)
        d = d.amax(-1, keepdim=True) + 8 * U32 * s.abs().amax(-1, keepdim=True) + 2.0 ** -21
        wide = torch.einsum("hgn,nhd->hgd", p, vv.abs())
        n = at.numel()
        up = 2.0 ** -11 if fp8 else half_step(q.dtype)  # weights are rounded to fp16, or to q's type
        e = (up * (1 + 2.0 ** -10) + 2 * d + (n + 64) * U32) * wide
        least = torch.exp(-lse[t].view(Hk, G, 1) + s.amax(-1, keepdim=True))  # 1 / (sum of weights)
        if fp8:  # the smallest weights: 2^-25 of the largest scale, each times a code
            e = e + n * 2.0 ** -25 * v_scale[at].double().amax() * 448 * least
        elif q.dtype == torch.float16:  # fp16 weights below its smallest step
            e = e + n * 2.0 ** -25 * vv.abs().amax() * least
        eo[t] = e.reshape(Hq, D)
        el[t] = (d.squeeze(-1) + (n + 64) * U32).view(-1) + 4 * U32 * lse[t].abs()
    return o, lse, eo, el


def check_attention(got, got_lse, ref, what=""):
    o, lse, eo, el = ref
    check_dense(got, o, eo, what)
    if got_lse is not None:
        none = torch.isneginf(lse)
        assert torch.equal(torch.isneginf(got_lse), none), f"{what}: empty rows"
        off = (got_lse.double() - lse)[~none].abs()
        assert bool((off <= el[~none]).all()), f"{what}: lse off by {float((off / el[~none]).max()):.2f} x the bound"
