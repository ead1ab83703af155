"""Plain 64-bit statements of attention over a paged cache and of eviction, on top of rows_ref."""
from __future__ import annotations

import torch

import rows_ref as ref


def slots_of(page_table, lengths, page, device):
    """int32 [B, longest]: the cache rows of every sequence's positions, -1 behind its length and on negative pages."""
    B, cols = page_table.shape
    n = lengths.clamp(0, cols * page).to(device)
    longest = max(1, int(n.max()) if B else 1)
    j = torch.arange(longest, device=device)
    if cols == 0:
        return torch.full((B, longest), -1, dtype=torch.int32, device=device)
    entry = page_table.long()[:, (j // page).clamp_max(cols - 1)]
    at = torch.where(entry >= 0, entry * page + j % page, -1)
    return torch.where(j < n.unsqueeze(1), at, -1).to(torch.int32)


def attention(q, k, v, page_table, lengths, page, softmax_scale=None, k_scale=None, v_scale=None):
    """rows_ref.attention over the sequences' rows: (out, lse, their bounds), and the rows."""
    at = slots_of(page_table, lengths, page, q.device)
    return ref.attention(q, k, v, at, None, softmax_scale, k_scale, v_scale), at


def weights(q, k, at, refs, softmax_scale=None, k_scale=None):
    """(sum of weights [B, Hk, longest], its bound): a weight is exp(score - lse), so what its score and the lse are off by (each by
    no more than lse's bound) it is off by, relative, and 2^-20 for exp2 and the factors; a group's sum adds a rounding per head."""
    (_, lse, _, el), B, Hq, Hk = refs, q.size(0), q.size(1), k.size(1)
    G = Hq // Hk
    scale = q.size(2) ** -0.5 if softmax_scale is None else softmax_scale
    w = torch.zeros(B, Hk, at.size(1), dtype=torch.float64, device=q.device)
    e = torch.zeros_like(w)
    for b in range(B):
        there = (at[b] >= 0) & (at[b] < k.size(0))
        rows = at[b][there].long()
        if rows.numel() == 0:
            continue
        kk = ref.cache_values(k[rows], None if k_scale is None else k_scale[rows])
        s = torch.einsum("hgd,nhd->hgn", q[b].double().view(Hk, G, -1), kk) * scale
        p = torch.exp(s - lse[b].view(Hk, G, 1))
        w[b][:, there] = p.sum(1)
        e[b][:, there] = (p * (2 * el[b].view(Hk, G, 1) + 2.0 ** -20)).sum(1) * 1.01 + (G + 2) * ref.U32 * p.sum(1) + 1e-37
    return w, e


def check_weights(got, before, lengths, w, e, what=""):
    """got [B, Hk, N] against before + w up to every sequence's length; behind it `got` has to be what it was (NaN here)."""
    N = w.size(2)
    j = torch.arange(got.size(2), device=got.device)
    inside = (j < lengths.to(got.device).clamp_min(0).unsqueeze(1)).unsqueeze(1).expand_as(got)
    assert bool(got[~inside].isnan().all()), f"{what}: written behind a length"
    n = min(N, got.size(2))
    want = w[..., :n] + (0.0 if before is None else before[..., :n].double())
    lim = e[..., :n] + 2 * ref.U32 * want.abs()
    off = torch.where(inside[..., :n], (got[..., :n].double() - want).abs(), 0.0)
    assert bool((off <= lim).all()), f"{what}: worst {float((off / lim).max()):.2f} x the bound"


def evict(weight, lengths, budget, recent, sinks):
    """(kept, lengths, weights) from the definition, sequence by sequence and head by head, on the CPU: weights are compared as they
    are (-0 equals 0, NaN above infinity), of equal ones the lower position stays."""
    weight = weight.cpu()
    B, H, N = weight.shape
    kept = torch.full((B, H, budget), -1, dtype=torch.int32)
    out = torch.zeros_like(weight)
    left = []
    for b, n in enumerate(lengths.tolist()):
        n = min(max(n, 0), N)
        left.append(min(n, budget))
        for h in range(H):
            stay = list(range(n))
            if n > budget:
                row = weight[b, h].tolist()
                order = sorted(range(sinks, n - recent), key=lambda j: (row[j] == row[j], -row[j] if row[j] == row[j] else 0.0, j))
                stay = sorted(list(range(sinks)) + list(range(n - recent, n)) + order[:budget - sinks - recent])
            kept[b, h, :len(stay)] = torch.tensor(stay, dtype=torch.int32)
            out[b, h, :len(stay)] = weight[b, h][stay]
    return kept, torch.tensor(left, dtype=torch.int32), out


def move(cache, kept, page_table, to_table, page):
    """What the rows of `cache` [slots, H, ..] (or a scale) hold afterwards."""
    out = cache.clone()
    src, dst = (x.view(torch.uint8) if x.dtype.itemsize == 1 else x for x in (cache, out))
    B, H, _ = kept.shape
    slots = cache.size(0)
    for b in range(B):
        for h in range(H):
            pos = kept[b, h][kept[b, h] >= 0].long().to(cache.device)
            i = torch.arange(pos.numel(), device=cache.device)
            p, t = page_table[b].long()[pos // page], to_table[b].long()[i // page]
            a, z = p * page + pos % page, t * page + i % page
            ok = (p >= 0) & (t >= 0) & (a < slots) & (z < slots)
            dst[z[ok], h] = src[a[ok], h]
    return out
