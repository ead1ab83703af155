"""Attention over an e4m3 cache whose rows' scales differ: what a row adds to a result is its weight times its scale, so a row of a
large scale and hardly any weight takes nothing from the others, and rows of tiny scales and most of the weight lose nothing."""
import math

import pytest
import torch

import rows_ref as ref
from jit_kernel.sparse_attention import sparse_attention
from test_sparse_attention_gpu import FP8, gen, rand, status  # noqa: F401

pytestmark = pytest.mark.gpu

FEW = [(3, 8, 1), (5, 32, 2), (1, 20, 1)]  # tokens, query heads, key heads: the kernel of 16 heads
N = 200


def statement(q, k, v, indices, k_scale, v_scale):
    """(out, lse, bound of out's error before its last rounding, bound of lse's), token by token in 64 bits.

    A weight p_j |v scale_j| is rounded to fp16: 2^-11 of it, and at least 2^-25 of the unit it is held in. The unit is no more than
    2^4 times the largest p_j |v scale_j| that the head meets, so a row is off by 2^-21 of that one times a code (448 at most); weights
    that vanish in 32 bits, below 2^-126 of the reference times a scale of up to 2^100, by less than that again. Scores are held
    against a reference that lies up to 100 away from them (log2)."""
    T, Hq, D = q.shape
    Hk = k.size(1)
    G = Hq // Hk
    scale = D ** -0.5
    o = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    eo, el = torch.zeros_like(o), torch.zeros_like(lse)
    for t in range(T):
        at = indices[t].long()
        at = at[at >= 0]
        n = at.numel()
        if n == 0:
            continue
        kk, vv = ref.cache_values(k[at], k_scale[at]), ref.cache_values(v[at], v_scale[at])
        qq = q[t].double().view(Hk, G, D)
        s = torch.einsum("hgd,nhd->hgn", qq, kk) * scale
        p = torch.softmax(s, -1)
        lse[t] = torch.logsumexp(s, -1).view(-1)
        o[t] = torch.einsum("hgn,nhd->hgd", p, vv).reshape(Hq, D)
        # scores: as in rows_ref.attention, and what is left of the reference's distance
        d = 4 * (D + 4) * ref.U32 * torch.einsum("hgd,nhd->hgn", qq.abs(), kk.abs()) * scale
        d = d + D * 2.0 ** -24 * qq.abs().amax(-1, keepdim=True) * kk.abs().amax() * scale
        d = d.amax(-1, keepdim=True) + 8 * ref.U32 * (s.abs().amax(-1, keepdim=True) + 100) + 2.0 ** -21
        wide = torch.einsum("hgn,nhd->hgd", p, vv.abs())
        largest = (p * v_scale[at].double().abs().t().unsqueeze(1)).amax(-1, keepdim=True)
        e = (2.0 ** -11 * (1 + 2.0 ** -10) + 2 * d + (n + 64) * ref.U32) * wide + n * 2.0 ** -20 * 448 * largest
        eo[t] = e.reshape(Hq, D)
        el[t] = (d.squeeze(-1) + (n + 64) * ref.U32).view(-1) + 4 * ref.U32 * (lse[t].abs() + 100)
    return o, lse, eo, el


def inputs(g, T, Hq, Hk, D, dtype, scores, exponents):
    """Queries that all look one way and keys along it, so that row j scores about scores[j]; v scales near 2^exponents[j]."""
    n = scores.numel()
    way = torch.where(torch.rand(D, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    q = (D ** -0.5 * (way + 0.05 * rand(g, T, Hq, D))).to(dtype)
    k, ks = ref.quantise(scores.view(n, 1, 1) * way + 0.3 * rand(g, n, Hk, D))
    v, vs = ref.quantise(rand(g, n, Hk, D))
    return q, k, v, ks, vs * torch.exp2(exponents).view(n, 1)


def orders(g, T, n):
    """The rows rising, falling and mixed, with none of them here and there and an empty list."""
    idx = torch.stack([torch.randperm(n, generator=g, device="cuda") for _ in range(T)]).to(torch.int32)
    up = torch.arange(n, device="cuda", dtype=torch.int32)
    idx[0] = up
    if T > 1:
        idx[1] = up.flip(0)
    if T > 2:
        idx[2, ::3] = -1
    if T > 4:
        idx[T - 1] = -1
        idx[T // 2, 1:] = -1
    return idx


def check(q, k, v, ks, vs, idx):
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, return_lse=True)
    o, l, eo, el = statement(q, k, v, idx, ks, vs)
    # what lies beyond the output's type (65,504 of fp16) is an infinity there; beside the border either is right
    most = torch.finfo(out.dtype).max
    beyond, beside = o.abs() - eo > 1.001 * most, (o.abs() + eo > 0.999 * most)
    assert torch.equal(out[beyond].double(), o[beyond].sign() * math.inf)
    ref.check_attention(torch.where(beside, 0, out), lse, (torch.where(beside, 0, o), l, eo, el))


def one_row_without_weight(g, T, Hq, Hk, D, dtype):
    """One row's v scale is 2^30 times the others', its score 40 below theirs (2^-57): it adds 2^-27 of what they do."""
    for where in (0, 1, 50, 131, N - 1):
        scores, exponents = rand(g, N, scale=0.5), torch.zeros(N, device="cuda")
        scores[where], exponents[where] = -40.0, 30.0
        check(*inputs(g, T, Hq, Hk, D, dtype, scores, exponents), orders(g, T, N))


def scales_against_scores(g, T, Hq, Hk, D, dtype):
    """v scales over 2^+-20 where a row's weight falls, or rises, with its scale; and where neither knows of the other."""
    exponents = torch.linspace(-20, 20, N, device="cuda")
    for power in (-1.5, -1.0, -0.5, 0.0, 0.5):
        scores = power * math.log(2.0) * exponents
        check(*inputs(g, T, Hq, Hk, D, dtype, scores, exponents), orders(g, T, N))
    check(*inputs(g, T, Hq, Hk, D, dtype, rand(g, N), rand(g, N, scale=15.0).clamp(-50, 50)), orders(g, T, N))


def rows_of_zeros(g, T, Hq, Hk, D, dtype):
    """Rows of zeros as the cache holds them (scale 2^-96 / 448), and scales of zero, with little and with most of the weight."""
    for score in (-20.0, 0.0, 20.0):
        scores = rand(g, N)
        scores[::3] = score
        q, k, v, ks, vs = inputs(g, T, Hq, Hk, D, dtype, scores, torch.zeros(N, device="cuda"))
        v.view(torch.uint8)[::3] = 0
        vs[::3] = 2.0 ** -96 / 448
        vs[::6] = 0.0
        idx = orders(g, T, N)
        idx[0, 1:] = -1  # (nothing but such a row)
        check(q, k, v, ks, vs, idx)


CASES = [one_row_without_weight, scales_against_scores, rows_of_zeros]


@pytest.mark.parametrize("T,Hq,Hk", FEW)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES)
def test_scales_few_tokens(case, dtype, D, T, Hq, Hk):
    case(gen(T * Hq + D), T, Hq, Hk, D, dtype)


MANY = [(12, 128, 1), (170, 100, 1), (40, 128, 2)]  # enough tokens for the kernel of 128 heads: keys split over CTAs, and not


@pytest.mark.parametrize("T,Hq,Hk", MANY)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES)
def test_scales_many_heads(case, dtype, D, T, Hq, Hk):
    case(gen(T * Hq + D), T, Hq, Hk, D, dtype)
