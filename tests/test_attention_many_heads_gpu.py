"""Attention of many heads to a key head over an e4m3 cache, with enough tokens that it goes to the kernel of 128 heads: scales of
either sign, heads of zeros, of tiny and of huge queries."""
import pytest
import torch

import rows_ref as ref
from jit_kernel.sparse_attention import sparse_attention
from test_sparse_attention_gpu import gen, make_cache, make_indices, rand, status  # noqa: F401

pytestmark = pytest.mark.gpu

MANY = [(12, 128, 1), (170, 100, 1), (40, 128, 2)]  # tokens, query heads, key heads; tests/test_attention_rule_cpu.py holds them to the rule


def case(g, T, Hq, Hk, D, dtype, n=500):
    q = rand(g, T, Hq, D, dtype=dtype, scale=2.0)
    k, ks = make_cache(g, n, Hk, D, dtype, True)
    v, vs = make_cache(g, n, Hk, D, dtype, True)
    return q, k, v, ks, vs, make_indices(g, T, 400, n)


@pytest.mark.parametrize("T,Hq,Hk", MANY)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_below_zero(dtype, D, T, Hq, Hk):
    g = gen(T)
    q, k, v, ks, vs, idx = case(g, T, Hq, Hk, D, dtype)
    sign = torch.where(torch.rand(500, Hk, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    for s, vv in ((sign, vs * sign), (sign, -vs), (-torch.ones_like(sign), vs)):
        out, lse = sparse_attention(q, k, v, idx, k_scale=ks * s, v_scale=vv, return_lse=True)
        _, l, eo, el = ref.attention(q, k, v, idx, None, None, ks * s, vv.abs())  # (its bounds want magnitudes)
        ref.check_attention(out, lse, (ref.attention(q, k, v, idx, None, None, ks * s, vv)[0], l, eo, el))


@pytest.mark.parametrize("T,Hq,Hk", MANY)
@pytest.mark.parametrize("D", [64, 128])
def test_queries_of_all_sizes(D, T, Hq, Hk):
    g = gen(T + 1)
    q, k, v, ks, vs, idx = case(g, T, Hq, Hk, D, torch.bfloat16)
    q[:, 0] *= 1e-30
    q[:, 1] *= 1e-3
    q[:, 33] = 0
    q[::2, Hq - 1] = 0
    q[1::2, Hq - 1] *= 1e-37
    for by in (1.0, 1e30):
        out, lse = sparse_attention(q * by, k, v, idx, k_scale=ks / by, v_scale=vs, return_lse=True)
        ref.check_attention(out, lse, ref.attention(q * by, k, v, idx, None, None, ks / by, vs))
