"""Lists that go on for millions of entries behind the last that names a row: a batch over one shared list, and a token of its own."""
import pytest
import torch

import rows_ref as ref
from jit_kernel.sparse_attention import sparse_attention
from test_sparse_attention_gpu import gen, make_cache, rand, status  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,Hq", [(160, 100), (12, 128), (3, 8)])
@pytest.mark.parametrize("K,at", [(3_000_001, (5, 1_000_000, 1_999_999)), (1 << 20, (0, 700)), ((1 << 20) + 1, (0,)), (1_100_000, (60_000, 52_000))])
def test_long_tails(K, at, T, Hq):
    g = gen(T + K)
    q = rand(g, T, Hq, 64, dtype=torch.bfloat16)
    (k, ks), (v, vs) = (make_cache(g, 500, 1, 64, torch.bfloat16, True) for _ in range(2))
    idx = torch.full((1, K), -1, device="cuda", dtype=torch.int32)
    rows = torch.randperm(500, generator=g, device="cuda")[:len(at)].to(torch.int32)
    idx[0, list(at)] = rows
    out, lse = sparse_attention(q, k, v, idx.expand(T, K), k_scale=ks, v_scale=vs, return_lse=True)
    short = rows.view(1, -1).expand(T, len(at))  # (the order of a list says nothing)
    ref.check_attention(out, lse, ref.attention(q, k, v, short, None, None, ks, vs))
