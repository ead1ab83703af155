"""Attention over selected rows where lists, scales and heads are unlike the ordinary: long lists, lists that begin with nothing,
many heads to a key head, scales of either sign, an empty cache, an output over the queries."""
import pytest
import torch

import rows_ref as ref
from jit_kernel.kv_cache import cache_read, cache_write
from jit_kernel.sparse_attention import sparse_attention
from test_sparse_attention_gpu import FP8, gen, make_cache, make_indices, rand, status  # noqa: F401

pytestmark = pytest.mark.gpu


def case(g, T, Hq, Hk, K, rows, fp8, D=128, dtype=torch.bfloat16):
    q = rand(g, T, Hq, D, dtype=dtype, scale=2.0)
    k, ks = make_cache(g, rows, Hk, D, dtype, fp8)
    v, vs = make_cache(g, rows, Hk, D, dtype, fp8)
    return q, k, v, ks, vs


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T,Hq,K", [(1, 8, 20000), (1, 64, 20000), (150, 8, 3001), (150, 24, 3001), (40, 128, 2500)])
def test_long_lists(T, Hq, K, fp8):
    g = gen(K + Hq)
    q, k, v, ks, vs = case(g, T, Hq, 1, K, 4000, fp8)
    idx = make_indices(g, T, K, 4000)
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, k, v, idx, None, None, ks, vs))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq", [8, 100])
@pytest.mark.parametrize("T", [2, 160])
def test_lists_that_begin_with_nothing(T, Hq, fp8):
    """Whole tiles without a row in front of, between and behind those that have some."""
    g = gen(21)
    q, k, v, ks, vs = case(g, T, Hq, 1, 1500, 900, fp8)
    idx = make_indices(g, T, 1500, 900, empty=False)
    idx[:, :700] = -1
    idx[0, 800:1300] = -1
    idx[T // 2, 1400:] = -1
    idx[T // 2, 703:1390] = -1
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, k, v, idx, None, None, ks, vs))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hk", [(17, 1), (300, 1), (128, 2), (129, 1), (258, 2), (16, 1), (32, 2)])
def test_heads(Hq, Hk, fp8):
    g = gen(Hq)
    q, k, v, ks, vs = case(g, 3, Hq, Hk, 300, 500, fp8)
    idx = make_indices(g, 3, 300, 500)
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, k, v, idx, None, None, ks, vs))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq", [8, 100])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-6, 3.0])
def test_softmax_scales(scale, Hq, fp8):
    g = gen(22)
    q, k, v, ks, vs = case(g, 3, Hq, 1, 400, 500, fp8)
    q[0, 1] = 0
    idx = make_indices(g, 3, 400, 500)
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, softmax_scale=scale, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, k, v, idx, None, scale, ks, vs))


@pytest.mark.parametrize("Hq", [8, 100])
def test_scales_below_zero(Hq):
    g = gen(23)
    q, k, v, ks, vs = case(g, 3, Hq, 1, 400, 500, True)
    sign = torch.where(torch.rand(500, 1, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    idx = make_indices(g, 3, 400, 500)
    for vv in (vs * sign, -vs):
        out, lse = sparse_attention(q, k, v, idx, k_scale=ks * sign, v_scale=vv, return_lse=True)
        want = ref.attention(q, k, v, idx, None, None, ks * sign, vv.abs())  # (its bounds want magnitudes)
        o, l, eo, el = want
        o = ref.attention(q, k, v, idx, None, None, ks * sign, vv)[0]
        ref.check_attention(out, lse, (o, l, eo, el))


@pytest.mark.parametrize("Hq", [8, 100])
def test_nothing_to_attend_to(Hq):
    q = torch.ones(3, Hq, 64, device="cuda", dtype=torch.bfloat16)
    for c, s in ((torch.empty(0, 1, 64, device="cuda", dtype=torch.bfloat16), None),
                 (torch.empty(0, 1, 64, device="cuda", dtype=torch.uint8).view(FP8), torch.empty(0, 1, device="cuda"))):
        for K in (0, 5, 300):
            idx = torch.full((3, K), -1, device="cuda", dtype=torch.int32)
            out, lse = sparse_attention(q, c, c, idx, k_scale=s, v_scale=s, return_lse=True)
            assert bool((out == 0).all()) and bool(lse.isneginf().all())
    assert bool((cache_read(c, s, torch.full((4,), -1, device="cuda", dtype=torch.int32)) == 0).all())
    cache_write(q[:, :1], torch.full((3,), -1, device="cuda", dtype=torch.int32), c, s)


@pytest.mark.parametrize("T", [2, 300])
@pytest.mark.parametrize("Hq", [8, 100])
def test_output_over_the_queries(Hq, T):
    g = gen(24)
    q, k, v, ks, vs = case(g, T, Hq, 1, 500, 900, True)
    idx = make_indices(g, T, 500, 900)
    want = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs)
    got = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq", [8, 100])
def test_two_at_once(Hq, fp8):
    """Calls of different sizes on two streams that overlap give what each gives alone."""
    g = gen(25)
    cases = []
    for T, K in ((3, 2048), (170, 700)):
        q, k, v, ks, vs = case(g, T, Hq, 1, K, 3000, fp8)
        idx = make_indices(g, T, K, 3000)
        cases.append(lambda q=q, k=k, v=v, ks=ks, vs=vs, idx=idx: sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs))
    want = [c() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for s, c, o in zip(streams, cases, got):
            with torch.cuda.stream(s):
                o.append(c())
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(torch.equal(w, x) for x in o)
