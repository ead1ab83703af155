"""Attention over selected rows where lists, scales and heads are unlike the ordinary: long lists, lists that begin with nothing,
many heads to a key head, scales of either sign, an empty cache, an output over the queries."""
import pytest
import torch

import rows_ref as ref
from jit_kernel import _native
from jit_kernel.kv_cache import cache_read, cache_write
from jit_kernel.sparse_attention import sparse_attention
from test_sparse_attention_gpu import FP8, gen, make_cache, make_indices, rand, status, take_status  # noqa: F401

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
            if K:
                many = torch.ones(60, Hq, 64, device="cuda", dtype=torch.bfloat16)
                for x in (q, many):
                    out, lse = sparse_attention(x, c, c, idx[:1].abs().expand(x.size(0), K), k_scale=s, v_scale=s, return_lse=True)
                    assert take_status() == _native.ST_BAD_INDEX
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


# Enough tokens for the kernel of many heads: below that the call goes another way (a token's keys are split over 8, 4, 2 CTAs or
# one; CTAs that take one token after the other).
MANY = [(12, 128, 1), (24, 100, 1), (50, 64, 1), (100, 33, 1), (40, 128, 2), (310, 128, 1), (60, 300, 1), (200, 64, 2)]


@pytest.mark.parametrize("T,Hq,Hk", MANY)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_tokens(dtype, fp8, D, T, Hq, Hk):
    g = gen(T + D)
    K, rows = {12: 2048, 310: 515, 200: 129}.get(T, 700), 1100
    layout = "wide" if T % 3 else "dense"
    q = rand(g, T, Hq + 1, D, dtype=dtype, scale=2.0)[:, 1:]
    k, ks = make_cache(g, rows, Hk, D, dtype, fp8, layout)
    v, vs = make_cache(g, rows, Hk, D, dtype, fp8, layout)
    idx = make_indices(g, T, K, rows - 100)
    idx[2, : K // 2] = -1
    idx[T // 2] = -1
    idx[T // 3, 1:] = -1
    off = torch.randint(0, 100, (T,), generator=g, device="cuda", dtype=torch.int32)
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, offsets=off, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, k, v, idx, off, None, ks, vs))
    again = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, offsets=off)
    assert torch.equal(again, out)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T", [12, 170])
def test_many_tokens_with_anything(T, fp8):
    """Far scores, negative and zero softmax scales, NaN rows, indices beyond the cache, an output with gaps."""
    g = gen(31)
    q, k, v, ks, vs = case(g, T, 128, 1, 600, 900, fp8)
    idx = make_indices(g, T, 600, 800)
    for scale in (5.0, -0.3, 0.0):
        out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, softmax_scale=scale, return_lse=True)
        ref.check_attention(out, lse, ref.attention(q, k, v, idx, None, scale, ks, vs))
    if fp8:
        wild = vs * 10.0 ** torch.linspace(-6, 6, 900, device="cuda").unsqueeze(1)
        up = idx.sort(dim=1).values
        for i in (up, up.flip(1)):
            out, lse = sparse_attention(q, k, v, i, k_scale=ks, v_scale=wild, return_lse=True)
            ref.check_attention(out, lse, ref.attention(q, k, v, i, None, None, ks, wild))
    beyond = idx.clone()
    beyond[::2, 5] = 900
    beyond[1::3, 300] = 2147483647
    wide = torch.full((T, 129, 130), 7.0, device="cuda", dtype=torch.bfloat16)
    out, lse = sparse_attention(q, k, v, beyond, k_scale=ks, v_scale=vs, out=wide[:, :128, 1:129], return_lse=True)
    assert take_status() == _native.ST_BAD_INDEX
    ref.check_attention(out, lse, ref.attention(q, k, v, beyond, None, None, ks, vs))
    assert bool((wide[:, 128] == 7).all()) and bool((wide[..., 0] == 7).all()) and bool((wide[..., 129] == 7).all())
    for c in (k, v):
        if fp8:
            c.view(torch.uint8)[850, 0, 3] = 0x7f
        else:
            c[850, 0, 3] = float("nan")
    asks = idx.clone()
    asks[1] = -1
    asks[1, 7] = 850
    asks[4, 599] = 850
    out, lse = sparse_attention(q, k, v, asks, k_scale=ks, v_scale=vs, return_lse=True)
    hit = torch.tensor([1, 4], device="cuda")
    assert bool(out[hit].isnan().all()) and bool(lse[hit].isnan().all())
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[hit] = False
    ref.check_attention(out[rest], lse[rest], ref.attention(q[rest], k, v, asks[rest], None, None, ks, vs))


@pytest.mark.parametrize("fp8", [False, True])
def test_many_tokens_in_a_graph(fp8):
    g = gen(32)
    q, k, v, ks, vs = case(g, 20, 128, 1, 700, 900, fp8)
    idx = make_indices(g, 20, 700, 900)
    call = lambda: sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, return_lse=True)  # noqa: E731
    call()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = call()
    q.copy_(rand(g, 20, 128, 128, dtype=torch.bfloat16))
    idx.copy_(make_indices(g, 20, 700, 900))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.replay()
        graph.replay()
    eager = call()
    torch.cuda.synchronize()
    assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])


def test_many_tokens_on_a_long_cache():
    """Rows beyond 2^31 elements and 2^32 bytes, and scales beyond neither."""
    rows = (1 << 31) // 128 + 5000
    cache = torch.zeros(rows, 1, 128, device="cuda", dtype=torch.bfloat16)
    g = gen(33)
    idx = torch.randint(rows - 4000, rows, (12, 300), generator=g, device="cuda", dtype=torch.int32)
    idx[1, ::2] = torch.randint(0, 4000, (150,), generator=g, device="cuda", dtype=torch.int32)
    cache[-4000:] = rand(g, 4000, 1, 128, dtype=torch.bfloat16)
    cache[:4000] = rand(g, 4000, 1, 128, dtype=torch.bfloat16)
    q = rand(g, 12, 128, 128, dtype=torch.bfloat16)
    out, lse = sparse_attention(q, cache, cache, idx, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, cache, cache, idx))
