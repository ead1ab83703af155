"""Inputs and results of the paged cache's ops side by side in one buffer, row by row: the same bits as apart. On one another: refused."""
import pytest
import torch

import paged_ref as paged
from jit_kernel.kv_cache import cache_evict
from jit_kernel.paged_attention import paged_attention
from jit_kernel.topk_indexer import _status_word, kernel_status
from test_cache_evict_gpu import bits, make, weights
from test_paged_attention_gpu import gen, make_cache, make_pages, rand

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def status():
    if torch.cuda.is_available():
        _status_word(torch.device("cuda", 0)).zero_()
    yield
    if torch.cuda.is_available():
        assert kernel_status() == 0


def pair(x, y, dim):
    """x and y in one buffer, in turn along `dim`: (x, y, buffer)"""
    buffer = torch.stack([bits(x), bits(y)], dim)
    return buffer.select(dim, 0).view(x.dtype), buffer.select(dim, 1).view(y.dtype), buffer


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [0, 1, 2])
@pytest.mark.parametrize("extra", [0, 3000])
def test_attention(fp8, dim, extra):
    g = gen(dim)
    B, Hq, Hk, D, page, lens = 3, 16, 2, 128, 16, [300, 0, 77]
    table, pages = make_pages(g, lens, page, extra // page + 1)
    q = rand(g, B, Hq, D, dtype=torch.bfloat16, scale=2.0)
    k, ks = make_cache(g, pages * page, Hk, D, torch.bfloat16, fp8)
    v, vs = make_cache(g, pages * page, Hk, D, torch.bfloat16, fp8)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    before = weights(g, B, Hk, 301)
    after = torch.full_like(before, -1.0)
    kw = dict(page_size=page, return_lse=True)
    want, lse = paged_attention(q, k, v, table, n, k_scale=ks, v_scale=vs, weight=before, weight_out=after, **kw)
    q2, out, _ = pair(q, torch.zeros_like(q), dim)
    k2, v2, _ = pair(k, v, dim)
    ks2, vs2 = pair(ks, vs, dim)[:2] if fp8 else (None, None)
    w2, wo2, _ = pair(before, torch.full_like(before, -1.0), dim)
    got, lse2 = paged_attention(q2, k2, v2, table, n, k_scale=ks2, v_scale=vs2, weight=w2, weight_out=wo2, out=out, **kw)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want) and torch.equal(lse2, lse) and torch.equal(wo2, after)
    assert torch.equal(q2, q) and torch.equal(w2, before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
@pytest.mark.parametrize("dim", [0, 1, 2])
def test_evict(dtype, dim):
    g = gen(10 + dim)
    lens, budget, page, H = [300, 41, 0], 100, 16, 3
    data, scales, table, to = make(g, lens, budget, H, 24, page, dtype)
    w = weights(g, 3, H, 301)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    kept, left, out = paged.evict(w, n, budget, 7, 2)
    want = [None if x is None else paged.move(x, kept, table, to, page) for x in (*data, *scales)]
    k, v, _ = pair(*data, dim)
    ks, vs = pair(*scales, dim)[:2] if dtype is FP8 else (None, None)
    w2, wo2, _ = pair(w, torch.full_like(w, -1.0), dim)
    got = cache_evict(k, v, w2, table, n, to, page_size=page, budget=budget, recent=7, sinks=2, k_scale=ks, v_scale=vs, weight_out=wo2)
    assert torch.equal(got[0].cpu(), kept) and torch.equal(got[1].cpu(), left) and torch.equal(bits(wo2.cpu()), bits(out)) and torch.equal(w2, w)
    for x, y in zip((k, v, ks, vs), want):
        assert x is None or torch.equal(bits(x), bits(y))


def test_on_one_another():
    g = gen(20)
    B, Hq, Hk, D, page, lens = 3, 16, 2, 128, 16, [300, 0, 77]
    table, pages = make_pages(g, lens, page)
    buffer = rand(g, B + 1, Hq + 1, D, dtype=torch.bfloat16)
    q = buffer[:B, :Hq]
    k, _ = make_cache(g, pages * page, Hk, D, torch.bfloat16, False)
    v, _ = make_cache(g, pages * page, Hk, D, torch.bfloat16, False)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    w = torch.zeros(B + 1, Hk + 1, 310, device="cuda")
    keep = buffer.clone()
    for out in (q, buffer[1:, :Hq], buffer[:B, 1:], buffer[1:, 1:], buffer.view(-1)[64:64 + B * Hq * D].view(B, Hq, D)):
        with pytest.raises(RuntimeError):
            paged_attention(q, k, v, table, n, page_size=page, out=out)
    with pytest.raises(RuntimeError):  # (rows of its own sequences on one another, strides of a row or more)
        paged_attention(q, k, v, table, n, page_size=page, out=torch.as_strided(torch.empty_like(buffer), (B, Hq, D), (2 * D, D, 1)))
    place = w[:B, :Hk, :300]
    spare = torch.tensor([[0], [1], [2]], device="cuda", dtype=torch.int32)
    for other in (w[1:, :Hk, :300], w[:B, 1:, :300], w[:B, :Hk, 1:301], w[:B, :Hk, 10:]):
        with pytest.raises(RuntimeError):
            paged_attention(q, k, v, table, n, page_size=page, weight=place, weight_out=other)
        with pytest.raises(RuntimeError):
            cache_evict(k, v, place, table, n, spare, page_size=page, budget=16, weight_out=other)
    torch.cuda.synchronize()
    assert torch.equal(buffer, keep) and bool((w == 0).all())
