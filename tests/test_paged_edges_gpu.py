"""Attention over a paged cache and eviction from it at the edges of their launch plans and arguments."""
import math

import pytest
import torch

import paged_ref as paged
import rows_ref as ref
from jit_kernel.kv_cache import cache_evict
from jit_kernel.paged_attention import paged_attention
from jit_kernel.topk_indexer import _status_word, kernel_status
from test_cache_evict_gpu import check, make, weights
from test_paged_attention_gpu import SHAPES, gen, make_cache, make_pages, ragged, rand

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def status():
    if torch.cuda.is_available():
        _status_word(torch.device("cuda", 0)).zero_()
    yield
    if torch.cuda.is_available():
        assert kernel_status() == 0


def attend(g, lens, Hq, Hk, page, D, dtype, fp8, weigh=True, extra=1, **kw):
    table, pages = make_pages(g, lens, page, extra)
    q = rand(g, len(lens), Hq, D, dtype=dtype, scale=2.0)
    k, ks = make_cache(g, pages * page, Hk, D, dtype, fp8)
    v, vs = make_cache(g, pages * page, Hk, D, dtype, fp8)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    after = torch.full((len(lens), Hk, max(lens)), float("nan"), device="cuda") if weigh else None
    out, lse = paged_attention(q, k, v, table, n, page_size=page, k_scale=ks, v_scale=vs, weight_out=after, return_lse=True, **kw)
    want, at = paged.attention(q, k, v, table, n, page, kw.get("softmax_scale"), ks, vs)
    ref.check_attention(out, lse, want)
    if weigh:
        paged.check_weights(after, None, n, *paged.weights(q, k, at, want, kw.get("softmax_scale"), ks))
    return out


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hk", [(700, 700), (600, 300), (1200, 40)])
def test_more_key_heads_than_ctas(fp8, Hq, Hk):
    """A run for each key head, in several waves; and few runs of many heads."""
    attend(gen(Hq), [70, 0, 33], Hq, Hk, 16, 64, torch.bfloat16, fp8)


@pytest.mark.parametrize("B,Hq,longest", [(1000, 8, 40), (333, 12, 600), (2100, 1, 5)])
def test_many_sequences(B, Hq, longest):
    """More sequences than a warp has lanes, many times over, empty ones among them; several to a warp in the join."""
    g = gen(B)
    lens = torch.randint(0, longest + 1, (B,), generator=g, device="cuda").tolist()
    lens[:3], lens[-2:] = [longest, 0, 1], [longest, 0]
    attend(g, lens, Hq, 1, 8, 64, torch.float16, B % 2 == 0)


@pytest.mark.parametrize("room,Hq,Hk,page,lengths", [(52000, *x) for x in SHAPES] + [
    (7000, *x) for x in SHAPES + [(8, 1, 8, (1000, 40)), (12, 1, 8, (333, 600)), (3, 3, 16, (2100, 5))]])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
def test_wide_tables(fp8, D, room, Hq, Hk, page, lengths):
    """Tables with room for 7,000 and 52,000 positions, most of it unused: clusters whose CTAs have less than a block each; runs that hold many
    sequences and parts of them, several pairs to a warp of the join."""
    g = gen(Hq * page + D + 1)
    lens = ragged(g, *lengths) if isinstance(lengths, tuple) else lengths
    attend(g, lens, Hq, Hk, page, D, torch.bfloat16, fp8, extra=room // page)


@pytest.mark.parametrize("fp8", [False, True])
def test_runs_and_their_join_in_a_graph(fp8):
    """Room for long sequences: equal runs and a second kernel, captured with lengths that change between replays, two graphs side by side."""
    g = gen(17)
    page, Hk = 64, 4
    table, pages = make_pages(g, [13000, 9000, 20000], page)
    q = rand(g, 3, 32, 128, dtype=torch.bfloat16)
    k, ks = make_cache(g, pages * page, Hk, 128, torch.bfloat16, fp8)
    v, vs = make_cache(g, pages * page, Hk, 128, torch.bfloat16, fp8)
    n = torch.tensor([13000, 9000, 20000], device="cuda", dtype=torch.int32)
    kw = dict(page_size=page, k_scale=ks, v_scale=vs, return_lse=True)
    w = [torch.zeros(3, Hk, 20000, device="cuda") for _ in range(3)]
    paged_attention(q, k, v, table, n, weight_out=w[2], **kw)
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = paged_attention(q, k, v, table, n, weight_out=w[i] if i else None, **kw)
        graphs.append((graph, r))
    for lens in ([13000, 9000, 20000], [1, 0, 19999], [0, 0, 0], [12999, 17, 64]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        for x in w:
            x.fill_(float("nan"))
        for graph, _ in graphs:
            graph.replay()
        a = paged_attention(q, k, v, table, n, weight_out=w[2], **kw)
        want, at = paged.attention(q, k, v, table, n, page, None, ks, vs)
        ref.check_attention(*a, want)
        for _, r in graphs:
            assert torch.equal(r[0], a[0]) and torch.equal(r[1], a[1])
        assert torch.equal(w[1].view(torch.int32), w[2].view(torch.int32))
        paged.check_weights(w[2], None, n, *paged.weights(q, k, at, want, None, ks))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens", [[60000] + [3] * 40, [3] * 40 + [60000], [1, 50001, 0, 2]])
def test_one_long_sequence_among_short_ones(fp8, lens):
    attend(gen(len(lens)), lens, 8, 2, 64, 128, torch.bfloat16, fp8)


def test_pages_longer_than_sequences():
    attend(gen(5), [100, 31, 1], 8, 2, 1 << 12, 64, torch.bfloat16, True)
    attend(gen(6), [100, 31, 1], 8, 2, 4001, 64, torch.bfloat16, True)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-6])
def test_softmax_scales(fp8, scale):
    attend(gen(7), [300, 17], 16, 2, 16, 128, torch.float16, fp8, softmax_scale=scale)


@pytest.mark.parametrize("fp8", [False, True])
def test_a_scale_that_is_nan(fp8):
    """NaN for every sequence that has a row, zeros for the others, as ever."""
    g = gen(8)
    table, pages = make_pages(g, [300, 0], 16)
    q = rand(g, 2, 8, 128, dtype=torch.bfloat16)
    k, ks = make_cache(g, pages * 16, 1, 128, torch.bfloat16, fp8)
    n = torch.tensor([300, 0], device="cuda", dtype=torch.int32)
    out, lse = paged_attention(q, k, k, table, n, page_size=16, k_scale=ks, v_scale=ks, softmax_scale=math.nan, return_lse=True)
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all()) and bool((out[1] == 0).all()) and bool(lse[1].isneginf().all())


def test_row_strides_that_do_not_fit_32_bits_are_refused():
    base = torch.zeros(64, device="cuda", dtype=torch.bfloat16)
    far = torch.as_strided(base, (1, 1, 64), (1 << 32, 64, 1))  # (a lone slot's stride says nothing)
    q = torch.zeros(1, 1, 64, device="cuda", dtype=torch.bfloat16)
    t, n = torch.zeros(1, 1, device="cuda", dtype=torch.int32), torch.ones(1, device="cuda", dtype=torch.int32)
    assert bool((paged_attention(q, far, far, t, n, page_size=1) == 0).all())


@pytest.mark.parametrize("H,lens,budget", [(1, [262145], 5000), (3, [17000, 16384, 16385, 8193, 8192], 8192), (300, [600, 599], 100), (1, [4] * 700, 3)])
def test_evict_plans(H, lens, budget):
    """Clusters, keys that do and do not fit shared memory, more units than CTAs at once."""
    g = gen(len(lens) * H)
    data, scales, table, to = make(g, lens, budget, H, 8, 16, FP8)
    check(data, scales, table, to, weights(g, len(lens), H, max(lens)), lens, 16, budget, min(2, budget), 1)


def test_evict_by_parts_of_a_wider_pool():
    """Rows of one sequence after another into the same pages, freed in between; weights not contiguous."""
    g = gen(31)
    data, scales, table, to = make(g, [90, 80], 32, 2, 16, 16, torch.bfloat16)
    w = weights(g, 2, 2, 200)[..., 50:150]
    for b in (0, 1):
        part = [x.clone() for x in data]
        n = torch.tensor([[90, 80][b]], device="cuda", dtype=torch.int32)
        kept, left, out = paged.evict(w[b:b + 1], n, 32, 4, 4)
        got = cache_evict(*part, w[b:b + 1], table[b:b + 1], n, to[:1], page_size=16, budget=32, recent=4, sinks=4)
        assert torch.equal(got[0].cpu(), kept) and torch.equal(got[1].cpu(), left) and torch.equal(got[2].cpu(), out)
        for x, y in zip(part, data):
            assert torch.equal(x.view(torch.int16), paged.move(y, kept, table[b:b + 1], to[:1], 16).view(torch.int16))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,page", [(8, 16), (16, 16), (16, 5), (5, 32)])
@pytest.mark.parametrize("extra", [0, 3000])
def test_weights_onto_large_ones(fp8, Hq, page, extra):
    """What many calls have added up is rounded once more by this one (by two eights of heads: twice), not once for every head."""
    g = gen(Hq * page)
    lens = [900, 31, 0]
    table, pages = make_pages(g, lens, page, extra)
    q = rand(g, 3, Hq, 128, dtype=torch.bfloat16, scale=2.0)
    k, ks = make_cache(g, pages * page, 1, 128, torch.bfloat16, fp8)
    v, vs = make_cache(g, pages * page, 1, 128, torch.bfloat16, fp8)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    before = 3e4 + 3e4 * torch.rand(3, 1, 900, generator=g, device="cuda")
    after = torch.full_like(before, float("nan"))
    paged_attention(q, k, v, table, n, page_size=page, k_scale=ks, v_scale=vs, weight=before, weight_out=after)
    want, at = paged.attention(q, k, v, table, n, page, None, ks, vs)
    paged.check_weights(after, before, n, *paged.weights(q, k, at, want, None, ks))


@pytest.mark.parametrize("fp8", [False, True])
def test_broadcast_views(fp8):
    """One query for all sequences and heads, one table row for all sequences, weights that key heads share: read as they are. As results
    they are refused."""
    g = gen(91)
    B, Hq, Hk, D, page, n = 3, 8, 2, 64, 16, 150
    table, pages = make_pages(g, [n], page)
    table = table.expand(B, -1)
    q = rand(g, 1, 1, D, dtype=torch.float16, scale=2.0).expand(B, Hq, D)
    k, ks = make_cache(g, pages * page, Hk, D, torch.float16, fp8)
    v, vs = make_cache(g, pages * page, Hk, D, torch.float16, fp8)
    lens = torch.tensor([n, 77, 0], device="cuda", dtype=torch.int32)
    before = weights(g, B, 1, n).expand(B, Hk, n)
    after = torch.full((B, Hk, n), float("nan"), device="cuda")
    scales = dict(page_size=page, k_scale=ks, v_scale=vs)
    out, lse = paged_attention(q, k, v, table, lens, weight=before, weight_out=after, return_lse=True, **scales)
    want, at = paged.attention(q, k, v, table, lens, page, None, ks, vs)
    ref.check_attention(out, lse, want)
    paged.check_weights(after, before, lens, *paged.weights(q, k, at, want, None, ks))
    with pytest.raises(RuntimeError):
        paged_attention(q, k, v, table, lens, weight=before, **scales)
    with pytest.raises(RuntimeError):
        paged_attention(q, k, v, table, lens, out=torch.empty_like(out[:1]).expand(B, Hq, D), **scales)
    to = torch.arange(B * 4, device="cuda", dtype=torch.int32).view(B, 4) % pages
    with pytest.raises(RuntimeError):
        cache_evict(k, v, after, table, lens, to, budget=40, weight_out=before, **scales)
    with pytest.raises(RuntimeError):
        cache_evict(k[:, :1].expand_as(k), v, after, table, lens, to, budget=40, **scales)
