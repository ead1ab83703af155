"""Attention over a paged cache, and the weights its rows have had, against 64-bit statements of them."""
import pytest
import torch

import paged_ref as paged
import rows_ref as ref
from jit_kernel import _native
from jit_kernel.paged_attention import paged_attention
from jit_kernel.topk_indexer import _status_word, kernel_status

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def status():
    if torch.cuda.is_available():
        _status_word(torch.device("cuda", 0)).zero_()
    yield
    if torch.cuda.is_available():
        assert kernel_status() == 0


def take_status():
    st = kernel_status()
    _status_word(torch.device("cuda", 0)).zero_()
    return st


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def make_cache(g, rows, H, D, dtype, fp8, wide=False):
    """(cache, scale or None); wide: strided, with NaN between the rows"""
    x = rand(g, rows, H, D) * (0.2 + torch.rand(rows, H, 1, generator=g, device="cuda"))
    if fp8:
        x, s = ref.quantise(x)
        if not wide:
            return x, s
        y = torch.full((H, rows, 2 * D), 0x7f, device="cuda", dtype=torch.uint8).transpose(0, 1)
        y[..., D:] = x.view(torch.uint8)
        return y[..., D:].view(FP8), s.t().contiguous().t()
    if not wide:
        return x.to(dtype), None
    y = torch.full((H, rows, 2 * D), float("nan"), device="cuda", dtype=dtype).transpose(0, 1)
    y[..., D:] = x.to(dtype)
    return y[..., D:], None


def make_pages(g, lengths, page, extra=1):
    """(page table, pages of the cache): pages in no order; behind a sequence's pages entries that may not be followed."""
    need = [-(-n // page) for n in lengths]
    cols = max(need) + extra
    order = torch.randperm(sum(need) + 2, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), cols), 0x7fffffff, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 2


def ragged(g, B, longest):
    n = torch.randint(0, longest + 1, (B,), generator=g, device="cuda").tolist()
    n[0] = longest
    if B > 2:
        n[1], n[2] = 0, 1
    return n


SHAPES = [  # q heads, kv heads, page, lengths (or sequences and the longest)
    (1, 1, 1, [1]), (64, 8, 16, [100]), (21, 3, 5, [777, 0, 1]), (128, 1, 64, [1000, 333]), (16, 2, 24, (70, 300)), (8, 8, 128, [5, 9]),
    (40, 2, 3, (9, 500)), (64, 8, 64, [9000]), (6, 6, 16, (5, 1000)), (64, 1, 64, (160, 200)), (32, 2, 16, [0, 0, 17, 0]), (9, 1, 7, [0]),
    (8, 1, 1, [63, 64, 65])]


@pytest.mark.parametrize("Hq,Hk,page,lengths", SHAPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention(dtype, fp8, D, Hq, Hk, page, lengths):
    g = gen(Hq * page + D)
    lens = ragged(g, *lengths) if isinstance(lengths, tuple) else lengths
    B = len(lens)
    table, pages = make_pages(g, lens, page)
    q = rand(g, B, Hq + 2, D, dtype=dtype, scale=2.0)[:, 1:Hq + 1]
    k, ks = make_cache(g, pages * page, Hk, D, dtype, fp8, page % 2 == 1)
    v, vs = make_cache(g, pages * page, Hk, D, dtype, fp8, page % 2 == 1)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    before = torch.rand(B, Hk, max(lens) + 3, generator=g, device="cuda")
    after = torch.full_like(before, float("nan"))
    out, lse = paged_attention(q, k, v, table, n, page_size=page, k_scale=ks, v_scale=vs, return_lse=True)
    want, at = paged.attention(q, k, v, table, n, page, None, ks, vs)
    ref.check_attention(out, lse, want)
    again, lse2 = paged_attention(q, k, v, table, n, page_size=page, k_scale=ks, v_scale=vs, weight=before, weight_out=after, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    paged.check_weights(after, before, n, *paged.weights(q, k, at, want, None, ks))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq", [8, 32])
def test_scale_out_and_table_strides(fp8, Hq):
    g = gen(7)
    lens, page = [300, 41, 0, 160], 16
    wide = torch.full((4, 40), 1 << 30, device="cuda", dtype=torch.int32)
    t, pages = make_pages(g, lens, page)
    wide[:, 3:3 + t.size(1)] = t
    table = wide[:, 3:3 + t.size(1)]
    q = rand(g, 4, Hq, 128, dtype=torch.bfloat16)
    k, ks = make_cache(g, pages * page, 2, 128, torch.bfloat16, fp8)
    v, vs = make_cache(g, pages * page, 2, 128, torch.bfloat16, fp8)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    out = torch.full((4, Hq + 1, 130), 7.0, device="cuda", dtype=torch.bfloat16)
    o = out[:, :Hq, 1:129]
    r = paged_attention(q, k, v, table, n, page_size=page, k_scale=ks, v_scale=vs, softmax_scale=0.3, out=o)
    assert r.data_ptr() == o.data_ptr()
    want, _ = paged.attention(q, k, v, table, n, page, 0.3, ks, vs)
    ref.check_attention(o, None, want)
    assert bool((out[:, Hq:] == 7).all()) and bool((out[..., 0] == 7).all()) and bool((out[..., 129] == 7).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_weights_in_place_and_alone(fp8):
    g = gen(11)
    lens, page, Hk = [700, 0, 33], 8, 2
    table, pages = make_pages(g, lens, page)
    q = rand(g, 3, 14, 64, dtype=torch.float16, scale=2.0)
    k, ks = make_cache(g, pages * page, Hk, 64, torch.float16, fp8)
    v, vs = make_cache(g, pages * page, Hk, 64, torch.float16, fp8)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    want, at = paged.attention(q, k, v, table, n, page, None, ks, vs)
    w, e = paged.weights(q, k, at, want, None, ks)
    kw = dict(page_size=page, k_scale=ks, v_scale=vs)
    alone = torch.full((3, Hk, 800), float("nan"), device="cuda")
    paged_attention(q, k, v, table, n, weight_out=alone, **kw)
    paged.check_weights(alone, None, n, w, e)
    # (heads before sequences in memory; NaN behind the lengths stays)
    place = torch.full((Hk, 3, 801), float("nan"), device="cuda").transpose(0, 1)
    first = torch.rand(3, Hk, 801, generator=g, device="cuda")
    j = torch.arange(801, device="cuda")
    place.copy_(torch.where((j < n.unsqueeze(1)).unsqueeze(1), first, float("nan")))
    paged_attention(q, k, v, table, n, weight=place, **kw)
    paged.check_weights(place, first, n, w, e)


def test_pages_shared_by_sequences():
    """A prompt's pages in several sequences, and a page twice in one: every sequence has its own weights."""
    g = gen(12)
    page, Hk = 16, 4
    table = torch.tensor([[3, 1, 0], [3, 1, 2], [2, 2, 2]], device="cuda", dtype=torch.int32)
    n = torch.tensor([48, 40, 47], device="cuda", dtype=torch.int32)
    q = rand(g, 3, 32, 128, dtype=torch.bfloat16)
    k, _ = make_cache(g, 4 * page, Hk, 128, torch.bfloat16, False)
    v, _ = make_cache(g, 4 * page, Hk, 128, torch.bfloat16, False)
    after = torch.full((3, Hk, 48), float("nan"), device="cuda")
    out, lse = paged_attention(q, k, v, table, n, page_size=page, weight_out=after, return_lse=True)
    want, at = paged.attention(q, k, v, table, n, page)
    ref.check_attention(out, lse, want)
    paged.check_weights(after, None, n, *paged.weights(q, k, at, want))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq", [16, 64])
def test_bad_pages_and_lengths(fp8, Hq):
    """Rows in front of and behind the cache are NaN: none of them is read. Negative pages are left out without a word, rows beyond
    the cache and positions beyond the table with a status bit."""
    g = gen(8)
    whole = torch.full((120, 1, 128), float("nan"), device="cuda", dtype=torch.bfloat16)
    if fp8:
        whole = torch.full((120, 1, 128), 0x7f, device="cuda", dtype=torch.uint8).view(FP8)
    k, ks = make_cache(g, 100, 1, 128, torch.bfloat16, fp8)
    whole.view(torch.uint8)[10:110] = k.view(torch.uint8)
    cache = whole[10:110]
    q = rand(g, 4, Hq, 128, dtype=torch.bfloat16)
    n = torch.tensor([64, 48, -5, 16], device="cuda", dtype=torch.int32)
    table = torch.tensor([[0, -1, 2, -7], [-1, -2, -1, 9], [1, 1, 1, 1], [-1, 0, 0, 0]], device="cuda", dtype=torch.int32)
    after = torch.full((4, 1, 64), float("nan"), device="cuda")
    kw = dict(page_size=16, k_scale=ks, v_scale=ks)
    out, lse = paged_attention(q, cache, cache, table, n, weight_out=after, return_lse=True, **kw)
    want, at = paged.attention(q, cache, cache, table, n, 16, None, ks, ks)
    ref.check_attention(out, lse, want)
    paged.check_weights(after, None, n, *paged.weights(q, cache, at, want, None, ks))
    assert bool((out[1:] == 0).all()) and bool(lse[1:].isneginf().all()) and take_status() == 0
    # page 6 holds rows 96 to 111 (of 100), page 7 none
    table = torch.tensor([[0, 6, 2, 7], [6, 0x7fffffff, 3, 3], [1, 1, 1, 1], [2, 0, 0, 0]], device="cuda", dtype=torch.int32)
    n = torch.tensor([64, 64, 65, 1 << 30], device="cuda", dtype=torch.int32)
    for b in range(4):
        after = torch.full((1, 1, 64), float("nan"), device="cuda")
        out, lse = paged_attention(q[b:b + 1], cache, cache, table[b:b + 1], n[b:b + 1], weight_out=after, return_lse=True, **kw)
        want, at = paged.attention(q[b:b + 1], cache, cache, table[b:b + 1], n[b:b + 1], 16, None, ks, ks)
        ref.check_attention(out, lse, want)
        paged.check_weights(after, None, n[b:b + 1], *paged.weights(q[b:b + 1], cache, at, want, None, ks))
        assert take_status() == _native.ST_BAD_INDEX


def test_weights_shorter_than_a_sequence():
    g = gen(9)
    q, (k, _) = rand(g, 1, 8, 64, dtype=torch.float16), make_cache(g, 64, 1, 64, torch.float16, False)
    table, n = torch.tensor([[0, 1, 2, 3]], device="cuda", dtype=torch.int32), torch.tensor([50], device="cuda", dtype=torch.int32)
    guard = torch.full((1, 1, 64), float("nan"), device="cuda")
    paged_attention(q, k, k, table, n, page_size=16, weight_out=guard[..., :40])
    assert take_status() == _native.ST_BAD_INDEX
    want, at = paged.attention(q, k, k, table, n, 16)
    w, e = paged.weights(q, k, at, want)
    paged.check_weights(guard, None, torch.tensor([40]), w[..., :40], e[..., :40])


@pytest.mark.parametrize("fp8", [False, True])
def test_empty_caches_and_batches(fp8):
    q = torch.ones(2, 8, 64, device="cuda", dtype=torch.bfloat16)
    c = torch.zeros(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    s = None
    if fp8:
        c, s = c.to(FP8), torch.zeros(0, 2, device="cuda")
    kw = dict(page_size=4, k_scale=s, v_scale=s, return_lse=True)
    n = torch.tensor([3, 0], device="cuda", dtype=torch.int32)
    out, lse = paged_attention(q, c, c, torch.zeros(2, 1, device="cuda", dtype=torch.int32), n, **kw)
    assert bool((out == 0).all()) and bool(lse.isneginf().all()) and take_status() == _native.ST_BAD_INDEX
    out, lse = paged_attention(q, c, c, torch.zeros(2, 0, device="cuda", dtype=torch.int32), n * 0, **kw)
    assert bool((out == 0).all()) and bool(lse.isneginf().all())
    out, lse = paged_attention(q[:0], c, c, torch.zeros(0, 1, device="cuda", dtype=torch.int32), n[:0], **kw)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)


@pytest.mark.parametrize("fp8", [False, True])
def test_large_scores_nan_and_infinities(fp8):
    """Scores of +-1e4; a NaN key row makes the sequence's heads NaN and no other sequence's; infinities in rows behind a length and
    on pages that nothing names touch nothing."""
    g = gen(13)
    page, lens = 8, [100, 100, 90]
    table, pages = make_pages(g, lens, page)
    q = rand(g, 3, 8, 128, dtype=torch.bfloat16, scale=30.0)
    k, ks = make_cache(g, pages * page, 1, 128, torch.bfloat16, fp8)
    v, vs = make_cache(g, pages * page, 1, 128, torch.bfloat16, fp8)
    if fp8:
        ks = ks * 30
    else:
        k = k * 30
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    named = paged.slots_of(table, n, page, "cuda")
    free = torch.ones(pages * page, device="cuda", dtype=torch.bool)
    free[named[named >= 0].long()] = False
    for x in (k, v):
        x.view(torch.uint8)[free] = 0x7f if fp8 else torch.full((1,), float("inf"), dtype=x.dtype, device="cuda").view(torch.uint8).repeat(128)
    want, _ = paged.attention(q, k, v, table, n, page, None, ks, vs)
    out, lse = paged_attention(q, k, v, table, n, page_size=page, k_scale=ks, v_scale=vs, return_lse=True)
    ref.check_attention(out, lse, want)
    row = int(named[1, 37])
    k.view(torch.uint8)[row] = 0x7f if fp8 else torch.full((1,), float("nan"), dtype=k.dtype, device="cuda").view(torch.uint8).repeat(128)
    bad, bad_lse = paged_attention(q, k, v, table, n, page_size=page, k_scale=ks, v_scale=vs, return_lse=True)
    assert bool(bad[1].isnan().all()) and bool(bad_lse[1].isnan().all())
    assert torch.equal(bad[0], out[0]) and torch.equal(bad[2], out[2])


def test_v_scales_far_apart():
    """Rows of v scales of 2^-90, below zero, zero, and of 2^20 with hardly any weight behind it: the others are as exact as ever."""
    g = gen(14)
    page, lens = 16, [200]
    table, pages = make_pages(g, lens, page)
    q = rand(g, 1, 8, 128, dtype=torch.bfloat16, scale=2.0)
    k, ks = make_cache(g, pages * page, 1, 128, torch.bfloat16, True)
    v, vs = make_cache(g, pages * page, 1, 128, torch.bfloat16, True)
    at = paged.slots_of(table, torch.tensor(lens), page, "cuda")[0].long()
    vs[at[5]], vs[at[6]], vs[at[7]] = 2.0 ** -90, -vs[at[7]], 0.0
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    want, _ = paged.attention(q, k, v, table, n, page, None, ks, vs)
    out, lse = paged_attention(q, k, v, table, n, page_size=page, k_scale=ks, v_scale=vs, return_lse=True)
    ref.check_attention(out, lse, want)
    # a row whose score is far below the others' and whose v scale is 2^20: it takes nothing from the others
    ks[at[9]] = 0
    q2 = q.abs() * 4
    k.view(torch.uint8)[at] = k[at].float().abs().to(FP8).view(torch.uint8)
    vs[at[9]] = 2.0 ** 20
    want, _ = paged.attention(q2, k, v, table, n, page, None, ks, vs)
    out, lse = paged_attention(q2, k, v, table, n, page_size=page, k_scale=ks, v_scale=vs, return_lse=True)
    ref.check_attention(out, lse, want)


def test_offsets_beyond_32_bits():
    """Rows whose elements lie beyond 2^32 bytes and 2^31 elements of the cache."""
    g = gen(15)
    slots, page = 2_200_000, 100
    cache = torch.zeros(slots, 8, 128, device="cuda", dtype=torch.uint8)
    scale = torch.zeros(slots, 8, device="cuda")
    c, s = make_cache(g, 300, 8, 128, torch.bfloat16, True)
    for i, at in enumerate((0, 10_000 * page, slots - page)):
        cache[at:at + page] = c[i * page:(i + 1) * page].view(torch.uint8)
        scale[at:at + page] = s[i * page:(i + 1) * page]
    table = torch.tensor([[slots // page - 1, 0, 10_000]], device="cuda", dtype=torch.int32)
    n = torch.tensor([289], device="cuda", dtype=torch.int32)
    q = rand(g, 1, 64, 128, dtype=torch.bfloat16)
    cache = cache.view(FP8)
    out, lse = paged_attention(q, cache, cache, table, n, page_size=page, k_scale=scale, v_scale=scale, return_lse=True)
    small = torch.tensor([[2, 0, 1]], device="cuda", dtype=torch.int32)
    want, _ = paged.attention(q, c, c, small, n, page, None, s, s)
    ref.check_attention(out, lse, want)
    a, b = paged_attention(q, c, c, small, n, page_size=page, k_scale=s, v_scale=s, return_lse=True)
    assert torch.equal(out, a) and torch.equal(lse, b)


def test_streams_graphs_and_repeats():
    """On a stream of its own beside another call, captured with lengths that change between replays, and twice with the same bits."""
    g = gen(16)
    page, lens, Hk = 16, [900, 1500, 20], 8
    table, pages = make_pages(g, [1600] * 3, page)
    q = rand(g, 3, 64, 128, dtype=torch.bfloat16)
    k, _ = make_cache(g, pages * page, Hk, 128, torch.bfloat16, False)
    v, _ = make_cache(g, pages * page, Hk, 128, torch.bfloat16, False)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    w = [torch.zeros(3, Hk, 1600, device="cuda") for _ in range(4)]
    first = paged_attention(q, k, v, table, n, page_size=page, weight_out=w[0], return_lse=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            for _ in range(3):
                got.append(paged_attention(q, k, v, table, n, page_size=page, weight_out=w[1 + i], return_lse=True))
    torch.cuda.synchronize()
    for o, l in got:
        assert torch.equal(o, first[0]) and torch.equal(l, first[1])
    assert torch.equal(w[1], w[0]) and torch.equal(w[2], w[0])
    graphs = []
    for _ in range(2):  # (two graphs, each with a workspace of its own, replayed in turn and side by side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, l = paged_attention(q, k, v, table, n, page_size=page, weight_out=w[3], return_lse=True)
        graphs.append((graph, o, l))
    for new in ([900, 1500, 20], [1, 0, 1600], [1600, 1599, 17], [0, 0, 0]):
        n.copy_(torch.tensor(new, dtype=torch.int32))
        w[3].zero_()
        for graph, _, _ in graphs:
            graph.replay()
        o, l = paged_attention(q, k, v, table, n, page_size=page, return_lse=True)
        wo = torch.zeros_like(w[3])
        paged_attention(q, k, v, table, n, page_size=page, weight_out=wo)
        for _, go, gl in graphs:
            assert torch.equal(go, o) and torch.equal(gl, l)
        assert torch.equal(w[3], wo)
        want, _ = paged.attention(q, k, v, table, n, page)
        ref.check_attention(o, l, want)


def test_refusals():
    q = torch.zeros(2, 8, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(32, 2, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(2, 2, device="cuda", dtype=torch.int32)
    n = torch.zeros(2, device="cuda", dtype=torch.int32)
    w = torch.zeros(2, 2, 32, device="cuda")
    good = dict(q=q, k_cache=k, v_cache=k, page_table=t, lengths=n, page_size=16)
    paged_attention(**good)
    x8 = k.to(FP8)
    for bad in (dict(q=q[0]), dict(q=q.float()), dict(q=q[..., :32]), dict(q=q.transpose(0, 2)), dict(q=q[:, :7]), dict(q=q[:1]),
                dict(k_cache=k[0]), dict(k_cache=k.half()), dict(v_cache=k.half()), dict(v_cache=k[:16]), dict(k_cache=x8, v_cache=x8),
                dict(k_scale=w[0], v_scale=w[0]), dict(k_cache=k[:, :0], v_cache=k[:, :0]), dict(page_table=t.long()), dict(page_table=t[0]),
                dict(page_table=t[:1]), dict(page_table=torch.zeros(2, 4, device="cuda", dtype=torch.int32)[:, ::2]), dict(page_table=t.cpu()),
                dict(lengths=n.long()), dict(lengths=n[:1]), dict(lengths=n.cpu()), dict(lengths=None), dict(page_size=0), dict(page_size=-1),
                dict(page_size=1 << 31), dict(page_size=0x7fffffff), dict(weight=w[:1]), dict(weight=w[:, :1]), dict(weight=w.double()),
                dict(weight=w[..., ::2]), dict(weight=w.cpu()), dict(weight=w, weight_out=w[..., :8]), dict(weight_out=w.half()),
                dict(out=q.float()), dict(out=q[:1]), dict(q=q.clone().requires_grad_()), dict(weight=w.clone().requires_grad_()),
                dict(k_cache=torch.zeros(32 * 128 + 8, device="cuda", dtype=torch.bfloat16)[4:-4].view(32, 2, 64))):
        with pytest.raises((RuntimeError, AttributeError)):
            paged_attention(**{**good, **bad})
    torch.cuda.synchronize()
