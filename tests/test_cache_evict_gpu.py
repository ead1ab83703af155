"""Eviction from a paged cache by accumulated weight against its definition: exact, ties and untouched rows included."""
import pytest
import torch

import paged_ref as paged
from jit_kernel import _native
from jit_kernel.kv_cache import cache_evict
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


def make(g, lens, budget, H, D, page, dtype, wide=False):
    """(caches and scales, page table, pages to move to): the two kinds of pages in no order, entries behind them not to be followed"""
    need, more = [-(-n // page) for n in lens], -(-budget // page)
    B, pages = len(lens), sum(need) + len(lens) * more + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, max(need + [1])), 0x7fffffff, dtype=torch.int32, device="cuda")
    to = torch.full((B, more + 1), 0x7fffffff, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        to[b, :more] = order[at + n:at + n + more]
        at += n + more
    slots = pages * page
    data = []
    for _ in range(2):
        if dtype is FP8:
            x = torch.randint(0, 256, (slots, H, D), generator=g, device="cuda", dtype=torch.uint8)
        else:
            x = torch.randint(-32768, 32767, (slots, H, D), generator=g, device="cuda", dtype=torch.int16)
        if wide:  # strided, heads in front, rows on an odd boundary
            y = torch.zeros(H, slots, 2 * D + 1, device="cuda", dtype=x.dtype).transpose(0, 1)
            y[..., D + 1:] = x
            x = y[..., D + 1:]
        data.append(x.view(dtype))
    scales = [torch.rand(slots, H, generator=g, device="cuda") for _ in range(2)] if dtype is FP8 else [None, None]
    return data, scales, table, to[:, :more] if more else to[:, :0]


def weights(g, B, H, N, kind="heavy"):
    w = torch.exp(torch.randn(B, H, N, generator=g, device="cuda") * 3 - 6)
    if kind == "ties":
        w = torch.randint(0, 4, (B, H, N), generator=g, device="cuda").float() / 4
    elif kind == "same":
        w = torch.full((B, H, N), 0.125, device="cuda")
    elif kind == "odd":  # zeros of both signs, negatives, infinities, NaN, subnormals
        values = torch.tensor([0.0, -0.0, -1.0, 1e-42, -1e-42, float("inf"), float("-inf"), float("nan"), 3.0, 3.0000002], device="cuda")
        w = values[torch.randint(0, 10, (B, H, N), generator=g, device="cuda")]
    elif kind == "near":  # keys that differ in their lowest bits only
        w = (0x3f800000 + torch.randint(0, 700, (B, H, N), generator=g, device="cuda", dtype=torch.int32)).view(torch.float32)
    return w


def bits(x):
    return x.contiguous().view(torch.int32 if x.dtype.itemsize == 4 else torch.int16 if x.dtype.itemsize == 2 else torch.uint8)


def check(data, scales, table, to, w, lens, page, budget, recent, sinks, **kw):
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    kept, left, out = paged.evict(w, n, budget, recent, sinks)
    want = [None if x is None else paged.move(x, kept, table, to, page) for x in (*data, *scales)]
    got_kept, got_left, got_w = cache_evict(*data, w, table, n, to, page_size=page, budget=budget, recent=recent, sinks=sinks,
                                            k_scale=scales[0], v_scale=scales[1], **kw)
    assert torch.equal(got_left.cpu(), left)
    assert torch.equal(got_kept.cpu(), kept)
    assert torch.equal(bits(got_w.cpu()), bits(out))
    for x, y in zip((*data, *scales), want):
        assert x is None or torch.equal(bits(x), bits(y))
    return got_kept, got_left, got_w


SHAPES = [  # heads, page, lengths, budget, recent, sinks
    (1, 1, [1], 1, 0, 0), (1, 1, [2], 1, 0, 0), (2, 16, [100, 0, 17, 64], 64, 8, 4), (3, 5, [777, 1, 0, 1001], 300, 0, 0), (8, 64, [1500] * 3, 1000, 100, 4),
    (1, 24, [5000], 4999, 0, 0), (2, 7, [3000], 40, 20, 20), (1, 128, [20000], 9000, 512, 4), (40, 3, [33, 65, 97, 129, 31], 32, 1, 1), (2, 64, [70], 0, 0, 0)]


@pytest.mark.parametrize("H,page,lens,budget,recent,sinks", SHAPES)
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (FP8, 128), (torch.float16, 64), (FP8, 8), (torch.bfloat16, 80), (FP8, 256)])
def test_evict(dtype, D, H, page, lens, budget, recent, sinks):
    g = gen(H * page + budget + D)
    data, scales, table, to = make(g, lens, budget, H, D, page, dtype)
    w = weights(g, len(lens), H, max(lens) + 5)
    check(data, scales, table, to, w, lens, page, budget, recent, sinks)


@pytest.mark.parametrize("kind", ["ties", "same", "odd", "near"])
@pytest.mark.parametrize("lens,budget,recent,sinks", [([500, 333], 100, 10, 3), ([3000], 1500, 0, 0), ([30000], 7001, 100, 0), ([200], 199, 0, 0), ([90, 80], 16, 8, 8)])
def test_weights_of_every_kind(kind, lens, budget, recent, sinks):
    g = gen(budget)
    data, scales, table, to = make(g, lens, budget, 2, 16, 16, torch.bfloat16)
    check(data, scales, table, to, weights(g, len(lens), 2, max(lens), kind), lens, 16, budget, recent, sinks)


@pytest.mark.parametrize("n", [8191, 163841, 200003])
def test_longer_than_shared_memory(n):
    """One unit over a cluster, keys beyond shared memory's room read again; and many units, a CTA each."""
    g = gen(n)
    for H in (1, 200 if n < 10000 else 2):
        data, scales, table, to = make(g, [n], n // 3, H, 8, 64, FP8)
        check(data, scales, table, to, weights(g, 1, H, n), [n], 64, n // 3, 100, 4)


def test_one_cta_beyond_shared_memory():
    g = gen(5)
    n, H = 30001, 160
    data, scales, table, to = make(g, [n], 64, H, 8, 64, FP8)
    check(data, scales, table, to, weights(g, 1, H, n, "near"), [n], 64, 64, 1, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
def test_strides_and_outputs(dtype):
    g = gen(21)
    lens, page, budget, H = [300, 41, 0], 16, 100, 3
    data, scales, table, to = make(g, lens, budget, H, 24, page, dtype, wide=True)
    if scales[0] is not None:
        scales = [s.t().contiguous().t() for s in scales]
    wide = torch.full((H, 3, 700), float("nan"), device="cuda")
    w = wide.transpose(0, 1)[..., 100:400]
    w.copy_(weights(g, 3, H, 300))
    place = torch.full((3, H, 302), 7.0, device="cuda")
    t2 = torch.full((3, 90), 0x7fffffff, device="cuda", dtype=torch.int32)
    t2[:, 5:5 + table.size(1)] = table
    _, _, got = check(data, scales, t2[:, 5:5 + table.size(1)], to, w, lens, page, budget, 7, 2, weight_out=place[..., 1:301])
    assert got.data_ptr() == place[..., 1:].data_ptr()
    assert bool((place[..., 0] == 7).all()) and bool((place[..., 301] == 7).all())


def test_bad_pages_and_lengths():
    """Rows on negative pages, or beyond the cache, are not copied - on either side -, and nothing is written where they would go."""
    g = gen(22)
    data, scales, table, to = make(g, [160], 64, 2, 32, 16, FP8)
    slots = data[0].size(0)
    for t, z in (((3, -1), None), ((3, slots // 16), None), (None, (1, -5)), (None, (1, 0x7fffffff)), ((0, 0x7fffffff), (0, slots // 16))):
        a, c = table.clone(), to.clone()
        if t:
            a[0, t[0]] = t[1]
        if z:
            c[0, z[0]] = z[1]
        check([x.clone() for x in data], [x.clone() for x in scales], a, c, weights(g, 1, 2, 160), [160], 16, 64, 60, 4)
        st = take_status()
        # (rows in the middle of page 3 need not be among those that stay)
        assert st in (0, _native.ST_BAD_INDEX) and (st or not z)
    # lengths beyond the table, beyond the weights, below zero
    for n, cols in ((161, 200), (160, 100), (1 << 30, 200)):
        w = weights(g, 1, 2, cols)
        m = min(n, 160, cols)
        kept, left, out = paged.evict(w, torch.tensor([m]), 64, 8, 0)
        got = cache_evict(*data, w, table, torch.tensor([n], device="cuda", dtype=torch.int32), to, page_size=16, budget=64, recent=8,
                          k_scale=scales[0], v_scale=scales[1])
        assert torch.equal(got[0].cpu(), kept) and torch.equal(got[1].cpu(), left) and torch.equal(got[2].cpu(), out)
        assert take_status() == _native.ST_BAD_INDEX
    check(data, scales, table, to, weights(g, 1, 2, 160), [-3], 16, 64, 8, 0)


def test_empty():
    c, s = torch.zeros(0, 2, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(3, 2, 0, device="cuda")
    t, n = torch.zeros(3, 0, device="cuda", dtype=torch.int32), torch.zeros(3, device="cuda", dtype=torch.int32)
    kept, left, out = cache_evict(c, c.clone(), s, t, n, t, page_size=4, budget=0)
    assert kept.shape == (3, 2, 0) and bool((left == 0).all()) and out.shape == s.shape
    kept, left, out = cache_evict(c, c.clone(), s[:0], t[:0], n[:0], t[:0], page_size=4, budget=0)
    assert kept.shape == (0, 2, 0) and left.shape == (0,)


def test_streams_and_graphs():
    g = gen(23)
    lens, budget, page, H = [900, 30, 1000], 128, 16, 8
    data, scales, table, to = make(g, lens, budget, H, 64, page, torch.float16)
    start = [x.clone() for x in data]
    w = weights(g, 3, H, 1000)
    n = torch.tensor(lens, device="cuda", dtype=torch.int32)
    kw = dict(page_size=page, budget=budget, recent=16, sinks=4)
    graph = torch.cuda.CUDAGraph()
    cache_evict(*data, w, table, n, to, **kw)
    with torch.cuda.graph(graph):
        kept, left, out = cache_evict(*data, w, table, n, to, **kw)
    for new in (lens, [128, 129, 0], [1, 1000, 999]):
        n.copy_(torch.tensor(new, dtype=torch.int32))
        w.copy_(weights(g, 3, H, 1000))
        for x, y in zip(data, start):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        a, b, c = paged.evict(w, n, budget, 16, 4)
        assert torch.equal(kept.cpu(), a) and torch.equal(left.cpu(), b) and torch.equal(bits(out.cpu()), bits(c))
        for x, y in zip(data, start):
            assert torch.equal(bits(x), bits(paged.move(y, a, table, to, page)))
    # (the second sequence has pages for 30 rows: the replays with longer ones say so)
    assert take_status() == _native.ST_BAD_INDEX
    # two streams at once, on caches of their own
    sets = [[x.clone() for x in start] for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for mine in sets:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(3):
                r = cache_evict(*mine, w, table, n, to, **kw)
            got.append(r)
    torch.cuda.synchronize()
    for mine, r in zip(sets, got):
        assert torch.equal(r[0], kept) and all(torch.equal(bits(x), bits(y)) for x, y in zip(mine, data))
    assert take_status() == _native.ST_BAD_INDEX


def test_refusals():
    k = torch.zeros(64, 2, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(2, 2, 32, device="cuda")
    t = torch.zeros(2, 2, device="cuda", dtype=torch.int32)
    n = torch.zeros(2, device="cuda", dtype=torch.int32)
    good = dict(k_cache=k, v_cache=k.clone(), weight=w, page_table=t, lengths=n, to_table=t + 2, page_size=16, budget=32)
    cache_evict(**good)
    x8 = k.to(FP8)
    for bad in (dict(k_cache=k[0]), dict(v_cache=k.half()), dict(v_cache=k[:32]), dict(k_cache=k.float(), v_cache=k.float()), dict(k_cache=x8, v_cache=x8),
                dict(k_scale=w[0], v_scale=w[0]), dict(k_cache=k[..., :12], v_cache=k[..., :12]), dict(k_cache=k[..., ::2], v_cache=k[..., ::2]),
                dict(weight=w.double()), dict(weight=w[0]), dict(weight=w[:, :1]), dict(weight=w[:1]), dict(weight=w[..., ::2]), dict(weight=w.cpu()),
                dict(page_table=t.long()), dict(page_table=t[:1]), dict(to_table=t[:1]), dict(to_table=t.cpu()), dict(lengths=n.long()),
                dict(lengths=n[:1]), dict(lengths=None), dict(page_size=0), dict(page_size=1 << 31), dict(budget=-1), dict(budget=33), dict(recent=-1),
                dict(sinks=-1), dict(recent=20, sinks=13), dict(weight_out=w), dict(weight_out=w[..., :16]), dict(weight_out=w.half()),
                dict(k_cache=k.clone().requires_grad_()), dict(weight=w.clone().requires_grad_())):
        with pytest.raises((RuntimeError, AttributeError)):
            cache_evict(**{**good, **bad})
    torch.cuda.synchronize()
