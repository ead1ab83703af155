"""Attention over selected cache rows against a 64-bit statement of it, and the whole chain: indexer inputs, selection, attention."""
import pytest
import torch

import rows_ref as ref
from jit_kernel import _native
from jit_kernel.indexer import FusedIndexerTopk, reference_logits
from jit_kernel.kv_cache import cache_write
from jit_kernel.norm_rope import indexer_qk_write, qkv_norm_rope_write
from jit_kernel.sparse_attention import sparse_attention
from jit_kernel.topk_indexer import _status_word, fast_topk_transform_ragged_fused, kernel_status

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def status():
    if torch.cuda.is_available():
        _status_word(torch.device("cuda", 0)).zero_()
    yield
    if torch.cuda.is_available():
        assert kernel_status() & ~_native.ST_GUESS_MISSED == 0


def take_status():
    st = kernel_status()
    _status_word(torch.device("cuda", 0)).zero_()
    return st


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def make_cache(g, rows, H, D, dtype, fp8, layout="dense"):
    """(cache, scale or None)"""
    x = rand(g, rows, H, D) * (0.2 + torch.rand(rows, H, 1, generator=g, device="cuda"))
    if not fp8:
        if layout == "dense":
            return x.to(dtype), None
        wide = torch.full((H, rows, 2 * D), float("nan"), device="cuda", dtype=dtype).transpose(0, 1)
        wide[..., D:] = x.to(dtype)
        return wide[..., D:], None
    c, s = ref.quantise(x)
    if layout == "dense":
        return c, s
    wide = torch.full((H, rows, 2 * D), 0x7f, device="cuda", dtype=torch.uint8).transpose(0, 1)
    wide[..., D:] = c.view(torch.uint8)
    return wide[..., D:].view(FP8), s.t().contiguous().t()


def make_indices(g, T, K, rows, empty=True):
    """Rows of picks with -1 strewn in, a tail of -1, one row (where there are several) without any."""
    idx = torch.randint(0, rows, (T, K), generator=g, device="cuda", dtype=torch.int32)
    drop = torch.rand(T, K, generator=g, device="cuda") < torch.rand(T, 1, generator=g, device="cuda") * 0.5
    idx[drop] = -1
    if T > 1:
        idx[1, K // 3:] = -1
        if empty:
            idx[T - 1] = -1
    return idx


SHAPES = [  # T, q heads, kv heads, picks, cache rows
    (1, 1, 1, 1, 1), (1, 64, 8, 2048, 5000), (3, 21, 3, 1000, 777), (4, 128, 1, 257, 4000), (2, 33, 1, 17, 64),
    (70, 16, 2, 40, 300), (2, 8, 8, 5, 9), (9, 40, 2, 129, 500), (1, 128, 1, 2048, 3000), (5, 6, 6, 128, 1000), (160, 64, 1, 64, 999)]


@pytest.mark.parametrize("T,Hq,Hk,K,rows", SHAPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention(dtype, fp8, D, T, Hq, Hk, K, rows):
    g = gen(T * K + D)
    layout = "dense" if K % 2 else "wide"
    q = rand(g, T, Hq + 2, D, dtype=dtype, scale=2.0)[:, 1:Hq + 1]
    k, ks = make_cache(g, rows, Hk, D, dtype, fp8, layout)
    v, vs = make_cache(g, rows, Hk, D, dtype, fp8, layout)
    idx = make_indices(g, T, K, rows)
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, k, v, idx, None, None, ks, vs))
    if T > 1:
        assert bool((out[T - 1] == 0).all()) and bool(lse[T - 1].isneginf().all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq", [8, 128])
def test_offsets_scale_out_and_strides(fp8, Hq):
    g = gen(7)
    T, rows = 6, 400
    q = rand(g, T, Hq, 128, dtype=torch.bfloat16)
    k, ks = make_cache(g, T * rows, 1, 128, torch.bfloat16, fp8)
    v, vs = make_cache(g, T * rows, 1, 128, torch.bfloat16, fp8)
    wide = torch.full((T, 700), 1 << 30, device="cuda", dtype=torch.int32)
    wide[:, :333] = make_indices(g, T, 333, rows)
    off = torch.arange(T, device="cuda", dtype=torch.int32) * rows
    out = torch.full((T, Hq + 1, 130), 7.0, device="cuda", dtype=torch.bfloat16)
    o = out[:, :Hq, 1:129]
    r = sparse_attention(q, k, v, wide[:, :333], k_scale=ks, v_scale=vs, offsets=off, softmax_scale=0.3, out=o)
    assert r.data_ptr() == o.data_ptr()
    ref.check_attention(o, None, ref.attention(q, k, v, wide[:, :333], off, 0.3, ks, vs))
    assert bool((out[:, Hq:] == 7).all()) and bool((out[..., 0] == 7).all()) and bool((out[..., 129] == 7).all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq", [16, 64])
def test_bad_indices_are_left_out(fp8, Hq):
    """Rows in front of and behind the cache are NaN: none of them is read. An index beyond the cache raises a status bit."""
    g = gen(8)
    whole = torch.full((120, 1, 128), float("nan"), device="cuda", dtype=torch.bfloat16)
    if fp8:
        whole = torch.full((120, 1, 128), 0x7f, device="cuda", dtype=torch.uint8).view(FP8)
    k, ks = make_cache(g, 100, 1, 128, torch.bfloat16, fp8)
    whole.view(torch.uint8)[10:110] = k.view(torch.uint8)
    cache = whole[10:110]
    scale = None
    if fp8:
        sw = torch.full((120, 1), float("nan"), device="cuda")
        sw[10:110] = ks
        scale = sw[10:110]
    q = rand(g, 3, Hq, 128, dtype=torch.bfloat16)
    idx = torch.tensor([[0, 99, 100, 5, -1, 2147483647], [100, 101, -5, -2147483648, 109, 1 << 30], [3, 3, 3, -1, 1, 2]],
                       device="cuda", dtype=torch.int32)
    out, lse = sparse_attention(q, cache, cache, idx, k_scale=scale, v_scale=scale, return_lse=True)
    assert take_status() == _native.ST_BAD_INDEX
    ref.check_attention(out, lse, ref.attention(q, cache, cache, idx, None, None, scale, scale))
    assert bool((out[1] == 0).all()) and bool(lse[1].isneginf().all())
    # an offset that takes entries below the cache
    off = torch.tensor([-50, -101, 97], device="cuda", dtype=torch.int32)
    out, lse = sparse_attention(q, cache, cache, idx, k_scale=scale, v_scale=scale, offsets=off, return_lse=True)
    assert take_status() == _native.ST_BAD_INDEX
    ref.check_attention(out, lse, ref.attention(q, cache, cache, idx, off, None, scale, scale))


@pytest.mark.parametrize("Hq", [4, 128])
def test_far_scores(Hq):
    """Scores of +-1e4 and more: the running maximum carries them; a later key may dwarf all before it."""
    g = gen(9)
    q = rand(g, 2, Hq, 128, dtype=torch.bfloat16, scale=30.0)
    k, v = rand(g, 700, 1, 128, dtype=torch.bfloat16, scale=30.0), rand(g, 700, 1, 128, dtype=torch.bfloat16)
    idx = torch.arange(700, device="cuda", dtype=torch.int32).repeat(2, 1)
    out, lse = sparse_attention(q, k, v, idx, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, k, v, idx))
    q.fill_(0)
    out, lse = sparse_attention(q, k, v, idx, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, k, v, idx))


@pytest.mark.parametrize("Hq", [4, 128])
def test_scales_of_all_sizes(Hq):
    """fp8: v scales over twelve decades, growing and falling along the list; q of huge and tiny heads."""
    g = gen(10)
    k, ks = make_cache(g, 600, 1, 64, torch.bfloat16, True)
    v, vs = make_cache(g, 600, 1, 64, torch.bfloat16, True)
    vs = vs * 10.0 ** torch.linspace(-6, 6, 600, device="cuda").unsqueeze(1)
    q = rand(g, 2, Hq, 64, dtype=torch.bfloat16)
    q[:, 0] *= 1e-30
    q[:, 1] *= 1e-3
    q[0, 2] = 0
    up = torch.arange(600, device="cuda", dtype=torch.int32)
    idx = torch.stack([up, up.flip(0)])
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, k, v, idx, None, None, ks, vs))
    big = q * 1e30
    out, lse = sparse_attention(big, k, v, idx, k_scale=ks * 1e-30, v_scale=vs, return_lse=True)
    ref.check_attention(out, lse, ref.attention(big, k, v, idx, None, None, ks * 1e-30, vs))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq", [4, 128])
def test_nan_stays_with_who_asks_for_it(fp8, Hq):
    g = gen(11)
    q = rand(g, 4, Hq, 128, dtype=torch.float16)
    k, ks = make_cache(g, 300, 1, 128, torch.float16, fp8)
    v, vs = make_cache(g, 300, 1, 128, torch.float16, fp8)
    nan = (lambda c: c.view(torch.uint8).__setitem__((17, 0, 3), 0x7f)) if fp8 else (lambda c: c.__setitem__((17, 0, 3), float("nan")))
    nan(k)
    nan(v)
    idx = torch.randint(20, 300, (4, 200), generator=g, device="cuda", dtype=torch.int32)
    idx[1, 60] = 17
    idx[2] = -1
    idx[2, 5] = 17
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, return_lse=True)
    assert bool(out[1:3].isnan().all()) and bool(lse[1:3].isnan().all())
    good = torch.tensor([0, 3], device="cuda")
    ref.check_attention(out[good], lse[good], ref.attention(q[good], k, v, idx[good], None, None, ks, vs))


def test_no_picks_and_no_tokens():
    q = torch.ones(3, 4, 64, device="cuda", dtype=torch.float16)
    c = torch.ones(5, 2, 64, device="cuda", dtype=torch.float16)
    out, lse = sparse_attention(q, c, c, torch.empty(3, 0, device="cuda", dtype=torch.int32), return_lse=True)
    assert bool((out == 0).all()) and bool(lse.isneginf().all())
    out, lse = sparse_attention(q, c[:0], c[:0], torch.full((3, 7), -1, device="cuda", dtype=torch.int32), return_lse=True)
    assert bool((out == 0).all()) and bool(lse.isneginf().all())
    assert sparse_attention(q[:0], c, c, torch.empty(0, 9, device="cuda", dtype=torch.int32)).shape == (0, 4, 64)


@pytest.mark.parametrize("Hq", [8, 128])
def test_long_cache(Hq):
    """Rows beyond 2^31 elements and 2^32 bytes."""
    rows = (1 << 31) // 128 + 5000
    cache = torch.zeros(rows, 1, 128, device="cuda", dtype=torch.bfloat16)
    g = gen(12)
    idx = torch.randint(rows - 4000, rows, (2, 300), generator=g, device="cuda", dtype=torch.int32)
    idx[1, ::2] = torch.randint(0, 4000, (150,), generator=g, device="cuda", dtype=torch.int32)
    cache[-4000:] = rand(g, 4000, 1, 128, dtype=torch.bfloat16)
    cache[:4000] = rand(g, 4000, 1, 128, dtype=torch.bfloat16)
    q = rand(g, 2, Hq, 128, dtype=torch.bfloat16)
    out, lse = sparse_attention(q, cache, cache, idx, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, cache, cache, idx))


@pytest.mark.parametrize("Hq", [8, 128])
def test_streams_graphs_and_repeats(Hq):
    """Two calls at once on two streams, one captured and replayed on new contents; the same call gives the same bits."""
    g = gen(13)
    T = 8
    q = rand(g, T, Hq, 128, dtype=torch.bfloat16)
    k, ks = make_cache(g, 4000, 1, 128, torch.bfloat16, True)
    v, vs = make_cache(g, 4000, 1, 128, torch.bfloat16, True)
    idx = make_indices(g, T, 2048, 4000)
    call = lambda: sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, return_lse=True)  # noqa: E731
    first = call()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = call()
    q.copy_(rand(g, T, Hq, 128, dtype=torch.bfloat16))
    idx.copy_(make_indices(g, T, 2048, 4000))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.replay()
    eager = call()
    torch.cuda.synchronize()
    assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])
    assert not torch.equal(first[0], eager[0])
    for _ in range(5):
        again = call()
        assert torch.equal(again[0], eager[0]) and torch.equal(again[1], eager[1])


@pytest.mark.parametrize("Hq,Hk", [(32, 4), (128, 1)])
def test_tree_of_drafts(Hq, Hk):
    """Drafted tokens written behind the context; each attends to its picks of the context and to its ancestors."""
    g = gen(14)
    context, parents = 3000, [-1, 0, 0, 1, 1, 2, 5]
    n = len(parents)
    k, ks = make_cache(g, context + 50, Hk, 128, torch.bfloat16, True)
    v, vs = make_cache(g, context + 50, Hk, 128, torch.bfloat16, True)
    slots = torch.arange(context, context + n, device="cuda", dtype=torch.int32)
    cache_write(rand(g, n, Hk, 128, dtype=torch.bfloat16), slots, k, ks, rand(g, n, Hk, 128, dtype=torch.bfloat16), v, vs)
    idx = torch.full((n, 2048 + n), -1, device="cuda", dtype=torch.int32)
    for t in range(n):
        idx[t, :2048] = torch.randperm(context, generator=g, device="cuda")[:2048].to(torch.int32)
        a, j = t, 2048
        while a >= 0:
            idx[t, j] = context + a
            a, j = parents[a], j + 1
    q = rand(g, n, Hq, 128, dtype=torch.bfloat16)
    out, lse = sparse_attention(q, k, v, idx, k_scale=ks, v_scale=vs, return_lse=True)
    ref.check_attention(out, lse, ref.attention(q, k, v, idx, None, None, ks, vs))


@pytest.mark.parametrize("Hq,Hk", [(32, 4), (128, 1)])
def test_decode_step(Hq, Hk):
    """One layer's decode step as it would be used: the indexer's q and k, the selection on its key cache, q, k and v of the
    attention into theirs, attention over what was selected. Each op against its own statement, on what the one before it made."""
    g = gen(15)
    B, rows, D = 5, 6000, 128
    lengths = torch.tensor([6000, 2049, 3500, 1000, 1], device="cuda", dtype=torch.int32)
    base = torch.arange(B, device="cuda", dtype=torch.int32) * rows
    pos = lengths - 1
    slots = base + pos
    table = ref.angles(rows, 64, "cuda")
    ik, isc = ref.quantise(rand(g, B, rows, D))
    q, k, w = rand(g, B, 64, D, dtype=torch.bfloat16), rand(g, B, D, dtype=torch.bfloat16), torch.rand(B, 64, generator=g, device="cuda")
    q8, w8 = indexer_qk_write(q, k, w, pos, table, slots, ik, isc)
    picker = FusedIndexerTopk(B, rows)
    idx = picker(q8, ik, w8, lengths, k_scale=isc)
    logits = reference_logits(q8, ik, w8, isc)
    for b in range(B):
        n = int(lengths[b])
        row = idx[b][idx[b] >= 0].long()
        assert row.numel() == min(n, 2048) and row.unique().numel() == row.numel() and int(row.max()) < n
        if n > 2048:
            worst = logits[b, row].min()
            rest = logits[b, :n].clone()
            rest[row] = -1e30
            assert float(rest.max() - worst) <= 2e-5 * float(logits[b, :n].abs().max())
    # the quantised indexer ranks as the unquantised one would, to the 2^-4 of q and of k that e4m3 rounds
    (kc, ks), (vc, vs) = (make_cache(g, B * rows, Hk, D, torch.bfloat16, True) for _ in range(2))
    qa, ka, va = (rand(g, B, h, D, dtype=torch.bfloat16) for h in (Hq, Hk, Hk))
    full = ref.angles(rows, D, "cuda")
    qr = qkv_norm_rope_write(qa, ka, va, pos, full, slots, kc, ks, vc, vs)
    ref.check_dense(qr, *ref.head_rows(qa, "rms", positions=pos, cos_sin=full))
    y, e = ref.head_rows(ka, "rms", positions=pos, cos_sin=full)
    ref.check_quantised(kc.view(torch.uint8)[slots.long()].view(FP8), ks[slots.long()], y, e)
    out, lse = sparse_attention(qr, kc, vc, idx, k_scale=ks, v_scale=vs, offsets=base, return_lse=True)
    ref.check_attention(out, lse, ref.attention(qr, kc, vc, idx, base, None, ks, vs))
    # the same slots from the selector that adds the offsets itself
    ragged = fast_topk_transform_ragged_fused(picker.logits[:B], lengths, base, 2048)
    again = sparse_attention(qr, kc, vc, ragged, k_scale=ks, v_scale=vs)
    ref.check_attention(again, None, ref.attention(qr, kc, vc, ragged, None, None, ks, vs))
