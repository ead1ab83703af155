"""Norm, rotation and quantisation of head rows, and the cache's rows read back, against 64-bit statements of the same."""
import pytest
import torch

import rows_ref as ref
from jit_kernel import _native
from jit_kernel.kv_cache import cache_read, cache_write
from jit_kernel.norm_rope import indexer_qk_write, qk_norm_rope, qkv_norm_rope_write
from jit_kernel.topk_indexer import _status_word, kernel_status

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
DT = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def status():
    """Every test leaves the device's status word as it found it: zero, but for the bits it takes itself."""
    if torch.cuda.is_available():
        _status_word(torch.device("cuda", 0)).zero_()
    yield
    if torch.cuda.is_available():
        assert kernel_status() == 0


def take_status():
    st = kernel_status()
    _status_word(torch.device("cuda", 0)).zero_()
    return st


def rand(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows_case(g, T, H, D, dtype, layout):
    """Activations [T, H, D]: dense, a slice of a fused projection, or starting off 16 bytes."""
    if layout == "dense":
        return rand(g, T, H, D, dtype=dtype)
    if layout == "slice":
        return rand(g, T, H + 3, D, dtype=dtype)[:, 1:H + 1]
    flat = rand(g, T * H * D + 1, dtype=dtype)
    return flat[1:].view(T, H, D)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,Hq,Hk,D,R,layout", [
    (1, 1, 1, 8, None, "dense"), (1, 64, 1, 128, 64, "dense"), (3, 5, 2, 64, 64, "slice"), (17, 7, 3, 80, 48, "slice"),
    (5, 4, 1, 96, 16, "odd"), (33, 9, 5, 256, 256, "dense"), (2, 3, 2, 136, 112, "slice"), (1300, 33, 4, 128, 128, "slice"),
    (1, 2, 1, 24, 16, "odd"), (2100, 21, 1, 40, 32, "dense")])
@pytest.mark.parametrize("norm,interleaved", [("rms", False), ("layer", True), (None, True), ("rms", True), ("layer", False)])
def test_norm_rope(dtype, T, Hq, Hk, D, R, layout, norm, interleaved):
    g = gen(T + D)
    q, k = rows_case(g, T, Hq, D, dtype, layout), rows_case(g, T, Hk, D, dtype, layout)
    q[0, 0] = 0
    table = None if R is None else ref.angles(500, R, "cuda")
    pos = None if R is None else torch.randint(0, 500, (T,), generator=g, device="cuda", dtype=torch.int32)
    qw = rand(g, D, dtype=dtype) if norm else None
    kw = rand(g, D) if norm else None
    kb = rand(g, D) if norm == "layer" else None
    qo, ko = qk_norm_rope(q, k, pos, table, q_norm=norm, k_norm=norm, q_weight=qw, k_weight=kw, k_bias=kb, eps=1e-5,
                          interleaved=interleaved)
    ref.check_dense(qo, *ref.head_rows(q, norm, qw, None, 1e-5, pos, table, interleaved), "q")
    ref.check_dense(ko, *ref.head_rows(k, norm, kw, kb, 1e-5, pos, table, interleaved), "k")


@pytest.mark.parametrize("dtype", DT)
def test_in_place_and_out(dtype):
    g = gen(1)
    qkv = rand(g, 50, 12, 128, dtype=dtype)
    table, pos = ref.angles(64, 64, "cuda"), torch.arange(50, device="cuda", dtype=torch.int32)
    q, k = qkv[:, :8], qkv[:, 8:10]
    want = [ref.head_rows(x, "rms", positions=pos, cos_sin=table) for x in (q, k)]
    rest = qkv[:, 10:].clone()
    a, b = qk_norm_rope(q, k, pos, table, q_out=q, k_out=k)
    assert a.data_ptr() == q.data_ptr() and b.data_ptr() == k.data_ptr()
    ref.check_dense(q, *want[0], "q")
    ref.check_dense(k, *want[1], "k")
    assert torch.equal(qkv[:, 10:], rest)


def test_far_values():
    """Large means, tiny and huge magnitudes, NaN and infinities stay in their rows."""
    x = rand(gen(2), 6, 1, 128)
    x[0] += 1000.0
    x[1] *= 1e-18
    x[2] *= 1e15
    x[3, 0, 5] = float("nan")
    x[4, 0, 7] = float("inf")
    y, _ = qk_norm_rope(x, None, None, None, q_norm="layer")
    want, bound = ref.head_rows(x[[0, 1, 2, 5]], "layer")
    ref.check_dense(y[[0, 1, 2, 5]], want, bound)
    assert bool(y[3].isnan().all()) and bool(y[4].isnan().all())


def test_position_beyond_the_table():
    g = gen(3)
    q = rand(g, 4, 2, 64, dtype=torch.bfloat16)
    table = ref.angles(10, 32, "cuda")
    pos = torch.tensor([0, 10, -1, 9], device="cuda", dtype=torch.int32)
    y, _ = qk_norm_rope(q, None, pos, table, q_norm=None)
    assert take_status() == _native.ST_BAD_INDEX
    good = torch.tensor([0, 3], device="cuda")
    ref.check_dense(y[good], *ref.head_rows(q[good], positions=pos[good], cos_sin=table))
    assert bool(y[1:3, :, :32].isnan().all()) and torch.equal(y[1:3, :, 32:], q[1:3, :, 32:])


def empty_cache(rows, H, D, layout="dense"):
    if layout == "dense":
        return torch.zeros(rows, H, D, device="cuda", dtype=torch.uint8).view(FP8), torch.full((rows, H), -1.0, device="cuda")
    if layout == "pair":  # keys and values side by side, scales in another order
        return (torch.zeros(rows, H, 2, D, device="cuda", dtype=torch.uint8)[:, :, 1].view(FP8),
                torch.full((H, rows), -1.0, device="cuda").t())
    return (torch.zeros(rows * H * D + 1, device="cuda", dtype=torch.uint8)[1:].view(rows, H, D).view(FP8),
            torch.full((rows, H), -1.0, device="cuda"))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,H,D,layout", [(1, 1, 128, "dense"), (1, 8, 64, "pair"), (37, 3, 80, "dense"), (5, 2, 256, "odd"),
                                          (700, 8, 128, "pair"), (9000, 5, 128, "dense"), (3, 1, 8, "odd")])
def test_cache_write_and_read(dtype, T, H, D, layout):
    g = gen(T)
    k, v = rand(g, T, H, D, dtype=dtype, scale=3.0), rows_case(g, T, H, D, dtype, "slice")
    rows = 2 * T + 5
    (kc, ks), (vc, vs) = empty_cache(rows, H, D, layout), empty_cache(rows, H, D)
    slots = torch.randperm(rows, generator=g, device="cuda")[:T].to(torch.int32)
    if T > 2:
        slots[1] = -1
        k[0, 0] = 0
    cache_write(k, slots, kc, ks, v, vc, vs)
    on = slots >= 0
    at = slots[on].long()
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        y, e = ref.head_rows(x[on])
        ref.check_quantised(c.view(torch.uint8)[at].view(FP8), s[at], y, e * 0)
        left = torch.ones(rows, dtype=torch.bool, device="cuda")
        left[at] = False
        assert bool((s[left] == -1.0).all()) and int(c.view(torch.uint8)[left].max()) == 0
    # back: every row, some twice, some none
    ask = torch.cat([slots, slots[:1], torch.tensor([-1], device="cuda", dtype=torch.int32)])
    for out_dtype in DT:
        got = cache_read(kc, ks, ask, dtype=out_dtype)
        want = ref.cache_values(kc.view(torch.uint8)[ask.long().clamp_min(0)].view(FP8), ks[ask.long().clamp_min(0)])
        want[ask < 0] = 0
        ref.check_dense(got, want, want.abs() * ref.U32)


def test_quantised_values_at_the_edges():
    """Rows of zeros, tiny ones, infinities, NaN; halves go to even; the largest becomes 448 exactly."""
    x = torch.zeros(8, 1, 16, device="cuda")
    x[1] = 1e-35
    x[2, 0, 3] = float("inf")
    x[2, 0, 4] = -2.0
    x[3, 0, 0], x[3, 0, 1] = float("nan"), 1.0
    x[4, 0] = torch.tensor([448.0, 17.0, 19.0, -17.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11, 0.5, -448, 240, 248, 9.5, 1, 2, 3, 4])
    x[5] = 3e38
    x[6, 0, 2] = -float("inf")
    c, s = empty_cache(8, 1, 16)
    cache_write(x, torch.arange(8, device="cuda", dtype=torch.int32), c, s)
    f = c.float()[:, 0]
    assert bool((s > 0).all()) and bool(s.isfinite().all())
    assert bool((f[0] == 0).all()) and bool((f[1] == 0).all())
    assert f[2, 3] == 448 and f[2, 4] == -448 and s[2, 0] == torch.tensor(2.0) / 448
    assert bool(f[3, 0].isnan()) and f[3, 1] == 448
    want = torch.tensor([448, 16, 20, -16, 0, 2.0 ** -8, 0, 0.5, -448, 240, 256, 9, 1, 2, 3, 4], device="cuda")
    want[11] = 10.0  # 9.5 lies halfway between 9 and 10: to the even code
    assert torch.equal(f[4], want), f[4]
    assert s[4, 0] == 1.0
    assert bool((f[5] == 448).all()) and f[6, 2] == -448 and bool((f[7] == 0).all())
    back = cache_read(c, s, torch.tensor([[3, 5]], device="cuda", dtype=torch.int32), dtype=torch.float32)
    assert bool(back[0, 0, 0, 0].isnan()) and bool(back[0, 1].isfinite().all())


def test_slots_beyond_the_cache():
    g = gen(4)
    x = rand(g, 6, 2, 64, dtype=torch.bfloat16)
    c, s = empty_cache(10, 2, 64)
    guard = torch.zeros(12, 2, 64, device="cuda", dtype=torch.uint8)
    inner, sc = guard[1:11].view(FP8), torch.zeros(12, 2, device="cuda")
    slots = torch.tensor([9, 10, 2147483647, -2147483648, -1, 0], device="cuda", dtype=torch.int32)
    cache_write(x, slots, inner, sc[1:11])
    assert take_status() == _native.ST_BAD_INDEX
    assert int(guard[0].max()) == 0 and int(guard[11].max()) == 0 and int(guard[2:10].max()) == 0
    assert float(sc[0].abs().max()) == 0 and float(sc[11].abs().max()) == 0
    ref.check_quantised(inner[[9, 0]], sc[1:11][[9, 0]], x[[0, 5]].double(), x[[0, 5]].double() * 0)
    ask = torch.tensor([[9, 10], [-1, 0]], device="cuda", dtype=torch.int32)
    got = cache_read(inner, sc[1:11], ask, offsets=torch.tensor([0, 9], device="cuda", dtype=torch.int32), dtype=torch.float32)
    assert take_status() == _native.ST_BAD_INDEX
    assert torch.equal(got[0, 0], got[1, 1]) and bool((got[0, 1] == 0).all()) and bool((got[1, 0] == 0).all())
    assert float(got[0, 0].abs().max()) > 0
    # an offset that takes an entry below zero
    got = cache_read(inner, sc[1:11], ask, offsets=torch.tensor([-20, -1], device="cuda", dtype=torch.int32))
    assert take_status() == _native.ST_BAD_INDEX and bool((got == 0).all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,H,R,interleaved", [(1, 64, 64, False), (5, 7, 128, True), (130, 64, 64, True), (700, 16, 32, False)])
def test_indexer_qk_write(dtype, T, H, R, interleaved):
    g = gen(T)
    q, k = rand(g, T, H, 128, dtype=dtype), rows_case(g, T, 1, 128, dtype, "slice")[:, 0]
    w = rand(g, T, H)
    kw, kb = rand(g, 128), rand(g, 128, scale=0.1)
    table = ref.angles(900, R, "cuda")
    pos = torch.randint(0, 900, (T,), generator=g, device="cuda", dtype=torch.int32)
    cache, scale = empty_cache(3 * 400, 1, 128)
    cache, scale = cache.view(3, 400, 128), scale.view(3, 400)
    slots = torch.randperm(1200, generator=g, device="cuda")[:T].to(torch.int32)
    q8, w8 = indexer_qk_write(q, k, w, pos, table, slots, cache, scale, k_weight=kw, k_bias=kb, interleaved=interleaved)
    y, e = ref.head_rows(q, positions=pos, cos_sin=table, interleaved=interleaved)
    # (w8 / w is the row's scale, with the rounding of the product)
    ref.check_quantised(q8, w8.double() / w.double(), y, e + U(y))
    y, e = ref.head_rows(k.unsqueeze(1), "layer", kw, kb, 1e-6, pos, table, interleaved)
    at = slots.long()
    ref.check_quantised(cache.view(-1, 1, 128).view(torch.uint8)[at].view(FP8), scale.view(-1, 1)[at], y, e)


def U(y):
    return 4 * ref.U32 * y.abs().amax(-1, keepdim=True)


@pytest.mark.parametrize("T", [1, 40, 900])
def test_one_launch_is_the_two_calls(T):
    g = gen(T)
    q, k, v = (rand(g, T, h, 128, dtype=torch.bfloat16) for h in (16, 4, 4))
    table, pos = ref.angles(1000, 128, "cuda"), torch.arange(T, device="cuda", dtype=torch.int32)
    slots = torch.randperm(T + 9, generator=g, device="cuda")[:T].to(torch.int32)
    qw = rand(g, 128)
    a = [empty_cache(T + 9, 4, 128) for _ in range(4)]
    qo = qkv_norm_rope_write(q, k, v, pos, table, slots, *a[0], *a[1], q_weight=qw, k_weight=qw)
    want, _ = qk_norm_rope(q, None, pos, table, q_weight=qw)
    k32, _ = qk_norm_rope(k.float(), None, pos, table, q_weight=qw)
    cache_write(k32, slots, *a[2])
    cache_write(v, slots, *a[3])
    assert torch.equal(qo, want)
    for x, y in ((a[0], a[2]), (a[1], a[3])):
        assert torch.equal(x[0].view(torch.uint8), y[0].view(torch.uint8)) and torch.equal(x[1], y[1])


def test_offsets_beyond_32_bits():
    """Rows of a cache of more than 2^32 bytes, and of its scales."""
    rows = (1 << 32) // 256 + 100
    cache = torch.empty(rows, 2, 128, device="cuda", dtype=torch.uint8).view(FP8)
    scale = torch.empty(rows, 2, device="cuda")
    x = rand(gen(5), 4, 2, 128, dtype=torch.bfloat16)
    slots = torch.tensor([rows - 1, 0, (1 << 24) + 1, rows - 50], device="cuda", dtype=torch.int32)
    cache_write(x, slots, cache, scale)
    at = slots.long()
    y, e = ref.head_rows(x)
    ref.check_quantised(cache.view(torch.uint8)[at].view(FP8), scale[at], y, e * 0)
    got = cache_read(cache, scale, slots, dtype=torch.float32)
    ref.check_dense(got, ref.cache_values(cache.view(torch.uint8)[at].view(FP8), scale[at]), y.abs() * 2 * ref.U32)


def test_streams_and_graphs():
    """A captured call replays on new contents, on a stream of its own, beside an eager one."""
    g = gen(6)
    T = 64
    q, k = rand(g, T, 64, 128, dtype=torch.bfloat16), rand(g, T, 128, dtype=torch.bfloat16)
    w = rand(g, T, 64)
    table, pos = ref.angles(T, 64, "cuda"), torch.arange(T, device="cuda", dtype=torch.int32)
    (c1, s1), (c2, s2) = empty_cache(T, 1, 128), empty_cache(T, 1, 128)
    args = lambda c, s: (q, k, w, pos, table, pos, c.view(T, 128), s.view(T))  # noqa: E731
    indexer_qk_write(*args(c1, s1))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        q8, w8 = indexer_qk_write(*args(c1, s1))
    q.copy_(rand(g, T, 64, 128, dtype=torch.bfloat16))
    k.copy_(rand(g, T, 128, dtype=torch.bfloat16))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.replay()
    e8, ew = indexer_qk_write(*args(c2, s2))
    torch.cuda.synchronize()
    assert torch.equal(q8.view(torch.uint8), e8.view(torch.uint8)) and torch.equal(w8, ew)
    assert torch.equal(c1.view(torch.uint8), c2.view(torch.uint8)) and torch.equal(s1, s2)


def test_empty_calls():
    z = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16)
    none = torch.empty(0, device="cuda", dtype=torch.int32)
    a, b = qk_norm_rope(z, z, none, ref.angles(4, 64, "cuda"))
    assert a.shape == z.shape and b.shape == z.shape
    c, s = empty_cache(4, 4, 64)
    cache_write(z, none, c, s)
    assert cache_read(c, s, none).shape == (0, 4, 64)
    assert cache_read(c, s, torch.empty(3, 0, device="cuda", dtype=torch.int32)).shape == (3, 0, 4, 64)


@pytest.mark.parametrize("D", [8, 16, 24, 40])
def test_many_short_rows(D):
    """Heads of fewer channels than an item has rows: every row's scale is written."""
    g = gen(D)
    T, H = 9000, 5
    x = rand(g, T, H, D, dtype=torch.bfloat16)
    c, s = empty_cache(T, H, D)
    cache_write(x, torch.arange(T, device="cuda", dtype=torch.int32), c, s)
    y, e = ref.head_rows(x)
    ref.check_quantised(c, s, y, e * 0)
    w = torch.rand(T, H, generator=g, device="cuda")
    kc, ks = empty_cache(T, 1, D)
    q8, w8 = indexer_qk_write(x, x[:, 0], w, None, None, torch.arange(T, device="cuda", dtype=torch.int32), kc[:, 0], ks[:, 0].contiguous(),
                              k_norm=None)
    ref.check_quantised(q8, w8.double() / w.double(), y, e * 0 + U(y))
