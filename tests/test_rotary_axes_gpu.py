"""Rotation by positions with several axes against a 64-bit statement of it, and against the one-position ops where the axes agree."""
import pytest
import torch

import rows_ref as ref
from jit_kernel import _native
from jit_kernel.norm_rope import indexer_qk_write, qk_norm_rope, qkv_norm_rope_write, rotary_axes
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


def head_rows(x, norm, weight, bias, eps, positions, table, axes, interleaved):
    """ref.head_rows with a table row per token: the cosine and sine of every pair from its axis' row"""
    R = table.size(1)
    i = torch.arange(R // 2, device=x.device)
    at = positions[torch.tensor(axes, device=x.device)].long()  # [pairs, tokens]
    own = torch.cat([table[at, i.unsqueeze(1)].t(), table[at, (i + R // 2).unsqueeze(1)].t()], 1)
    return ref.head_rows(x, norm, weight, bias, eps, torch.arange(x.size(0), device=x.device), own, interleaved)


def make_axes(kind, pairs, n):
    if kind == "turn":
        return rotary_axes([pairs // n + (a < pairs % n) for a in range(n)], interleaved=True)
    if kind == "blocks":
        return rotary_axes([pairs // n + (a < pairs % n) for a in range(n)])
    return tuple((i * i + 3 * i // 5) % n for i in range(pairs))  # in no order


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,Hq,Hk,D,R,odd", [(1, 1, 1, 16, 16, False), (1, 64, 8, 128, 128, False), (17, 7, 3, 80, 48, False), (5, 4, 1, 96, 16, True),
                                             (33, 9, 5, 256, 256, False), (1300, 33, 4, 128, 64, False), (2100, 21, 1, 40, 32, False)])
@pytest.mark.parametrize("kind,n,norm,interleaved", [("turn", 3, "rms", False), ("blocks", 3, "layer", True), ("none", 4, None, False), ("blocks", 2, "rms", False),
                                                     ("turn", 4, "rms", True), ("blocks", 1, None, False)])
def test_axes(dtype, T, Hq, Hk, D, R, odd, kind, n, norm, interleaved):
    g = gen(T + D + n)
    flat = rand(g, T * (Hq + Hk + 1) * D + odd, dtype=dtype)[int(odd):].view(T, Hq + Hk + 1, D)
    q, k = flat[:, :Hq], flat[:, Hq:Hq + Hk]
    table = ref.angles(700, R, "cuda")
    wide = torch.randint(0, 700, (n, T + 3), generator=g, device="cuda", dtype=torch.int32)
    pos = wide[:, 2:T + 2]
    axes = make_axes(kind, R // 2, n)
    qw = rand(g, D, dtype=dtype) if norm else None
    kb = rand(g, D) if norm == "layer" else None
    qo, ko = qk_norm_rope(q, k, pos, table, axes=axes, q_norm=norm, k_norm=norm, q_weight=qw, k_bias=kb, eps=1e-5, interleaved=interleaved)
    ref.check_dense(qo, *head_rows(q, norm, qw, None, 1e-5, pos, table, axes, interleaved), "q")
    ref.check_dense(ko, *head_rows(k, norm, None, kb, 1e-5, pos, table, axes, interleaved), "k")


@pytest.mark.parametrize("T", [3, 2000])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes_that_agree(T, interleaved):
    """Text tokens, whose axes are all at the same position, and the writing ops: the same bits as with one position."""
    g = gen(T)
    qkv = rand(g, T, 20, 128, dtype=torch.bfloat16)
    q, k, v = qkv[:, :16], qkv[:, 16:18], qkv[:, 18:]
    table, one = ref.angles(3000, 128, "cuda"), torch.randint(0, 3000, (T,), generator=g, device="cuda", dtype=torch.int32)
    three, axes = one.expand(3, T), rotary_axes((16, 24, 24))
    slots = torch.randperm(T + 5, generator=g, device="cuda")[:T].to(torch.int32)
    slots[T // 2] = -1

    def caches(H):
        return torch.zeros(T + 5, H, 128, device="cuda", dtype=torch.uint8).view(FP8), torch.zeros(T + 5, H, device="cuda")

    got = []
    for pos, kw in ((one, {}), (three, dict(axes=axes))):
        (kc, ks), (vc, vs), (ic, is_) = caches(2), caches(2), caches(1)
        a = qkv_norm_rope_write(q, k, v, pos, table, slots, kc, ks, vc, vs, interleaved=interleaved, **kw)
        b, w = indexer_qk_write(q, k[:, 0].contiguous(), torch.ones(T, 16, device="cuda"), pos, table, slots, ic[:, 0], is_[:, 0].contiguous(),
                                interleaved=interleaved, **kw)
        got.append([a, b.view(torch.uint8), w] + [x.view(torch.uint8) if x.dtype is FP8 else x for x in (kc, ks, vc, vs, ic)])
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_quantised_writes():
    g = gen(3)
    T, axes = 70, make_axes("turn", 32, 3)
    q, k, v = (rand(g, T, h, 128, dtype=torch.float16) for h in (8, 2, 2))
    table, pos = ref.angles(100, 64, "cuda"), torch.randint(0, 100, (3, T), generator=g, device="cuda", dtype=torch.int32)
    kc, vc = (torch.zeros(T, 2, 128, device="cuda", dtype=torch.uint8).view(FP8) for _ in range(2))
    ks, vs = (torch.zeros(T, 2, device="cuda") for _ in range(2))
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    qo = qkv_norm_rope_write(q, k, v, pos, table, slots, kc, ks, vc, vs, axes=axes)
    ref.check_dense(qo, *head_rows(q, "rms", None, None, 1e-6, pos, table, axes, False), "q")
    ref.check_quantised(kc, ks, *head_rows(k, "rms", None, None, 1e-6, pos, table, axes, False), "k")
    ref.check_quantised(vc, vs, *ref.head_rows(v), "v")


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_beyond_the_table(interleaved):
    """One axis out of the table makes its own channels NaN and no others; an axis that no pair turns by may be anything; a padding token's
    positions too."""
    g = gen(4)
    q, table = rand(g, 4, 2, 64, dtype=torch.bfloat16), ref.angles(10, 32, "cuda")
    pos = torch.tensor([[1, 2, 3, 4], [5, 10, -1, 6], [99, -7, 1 << 30, -(1 << 31)]], device="cuda", dtype=torch.int32)
    axes = tuple(i % 2 for i in range(16))
    out, _ = qk_norm_rope(q, None, pos, table, axes=axes, interleaved=interleaved)
    assert take_status() == _native.ST_BAD_INDEX
    bad = torch.zeros(64, dtype=torch.bool)
    for i in range(1, 16, 2):
        bad[[2 * i, 2 * i + 1] if interleaved else [i, i + 16]] = True
    fine = head_rows(q, "rms", None, None, 1e-6, pos.clamp(0, 9), table, axes, interleaved)
    nan = out.isnan().cpu()
    for t in range(4):
        assert bool((nan[t] == (bad if t in (1, 2) else torch.zeros_like(bad))).all())
    ref.check_dense(torch.where(out.isnan(), fine[0].to(out.dtype), out), *fine, "q")
    out, _ = qk_norm_rope(q[::3], None, pos[:, ::3].contiguous(), table, axes=axes, interleaved=interleaved)  # (the third axis only is out)
    assert not bool(out.isnan().any())
    c, s = torch.zeros(8, 2, 64, device="cuda", dtype=torch.uint8).view(FP8), torch.zeros(8, 2, device="cuda")
    slots = torch.tensor([0, -1, -1, 1], device="cuda", dtype=torch.int32)
    qkv_norm_rope_write(q, q, q, pos, table, slots, c, s, c.clone(), s.clone(), axes=axes, interleaved=interleaved)


def test_graph():
    g = gen(5)
    q, table = rand(g, 50, 8, 128, dtype=torch.bfloat16), ref.angles(500, 128, "cuda")
    pos = torch.randint(0, 500, (3, 50), generator=g, device="cuda", dtype=torch.int32)
    axes = list(rotary_axes((24, 20, 20), interleaved=True))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = qk_norm_rope(q, None, pos, table, axes=axes)
    for i in range(3):
        pos.copy_(torch.randint(0, 500, (3, 50), generator=g, device="cuda", dtype=torch.int32))
        graph.replay()
        ref.check_dense(out, *head_rows(q, "rms", None, None, 1e-6, pos, table, axes, False), "q")


def test_refusals():
    q, table = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(10, 32, device="cuda")
    pos, axes = torch.zeros(3, 4, device="cuda", dtype=torch.int32), (0, 1, 2, 0) * 4
    qk_norm_rope(q, None, pos, table, axes=axes)
    for p, c, a in ((pos, table, axes[:-1]), (pos, table, axes + (0,)), (pos, table, (3,) + axes[1:]), (pos, table, (-1,) + axes[1:]),
                    (pos, table, (0.0,) + axes[1:]), (pos[0], table, axes), (pos[:, :3], table, axes), (pos.long(), table, axes), (pos.cpu(), table, axes),
                    (pos.t().contiguous().t(), table, axes), (pos, None, axes), (None, None, axes), (pos, table, None),
                    (torch.zeros(5, 4, device="cuda", dtype=torch.int32), table, axes), (pos[:0], table, axes)):
        with pytest.raises((RuntimeError, AttributeError)):
            qk_norm_rope(q, None, p, c, axes=a)
