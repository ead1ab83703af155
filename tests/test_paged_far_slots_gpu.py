"""Caches whose slots lie as far from one another as strides of 32 bits reach, and lone slots, whose stride says nothing."""
import pytest
import torch

import paged_ref as paged
import rows_ref as ref
from jit_kernel.kv_cache import cache_evict
from jit_kernel.paged_attention import paged_attention
from jit_kernel.topk_indexer import _status_word, kernel_status
from test_cache_evict_gpu import bits
from test_paged_attention_gpu import gen, make_cache, rand

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def status():
    if torch.cuda.is_available():
        _status_word(torch.device("cuda", 0)).zero_()
    yield
    if torch.cuda.is_available():
        assert kernel_status() == 0


@pytest.mark.parametrize("dtype", [FP8, torch.bfloat16])
def test_a_lone_slot_has_no_stride(dtype):
    """Its row is read where it is, whatever the stride says."""
    g = gen(4)
    q = rand(g, 2, 4, 64, dtype=torch.bfloat16)
    k, ks = make_cache(g, 1, 2, 64, torch.bfloat16, dtype is FP8)
    v, vs = make_cache(g, 1, 2, 64, torch.bfloat16, dtype is FP8)
    far = [torch.as_strided(x, (1, 2, 64), (1 << 33, 64, 1)) for x in (k, v)]
    t, n = torch.zeros(2, 1, device="cuda", dtype=torch.int32), torch.tensor([1, 0], device="cuda", dtype=torch.int32)
    out, lse = paged_attention(q, *far, t, n, page_size=1, k_scale=ks, v_scale=vs, return_lse=True)
    want, _ = paged.attention(q, k, v, t, n, 1, None, ks, vs)
    ref.check_attention(out, lse, want)
    assert bool((out[0] != 0).any())


@pytest.mark.parametrize("fp8", [False, True])
def test_slots_nearly_four_gigabytes_apart(fp8):
    """The longest strides that are taken, over rows of both slots."""
    g = gen(5)
    H, D = 2, 64
    stride = (1 << 32) - 16 if fp8 else (1 << 31) - 8
    c, s = make_cache(g, 2, H, D, torch.bfloat16, fp8)
    buffer = torch.empty(stride + H * D, device="cuda", dtype=torch.uint8 if fp8 else torch.bfloat16)
    for i in range(2):
        buffer[i * stride:i * stride + H * D] = (c.view(torch.uint8) if fp8 else c)[i].reshape(-1)
    far = torch.as_strided(buffer, (2, H, D), (stride, D, 1)).view(c.dtype)
    q = rand(g, 2, 8, D, dtype=torch.bfloat16, scale=2.0)
    for page, table, lens in ((1, [[1, 0], [1, 1]], [2, 1]), (32, [[0], [0]], [2, 1])):
        t, n = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in (table, lens))
        out, lse = paged_attention(q, far, far, t, n, page_size=page, k_scale=s, v_scale=s, return_lse=True)
        want, _ = paged.attention(q, c, c, t, n, page, None, s, s)
        ref.check_attention(out, lse, want)
    # eviction: the row of slot 0 to slot 1
    w, n = torch.ones(1, H, 1, device="cuda"), torch.ones(1, device="cuda", dtype=torch.int32)
    t, to = (torch.full((1, 1), i, device="cuda", dtype=torch.int32) for i in (0, 1))
    scales = [s.clone(), s.clone()] if fp8 else [None, None]
    cache_evict(far, far, w, t, n, to, page_size=1, budget=1, k_scale=scales[0], v_scale=scales[1])
    for i in range(2):
        assert torch.equal(buffer[i * stride:i * stride + H * D], bits(c[0]).view(buffer.dtype).reshape(-1))
    assert not fp8 or all(torch.equal(x, s[:1].expand(2, -1)) for x in scales)
