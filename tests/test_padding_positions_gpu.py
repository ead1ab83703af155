"""Padding tokens (slot -1) have no position: whatever stands in its place is not an error, and the other tokens' results are those
of a call without them."""
import pytest
import torch

import rows_ref as ref
from jit_kernel import _native
from jit_kernel.norm_rope import indexer_qk_write, qk_norm_rope, qkv_norm_rope_write
from test_norm_rope_gpu import empty_cache, gen, rand, status, take_status  # noqa: F401

pytestmark = pytest.mark.gpu


def batch(T, rows, R):
    """Tokens whose every third, and last, is padding with a position outside the table."""
    g = gen(T)
    pos = torch.randint(0, rows, (T,), generator=g, device="cuda", dtype=torch.int32)
    slots = torch.randperm(2 * T, generator=g, device="cuda")[:T].to(torch.int32)
    pad = torch.zeros(T, dtype=torch.bool, device="cuda")
    pad[1::3] = True
    pad[T - 1] = True
    slots[pad] = -1
    wild = pos.clone()
    wild[pad] = -1
    wild[T - 1] = rows
    return g, ref.angles(rows, R, "cuda"), wild, slots, pad


@pytest.mark.parametrize("T", [2, 50, 3000])
@pytest.mark.parametrize("interleaved", [False, True])
def test_indexer_qk_write(T, interleaved):
    g, table, pos, slots, pad = batch(T, 700, 64)
    q, k, w = rand(g, T, 64, 128, dtype=torch.bfloat16), rand(g, T, 128, dtype=torch.bfloat16), rand(g, T, 64)
    (c, s), (c1, s1) = empty_cache(2 * T, 1, 128), empty_cache(2 * T, 1, 128)
    q8, w8 = indexer_qk_write(q, k, w, pos, table, slots, c[:, 0], s[:, 0], interleaved=interleaved)
    assert take_status() == 0
    on = ~pad
    r8, v8 = indexer_qk_write(q[on], k[on], w[on], pos[on], table, slots[on], c1[:, 0], s1[:, 0], interleaved=interleaved)
    assert torch.equal(q8.view(torch.uint8)[on], r8.view(torch.uint8)) and torch.equal(w8[on], v8)
    assert torch.equal(c.view(torch.uint8), c1.view(torch.uint8)) and torch.equal(s, s1)


@pytest.mark.parametrize("T", [2, 50, 3000])
def test_qkv_norm_rope_write(T):
    g, table, pos, slots, pad = batch(T, 700, 128)
    q, k, v = (rand(g, T, h, 128, dtype=torch.bfloat16) for h in (16, 2, 2))
    caches, others = ([empty_cache(2 * T, 2, 128) for _ in range(2)] for _ in range(2))
    out = qkv_norm_rope_write(q, k, v, pos, table, slots, *caches[0], *caches[1])
    assert take_status() == 0
    on = ~pad
    want = qkv_norm_rope_write(q[on], k[on], v[on], pos[on], table, slots[on], *others[0], *others[1])
    assert torch.equal(out[on], want)
    for (c, s), (c1, s1) in zip(caches, others):
        assert torch.equal(c.view(torch.uint8), c1.view(torch.uint8)) and torch.equal(s, s1)


def test_the_others_are_still_told():
    """A token that is written, and one of a call without slots, needs a position of the table."""
    T = 40
    g, table, pos, slots, pad = batch(T, 700, 128)
    q, k, v = (rand(g, T, h, 128, dtype=torch.bfloat16) for h in (16, 2, 2))
    caches = [empty_cache(2 * T, 2, 128) for _ in range(2)]
    qk_norm_rope(q, k, pos, table)
    assert take_status() == _native.ST_BAD_INDEX
    pos[0] = 700
    qkv_norm_rope_write(q, k, v, pos, table, slots, *caches[0], *caches[1])
    assert take_status() == _native.ST_BAD_INDEX
