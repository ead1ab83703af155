"""Requests of text and images decoded over a paged fp8 cache: rotation by several axes as the rows are written, attention that adds up
the rows' weights, eviction to other pages, and on from there - eager, and with the step captured into a graph."""
import pytest
import torch

import paged_ref as paged
import rows_ref as ref
from jit_kernel.kv_cache import cache_evict
from jit_kernel.norm_rope import qkv_norm_rope_write, rotary_axes
from jit_kernel.paged_attention import paged_attention
from jit_kernel.topk_indexer import _status_word, kernel_status

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
B, Hq, Hk, D, PAGE, COLS = 3, 8, 2, 128, 16, 6
BUDGET, RECENT, SINKS = 32, 8, 2


@pytest.fixture(autouse=True)
def status():
    if torch.cuda.is_available():
        _status_word(torch.device("cuda", 0)).zero_()
    yield
    if torch.cuda.is_available():
        assert kernel_status() == 0


def slot_of(table, position):
    """The cache rows of one position of each sequence"""
    return (table[torch.arange(B, device="cuda"), (position // PAGE).long()] * PAGE + position % PAGE).to(torch.int32)


@pytest.mark.parametrize("captured", [False, True])
def test_decode(captured):
    g = torch.Generator(device="cuda").manual_seed(3)
    pages = 2 * B * COLS
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = order[:B * COLS].view(B, COLS).clone()
    spare = order[B * COLS:].view(B, COLS)
    kc, vc = (torch.zeros(pages * PAGE, Hk, D, device="cuda", dtype=torch.uint8).view(FP8) for _ in range(2))
    ks, vs = (torch.zeros(pages * PAGE, Hk, device="cuda") for _ in range(2))
    weight = torch.zeros(B, Hk, COLS * PAGE, device="cuda")
    cos_sin, axes = ref.angles(400, D, "cuda"), rotary_axes((24, 20, 20), interleaved=True)

    def activations(T):
        return [torch.randn(T, h, D, generator=g, device="cuda").to(torch.bfloat16) for h in (Hq, Hk, Hk)]

    # prompts: text, then a piece of an image (rows of seven patches)
    start = torch.tensor([70, 33, 5], device="cuda", dtype=torch.int32)
    for b in range(B):
        n = int(start[b])
        i = torch.arange(n, device="cuda", dtype=torch.int32)
        pos = torch.stack([i.clamp_max(20), torch.where(i > 20, 20 + (i - 20) // 7, i), torch.where(i > 20, 20 + (i - 20) % 7, i)])
        slots = (table[b, (i // PAGE).long()] * PAGE + i % PAGE).to(torch.int32)
        q, k, v = activations(n)
        qkv_norm_rope_write(q, k, v, pos, cos_sin, slots, kc, ks, vc, vs, axes=axes)

    # a decode step's inputs and outputs have places of their own: a graph is replayed on them
    q, k, v = activations(B)
    lengths, text = start.clone(), torch.tensor([100, 60, 5], device="cuda", dtype=torch.int32)
    out, lse = torch.empty(B, Hq, D, device="cuda", dtype=torch.bfloat16), torch.empty(B, Hq, device="cuda")

    def step():
        slots = slot_of(table, lengths)
        lengths.add_(1)
        qr = qkv_norm_rope_write(q, k, v, text.expand(3, B), cos_sin, slots, kc, ks, vc, vs, axes=axes)
        o, l = paged_attention(qr, kc, vc, table, lengths, page_size=PAGE, k_scale=ks, v_scale=vs, weight=weight, return_lse=True)
        out.copy_(o)
        lse.copy_(l)
        text.add_(1)
        return qr

    def evict():
        return cache_evict(kc, vc, weight, table, lengths, spare, page_size=PAGE, budget=BUDGET, recent=RECENT, sinks=SINKS, k_scale=ks, v_scale=vs)

    run = step
    if captured:
        keep = [x.clone() for x in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs, weight, lengths, text)]
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            qr = step()
        for x, y in zip((kc.view(torch.uint8), vc.view(torch.uint8), ks, vs, weight, lengths, text), keep):
            x.copy_(y)

        def run():
            graph.replay()
            return qr

    for i in range(9):
        if i in (3, 6):
            before = [x.clone() for x in (kc, vc, ks, vs)]
            kept, left, after = paged.evict(weight, lengths, BUDGET, RECENT, SINKS)
            got = evict()
            assert torch.equal(got[0].cpu(), kept) and torch.equal(got[1].cpu(), left) and torch.equal(got[2].cpu(), after)
            for x, y in zip((kc, vc, ks, vs), before):
                want = paged.move(y, kept, table, spare, PAGE)
                assert torch.equal(x.view(torch.uint8), want.view(torch.uint8))
            # (the old pages are the spare ones now)
            old = table.clone()
            table.copy_(spare)
            spare.copy_(old)
            lengths.copy_(got[1])
            weight.copy_(got[2])
        for x, y in zip((q, k, v), activations(B)):
            x.copy_(y)
        had, n = weight.clone(), lengths + 1
        rotated = run()
        assert torch.equal(lengths, n)
        want, at = paged.attention(rotated, kc, vc, table, lengths, PAGE, None, ks, vs)
        ref.check_attention(out, lse, want, f"step {i}")
        w, e = paged.weights(rotated, kc, at, want, None, ks)
        m = w.size(2)
        off = (weight[..., :m].double() - had[..., :m].double() - w).abs()
        assert bool((off <= e + 2 * ref.U32 * (had[..., :m].double() + w)).all()) and torch.equal(weight[..., m:], had[..., m:])
        # (a token's weights are shares of its sequence's group: they add up to the group's size)
        assert bool(((w.sum(2) - Hq // Hk).abs() < 1e-9).all())
    assert int(lengths.max()) == BUDGET + 3
