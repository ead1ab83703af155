"""Calls of the paged cache's entries that are refused before anything is enqueued: no device is needed, and the pointers named
here are never followed."""
import ctypes

import pytest
import torch

from jit_kernel import _native
from jit_kernel.kv_cache import _EVICT, cache_evict
from jit_kernel.paged_attention import _ARGS, paged_attention

EINVAL, ERANGE = -1, -4
A = 1 << 20  # an aligned address

CALL = dict(q=A, qs=1024, qh=128, k=A, ks=128, kh=128, v=A, vs=128, vh=128, k_scale=0, kss=0, ksh=0, v_scale=0, vss=0, vsh=0, table=A, row=8,
            lengths=A, out=A, os=1024, oh=128, lse=0, w=0, ws=0, wh=0, wo=0, wos=0, woh=0, cols=0, seqs=2, slots=100, q_heads=8, kv_heads=1,
            D=128, pages=8, page_size=16, dtype=1, scale=0.1, reserved=0)


def test_struct_size():
    """The packed arguments have the C struct's size: pointers and 64-bit fields, then eight 32-bit ones."""
    assert _ARGS.size == 31 * 8 + 8 * 4


@pytest.mark.parametrize("want,call", [
    (EINVAL, dict(seqs=-1)), (EINVAL, dict(q_heads=-1)), (EINVAL, dict(kv_heads=-1)), (EINVAL, dict(pages=-1)), (EINVAL, dict(page_size=0)),
    (EINVAL, dict(slots=-1)), (EINVAL, dict(cols=-1)), (EINVAL, dict(dtype=2)), (ERANGE, dict(D=96)), (ERANGE, dict(D=256)),
    (EINVAL, dict(kv_heads=0)), (EINVAL, dict(kv_heads=3)), (EINVAL, dict(k_scale=A)), (EINVAL, dict(v_scale=A)), (EINVAL, dict(q=0)),
    (EINVAL, dict(out=0)), (EINVAL, dict(table=0)), (EINVAL, dict(lengths=0)), (EINVAL, dict(k=0)), (EINVAL, dict(v=0)), (EINVAL, dict(q=A + 8)),
    (EINVAL, dict(k=A + 8)), (EINVAL, dict(v=A + 8)), (EINVAL, dict(qs=1028)), (EINVAL, dict(qh=68)), (EINVAL, dict(ks=132)),
    (EINVAL, dict(vs=132)), (EINVAL, dict(kv_heads=2, kh=68)), (EINVAL, dict(out=A + 1)), (EINVAL, dict(table=A + 2)),
    (EINVAL, dict(lengths=A + 1)), (EINVAL, dict(lse=A + 2)), (EINVAL, dict(k_scale=A + 2, v_scale=A)), (EINVAL, dict(w=A)),
    (EINVAL, dict(wo=A + 2)), (ERANGE, dict(slots=1 << 31)), (ERANGE, dict(seqs=1 << 31)), (0, dict(seqs=0)), (0, dict(q_heads=0))])
def test_paged_attention(want, call):
    blob, n = _ARGS.pack(*{**CALL, **call}.values()), ctypes.c_size_t(7)
    assert _native.lib().fftopk_paged_attention(blob, None, 0, None, None) == want
    assert _native.lib().fftopk_paged_workspace_bytes(blob, ctypes.byref(n)) == want and n.value == 0


@pytest.mark.parametrize("call", [
    dict(os=127), dict(os=0), dict(oh=0), dict(oh=-127), dict(wo=A, cols=8, wos=7), dict(wo=A, cols=8, wos=0), dict(w=A, wo=A, cols=1),
    dict(wo=A, cols=8, wos=16, kv_heads=2, kh=128, woh=7)])
def test_results_on_one_another(call):
    """Broadcast views as results: their rows would hold whichever was written last."""
    assert _native.lib().fftopk_paged_attention(_ARGS.pack(*{**CALL, **call}.values()), None, 0, None, None) == EINVAL


def test_without_arguments():
    n = ctypes.c_size_t()
    assert _native.lib().fftopk_paged_attention(None, None, 0, None, None) == EINVAL
    assert _native.lib().fftopk_paged_workspace_bytes(None, ctypes.byref(n)) == EINVAL
    assert _native.lib().fftopk_paged_workspace_bytes(_ARGS.pack(*CALL.values()), None) == EINVAL


EVICT = dict(k=A, ks=128, kh=128, v=A, vs=128, vh=128, k_scale=0, kss=0, ksh=0, v_scale=0, vss=0, vsh=0, w=A, ws=64, wh=64, wo=2 * A, wos=64,
             woh=64, table=A, row=8, to=A, to_row=8, lengths=A, new=A, kept=A, cols=64, seqs=2, slots=100, heads=1, D=128, elem=2, pages=8,
             to_pages=4, page_size=16, budget=32, recent=4, sinks=4, reserved=0)


@pytest.mark.parametrize("want,call", [
    (EINVAL, dict(seqs=-1)), (EINVAL, dict(heads=-1)), (EINVAL, dict(slots=-1)), (EINVAL, dict(pages=-1)), (EINVAL, dict(to_pages=-1)),
    (EINVAL, dict(page_size=0)), (EINVAL, dict(budget=-1, recent=0, sinks=0)), (EINVAL, dict(recent=-1)), (EINVAL, dict(sinks=-1)), (EINVAL, dict(cols=-1)),
    (EINVAL, dict(recent=29)), (EINVAL, dict(recent=0x7fffffff, sinks=0x7fffffff)), (EINVAL, dict(elem=4)), (EINVAL, dict(elem=0)), (ERANGE, dict(D=4)),
    (ERANGE, dict(D=12)), (ERANGE, dict(D=264)), (EINVAL, dict(k_scale=A)), (EINVAL, dict(v_scale=A)), (EINVAL, dict(lengths=0)), (EINVAL, dict(new=0)),
    (EINVAL, dict(kept=0)), (EINVAL, dict(table=0)), (EINVAL, dict(to=0)), (EINVAL, dict(w=0)), (EINVAL, dict(wo=0)), (EINVAL, dict(wo=A)),
    (EINVAL, dict(k=0)), (EINVAL, dict(v=0)), (EINVAL, dict(k=A + 1)), (EINVAL, dict(v=A + 1)), (EINVAL, dict(w=A + 2)), (EINVAL, dict(kept=A + 2)),
    (EINVAL, dict(table=A + 1)), (EINVAL, dict(to=A + 2)), (EINVAL, dict(lengths=A + 2)), (EINVAL, dict(new=A + 2)), (ERANGE, dict(slots=1 << 31)),
    (ERANGE, dict(seqs=1 << 31)), (ERANGE, dict(seqs=1 << 30, heads=4)), (ERANGE, dict(budget=65)), (ERANGE, dict(pages=0x7fffffff, cols=1 << 31)),
    (ERANGE, dict(seqs=1 << 27, budget=1 << 20, to_pages=1 << 16)), (0, dict(seqs=0)), (0, dict(heads=0))])
def test_cache_evict(want, call):
    assert _native.lib().fftopk_cache_evict(_EVICT.pack(*{**EVICT, **call}.values()), None, None) == want


@pytest.mark.parametrize("call", [
    dict(wos=63), dict(wos=0), dict(heads=2, wos=128, kh=12800, vh=12800, woh=0), dict(heads=2, wos=128, kh=0, vh=12800),
    dict(heads=2, wos=128, kh=12800, vh=127), dict(ks=0), dict(vs=127), dict(k_scale=A, v_scale=A, kss=0, vss=1),
    dict(k_scale=A, v_scale=A, kss=1, vss=0), dict()])
def test_evict_results_on_one_another(call):
    """Broadcast views as results; and (the last) lengths that would be read while the new ones are written."""
    blob = _EVICT.pack(*{**EVICT, "new": 2 * A if call else A, **call}.values())
    assert _native.lib().fftopk_cache_evict(blob, None, None) == EINVAL


def test_evict_without_arguments():
    assert _EVICT.size == 28 * 8 + 10 * 4
    assert _native.lib().fftopk_cache_evict(None, None, None) == EINVAL


def test_cpu_tensors_are_refused():
    x, c, i = torch.zeros(2, 4, 64).half(), torch.zeros(8, 4, 64).half(), torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        paged_attention(x, c, c, i, i[:, 0].contiguous(), page_size=4)
    with pytest.raises(RuntimeError):
        cache_evict(c, c, torch.zeros(2, 4, 8), i, i[:, 0].contiguous(), i, page_size=4, budget=4)
