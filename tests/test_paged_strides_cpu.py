"""Slots of a cache whose distance does not fit the kernels' 32-bit strides: refused before anything is enqueued, whether the call asks for its workspace
or runs. No device is needed, and the pointers named here are never followed."""
import ctypes

import pytest

from jit_kernel import _native
from jit_kernel.paged_attention import _ARGS
from test_paged_overlap_cpu import A, CALL, FAR, attend, evict

ERANGE = -4
CODES = dict(k_scale=A + 6 * FAR, kss=2, ksh=1, v_scale=A + 7 * FAR, vss=2, vsh=1)

# (2^32 bytes and more between two slots, and slots one in front of the other)
FAR_SLOTS = [(2, x) for x in (1 << 31, (1 << 31) + 8, 1 << 40, -128, -(1 << 33))] + [(1, x) for x in (1 << 32, (1 << 32) + 16, 1 << 40, -128, -(1 << 33))]


@pytest.mark.parametrize("which", ["ks", "vs"])
@pytest.mark.parametrize("elem,stride", FAR_SLOTS)
@pytest.mark.parametrize("slots", [2, 100])
def test_attention(slots, elem, stride, which):
    call = {"slots": slots, which: stride, **(CODES if elem == 1 else {})}
    assert attend(**call) == ERANGE
    n = ctypes.c_size_t(7)
    assert _native.lib().fftopk_paged_workspace_bytes(_ARGS.pack(*{**CALL, **call}.values()), ctypes.byref(n)) == ERANGE and n.value == 0


@pytest.mark.parametrize("which", ["ks", "vs"])
@pytest.mark.parametrize("elem,stride", FAR_SLOTS)
@pytest.mark.parametrize("slots", [2, 100])
def test_evict(slots, elem, stride, which):
    assert evict(**{"slots": slots, "elem": elem, which: stride, **(CODES if elem == 1 else {})}) == ERANGE
