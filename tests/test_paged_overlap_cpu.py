"""Results of the paged cache's entries whose rows lie on one another in ways that no single stride shows: refused before anything is enqueued.
No device is needed, and the pointers named here are never followed."""
import ctypes
import itertools
import subprocess
from pathlib import Path

import pytest
from hypothesis import given, settings, strategies as st

from jit_kernel import _native
from jit_kernel.kv_cache import _EVICT
from jit_kernel.paged_attention import _ARGS

EINVAL = -1
A = 1 << 20  # an aligned address; the arrays named here lie 2^40 bytes from one another
FAR = 1 << 40
CSRC = Path(__file__).resolve().parent.parent / "flash-float-jit-kernels_b200" / "csrc"

CALL = dict(q=A, qs=1024, qh=128, k=A + FAR, ks=256, kh=128, v=A + 2 * FAR, vs=256, vh=128, k_scale=0, kss=0, ksh=0, v_scale=0, vss=0, vsh=0,
            table=A + 3 * FAR, row=8, lengths=A + 4 * FAR, out=A + 5 * FAR, os=1024, oh=128, lse=0, w=0, ws=0, wh=0, wo=0, wos=0, woh=0, cols=0,
            seqs=2, slots=100, q_heads=8, kv_heads=2, D=128, pages=8, page_size=16, dtype=1, scale=0.1, reserved=0)
EVICT = dict(k=A, ks=256, kh=128, v=A + FAR, vs=256, vh=128, k_scale=0, kss=0, ksh=0, v_scale=0, vss=0, vsh=0, w=A + 2 * FAR, ws=128, wh=64,
             wo=A + 3 * FAR, wos=128, woh=64, table=A + 4 * FAR, row=8, to=A + 5 * FAR, to_row=8, lengths=A + 6 * FAR, new=A + 7 * FAR, kept=A + 8 * FAR,
             cols=64, seqs=2, slots=100, heads=2, D=128, elem=2, pages=8, to_pages=4, page_size=16, budget=32, recent=4, sinks=4, reserved=0)


def attend(**call):
    return _native.lib().fftopk_paged_attention(_ARGS.pack(*{**CALL, **call}.values()), None, 0, None, None)


def evict(**call):
    return _native.lib().fftopk_cache_evict(_EVICT.pack(*{**EVICT, **call}.values()), None, None)


# (every stride by itself is a row or more: row 1 of one sequence is row 0 of another, or overlaps it)
@pytest.mark.parametrize("call", [
    dict(os=128, oh=128), dict(os=256, oh=128), dict(os=128, oh=256, seqs=3), dict(os=192, oh=128), dict(os=-128, oh=128), dict(os=896, oh=128),
    dict(os=1000, oh=128), dict(wo=A + 6 * FAR, cols=8, wos=8, woh=8), dict(wo=A + 6 * FAR, cols=8, wos=12, woh=8),
    dict(wo=A + 6 * FAR, cols=8, wos=9, woh=17, seqs=3)])
def test_attention_results_on_one_another(call):
    assert attend(**call) == EINVAL


@pytest.mark.parametrize("call", [
    dict(wos=64, woh=64), dict(wos=100, woh=64), dict(wos=64, woh=96), dict(ks=128, kh=128), dict(vs=128, vh=128), dict(ks=128, kh=200), dict(vs=128, vh=12672),
    dict(k_scale=A + 9 * FAR, v_scale=A + 10 * FAR, kss=1, ksh=1, vss=2, vsh=1), dict(k_scale=A + 9 * FAR, v_scale=A + 10 * FAR, kss=2, ksh=1, vss=1, vsh=1),
    dict(k_scale=A + 9 * FAR, v_scale=A + 10 * FAR, kss=2, ksh=1, vss=1, vsh=99)])
def test_evict_results_on_one_another(call):
    assert evict(**call) == EINVAL


@pytest.fixture(scope="module")
def extents(tmp_path_factory):
    out = tmp_path_factory.mktemp("extents") / "libextents.so"
    source = out.with_suffix(".cpp")
    source.write_text('#include "fftopk_extent.h"\nextern "C" int apart(int64_t a, int64_t b, int64_t c, int64_t d, int64_t w)'
                      " { return fftopk::rows_apart(a, b, c, d, w); }\n")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(out), str(source)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.apart.argtypes = [ctypes.c_int64] * 5
    return lib


def rows(seqs, seq, heads, head, width):
    return [set(range(s * seq + h * head, s * seq + h * head + width)) for s in range(seqs) for h in range(heads)]


@settings(deadline=None, max_examples=2000)
@given(st.integers(0, 6), st.integers(-40, 40), st.integers(0, 6), st.integers(-40, 40), st.integers(1, 9))
def test_rows_apart(extents, seqs, seq, heads, head, width):
    """Against every pair of rows: nothing that lies apart is refused, interleaved views included."""
    want = all(not x & y for x, y in itertools.combinations(rows(seqs, seq, heads, head, width), 2))
    assert bool(extents.apart(seqs, seq, heads, head, width)) == want


def test_rows_apart_at_large_sizes(extents):
    big = (1 << 63) - 1
    assert extents.apart(1 << 31, 1024, 8, 128, 128) and extents.apart(1 << 31, 128, 8, 1 << 38, 128)
    assert not extents.apart(1 << 31, 128, 8, (1 << 38) - 1, 128) and not extents.apart(1 << 31, 1024, 9, 128, 128)
    assert extents.apart(big, 1, 1, big, 1) and not extents.apart(big, big, 2, big, big) and not extents.apart(1 << 20, -big - 1, 3, -big - 1, 8)
    assert extents.apart(1 << 20, 3, 2, 1, 1) and not extents.apart(1 << 20, 3, 4, 1, 1)
