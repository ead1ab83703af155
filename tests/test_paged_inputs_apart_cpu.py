"""Results of the paged cache's entries that lie on their inputs: refused before anything is enqueued. No device is needed, and the pointers named here
are never followed."""
import ctypes
import subprocess

import pytest
from hypothesis import given, settings, strategies as st

from test_paged_overlap_cpu import A, CALL, CSRC, EINVAL, EVICT, FAR, attend, evict, rows

W = A + 8 * FAR


# (2 sequences, 8 query heads and 2 key heads of 128, weights [2, 2, 64])
@pytest.mark.parametrize("call", [
    dict(out=A), dict(out=A, os=128, oh=256), dict(out=A + 16), dict(out=A + 2 * 15 * 128 + 254), dict(out=A - 2 * 15 * 128 - 254), dict(out=A + 2 * 1024),
    dict(out=A + 2 * 128, os=2048), dict(out=A, q_heads=2, seqs=1), dict(out=A, qs=0, qh=0), dict(out=A + 64, qs=0, qh=128),
    dict(out=A + 2 * 128, qs=2048, qh=256, os=2048, oh=128), dict(out=A + 6, qs=2080, qh=136, os=1088, oh=130),
    dict(w=W, wo=W + 4, ws=128, wh=64, wos=128, woh=64, cols=64), dict(w=W, wo=W, ws=128, wh=64, wos=64, woh=128, cols=64),
    dict(w=W, wo=W, ws=128, wh=0, wos=128, woh=64, cols=64), dict(w=W, wo=W, ws=0, wh=64, wos=128, woh=64, cols=64),
    dict(w=W, wo=W + 4 * 64, ws=128, wh=64, wos=128, woh=64, cols=64), dict(w=W, wo=W - 4 * 255, ws=128, wh=64, wos=128, woh=64, cols=64)])
def test_attention(call):
    assert attend(**call) == EINVAL


@pytest.mark.parametrize("call", [
    dict(wo=EVICT["w"] + 4), dict(wo=EVICT["w"] + 4 * 64), dict(wo=EVICT["w"] - 4 * 255), dict(wo=EVICT["w"] + 4 * 128, ws=256, wos=64, woh=128),
    dict(wo=EVICT["w"] + 4 * 64, wh=0)])
def test_evict(call):
    assert evict(**call) == EINVAL


@pytest.fixture(scope="module")
def extents(tmp_path_factory):
    out = tmp_path_factory.mktemp("extents") / "libextents.so"
    source = out.with_suffix(".cpp")
    source.write_text('#include "fftopk_extent.h"\nextern "C" int meet(int64_t at, int64_t as, int64_t ah, int64_t bs, int64_t bh, int64_t n, int64_t h, int64_t w, int e)'
                      "{ char* p = (char*)(1 << 20); return fftopk::rows_meet(p, as, ah, p + at, bs, bh, n, h, w, e); }\n")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(out), str(source)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.meet.argtypes = [ctypes.c_int64] * 8 + [ctypes.c_int]
    return lib


@settings(deadline=None, max_examples=3000)
@given(st.integers(-150, 150), *[st.integers(-40, 40)] * 4, st.integers(0, 5), st.integers(0, 5), st.integers(0, 9), st.booleans())
def test_rows_meet(extents, at, a_seq, a_head, b_seq, b_head, seqs, heads, width, same):
    """Against every row of either: what lies between the other one's rows is told from what lies on them. (Two bytes an element)"""
    if same:
        b_seq, b_head = a_seq, a_head
    # (in halves of elements: an address may lie between two of them)
    a, b = (rows(seqs, 2 * s, heads, 2 * h, 2 * width) for s, h in ((a_seq, a_head), (b_seq, b_head)))
    b = [{x + at for x in row} for row in b]
    want = any(x & y for x in a for y in b)
    assert bool(extents.meet(at, a_seq, a_head, b_seq, b_head, seqs, heads, width, 2)) == want


def test_rows_meet_at_large_sizes(extents):
    n, h, w = 1 << 20, 1 << 10, 128
    assert extents.meet(2 * n * h * w - 2, h * w, w, h * w, w, n, h, w, 2) and not extents.meet(2 * n * h * w, h * w, w, h * w, w, n, h, w, 2)
    assert not extents.meet(2 * h * w, 2 * h * w, w, 2 * h * w, w, n, h, w, 2) and extents.meet(2 * h * w - 2, 2 * h * w, w, 2 * h * w, w, n, h, w, 2)
    assert not extents.meet(2 * w, h * 2 * w, 2 * w, h * 2 * w, 2 * w, n, h, w, 2)  # (heads of either in turn)


def test_the_call_itself_is_not_refused_for_its_inputs():
    assert len({CALL[x] for x in ("q", "k", "v", "table", "lengths", "out")}) == 6 and len({EVICT[x] for x in ("k", "v", "w", "wo", "lengths", "new")}) == 6
