"""The rule that sends a call of attention to the kernel of many heads, and that the GPU tests written for either kernel reach it.
The kernels' host code takes the rule from csrc/fftopk_decide.h; here g++ compiles the same header."""
import ctypes
import subprocess
from pathlib import Path

import pytest

import test_attention_many_heads_gpu as many_heads
import test_attention_scales_gpu as scales
import test_sparse_attention_edges_gpu as edges

REPO = Path(__file__).resolve().parent.parent
SMS = 148
HARNESS = """
#include "fftopk_decide.h"
extern "C" int is_wide(int64_t tokens, int kv_heads, int group, int fp8, int sms) {
  return fftopk::attend_is_wide(tokens, kv_heads, group, fp8 != 0, sms);
}
"""


@pytest.fixture(scope="module")
def is_wide(tmp_path_factory):
    at = tmp_path_factory.mktemp("rule")
    (at / "rule.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", str(REPO / "flash-float-jit-kernels_b200" / "csrc"), "-o",
                    str(at / "rule.so"), str(at / "rule.cpp")], check=True)
    f = ctypes.CDLL(str(at / "rule.so")).is_wide
    f.argtypes = [ctypes.c_int64] + [ctypes.c_int] * 4
    return lambda T, Hq, Hk, fp8: bool(f(T, Hk, Hq // Hk, fp8, SMS))


@pytest.mark.parametrize("T,Hq,Hk", many_heads.MANY + scales.MANY + [(12, 128, 1), (170, 128, 1), (20, 128, 1)])
@pytest.mark.parametrize("fp8", [False, True])
def test_cases_of_many_heads(is_wide, fp8, T, Hq, Hk):
    assert is_wide(T, Hq, Hk, fp8)


@pytest.mark.parametrize("T,Hq,Hk", edges.MANY)
@pytest.mark.parametrize("fp8", [False, True])
def test_cases_of_many_tokens(is_wide, fp8, T, Hq, Hk):
    """(32 heads to a key head over e4m3 stay where they are: see the rule)"""
    assert is_wide(T, Hq, Hk, fp8) == (not fp8 or Hq // Hk > 32)


@pytest.mark.parametrize("T,Hq,Hk", scales.FEW)
@pytest.mark.parametrize("fp8", [False, True])
def test_cases_of_few_tokens(is_wide, fp8, T, Hq, Hk):
    assert not is_wide(T, Hq, Hk, fp8)


@pytest.mark.parametrize("fp8", [False, True])
def test_where_the_rule_turns(is_wide, fp8):
    assert not is_wide(1 << 20, 16, 1, fp8) and not is_wide(1 << 20, 128, 8, fp8)
    assert is_wide(1 << 20, 17, 1, fp8) == (not fp8) and is_wide(1 << 20, 33, 1, fp8)
    # four CTAs for each of its pieces: 8 pieces to a token of 128 heads
    assert not is_wide(9, 128, 1, fp8) and is_wide(10, 128, 1, fp8)


def test_limits_of_waits():
    """Set and restored without a device."""
    from jit_kernel import _native
    stop = _native.lib().fftopk_set_attend_stop
    assert stop(200_000_001, -1) == _native.E_RANGE and stop(-1, 1 << 31) == _native.E_RANGE
    assert stop(1, 0) == 0 and stop(-1, -1) == 0


@pytest.mark.parametrize("tokens,q_heads,kv_heads", [((1 << 31) - 1, (1 << 31) - 1, (1 << 31) - 1), (1 << 28, 8, 8), ((1 << 31) - 1, 1 << 30, 1)])
def test_more_pieces_of_work_than_a_grid_has(tokens, q_heads, kv_heads):
    """Refused before anything is multiplied out of 64 bits, and before a device is asked."""
    from jit_kernel import _native
    from test_rows_refusals_cpu import ATTEND
    from jit_kernel.sparse_attention import _ARGS
    args = {**ATTEND, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "kh": 128}
    assert _native.lib().fftopk_sparse_attention(_ARGS.pack(*args.values()), None, None) == _native.E_RANGE


def test_more_head_rows_than_a_call_takes():
    from jit_kernel import _native
    from test_rows_refusals_cpu import rows
    for tokens, heads, n in ((1 << 61, 8, 1), ((1 << 31) - 1, (1 << 31) - 1, 3), (1 << 40, 1, 1), (16, 1 << 30, 2)):
        assert rows(tokens=tokens, heads=heads, n_parts=n) == _native.E_RANGE
