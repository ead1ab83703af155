"""Calls of the head-row, cache and attention entries that are refused before anything is enqueued: no device is needed, and the
pointers named here are never followed."""
import pytest
import torch

from jit_kernel import _native
from jit_kernel.kv_cache import cache_read, cache_write
from jit_kernel.norm_rope import _PART, indexer_qk_write, qk_norm_rope
from jit_kernel.sparse_attention import _ARGS, sparse_attention

EINVAL, ERANGE = -1, -4
A = 1 << 20  # an aligned address

PART = dict(x=A, xt=1024, xh=128, weight=0, bias=0, out=A, ot=1024, oh=128, scale=0, st=0, sh=0, mul=0, slots=0, n_slots=0, heads=8,
            norm=0, rotate=0, wd=0, eps=1e-6, reserved=0)


def rows(tokens=4, D=128, dtype=1, positions=A, table=A, table_rows=10, rotary=64, n_parts=1, parts=None, **fields):
    blob = _PART.pack(*{**PART, **fields}.values()) * n_parts if parts is None else parts
    return _native.lib().fftopk_head_rows(blob, n_parts, tokens, D, dtype, positions, table, table_rows, rotary, 0, None, None)


@pytest.mark.parametrize("want,call", [
    (EINVAL, dict(tokens=-1)), (EINVAL, dict(dtype=3)), (EINVAL, dict(dtype=-1)), (ERANGE, dict(D=0)), (ERANGE, dict(D=12)),
    (ERANGE, dict(D=264)), (EINVAL, dict(n_parts=0)), (EINVAL, dict(n_parts=4)), (EINVAL, dict(heads=-1)), (EINVAL, dict(norm=3)),
    (EINVAL, dict(weight=A)), (EINVAL, dict(bias=A)), (EINVAL, dict(norm=1, weight=A, wd=5)), (EINVAL, dict(norm=1, weight=A + 1, wd=1)),
    (EINVAL, dict(x=0)), (EINVAL, dict(out=0)), (EINVAL, dict(x=A + 1)), (EINVAL, dict(out=A + 1)), (EINVAL, dict(scale=A + 2)),
    (EINVAL, dict(slots=A + 2)), (EINVAL, dict(mul=A)), (EINVAL, dict(slots=A, n_slots=-1)),
    (ERANGE, dict(rotate=1, rotary=8)), (ERANGE, dict(rotate=1, rotary=72)), (ERANGE, dict(rotate=1, rotary=144)),
    (EINVAL, dict(rotate=1, positions=None)), (EINVAL, dict(rotate=1, table=None)), (EINVAL, dict(rotate=1, table=A + 8)),
    (EINVAL, dict(rotate=1, table_rows=-1)), (ERANGE, dict(tokens=1 << 31)), (ERANGE, dict(tokens=1 << 30, heads=8)),
    (0, dict(tokens=0)), (0, dict(heads=0)), (0, dict(tokens=0, x=0, out=0))])
def test_head_rows(want, call):
    assert rows(**call) == want


def test_head_rows_without_parts():
    assert _native.lib().fftopk_head_rows(None, 1, 4, 128, 1, None, None, 0, 0, 0, None, None) == EINVAL


READ = dict(cache=A, ss=256, hs=128, n_slots=10, heads=2, D=128, scale=A, cs=2, ch=1, slots=A, rows=2, per_row=3, offsets=None, out=A,
            dtype=1)


@pytest.mark.parametrize("want,call", [
    (EINVAL, dict(n_slots=-1)), (EINVAL, dict(heads=-1)), (EINVAL, dict(rows=-1)), (EINVAL, dict(per_row=-1)), (EINVAL, dict(dtype=4)),
    (ERANGE, dict(D=4)), (ERANGE, dict(D=300)), (EINVAL, dict(cache=None)), (EINVAL, dict(scale=None)), (EINVAL, dict(slots=None)),
    (EINVAL, dict(out=None)), (EINVAL, dict(out=A + 8)), (EINVAL, dict(scale=A + 1)), (EINVAL, dict(offsets=A + 2)),
    (ERANGE, dict(rows=1 << 16, per_row=1 << 16)), (ERANGE, dict(rows=1 << 31)), (ERANGE, dict(rows=1 << 30, per_row=1, heads=4)),
    (0, dict(rows=0)), (0, dict(per_row=0)), (0, dict(heads=0))])
def test_cache_read(want, call):
    assert _native.lib().fftopk_cache_read(*{**READ, **call}.values(), None, None) == want


ATTEND = dict(q=A, qt=1024, qh=128, k=A, ks=128, kh=128, v=A, vs=128, vh=128, k_scale=0, kss=0, ksh=0, v_scale=0, vss=0, vsh=0,
              indices=A, row=64, offsets=0, out=A, ot=1024, oh=128, lse=0, tokens=2, slots=100, q_heads=8, kv_heads=1, D=128, picks=64,
              dtype=1, scale=0.1)


@pytest.mark.parametrize("want,call", [
    (EINVAL, dict(tokens=-1)), (EINVAL, dict(q_heads=-1)), (EINVAL, dict(kv_heads=-1)), (EINVAL, dict(picks=-1)),
    (EINVAL, dict(slots=-1)), (EINVAL, dict(dtype=2)), (ERANGE, dict(D=96)), (ERANGE, dict(D=256)), (EINVAL, dict(kv_heads=0)),
    (EINVAL, dict(kv_heads=3)), (EINVAL, dict(k_scale=A)), (EINVAL, dict(v_scale=A)), (EINVAL, dict(q=0)), (EINVAL, dict(out=0)),
    (EINVAL, dict(indices=0)), (EINVAL, dict(k=0)), (EINVAL, dict(v=0)), (EINVAL, dict(q=A + 8)), (EINVAL, dict(k=A + 8)),
    (EINVAL, dict(v=A + 8)), (EINVAL, dict(qt=1028)), (EINVAL, dict(qh=68)), (EINVAL, dict(ks=132)), (EINVAL, dict(vs=132)),
    (EINVAL, dict(kv_heads=2, kh=68)), (EINVAL, dict(out=A + 1)), (EINVAL, dict(indices=A + 2)), (EINVAL, dict(offsets=A + 1)),
    (EINVAL, dict(lse=A + 2)), (EINVAL, dict(k_scale=A + 2, v_scale=A)), (ERANGE, dict(slots=1 << 31)), (ERANGE, dict(tokens=1 << 31)),
    (0, dict(tokens=0)), (0, dict(q_heads=0))])
def test_sparse_attention(want, call):
    assert _native.lib().fftopk_sparse_attention(_ARGS.pack(*{**ATTEND, **call}.values()), None, None) == want


def test_sparse_attention_without_arguments():
    assert _native.lib().fftopk_sparse_attention(None, None, None) == EINVAL


def test_cpu_tensors_are_refused():
    x, i = torch.zeros(2, 4, 64), torch.zeros(2, dtype=torch.int32)
    c, s = torch.zeros(8, 4, 64, dtype=torch.float8_e4m3fn), torch.ones(8, 4)
    with pytest.raises(RuntimeError):
        qk_norm_rope(x, None, None, None)
    with pytest.raises(RuntimeError):
        indexer_qk_write(x, x[:, 0], torch.zeros(2, 4), None, None, i, c[:, 0], s[:, 0])
    with pytest.raises(RuntimeError):
        cache_write(x, i, c, s)
    with pytest.raises(RuntimeError):
        cache_read(c, s, i)
    with pytest.raises(RuntimeError):
        sparse_attention(x.half(), c, c, i.view(2, 1), k_scale=s, v_scale=s)
