"""The axes of rotated pairs, and calls of the entry that takes them that are refused before anything is enqueued."""
import pytest

from jit_kernel import _native
from jit_kernel.norm_rope import _PART, _axes_bytes, rotary_axes

EINVAL, ERANGE = -1, -4
A = 1 << 20  # an aligned address

PART = dict(x=A, xt=1024, xh=128, weight=0, bias=0, out=A, ot=1024, oh=128, scale=0, st=0, sh=0, mul=0, slots=0, n_slots=0, heads=8,
            norm=0, rotate=1, wd=0, eps=1e-6, reserved=0)


def test_rotary_axes():
    assert rotary_axes((2, 3, 1)) == (0, 0, 1, 1, 1, 2)
    assert rotary_axes((3, 1, 2), interleaved=True) == (0, 1, 2, 0, 2, 0)
    assert rotary_axes(()) == rotary_axes((), interleaved=True) == ()


def test_axes_bytes():
    assert _axes_bytes((0, 2, 1, 0), 4, 3) == b"\0\2\1\0"
    for axes, pairs, n in (((0, 1), 3, 2), ((0, 2), 2, 2), ((0, -1), 2, 2), ((0, 1.0), 2, 2), ((0, 0), 2, 0), ((0, 4), 2, 5)):
        with pytest.raises(RuntimeError):
            _axes_bytes(axes, pairs, n)


def rows(tokens=4, D=128, positions=A, n_axes=3, axes=bytes(i % 3 for i in range(32)), table=A, rotary=64, workspace=None, **fields):
    return _native.lib().fftopk_head_rows_axes(_PART.pack(*{**PART, **fields}.values()), 1, tokens, D, 1, positions, 4, n_axes, axes, table, 10,
                                               rotary, 0, workspace, None, None)


@pytest.mark.parametrize("want,call", [
    (EINVAL, dict(axes=None)), (EINVAL, dict(workspace=A + 8)), (EINVAL, dict(n_axes=0)), (EINVAL, dict(n_axes=-1)), (ERANGE, dict(n_axes=5)), (EINVAL, dict(n_axes=2)),
    (EINVAL, dict(axes=bytes(31) + b"\3")), (EINVAL, dict(axes=b"\xff" + bytes(31))), (EINVAL, dict(positions=None)), (EINVAL, dict(positions=A + 2)),
    (EINVAL, dict(table=None)), (ERANGE, dict(rotary=8)), (ERANGE, dict(rotary=144)), (EINVAL, dict(tokens=-1)), (ERANGE, dict(D=12)), (0, dict(tokens=0)),
    (0, dict(heads=0)), (ERANGE, dict(tokens=1 << 31))])
def test_head_rows_axes(want, call):
    assert rows(**call) == want
