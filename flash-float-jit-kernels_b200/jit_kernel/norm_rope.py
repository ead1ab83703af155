"""Norm and position rotation of queries and keys, head by head and in one pass (no counterpart in the reference, which starts
from finished logits; README.md:24 names the steps in front of them).

``qk_norm_rope`` hands q and k back in their own type; ``qkv_norm_rope_write`` writes k and v into a quantised cache in the same
launch; ``indexer_qk_write`` makes what ``FusedIndexerTopk`` reads in fp8: q as e4m3 with its scales folded into the head weights,
k quantised into the indexer's key cache as it is written. All are enqueue-only on the current stream, work in 32 bits whatever the
inputs' type and round once. They serve: none has a gradient, and a tensor that asks for one is refused."""
from __future__ import annotations

import struct
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native
from .topk_indexer import _launch

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_NORMS = {None: 0, "rms": 1, "layer": 2}
#: fftopk_head_part (include/fftopk.h)
_PART = struct.Struct("@PqqPPPqqPqqPPqiiiifi")
FP8 = torch.float8_e4m3fn
_DENSE = torch.contiguous_format


# An eager call on a few tokens is as long as its Python: every tensor is asked once for each of its properties, and the
# pieces below hand on what they have asked for.
def _no_grad(*tensors) -> None:
    """Every floating tensor of a call, outputs and caches too: none may ask for a gradient, or carry a forward-mode tangent."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("this op has no gradient: call it under torch.no_grad() or detach its inputs")
    # (the level's name is private: where it is missing, every tensor is asked)
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("this op has no gradient: a tensor carries a forward-mode tangent")


def _check_rows(x: torch.Tensor, what: str, idx: int, dtype: torch.dtype, tokens: int, dim: int, heads: int = -1):
    """(heads, strides) of x [tokens, heads, dim]"""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != tokens or shape[2] != dim or (heads >= 0 and shape[1] != heads):
        raise RuntimeError(f"{what} must be [tokens, heads, D] with the tokens and the D of the others, and an output of its input's shape")
    if x.dtype is not dtype or x.get_device() != idx:
        raise RuntimeError(f"{what} must be of the others' type and on their device")
    if stride[2] != 1 and dim > 1:
        raise RuntimeError(f"{what} must have unit inner stride")
    return shape[1], stride


def _check_vector(t: Optional[torch.Tensor], what: str, idx: int, n: int) -> int:
    """The address of an int32 vector of n (0: None)"""
    if t is None:
        return 0
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous() or t.get_device() != idx:
        raise RuntimeError(f"{what} must be a contiguous int32 tensor of shape [{n}] on the inputs' device")
    return t.data_ptr()


def _check_norm(norm, weight, bias, what: str, idx: int, dim: int):
    """(weight's address, bias', their type, the norm) as the C entry takes them"""
    if norm is None:
        if weight is not None or bias is not None:
            raise RuntimeError(f"{what}_weight and {what}_bias go with a norm")
        return 0, 0, 0, 0
    if norm not in _NORMS:
        raise RuntimeError(f"{what}_norm must be None, 'rms' or 'layer'")
    at, kind = [0, 0], None
    for i, t in enumerate((weight, bias)):
        if t is None:
            continue
        if t.dtype not in _DTYPES or t.shape != (dim,) or not t.is_contiguous() or t.get_device() != idx:
            raise RuntimeError(f"{what}_weight and {what}_bias must be contiguous floating tensors of shape [D] on the inputs' device")
        if kind is not None and t.dtype is not kind:
            raise RuntimeError(f"{what}_weight and {what}_bias must have the same type")
        at[i], kind = t.data_ptr(), t.dtype
    return at[0], at[1], 0 if kind is None else _DTYPES[kind], _NORMS[norm]


def _check_cache(cache: torch.Tensor, scale: torch.Tensor, what: str, idx: int, heads: int, dim: int):
    """(slots, strides, scale's strides) of a quantised cache [slots, heads, dim]"""
    shape, stride = cache.shape, cache.stride()
    if cache.dtype is not FP8 or len(shape) != 3 or shape[1] != heads or shape[2] != dim or cache.get_device() != idx:
        raise RuntimeError(f"{what}_cache must be float8_e4m3fn [slots, heads, D] on the inputs' device")
    if stride[2] != 1 and dim > 1:
        raise RuntimeError(f"{what}_cache must have unit inner stride")
    if scale is None or scale.dtype is not torch.float32 or scale.shape != shape[:2] or scale.get_device() != idx:
        raise RuntimeError(f"{what}_scale must be float32 [slots, heads] on the inputs' device")
    return shape[0], stride, scale.stride()


_PLAIN = (0, 0, 0, 0)


def _dense(x, xs, heads, out, os, norm=_PLAIN, rotate=0, eps=0.0) -> bytes:
    """A part as the C entry takes it: x [T, H, D] into `out` of the same type."""
    return _PART.pack(x.data_ptr(), xs[0], xs[1], norm[0], norm[1], out.data_ptr(), os[0], os[1], 0, 0, 0, 0, 0, 0, heads, norm[3], rotate,
                      norm[2], eps, 0)


def _quantised(x, xs, heads, out, os, scale, ss, slots=0, n=0, mul=0, norm=_PLAIN, rotate=0, eps=0.0) -> bytes:
    """A part that ends as e4m3 in `out`, with its scales."""
    return _PART.pack(x.data_ptr(), xs[0], xs[1], norm[0], norm[1], out.data_ptr(), os[0], os[1], scale.data_ptr(), ss[0], ss[1], mul, slots,
                      n, heads, norm[3], rotate, norm[2], eps, 0)


def _rows(idx: int, parts: bytes, tokens: int, dim: int, dtype: torch.dtype, table=(0, 0, 0, 0), interleaved: bool = False) -> None:
    _launch(_native.lib().fftopk_head_rows, "fftopk_head_rows", idx, parts, len(parts) // _PART.size, tokens, dim, _DTYPES[dtype], table[0],
            table[1], table[2], table[3], interleaved)


def _check_first(x: torch.Tensor, what: str):
    """(device, tokens, D, type) of the first input, which the others go by"""
    shape, dtype, idx = x.shape, x.dtype, x.get_device()
    if idx < 0:
        raise RuntimeError("the inputs must be CUDA tensors")
    if len(shape) != 3:
        raise RuntimeError(f"{what} must be [tokens, heads, D]")
    if dtype not in _DTYPES:
        raise RuntimeError("the inputs must be float16, bfloat16 or float32")
    dim = shape[2]
    if dim % 8 or not 8 <= dim <= 256:
        raise RuntimeError("D must be a multiple of 8 up to 256")
    return idx, shape[0], dim, dtype


def _check_table(positions, cos_sin, idx: int, tokens: int, dim: int):
    """(positions' address, cos_sin's, its rows, its columns); zeros without a rotation"""
    if cos_sin is None:
        if positions is not None:
            raise RuntimeError("positions and cos_sin go together")
        return 0, 0, 0, 0
    if positions is None:
        raise RuntimeError("positions and cos_sin go together")
    shape = cos_sin.shape
    if cos_sin.dtype is not torch.float32 or len(shape) != 2 or not cos_sin.is_contiguous() or cos_sin.get_device() != idx:
        raise RuntimeError("cos_sin must be a contiguous float32 tensor [positions, rotary] on the inputs' device")
    if shape[1] % 16 or not 16 <= shape[1] <= dim:
        raise RuntimeError("the rotated channels (cos_sin's columns) must be a multiple of 16 up to D")
    return _check_vector(positions, "positions", idx, tokens), cos_sin.data_ptr(), shape[0], shape[1]


def qk_norm_rope(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: Optional[torch.Tensor],
    cos_sin: Optional[torch.Tensor],
    *,
    q_norm: Optional[str] = "rms",
    k_norm: Optional[str] = "rms",
    q_weight: Optional[torch.Tensor] = None,
    q_bias: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    k_bias: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
):
    """
    Norm of every head of q and k, then rotation of its first channels by the token's position.
    Args:
        q, k: [T, Hq, D] and [T, Hk, D] of one type (float16, bfloat16, float32), CUDA, unit inner stride - slices of a fused
            projection's output, for instance; k may be None. D is a multiple of 8 up to 256.
        positions: int32 [T], rows of cos_sin; with cos_sin None: no rotation.
        cos_sin: float32 [positions, R], contiguous: R/2 cosines, then R/2 sines. R, a multiple of 16 up to D, is the number of
            channels that are rotated. A position beyond the table makes them NaN and shows up in kernel_status().
        q_norm, k_norm: None, "rms" or "layer", over the D channels of a head; weight and bias [D] (default 1 and 0) and eps go
            with them.
        interleaved: pairs (2i, 2i + 1) instead of (i, i + R/2).
        q_out, k_out: where the results go (default: new tensors); q and k themselves are allowed.
    Returns:
        (q_out, k_out), of q's and k's shapes and type.
    """
    idx, T, D, dtype = _check_first(q, "q")
    table = _check_table(positions, cos_sin, idx, T, D)
    rotate = 1 if cos_sin is not None else 0
    heads, xs = _check_rows(q, "q", idx, dtype, T, D)
    norm = _check_norm(q_norm, q_weight, q_bias, "q", idx, D)
    _no_grad(q, k, cos_sin, q_weight, k_weight, q_bias, k_bias, q_out, k_out)
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=_DENSE)
        os = (heads * D, D)
    else:
        _, os = _check_rows(q_out, "q_out", idx, dtype, T, D, heads)
    parts = _dense(q, xs, heads, q_out, os, norm, rotate, eps)
    if k is not None:
        heads, xs = _check_rows(k, "k", idx, dtype, T, D)
        norm = _check_norm(k_norm, k_weight, k_bias, "k", idx, D)
        if k_out is None:
            k_out = torch.empty_like(k, memory_format=_DENSE)
            os = (heads * D, D)
        else:
            _, os = _check_rows(k_out, "k_out", idx, dtype, T, D, heads)
        parts += _dense(k, xs, heads, k_out, os, norm, rotate, eps)
    if T:
        _rows(idx, parts, T, D, dtype, table, interleaved)
    return q_out, k_out


def qkv_norm_rope_write(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: Optional[torch.Tensor],
    cos_sin: Optional[torch.Tensor],
    slots: torch.Tensor,
    k_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_cache: torch.Tensor,
    v_scale: torch.Tensor,
    *,
    q_norm: Optional[str] = "rms",
    k_norm: Optional[str] = "rms",
    q_weight: Optional[torch.Tensor] = None,
    q_bias: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    k_bias: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    q_out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """qk_norm_rope and kv_cache.cache_write in one launch: q comes back normed and rotated, k is normed, rotated and quantised
    into row slots[t] of k_cache, v quantised into v_cache. Arguments as for those two; padding tokens (slot -1) may have any
    position (outside the table: q's rotated channels are NaN, and kernel_status() says nothing)."""
    idx, T, D, dtype = _check_first(q, "q")
    table = _check_table(positions, cos_sin, idx, T, D)
    rotate = 1 if cos_sin is not None else 0
    (qh, qs), (kh, ks), (vh, vs) = (_check_rows(x, what, idx, dtype, T, D) for x, what in ((q, "q"), (k, "k"), (v, "v")))
    q_how, k_how = _check_norm(q_norm, q_weight, q_bias, "q", idx, D), _check_norm(k_norm, k_weight, k_bias, "k", idx, D)
    at = _check_vector(slots, "slots", idx, T)
    kn, kcs, kss = _check_cache(k_cache, k_scale, "k", idx, kh, D)
    vn, vcs, vss = _check_cache(v_cache, v_scale, "v", idx, vh, D)
    _no_grad(q, k, v, cos_sin, k_cache, k_scale, v_cache, v_scale, q_weight, k_weight, q_bias, k_bias, q_out)
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=_DENSE)
        os = (qh * D, D)
    else:
        _, os = _check_rows(q_out, "q_out", idx, dtype, T, D, qh)
    if T:
        _rows(idx, _dense(q, qs, qh, q_out, os, q_how, rotate, eps)
              + _quantised(k, ks, kh, k_cache, kcs, k_scale, kss, at, kn, 0, k_how, rotate, eps)
              + _quantised(v, vs, vh, v_cache, vcs, v_scale, vss, at, vn), T, D, dtype, table, interleaved)
    return q_out


def indexer_qk_write(
    q: torch.Tensor,
    k: torch.Tensor,
    w: torch.Tensor,
    positions: Optional[torch.Tensor],
    cos_sin: Optional[torch.Tensor],
    slots: torch.Tensor,
    k_cache: torch.Tensor,
    k_scale: torch.Tensor,
    *,
    q_norm: Optional[str] = None,
    k_norm: Optional[str] = "layer",
    q_weight: Optional[torch.Tensor] = None,
    q_bias: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    k_bias: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
):
    """
    The step in front of ``FusedIndexerTopk`` with an fp8 key cache.
    Args:
        q: [T, H, D] (H = 64, D = 128 for FusedIndexerTopk); k: [T, D], one key per token; as for qk_norm_rope.
        w: float32 [T, H], contiguous: the head weights.
        slots: int32 [T]: the token's row of the cache, counted through the sequences (b * rows + position for a cache
            [B, rows, D]); -1 for padding tokens, whose keys are not written and whose positions may be anything (outside the
            table: q's rotated channels are NaN). The slots of one call differ from one another.
        k_cache: float8_e4m3fn, contiguous, last dimension D: [B, rows, D] as FusedIndexerTopk takes it, or [rows, D];
            k_scale: float32, contiguous, of k_cache's shape without D. Both are written at `slots`.
    Returns:
        (q8, w8): q as float8_e4m3fn [T, H, D] and w times the scale of each head's row, float32 [T, H] - relu(s x) = s relu(x)
        for a positive scale, so FusedIndexerTopk(q8, k_cache, w8, lengths, k_scale=k_scale) ranks as with q itself.
    """
    idx, T, D, dtype = _check_first(q, "q")
    table = _check_table(positions, cos_sin, idx, T, D)
    rotate = 1 if cos_sin is not None else 0
    H, qs = _check_rows(q, "q", idx, dtype, T, D)
    ks = k.stride()
    if k.shape != (T, D) or k.dtype is not dtype or k.get_device() != idx or ks[1] != 1:
        raise RuntimeError("k must be [tokens, D], of q's type and on its device, with unit inner stride")
    q_how, k_how = _check_norm(q_norm, q_weight, q_bias, "q", idx, D), _check_norm(k_norm, k_weight, k_bias, "k", idx, D)
    at = _check_vector(slots, "slots", idx, T)
    if w.dtype is not torch.float32 or w.shape != (T, H) or not w.is_contiguous() or w.get_device() != idx:
        raise RuntimeError("w must be a contiguous float32 tensor [tokens, heads] on the inputs' device")
    shape = k_cache.shape
    if k_cache.dtype is not FP8 or len(shape) < 2 or shape[-1] != D or not k_cache.is_contiguous() or k_cache.get_device() != idx:
        raise RuntimeError("k_cache must be contiguous float8_e4m3fn [.., rows, D] on the inputs' device")
    if k_scale.dtype is not torch.float32 or k_scale.shape != shape[:-1] or not k_scale.is_contiguous() or k_scale.get_device() != idx:
        raise RuntimeError("k_scale must be contiguous float32 of k_cache's shape without D on the inputs' device")
    _no_grad(q, k, w, cos_sin, k_cache, k_scale, q_weight, k_weight, q_bias, k_bias)
    q8 = torch.empty_like(q, dtype=FP8, memory_format=_DENSE)
    w8 = torch.empty_like(w)
    if T:
        _rows(idx, _quantised(q, qs, H, q8, (H * D, D), w8, (H, 1), 0, 0, w.data_ptr(), q_how, rotate, eps)
              + _quantised(k, (ks[0], D), 1, k_cache, (D, D), k_scale, (1, 1), at, k_scale.numel(), 0, k_how, rotate, eps), T, D, dtype,
              table, interleaved)
    return q8, w8
