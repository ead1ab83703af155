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

from . import _native
from .topk_indexer import _launch

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_NORMS = {None: 0, "rms": 1, "layer": 2}
#: fftopk_head_part (include/fftopk.h)
_PART = struct.Struct("@PqqPPPqqPqqPPqiiiifi")
FP8 = torch.float8_e4m3fn


def _no_grad(*tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("this op has no gradient: call it under torch.no_grad() or detach its inputs")


def _check_rows(x: torch.Tensor, what: str, idx: int, dtype: torch.dtype, tokens: int, dim: int) -> None:
    if x.dim() != 3 or x.size(0) != tokens or x.size(2) != dim:
        raise RuntimeError(f"{what} must be [tokens, heads, D] with the tokens and the D of the others")
    if x.dtype != dtype or x.get_device() != idx:
        raise RuntimeError(f"{what} must be of the others' type and on their device")
    if x.stride(2) != 1 and dim > 1:
        raise RuntimeError(f"{what} must have unit inner stride")


def _check_vector(t: Optional[torch.Tensor], what: str, idx: int, n: int, dtype: torch.dtype = torch.int32) -> None:
    if t is not None and (t.dtype != dtype or t.dim() != 1 or t.size(0) != n or not t.is_contiguous() or t.get_device() != idx):
        raise RuntimeError(f"{what} must be a contiguous {dtype} tensor of shape [{n}] on the inputs' device")


def _check_norm(norm, weight, bias, what: str, idx: int, dim: int) -> None:
    if norm not in _NORMS:
        raise RuntimeError(f"{what}_norm must be None, 'rms' or 'layer'")
    if norm is None and (weight is not None or bias is not None):
        raise RuntimeError(f"{what}_weight and {what}_bias go with a norm")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.dtype not in _DTYPES or t.dim() != 1 or t.size(0) != dim or not t.is_contiguous()
                              or t.get_device() != idx):
            raise RuntimeError(f"{what}_{name} must be a contiguous floating tensor of shape [D] on the inputs' device")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"{what}_weight and {what}_bias must have the same type")


def _check_cache(cache: torch.Tensor, scale: torch.Tensor, what: str, idx: int, heads: int, dim: int) -> None:
    if cache.dtype != FP8 or cache.dim() != 3 or cache.size(1) != heads or cache.size(2) != dim or cache.get_device() != idx:
        raise RuntimeError(f"{what}_cache must be float8_e4m3fn [slots, heads, D] on the inputs' device")
    if cache.stride(2) != 1 and dim > 1:
        raise RuntimeError(f"{what}_cache must have unit inner stride")
    if scale is None or scale.dtype != torch.float32 or scale.shape != cache.shape[:2] or scale.get_device() != idx:
        raise RuntimeError(f"{what}_scale must be float32 [slots, heads] on the inputs' device")


def _part(x, out, norm=None, weight=None, bias=None, rotate=False, eps=0.0, scale=None, mul=None, slots=None) -> bytes:
    """A part as the C entry takes it: x [T, H, D] into `out` [T or slots, H, D] (and scale [.., H])."""
    wd = weight if weight is not None else bias
    return _PART.pack(
        x.data_ptr(), x.stride(0), x.stride(1), 0 if weight is None else weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
        out.data_ptr(), out.stride(0), out.stride(1), 0 if scale is None else scale.data_ptr(),
        0 if scale is None else scale.stride(0), 0 if scale is None else scale.stride(1), 0 if mul is None else mul.data_ptr(),
        0 if slots is None else slots.data_ptr(), 0 if slots is None else out.size(0), x.size(1), _NORMS[norm], int(rotate),
        0 if wd is None else _DTYPES[wd.dtype], eps, 0)


def _rows(idx: int, parts, tokens: int, dim: int, dtype: torch.dtype, positions, cos_sin, interleaved: bool) -> None:
    _launch(_native.lib().fftopk_head_rows, "fftopk_head_rows", idx, b"".join(parts), len(parts), tokens, dim, _DTYPES[dtype],
            None if positions is None else positions.data_ptr(), None if cos_sin is None else cos_sin.data_ptr(),
            0 if cos_sin is None else cos_sin.size(0), 0 if cos_sin is None else cos_sin.size(1), int(interleaved))


def _check_call(x: torch.Tensor, positions, cos_sin, dim: int) -> int:
    if not x.is_cuda:
        raise RuntimeError("the inputs must be CUDA tensors")
    if x.dtype not in _DTYPES:
        raise RuntimeError("the inputs must be float16, bfloat16 or float32")
    if dim % 8 or not 8 <= dim <= 256:
        raise RuntimeError("D must be a multiple of 8 up to 256")
    idx = x.get_device()
    if (positions is None) != (cos_sin is None):
        raise RuntimeError("positions and cos_sin go together")
    if cos_sin is not None:
        _check_vector(positions, "positions", idx, x.size(0))
        if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.get_device() != idx:
            raise RuntimeError("cos_sin must be a contiguous float32 tensor [positions, rotary] on the inputs' device")
        if cos_sin.size(1) % 16 or not 16 <= cos_sin.size(1) <= dim:
            raise RuntimeError("the rotated channels (cos_sin's columns) must be a multiple of 16 up to D")
    return idx


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
    if q.dim() != 3:
        raise RuntimeError("q must be [tokens, heads, D]")
    T, _, D = q.shape
    idx = _check_call(q, positions, cos_sin, D)
    _check_rows(q, "q", idx, q.dtype, T, D)
    _check_norm(q_norm, q_weight, q_bias, "q", idx, D)
    _no_grad(q, k, q_weight, k_weight, q_bias, k_bias)
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check_rows(q_out, "q_out", idx, q.dtype, T, D)
        if q_out.size(1) != q.size(1):
            raise RuntimeError("q_out must have q's shape")
    rotate = cos_sin is not None
    parts = [_part(q, q_out, q_norm, q_weight, q_bias, rotate, eps)]
    if k is not None:
        _check_rows(k, "k", idx, q.dtype, T, D)
        _check_norm(k_norm, k_weight, k_bias, "k", idx, D)
        if k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        else:
            _check_rows(k_out, "k_out", idx, q.dtype, T, D)
            if k_out.size(1) != k.size(1):
                raise RuntimeError("k_out must have k's shape")
        parts.append(_part(k, k_out, k_norm, k_weight, k_bias, rotate, eps))
    if T:
        _rows(idx, parts, T, D, q.dtype, positions, cos_sin, interleaved)
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
    into row slots[t] of k_cache, v quantised into v_cache. Arguments as for those two."""
    if q.dim() != 3:
        raise RuntimeError("q must be [tokens, heads, D]")
    T, _, D = q.shape
    idx = _check_call(q, positions, cos_sin, D)
    for x, what in ((q, "q"), (k, "k"), (v, "v")):
        _check_rows(x, what, idx, q.dtype, T, D)
    _check_norm(q_norm, q_weight, q_bias, "q", idx, D)
    _check_norm(k_norm, k_weight, k_bias, "k", idx, D)
    _check_vector(slots, "slots", idx, T)
    _check_cache(k_cache, k_scale, "k", idx, k.size(1), D)
    _check_cache(v_cache, v_scale, "v", idx, v.size(1), D)
    _no_grad(q, k, v, q_weight, k_weight, q_bias, k_bias)
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check_rows(q_out, "q_out", idx, q.dtype, T, D)
        if q_out.size(1) != q.size(1):
            raise RuntimeError("q_out must have q's shape")
    rotate = cos_sin is not None
    if T:
        _rows(idx, [_part(q, q_out, q_norm, q_weight, q_bias, rotate, eps),
                    _part(k, k_cache, k_norm, k_weight, k_bias, rotate, eps, k_scale, None, slots),
                    _part(v, v_cache, scale=v_scale, slots=slots)], T, D, q.dtype, positions, cos_sin, interleaved)
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
            [B, rows, D]); -1 for padding tokens, whose keys are not written. The slots of one call differ from one another.
        k_cache: float8_e4m3fn, contiguous, last dimension D: [B, rows, D] as FusedIndexerTopk takes it, or [rows, D];
            k_scale: float32, contiguous, of k_cache's shape without D. Both are written at `slots`.
    Returns:
        (q8, w8): q as float8_e4m3fn [T, H, D] and w times the scale of each head's row, float32 [T, H] - relu(s x) = s relu(x)
        for a positive scale, so FusedIndexerTopk(q8, k_cache, w8, lengths, k_scale=k_scale) ranks as with q itself.
    """
    if q.dim() != 3 or k.dim() != 2:
        raise RuntimeError("q must be [tokens, heads, D] and k [tokens, D]")
    T, H, D = q.shape
    idx = _check_call(q, positions, cos_sin, D)
    k3 = k.unsqueeze(1)
    _check_rows(q, "q", idx, q.dtype, T, D)
    _check_rows(k3, "k", idx, q.dtype, T, D)
    _check_norm(q_norm, q_weight, q_bias, "q", idx, D)
    _check_norm(k_norm, k_weight, k_bias, "k", idx, D)
    _check_vector(slots, "slots", idx, T)
    if w.dtype != torch.float32 or w.shape != (T, H) or not w.is_contiguous() or w.get_device() != idx:
        raise RuntimeError("w must be a contiguous float32 tensor [tokens, heads] on the inputs' device")
    if k_cache.dim() < 2 or not k_cache.is_contiguous() or not k_scale.is_contiguous() or k_scale.shape != k_cache.shape[:-1]:
        raise RuntimeError("k_cache must be contiguous [.., rows, D] and k_scale contiguous of its shape without D")
    rows, scales = k_cache.view(-1, 1, k_cache.size(-1)), k_scale.view(-1, 1)
    _check_cache(rows, scales, "k", idx, 1, D)
    _no_grad(q, k, w, q_weight, k_weight, q_bias, k_bias)
    q8 = torch.empty((T, H, D), dtype=FP8, device=q.device)
    w8 = torch.empty((T, H), dtype=torch.float32, device=q.device)
    rotate = cos_sin is not None
    if T:
        _rows(idx, [_part(q, q8, q_norm, q_weight, q_bias, rotate, eps, w8, w),
                    _part(k3, rows, k_norm, k_weight, k_bias, rotate, eps, scales, None, slots)], T, D, q.dtype, positions, cos_sin,
              interleaved)
    return q8, w8
