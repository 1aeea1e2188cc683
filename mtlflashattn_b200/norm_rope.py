"""Per-head RMS norm of queries and keys with the position rotation, in one pass: what stands
between a model's q/k projection and the attention (no counterpart in the reference)."""
from __future__ import annotations

import struct

import torch

from . import _kernel, _lib
from ._grad import _guard_grad
from ._kernel import _DTYPES, MAX_HEAD_DIM

__all__ = ["qk_norm_rope"]

_FORMAT = struct.Struct(_lib.NORM_ROPE_FORMAT)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _side_dtype(name, tensors, dtype):
    """Type code of the given weights or tables: all fp32, or all of q's type."""
    ds = {t.dtype for t in tensors if t is not None}
    if not ds:
        return _DTYPES[dtype]
    if len(ds) > 1 or not ds <= {dtype, torch.float32}:
        raise ValueError(f"mtlflashattn_b200: {name} must all be {dtype} or all fp32")
    return _DTYPES[ds.pop()]


def qk_norm_rope(q, k, q_weight=None, k_weight=None, rotary_cos=None, rotary_sin=None,
                 positions=None, eps=1e-6, interleaved=False):
    """Normalise every head of q and k and rotate it by its token's position (forward only).

    q: [B, L, Hq, D]; k: [B, L, Hkv, D] (or packed [total, H, D]), any strides, fp16/bf16/fp32,
    D <= 128. Each head row x becomes x / sqrt(mean(x^2) + eps) * weight, then its first R dims
    are rotated: pairs (i, i + R/2), or (2i, 2i + 1) if ``interleaved``, turn by the angle whose
    cosine and sine stand in ``rotary_cos``/``rotary_sin`` [max_position, R/2] at the token's
    position. Everything is fp32 up to one rounding at the end.

    ``q_weight``/``k_weight``: [D] in q's type or fp32 (None: ones). The tables are in q's type or
    fp32; without them there is no rotation. ``positions``: int32 or int64, [B, L] or [L]
    (packed: [total]); None means 0 .. L - 1. A token whose position is outside of the tables gets
    rows of zeros, and ``check_device_errors`` reports it.

    Returns contiguous (q, k) of the inputs' shapes and type.
    """
    dtype, dev = q.dtype, q.device
    if not q.is_cuda:
        raise NotImplementedError(
            f"mtlflashattn_b200: device {dev.type!r} not supported (CUDA only)")
    if dtype not in _DTYPES or k.dtype != dtype:
        raise NotImplementedError(
            f"mtlflashattn_b200: dtype {dtype} (q/k must match, fp16/bf16/fp32)")
    shape = q.shape
    nd = len(shape)
    if nd not in (3, 4) or k.dim() != nd:
        raise ValueError("mtlflashattn_b200: expected 4-D [B,L,H,D] or 3-D [total,H,D] q and k")
    if k.shape[:-2] != shape[:-2] or k.shape[-1] != shape[-1]:
        raise ValueError("mtlflashattn_b200: q/k tokens or head_dim mismatch")
    *lead, Hq, D = shape
    Hkv = k.shape[-2]
    if D > MAX_HEAD_DIM:
        raise NotImplementedError(f"mtlflashattn_b200: head_dim {D} > {MAX_HEAD_DIM}")
    if D == 0 or Hq == 0 or Hkv == 0:
        raise ValueError("mtlflashattn_b200: q and k need at least one head and one dim")
    if not eps >= 0:
        raise ValueError("mtlflashattn_b200: eps must be >= 0")
    B, L = lead if nd == 4 else (1, lead[0])
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and tuple(w.shape) != (D,):
            raise ValueError(f"mtlflashattn_b200: {name} must be [{D}], got {tuple(w.shape)}")
    w_dtype = _side_dtype("q_weight and k_weight", (q_weight, k_weight), dtype)
    R = rows = cos_row = sin_row = 0
    if (rotary_cos is None) != (rotary_sin is None):
        raise ValueError("mtlflashattn_b200: rotary_cos and rotary_sin go together")
    if rotary_cos is not None:
        if rotary_cos.dim() != 2 or rotary_cos.shape != rotary_sin.shape:
            raise ValueError("mtlflashattn_b200: rotary_cos/rotary_sin must be [max_position, R/2]")
        rows, R = rotary_cos.shape[0], 2 * rotary_cos.shape[1]
        if R > D:
            raise ValueError(f"mtlflashattn_b200: rotation of {R} dims of a head_dim of {D}")
    rot_dtype = _side_dtype("rotary_cos and rotary_sin", (rotary_cos, rotary_sin), dtype)
    pos_b = pos_l = 0
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("mtlflashattn_b200: positions must be int32 or int64")
        ps = tuple(positions.shape)
        if ps == (L,):
            pos_l = positions.stride(0)
        elif nd == 4 and ps == (B, L):
            pos_b, pos_l = positions.stride()
        else:
            raise ValueError(f"mtlflashattn_b200: positions must be one per token, got {ps}")
    for t in (k, q_weight, k_weight, rotary_cos, rotary_sin, positions):
        if t is not None and t.device != dev:
            raise ValueError("mtlflashattn_b200: all tensors must be on q's device")
    args = (q, k)
    q, k = _kernel._last_dim_contig(q), _kernel._last_dim_contig(k)
    if q_weight is not None:
        q_weight = _kernel._last_dim_contig(q_weight)
    if k_weight is not None:
        k_weight = _kernel._last_dim_contig(k_weight)
    if rotary_cos is not None:
        rotary_cos = _kernel._last_dim_contig(rotary_cos)
        rotary_sin = _kernel._last_dim_contig(rotary_sin)
        cos_row, sin_row = rotary_cos.stride(0), rotary_sin.stride(0)
    q_out = torch.empty(shape, dtype=dtype, device=dev)
    k_out = torch.empty(k.shape, dtype=dtype, device=dev)
    qs, ks = q.stride(), k.stride()
    if nd == 3:
        qs, ks = (0, *qs), (0, *ks)
    p = _kernel._scratch("norm_rope", _FORMAT)
    _FORMAT.pack_into(
        p, 0, q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), *qs[:3], *ks[:3],
        _ptr(q_weight), _ptr(k_weight), _ptr(rotary_cos), _ptr(rotary_sin), cos_row, sin_row,
        _ptr(positions), pos_b, pos_l, B, L, Hq, Hkv, D, R, min(rows, 2**31 - 1),
        positions is not None and positions.dtype == torch.int64, _DTYPES[dtype], w_dtype,
        rot_dtype, bool(interleaved), float(eps), _kernel._err_word(dev).data_ptr())
    _kernel._call(dev, "qk_norm_rope", _lib.qk_norm_rope, p)
    if torch.is_grad_enabled():
        extra = (q_weight, k_weight, rotary_cos, rotary_sin)
        return _guard_grad(q_out, *args, *extra), _guard_grad(k_out, *args, *extra)
    return q_out, k_out
