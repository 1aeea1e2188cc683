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


def _side(name, a, b, code, dtype):
    """Type code of two optional weights or tables: both fp32, or both of q's type."""
    if a is None:
        a = b
    if a is None:
        return code
    if b is not None and b.dtype is not a.dtype:
        raise ValueError(f"mtlflashattn_b200: {name} must be of one type")
    if a.dtype is torch.float32:
        return _lib.FP32
    if a.dtype is not dtype:
        raise ValueError(f"mtlflashattn_b200: {name} must be {dtype} or fp32")
    return code


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
    dtype, index = q.dtype, q.get_device()
    if index < 0:
        raise NotImplementedError(
            f"mtlflashattn_b200: device {q.device.type!r} not supported (CUDA only)")
    code = _DTYPES.get(dtype)
    if code is None or k.dtype is not dtype:
        raise NotImplementedError(
            f"mtlflashattn_b200: dtype {dtype} (q/k must match, fp16/bf16/fp32)")
    q_shape, k_shape = q.shape, k.shape
    nd = len(q_shape)
    if nd == 4 and len(k_shape) == 4:
        B, L, Hq, D = q_shape
        kB, kL, Hkv, kD = k_shape
    elif nd == 3 and len(k_shape) == 3:
        B = kB = 1
        L, Hq, D = q_shape
        kL, Hkv, kD = k_shape
    else:
        raise ValueError("mtlflashattn_b200: expected 4-D [B,L,H,D] or 3-D [total,H,D] q and k")
    if kB != B or kL != L or kD != D:
        raise ValueError("mtlflashattn_b200: q/k tokens or head_dim mismatch")
    if D > MAX_HEAD_DIM:
        raise NotImplementedError(f"mtlflashattn_b200: head_dim {D} > {MAX_HEAD_DIM}")
    if D == 0 or Hq == 0 or Hkv == 0:
        raise ValueError("mtlflashattn_b200: q and k need at least one head and one dim")
    if not eps >= 0:
        raise ValueError("mtlflashattn_b200: eps must be >= 0")
    same = k.get_device() == index
    wq = wk = cos = sin = pos = R = rows = cos_row = sin_row = pos_b = pos_l = pos64 = 0
    if q_weight is not None:
        if q_weight.shape != (D,):
            raise ValueError(f"mtlflashattn_b200: q_weight must be [{D}]")
        same = same and q_weight.get_device() == index
        q_weight = _kernel._last_dim_contig(q_weight)
        wq = q_weight.data_ptr()
    if k_weight is not None:
        if k_weight.shape != (D,):
            raise ValueError(f"mtlflashattn_b200: k_weight must be [{D}]")
        same = same and k_weight.get_device() == index
        k_weight = _kernel._last_dim_contig(k_weight)
        wk = k_weight.data_ptr()
    w_code = _side("q_weight and k_weight", q_weight, k_weight, code, dtype)
    if rotary_cos is not None and rotary_sin is not None:
        table = rotary_cos.shape
        if len(table) != 2 or rotary_sin.shape != table:
            raise ValueError("mtlflashattn_b200: rotary_cos/rotary_sin must be [max_position, R/2]")
        rows, R = table[0], 2 * table[1]
        if R > D:
            raise ValueError(f"mtlflashattn_b200: rotation of {R} dims of a head_dim of {D}")
        same = same and rotary_cos.get_device() == index and rotary_sin.get_device() == index
        rotary_cos = _kernel._last_dim_contig(rotary_cos)
        rotary_sin = _kernel._last_dim_contig(rotary_sin)
        cos, sin = rotary_cos.data_ptr(), rotary_sin.data_ptr()
        cos_row, sin_row = rotary_cos.stride(0), rotary_sin.stride(0)
    elif rotary_cos is not None or rotary_sin is not None:
        raise ValueError("mtlflashattn_b200: rotary_cos and rotary_sin go together")
    rot_code = _side("rotary_cos and rotary_sin", rotary_cos, rotary_sin, code, dtype)
    if positions is not None:
        if positions.dtype is torch.int64:
            pos64 = 1
        elif positions.dtype is not torch.int32:
            raise ValueError("mtlflashattn_b200: positions must be int32 or int64")
        ps = positions.shape
        if nd == 4 and ps == (B, L):
            pos_b, pos_l = positions.stride()
        elif ps == (L,):
            pos_l = positions.stride(0)
        else:
            raise ValueError(f"mtlflashattn_b200: positions must be one per token, got {tuple(ps)}")
        same = same and positions.get_device() == index
        pos = positions.data_ptr()
    if not same:
        raise ValueError("mtlflashattn_b200: all tensors must be on q's device")
    dev = q.device
    x, y = q, k
    qs, ks = q.stride(), k.stride()
    if qs[-1] != 1:
        x = q.contiguous()
        qs = x.stride()
    if ks[-1] != 1:
        y = k.contiguous()
        ks = y.stride()
    if nd == 3:
        qs, ks = (0, *qs), (0, *ks)
    q_out = torch.empty(q_shape, dtype=dtype, device=dev)
    k_out = torch.empty(k_shape, dtype=dtype, device=dev)
    p = _kernel._scratch("norm_rope", _FORMAT)
    _FORMAT.pack_into(
        p, 0, x.data_ptr(), y.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), qs[0], qs[1], qs[2],
        ks[0], ks[1], ks[2], wq, wk, cos, sin, cos_row, sin_row, pos, pos_b, pos_l, B, L, Hq, Hkv,
        D, R, min(rows, 2**31 - 1), pos64, code, w_code, rot_code, bool(interleaved), eps,
        _kernel._err_ptr(dev))
    _kernel._call(dev, "qk_norm_rope", _lib.qk_norm_rope, p)
    if torch.is_grad_enabled():
        extra = (q, k, q_weight, k_weight, rotary_cos, rotary_sin)
        return _guard_grad(q_out, *extra), _guard_grad(k_out, *extra)
    return q_out, k_out
