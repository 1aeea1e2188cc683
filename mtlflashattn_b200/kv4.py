"""A paged key/value cache held in 4 bits, and attention over it (no counterpart in the
reference, whose block_table and KV cache are not supported).

Each group of 16 dims of one head of one token shares a scale in e4m3 and holds e2m1 codes: 4.5
bits a value, against 16. ``kv4_append`` quantises new rows into the sequences' pages,
``flash_attn_with_kv4cache`` attends over what is cached straight from the codes, ``kv4_gather``
reads tokens back. Sequences own pages through an int32 ``block_table`` [B, max_pages]: token t of
sequence b is slot t % page_size of page block_table[b, t // page_size]. All lengths and tables
stay on the device, so a decode step can be captured in a CUDA graph. A page index or token
outside of the pool is skipped, never dereferenced, and ``check_device_errors`` reports it.
"""
from __future__ import annotations

import math
import struct

import torch

from . import _kernel, _lib
from ._grad import _guard_grad
from ._kernel import _DTYPES, _broadcast_alibi_slopes, _check_sink

__all__ = ["KV4Cache", "kv4_cache", "kv4_append", "kv4_gather", "flash_attn_with_kv4cache"]

_CACHE = struct.Struct(_lib.KV4_CACHE_FORMAT)
_ROWS = struct.Struct(_lib.KV4_ROWS_FORMAT)
_FWD = struct.Struct(_lib.KV4_FWD_FORMAT)
_WS = struct.Struct("<QQ")
_I32 = torch.int32


def _is_unit(u):
    return isinstance(u, (int, float)) and math.frexp(u)[0] == 0.5 and 2.0**-14 <= u <= 2.0**4


class KV4Cache:
    """The pool of pages: ``k``/``v`` uint8 [num_pages, Hkv, page_size, D/2] and
    ``k_scale``/``v_scale`` float8_e4m3fn [num_pages, Hkv, page_size, D/16], contiguous CUDA
    tensors (for instance one layer's slice of a larger allocation). D is 64 or 128, page_size a
    power of two from 16 to 1024. ``k_unit``/``v_unit``, powers of two from 2^-14 to 2^4,
    multiply every held value: scales in e4m3 are finest for groups whose largest value lies
    between unit / 10 and 2688 unit."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "k_unit", "v_unit")

    def __init__(self, k, v, k_scale, v_scale, k_unit=1.0, v_unit=1.0):
        shape = k.shape
        if len(shape) != 4 or v.shape != shape:
            raise ValueError("mtlflashattn_b200: k and v must be [num_pages, Hkv, page_size, D/2]")
        scales = (shape[0], shape[1], shape[2], shape[3] // 8)
        if k_scale.shape != scales or v_scale.shape != scales:
            raise ValueError(
                f"mtlflashattn_b200: k_scale and v_scale must be {scales} (one per 16 dims)")
        e4m3 = torch.float8_e4m3fn
        if (k.dtype != torch.uint8 or v.dtype != torch.uint8 or k_scale.dtype != e4m3
                or v_scale.dtype != e4m3):
            raise ValueError("mtlflashattn_b200: codes are uint8 and scales float8_e4m3fn")
        if shape[3] not in (32, 64):
            raise NotImplementedError(
                f"mtlflashattn_b200: 4-bit cache of head_dim {2 * shape[3]} (64 or 128)")
        size = shape[2]
        if size < 16 or size > 1024 or size & (size - 1):
            raise NotImplementedError(
                f"mtlflashattn_b200: page_size {size} (a power of two from 16 to 1024)")
        if shape[1] == 0:
            raise ValueError("mtlflashattn_b200: the cache needs at least one head")
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous()
                and v_scale.is_contiguous()):
            raise ValueError("mtlflashattn_b200: the cache's tensors must be contiguous")
        dev = k.device
        if v.device != dev or k_scale.device != dev or v_scale.device != dev:
            raise ValueError("mtlflashattn_b200: the cache's tensors must be on one device")
        if not (_is_unit(k_unit) and _is_unit(v_unit)):
            raise ValueError(
                "mtlflashattn_b200: k_unit and v_unit must be powers of two from 2^-14 to 2^4")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.k_unit, self.v_unit = float(k_unit), float(v_unit)
        if k.is_cuda:
            _kernel._err_ptr(dev)  # there before a first call that may be captured

    @property
    def num_pages(self):
        return self.k.shape[0]

    @property
    def page_size(self):
        return self.k.shape[2]

    @property
    def num_heads_kv(self):
        return self.k.shape[1]

    @property
    def head_dim(self):
        return 2 * self.k.shape[3]


def kv4_cache(num_pages, page_size, num_heads_kv, head_dim, device=None, k_unit=1.0, v_unit=1.0):
    """A new, zeroed ``KV4Cache`` (every token in it is held as 0)."""
    if head_dim not in (64, 128):
        raise NotImplementedError(
            f"mtlflashattn_b200: 4-bit cache of head_dim {head_dim} (64 or 128)")
    device = torch.device("cuda") if device is None else device
    shape = (num_pages, num_heads_kv, page_size)

    def zeros(n):
        return torch.zeros(*shape, n, dtype=torch.uint8, device=device)

    e4m3 = torch.float8_e4m3fn
    return KV4Cache(zeros(head_dim // 2), zeros(head_dim // 2), zeros(head_dim // 16).view(e4m3),
                    zeros(head_dim // 16).view(e4m3), k_unit, v_unit)


def _check_lens(name, t, B, index):
    if t.dtype is not _I32 or t.shape != (B,) or not t.is_contiguous():
        raise ValueError(f"mtlflashattn_b200: {name} must be a contiguous int32 tensor of [{B}]")
    if t.get_device() != index:
        raise ValueError("mtlflashattn_b200: all tensors must be on the cache's device")


def _pack_cache(cache, block_table, B, dev, max_seqlen=None):
    """The cache and table as ``mfa_kv4_cache`` in this thread's buffer; ``max_seqlen``: only as
    many of the table's columns as hold that many tokens."""
    if not isinstance(cache, KV4Cache):
        raise TypeError("mtlflashattn_b200: cache must be a KV4Cache")
    k = cache.k
    index = k.get_device()
    if index < 0:
        raise NotImplementedError(
            f"mtlflashattn_b200: device {k.device.type!r} not supported (CUDA only)")
    table = block_table.shape
    if block_table.dtype is not _I32 or len(table) != 2 or table[0] != B:
        raise ValueError(f"mtlflashattn_b200: block_table must be int32 [{B}, max_pages]")
    if dev.index != index or dev.type != "cuda" or block_table.get_device() != index:
        raise ValueError("mtlflashattn_b200: all tensors must be on the cache's device")
    pages, heads, size, half = k.shape
    max_pages = table[1] if max_seqlen is None else min(table[1], -(-max_seqlen // size))
    if max_pages * size > 2**31 - 4096:
        raise ValueError("mtlflashattn_b200: block_table covers more than 2^31 - 4096 tokens")
    stride = block_table.stride()
    if max_pages > 1 and stride[1] != 1:
        raise ValueError("mtlflashattn_b200: block_table must have a contiguous last dimension")
    p = _kernel._scratch("kv4_cache", _CACHE)
    _CACHE.pack_into(
        p, 0, k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(),
        cache.v_scale.data_ptr(), block_table.data_ptr(), stride[0], pages, size, heads, 2 * half,
        B, max_pages, cache.k_unit, cache.v_unit, _kernel._err_ptr(dev))
    return p


def _check_max_seqlen(n):
    if not isinstance(n, int) or isinstance(n, bool) or n < 0:
        raise ValueError("mtlflashattn_b200: max_seqlen must be an int >= 0")


def _in_pieces(t):
    """t, or a copy of it, with rows that can be read in 16-byte pieces."""
    sb, ss, sh, sd = t.stride()
    if sd != 1 or (sb | ss | sh) % 8 or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _pack_rows(k, v, start, lens):
    p = _kernel._scratch("kv4_rows", _ROWS)
    _ROWS.pack_into(
        p, 0, k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3],
        0 if start is None else start.data_ptr(), 0 if lens is None else lens.data_ptr(),
        k.shape[1], _DTYPES[k.dtype])
    return p


def kv4_append(cache, k, v, block_table, cache_seqlens, new_lens=None):
    """Quantise k, v [B, L, Hkv, D] (fp16/bf16, any strides) into the sequences' pages, in place.

    Row j of sequence b becomes token cache_seqlens[b] + j, where ``cache_seqlens`` (int32 [B]) is
    the length before the call; advancing it is the caller's. ``new_lens`` (int32 [B]): only the
    first new_lens[b] rows count, as in a padded batch. Rows without a page are skipped and
    reported by ``check_device_errors``. No two rows may go to one slot (pages that sequences
    share are read, not written): what such a slot then holds is undefined.

    A value x is held as code * scale * unit with, for its group of 16,
    scale = e4m3(min(max|x / unit| / 6, 448)) and code the e2m1 number nearest to
    x / unit / scale, ties to the even code. A NaN makes its whole group NaN.
    """
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError("mtlflashattn_b200: k and v must be [B, L, Hkv, D]")
    if k.dtype not in (torch.float16, torch.bfloat16) or v.dtype != k.dtype:
        raise NotImplementedError(f"mtlflashattn_b200: dtype {k.dtype} (k/v must match, fp16/bf16)")
    B, dev = k.shape[0], k.device
    c = _pack_cache(cache, block_table, B, dev)
    if v.device != dev:
        raise ValueError("mtlflashattn_b200: all tensors must be on the cache's device")
    if k.shape[2] != cache.num_heads_kv or k.shape[3] != cache.head_dim:
        raise ValueError("mtlflashattn_b200: k and v do not have the cache's heads and head_dim")
    _check_lens("cache_seqlens", cache_seqlens, B, dev.index)
    if new_lens is not None:
        _check_lens("new_lens", new_lens, B, dev.index)
    k, v = _in_pieces(k), _in_pieces(v)
    r = _pack_rows(k, v, cache_seqlens, new_lens)
    _kernel._call(dev, "kv4_append", _lib.kv4_append, c, r)


def kv4_gather(cache, block_table, cache_seqlens, max_seqlen, starts=None, dtype=torch.bfloat16):
    """Read tokens back: (k, v), each [B, max_seqlen, Hkv, D] in ``dtype`` (fp16/bf16/fp32).

    Row j of sequence b is token starts[b] + j (``starts``: int32 [B], None for 0); rows at or
    past ``cache_seqlens[b]`` are 0. The values are exactly those that the attention uses.
    """
    if dtype not in _DTYPES:
        raise NotImplementedError(f"mtlflashattn_b200: dtype {dtype} (fp16/bf16/fp32)")
    _check_max_seqlen(max_seqlen)
    B, dev = block_table.shape[0], block_table.device
    c = _pack_cache(cache, block_table, B, dev)
    _check_lens("cache_seqlens", cache_seqlens, B, dev.index)
    if starts is not None:
        _check_lens("starts", starts, B, dev.index)
    shape = (B, max_seqlen, cache.num_heads_kv, cache.head_dim)
    k = torch.empty(shape, dtype=dtype, device=dev)
    v = torch.empty(shape, dtype=dtype, device=dev)
    r = _pack_rows(k, v, starts, cache_seqlens)
    _kernel._call(dev, "kv4_gather", _lib.kv4_gather, c, r)
    return k, v


def flash_attn_with_kv4cache(q, cache, block_table, cache_seqlens, softmax_scale=None,
                             causal=False, window_size=(-1, -1), softcap=0.0, alibi_slopes=None,
                             sink_tokens=0, max_seqlen=None):
    """Attention of q [B, Lq, Hq, D] (fp16/bf16) over the cached keys and values (forward only).

    ``cache_seqlens`` (int32 [B]) counts the keys of each sequence; q holds its newest Lq rows,
    whose keys are appended before the call. Masks, scale, softcap, ALiBi and ``sink_tokens`` are
    those of ``flash_attn_func`` with k and v of length cache_seqlens[b]; a row that sees no key
    is 0. Pages whose tokens no row sees are not looked at: their entries in ``block_table`` may
    be anything (-1, or a page that others use by now). Returns [B, Lq, Hq, D] in q.dtype.

    ``max_seqlen``, an int that no length exceeds (None: the tokens that ``block_table`` has
    columns for). More than 48 query rows per KV head (16 at D = 64) are attended by way of keys and
    values in 16 bits: time and workspace of such calls follow this bound, not the lengths, so give
    it where the table is much wider than they are (the workspace, up to 512 MiB or one sequence's
    bound where that is more, is kept for the stream's next calls). A longer sequence is cut after
    the page of the bound's last token and reported by ``check_device_errors``.
    """
    if q.dim() != 4:
        raise ValueError(f"mtlflashattn_b200: expected 4-D [B,S,H,D] q, got q.dim()={q.dim()}")
    if (
        not isinstance(window_size, (tuple, list))
        or len(window_size) != 2
        or any(not isinstance(w, int) or isinstance(w, bool) or w < -1 for w in window_size)
    ):
        raise ValueError(
            "mtlflashattn_b200: window_size must be a (left, right) pair of ints >= -1 "
            "(-1 = unbounded on that side)"
        )
    if not softcap >= 0:
        raise ValueError("mtlflashattn_b200: softcap must be >= 0 (0 disables capping)")
    sink = _check_sink(sink_tokens)
    if max_seqlen is not None:
        _check_max_seqlen(max_seqlen)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise NotImplementedError(f"mtlflashattn_b200: dtype {q.dtype} (fp16/bf16)")
    B, Lq, Hq, D = q.shape
    dev = q.device
    c = _pack_cache(cache, block_table, B, dev, max_seqlen)
    Hkv = cache.num_heads_kv
    if D != cache.head_dim:
        raise ValueError("mtlflashattn_b200: q does not have the cache's head_dim")
    if Hq == 0 or Hq % Hkv != 0:
        raise ValueError(f"mtlflashattn_b200: num_heads_kv ({Hkv}) must divide num_heads_q ({Hq})")
    _check_lens("cache_seqlens", cache_seqlens, B, dev.index)
    alibi = None
    if alibi_slopes is not None:
        if not torch.is_tensor(alibi_slopes):
            raise TypeError("mtlflashattn_b200: alibi_slopes must be a tensor of per-head slopes")
        alibi = _broadcast_alibi_slopes(alibi_slopes, B, Hq, dev)
    x = _in_pieces(q)
    if 0 in x.stride():  # many broadcast rows would run on the CUDA cores: TMA takes no stride of 0
        x = x.contiguous()
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D)
    far = 2**31 - 1
    p = _kernel._scratch("kv4_fwd", _FWD)
    _FWD.pack_into(
        p, 0, x.data_ptr(), out.data_ptr(), *x.stride()[:3], *out.stride()[:3],
        cache_seqlens.data_ptr(), Lq, Hq, _DTYPES[q.dtype], scale, softcap, bool(causal),
        min(window_size[0], far), min(window_size[1], far), sink,
        0 if alibi is None else alibi.data_ptr(), 0, 0)
    _kernel._call(dev, "flash_attn_with_kv4cache", _launch, c, p, dev)
    return _guard_grad(out, q)


def _launch(c, p, dev, stream):
    with _kernel._workspace_lock:
        # the stream's workspace is usually there and large enough: no need to ask first
        ws = _kernel._workspaces.get((dev, stream))
        if ws is not None and not torch.cuda.is_current_stream_capturing():
            _WS.pack_into(p, _lib.KV4_FWD_WORKSPACE_OFFSET, ws.data_ptr(), ws.numel())
            rc = _lib.kv4_fwd(c, p, stream)
            if rc != _lib.ERR_SCRATCH_TOO_SMALL:
                return rc
        need = _lib.kv4_fwd_workspace_size(c, p)
        if need > 0:
            ws = _kernel._workspace(dev, stream, need)
            _WS.pack_into(p, _lib.KV4_FWD_WORKSPACE_OFFSET, ws.data_ptr(), need)
        return _lib.kv4_fwd(c, p, stream)
