"""The 4-bit cache's definition in plain torch: quantisation, the layout of its rows, and the
values that they stand for. Test infrastructure, as the rest of this package."""
import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantise(x, unit=1.0):
    """x [..., D] -> (codes [..., D] int64 in 0..15, scales [..., D / 16] e4m3)."""
    g = x.double().unflatten(-1, (x.shape[-1] // 16, 16)) / unit
    top = g.abs().amax(-1)  # amax passes a NaN on
    s8 = torch.clamp((top / 6.0).float(), max=448.0).to(torch.float8_e4m3fn)
    s = s8.double()[..., None]
    a = g.abs()
    # borders between neighbouring codes; a value on a border goes to the even one
    code = torch.zeros_like(a, dtype=torch.int64)
    for n, border in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a > border * s) | ((a == border * s) & (n % 2 == 1))
    code = torch.where(s > 0, code, torch.zeros_like(code))  # also for a NaN scale
    code = code + 8 * (g < 0)
    return code.flatten(-2), s8


def value(codes, scales, unit=1.0):
    """What codes [..., D] with scales [..., D / 16] stand for, in 64 bits."""
    mag = torch.tensor(MAGNITUDES, dtype=torch.float64, device=codes.device)[codes & 7]
    x = torch.where(codes >= 8, -mag, mag).unflatten(-1, (codes.shape[-1] // 16, 16))
    return (x * scales.double()[..., None] * unit).flatten(-2)


def held(x, unit=1.0):
    """What the cache stands for after x [..., D] was appended, in 64 bits."""
    return value(*quantise(x, unit), unit)


def places(D, keys):
    """(byte, half) of each dim within a row."""
    d = torch.arange(D)
    i, j = d // 16, d % 16
    if keys:
        return (j // 4) * (D // 8) + 2 * i + (j % 4) // 2, (j % 4) % 2
    return (j % 8) * (D // 16) + i, j // 8


def unpack(rows, keys):
    """Byte rows [..., D / 2] -> codes [..., D]."""
    byte, half = (t.to(rows.device) for t in places(2 * rows.shape[-1], keys))
    return (rows[..., byte].to(torch.int64) >> (4 * half)) & 15


def tokens(cache, table, length, keys):
    """Tokens [0, length) of the pages in ``table`` (a 1-D row of a block table), in 64 bits:
    [length, Hkv, D]."""
    at = torch.arange(length, device=cache.k.device)
    page, slot = table.long()[at // cache.page_size], at % cache.page_size
    rows = (cache.k if keys else cache.v)[page, :, slot]
    scales = (cache.k_scale if keys else cache.v_scale).view(torch.uint8)[page, :, slot]
    return value(unpack(rows, keys), scales.view(torch.float8_e4m3fn),
                 cache.k_unit if keys else cache.v_unit)


def attention(q, k, v, causal=False, window=(-1, -1), softcap=0.0, slopes=None, sink=0,
              scale=None):
    """One sequence in 64 bits: q [Lq, Hq, D], k, v [Lk, Hkv, D]. Masked keys do not count at all,
    whatever they hold; a row without keys is 0."""
    Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[:2]
    q, k, v = q.double(), k.double(), v.double()
    c = torch.arange(Lk - Lq, Lk, device=q.device)[:, None]
    j = torch.arange(Lk, device=q.device)[None]
    seen = torch.ones(Lq, Lk, dtype=torch.bool, device=q.device)
    if window[0] >= 0:
        seen &= (j >= c - window[0]) | (j < sink)
    if window[1] >= 0:
        seen &= j <= c + window[1]
    if causal:
        seen &= j <= c
    out = torch.zeros(Lq, Hq, D, dtype=torch.float64, device=q.device)
    for i in range(Lq):
        if not bool(seen[i].any()):
            continue
        kk = k[seen[i]].repeat_interleave(Hq // Hkv, 1)
        vv = v[seen[i]].repeat_interleave(Hq // Hkv, 1)
        s = torch.einsum("hd,nhd->hn", q[i], kk) * (scale if scale is not None else D**-0.5)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            s = s - slopes.double()[:, None] * (c[i] - j[0][seen[i]]).abs()
        out[i] = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), vv)
    return out
