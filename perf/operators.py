"""Cases of the operators that surround the attention forward in a serving loop with a long,
4-bit cache: per-head norms with the position rotation, sliding-window attention whose first
tokens stay visible, appending keys and values to a paged 4-bit cache, and attention over that
cache. ``run`` computes them in a plain form (elementary torch operations, in 32 bits) or, where
``own`` is true, through this package's entry points.

The cache. A group of 16 consecutive values of one head of one token shares a scale in e4m3,
scale = e4m3(min(max|x| / 6, 448)), and each value is held as e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6
and a sign), the nearest to x / scale with ties to the even code. Pages of tokens hold
  codes   [pages, kv heads, page size, D / 2]   two codes per byte, the first in the low half
  scales  [pages, kv heads, page size, D / 16]  one e4m3 byte per group
Within a token's row of codes the dims are permuted (d = 16 i + j):
  keys    byte (j / 4) (D / 8) + 2 i + (j % 4) / 2, half (j % 4) % 2
  values  byte (j % 8) (D / 16) + i, half j / 8
"""
import math
import random

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token for each of 8 sequences: latency
        dict(name="norm_rope decode", op="norm_rope", B=8, L=1, Hq=32, Hkv=8, D=128, R=128,
             interleaved=False, dtype="bf16"),
        # a ragged chunk: odd length, D = 64, rotation of half the dims in interleaved pairs
        dict(name="norm_rope chunk", op="norm_rope", B=3, L=333, Hq=16, Hkv=16, D=64, R=32,
             interleaved=True, dtype="fp16"),
        # prefill of 16 sequences, GQA 32/8
        dict(name="norm_rope prefill", op="norm_rope", B=16, L=1024, Hq=32, Hkv=8, D=128, R=128,
             interleaved=False, dtype="bf16"),
        # prefill of one long sequence, 16 heads, D = 128
        dict(name="sink prefill", op="sink", varlen=False, B=1, Lq=8192, Lk=8192, Hq=16, Hkv=16,
             D=128, left=1024, sink=4, dtype="bf16"),
        # packed sequences of different lengths, GQA 32/8, odd window
        dict(name="sink varlen", op="sink", varlen=True, B=7, Lq=1999, Lk=1999, Hq=32, Hkv=8,
             D=64, left=255, sink=16, dtype="fp16"),
        # single tokens against long caches
        dict(name="sink decode", op="sink", varlen=False, B=4, Lq=1, Lk=16384, Hq=64, Hkv=8,
             D=128, left=4095, sink=4, dtype="bf16"),
        # one token for each of 64 sequences, read back
        dict(name="append decode", op="append", B=64, L=1, Hkv=8, D=128, page=16, dtype="bf16"),
        # the prompts of two sequences
        dict(name="append prefill", op="append", B=2, L=8192, Hkv=8, D=128, page=64,
             dtype="bf16"),
        # one sequence's next token at a moderate length: latency
        dict(name="attend short", op="attend", B=1, Lq=1, Lk=4096, Hq=32, Hkv=8, D=128, page=64,
             left=-1, sink=0, dtype="bf16"),
        # a serving batch with ragged lengths
        dict(name="attend batch", op="attend", B=32, Lq=1, Lk=8192, Hq=32, Hkv=8, D=128, page=64,
             left=-1, sink=0, dtype="bf16"),
        # one very long sequence
        dict(name="attend long", op="attend", B=1, Lq=1, Lk=131072, Hq=64, Hkv=8, D=128, page=128,
             left=-1, sink=0, dtype="fp16"),
        # a chunk of a prompt against what is cached, window and first tokens, odd sizes
        dict(name="attend chunk", op="attend", B=2, Lq=509, Lk=8001, Hq=16, Hkv=4, D=64, page=32,
             left=4000, sink=8, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm_rope", "sink", "append", "attend"))
    Hkv = rng.choice((1, 2, 4, 8))
    Hq = Hkv * rng.choice((1, 2, 3, 4, 5, 8))
    page = rng.choice((16, 32, 64, 128))
    if op == "norm_rope":
        D = rng.choice((32, 64, 80, 96, 128))
        L = _log(rng, 1, 2048)
        B = max(1, min(_log(rng, 1, 64), 16384 * 5120 // (L * (Hq + Hkv) * D)))
        return dict(op=op, B=B, L=L, Hq=Hq, Hkv=Hkv, D=D, R=rng.choice((D, D // 2)),
                    interleaved=rng.random() < 0.5, dtype=rng.choice(("fp16", "bf16", "fp32")))
    dtype = rng.choice(("fp16", "bf16"))
    if op == "sink":
        D = rng.choice((32, 64, 128))
        sink, left = _log(rng, 1, 150), _log(rng, 1, 5000)
        if rng.random() < 0.5:
            L = _log(rng, 30, 4096)
            B = max(1, min(rng.randint(1, 9), 2 * 10**8 // (L * L * Hq)))
            return dict(op=op, varlen=rng.random() < 0.5, B=B, Lq=L, Lk=L, Hq=Hq, Hkv=Hkv, D=D,
                        left=left, sink=sink, dtype=dtype)
        Lk = _log(rng, 100, 16384)
        return dict(op=op, varlen=False, B=rng.randint(1, 4), Lq=min(Lk, rng.choice((1, 1, 3, 16))),
                    Lk=Lk, Hq=Hq, Hkv=Hkv, D=D, left=left, sink=sink, dtype=dtype)
    D = rng.choice((64, 128))
    if op == "append":
        L = _log(rng, 1, 8192)
        return dict(op=op, B=max(1, min(_log(rng, 1, 64), 16384 // L)), L=L, Hkv=Hkv, D=D,
                    page=page, dtype=dtype)
    Lk = _log(rng, 60, 65536)
    B = max(1, min(_log(rng, 1, 32), 200000 // Lk))
    Lq = min(Lk, rng.choice((1, 1, 1, 2, 5, 16, _log(rng, 17, 600))))
    while Lq > 1 and B * Lq * Lk * Hq > 3 * 10**8:
        Lq = max(1, Lq // 2)
    windowed = rng.random() < 0.5
    return dict(op=op, B=B, Lq=Lq, Lk=Lk, Hq=Hq, Hkv=Hkv, D=D, page=page,
                left=_log(rng, 16, 8192) if windowed else -1,
                sink=_log(rng, 1, 100) if windowed else 0, dtype=dtype)


def _lens(c, least):
    """Lengths of the case's sequences: the first has the full length, the others any."""
    rng = random.Random("%d %d" % (c["B"], c["Lk"]))
    return [c["Lk"]] + [rng.randint(least, c["Lk"]) for _ in range(c["B"] - 1)]


# ------------------------------------------------------------------- the 4-bit form, in torch
def _nibble(x, scale):
    """e2m1 code (0..15) nearest to x / scale; every comparison is of exact products."""
    a = x.abs()
    c = (a > 0.25 * scale).to(torch.uint8)
    c += a >= 0.75 * scale
    c += a > 1.25 * scale
    c += a >= 1.75 * scale
    c += a > 2.5 * scale
    c += a >= 3.5 * scale
    c += a > 5.0 * scale
    c = torch.where(scale > 0, c, torch.zeros_like(c))
    return c | ((x < 0).to(torch.uint8) << 3)


def _quantise(x):
    """x [..., D] -> codes [..., D] uint8 and e4m3 scales [..., D / 16]."""
    g = x.float().unflatten(-1, (-1, 16))
    s = (g.abs().amax(-1) / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn)
    return _nibble(g, s.float()[..., None]).flatten(-2), s


def _bytes(n):
    n = n.unflatten(-1, (-1, 2))
    return n[..., 0] | (n[..., 1] << 4)


def _pack_k(codes):
    i = codes.shape[-1] // 16
    return _bytes(codes.unflatten(-1, (i, 4, 4)).transpose(-3, -2).flatten(-3))


def _pack_v(codes):
    i = codes.shape[-1] // 16
    return _bytes(codes.unflatten(-1, (i, 2, 8)).movedim(-1, -3).flatten(-3))


def _values(packed, scales):
    """The values of a permuted row, in 32 bits, still permuted: [..., bytes, 2]."""
    n = torch.stack((packed & 15, packed >> 4), -1)
    mag = torch.tensor(LEVELS, device=n.device)[(n & 7).int()]
    return torch.where(n > 7, -mag, mag)


def _unpack_k(packed, scales):
    x = _values(packed, scales).flatten(-2)
    x = x.unflatten(-1, (4, -1, 4)).transpose(-3, -2).flatten(-2)
    return (x * scales.float()[..., None]).flatten(-2)


def _unpack_v(packed, scales):
    x = _values(packed, scales).flatten(-2)
    x = x.unflatten(-1, (8, -1, 2)).movedim(-3, -1).flatten(-2)
    return (x * scales.float()[..., None]).flatten(-2)


def _cached(s, table):
    """Keys and values of the pages in ``table``, 32 bits: [B, kv heads, tokens, D] each."""
    t = table.long()
    k = _unpack_k(s["k"][t], s["k_scale"][t])
    v = _unpack_v(s["v"][t], s["v_scale"][t])
    return k.transpose(1, 2).flatten(2, 3), v.transpose(1, 2).flatten(2, 3)


# ----------------------------------------------------------------------------------- prepare
def _cache(c, g, dev, tokens):
    """Empty pages for the case's sequences, handed out in no order, and the block table."""
    each = -(-tokens // c["page"])
    pages = c["B"] * each
    shape = (pages, c["Hkv"], c["page"])
    s = dict(
        k=torch.zeros(*shape, c["D"] // 2, dtype=torch.uint8, device=dev),
        v=torch.zeros(*shape, c["D"] // 2, dtype=torch.uint8, device=dev),
        k_scale=torch.zeros(*shape, c["D"] // 16, device=dev).to(torch.float8_e4m3fn),
        v_scale=torch.zeros(*shape, c["D"] // 16, device=dev).to(torch.float8_e4m3fn),
        table=torch.randperm(pages, device=dev, generator=g).to(torch.int32).view(c["B"], each))
    return s


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    if c["op"] == "norm_rope":
        # q, k and v leave one fused projection; positions lie anywhere in a long context
        heads = c["Hq"] + 2 * c["Hkv"]
        qkv = (3 * normal(c["B"], c["L"], heads, c["D"])).to(dt)
        far = 32768
        freq = 10000.0 ** (-torch.arange(0, c["R"], 2, device=dev, dtype=torch.float64) / c["R"])
        angle = torch.arange(far, device=dev, dtype=torch.float64)[:, None] * freq
        first = torch.randint(0, far - c["L"] + 1, (c["B"], 1), device=dev, generator=g)
        return dict(case=c, q=qkv[:, :, :c["Hq"]], k=qkv[:, :, c["Hq"]:c["Hq"] + c["Hkv"]],
                    q_weight=(1 + 0.2 * normal(c["D"])).to(dt),
                    k_weight=(1 + 0.2 * normal(c["D"])).to(dt),
                    cos=angle.cos().float(), sin=angle.sin().float(),
                    positions=first + torch.arange(c["L"], device=dev))
    if c["op"] == "sink":
        if c["varlen"]:
            lens = _lens(c, 1)
            cu = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
            rows = sum(lens)
            return dict(case=c, lens=lens, cu=cu, longest=max(lens),
                        q=normal(rows, c["Hq"], c["D"]).to(dt),
                        k=normal(rows, c["Hkv"], c["D"]).to(dt),
                        v=normal(rows, c["Hkv"], c["D"]).to(dt))
        return dict(case=c, q=normal(c["B"], c["Lq"], c["Hq"], c["D"]).to(dt),
                    k=normal(c["B"], c["Lk"], c["Hkv"], c["D"]).to(dt),
                    v=normal(c["B"], c["Lk"], c["Hkv"], c["D"]).to(dt))
    if c["op"] == "append":
        # sequences that already hold up to 100 tokens when there is one new one, else none
        old = 100 if c["L"] == 1 else 0
        start = torch.randint(0, old + 1, (c["B"],), device=dev, generator=g).to(torch.int32)
        s = _cache(c, g, dev, old + c["L"])
        return dict(s, case=c, start=start, end=start + c["L"],
                    new_k=(2 * normal(c["B"], c["L"], c["Hkv"], c["D"])).to(dt),
                    new_v=normal(c["B"], c["L"], c["Hkv"], c["D"]).to(dt))
    s = _cache(c, g, dev, c["Lk"])
    pages = s["k"].shape[0]
    step = max(1, 2**27 // (c["Hkv"] * c["page"] * c["D"]))
    for i in range(0, pages, step):
        shape = (min(step, pages - i), c["Hkv"], c["page"], c["D"])
        for x, pack, name in ((2 * normal(*shape), _pack_k, "k"), (normal(*shape), _pack_v, "v")):
            codes, scale = _quantise(x.to(dt))
            s[name][i:i + step] = pack(codes)
            s[name + "_scale"][i:i + step] = scale
    lens = torch.tensor(_lens(c, c["Lq"]), dtype=torch.int32, device=dev)
    return dict(s, case=c, seqlens=lens, q=normal(c["B"], c["Lq"], c["Hq"], c["D"]).to(dt))


# ------------------------------------------------------------------------------- plain forms
def _norm_rope(x, weight, cos, sin, c):
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    r, rest = y[..., :c["R"]], y[..., c["R"]:]
    if c["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = r.chunk(2, -1)
        r = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((r, rest), -1).to(TYPES[c["dtype"]])


def _attention(q, k, v, visible):
    """q [B, Lq, Hq, D]; k, v [B, Hkv, Lk, D], 32 bits; visible [B or 1, Lq, Lk]."""
    B, Lq, Hq, D = q.shape
    Hkv = k.shape[1]
    q = q.float().view(B, Lq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)  # [B, Hkv, G, Lq, D]
    s = q.flatten(2, 3) @ k.transpose(-1, -2) * (1.0 / math.sqrt(D))
    s = s.unflatten(2, (Hq // Hkv, Lq)).masked_fill_(~visible[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (Hq // Hkv, Lq)) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Lq, Hq, D)


def _visible(lq, lk, n, m, left, sink, dev):
    """[B, n, m]: key j is seen by row i of a sequence of lq rows and lk keys."""
    i = torch.arange(n, device=dev)[None, :, None] + (lk - lq)[:, None, None]
    j = torch.arange(m, device=dev)[None, None, :]
    seen = j <= i
    if left >= 0:
        seen &= (j >= i - left) | (j < sink)
    return seen & (j < lk[:, None, None])


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    if c["op"] == "norm_rope":
        cos, sin = (s[t][s["positions"]][:, :, None] for t in ("cos", "sin"))
        return (_norm_rope(s["q"], s["q_weight"], cos, sin, c),
                _norm_rope(s["k"], s["k_weight"], cos, sin, c))
    dt = TYPES[c["dtype"]]
    if c["op"] == "sink":
        dev = s["q"].device
        q, k, v = s["q"], s["k"], s["v"]
        if c["varlen"]:
            # padded to the longest sequence, and packed again
            lens = (s["cu"][1:] - s["cu"][:-1]).long()
            n = s["longest"]
            held = torch.arange(n, device=dev) < lens[:, None]
            at = (s["cu"][:-1, None] + torch.arange(n, device=dev)).clamp(max=q.shape[0] - 1)
            q, k, v = q[at], k[at], v[at]
            seen = _visible(lens, lens, n, n, c["left"], c["sink"], dev)
            o = _attention(q, k.float().transpose(1, 2), v.float().transpose(1, 2), seen)
            return o[held].to(dt)
        lq, lk = (torch.full((1,), n, device=dev) for n in (c["Lq"], c["Lk"]))
        seen = _visible(lq, lk, c["Lq"], c["Lk"], c["left"], c["sink"], dev)
        return _attention(q, k.float().transpose(1, 2), v.float().transpose(1, 2), seen).to(dt)
    dev = s["table"].device
    if c["op"] == "append":
        at = s["start"][:, None].long() + torch.arange(c["L"], device=dev)
        page = s["table"].long().gather(1, at // c["page"])
        slot = at % c["page"]
        for x, pack, name in ((s["new_k"], _pack_k, "k"), (s["new_v"], _pack_v, "v")):
            codes, scale = _quantise(x)
            s[name][page, :, slot] = pack(codes)
            s[name + "_scale"].view(torch.uint8)[page, :, slot] = scale.view(torch.uint8)
        k, v = (f(s[n][page, :, slot], s[n + "_scale"].view(torch.uint8)[page, :, slot]
                  .view(torch.float8_e4m3fn)).to(dt)
                for n, f in (("k", _unpack_k), ("v", _unpack_v)))
        return k, v
    k, v = _cached(s, s["table"])
    lens = s["seqlens"].long()
    seen = _visible(torch.full_like(lens, c["Lq"]), lens, c["Lq"], k.shape[2], c["left"],
                    c["sink"], dev)
    held = torch.arange(k.shape[2], device=dev) < lens[:, None]
    v = v.masked_fill_(~held[:, None, :, None], 0.0)
    return _attention(s["q"], k, v, seen).to(dt)


def _run_own(s, c):
    import mtlflashattn_b200 as mfa
    if c["op"] == "norm_rope":
        return mfa.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"],
                                s["positions"], eps=1e-6, interleaved=c["interleaved"])
    window = (c.get("left", -1), -1)
    if c["op"] == "sink":
        if c["varlen"]:
            return mfa.flash_attn_varlen_func(
                s["q"], s["k"], s["v"], s["cu"], s["cu"], s["longest"], s["longest"],
                causal=True, window_size=window, sink_tokens=c["sink"])
        return mfa.flash_attn_func(s["q"], s["k"], s["v"], causal=True, window_size=window,
                                   sink_tokens=c["sink"])
    cache = mfa.KV4Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if c["op"] == "append":
        mfa.kv4_append(cache, s["new_k"], s["new_v"], s["table"], s["start"])
        return mfa.kv4_gather(cache, s["table"], s["end"], c["L"], starts=s["start"],
                              dtype=TYPES[c["dtype"]])
    return mfa.flash_attn_with_kv4cache(s["q"], cache, s["table"], s["seqlens"], causal=True,
                                        window_size=window, sink_tokens=c["sink"])


# -------------------------------------------------------------------------------------- work
def _pairs(lq, lk, left, sink):
    """(query, key) pairs that are visible, and how many keys any row sees."""
    total, low = 0, lk
    i = torch.arange(lk - lq, lk)
    lo = (i - left).clamp(min=0) if left >= 0 else torch.zeros_like(i)
    low = int(lo.min()) if lq else lk
    first = torch.minimum(lo, torch.tensor(min(sink, lk))) if left >= 0 else torch.zeros_like(i)
    total = int((i + 1 - lo + first).sum())
    return total, lk - low + min(low, sink if left >= 0 else 0)


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "norm_rope":
        n = c["B"] * c["L"] * (c["Hq"] + c["Hkv"]) * c["D"]
        tables = c["B"] * c["L"] * (c["R"] * 4 + 8)
        return {"bytes": 2 * n * size + tables + 2 * c["D"] * size, "flops": 9 * n}
    if c["op"] == "append":
        n = 2 * c["B"] * c["L"] * c["Hkv"] * c["D"]
        held = n // 2 + n // 16
        # rows in and the cache out, then the cache in and the values out
        return {"bytes": 2 * n * size + 2 * held, "flops": 6 * n}
    lens = _lens(c, c["Lq"]) if c["op"] == "attend" else \
        _lens(c, 1) if c["varlen"] else [c["Lk"]] * c["B"]
    pairs = keys = rows = 0
    for n in lens:
        lq = n if c["op"] == "sink" and c["varlen"] else c["Lq"]
        p, k = _pairs(lq, n, c["left"], c["sink"])
        pairs, keys, rows = pairs + p, keys + k, rows + lq
    io = 2 * rows * c["Hq"] * c["D"] * size
    row = c["D"] * size if c["op"] == "sink" else c["D"] // 2 + c["D"] // 16
    return {"bytes": io + 2 * keys * c["Hkv"] * row, "flops": 4 * c["D"] * pairs * c["Hq"]}


# ------------------------------------------------------------------------------------- exact
def _exact_rows(q, k, v, left, sink):
    """One sequence, one query head at a time, 64 bits: q [Lq, Hq, D], k, v [Lk, Hkv, D]."""
    Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[:2]
    out = torch.zeros(Lq, Hq, D, dtype=torch.float64, device=q.device)
    at = torch.arange(Lk - Lq, Lk, device=q.device)
    key = torch.arange(Lk, device=q.device)
    for a in range(0, Lq, 2048):
        n = at[a:a + 2048, None]
        hidden = key > n
        if left >= 0:
            hidden |= (key < n - left) & (key >= sink)
        for h in range(Hq):
            kv = h // (Hq // Hkv)
            s = q[a:a + 2048, h].double() @ k[:, kv].double().T / math.sqrt(D)
            s.masked_fill_(hidden, -math.inf)
            out[a:a + 2048, h] = torch.softmax(s, -1).nan_to_num_(0.0) @ v[:, kv].double()
    return out


def _exact_held(x):
    """What the cache stands for after x [..., D] was put in: nearest level, ties to even."""
    x = x.double()
    parts = []
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    for a in range(0, x.shape[-1], 16):
        p = x[..., a:a + 16]
        # the scale is e4m3 by definition: the quotient is rounded to it, by way of 32 bits
        s = (p.abs().amax(-1, keepdim=True) / 6).float().clamp(max=448)
        s = s.to(torch.float8_e4m3fn).double()
        y = torch.where(s > 0, p.abs() / torch.where(s > 0, s, 1.0), 0.0)
        off = (y[..., None] - levels).abs()
        # of two levels as near, the one of even index
        best = (off + torch.arange(8, device=x.device).remainder(2) * 1e-9).argmin(-1)
        parts.append(torch.copysign(levels[best], p) * s)
    return torch.cat(parts, -1)


def _exact_rotated(x, weight, cos, sin, c):
    x = x.double()
    y = x / (x.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-6).sqrt() * weight.double()
    half = c["R"] // 2
    out = y.clone()
    for p in range(half):
        a, b = (2 * p, 2 * p + 1) if c["interleaved"] else (p, p + half)
        co, si = cos[..., p], sin[..., p]
        out[..., a] = y[..., a] * co - y[..., b] * si
        out[..., b] = y[..., b] * co + y[..., a] * si
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "norm_rope":
        cos, sin = (s[t].double()[s["positions"].flatten()].view(c["B"], c["L"], 1, -1)
                    for t in ("cos", "sin"))
        return (_exact_rotated(s["q"], s["q_weight"], cos, sin, c),
                _exact_rotated(s["k"], s["k_weight"], cos, sin, c))
    if c["op"] == "append":
        return _exact_held(s["new_k"]), _exact_held(s["new_v"])
    if c["op"] == "sink":
        if not c["varlen"]:
            return torch.stack([_exact_rows(s["q"][b], s["k"][b], s["v"][b], c["left"], c["sink"])
                                for b in range(c["B"])])
        at = s["cu"].tolist()
        return torch.cat([_exact_rows(s["q"][a:b], s["k"][a:b], s["v"][a:b], c["left"], c["sink"])
                          for a, b in zip(at, at[1:])])
    out = []
    D, page = c["D"], c["page"]
    d = torch.arange(D, device="cuda")
    i, j = d // 16, d % 16
    place = {"k": ((j // 4) * (D // 8) + 2 * i + (j % 4) // 2, (j % 4) % 2),
             "v": ((j % 8) * (D // 16) + i, j // 8)}
    for b, n in enumerate(s["seqlens"].tolist()):
        at = torch.arange(n, device="cuda")
        page_of, slot = s["table"][b, at // page].long(), at % page
        kv = []
        for name in ("k", "v"):
            byte, half = place[name]
            code = (s[name][page_of, :, slot][..., byte] >> (4 * half)) & 15
            e, m = (code >> 1) & 3, (code & 1).double()
            size = torch.where(e == 0, m / 2, (1 + m / 2) * 2.0 ** (e.double() - 1))
            sign = 1 - 2 * (code >> 3).double()
            scale = s[name + "_scale"].view(torch.uint8)[page_of, :, slot]
            kv.append(sign * size * scale.view(torch.float8_e4m3fn).double()[..., i])
        out.append(_exact_rows(s["q"][b], kv[0], kv[1], c["left"], c["sink"]))
    return torch.stack(out)
