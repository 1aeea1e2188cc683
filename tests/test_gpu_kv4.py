"""The paged 4-bit cache against its definition (oracle/kv4.py): what append holds, exactly, and
attention over it in 64 bits on the same held values."""
import pytest
import torch

import mtlflashattn_b200 as mfa
from mtlflashattn_b200 import _kernel, _lib
from oracle import kv4 as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def table_of(B, each, extra=0, seed=0):
    """A block table over shuffled pages: (int32 [B, each], number of pages)."""
    n = B * each + extra
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randperm(n, device=DEV, generator=g)[:B * each].view(B, each).int(), n


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def dirty(cache):
    """Every byte set, the scales to NaN: what memory may hold where nothing was appended."""
    cache.k.fill_(0xE7)
    cache.v.fill_(0x7E)
    cache.k_scale.view(torch.uint8).fill_(0x7F)
    cache.v_scale.view(torch.uint8).fill_(0xFF)
    return cache


def reported():
    with pytest.raises(_lib.MfaError):
        _kernel.check_device_errors()


# ---------------------------------------------------------------------------- append and gather
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("B,L,Hkv", [(1, 1, 1), (3, 1, 8), (2, 37, 3), (1, 130, 2)])
def test_append_holds_exactly_what_is_defined(dtype, D, page, B, L, Hkv):
    g = torch.Generator(device=DEV).manual_seed(B + L)
    start = [0, 13, 50][:B]
    each = -(-(50 + L) // page)
    table, pages = table_of(B, each, 2)
    cache = dirty(mfa.kv4_cache(pages, page, Hkv, D, DEV, k_unit=2.0**-3, v_unit=2.0))
    k, v = (torch.randn(B, L, Hkv, D, device=DEV, generator=g) for _ in range(2))
    k *= torch.exp(2 * torch.randn(B, L, Hkv, 1, device=DEV, generator=g))  # rows of other sizes
    k, v = k.to(dtype), v.to(dtype)
    before = [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    mfa.kv4_append(cache, k, v, table, i32(*start))
    end = i32(*(s + L for s in start))
    written = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
    for b, s in enumerate(start):
        for x, keys, unit in ((k, True, 2.0**-3), (v, False, 2.0)):
            got = ref.tokens(cache, table[b], s + L, keys)[s:]
            assert torch.equal(got, ref.held(x[b], unit))
        at = torch.arange(s, s + L, device=DEV)
        written[table[b].long()[at // page], at % page] = True
    for t, old in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), before):
        new = t.view(torch.uint8).transpose(1, 2)
        assert torch.equal(new[~written], old.transpose(1, 2)[~written])  # nothing else
    for out in (dtype, torch.float32):
        gk, gv = mfa.kv4_gather(cache, table, end, L + 3, starts=i32(*start), dtype=out)
        for x, got, unit in ((k, gk, 2.0**-3), (v, gv, 2.0)):
            want = torch.stack([ref.held(x[b], unit) for b in range(B)])
            assert got.dtype == out
            assert torch.equal(got[:, :L].double(), want) and bool((got[:, L:] == 0).all())
    _kernel.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_borders_zeros_and_what_is_not_finite(dtype):
    rows = []
    for top in (6.0, 0.75, 6 * 448.0, 6 * 2.0**-9, 6 * 13 * 2.0**-4, 3 * 2.0**-10, 1e-5, 3000.0):
        s = ref.quantise(torch.full((16,), top))[1].float().item()
        for sign in (1, -1):
            # every border of the codes and its neighbours, with the value that sets the scale
            borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]) * s * sign
            edge = borders.to(dtype)
            up = torch.nextafter(edge, torch.full_like(edge, 6e4))
            down = torch.nextafter(edge, torch.full_like(edge, -6e4))
            for x in (edge, up, down):
                rows.append(torch.cat((torch.tensor([top, 0.0]).to(dtype), x,
                                       torch.zeros(7, dtype=dtype))))
    nan, inf = float("nan"), float("inf")
    for special in ([0.0] * 16, [-0.0] * 16, [nan] + [1.0] * 15, [1.0] * 15 + [nan],
                    [inf] + [1.0] * 15, [2.0] * 7 + [-inf] + [3.0] * 8, [inf, nan] + [0.0] * 14,
                    [torch.finfo(dtype).max] * 16, [torch.finfo(dtype).smallest_normal] * 16,
                    [torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps] * 16):
        rows.append(torch.tensor(special).to(dtype))
    while len(rows) % 4:
        rows.append(torch.ones(16, dtype=dtype))
    x = torch.cat(rows).view(1, -1, 1, 64).to(DEV)
    L = x.shape[1]
    for unit in (1.0, 2.0**-14, 16.0):
        cache = dirty(mfa.kv4_cache(-(-L // 16), 16, 1, 64, DEV, k_unit=unit, v_unit=unit))
        table = torch.arange(cache.num_pages, device=DEV).int()[None]
        mfa.kv4_append(cache, x, x, table, i32(0))
        want = ref.held(x[0], unit)
        got = mfa.kv4_gather(cache, table, i32(L), L, dtype=torch.float32)
        for t in got:
            torch.testing.assert_close(t[0].double(), want, atol=0, rtol=0, equal_nan=True)
        # exact in 16 bits too, but where a saturated value passes the type's range
        half = mfa.kv4_gather(cache, table, i32(L), L, dtype=dtype)[0][0]
        torch.testing.assert_close(half.double(), want, atol=0, rtol=0, equal_nan=True)


def test_padded_rows_views_and_rows_without_a_page():
    B, L, Hkv, D, page = 4, 6, 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(7)
    qkv = torch.randn(B, L, 4 + 2 * Hkv, D, device=DEV, generator=g).bfloat16()
    k, v = qkv[:, :, 4:4 + Hkv], qkv[:, :, 4 + Hkv:]
    table, pages = table_of(B, 2)
    cache = dirty(mfa.kv4_cache(pages, page, Hkv, D, DEV))
    lens = (6, 0, 3, 99)  # the last: all of them
    mfa.kv4_append(cache, k, v, table, i32(0, 5, 14, 20), new_lens=i32(*lens))
    _kernel.check_device_errors()
    for b, (s, n) in enumerate(zip((0, 5, 14, 20), (6, 0, 3, 6))):
        got = ref.tokens(cache, table[b], 32, True)
        assert torch.equal(got[s:s + n], ref.held(k[b, :n]))
        rest = torch.ones(32, dtype=torch.bool)
        rest[s:s + n] = False
        assert bool(got[rest.to(DEV)].isnan().all())
    # outside of the table, a page that does not exist, a negative length: skipped and reported
    snap = [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    for start, spoil in ((32, None), (-6, None), (2**31 - 1, None), (0, pages), (0, -1),
                         (0, 2**31 - 1), (0, -2**31)):
        bad = table.clone()
        if spoil is not None:
            bad[1, 0] = spoil
        only = i32(0, 6, 0, 0)
        mfa.kv4_append(cache, k, v, bad, i32(0, start, 0, 0), new_lens=only)
        reported()
        for t, old in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), snap):
            assert torch.equal(t.view(torch.uint8), old)
        gk, gv = mfa.kv4_gather(cache, bad, i32(0, min(start, 2**31 - 8) + 6, 0, 0), 6,
                                starts=i32(0, min(start, 2**31 - 8), 0, 0))
        reported()
        assert bool((gk[1] == 0).all()) and bool((gv[1] == 0).all())
    # across the end of the table: the rows that have a page are written
    mfa.kv4_append(cache, k, v, table, i32(0, 29, 0, 0), new_lens=i32(0, 6, 0, 0))
    reported()
    assert torch.equal(ref.tokens(cache, table[1], 32, False)[29:], ref.held(v[1, :3]))


def test_pool_beyond_32_bits():
    page, Hkv, D = 1024, 8, 128
    pages = 2**31 // (page * Hkv * D // 2) + 9
    cache = mfa.kv4_cache(pages, page, Hkv, D, DEV)
    table = i32(pages - 1, 3, pages - 2).view(1, 3)
    g = torch.Generator(device=DEV).manual_seed(8)
    k, v = (torch.randn(1, 2 * page + 70, Hkv, D, device=DEV, generator=g).bfloat16()
            for _ in range(2))
    n = k.shape[1]
    mfa.kv4_append(cache, k, v, table, i32(0))
    gk, gv = mfa.kv4_gather(cache, table, i32(n), n)
    assert torch.equal(gk[0].double(), ref.held(k[0])) and torch.equal(gv[0].double(), ref.held(v[0]))
    q = torch.randn(1, 1, 8, D, device=DEV, generator=g).bfloat16()
    out = mfa.flash_attn_with_kv4cache(q, cache, table, i32(n), causal=True)
    check(out[0], ref.attention(q[0], gk[0], gv[0]), gv[0])
    _kernel.check_device_errors()


# ------------------------------------------------------------------------------------ attention
def check(out, want, v, rows=1, softcap=0.0):
    if rows > 64:  # the tensor-core forward: probabilities in the output's type, 7.5e-5 of the
        # exponentials from the FMA pipe, logits and output as below; softcap's hardware tanh moves
        # a logit by softcap * 2^-11, twice
        top = float(v.double().nan_to_num(0.0).abs().amax()) if v.numel() else 0.0
        step = torch.finfo(out.dtype).eps / 2
        torch.testing.assert_close(out.double(), want, rtol=step, equal_nan=True,
                                   atol=top * (step + 1.5e-4 + 2**-9 + 2 * softcap * 2**-11))
        return
    # Probabilities are rounded to fp16 and once more with the value's scale (2^-11 each), and are
    # off by what moves a logit: its fp32 sum of 128 products, 2^-16 of sum|q k| / sqrt(D) (under
    # 64 here) = 2^-10, twice (numerator and sum). With sum p = 1 that is 2^-8.4 max|v| at most.
    # Then one rounding to the output's type.
    top = v.double().nan_to_num(0.0).abs().amax() if v.numel() else 0.0
    step = torch.finfo(out.dtype).eps / 2
    torch.testing.assert_close(out.double(), want, atol=float(top) * 2**-8.4, rtol=step,
                               equal_nan=True)
    # as independent roundings they cancel: the 2-norm is far below the bound
    w = want.nan_to_num(0.0)
    off = (out.double().nan_to_num(0.0) - w).norm()
    assert off <= 2 * (step + 2**-11) * w.norm() + 1e-30


def filled(lens, page, Hkv, D, seed=0, **unit):
    """A cache of normal keys and values for sequences of these lengths, NaN everywhere else."""
    B = len(lens)
    each = max(1, -(-max(lens) // page))
    table, pages = table_of(B, each, 1, seed)
    cache = dirty(mfa.kv4_cache(pages, page, Hkv, D, DEV, **unit))
    g = torch.Generator(device=DEV).manual_seed(seed)
    L = max(max(lens), 1)
    k, v = (torch.randn(B, L, Hkv, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    mfa.kv4_append(cache, k, v, table, i32(*[0] * B), new_lens=i32(*lens))
    return cache, table, g


def compare(cache, table, lens, q, **kw):
    n = i32(*lens)
    out = mfa.flash_attn_with_kv4cache(q, cache, table, n, causal=kw.get("causal", False),
                                       window_size=kw.get("window", (-1, -1)),
                                       softcap=kw.get("softcap", 0.0),
                                       alibi_slopes=kw.get("slopes"),
                                       sink_tokens=kw.get("sink", 0),
                                       softmax_scale=kw.get("scale"))
    _kernel.check_device_errors()
    assert out.shape == q.shape and out.dtype == q.dtype
    for b, length in enumerate(lens):
        k = ref.tokens(cache, table[b], length, True)
        v = ref.tokens(cache, table[b], length, False)
        check(out[b], ref.attention(q[b], k, v, **kw), v, q.shape[1] * q.shape[2] // k.shape[1],
              kw.get("softcap", 0.0))
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 4, 4), (128, 32, 4), (64, 16, 1), (64, 6, 2),
                                      (128, 5, 1), (64, 24, 2)])
@pytest.mark.parametrize("Lq,page,kw", [
    (1, 16, dict(causal=True)),
    (1, 64, dict(causal=True, window=(100, -1), sink=5)),
    (3, 32, dict(causal=True)),
    (5, 128, dict(causal=True, window=(33, -1), sink=40)),
    (2, 16, dict(window=(20, 3), sink=1)),
    (7, 64, dict(causal=False, scale=-0.2)),
    (40, 16, dict(causal=True, window=(300, -1), sink=17)),
])
def test_attention_against_formula(dtype, D, Hq, Hkv, Lq, page, kw):
    lens = (0, 1, 15, 16, 17, 200, 531, 64)
    cache, table, g = filled(lens, page, Hkv, D, seed=Lq)
    q = torch.randn(len(lens), Lq, Hq, D, device=DEV, generator=g).to(dtype)
    compare(cache, table, lens, q, **kw)


@pytest.mark.parametrize("kw", [dict(softcap=20.0), dict(slopes=True),
                                dict(softcap=5.0, slopes=True, window=(200, -1), sink=9)])
@pytest.mark.parametrize("Lq", [1, 4])
def test_attention_softcap_alibi_units(kw, Lq):
    lens = (700, 3, 90)
    cache, table, g = filled(lens, 32, 2, 128, seed=3, k_unit=0.25, v_unit=2.0**-5)
    q = torch.randn(3, Lq, 8, 128, device=DEV, generator=g).half()
    if kw.get("slopes"):
        kw = dict(kw, slopes=torch.tensor([0.5 ** (i + 1) for i in range(8)], device=DEV))
    compare(cache, table, lens, q, causal=True, **kw)


@pytest.mark.parametrize("B,lk,Lq,Hq,Hkv", [(1, 20000, 1, 16, 2), (2, 5000, 1, 8, 8),
                                            (1, 9000, 3, 8, 1)])
def test_split_over_a_long_cache(B, lk, Lq, Hq, Hkv):
    lens = tuple(lk - 37 * b * b for b in range(B))
    cache, table, g = filled(lens, 64, Hkv, 128, seed=B)
    q = torch.randn(B, Lq, Hq, 128, device=DEV, generator=g).bfloat16()
    for kw in (dict(), dict(window=(3000, -1), sink=4), dict(window=(1, -1), sink=2500)):
        a = compare(cache, table, lens, q, causal=True, **kw)
        n = i32(*lens)
        again = mfa.flash_attn_with_kv4cache(q, cache, table, n, causal=True,
                                             window_size=kw.get("window", (-1, -1)),
                                             sink_tokens=kw.get("sink", 0))
        assert torch.equal(a, again)


@pytest.mark.parametrize("Lq,Hq,Hkv,D", [(130, 8, 2, 64), (300, 4, 4, 128), (257, 6, 1, 128)])
def test_chunk_of_a_prompt(Lq, Hq, Hkv, D):
    lens = (700, Lq, 0, 40)  # the last two: rows before the first key see nothing
    cache, table, g = filled(lens, 32, Hkv, D, seed=Lq)
    q = torch.randn(4, Lq, Hq, D, device=DEV, generator=g).bfloat16()
    compare(cache, table, lens, q, causal=True)
    compare(cache, table, lens, q, causal=True, window=(100, -1), sink=6)


def test_chunk_with_softcap_and_alibi():
    lens = (500, 260)
    cache, table, g = filled(lens, 64, 2, 128, seed=21, k_unit=0.5, v_unit=2.0**-4)
    q = torch.randn(2, 100, 8, 128, device=DEV, generator=g).half()
    slopes = torch.tensor([0.5 ** (i + 1) for i in range(8)], device=DEV)
    compare(cache, table, lens, q, causal=True, softcap=10.0, slopes=slopes, window=(90, -1), sink=5)
    compare(cache, table, lens, q, slopes=slopes)


@pytest.mark.parametrize("D,Hq,Hkv,Lq,page", [
    (64, 71, 1, 1, 64), (128, 71, 1, 1, 64),   # more heads per KV head than rows read directly
    (128, 48, 1, 1, 16), (128, 9, 1, 5, 1024), (64, 16, 1, 1, 1024), (64, 2, 2, 16, 16),
    (128, 7, 7, 1, 32), (128, 3, 1, 16, 128)])
def test_row_counts_and_pages(D, Hq, Hkv, Lq, page):
    lens = (300, 1025, Lq)
    cache, table, g = filled(lens, page, Hkv, D, seed=Hq)
    q = torch.randn(3, Lq, Hq, D, device=DEV, generator=g).bfloat16()
    compare(cache, table, lens, q, causal=True)
    compare(cache, table, lens, q, window=(70, 2), sink=3)
    compare(cache, table, lens, q, causal=True, window=(2**40, -1), sink=10**15)


@pytest.mark.parametrize("Hq,Lq", [(48, 1), (49, 1), (64, 1), (65, 1), (16, 4), (13, 5), (1, 49), (7, 9)])
def test_rows_around_the_direct_limit(Hq, Lq):
    """The last row counts whose codes are read directly, and the first that go through 16 bits."""
    lens = (1300, Lq, 700)
    cache, table, g = filled(lens, 32, 1, 128, seed=Hq)
    q = torch.randn(3, Lq, Hq, 128, device=DEV, generator=g).half()
    compare(cache, table, lens, q, causal=True)
    compare(cache, table, lens, q, causal=True, window=(200, -1), sink=130)


@pytest.mark.parametrize("B,Lq", [(400, 1), (333, 2)])
def test_more_sequences_than_threads(B, Lq):
    lens = tuple((7 * b * b) % 90 if b % 5 else 0 for b in range(B))
    cache, table, g = filled(lens, 16, 1, 64, seed=B)
    q = torch.randn(B, Lq, 3, 64, device=DEV, generator=g).half()
    compare(cache, table, lens, q, causal=True)


def test_one_long_and_many_short_sequences():
    """The line of blocks is cut anywhere: a unit over many CTAs next to many units in one."""
    lens = (30000, *[1 + 13 * b % 200 for b in range(60)], 9000)
    cache, table, g = filled(lens, 64, 2, 128, seed=31)
    q = torch.randn(len(lens), 1, 8, 128, device=DEV, generator=g).bfloat16()
    compare(cache, table, lens, q, causal=True)


@pytest.mark.parametrize("Hq,Hkv,B", [(8, 8, 60), (16, 1, 450), (8, 8, 1)])
@pytest.mark.parametrize("mean,sd", [(0.03, 0.02), (0.1, 0.05), (3.0, 2.0)])
def test_small_values_beside_a_dominant_key(Hq, Hkv, B, mean, sd):
    """A first key with most of the weight and the value 0, as sink tokens have it: the output is
    what the other keys, each of about 2^-23 of its weight, add up to. With the batches one CTA
    holds a sequence's KV head, and one warp all of what it shares with the first key."""
    n, D, page = 8192, 128, 64
    g = torch.Generator(device=DEV).manual_seed(B)
    cache = mfa.kv4_cache(n // page, page, Hkv, D, DEV)
    table = torch.arange(n // page, device=DEV).int()[None]
    one = torch.randn(Hkv, 1, D, device=DEV, generator=g).bfloat16()  # alike in a group's heads
    q = one.expand(Hkv, Hq // Hkv, D).reshape(1, 1, Hq, D)
    k = torch.randn(1, n, Hkv, D, device=DEV, generator=g)
    v = mean + sd * torch.randn(1, n, Hkv, D, device=DEV, generator=g)
    u = one[:, 0].float()
    k[0, 0] = u * (16 * D**0.5 / u.square().sum(-1, keepdim=True))  # a logit of 16
    v[0, 0] = 0
    mfa.kv4_append(cache, k.bfloat16(), v.bfloat16(), table, i32(0))
    out = mfa.flash_attn_with_kv4cache(q.expand(B, 1, Hq, D), cache, table.expand(B, -1),
                                       torch.full((B,), n, dtype=torch.int32, device=DEV))
    want = ref.attention(q[0], ref.tokens(cache, table[0], n, True),
                         ref.tokens(cache, table[0], n, False))
    # Relative to the output, in the 2-norm: 2^-9 of its rounding to bf16; 2^-11 of that of the
    # probabilities, which are normal fp16 numbers here; 2^-13 and 2^-14 of what moves the first
    # key's logit and another's (fp32 sums, 2^-17 of sum|q k| / sqrt(D) = 16 and about 7)
    for b in {0, B // 2, B - 1}:
        off = (out[b].double() - want).norm() / want.norm()
        assert off <= 2**-9 + 2**-11 + 2**-13 + 2**-14, (b, off)
    _kernel.check_device_errors()


def test_extreme_queries():
    """Query rows far outside of fp16's range in bf16, zeros, and infinities in one row only."""
    lens = (300,)
    cache, table, g = filled(lens, 32, 1, 64, seed=5)
    q = torch.randn(1, 1, 8, 64, device=DEV, generator=g).bfloat16()
    size = torch.tensor([1e-30, 1e-8, 1e-3, 1.0, 3.0, 0.0, 1e-38, 1.0], device=DEV)
    q = (q.float() * size[:, None]).bfloat16()
    compare(cache, table, lens, q)
    scaled = (q.float() * 2.0**100).bfloat16()
    scaled[0, 0, 2:5] = 0
    scaled[0, 0, 7] = 0
    out = mfa.flash_attn_with_kv4cache(scaled, cache, table, i32(300), softmax_scale=2.0**-103)
    want = mfa.flash_attn_with_kv4cache((scaled.float() * 2.0**-100).bfloat16(), cache, table,
                                        i32(300), softmax_scale=2.0**-3)
    assert torch.equal(out[0, 0, :2], want[0, 0, :2]) and torch.equal(out[0, 0, 5:], want[0, 0, 5:])
    good = mfa.flash_attn_with_kv4cache(q, cache, table, i32(300))
    q[0, 0, 3, 10] = float("nan")
    q[0, 0, 6] = float("inf")
    out = mfa.flash_attn_with_kv4cache(q, cache, table, i32(300))
    rest = [0, 1, 2, 4, 5, 7]
    assert torch.equal(out[0, 0, rest], good[0, 0, rest])
    assert bool(out[0, 0, 3].isnan().all()) and bool(out[0, 0, 6].isnan().all())


def test_what_masked_tokens_hold_does_not_matter():
    """NaN keys and values that a row does not see, next to ones that it does, in one tile."""
    page, D, n = 16, 64, 100
    cache, table, g = filled((n,), page, 2, D, seed=6)
    q = torch.randn(1, 4, 4, D, device=DEV, generator=g).bfloat16()
    kw = dict(causal=True, window_size=(20, -1), sink_tokens=3)
    good = mfa.flash_attn_with_kv4cache(q, cache, table, i32(n), **kw)
    k = torch.full((1, 70, 2, D), float("nan"), device=DEV).bfloat16()
    mfa.kv4_append(cache, k, k, table, i32(4))  # hidden from every row: tokens 4 .. 73
    assert torch.equal(mfa.flash_attn_with_kv4cache(q, cache, table, i32(n), **kw), good)
    one = k[:, :1]
    mfa.kv4_append(cache, one, one, table, i32(77))  # only the first two rows see it
    out = mfa.flash_attn_with_kv4cache(q, cache, table, i32(n), **kw)
    assert bool(out[0, :2].isnan().all()) and torch.equal(out[0, 2:], good[0, 2:])
    mfa.kv4_append(cache, one, one, table, i32(99))  # only the newest row sees it
    out = mfa.flash_attn_with_kv4cache(q, cache, table, i32(n), **kw)
    assert bool(out[0, 3].isnan().all()) and torch.equal(out[0, 2], good[0, 2])


@pytest.mark.parametrize("shape", [(2, 60, 1), (2, 1, 4), (1, 60, 4), (1, 1, 4)])
def test_broadcast_queries_give_the_same_bits(shape):
    """Expanded over heads, rows or the batch: the same kernels as for a copy, so the same bits."""
    lens = (500, 77)
    cache, table, g = filled(lens, 16, 2, 64, seed=16)
    for rows in (60, 1):
        if shape[1] > rows:
            continue
        q = torch.randn(*shape, 64, device=DEV, generator=g).bfloat16().expand(2, rows, 4, 64)
        want = mfa.flash_attn_with_kv4cache(q.contiguous(), cache, table, i32(*lens), causal=True)
        got = mfa.flash_attn_with_kv4cache(q, cache, table, i32(*lens), causal=True)
        assert torch.equal(got, want)


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 4, 2), (64, 4, 1), (128, 2, 1), (128, 8, 2), (128, 12, 1)])
@pytest.mark.parametrize("page", [16, 128])
def test_nan_values_reach_their_dims_of_the_rows_that_see_them(D, Hq, Hkv, page):
    """A NaN among a token's values (its keys are finite) makes NaN of the 16 dims that share its
    scale, in the rows that see it; all else is as if it were not there."""
    n, Lq = 300, 4
    g = torch.Generator(device=DEV).manual_seed(18)
    table, pages = table_of(1, -(-n // page))
    cache = dirty(mfa.kv4_cache(pages, page, Hkv, D, DEV))
    k, v = (torch.randn(1, n, Hkv, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    mfa.kv4_append(cache, k, v, table, i32(0))
    q = torch.randn(1, Lq, Hq, D, device=DEV, generator=g).bfloat16()
    kw = dict(causal=True, window=(60, -1), sink=130)
    good = compare(cache, table, (n,), q, **kw)
    # the newest token but one: two rows see it; the oldest of the window: one; hidden; first keys
    for token in (n - 2, n - Lq - 60, 200, 5):
        bad = v.clone()
        bad[0, token, 0, 33] = float("nan")
        mfa.kv4_append(cache, k, bad, table, i32(0))
        out = compare(cache, table, (n,), q, **kw)  # the oracle leaves out what is hidden
        rows = [i for i in range(Lq) if token <= n - Lq + i
                and (token >= n - Lq + i - 60 or token < 130)]
        touched = torch.zeros(1, Lq, Hq, D, dtype=torch.bool, device=DEV)
        touched[0, rows, :Hq // Hkv, 32:48] = True
        assert bool(out[touched].isnan().all())
        assert torch.equal(out[~touched], good[~touched])
    _kernel.check_device_errors()


def test_bad_tables_and_lengths_are_reported():
    lens = (90, 90)
    cache, table, g = filled(lens, 16, 2, 64, seed=9)
    for Lq in (1, 200):
        q = torch.randn(2, Lq, 4, 64, device=DEV, generator=g).bfloat16()
        good = mfa.flash_attn_with_kv4cache(q, cache, table, i32(*lens))
        for page in (-1, cache.num_pages, 2**31 - 1):
            bad = table.clone()
            bad[1, 2] = page
            out = mfa.flash_attn_with_kv4cache(q, cache, bad, i32(*lens))
            reported()
            assert torch.equal(out[0], good[0]) and bool(out[1].isfinite().all())
            if Lq == 1:  # read directly, the tokens are left out; by way of 16 bits they are 0
                k, v = (torch.cat((t[:32], t[48:])) for t in
                        (ref.tokens(cache, table[1], 90, keys) for keys in (True, False)))
                check(out[1], ref.attention(q[1], k, v), v)
        full = mfa.flash_attn_with_kv4cache(q, cache, table, i32(90, 96))
        for n in (97, 2**31 - 1):  # more than the table covers: what it covers
            out = mfa.flash_attn_with_kv4cache(q, cache, table, i32(90, n))
            reported()
            torch.testing.assert_close(out, full, atol=0, rtol=0, equal_nan=True)
        out = mfa.flash_attn_with_kv4cache(q, cache, table, i32(90, -5))
        reported()
        assert bool((out[1] == 0).all()) and torch.equal(out[0], good[0])
    empty = table[:, :0]
    out = mfa.flash_attn_with_kv4cache(q, cache, empty, i32(0, 0))
    _kernel.check_device_errors()
    assert bool((out == 0).all())


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("Lq,Hq,D", [(1, 4, 64), (3, 32, 128), (60, 4, 64), (40, 8, 128)])
@pytest.mark.parametrize("kw", [dict(causal=True, window=(40, -1), sink=5),
                                dict(causal=True, window=(300, -1), sink=150),
                                dict(causal=True, window=(17, -1)),
                                dict(window=(100, 3), sink=20)])
def test_pages_that_no_row_sees_may_be_missing(page, Lq, Hq, D, kw):
    """What a window has left behind may have been given back, whichever way the call goes."""
    lens = (1500, 700, Lq)
    cache, table, g = filled(lens, page, 2, D, seed=page)
    q = torch.randn(3, Lq, Hq, D, device=DEV, generator=g).bfloat16()
    want = compare(cache, table, lens, q, **kw)
    bare = table.clone()
    for b, n in enumerate(lens):
        first, sink = max(0, n - Lq - kw["window"][0]), kw.get("sink", 0)
        for p in range(table.shape[1]):
            seen = range(max(p * page, first), min((p + 1) * page, n))
            if not (len(seen) or p * page < min(sink, n)):
                bare[b, p] = (-1, cache.num_pages, 2**31 - 1)[p % 3]
    assert bool((bare != table).any())
    got = mfa.flash_attn_with_kv4cache(q, cache, bare, i32(*lens), causal=kw.get("causal", False),
                                       window_size=kw["window"], sink_tokens=kw.get("sink", 0))
    _kernel.check_device_errors()
    assert torch.equal(got, want)
    # one that is seen is still reported
    bare[0, (lens[0] - 1) // page] = -1
    mfa.flash_attn_with_kv4cache(q, cache, bare, i32(*lens), causal=kw.get("causal", False),
                                 window_size=kw["window"], sink_tokens=kw.get("sink", 0))
    reported()


@pytest.mark.parametrize("Lq", [1, 60])
@pytest.mark.parametrize("window,sink", [((20, -1), 0), ((20, -1), 4), ((200, -1), 0)])
def test_lengths_past_the_table_under_a_window(Lq, window, sink):
    """A length beyond the table counts as what the table covers, and the window ends there: the
    keys that it then shows are this cache's, not what an earlier call left in the workspace."""
    n = 608
    cache, table, g = filled((n,), 16, 2, 64, seed=13)
    other, _, _ = filled((n,), 16, 2, 64, seed=14)
    q = torch.randn(1, Lq, 4, 64, device=DEV, generator=g).bfloat16()
    kw = dict(causal=True, window_size=window, sink_tokens=sink)
    want = mfa.flash_attn_with_kv4cache(q, cache, table, i32(n), **kw)
    for length in (n + 1, 900, 2**31 - 1):
        mfa.flash_attn_with_kv4cache(q, other, table, i32(n), **kw)
        out = mfa.flash_attn_with_kv4cache(q, cache, table, i32(length), **kw)
        reported()
        assert torch.equal(out, want)


def test_many_rows_over_a_table_without_pages():
    """All rows are 0, in time that grows with the rows alone: 4096 x 32 rows write 34 MB, 6 us of
    a copy; 20 ms is far more than that, and than a launch per row block would take."""
    cache, table, g = filled((40,), 16, 8, 128, seed=15)
    q = torch.randn(1, 4096, 32, 128, device=DEV, generator=g).bfloat16()
    empty = table[:, :0]
    mfa.flash_attn_with_kv4cache(q, cache, empty, i32(0))
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    out = mfa.flash_attn_with_kv4cache(q, cache, empty, i32(0), causal=True)
    end.record()
    end.synchronize()
    _kernel.check_device_errors()
    assert bool((out == 0).all())
    assert start.elapsed_time(end) < 20
    mfa.flash_attn_with_kv4cache(q, cache, empty, i32(7))  # a length that no page holds
    reported()


@pytest.mark.parametrize("Lq,Hq,D", [(1, 4, 64), (100, 8, 64), (200, 4, 128)])
def test_wide_tables_and_a_bound_of_the_lengths(Lq, Hq, D):
    """With a bound, a table as wide as the longest context asks for no more workspace than a
    narrow one, and gives the same bits; a longer sequence is cut at the bound's page and
    reported."""
    lens = (700, 256, 0)
    cache, table, g = filled(lens, 16, 2, D, seed=17)
    q = torch.randn(3, Lq, Hq, D, device=DEV, generator=g).bfloat16()
    wide = torch.full((3, 2**17 // 16), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    sizes = []  # of the workspaces of streams that make no other call
    kw = dict(causal=True, window_size=(400, -1), sink_tokens=3)
    for t, bound in ((table, None), (wide, 700), (wide, table.shape[1] * 16)):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = mfa.flash_attn_with_kv4cache(q, cache, t, i32(*lens), max_seqlen=bound, **kw)
            sizes.append(_kernel._workspaces.pop((q.device, side.cuda_stream)).numel())
        side.synchronize()
        if bound is None:
            want = out
        assert torch.equal(out, want)
    assert sizes[0] == sizes[1] == sizes[2] < 16 << 20
    compare(cache, wide, lens, q, causal=True, window=(400, -1), sink=3)
    _kernel.check_device_errors()
    cut = mfa.flash_attn_with_kv4cache(q, cache, wide, i32(700, 256, 0), max_seqlen=600, **kw)
    reported()
    assert torch.equal(cut, mfa.flash_attn_with_kv4cache(q, cache, table, i32(608, 256, 0), **kw))
    assert bool((mfa.flash_attn_with_kv4cache(q, cache, wide, i32(0, 0, 0), max_seqlen=0) == 0).all())
    _kernel.check_device_errors()


def test_strided_queries_and_empty_batches():
    lens = (50, 33)
    cache, table, g = filled(lens, 16, 2, 64, seed=10)
    big = torch.randn(2, 6, 12, 65, device=DEV, generator=g).half()
    q = big[:, ::2, 1:9, 1:]
    want = mfa.flash_attn_with_kv4cache(q.contiguous(), cache, table, i32(*lens), causal=True)
    assert torch.equal(mfa.flash_attn_with_kv4cache(q, cache, table, i32(*lens), causal=True), want)
    wide = torch.zeros(2, 9, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + table.shape[1]] = table
    assert torch.equal(mfa.flash_attn_with_kv4cache(q, cache, wide[:, 2:2 + table.shape[1]],
                                                    i32(*lens), causal=True), want)
    assert mfa.flash_attn_with_kv4cache(q[:, :0], cache, table, i32(*lens)).shape == (2, 0, 8, 64)
    assert mfa.flash_attn_with_kv4cache(q[:0], cache, table[:0], i32()).shape == (0, 3, 8, 64)
    mfa.kv4_append(cache, big[:0, :, :2, :64], big[:0, :, :2, :64], table[:0], i32())
    assert mfa.kv4_gather(cache, table, i32(*lens), 0)[0].shape == (2, 0, 2, 64)


def test_refusals_on_the_gpu():
    cache, table, g = filled((40, 40), 16, 2, 64)
    q = torch.zeros(2, 1, 4, 64, device=DEV, dtype=torch.float16)
    kv = torch.zeros(2, 1, 2, 64, device=DEV, dtype=torch.float16)
    n = i32(40, 40)
    attend = [(q, cache, table, n.long()), (q, cache, table, i32(40)), (q, cache, table.long(), n),
              (q, cache, table[:1], n), (q, cache, table.cpu(), n), (q, cache, table, n.cpu()),
              (q[..., :32], cache, table, n), (q[:, :, :3], cache, table, n),
              (q, cache, table.t().contiguous().t(), n), (q, cache, table[0], n)]
    for args in attend:
        with pytest.raises(ValueError):
            mfa.flash_attn_with_kv4cache(*args)
    for args in ((kv[:, :, :1], kv[:, :, :1], table, n), (kv[..., :32], kv[..., :32], table, n),
                 (kv, kv, table, n.long()), (kv, kv, table, n, n.long()), (kv, kv.cpu(), table, n)):
        with pytest.raises(ValueError):
            mfa.kv4_append(cache, *args)
    with pytest.raises(ValueError):
        mfa.kv4_gather(cache, table, n, 4, starts=n.long())
    out = mfa.flash_attn_with_kv4cache(q.requires_grad_(), cache, table, n)
    with pytest.raises(NotImplementedError):
        out.float().sum().backward()


# ----------------------------------------------------------------------------- as they are used
def test_serving_loop():
    """Prompt, then token by token: norm and rotation, append, attention with a window and first
    tokens, against the same steps in 64 bits on the held values; the prompt's own attention is
    the framework's dense forward with the same mask."""
    B, Hq, Hkv, D, page, prompt = 2, 8, 2, 128, 16, 45
    steps, window, sink = 20, (24, -1), 3
    g = torch.Generator(device=DEV).manual_seed(11)
    table, pages = table_of(B, 5)
    cache = dirty(mfa.kv4_cache(pages, page, Hkv, D, DEV))
    f = 1e4 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    angle = torch.arange(100, device=DEV, dtype=torch.float64)[:, None] * f
    cos, sin = angle.cos().float(), angle.sin().float()
    lens = i32(0, 0)
    for step in range(steps):
        n = prompt if step == 0 else 1
        qkv = torch.randn(B, n, Hq + 2 * Hkv, D, device=DEV, generator=g).bfloat16()
        pos = lens[:, None] + torch.arange(n, device=DEV)
        q, k = mfa.qk_norm_rope(qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], None, None, cos, sin, pos)
        v = qkv[:, :, Hq + Hkv:]
        mfa.kv4_append(cache, k, v, table, lens)
        lens += n
        out = mfa.flash_attn_with_kv4cache(q, cache, table, lens, causal=True, window_size=window,
                                           sink_tokens=sink)
        m = prompt + step
        hk, hv = mfa.kv4_gather(cache, table, lens, m)
        dense = mfa.flash_attn_func(q, hk, hv, causal=True, window_size=window, sink_tokens=sink)
        for b in range(B):
            assert torch.equal(hk[b, m - n:].double(), ref.held(k[b]))
            want = ref.attention(q[b], hk[b], hv[b], True, window, sink=sink)
            check(out[b], want, hv[b])
        # the dense forward rounds its probabilities to bf16 (half a step each) and its output once
        top = float(hv.abs().max())
        torch.testing.assert_close(out, dense, atol=2 * top * 2**-8, rtol=2**-7)
    _kernel.check_device_errors()


def test_captured_steps_replayed_together():
    """Two decode steps with splits, captured on one stream, replayed on two: each graph has its
    own workspace, and lengths are read at replay."""
    lens = (6000,)
    sets = []
    for seed in (1, 2):
        cache, table, g = filled((6100,), 64, 2, 128, seed=seed)
        q = torch.randn(1, 1, 16, 128, device=DEV, generator=g).bfloat16()
        kv = torch.randn(1, 1, 2, 128, device=DEV, generator=g).bfloat16()
        sets.append((cache, table, q, kv, i32(*lens)))

    def step(cache, table, q, kv, n):
        mfa.kv4_append(cache, kv, kv, table, n)
        n += 1
        return mfa.flash_attn_with_kv4cache(q, cache, table, n, causal=True)

    side = torch.cuda.Stream()
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step(*s))
        graphs.append(graph)
    for s in sets:
        s[4].fill_(lens[0])  # capture ran nothing
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(30):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (cache, table, q, kv, n), out in zip(sets, outs):
        assert n.item() == lens[0] + 30
        want = mfa.flash_attn_with_kv4cache(q, cache, table, n, causal=True)
        assert torch.equal(out, want)
        k, v = (ref.tokens(cache, table[0], n.item(), keys) for keys in (True, False))
        assert torch.equal(k[-30:], ref.held(kv[0]).expand(30, -1, -1))
        check(out[0], ref.attention(q[0], k, v, True), v)
    _kernel.check_device_errors()


def test_first_call_of_a_process_captured():
    """No eager call before: nothing that the capture made may be missing at replay."""
    import os
    import subprocess
    import sys
    import textwrap
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = textwrap.dedent("""
        import torch, mtlflashattn_b200 as mfa
        from mtlflashattn_b200 import _kernel
        cache = mfa.kv4_cache(64, 64, 2, 128, "cuda")
        table = torch.arange(64, device="cuda").int().view(1, 64)
        n = torch.tensor([3000], dtype=torch.int32, device="cuda")
        kv = torch.randn(1, 3000, 2, 128, device="cuda").bfloat16()
        q = torch.randn(1, 1, 8, 128, device="cuda").bfloat16()
        zero = torch.zeros(1, dtype=torch.int32, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            qq, _ = mfa.qk_norm_rope(q, kv[:, :1])
            mfa.kv4_append(cache, kv, kv, table, zero)
            out = mfa.flash_attn_with_kv4cache(qq, cache, table, n, causal=True)
            dense = mfa.flash_attn_func(qq, kv, kv, causal=True, window_size=(500, -1), sink_tokens=4)
        _kernel.check_device_errors("cuda")
        g.replay()
        torch.cuda.synchronize()
        qq, _ = mfa.qk_norm_rope(q, kv[:, :1])
        assert torch.equal(out, mfa.flash_attn_with_kv4cache(qq, cache, table, n, causal=True))
        assert torch.equal(dense, mfa.flash_attn_func(qq, kv, kv, causal=True,
                                                      window_size=(500, -1), sink_tokens=4))
        _kernel.check_device_errors("cuda")
        print("same")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root,
                       timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout[-1000:] + r.stderr[-3000:]


def test_reports_of_a_process_under_inference_mode(monkeypatch):
    monkeypatch.setattr(_kernel, "_err_words", {})
    cache, table, g = filled((40,), 16, 2, 64)
    torch.cuda.synchronize()
    _kernel._err_words.clear()
    with torch.inference_mode():
        q = torch.zeros(1, 1, 4, 64, device=DEV).half()
        mfa.flash_attn_with_kv4cache(q, cache, torch.full_like(table, -1), i32(40))
    reported()
    _kernel.check_device_errors()  # and is quiet again


def test_a_first_call_that_is_captured_still_reports():
    """Nothing but the cache was made before the capture."""
    import os
    import subprocess
    import sys
    import textwrap
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = textwrap.dedent("""
        import torch, mtlflashattn_b200 as mfa
        from mtlflashattn_b200 import _kernel, _lib
        cache = mfa.kv4_cache(8, 16, 2, 64, "cuda")
        table = torch.arange(4, device="cuda").int().view(1, 4)
        n = torch.tensor([50], dtype=torch.int32, device="cuda")
        q = torch.zeros(1, 1, 4, 64, device="cuda").half()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = mfa.flash_attn_with_kv4cache(q, cache, table, n, causal=True)
        g.replay()
        _kernel.check_device_errors("cuda")
        table[0, 1] = 8
        g.replay()
        try:
            _kernel.check_device_errors("cuda")
        except _lib.MfaError:
            print("told")
        table[0, 1] = 1
        g.replay()
        _kernel.check_device_errors("cuda")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root,
                       timeout=300)
    assert r.returncode == 0 and "told" in r.stdout, r.stdout[-1000:] + r.stderr[-3000:]


def test_two_threads_on_two_streams():
    import threading
    cache, table, g = filled((5000,), 64, 2, 64, seed=12)
    qs = [torch.randn(1, 1, 8, 64, device=DEV, generator=g).half() for _ in range(2)]
    n = i32(5000)
    want = [mfa.flash_attn_with_kv4cache(q, cache, table, n) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                out = mfa.flash_attn_with_kv4cache(qs[i], cache, table, n)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(out, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_threads_that_share_a_stream():
    """Two host threads whose calls share a stream, and with it the workspace that an attention
    kernel leaves partial sums in for the kernel that joins them."""
    import threading

    lens = (5000, 900)
    cases = []
    for seed in (1, 2):
        cache, table, g = filled(lens, 64, 2, 128, seed=seed)
        q = torch.randn(2, 1, 8, 128, device=DEV, generator=g).half()
        k = torch.randn(1, 9000, 2, 128, device=DEV, generator=g).half()

        def paged(q=q, cache=cache, table=table):
            return mfa.flash_attn_with_kv4cache(q, cache, table, i32(*lens), causal=True)

        def dense(q=q, k=k):  # few rows over long keys: split as well
            return mfa.flash_attn_func(q[:1], k, k)
        cases += [(paged, paged()), (dense, dense())]
    torch.cuda.synchronize()
    wrong, stop = [], threading.Event()

    def work(mine):
        try:
            for _ in range(300):
                if stop.is_set():
                    return
                for fn, want in mine:
                    if not torch.equal(fn(), want):
                        wrong.append(fn)
                        stop.set()
        except BaseException as e:  # shown by the assertion below
            wrong.append(e)
            stop.set()

    threads = [threading.Thread(target=work, args=(cases[i::4],)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong
