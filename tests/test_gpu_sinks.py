"""Sliding-window attention whose first tokens stay visible (sink_tokens), against the formula in
64 bits: key j is seen by row i (centre c = i + Lk - Lq) iff c - left <= j or j < sink, and the
causal and right limits hold."""
import math

import pytest
import torch

import mtlflashattn_b200 as mfa
from mtlflashattn_b200 import _kernel

pytestmark = pytest.mark.gpu


def formula(q, k, v, causal, window, sink, softcap=0.0, slopes=None):
    """q [B, Lq, Hq, D], k/v [B, Lk, Hkv, D] -> [B, Lq, Hq, D], 64 bits; empty rows are 0."""
    B, Lq, Hq, D = q.shape
    Lk, g = k.shape[1], Hq // k.shape[2]
    q, k, v = (t.double() for t in (q, k, v))
    k, v = k.repeat_interleave(g, 2), v.repeat_interleave(g, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(D)
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    c = torch.arange(Lk - Lq, Lk, device=q.device)[:, None]
    j = torch.arange(Lk, device=q.device)[None]
    if slopes is not None:
        s = s - slopes.double()[None, :, None, None] * (c - j).abs()
    seen = torch.ones(Lq, Lk, dtype=torch.bool, device=q.device)
    if window[0] >= 0:
        seen &= (j >= c - window[0]) | (j < sink)
    if window[1] >= 0:
        seen &= j <= c + window[1]
    if causal:
        seen &= j <= c
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
    return torch.einsum("bhij,bjhd->bihd", p, v)


def inputs(B, Lq, Lk, Hq, Hkv, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(B, n, h, D, device="cuda", generator=g).to(dtype)
            for n, h in ((Lq, Hq), (Lk, Hkv), (Lk, Hkv))]


def check(out, want, dtype, softcap=0.0):
    # p is rounded to the input type before P.V (half a step, eps / 2, of each p; |v| <= 6 and
    # sum p = 1), and the output once more; exponentials from the FMA pipe are off by up to 7.5e-5
    # and the softcap's hardware tanh moves a logit by up to softcap * 2^-11 (twice, for the
    # numerator and the sum). fp32: 2e-6 of accumulated rounding.
    step = torch.finfo(dtype).eps / 2
    if dtype == torch.float32:
        atol, rtol = 2e-5, 1e-4
    else:
        atol, rtol = 6 * (step + 1.5e-4 + 2 * softcap * 2**-11), step
    torch.testing.assert_close(out.double(), want, atol=atol, rtol=rtol)


@pytest.mark.parametrize("dtype,D,Hq,Hkv", [
    (torch.bfloat16, 128, 4, 4), (torch.float16, 64, 4, 2), (torch.float32, 64, 2, 1),
    (torch.bfloat16, 100, 2, 2), (torch.float16, 128, 8, 1), (torch.bfloat16, 64, 6, 2)])
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 700), (5, 300), (130, 130), (300, 700), (700, 700),
                                   (400, 260)])
@pytest.mark.parametrize("window,sink,causal", [
    ((0, -1), 1, True), ((37, -1), 4, True), ((129, 5), 130, False), ((64, 0), 1000, True),
    ((300, 40), 3, True), ((10, -1), 129, False)])
def test_against_formula(dtype, D, Hq, Hkv, Lq, Lk, window, sink, causal):
    q, k, v = inputs(2, Lq, Lk, Hq, Hkv, D, dtype, seed=Lq + Lk + D)
    out = mfa.flash_attn_func(q, k, v, causal=causal, window_size=window, sink_tokens=sink)
    check(out, formula(q, k, v, causal, window, sink), dtype)
    _kernel.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kw", [dict(softcap=15.0), dict(slopes=True),
                                dict(softcap=15.0, slopes=True)])
@pytest.mark.parametrize("Lq,Lk", [(600, 600), (3, 900)])
def test_with_softcap_and_alibi(dtype, D, kw, Lq, Lk):
    q, k, v = inputs(1, Lq, Lk, 4, 2, D, dtype)
    cap = kw.get("softcap", 0.0)
    slopes = torch.tensor([0.5, 0.1, 0.02, 0.004], device="cuda") if kw.get("slopes") else None
    out = mfa.flash_attn_func(q, k, v, causal=True, window_size=(150, -1), softcap=cap,
                              alibi_slopes=slopes, sink_tokens=7)
    check(out, formula(q, k, v, True, (150, -1), 7, cap, slopes), dtype, cap)


def test_key_split_of_long_decode():
    """Few query rows against many keys: the launch splits the keys, the first of which are in
    another split than the window, or in several when there are many of them."""
    for sink in (1, 5, 3000, 20000):
        q, k, v = inputs(1, 2, 40000, 8, 2, 128, torch.bfloat16, seed=sink)
        out = mfa.flash_attn_func(q, k, v, causal=True, window_size=(1000, -1), sink_tokens=sink)
        check(out, formula(q, k, v, True, (1000, -1), sink), torch.bfloat16)


@pytest.mark.parametrize("window,sink", [(2040, 7), (2040, 8), (100, 1947), (100, 1948), (60, 9000),
                                         (2500, 3)])
@pytest.mark.parametrize("Hq,Hkv,softcap", [(2, 2, 0.0), (4, 1, 20.0)])
def test_walks_around_the_tile_rule(window, sink, Hq, Hkv, softcap):
    """Window and first keys together decide between CTAs of one and of two tiles at D = 128."""
    q, k, v = inputs(1, 2900, 2900, Hq, Hkv, 128, torch.bfloat16, seed=window + sink)
    out = mfa.flash_attn_func(q, k, v, causal=True, window_size=(window, -1), softcap=softcap,
                              sink_tokens=sink)
    check(out, formula(q, k, v, True, (window, -1), sink, softcap), torch.bfloat16, softcap)
    lens = torch.tensor([0, 2900], device="cuda").int()
    flat = mfa.flash_attn_varlen_func(q[0], k[0], v[0], lens, lens, 2900, 2900, causal=True,
                                      window_size=(window, -1), softcap=softcap, sink_tokens=sink)
    check(flat[None], formula(q, k, v, True, (window, -1), sink, softcap), torch.bfloat16, softcap)
    _kernel.check_device_errors()


def test_varlen_sequences_have_their_own_first_tokens():
    lens_q, lens_k = [1, 300, 0, 77, 500], [400, 300, 9, 77, 513]
    cq = torch.tensor([0, *lens_q], device="cuda").cumsum(0).to(torch.int32)
    ck = torch.tensor([0, *lens_k], device="cuda").cumsum(0).to(torch.int32)
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(n, h, 64, device="cuda", generator=g).bfloat16()
               for n, h in ((sum(lens_q), 8), (sum(lens_k), 2), (sum(lens_k), 2)))
    out = mfa.flash_attn_varlen_func(q, k, v, cq, ck, 500, 513, causal=True,
                                     window_size=(50, -1), sink_tokens=6)
    for b in range(5):
        if lens_q[b]:
            sq, sk = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
            want = formula(q[None, sq], k[None, sk], v[None, sk], True, (50, -1), 6)[0]
            check(out[sq], want, torch.bfloat16)


def test_same_bits_where_it_changes_nothing():
    q, k, v = inputs(1, 513, 513, 4, 2, 128, torch.bfloat16)
    want = mfa.flash_attn_func(q, k, v, causal=True)
    assert torch.equal(mfa.flash_attn_func(q, k, v, causal=True, sink_tokens=9), want)
    # every key a first one: the window hides nothing, and the blocks are walked in one order
    got = mfa.flash_attn_func(q, k, v, causal=True, window_size=(3, -1), sink_tokens=10**12)
    torch.testing.assert_close(got, want, atol=2**-6, rtol=2**-7)


def test_other_entry_points_take_it():
    q, k, v = inputs(1, 300, 300, 4, 4, 64, torch.float16)
    want = mfa.flash_attn_func(q, k, v, causal=True, window_size=(40, -1), sink_tokens=5)
    kw = dict(causal=True, window_size=(40, -1), sink_tokens=5)
    assert torch.equal(mfa.flash_attn_qkvpacked_func(torch.stack((q, k, v), 2), **kw), want)
    assert torch.equal(mfa.flash_attn_kvpacked_func(q, torch.stack((k, v), 2), **kw), want)
    heads = mfa.flash_attn_forward(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2),
                                   0.125, True, window_left=40, sink_tokens=5)
    assert torch.equal(heads.transpose(1, 2), want)
    host = mfa.flash_attn_host(*(t.cpu().pin_memory() for t in (q, k, v)), chunks=3, **kw)
    torch.testing.assert_close(host, want.cpu(), atol=2**-9, rtol=2**-10)


def test_captured_and_replayed():
    """A split launch in two graphs captured on one stream: each has its own workspace."""
    sets = [inputs(1, 1, 20000, 8, 2, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    kw = dict(causal=True, window_size=(9000, -1), sink_tokens=4)
    eager = [mfa.flash_attn_func(*t, **kw) for t in sets]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for t in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(mfa.flash_attn_func(*t, **kw))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, want in zip(outs, eager):
            assert torch.equal(o, want)
