"""qk_norm_rope against the formula in 64 bits."""
import pytest
import torch

import mtlflashattn_b200 as mfa
from mtlflashattn_b200 import _kernel, _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tables(rows, R, dtype=torch.float32):
    f = 10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / max(R, 1))
    angle = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * f
    return angle.cos().to(dtype), angle.sin().to(dtype)


def formula(x, w, cos, sin, pos, eps, interleaved):
    """(result, a bound of the magnitudes that were added), 64 bits: x [B, L, H, D], pos [B, L]."""
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double()
    out, size = y.clone(), y.abs()
    if cos is not None:
        R = 2 * cos.shape[1]
        c, s = cos.double()[pos][:, :, None], sin.double()[pos][:, :, None]
        i = torch.arange(R // 2, device=x.device)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., a] * s + y[..., b] * c
        size[..., a] = size[..., b] = y[..., a].abs() + y[..., b].abs()
    return out, size


def check(got, x, *rest):
    want, size = formula(x, *rest)
    # a sum of up to 128 squares by at most 20 additions in a row: 20 * 2^-24 of it, half of that
    # after the square root, then about 8 roundings more: 32 * 2^-24 of what is added; and one
    # rounding to the type (at least half of its smallest number)
    t = torch.finfo(got.dtype)
    bound = 32 * 2.0**-24 * size + t.eps / 2 * (want.abs() + 32 * 2.0**-24 * size)
    bound += t.smallest_normal * t.eps / 2
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (off - bound).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,Hq,Hkv,D,R", [
    (1, 1, 1, 1, 64, 64), (2, 3, 4, 2, 128, 128), (3, 17, 5, 1, 128, 64), (1, 333, 40, 8, 128, 128),
    (2, 9, 6, 3, 96, 96), (1, 20, 4, 4, 80, 80), (1, 20, 3, 3, 80, 40), (2, 5, 9, 3, 32, 32),
    (1, 6, 7, 1, 16, 16), (2, 7, 2, 2, 48, 16), (1, 5, 3, 1, 100, 20), (1, 5, 3, 3, 33, 32),
    (1, 4, 2, 1, 1, 0), (2, 4, 2, 1, 64, 0), (1, 4, 2, 1, 64, 36), (1, 2500, 3, 2, 64, 24)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_against_formula(dtype, B, L, Hq, Hkv, D, R, interleaved):
    g = torch.Generator(device=DEV).manual_seed(D + L)
    q, k = (3 * torch.randn(B, L, h, D, device=DEV, generator=g) for h in (Hq, Hkv))
    q, k = q.to(dtype), k.to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(D, device=DEV, generator=g)).to(dtype) for _ in range(2))
    cos, sin = tables(5000, R) if R else (None, None)
    pos = torch.randint(0, 5000, (B, L), device=DEV, generator=g)
    oq, ok = mfa.qk_norm_rope(q, k, wq, wk, cos, sin, pos if R else None, 1e-5, interleaved)
    assert oq.shape == q.shape and ok.shape == k.shape and oq.dtype == dtype
    check(oq, q, wq, cos, sin, pos, 1e-5, interleaved)
    check(ok, k, wk, cos, sin, pos, 1e-5, interleaved)
    _kernel.check_device_errors()


def test_views_of_one_projection_and_packed_tokens():
    g = torch.Generator(device=DEV).manual_seed(1)
    cos, sin = tables(64, 128, torch.bfloat16)
    qkv = torch.randn(2, 11, 4 + 2 + 2, 128, device=DEV, generator=g).bfloat16()
    pos = torch.arange(11, device=DEV).expand(2, 11)
    for q, k in ((qkv[:, :, :4], qkv[:, :, 4:6]),
                 (qkv.transpose(1, 2).contiguous().transpose(1, 2)[:, :, 1:5], qkv[:, :, 6:])):
        oq, ok = mfa.qk_norm_rope(q, k, None, None, cos, sin)
        check(oq, q, None, cos, sin, pos, 1e-6, False)
        check(ok, k, None, cos, sin, pos, 1e-6, False)
        for p in (pos, pos[0], pos.int(), pos[0].int(), pos[:1].repeat(2, 1)):
            again = mfa.qk_norm_rope(q, k, None, None, cos, sin, p)
            assert torch.equal(again[0], oq) and torch.equal(again[1], ok)
    flat = qkv.flatten(0, 1)
    fq, fk = mfa.qk_norm_rope(flat[:, :4], flat[:, 4:6], None, None, cos, sin,
                              pos.reshape(-1).int())
    q, k = mfa.qk_norm_rope(qkv[:, :, :4], qkv[:, :, 4:6], None, None, cos, sin)
    assert torch.equal(fq, q.flatten(0, 1)) and torch.equal(fk, k.flatten(0, 1))


def test_unaligned_and_strided_last_dim():
    g = torch.Generator(device=DEV).manual_seed(2)
    cos, sin = tables(32, 64)
    base = torch.randn(1, 5, 4, 140, device=DEV, generator=g).half()
    pos = torch.arange(5, device=DEV)[None]
    for q in (base[..., 1:65], base[..., 3:131:2], base[..., :64]):
        k = q[:, :, ::2]
        oq, ok = mfa.qk_norm_rope(q, k, None, None, cos, sin)
        check(oq, q, None, cos, sin, pos, 1e-6, False)
        check(ok, k, None, cos, sin, pos, 1e-6, False)


def test_weights_in_fp32_and_one_of_them():
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(1, 3, 2, 64, device=DEV, generator=g).half()
    w = torch.rand(64, device=DEV, generator=g)
    oq, ok = mfa.qk_norm_rope(q, q, w, None)
    pos = torch.zeros(1, 3, dtype=torch.long, device=DEV)
    check(oq, q, w, None, None, pos, 1e-6, False)
    check(ok, q, None, None, None, pos, 1e-6, False)


@pytest.mark.parametrize("D", [64, 100])
def test_positions_outside_of_the_tables(D):
    q = torch.ones(1, 4, 2, D, device=DEV, dtype=torch.bfloat16)
    cos, sin = tables(8, 32)
    pos = torch.tensor([[0, 8, -1, 7]], device=DEV)
    oq, ok = mfa.qk_norm_rope(q, q, None, None, cos, sin, pos)
    with pytest.raises(_lib.MfaError):
        _kernel.check_device_errors()
    assert bool((oq[0, 1:3] == 0).all()) and bool((ok[0, 1:3] == 0).all())
    keep = pos.clamp(0, 7)
    want = mfa.qk_norm_rope(q, q, None, None, cos, sin, keep)
    assert torch.equal(oq[0, [0, 3]], want[0][0, [0, 3]])
    _kernel.check_device_errors()


def test_values_that_are_not_finite_stay_in_their_head():
    g = torch.Generator(device=DEV).manual_seed(4)
    q = torch.randn(1, 2, 8, 128, device=DEV, generator=g).bfloat16()
    cos, sin = tables(8, 128)
    want, _ = mfa.qk_norm_rope(q, q, None, None, cos, sin)
    q[0, 0, 3, 5], q[0, 1, 6, 127] = float("nan"), float("inf")
    got, _ = mfa.qk_norm_rope(q, q, None, None, cos, sin)
    touched = torch.zeros(2, 8, dtype=torch.bool, device=DEV)
    touched[0, 3] = touched[1, 6] = True
    assert torch.equal(got[0][~touched], want[0][~touched])
    assert bool(got[0, 0, 3].isnan().all())
    zero = torch.zeros(1, 1, 1, 64, device=DEV, dtype=torch.float16)
    assert bool((mfa.qk_norm_rope(zero, zero)[0] == 0).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(128, 0), (128, 64), (64, 32), (128, 40), (48, 24), (96, 96)])
def test_dims_that_do_not_rotate_stay_alone(interleaved, D, R):
    """A dim that is not finite after the norm leaves the others that do not rotate as they are,
    wherever the rows lie in memory."""
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.randn(1, 4, 3, D, device=DEV, generator=g).bfloat16()
    w = torch.ones(D, device=DEV)
    for d in {R, D - 9, D - 1} - {D}:  # (in the last shape: dims that do rotate)
        w[d] = float("inf")
    x[0, 1, 2, D - 2] = float("inf")
    cos, sin = tables(9, R) if R else (None, None)
    base = torch.zeros(1, 4, 3, D + 3, device=DEV).bfloat16()
    base[..., 1:1 + D] = x
    a = mfa.qk_norm_rope(x, x, w, None, cos, sin, interleaved=interleaved)
    b = mfa.qk_norm_rope(base[..., 1:1 + D], base[..., 1:1 + D], w, None, cos, sin,
                         interleaved=interleaved)
    pos = torch.arange(4, device=DEV)[None]
    for got, odd, weight in zip(a, b, (w, None)):
        want, _ = formula(x, weight, cos, sin, pos, 1e-6, interleaved)
        for t in (got, odd):
            assert torch.equal(t.isnan(), want.isnan())
            assert torch.equal(t.isinf(), want.isinf())
        # two kernels whose sums add up in another order: 32 * 2^-24 of what is added, as in
        # check(), may move a rounding by one step
        torch.testing.assert_close(got, odd, rtol=2**-7, atol=2**-16, equal_nan=True)


def test_empty_refusals_and_gradients():
    q, k = (torch.randn(2, 3, h, 64, device=DEV).half() for h in (4, 2))
    cos, sin = tables(8, 64)
    for a, b in ((q[:, :0], k[:, :0]), (q[:0], k[:0])):
        oq, ok = mfa.qk_norm_rope(a, b, None, None, cos, sin)
        assert oq.shape == a.shape and ok.shape == b.shape
    bad = [((q, k.float()), {}, NotImplementedError), ((q, k[:, :2]), {}, ValueError),
           ((q[0, 0], k[0, 0]), {}, ValueError), ((q, k, torch.ones(63, device=DEV)), {}, ValueError),
           ((q, k, torch.ones(64, device=DEV).double()), {}, ValueError),
           ((q, k, torch.ones(64, device=DEV), torch.ones(64, device=DEV).half()), {}, ValueError),
           ((q, k, None, None, cos), {}, ValueError), ((q, k, None, None, cos, sin[:4]), {}, ValueError),
           ((q, k, None, None, cos, sin, torch.zeros(2, device=DEV)), {}, ValueError),
           ((q, k, None, None, cos, sin, torch.zeros(2, 4, device=DEV).long()), {}, ValueError),
           ((q, k, torch.ones(64)), {}, ValueError), ((q, k), dict(eps=-1.0), ValueError),
           ((torch.cat((q, q, q), -1), torch.cat((k, k, k), -1)), {}, NotImplementedError),
           ((q, k, None, None, *tables(8, 80)), {}, ValueError)]
    for args, kw, exc in bad:
        with pytest.raises(exc):
            mfa.qk_norm_rope(*args, **kw)
    out, _ = mfa.qk_norm_rope(q.requires_grad_(), k, None, None, cos, sin)
    with pytest.raises(NotImplementedError):
        out.float().sum().backward()


def test_other_streams_and_replay():
    g = torch.Generator(device=DEV).manual_seed(5)
    q, k = (torch.randn(4, 1, h, 128, device=DEV, generator=g).bfloat16() for h in (32, 8))
    cos, sin = tables(100, 128)
    pos = torch.tensor([[3], [50], [99], [0]], device=DEV)
    want = mfa.qk_norm_rope(q, k, None, None, cos, sin, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mfa.qk_norm_rope(q, k, None, None, cos, sin, pos)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mfa.qk_norm_rope(q, k, None, None, cos, sin, pos)
    pos += 0  # same positions, new values of q
    q.copy_(q.flip(0))
    graph.replay()
    want = mfa.qk_norm_rope(q, k, None, None, cos, sin, pos)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
