"""The 4-bit cache and the norm with rotation without a GPU: struct layouts, refusals in Python and
in the library, and the oracle's own definition."""
import ctypes
import os
import shutil
import struct
import subprocess

import pytest
import torch

import mtlflashattn_b200 as mfa
from mtlflashattn_b200 import _lib
from oracle import kv4 as ref

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                      "mfa.h")
STRUCTS = [(_lib.MfaNormRopeParams, "mfa_norm_rope_params", _lib.NORM_ROPE_FORMAT),
           (_lib.MfaKv4Cache, "mfa_kv4_cache", _lib.KV4_CACHE_FORMAT),
           (_lib.MfaKv4Rows, "mfa_kv4_rows", _lib.KV4_ROWS_FORMAT),
           (_lib.MfaKv4FwdParams, "mfa_kv4_fwd_params", _lib.KV4_FWD_FORMAT)]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("cls,cname,fmt", STRUCTS)
def test_struct_layouts(tmp_path, cls, cname, fmt):
    names = [f[0] for f in cls._fields_]
    lines = [f'printf("%zu ", offsetof({cname}, {n}));' for n in names]
    src = tmp_path / "l.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n"
                   f'#include "{HEADER}"\nint main(void){{printf("%zu ", sizeof({cname}));'
                   + "".join(lines) + "return 0;}")
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "l")], check=True)
    got = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout
    size, *offs = map(int, got.split())
    assert size == ctypes.sizeof(cls) == struct.calcsize(fmt)
    assert offs == [getattr(cls, n).offset for n in names]


def test_packed_fields_land_where_the_struct_has_them():
    # each format fills the struct field by field: distinct numbers come back in order
    for cls, _, fmt in STRUCTS:
        n = len(struct.unpack(fmt, bytes(struct.calcsize(fmt))))
        raw = cls.from_buffer_copy(struct.pack(fmt, *range(n)))
        flat = []
        for name, _t in cls._fields_:
            x = getattr(raw, name)
            flat += list(x) if hasattr(x, "__len__") else [x or 0]
        assert flat == list(range(n)), cls.__name__
    assert _lib.MfaKv4FwdParams.workspace.offset == _lib.KV4_FWD_WORKSPACE_OFFSET


def test_two_threads_share_the_error_word(monkeypatch):
    """A word that one thread's launch points at must not be replaced by another's."""
    import threading

    from mtlflashattn_b200 import _kernel
    meet = threading.Barrier(2, timeout=20)
    zeros = torch.zeros

    def both_at_once(*args, **kw):
        meet.wait()
        return zeros(*args, **kw)

    monkeypatch.setattr(_kernel, "_err_words", {})
    monkeypatch.setattr(_kernel.torch, "zeros", both_at_once)
    got = []
    threads = [threading.Thread(target=lambda: got.append(_kernel._err_word(torch.device("cpu"))))
               for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 2 and got[0] is got[1] is _kernel._err_words[torch.device("cpu")]


def test_error_word_made_under_inference_mode(monkeypatch):
    from mtlflashattn_b200 import _kernel
    monkeypatch.setattr(_kernel, "_err_words", {})
    with torch.inference_mode():
        t = _kernel._err_word(torch.device("cpu"))
    t.fill_(_lib.ERR_INVALID)
    t.zero_()  # as check_device_errors does, outside of that mode
    assert t.item() == 0


def rows(shape=(2, 3, 2, 64), dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def test_cache_refusals():
    c = mfa.kv4_cache(3, 16, 2, 64, "cpu")
    assert (c.num_pages, c.page_size, c.num_heads_kv, c.head_dim) == (3, 16, 2, 64)
    parts = (c.k, c.v, c.k_scale, c.v_scale)
    for bad in (dict(k_unit=3.0), dict(v_unit=0.0), dict(k_unit=2.0**-15), dict(v_unit=32.0),
                dict(k_unit=-1.0), dict(k_unit=float("nan")), dict(v_unit=float("inf")),
                dict(k_unit="1")):
        with pytest.raises(ValueError, match="powers of two"):
            mfa.KV4Cache(*parts, **bad)
    with pytest.raises(NotImplementedError, match="page_size"):
        mfa.kv4_cache(3, 24, 2, 64, "cpu")
    with pytest.raises(NotImplementedError, match="page_size"):
        mfa.kv4_cache(3, 8, 2, 64, "cpu")
    with pytest.raises(NotImplementedError, match="head_dim"):
        mfa.kv4_cache(3, 16, 2, 96, "cpu")
    with pytest.raises(ValueError, match="one head"):
        mfa.kv4_cache(3, 16, 0, 64, "cpu")
    with pytest.raises(ValueError, match="k_scale"):
        mfa.KV4Cache(c.k, c.v, c.k_scale[:, :, :8], c.v_scale)
    with pytest.raises(ValueError, match="num_pages"):
        mfa.KV4Cache(c.k, c.v[:2], c.k_scale, c.v_scale)
    with pytest.raises(ValueError, match="float8"):
        mfa.KV4Cache(c.k, c.v, c.k_scale.view(torch.uint8), c.v_scale)
    with pytest.raises(ValueError, match="contiguous"):
        mfa.KV4Cache(*(t[::2] for t in parts))


def test_cpu_tensors_are_refused():
    c = mfa.kv4_cache(3, 16, 2, 64, "cpu")
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(NotImplementedError, match="CUDA"):
        mfa.kv4_append(c, rows(), rows(), table, lens)
    with pytest.raises(NotImplementedError, match="CUDA"):
        mfa.kv4_gather(c, table, lens, 4)
    with pytest.raises(NotImplementedError, match="CUDA"):
        mfa.flash_attn_with_kv4cache(rows(), c, table, lens)
    with pytest.raises(NotImplementedError, match="CUDA"):
        mfa.qk_norm_rope(rows(), rows())


@pytest.mark.parametrize("call,exc", [
    (lambda c, t, n: mfa.kv4_append(c, rows(), rows(dtype=torch.bfloat16), t, n),
     NotImplementedError),
    (lambda c, t, n: mfa.kv4_append(c, rows().float(), rows().float(), t, n), NotImplementedError),
    (lambda c, t, n: mfa.kv4_append(c, rows(), rows((2, 4, 2, 64)), t, n), ValueError),
    (lambda c, t, n: mfa.kv4_append("cache", rows(), rows(), t, n), TypeError),
    (lambda c, t, n: mfa.kv4_gather(c, t, n, -1), ValueError),
    (lambda c, t, n: mfa.kv4_gather(c, t, n, 4, dtype=torch.float64), NotImplementedError),
    (lambda c, t, n: mfa.flash_attn_with_kv4cache(rows()[0], c, t, n), ValueError),
    (lambda c, t, n: mfa.flash_attn_with_kv4cache(rows().float(), c, t, n), NotImplementedError),
    (lambda c, t, n: mfa.flash_attn_with_kv4cache(rows(), c, t, n, window_size=(1,)), ValueError),
    (lambda c, t, n: mfa.flash_attn_with_kv4cache(rows(), c, t, n, softcap=-1.0), ValueError),
    (lambda c, t, n: mfa.flash_attn_with_kv4cache(rows(), c, t, n, softcap=float("nan")),
     ValueError),
    (lambda c, t, n: mfa.flash_attn_with_kv4cache(rows(), c, t, n, sink_tokens=-1), ValueError),
])
def test_argument_refusals(call, exc):
    c = mfa.kv4_cache(3, 16, 2, 64, "cpu")
    with pytest.raises(exc):
        call(c, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("bad", [-1, 2.0, True, "9"])
def test_bounds_of_the_lengths_are_refused(bad):
    c = mfa.kv4_cache(3, 16, 2, 64, "cpu")
    table, n = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="max_seqlen"):
        mfa.flash_attn_with_kv4cache(rows(), c, table, n, max_seqlen=bad)
    with pytest.raises(ValueError, match="max_seqlen"):
        mfa.kv4_gather(c, table, n, bad)


def cache_params(**kw):
    c = _lib.MfaKv4Cache(k=16, v=16, k_scale=16, v_scale=16, block_table=4, table_stride=1,
                         num_pages=1, page_size=16, Hkv=2, D=64, B=1, max_pages=1, k_unit=1.0,
                         v_unit=1.0)
    for name, x in kw.items():
        setattr(c, name, x)
    return c


@pytest.mark.parametrize("kw,rc", [
    (dict(D=96), _lib.ERR_UNSUPPORTED), (dict(page_size=48), _lib.ERR_UNSUPPORTED),
    (dict(page_size=2048), _lib.ERR_UNSUPPORTED), (dict(Hkv=0), _lib.ERR_INVALID),
    (dict(k_unit=0.3), _lib.ERR_INVALID), (dict(v_unit=64.0), _lib.ERR_INVALID),
    (dict(k=24), _lib.ERR_INVALID), (dict(v_scale=None), _lib.ERR_INVALID),
    (dict(block_table=None), _lib.ERR_INVALID), (dict(num_pages=-1), _lib.ERR_INVALID),
    (dict(max_pages=2**27), _lib.ERR_INVALID), (dict(max_pages=2**27 - 255), _lib.ERR_INVALID), (dict(B=-1), _lib.ERR_INVALID)])
def test_library_checks_the_cache(kw, rc):
    r = _lib.MfaKv4Rows(k=16, v=16, L=1, dtype=_lib.BF16, lens=4)
    p = _lib.MfaKv4FwdParams(q=16, o=16, seqlens=4, Lq=1, Hq=2, dtype=_lib.BF16, scale=1.0,
                             win_left=-1, win_right=-1)
    c = cache_params(**kw)
    assert _lib.kv4_append(c, r, 0) == rc
    assert _lib.kv4_gather(c, r, 0) == rc
    assert _lib.kv4_fwd(c, p, 0) == rc
    assert _lib.kv4_fwd_workspace_size(c, p) == 0


def test_library_checks_the_rest(monkeypatch):
    c = cache_params()
    r = _lib.MfaKv4Rows(k=16, v=16, L=1, dtype=_lib.FP32)
    assert _lib.kv4_append(c, r, 0) == _lib.ERR_UNSUPPORTED
    assert _lib.kv4_gather(c, r, 0) == _lib.ERR_INVALID  # no lengths
    r.dtype, r.L = _lib.BF16, 0
    assert _lib.kv4_append(c, r, 0) == _lib.OK  # nothing to do
    for name, x in (("Hq", 3), ("Lq", -1), ("softcap", -1.0), ("win_left", -2), ("sink", -1),
                    ("seqlens", None), ("q", None)):
        p = _lib.MfaKv4FwdParams(q=16, o=16, seqlens=4, Lq=1, Hq=2, dtype=_lib.BF16, scale=1.0,
                                 win_left=-1, win_right=-1)
        setattr(p, name, x)
        assert _lib.kv4_fwd(c, p, 0) == _lib.ERR_INVALID, name
    n = _lib.MfaNormRopeParams(q=16, k=16, q_out=16, k_out=16, B=1, L=1, Hq=1, Hkv=1, D=64,
                               dtype=_lib.BF16, w_dtype=_lib.BF16, rot_dtype=_lib.FP32)
    for name, x, rc in (("D", 160, _lib.ERR_UNSUPPORTED), ("dtype", 7, _lib.ERR_UNSUPPORTED),
                        ("w_dtype", _lib.FP16, _lib.ERR_UNSUPPORTED), ("R", 7, _lib.ERR_INVALID),
                        ("R", 66, _lib.ERR_INVALID), ("R", 64, _lib.ERR_INVALID),
                        ("eps", -1.0, _lib.ERR_INVALID), ("k_out", None, _lib.ERR_INVALID)):
        m = _lib.MfaNormRopeParams.from_buffer_copy(n)
        setattr(m, name, x)
        assert _lib.qk_norm_rope(m, 0) == rc, name
    n.L = 0
    assert _lib.qk_norm_rope(n, 0) == _lib.OK
    monkeypatch.setenv("MFA_FAULT", "kv4,norm_rope")
    assert _lib.kv4_append(c, r, 0) == _lib.ERR_FAULT_INJECTED
    assert _lib.qk_norm_rope(n, 0) == _lib.ERR_FAULT_INJECTED


def test_oracle_layout_is_a_permutation():
    for D in (64, 128):
        for keys in (True, False):
            byte, half = ref.places(D, keys)
            assert sorted((2 * byte + half).tolist()) == list(range(D))


def test_oracle_rounds_to_the_nearest_code():
    """Against every code's distance, away from borders; on borders the even code."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 64, generator=g, dtype=torch.float64)
    codes, s = ref.quantise(x)
    got = ref.value(codes, s)
    levels = torch.tensor(ref.MAGNITUDES, dtype=torch.float64)
    levels = torch.cat((levels, -levels))
    grid = levels * s.double().repeat_interleave(16, -1)[..., None]
    best = (grid - x[..., None]).abs().amin(-1)
    torch.testing.assert_close((got - x).abs(), best, atol=0, rtol=0)
    tie = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] + [0.0] * 8])
    assert ref.held(tie)[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]
