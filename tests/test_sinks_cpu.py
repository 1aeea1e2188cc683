"""sink_tokens without a GPU: what is refused, and where it stands in the launch's parameters."""
import pytest
import torch

import mtlflashattn_b200 as mfa
from mtlflashattn_b200 import _kernel, _lib


@pytest.mark.parametrize("bad", [-1, 1.0, True, "4", None])
def test_bad_counts_are_refused(bad):
    t = torch.zeros(1, 8, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="sink_tokens"):
        _kernel._check_sink(bad)
    with pytest.raises(ValueError, match="sink_tokens"):
        mfa.flash_attn_host(t, t, t, sink_tokens=bad)
    with pytest.raises(ValueError, match="sink_tokens"):
        mfa.flash_attn_forward(t, t, t, 1.0, True, sink_tokens=bad)


def test_library_refuses_negative_counts():
    p = _lib.MfaFwdParams()
    p.B, p.Hq, p.Hkv, p.Lq, p.Lk, p.D, p.win_left, p.win_right = 1, 1, 1, 0, 8, 64, 3, -1
    assert _lib.fwd(p, 0) == _lib.OK
    p.sink = -1
    assert _lib.fwd(p, 0) == _lib.ERR_INVALID


def test_packed_parameters_carry_it():
    assert _lib.PARAMS_FORMAT.endswith("i4x")
    assert _kernel._check_sink(10**12) == 2**31 - 1
    assert _kernel._BiasParams(0.0, -1, -1, None).sink == 0
    raw = bytearray(_kernel._PACK.size)
    off = _lib.MfaFwdParams.sink.offset
    raw[off:off + 4] = (77).to_bytes(4, "little")
    assert _kernel._PACK.unpack(bytes(raw))[-1] == 77
