"""CPU checks of the norm and rotation of queries and keys: status codes, refusals
and the rotation's rates (nothing is launched)."""
import math

import pytest
import torch

from test_linear_checks import on
from tssm import _lib, qknorm

P = 1 << 20   # stand-in address, never dereferenced


def _fwd(dtype=1, norm=1, q=P, pos=P, pt=3, B=2, L=3, Hq=4, Hk=2, K=64, R=64):
    return _lib.lib().tssm_qk_norm_rotary_fwd(dtype, norm, 0, q, P, pos, pt, P, None, None, P, P,
                                              B, L, Hq, Hk, K, R, *[0] * 14, 1e-6, 1.0, None)


def _bwd(dw=P, ws=P, nbytes=1 << 30, q=P, K=64, B=2):
    return _lib.lib().tssm_qk_norm_rotary_bwd(1, 1, 0, P, P, q, P, P, 3, P, None, None, P, P, dw,
                                              None, B, 3, 4, 2, K, 64, *[0] * 20, 1e-6, 1.0, ws,
                                              nbytes, None)


def test_status():
    assert _fwd(dtype=3) == -4 and _fwd(pt=4) == -4 and _fwd(norm=3) == -6
    assert _fwd(q=None) == -1 and _fwd(pos=None) == -1
    assert _fwd(Hq=0) == -2 and _fwd(R=66) == -2 and _fwd(R=3) == -2 and _fwd(L=-1) == -2
    assert _fwd(K=257, R=0) == -6 and _fwd(B=1 << 20, L=1 << 12) == -6 and _fwd(Hq=1 << 20) == -6
    assert _fwd(K=1, R=0) == -6 and _fwd(K=1, R=0, norm=0, B=0) == 0
    assert _fwd(B=0) == 0 and _fwd(L=0) == 0
    assert _bwd(q=None) == -1 and _bwd(ws=None) == -5 and _bwd(nbytes=64) == -5
    assert _bwd(ws=P + 4) == -5 and _bwd(K=300) == -6
    assert _bwd(B=0, dw=None, ws=None) == 0
    assert _lib.lib().tssm_qk_norm_rotary_workspace_bytes(64) > 0
    assert _lib.lib().tssm_qk_norm_rotary_workspace_bytes(0) == -2
    assert _lib.lib().tssm_qk_norm_rotary_workspace_bytes(257) == -6


@pytest.fixture(autouse=True)
def no_library(monkeypatch):
    def called(*args):
        raise AssertionError("the library was called")
    monkeypatch.setattr(qknorm, "on_device", called)
    monkeypatch.setattr(qknorm, "stream_handle", lambda t: 0)


def operands(**change):
    d = dict(q=on(torch.zeros(2, 5, 4, 8)), k=on(torch.zeros(2, 5, 2, 8)),
             positions=on(torch.zeros(2, 5, dtype=torch.int64)),
             freqs=on(torch.zeros(4, dtype=torch.float64)), weight_q=on(torch.zeros(8)),
             weight_k=on(torch.zeros(8)))
    return dict(d, **change)


@pytest.mark.parametrize("change,error,match", [
    (dict(q=None), TypeError, "q: expected"),
    (dict(q=torch.zeros(2, 5, 4, 8)), ValueError, "HIP device"),
    (dict(q=on(torch.zeros(5, 8)), k=on(torch.zeros(5, 8))), ValueError, "expected q"),
    (dict(k=on(torch.zeros(2, 4, 2, 8))), ValueError, "k must be"),
    (dict(k=on(torch.zeros(2, 5, 2, 6))), ValueError, "k must be"),
    (dict(k=on(torch.zeros(2, 5, 2, 8, dtype=torch.float16))), TypeError, "k must be"),
    (dict(k=on(torch.zeros(2, 5, 0, 8))), ValueError, "sizes must be positive"),
    (dict(q=on(torch.zeros(2, 5, 4, 300)), k=on(torch.zeros(2, 5, 2, 300))), ValueError,
     "at most 256"),
    (dict(q=on(torch.zeros(2, 5, 4, 8, dtype=torch.int32))), TypeError, "unsupported dtype"),
    (dict(positions=None), ValueError, "go together"),
    (dict(freqs=None), ValueError, "go together"),
    (dict(freqs=on(torch.zeros(5))), ValueError, "rotate 10 channels of 8"),
    (dict(freqs=on(torch.zeros(2, 2))), ValueError, "freqs must be"),
    (dict(freqs=on(torch.zeros(4, dtype=torch.int64))), ValueError, "freqs must be"),
    (dict(positions=on(torch.zeros(2, 5, dtype=torch.int16))), TypeError, "unsupported dtype"),
    (dict(positions=on(torch.zeros(2, 6))), ValueError, "positions must be"),
    (dict(weight_q=on(torch.zeros(7))), ValueError, "weight_q must be"),
    (dict(weight_k=on(torch.zeros(8), True)), ValueError, "weight_k must be on device 0"),
    (dict(k=on(torch.zeros(2, 5, 2, 8), True)), ValueError, "k must be on device 0"),
    (dict(positions=on(torch.zeros(2, 5), True)), ValueError, "positions must be on device 0"),
    (dict(freqs=on(torch.zeros(4), True)), ValueError, "freqs must be on device 0"),
    (dict(q=on(torch.zeros(2, 5, 8, 4)).transpose(2, 3)), ValueError, "innermost"),
    (dict(norm="layer"), ValueError, "norm must be"),
    (dict(out_q=on(torch.zeros(2, 5, 4, 9))), ValueError, "out_q must be"),
    (dict(out_k=on(torch.zeros(2, 5, 2, 8, dtype=torch.float16))), TypeError, "out_k must be"),
    (dict(out_k=on(torch.zeros(2, 5, 2, 8), True)), ValueError, "out_k must be on device"),
    (dict(out_q=on(torch.zeros(2, 1, 4, 8)).expand(2, 5, 4, 8)), ValueError, "share memory"),
])
def test_refusals(change, error, match):
    with pytest.raises(error, match=match):
        qknorm.qk_norm_rotary_forward(**operands(**change))


def test_backward_refusals():
    d = operands()
    dq, dk = on(torch.zeros(2, 5, 4, 8)), on(torch.zeros(2, 5, 2, 8))
    with pytest.raises(ValueError, match="dq_out must be"):
        qknorm.qk_norm_rotary_backward(dk, dk, **d)
    with pytest.raises(TypeError, match="dk_out must be"):
        qknorm.qk_norm_rotary_backward(dq, dk.half(), **d)
    with pytest.raises(ValueError, match="dk_out must be on device"):
        qknorm.qk_norm_rotary_backward(dq, on(torch.zeros(2, 5, 2, 8), True), **d)


def test_frequencies():
    f = qknorm.rotary_frequencies(8)
    assert f.dtype == torch.float64
    assert f.tolist() == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-12)
    assert torch.equal(qknorm.rotary_frequencies(8, factor=4.0) * 4.0, f)
    b = qknorm.rotary_frequencies(8, factor=4.0, how="base")
    assert b[0] == 1.0 and float(b[3] * 4.0) == pytest.approx(0.001, rel=1e-12)
    # 1000 positions: 159, 15.9, 1.59 and 0.159 turns
    p = qknorm.rotary_frequencies(8, factor=4.0, how="parts", trained=1000, fast=32.0, slow=1.0)
    turns = 1000 / (2 * math.pi)
    mixed = [f[i] * (s + (1 - s) / 4) for i, s in
             ((1, (0.1 * turns - 1) / 31), (2, (0.01 * turns - 1) / 31))]
    assert p.tolist() == pytest.approx([1.0, *map(float, mixed), 0.00025], rel=1e-12)
    assert qknorm.rotary_amplitude(1.0) == 1.0
    assert qknorm.rotary_amplitude(math.e) == pytest.approx(1.1)
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, factor=0.5),
                dict(dim=8, how="other"), dict(dim=8, how="parts"),
                dict(dim=8, how="parts", trained=10, fast=1.0, slow=2.0),
                dict(dim=2, how="base", factor=2.0)):
        with pytest.raises(ValueError):
            qknorm.rotary_frequencies(**bad)
