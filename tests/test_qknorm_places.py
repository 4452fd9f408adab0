"""CPU checks of where the norm and rotation may write: over q and over k, and nowhere
else on what it still reads (nothing is launched)."""
import pytest
import torch

from test_linear_checks import on
from tssm import qknorm


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(qknorm, "stream_handle", lambda t: 0)
    monkeypatch.setattr(qknorm, "on_device", lambda device, f, *args: seen.append(args))
    return seen


def test_over_the_inputs(calls):
    packed = torch.zeros(2, 5, 6, 8)
    q, k = on(packed[:, :, :4]), on(packed[:, :, 4:])
    yq, yk = qknorm.qk_norm_rotary_forward(q, k, out_q=q, out_k=k)
    assert yq is q and yk is k
    k = on(torch.zeros(2, 5, 4, 8))
    qknorm.qk_norm_rotary_forward(q, k, out_q=q)
    qknorm.qk_norm_rotary_forward(q, k, out_k=k)
    qknorm.qk_norm_rotary_forward(q, k, out_k=on(torch.zeros(2, 4, 5, 8)).transpose(1, 2))
    one = on(torch.zeros(5, 4, 8))             # strides of one element say nothing
    qknorm.qk_norm_rotary_forward(one[None], k[:1], out_q=one.unsqueeze(1).transpose(0, 1))
    assert len(calls) == 5


@pytest.mark.parametrize("places", ["swapped", "q over k", "k over q", "one for both",
                                    "other strides"])
def test_refusals(calls, places):
    q, k = on(torch.zeros(2, 4, 4, 8)), on(torch.zeros(2, 4, 4, 8))
    out = dict(out_q=k, out_k=q) if places == "swapped" else dict(out_q=k) \
        if places == "q over k" else dict(out_k=q) if places == "k over q" else \
        dict(out_q=q, out_k=q) if places == "one for both" else dict(out_q=q.transpose(1, 2))
    with pytest.raises(ValueError, match="must not overlap"):
        qknorm.qk_norm_rotary_forward(q, k, **out)
    assert not calls


def test_nothing_overlaps_when_empty(calls):
    q = on(torch.zeros(0, 4, 4, 8))
    qknorm.qk_norm_rotary_forward(q, q, out_q=q, out_k=q)
