"""CPU checks that gradients which are expanded along their rows (those of sums) are
taken: what reaches the library has rows of its own (nothing is launched)."""
import pytest
import torch

from test_linear_checks import on
from tssm import delta, linear, qknorm

B, HK, HV, K, V = 2, 2, 4, 8, 6


@pytest.fixture
def calls(monkeypatch):
    """The arguments of the calls that would be made."""
    seen = []
    for module in (delta, linear, qknorm):
        monkeypatch.setattr(module, "stream_handle", lambda t: 0)
    for module in (linear, qknorm):
        monkeypatch.setattr(module, "on_device", lambda device, f, *args: seen.append(args))
    monkeypatch.setattr(delta.workspace, "call", lambda *args: seen.append(args))
    return seen


def gradients_of_sums(L):
    """dO of o.sum(), and of o.sum(-1) against weights, whose rows repeat one value."""
    one = torch.ones(()).expand(B, L, HV, V)
    return [one, torch.rand(B, L, HV)[..., None].expand(B, L, HV, V),
            torch.rand(B, L, 16 * HV)[:, :, ::16, None].expand(B, L, HV, V)]


@pytest.mark.parametrize("L", [1, 2, 40])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_linear_attention(calls, L, which):
    do = gradients_of_sums(L)[which]
    x = [on(torch.zeros(B, L, h, n)) for h, n in ((HK, K), (HK, K), (HV, V))]
    linear.linear_attention_backward(*x, on(torch.zeros(B, L, HV)), on(do))
    assert calls[0][0] == "tssm_linear_attention_backward"
    assert calls[0][-4:-1] == (L * HV * V, HV * V, V)      # dO's strides, before the scale
    linear.linear_attention_forward(*x[:2], on(do), on(torch.zeros(B, L, HV)))
    assert calls[1][0] == "tssm_linear_attention_forward"


@pytest.mark.parametrize("L", [1, 2, 40])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_delta_rule(calls, L, which):
    do = gradients_of_sums(L)[which]
    x = [on(torch.zeros(B, L, h, n)) for h, n in ((HK, K), (HK, K), (HV, V))]
    g = on(torch.zeros(B, L, HV))
    delta.gated_delta_backward(*x, g, g, on(do))
    assert calls[0][0] == "tssm_gated_delta_backward"
    assert calls[0][-4:-1] == (L * HV * V, HV * V, V)


@pytest.mark.parametrize("lead", [(3,), (2, 1), (2, 9)])
@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_norm_and_rotation(calls, lead, which):
    q, k = (on(torch.zeros(*lead, h, K)) for h in (HV, HK))
    dq, dk = (on(torch.rand(*lead, h)[..., None].expand(*lead, h, K) if which in (n, "both") else
                 torch.zeros(*lead, h, K)) for n, h in (("q", HV), ("k", HK)))
    qknorm.qk_norm_rotary_backward(dq, dk, q, k)
    name, *args = calls[0]
    assert name == "tssm_qk_norm_rotary_bwd"
    lead = lead if len(lead) == 2 else (lead[0], 1)
    at = args.index(HV, 14)                       # (B, L, Hq, Hk, K, R, strides)
    assert tuple(args[at - 2:at + 4]) == (*lead, HV, HK, K, 0)
    rows = args[at + 4:at + 10]
    step = 0 if q.dim() == 3 else 1
    assert rows[2::3] == [K, K] and rows[0::3] == [lead[1] * HV * K, lead[1] * HK * K]
    assert rows[1::3] == [step * HV * K, step * HK * K]


def test_other_rows_are_refused(calls):
    x = [on(torch.zeros(B, 3, h, n)) for h, n in ((HK, K), (HK, K), (HV, V))]
    with pytest.raises(ValueError, match="do: innermost"):
        linear.linear_attention_backward(*x, on(torch.zeros(B, 3, HV)),
                                         on(torch.zeros(B, 3, V, HV)).transpose(2, 3))
    q = on(torch.zeros(2, 3, HV, K))
    with pytest.raises(ValueError, match="dk_out: innermost"):
        qknorm.qk_norm_rotary_backward(q, on(torch.zeros(2, 3, K, HV)).transpose(2, 3), q, q)
