"""CPU checks that gradients which are expanded along their rows (those of sums) are
taken: what reaches the library has rows of its own (nothing is launched)."""
import pytest
import torch

from test_linear_checks import on
from tssm import delta, linear

B, HK, HV, K, V = 2, 2, 4, 8, 6


@pytest.fixture
def calls(monkeypatch):
    """The arguments of the calls that would be made."""
    seen = []
    for module in (delta, linear):
        monkeypatch.setattr(module, "stream_handle", lambda t: 0)
    monkeypatch.setattr(linear, "on_device", lambda device, f, *args: seen.append(args))
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


def test_other_rows_are_refused(calls):
    x = [on(torch.zeros(B, 3, h, n)) for h, n in ((HK, K), (HK, K), (HV, V))]
    with pytest.raises(ValueError, match="do: innermost"):
        linear.linear_attention_backward(*x, on(torch.zeros(B, 3, HV)),
                                         on(torch.zeros(B, 3, V, HV)).transpose(2, 3))
