"""CPU checks of the group norm's arguments (tensors that say they are on a
device; nothing is launched)."""
import pytest
import torch

from tssm import groupnorm


class On(torch.Tensor):
    """A CPU tensor that is on device ``dev`` by its own account."""
    dev = 0

    @property
    def is_cuda(self):
        return True

    def get_device(self):
        return self.dev


class OnOther(On):
    dev = 1


@pytest.fixture(autouse=True)
def no_library(monkeypatch):
    def called(*args):
        raise AssertionError("the library was called")
    monkeypatch.setattr(groupnorm.workspace, "call", called)


def on(t, other=False):
    return t.as_subclass(OnOther if other else On)


@pytest.mark.parametrize("name", ["weight", "bias", "gate", "out"])
def test_forward_operands_on_another_device(name):
    x = on(torch.zeros(3, 8))
    bad = {n: on(torch.zeros(8) if n in ("weight", "bias") else torch.zeros(3, 8), n == name)
           for n in ("weight", "bias", "gate", "out")}
    with pytest.raises(ValueError, match=f"{name} must be on x's device"):
        groupnorm.group_norm_act_forward(x, 2, **bad)


@pytest.mark.parametrize("name", ["dy", "mean", "rstd", "weight", "bias", "gate"])
def test_backward_operands_on_another_device(name):
    x, rows = on(torch.zeros(3, 8)), ("dy", "gate")
    a = {n: on(torch.zeros(3, 8) if n in rows else torch.zeros(8), n == name)
         for n in ("dy", "weight", "bias", "gate")}
    a["mean"] = on(torch.zeros(3, 2, dtype=torch.float64), name == "mean")
    a["rstd"] = on(torch.zeros(3, 2), name == "rstd")
    with pytest.raises(ValueError, match=f"{name} must be on x's device"):
        groupnorm.group_norm_act_backward(a["dy"], x, a["mean"], a["rstd"], 2, a["weight"],
                                          a["bias"], a["gate"])
