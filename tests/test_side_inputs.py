"""CPU checks of the small side inputs that kernels read as float32."""
import pytest
import torch

from tssm import launch


@pytest.fixture(autouse=True)
def on_host(monkeypatch):
    monkeypatch.setattr(launch, "need_gpu", lambda t, what: t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_other_float_types_are_converted_in_place(dtype):
    """Values and strides stay: the caller's strides describe the copy too."""
    t = torch.arange(24.0).reshape(2, 3, 4).to(dtype).permute(2, 0, 1)
    x = launch.as_f32(t, "g")
    assert x.dtype == torch.float32 and x.stride() == t.stride()
    assert torch.equal(x.double(), t.double())


def test_refusals():
    t = torch.zeros(2, 3)
    assert launch.as_f32(t, "g") is t
    with pytest.raises(TypeError, match="must be dense"):
        launch.as_f32(t.bfloat16()[:, :1].expand(2, 3), "g")
    with pytest.raises(TypeError, match="expected a float"):
        launch.as_f32(t.int(), "g")
