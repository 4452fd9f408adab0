"""Linear attention's gradients where one step of all value heads is longer than a chunk's
31 bits allow (66 heads of 2^16 columns in fp32: 17 MB a step)."""
import pytest
import torch

import test_gpu_linear as lin

pytestmark = pytest.mark.gpu


def test_backward(dev):
    d = lin.inputs(dev, 1, 3, 3, 66, 4, 1 << 16, lin.F32, seed=1, h0=True)
    assert d["v"].stride(1) * 4 * 129 >= 1 << 31
    lin.check_gradients(dev, d, lin.F32, seed=2)
    torch.cuda.empty_cache()
