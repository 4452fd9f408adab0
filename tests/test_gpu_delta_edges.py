"""GPU parity of the gated delta rule at its edges: step strides that are no
row's length, tensors past launch limits, values that are not finite in every
form of the kernels.  Tolerances as in test_gpu_delta."""
import pytest
import torch

from helpers import assert_close, np64
from oracle import mixer_oracle as M
from test_gpu_delta import BF16, F32, NAMES, TOL, gradients, inputs

pytestmark = pytest.mark.gpu


def compare_gradients(d, do, dh, dtype):
    ref = M.delta_backward(**{n: None if t is None else np64(t) for n, t in d.items()},
                           do=np64(do), dh_last=None if dh is None else np64(dh))
    for name, x, y in zip(NAMES, gradients(d, do, dh), ref):
        assert_close(x, y, TOL[dtype] if name in ("dq", "dk", "dv") else TOL[F32], name)


def one_step(t, layout):
    """t [B, 1, H, N] as a view whose step stride is no row's length."""
    B, _, H, N = t.shape
    if layout == "innermost":       # [B, H, N, L] with L = 1
        return t.new_empty(B, H, N, 1).permute(0, 3, 1, 2).copy_(t)
    if layout == "shared":          # one head for all
        return t[:, 0, 0][:, None].expand(B, H, N).unsqueeze(1)
    # 31 rows of this stride pass 32 bits
    return t.contiguous().as_strided(t.shape, (H * N, 1 << 30, N, 1))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout,step", [("innermost", 1), ("shared", 0), ("far", 1 << 30)])
def test_backward_of_one_step(dev, dtype, layout, step):
    """The stride of a dimension of one element says nothing."""
    r = torch.Generator().manual_seed(22)
    d = inputs(dev, 2, 1, 3, 3, 32, 32, dtype, seed=21, h0=True)
    do = torch.randn(2, 1, 3, 32, generator=r).to(dtype).to(dev)
    dh = torch.randn(2, 3, 32, 32, generator=r).to(dev)
    for n in ("q", "k", "v"):
        d[n] = one_step(d[n], layout)
        assert d[n].stride(1) == step
    compare_gradients(d, one_step(do, layout), dh, dtype)
