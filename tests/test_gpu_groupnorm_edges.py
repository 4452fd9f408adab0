"""GPU tests of the group norm at its edges."""
import pytest
import torch

from test_gpu_groupnorm import F32

pytestmark = pytest.mark.gpu


def test_many_short_series(dev):
    """20 million series of two positions: more workgroups than 2^32 work-items."""
    from tssm import group_norm_act_backward, group_norm_act_forward
    N, S, C = 20_000_000, 2, 4
    r = torch.Generator(device=dev).manual_seed(33)
    x = torch.randn(N, S, C, generator=r, device=dev)
    dy = torch.randn(N, S, C, generator=r, device=dev)
    y, mean, rstd = group_norm_act_forward(x, 1, act="none", return_stats=True)
    w = torch.ones(C, device=dev)
    dx, dw, _, _ = group_norm_act_backward(dy, x, mean, rstd, 1, w, act="none")
    total = torch.zeros(C, dtype=torch.float64, device=dev)
    for lo in range(0, N, 4_000_000):
        s = slice(lo, lo + 4_000_000)
        x64, d64 = x[s].double(), dy[s].double()
        m = x64.mean((1, 2), keepdim=True)
        rs = ((x64 - m).square().mean((1, 2), keepdim=True) + 1e-5).rsqrt()
        xh = (x64 - m) * rs
        want = rs * (d64 - d64.mean((1, 2), keepdim=True)
                     - xh * (d64 * xh).mean((1, 2), keepdim=True))
        assert (y[s].double() - xh).abs().max() <= 1e-5 * xh.abs().max(), lo
        assert (dx[s].double() - want).abs().max() <= 1e-5 * want.abs().max(), lo
        total += (d64 * xh).sum((0, 1))
    # dw is some 6e3, joined from 128 fp32 sums of 1.6e5 terms of both signs that reach
    # 6e2: roundings of at most 4e-5 each, 2e-2 a sum, 2e-1 in all
    assert (dw.double() - total).abs().max() <= 1.0


@pytest.mark.parametrize("shape", [(4, 0, 32), (3, 2, 0, 5, 32)])
def test_statistics_of_no_positions(dev, shape):
    """A mean over nothing is 0 / 0."""
    from tssm import group_norm_act_forward
    torch.full((4, 2), 7.0, device=dev, dtype=torch.float64)      # what free memory may hold
    y, mean, rstd = group_norm_act_forward(torch.empty(shape, device=dev), 2, return_stats=True)
    assert y.shape == shape and mean.shape == rstd.shape == (shape[0], 2)
    assert torch.isnan(mean).all() and torch.isnan(rstd).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("N,S,C", [(6, 1, 64), (3, 70, 64), (2, 1, 4 * 4099)])
def test_statistics_that_are_not_finite(dev, N, S, C, value):
    """rstd tells of a group that is not finite, in every form of the kernels."""
    from tssm import group_norm_act_forward
    x = torch.randn(N, S, C, generator=torch.Generator().manual_seed(31)).to(dev)
    x[1, 0, C // 4 + 4] = value
    y, mean, rstd = group_norm_act_forward(x, 4, return_stats=True)
    bad = torch.zeros(N, 4, dtype=torch.bool, device=dev)
    bad[1, 1] = True
    assert torch.equal(torch.isnan(rstd), bad)
    assert torch.equal(~torch.isfinite(mean), bad)
    assert torch.isnan(y[1, :, C // 4:C // 2]).all()


@pytest.mark.parametrize("N,S,G,C", [(64, 1, 4, 256), (64, 1, 4, 192), (5, 1, 2, 4099 * 2), (2, 500, 4, 256),
                                     (3, 7, 2, 24), (2, 9, 513, 1026)])
@pytest.mark.parametrize("gated", [False, True])
def test_offsets_of_many_deviations(dev, N, S, G, C, gated):
    """Values of 1e5 with a deviation of 1, in every form of the kernels.  x - mean is
    exact where the mean is what its two parts say (a 24-bit mean would be off by up
    to 4e-3), so the tolerance is the usual one."""
    from test_gpu_groupnorm import check, inputs
    d = inputs(dev, N, S, C, F32, gated, seed=C + S)
    d["x"] = d["x"] + 1e5
    check(d, G, "silu", F32)


@pytest.mark.parametrize("N,S,C,size", [(64, 1, 24, 1e10), (64, 333, 24, 1e10), (64, 5, 16800, 1e10),
                                        (64, 1, 16800, 1e15), (3, 400, 16800, 1e15)])
def test_large_constant_groups(dev, N, S, C, size):
    """Groups of one large value each: what rounding leaves of their variance may
    be below 0, which is no reason for NaN.  x - mean stays within 2^-46 of x (the
    mean's second part is good to 2^-24 of some 2^-24), rstd within eps^-1/2."""
    from tssm import group_norm_act_forward
    r = torch.Generator().manual_seed(32)
    x = (size * (1.0 + torch.rand(N, 1, 8, 1, generator=r))).expand(N, S, 8, C // 8)
    y, mean, rstd = group_norm_act_forward(x.reshape(N, S, C).to(dev), 8, act="none",
                                           return_stats=True)
    assert torch.isfinite(y).all()
    assert (rstd > 0).all() and (rstd <= 316.3).all()
    assert y.abs().max() <= 2.0 ** -45 * size * 316.3
