"""GPU gradients of the delta rule's decays where a strong decay stands among slow ones:
every term of dg_t has the factor e^(g_t), so dg_t is small there, and is compared with
its own size.

dg_t = <dR, R>, R = e^(g_t) S before the step's correction and dR = dS - k (beta du)^T,
whose terms' size is <|dS| + |k| |beta du|, |R|>.  What is off relative to it: the sums and
the corrections of a chunk, 1e-5 as everywhere (test_gpu_delta); exponents of up to 90 (60
nats in units of log 2) in 24 bits, 2^-18 x log 2 = 2.6e-6, for both of a weight's steps.
1.5e-5 holds them."""
import numpy as np
import pytest
import torch

from helpers import np64
from test_gpu_delta import BF16, F16, F32, gradients, inputs

pytestmark = pytest.mark.gpu

STRONG = (-10.0, -20.0, -30.0, -45.0, -60.0)


def of_decays(q, k, v, g, beta, do, h0, dh, scale):
    """dg and its size, step by step in 64 bits."""
    B, L, Hv, V = v.shape
    per = Hv // q.shape[2]
    q, k = np.repeat(q, per, 2) * scale, np.repeat(k, per, 2)
    S = np.zeros((B, Hv, q.shape[3], V)) if h0 is None else h0
    before = []
    for t in range(L):
        S = S * np.exp(g[:, t])[..., None, None]
        before.append(S)
        u = beta[:, t][..., None] * (v[:, t] - (k[:, t][..., None] * S).sum(-2))
        S = S + k[:, t][..., :, None] * u[..., None, :]
    dS = np.zeros_like(S) if dh is None else dh
    dg, size = np.empty_like(g), np.empty_like(g)
    for t in range(L - 1, -1, -1):
        dS = dS + q[:, t][..., :, None] * do[:, t][..., None, :]
        du = beta[:, t][..., None] * (k[:, t][..., None] * dS).sum(-2)
        back = k[:, t][..., :, None] * du[..., None, :]
        dg[:, t] = ((dS - back) * before[t]).sum((-2, -1))
        size[:, t] = ((np.abs(dS) + np.abs(back)) * np.abs(before[t])).sum((-2, -1))
        dS = (dS - back) * np.exp(g[:, t])[..., None, None]
    return dg, size


def check(d, do, dh):
    dg = np64(gradients(d, do, dh)[3])
    want, size = of_decays(*(np64(d[n]) for n in ("q", "k", "v", "g", "beta")), np64(do),
                           None if d["h0"] is None else np64(d["h0"]),
                           None if dh is None else np64(dh), d["q"].shape[-1] ** -0.5)
    off = np.abs(dg - want) / np.where(size > 0, size, 1.0)
    worst = np.unravel_index(off.argmax(), off.shape)
    assert off.max() <= 1.5e-5, (off.max(), worst, dg[worst], want[worst], size[worst])
    return dg


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Hk,Hv,K,V", [(2, 2, 64, 64), (1, 3, 40, 72), (1, 2, 128, 40)])
@pytest.mark.parametrize("at", [0, 1, 3, 4, 5, 15, 16, 17, 28, 30, 31])
def test_strong_among_slow(dev, dtype, Hk, Hv, K, V, at):
    """One strong step in each chunk of 32, at its edges and those of its groups."""
    L = 32 * len(STRONG) + 20
    d = inputs(dev, 1, L, Hk, Hv, K, V, dtype, seed=at + K, h0=at % 2 == 1)
    r = torch.Generator().manual_seed(at)
    d["g"] = (-0.02 * torch.rand(1, L, Hv, generator=r)).to(dev)
    for i, g in enumerate(STRONG):
        d["g"][:, 32 * i + at] = g
    do = torch.randn(1, L, Hv, V, generator=r).to(dtype).to(dev)
    check(d, do, torch.randn(1, Hv, K, V, generator=r).to(dev) if at % 3 else None)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("many", [2, 6])
def test_strong_ones_next_to_each_other(dev, dtype, many):
    """Several strong steps in a chunk, and segments of a long sequence."""
    L, Hv, K, V = 1500, 2, 48, 40
    d = inputs(dev, 1, L, 1, Hv, K, V, dtype, seed=many, h0=True)
    r = torch.Generator().manual_seed(many)
    d["g"] = (-0.02 * torch.rand(1, L, Hv, generator=r)).to(dev)
    for first in range(0, L, 32):
        at = first + torch.randperm(min(32, L - first), generator=r)[:many]
        d["g"][:, at.to(dev)] = -20.0 * torch.rand(many, 1, generator=r).to(dev)
    do = torch.randn(1, L, Hv, V, generator=r).to(dtype).to(dev)
    check(d, do, torch.randn(1, Hv, K, V, generator=r).to(dev))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_nothing_before_the_first_step(dev, dtype):
    """Without a state in, nothing passes step 0."""
    d = inputs(dev, 2, 150, 2, 4, 64, 64, dtype, seed=3)
    dg = check(d, d["v"].flip(1).contiguous(), None)
    assert not dg[:, 0].any()
