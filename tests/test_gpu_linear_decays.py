"""GPU gradients of linear attention's decays where a strong decay stands among slow
ones: every term of dg_t has the factor e^(g_t), so dg_t is small there, and is compared
with its own size.

dg_t = <dS, e^(g_t) S> over K x V products, whose size is <|dS|, e^(g_t) |S|>.  What is
off relative to it: the exponents of weights that cross the step, which have 24 bits of up
to 90 (60 nats in units of log 2), 2^-18 x log 2 = 2.6e-6 of the weight; the sums over K,
V and the steps, some hundred roundings of 2^-24 that add up like a walk's, 1e-6.  1e-5
holds both (the tolerance of all fp32 sums here)."""
import numpy as np
import pytest
import torch

from helpers import np64
from test_gpu_linear import BF16, F16, F32, gradients, inputs

pytestmark = pytest.mark.gpu

STRONG = (-10.0, -20.0, -30.0, -45.0, -60.0)


def of_decays(q, k, v, g, do, h0, dh, scale):
    """dg and its size, step by step in 64 bits."""
    B, L, Hv, V = v.shape
    per = Hv // q.shape[2]
    q, k = np.repeat(q, per, 2) * scale, np.repeat(k, per, 2)
    S = np.zeros((B, Hv, q.shape[3], V)) if h0 is None else h0
    before = []
    for t in range(L):
        S = S * np.exp(g[:, t])[..., None, None]
        before.append(S)
        S = S + k[:, t][..., :, None] * v[:, t][..., None, :]
    dS = np.zeros_like(S) if dh is None else dh
    dg, size = np.empty_like(g), np.empty_like(g)
    for t in range(L - 1, -1, -1):
        dS = dS + q[:, t][..., :, None] * do[:, t][..., None, :]
        dg[:, t] = (dS * before[t]).sum((-2, -1))
        size[:, t] = (np.abs(dS) * np.abs(before[t])).sum((-2, -1))
        dS = dS * np.exp(g[:, t])[..., None, None]
    return dg, size


def check(dev, d, do, dh):
    dg = np64(gradients(d, do, dh)[3])
    want, size = of_decays(*(np64(d[n]) for n in ("q", "k", "v", "g")), np64(do),
                           None if d["h0"] is None else np64(d["h0"]),
                           None if dh is None else np64(dh), d["q"].shape[-1] ** -0.5)
    off = np.abs(dg - want) / np.where(size > 0, size, 1.0)
    worst = np.unravel_index(off.argmax(), off.shape)
    assert off.max() <= 1e-5, (off.max(), worst, dg[worst], want[worst], size[worst])
    return dg


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Hk,Hv,K,V", [(2, 2, 64, 64), (1, 3, 40, 72), (1, 2, 128, 40),
                                       (2, 2, 32, 100)])
@pytest.mark.parametrize("at", [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 62, 63])
def test_strong_among_slow(dev, dtype, Hk, Hv, K, V, at):
    """One strong step in each chunk of 64, at its edges and those of its blocks."""
    L = 64 * len(STRONG) + 30
    d = inputs(dev, 1, L, Hk, Hv, K, V, dtype, seed=at + K, h0=at % 2 == 1)
    r = torch.Generator().manual_seed(at)
    d["g"] = (-0.02 * torch.rand(1, L, Hv, generator=r)).to(dev)
    for i, g in enumerate(STRONG):
        d["g"][:, 64 * i + at] = g
    do = torch.randn(1, L, Hv, V, generator=r).to(dtype).to(dev)
    check(dev, d, do, torch.randn(1, Hv, K, V, generator=r).to(dev) if at % 3 else None)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("many", [2, 6])
def test_strong_ones_next_to_each_other(dev, dtype, many):
    """Several strong steps in a chunk, and segments of a long sequence."""
    L, Hv, K, V = 1700, 2, 48, 40
    d = inputs(dev, 1, L, 1, Hv, K, V, dtype, seed=many, h0=True)
    r = torch.Generator().manual_seed(many)
    d["g"] = (-0.02 * torch.rand(1, L, Hv, generator=r)).to(dev)
    for first in range(0, L, 64):
        at = first + torch.randperm(min(64, L - first), generator=r)[:many]
        d["g"][:, at.to(dev)] = -20.0 * torch.rand(many, 1, generator=r).to(dev)
    do = torch.randn(1, L, Hv, V, generator=r).to(dtype).to(dev)
    check(dev, d, do, torch.randn(1, Hv, K, V, generator=r).to(dev))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_nothing_before_the_first_step(dev, dtype):
    """Without a state in, nothing passes step 0."""
    d = inputs(dev, 2, 150, 2, 4, 64, 64, dtype, seed=3)
    do = d["v"].flip(1).contiguous()
    dg = check(dev, d, do, None)
    assert not dg[:, 0].any()


@pytest.mark.parametrize("dtype,L,t0", [(F32, 40, 17), (BF16, 300, 70), (F16, 300, 64),
                                        (F32, 2000, 700), (BF16, 9, 4)])
def test_a_reset_drops_what_is_finite(dev, dtype, L, t0):
    """However large: the state before g = -inf is at 2^100, values there at 2^60 (2^15 in
    fp16), and what comes after has the bits of its own sequence."""
    from tssm import linear_attention_forward, linear_attention_step
    d = inputs(dev, 1, L, 1, 2, 64, 40, dtype, seed=L, h0=True, rate=0.1)
    d["g"][:, t0] = -float("inf")
    ops = [d[n] for n in ("q", "k", "v", "g")]
    want = linear_attention_forward(*ops, h0=d["h0"], return_state=True)
    d["v"][:, :t0] *= 2.0 ** 15 / d["v"].abs().max() if dtype == F16 else 2.0 ** 60
    d["k"][:, :t0] *= 2.0 ** 8
    got = linear_attention_forward(*ops, h0=d["h0"] * 2.0 ** 100, return_state=True)
    assert torch.equal(got[0][:, t0:], want[0][:, t0:]) and torch.equal(got[1], want[1])
    at, state = [t[:, t0] for t in ops], d["h0"] * 2.0 ** 100
    o, zero = linear_attention_step(*at, state), torch.zeros_like(state)
    assert torch.equal(o, linear_attention_step(*at, zero)) and torch.equal(state, zero)
