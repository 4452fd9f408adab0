"""The mixer of examples/delta_mixer.py: the delta rule and the group norm
together, against the formulas in 64 bits, in training and in serving."""
import copy
import importlib.util
import math
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

spec = importlib.util.spec_from_file_location(
    "delta_mixer", Path(__file__).resolve().parents[1] / "examples" / "delta_mixer.py")
M = importlib.util.module_from_spec(spec)
spec.loader.exec_module(M)


def test_recall_batch():
    """Every answer is the value that its key was given last."""
    keys, values = 5, 7
    key, value, answer = M.recall_batch(4, 40, keys, values, torch.Generator().manual_seed(2))
    for b in range(4):
        held = {}
        for k, v, a in zip(key[b].tolist(), value[b].tolist(), answer[b].tolist()):
            if v == values:
                assert a == held[k]
            else:
                assert a == -1
                held[k] = v
    assert (answer >= 0).any()


def plain(m, x):
    """DeltaMixer.forward by its formulas, in the precision of m and x."""
    B, L, _ = x.shape
    q, k, v, z, a, b = m.inp(x).split(m.parts, dim=-1)
    q, k = (F.normalize(t.reshape(B, L, m.Hk, m.K), dim=-1) for t in (q, k))
    q, k = (t.repeat_interleave(m.Hv // m.Hk, dim=2) for t in (q, k))
    v = F.silu(v).reshape(B, L, m.Hv, m.V)
    g, beta = -F.softplus(a + m.decay), torch.sigmoid(b)
    S, o = x.new_zeros(B, m.Hv, m.K, m.V), []
    for t in range(L):
        S = S * g[:, t, :, None, None].exp()
        u = beta[:, t, :, None] * (v[:, t] - (S * k[:, t, :, :, None]).sum(2))
        S = S + k[:, t, :, :, None] * u[:, :, None]
        o.append((S * q[:, t, :, :, None]).sum(2) * m.K ** -0.5)
    o = torch.stack(o, 1)
    o = o - o.mean(-1, keepdim=True)
    o = o * (o.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    return m.out(o.reshape(B, L, -1) * m.norm * F.silu(z))


# The longest sums have 1024 terms (an input weight's gradient): 32 x 6e-8 = 2e-6
# of their size, through five stages of the layer, and a row that the norm
# stretches by up to five (heads whose outputs are small): 5e-5 of the largest.
TOL = 5e-5


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,Hk,Hv,K,V", [(2, 70, 1, 2, 32, 32), (1, 7, 2, 4, 24, 40),
                                           (3, 33, 2, 2, 64, 48)])
def test_mixer_is_its_formulas(dev, B, L, Hk, Hv, K, V):
    torch.manual_seed(5)
    m = M.DeltaMixer(48, Hk, Hv, K, V, torch.float32)
    ref = copy.deepcopy(m).double()
    m = m.to(dev)
    x = torch.randn(B, L, 48, dtype=torch.float64)
    w = torch.randn(B, L, 48, dtype=torch.float64)
    want = plain(ref, x)
    (want * w).sum().backward()
    got = m(x.float().to(dev))
    (got * w.float().to(dev)).sum().backward()
    pairs = [("y", got, want)] + [(n, p.grad, r.grad) for (n, p), r in
                                  zip(m.named_parameters(), ref.parameters())]
    for name, a, b in pairs:
        err = (a.double().cpu() - b).abs().max() / b.abs().max()
        assert err <= TOL, f"{name}: {err:.2e}"


@pytest.mark.gpu
def test_prompt_and_steps_are_the_whole(dev):
    torch.manual_seed(6)
    model = M.Recall(9, 11, D=32, key_heads=1, heads=2, K=16, V=24, dtype=torch.float32).to(dev)
    key, value, _ = (t.to(dev) for t in M.recall_batch(3, 80, 9, 11,
                                                       torch.Generator().manual_seed(3)))
    with torch.no_grad():
        whole = model(key, value)
    for prompt in (1, 40, 79):
        served = M.serve(model, key, value, prompt)
        assert (served - whole).abs().max() <= TOL * whole.abs().max()


@pytest.mark.gpu
def test_mixer_learns_recall(dev):
    """The loss falls clearly below that of an answer at random, log(values)."""
    torch.manual_seed(7)
    keys, values = 8, 16
    model = M.Recall(keys, values, D=64, key_heads=2, heads=2).to(dev)
    losses = M.train(model, 150, 32, 64, keys, values, torch.Generator().manual_seed(4))
    assert all(math.isfinite(x) for x in losses)
    assert sum(losses[-10:]) / 10 < 0.75 * math.log(values)
