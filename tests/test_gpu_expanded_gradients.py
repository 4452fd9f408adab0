"""Gradients that are expanded along their rows, as those of sums are: the bits of
contiguous ones."""
import pytest
import torch

import test_gpu_delta as delta
import test_gpu_linear as lin
import test_gpu_qknorm as qk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [lin.F32, lin.BF16])
@pytest.mark.parametrize("L", [1, 2, 150])
def test_linear_attention(dev, dtype, L):
    d = lin.inputs(dev, 2, L, 2, 8, 32, 4, dtype, seed=L, h0=True)
    r = torch.Generator().manual_seed(1)
    weights = torch.randn(2, L, 8, generator=r).to(dev, dtype)
    for do in (torch.ones((), device=dev, dtype=dtype).expand(2, L, 8, 4),
               weights[..., None].expand(2, L, 8, 4)):
        want = lin.gradients(d, do.contiguous())
        assert all(torch.equal(x, y) for x, y in zip(lin.gradients(d, do), want))
        lin.compare_gradients(d, do, None, dtype)


@pytest.mark.parametrize("dtype", [lin.F32, lin.BF16])
@pytest.mark.parametrize("L", [1, 2, 70])
def test_delta_rule(dev, dtype, L):
    d = delta.inputs(dev, 2, L, 2, 8, 32, 4, dtype, seed=L, h0=True)
    weights = torch.randn(2, L, 8, generator=torch.Generator().manual_seed(1)).to(dev, dtype)
    for do in (torch.ones((), device=dev, dtype=dtype).expand(2, L, 8, 4),
               weights[..., None].expand(2, L, 8, 4)):
        want = delta.gradients(d, do.contiguous())
        assert all(torch.equal(x, y) for x, y in zip(delta.gradients(d, do), want))


@pytest.mark.parametrize("dtype", [lin.F32, lin.BF16])
@pytest.mark.parametrize("K,R", [(64, 64), (40, 20), (33, 8)])
def test_norm_and_rotation(dev, dtype, K, R):
    d = qk.inputs(dev, 2, 50, 4, 2, K, R, dtype, seed=K)
    for n in ("dq", "dk"):
        d[n] = d[n][..., :1].expand_as(d[n])
    got = qk.check(d)[1]
    want = qk.backward(dict(d, dq=d["dq"].contiguous(), dk=d["dk"].contiguous()))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    one = {n: t if t is None or n in ("wq", "wk", "freq") else t[:, 3] for n, t in d.items()}
    dq, dk = qk.backward(one)[:2]
    assert torch.equal(dq, got[0][:, 3]) and torch.equal(dk, got[1][:, 3])
