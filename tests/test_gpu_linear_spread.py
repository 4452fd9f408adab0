"""How far an input or gradient of linear attention's backward that is not finite reaches:
its chunk of 64 steps and what depends on it; other heads, sequences and chunks keep
their gradients.  Tolerances as in test_gpu_linear."""
import numpy as np
import pytest
import torch

from helpers import assert_close, np64
from oracle import mixer_oracle as M
from test_gpu_linear import BF16, F16, F32, NAMES, TOL, gradients, inputs

pytestmark = pytest.mark.gpu

# which chunks' gradients depend on a value of one step: its own and those before or after
BEFORE = {"q": ("dk", "dv", "dg"), "do": ("dk", "dv", "dg"), "k": (), "v": ()}
AFTER = {"q": (), "do": (), "k": ("dq", "dg"), "v": ("dq", "dg")}


@pytest.mark.parametrize("dtype,B,L,H,K,V", [(F32, 2, 300, 2, 64, 40), (BF16, 1, 330, 2, 128, 64),
                                             (F16, 2, 200, 1, 40, 72), (BF16, 1, 2000, 2, 64, 64)])
@pytest.mark.parametrize("t0", [70, 127])
@pytest.mark.parametrize("name", ["q", "k", "v", "do"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_not_finite(dev, dtype, B, L, H, K, V, t0, name, value):
    d = inputs(dev, B, L, H, H, K, V, dtype, seed=L + K, h0=True, rate=0.05)
    r = torch.Generator().manual_seed(1)
    do = torch.randn(B, L, H, V, generator=r).to(dtype).to(dev)
    dh = torch.randn(B, H, K, V, generator=r).to(dev)
    ref = M.linear_backward(*(np64(d[n]) for n in ("q", "k", "v", "g")), np64(do),
                            h0=np64(d["h0"]), dh_last=np64(dh))
    (do if name == "do" else d[name])[B - 1, t0, H - 1, 5] = value
    first = t0 // 64 * 64
    last = min(first + 64, L)
    touched = False
    for n, x, y in zip(NAMES, gradients(d, do, dh), ref):
        keep = np.ones(y.shape, dtype=bool)
        if n == "dh0":
            keep[B - 1, H - 1] = name in ("k", "v")
        else:
            keep[B - 1, first:last, H - 1] = False
            if n in BEFORE[name]:
                keep[B - 1, :first, H - 1] = False
            if n in AFTER[name]:
                keep[B - 1, last:, H - 1] = False
        tol = TOL[dtype] if n in ("dq", "dk", "dv") else TOL[F32]
        assert_close(np64(x)[keep], y[keep], tol, n)
        touched |= not np.isfinite(np64(x)).all()
    assert touched
