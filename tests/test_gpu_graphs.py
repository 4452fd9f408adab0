"""Calls of several launches captured in graphs, replayed after their stream's
workspace was replaced, with eager work between the replays."""
import pytest
import torch

from test_gpu_delta import BF16, F32, inputs
import test_gpu_groupnorm as norm

pytestmark = pytest.mark.gpu


def forward(d):
    from tssm import gated_delta_forward
    return gated_delta_forward(d["q"], d["k"], d["v"], d["g"], d["beta"], h0=d["h0"],
                               return_state=True)


def backward(d):
    from tssm import gated_delta_backward
    return gated_delta_backward(d["q"], d["k"], d["v"], d["g"], d["beta"], d["v"], h0=d["h0"])


def series(d):
    from tssm import group_norm_act_backward, group_norm_act_forward
    y, mean, rstd = group_norm_act_forward(d["x"], 4, d["w"], d["b"], return_stats=True)
    return (y, *group_norm_act_backward(d["dy"], d["x"], mean, rstd, 4, d["w"], d["b"])[:3])


def ssd(d):
    from tssm import ssd_scan_forward
    B, L, H, _ = d["v"].shape
    bc = torch.cat([d["q"], d["k"]], -1)
    return (ssd_scan_forward(d["v"], -d["g"], d["beta"][0, 0], bc, bc, fused=False),)


def delta(L, dtype=BF16):
    return lambda dev, seed: inputs(dev, 1, L, 2, 2, 32, 64, dtype, seed=seed, h0=True)


@pytest.mark.parametrize("run,make,larger", [
    (forward, delta(100), delta(9000)),
    (forward, delta(5000), delta(40000)),          # segments
    (backward, delta(100, F32), delta(5000, F32)),
    (series, lambda dev, seed: norm.inputs(dev, 3, 200, 64, F32, False, seed=seed),
     lambda dev, seed: norm.inputs(dev, 30, 2000, 256, F32, False, seed=seed)),
    (ssd, delta(100, F32), delta(9000, F32)),
])
def test_replays_after_a_larger_call(dev, run, make, larger):
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        d = make(dev, 1)
        run(d)                                     # loads the kernels, fills a workspace
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = run(d)
        run(larger(dev, 2))                        # a larger workspace takes its place
        for seed in (3, 4, 5):
            for t, new in zip(d.values(), make(dev, seed).values()):
                if t is not None:
                    t.copy_(new)
            rest = [torch.full((1 << 16,), seed, device=dev) for _ in range(8)]
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, run(d))), seed
            assert all((t == seed).all() for t in rest)
