"""Group norm with an activation, channels last, and its gradients (no
reference counterpart; the reference's own norm is ``layernorm_kernel``).

    xhat = (x - mean) rstd         over a group's C / groups channels and all S positions
    y = act(xhat w + b)            without a gate
    y = (xhat w + b) act(gate)     with one

x is [N, C] (statistics per row, as after a multi-head mixer) or [N, ..., C],
where the middle dimensions are positions that share their statistics.  Sums
and statistics are fp32, the mean 64 bits (fixed order: repeated runs give identical bits);
``weight`` and ``bias`` are read as float32 and their gradients are float32.
"""
from __future__ import annotations

import torch

from . import _lib, workspace
from .launch import as_f32, dcode, need_gpu, ptr, stream_handle

_ACT = {"none": 0, "silu": 1}


def _view(t, what):
    """t [N, ..., C] as (N, S, C, stride of n, stride of s): the middle
    dimensions must be one run of positions."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 2 and stride[1] == 1:
        return shape[0], 1, shape[1], stride[0], shape[1]
    if len(shape) < 2:
        raise ValueError(f"{what} must be [N, ..., C]")
    if stride[-1] != 1 and shape[-1] != 1:
        raise ValueError(f"{what}: innermost dimension must be contiguous")
    S, step = 1, None
    if 0 in shape[1:-1]:
        return shape[0], 0, shape[-1], stride[0], shape[-1]
    for n, s in zip(reversed(shape[1:-1]), reversed(stride[1:-1])):
        if n == 1:
            continue
        if step is None:
            step = s
        elif s != step * S:
            raise ValueError(f"{what}: the middle dimensions must be evenly strided "
                             "(one run of positions)")
        S *= n
    return shape[0], S, shape[-1], stride[0], step if step is not None else shape[-1]


def _same(t, what, x):
    need_gpu(t, what)
    if t.shape != x.shape:
        raise ValueError(f"{what} must be {list(x.shape)}, got {list(t.shape)}")
    if t.dtype != x.dtype:
        raise TypeError(f"{what} must be {x.dtype}, got {t.dtype}")
    if t.get_device() != x.get_device():
        raise ValueError(f"{what} must be on x's device")
    return _view(t, what)[3:]


def _channels(t, what, C, device):
    if t is None:
        return None
    need_gpu(t, what)
    if t.shape != (C,):
        raise ValueError(f"{what} must be [{C}], got {list(t.shape)}")
    if t.get_device() != device:
        raise ValueError(f"{what} must be on x's device")
    return t if t.dtype == torch.float32 and t.is_contiguous() else as_f32(t, what).contiguous()


def _operands(x, groups, weight, bias, gate, act):
    need_gpu(x, "x")
    code = dcode(x, "x")
    N, S, C, sx_n, sx_s = _view(x, "x")
    groups = int(groups)
    if groups <= 0 or C == 0 or C % groups:
        raise ValueError(f"groups = {groups} must divide the {C} channels")
    if act not in _ACT:
        raise ValueError(f"act must be 'none' or 'silu', got {act!r}")
    sg = _same(gate, "gate", x) if gate is not None else (0, 0)
    device = x.get_device()
    return (code, _ACT[act], N, S, groups, C // groups, (sx_n, sx_s), sg,
            _channels(weight, "weight", C, device), _channels(bias, "bias", C, device))


def group_norm_act_forward(x, groups, weight=None, bias=None, gate=None, *, act="silu",
                           eps=1e-5, return_stats=False, out=None):
    """Group norm of x [N, ..., C] (float32 / bfloat16 / float16) in ``groups``
    groups of neighbouring channels, with an activation ('silu' or 'none'),
    applied to the result or, where ``gate`` (shape and dtype of x) is given,
    to the gate that multiplies it.  weight, bias [C] or None.

    Returns y (dtype of x; ``out`` if given) and, with ``return_stats``, mean
    (float64: groups whose values almost agree need it) and rstd (float32)
    [N, groups], which the backward needs (NaN where there are no positions).
    """
    code, act_, N, S, G, Cg, sx, sg, w, b = _operands(x, groups, weight, bias, gate, act)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype) if out is None else out
    sy = _same(y, "out", x)
    mean = rstd = None
    if return_stats:
        mean = torch.empty(N, G, device=x.device, dtype=torch.float64)
        rstd = torch.empty(N, G, device=x.device, dtype=torch.float32)
    if N and (S or return_stats):
        workspace.call("tssm_group_norm_act_fwd", x, stream_handle(x),
                       _lib.lib().tssm_group_norm_workspace_bytes(N, S, G, Cg), code, act_,
                       x.data_ptr(), ptr(w), ptr(b), ptr(gate), y.data_ptr(), ptr(mean),
                       ptr(rstd), N, S, G, Cg, *sx, *sg, *sy, float(eps))
    return (y, mean, rstd) if return_stats else y


def group_norm_act_backward(dy, x, mean, rstd, groups, weight=None, bias=None, gate=None, *,
                            act="silu"):
    """Gradients of ``group_norm_act_forward`` for dy (shape and dtype of x),
    given its inputs and the statistics it returned.  Returns (dx, dw, db,
    dgate): dx and dgate of x's dtype, dw and db [C] float32; dw or db is None
    without weight or bias, dgate without a gate.
    """
    code, act_, N, S, G, Cg, sx, sg, w, b = _operands(x, groups, weight, bias, gate, act)
    sdy = _same(dy, "dy", x)
    for t, what, dtype in ((mean, "mean", torch.float64), (rstd, "rstd", torch.float32)):
        need_gpu(t, what)
        if t.shape != (N, G) or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous {dtype} [{N}, {G}]")
        if t.get_device() != x.get_device():
            raise ValueError(f"{what} must be on x's device")
    dx = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    dgate = torch.empty(x.shape, device=x.device, dtype=x.dtype) if gate is not None else None
    dw, db = torch.empty(2, G * Cg, device=x.device, dtype=torch.float32)
    sdx = _view(dx, "dx")[3:]
    workspace.call("tssm_group_norm_act_bwd", x, stream_handle(x),
                   _lib.lib().tssm_group_norm_workspace_bytes(N, S, G, Cg), code, act_,
                   dy.data_ptr(), x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), ptr(w), ptr(b),
                   ptr(gate), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ptr(dgate), N, S, G,
                   Cg, *sdy, *sx, *sg, *sdx, *sdx)
    return (dx, dw if weight is not None else None, db if bias is not None else None, dgate)
