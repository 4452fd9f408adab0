"""Gated delta rule: a state S [K, V] per value head whose every step corrects
what the state already holds for its key (no reference counterpart).

    u_t = beta_t (v_t - exp(g_t) S_{t-1}^T k_t)
    S_t = exp(g_t) S_{t-1} + k_t u_t^T
    o_t = scale S_t^T q_t

``gated_delta_forward``   whole sequences (prefill, training), any length
``gated_delta_backward``  every gradient of it
``gated_delta_step``      one step of many streams, the state in place (decode)

q and k have Hk heads, v, g and beta Hv, a multiple of Hk: value head h reads
key head h // (Hv // Hk).  The state and every sum that reaches it are fp32;
keys of unit length and beta in [0, 1] keep the recurrence contracting, which
is the caller's business: nothing is normalised here.  ``g`` (log decay) and
``beta`` are read as float32.
"""
from __future__ import annotations

import torch

from . import _lib, workspace
from .launch import DTYPES, as_f32, dcode, need_gpu, ptr, stream_handle


def _check(t, what, shape, dtype, device):
    need_gpu(t, what)
    if t.shape != shape:
        raise ValueError(f"{what} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{what} must be on device {device}")


def _rows(t, what):
    """Strides of every dimension but the innermost, which must be contiguous."""
    s = t.stride()
    if s[-1] != 1 and t.shape[-1] != 1:
        raise ValueError(f"{what}: innermost dimension must be contiguous")
    return s[:-1]


_F32 = torch.float32


def _operands(q, k, v, g, beta, lead):
    """Checks q, k, v, g, beta with ``lead`` leading dimensions; returns (sizes,
    dtype code, g, beta).  Decoding calls pay for every check, so what is right
    passes in one expression, and _explain() names what is not."""
    try:
        dev, dtype, rows, heads, shape = q.get_device(), q.dtype, q.shape, v.shape, g.shape
        right = (dev >= 0 and len(rows) == lead + 2 and rows == k.shape and shape == beta.shape
                 and heads[:-1] == shape and rows[:lead] == shape[:lead]
                 and dtype == k.dtype == v.dtype and dtype in DTYPES
                 and g.dtype == beta.dtype == _F32
                 and dev == k.get_device() == v.get_device() == g.get_device()
                 == beta.get_device())
    except (AttributeError, TypeError, IndexError):
        right = False
    if not right:
        g, beta = _explain(q, k, v, g, beta, lead)
        dtype, rows, heads = q.dtype, q.shape, v.shape
    Hk, K = rows[lead:]
    Hv, V = heads[lead:]
    if not (Hk and Hv and V and 0 < K <= 128) or Hv % Hk:
        _sizes(Hk, Hv, K, V)
    return (*rows[:lead], Hk, Hv, K, V), DTYPES[dtype], g, beta


def _sizes(Hk, Hv, K, V):
    if not (Hk and Hv and K and V) or Hv % Hk:
        raise ValueError(f"v's heads must be a multiple of q's, all sizes positive: Hk = {Hk}, "
                         f"Hv = {Hv}, K = {K}, V = {V}")
    if K > 128:
        raise ValueError(f"K = {K}: the key dimension may be at most 128")


def _explain(q, k, v, g, beta, lead):
    """Raises what is wrong with the operands; returns g and beta as float32 if
    it was their dtype alone."""
    for t, w in ((q, "q"), (k, "k"), (v, "v"), (g, "g"), (beta, "beta")):
        need_gpu(t, w)
    if q.dim() != lead + 2 or v.dim() != lead + 2:
        names = "[B, L, Hk, K] and v [B, L, Hv, V]" if lead == 2 else "[S, Hk, K] and v [S, Hv, V]"
        raise ValueError(f"expected q, k {names}")
    rows, (Hk, K), (Hv, V), dev = q.shape[:lead], q.shape[lead:], v.shape[lead:], q.get_device()
    _sizes(Hk, Hv, K, V)
    dcode(q, "q")
    _check(k, "k", q.shape, q.dtype, dev)
    _check(v, "v", rows + (Hv, V), q.dtype, dev)
    g, beta = as_f32(g, "g"), as_f32(beta, "beta")
    _check(g, "g", rows + (Hv,), _F32, dev)
    _check(beta, "beta", rows + (Hv,), _F32, dev)
    return g, beta


def _steps(t, chunks=False):
    """t [B, L, H, N], copied where its rows repeat one element (the gradient of a
    sum) or its steps overlap in memory (as expanded ones do): the chunked kernels
    take steps that lie one after the other.  With ``chunks`` (nothing but chunked
    kernels) also where a chunk of 32 steps and one more would pass 31 bits."""
    _, step, _, element = t.stride()
    if element == 0 and t.shape[3] > 1 or t.shape[1] > 1 and (
            step < t.shape[3] or chunks and step >= (1 << 31) // (33 * t.element_size())):
        return t.contiguous()
    return t


def _state(t, what, shape, device):
    if t is None:
        return None
    need_gpu(t, what)
    if t.dtype != _F32 or not t.is_contiguous():
        t = as_f32(t, what).contiguous()
    _check(t, what, shape, _F32, device)
    return t


def _out(out, v):
    """``out`` checked, or a new one like v."""
    if out is None:
        return torch.empty_like(v, memory_format=torch.contiguous_format)
    _check(out, "out", v.shape, v.dtype, v.get_device())
    return out


def gated_delta_forward(q, k, v, g, beta, *, scale=None, h0=None, return_state=False, out=None):
    """Gated delta rule over whole sequences.

    q, k   [B, L, Hk, K]  float32 / bfloat16 / float16, K <= 128
    v      [B, L, Hv, V]  dtype of q, Hv a multiple of Hk
    g      [B, L, Hv]     log decay of each step (<= 0)
    beta   [B, L, Hv]     step size
    scale  of q; None: K ** -0.5
    h0     [B, Hv, K, V] float32 or None (zero initial state)

    Returns o [B, L, Hv, V] (dtype of v; ``out`` if given) and, with
    ``return_state``, the final state [B, Hv, K, V] float32, which continues
    the sequence as the next call's ``h0`` or in ``gated_delta_step``.  An
    input that is not finite at some step changes no earlier output, and no
    other column of v.
    """
    (B, L, Hk, Hv, K, V), code, g, beta = _operands(q, k, v, g, beta, 2)
    q, k, v = _steps(q), _steps(k), _steps(v)
    h0 = _state(h0, "h0", (B, Hv, K, V), q.get_device())
    o = _out(out, v)
    h_last = None
    if return_state:
        h_last = torch.empty(B, Hv, K, V, device=v.device, dtype=_F32) if h0 is None else \
            torch.empty_like(h0)
    if B:
        nbytes = _lib.lib().tssm_gated_delta_workspace_bytes(B, L, Hk, Hv, K, V)
        workspace.call("tssm_gated_delta_forward", q, stream_handle(q), nbytes, code,
                       q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
                       ptr(h0), o.data_ptr(), ptr(h_last), B, L, Hk, Hv, K, V, *_rows(q, "q"),
                       *_rows(k, "k"), *_rows(v, "v"), *g.stride(), *beta.stride(),
                       *_rows(o, "out"), K ** -0.5 if scale is None else float(scale))
    return (o, h_last) if return_state else o


def gated_delta_backward(q, k, v, g, beta, do, *, scale=None, h0=None, dh_last=None):
    """Gradients of ``gated_delta_forward`` for its inputs and do [B, L, Hv, V]
    (dtype of v), the gradient of o, and dh_last [B, Hv, K, V] float32 or None,
    that of the final state.

    Returns (dq, dk, dv, dg, dbeta, dh0): dq, dk and dv of q's dtype, dg, dbeta
    and dh0 float32 (dh0 is None without h0).  dq and dk are summed over the
    value heads that share a key head; repeated calls give identical bits.  The
    states are formed again from the inputs: nothing but the inputs needs to be
    kept between the passes.  An input or gradient that is not finite makes its
    chunk of 32 steps, and what depends on it, not finite.
    """
    (B, L, Hk, Hv, K, V), code, g, beta = _operands(q, k, v, g, beta, 2)
    dev = q.get_device()
    _check(do, "do", v.shape, v.dtype, dev)
    q, k, v, do = (_steps(t, chunks=True) for t in (q, k, v, do))
    h0, dh_last = _state(h0, "h0", (B, Hv, K, V), dev), \
        _state(dh_last, "dh_last", (B, Hv, K, V), dev)
    dq = torch.empty(B, L, Hk, K, device=q.device, dtype=q.dtype)
    dk, dv = torch.empty_like(dq), torch.empty(B, L, Hv, V, device=q.device, dtype=q.dtype)
    dg, dbeta = torch.empty(2, B, L, Hv, device=q.device, dtype=torch.float32)
    dh0 = None if h0 is None else torch.empty(B, Hv, K, V, device=q.device, dtype=torch.float32)
    if B and L:
        nbytes = _lib.lib().tssm_gated_delta_backward_workspace_bytes(B, L, Hk, Hv, K, V)
        workspace.call("tssm_gated_delta_backward", q, stream_handle(q), nbytes, code,
                       q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
                       ptr(h0), do.data_ptr(), ptr(dh_last), dq.data_ptr(), dk.data_ptr(),
                       dv.data_ptr(), dg.data_ptr(), dbeta.data_ptr(), ptr(dh0), B, L, Hk, Hv, K,
                       V, *_rows(q, "q"), *_rows(k, "k"), *_rows(v, "v"), *g.stride(),
                       *beta.stride(), *_rows(do, "do"),
                       K ** -0.5 if scale is None else float(scale))
    elif dh0 is not None:
        dh0.zero_() if dh_last is None else dh0.copy_(dh_last)
    return dq, dk, dv, dg, dbeta, dh0


def gated_delta_step(q, k, v, g, beta, state, *, scale=None, out=None):
    """One step of S streams, the state updated in place.

    q, k [S, Hk, K], v [S, Hv, V] of one dtype (float32 / bfloat16 / float16),
    g, beta [S, Hv], state [S, Hv, K, V] float32 contiguous.  Returns o
    [S, Hv, V] (dtype of v; ``out`` if given).  The same step as
    ``gated_delta_forward`` with L = 1.
    """
    (S, Hk, Hv, K, V), code, g, beta = _operands(q, k, v, g, beta, 1)
    _check(state, "state", (S, Hv, K, V), torch.float32, q.get_device())
    if not state.is_contiguous():
        raise ValueError("state must be contiguous")
    o = _out(out, v)
    if S:
        _lib.call("tssm_gated_delta_step", code, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  g.data_ptr(), beta.data_ptr(), state.data_ptr(), o.data_ptr(), S, Hk, Hv, K, V,
                  *_rows(q, "q"), *_rows(k, "k"), *_rows(v, "v"), *g.stride(), *beta.stride(),
                  *_rows(o, "out"), K ** -0.5 if scale is None else float(scale),
                  stream_handle(q))
    return o
