"""Linear attention with a decay for each head: a state S [K, V] per value head
that sums outer products of keys and values and forgets at a rate of its own (no
reference counterpart).

    S_t = exp(g_t) S_{t-1} + k_t v_t^T
    o_t = scale S_t^T q_t

``linear_attention_forward``   whole sequences (prefill, training), any length
``linear_attention_backward``  every gradient of it
``linear_attention_step``      one step of many streams, the state in place (decode)

q and k have Hk heads, v and g Hv, a multiple of Hk: value head h reads key head
h // (Hv // Hk).  The state and every sum that reaches it are fp32.  With 16-bit
operands the weights between steps, and the state on its way to o and dv, count with 16
bits in products that fp32 sums add up: below the rounding of o, dq, dk and dv but where
their terms cancel by more than 2^8 (bfloat16) or 2^5 (float16).  ``g`` (log
decay, at most 0) is read as float32; one rate for each head is ``rate.expand(B,
L, Hv)``.  -inf at a step multiplies what came before by 0 and so drops it (several
sequences in one row, a stream that begins anew), as long as it is finite: 0 times a
NaN or infinity is NaN.  A state that holds one has to be zeroed instead, and a
sequence with one belongs in a row of its own.  ``qk_norm_rotary_forward`` prepares q
and k.
"""
from __future__ import annotations

import torch

from . import _lib, workspace
from .launch import DTYPES, as_f32, dcode, need_gpu, on_device, ptr, stream_handle

_F32 = torch.float32


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


def _operands(q, k, v, g, lead):
    """Checks q, k, v, g with ``lead`` leading dimensions; returns (sizes, dtype
    code, g).  Decoding calls pay for every check, so what is right passes in one
    expression, and _explain() names what is not."""
    try:
        dev, dtype, rows, heads, shape = q.get_device(), q.dtype, q.shape, v.shape, g.shape
        right = (dev >= 0 and len(rows) == lead + 2 and rows == k.shape and heads[:-1] == shape
                 and rows[:lead] == shape[:lead] and dtype == k.dtype == v.dtype
                 and dtype in DTYPES and g.dtype == _F32
                 and dev == k.get_device() == v.get_device() == g.get_device())
    except (AttributeError, TypeError, IndexError):
        right = False
    if not right:
        g = _explain(q, k, v, g, lead)
        dtype, rows, heads = q.dtype, q.shape, v.shape
    Hk, K = rows[lead:]
    Hv, V = heads[lead:]
    if not (Hk and Hv and V and 0 < K <= 128) or Hv % Hk:
        _sizes(Hk, Hv, K, V)
    return (*rows[:lead], Hk, Hv, K, V), DTYPES[dtype], g


def _sizes(Hk, Hv, K, V):
    if not (Hk and Hv and K and V) or Hv % Hk:
        raise ValueError(f"v's heads must be a multiple of q's, all sizes positive: Hk = {Hk}, "
                         f"Hv = {Hv}, K = {K}, V = {V}")
    if K > 128:
        raise ValueError(f"K = {K}: the key dimension may be at most 128")


def _explain(q, k, v, g, lead):
    """Raises what is wrong with the operands; returns g as float32 if it was its
    dtype alone."""
    for t, w in ((q, "q"), (k, "k"), (v, "v"), (g, "g")):
        need_gpu(t, w)
    if q.dim() != lead + 2 or v.dim() != lead + 2:
        names = "[B, L, Hk, K] and v [B, L, Hv, V]" if lead == 2 else "[S, Hk, K] and v [S, Hv, V]"
        raise ValueError(f"expected q, k {names}")
    rows, (Hk, K), (Hv, V), dev = q.shape[:lead], q.shape[lead:], v.shape[lead:], q.get_device()
    _sizes(Hk, Hv, K, V)
    dcode(q, "q")
    _check(k, "k", q.shape, q.dtype, dev)
    _check(v, "v", rows + (Hv, V), q.dtype, dev)
    if not g.is_floating_point():
        raise TypeError(f"g: expected a float tensor, got {g.dtype}")
    _check(g, "g", rows + (Hv,), g.dtype, dev)
    return g.to(_F32)


def _steps(t, chunks=False):
    """t [B, L, H, N], copied where its rows repeat one element (the gradient of a sum) or
    its steps overlap in memory (as expanded ones do): the chunked kernels take steps that
    lie one after the other.  With ``chunks`` (nothing but chunked kernels) also where a
    chunk of 128 steps and one more would pass 31 bits, heads first if one step is so long
    that it does not help to close the gaps."""
    _, step, _, element = t.stride()
    if element == 0 and t.shape[3] > 1 or t.shape[1] > 1 and step < t.shape[3]:
        t = t.contiguous()
    if chunks and t.shape[1] > 1:
        most = (1 << 31) // (129 * t.element_size())
        if t.stride(1) >= most:
            t = t.contiguous()
        if t.stride(1) >= most:
            t = t.transpose(1, 2).contiguous().transpose(1, 2)
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
    if any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError("out: elements must not share memory")
    return out


def linear_attention_forward(q, k, v, g, *, scale=None, h0=None, return_state=False, out=None):
    """Linear attention over whole sequences.

    q, k   [B, L, Hk, K]  float32 / bfloat16 / float16, K <= 128
    v      [B, L, Hv, V]  dtype of q, Hv a multiple of Hk
    g      [B, L, Hv]     log decay of each step (<= 0)
    scale  of q; None: K ** -0.5
    h0     [B, Hv, K, V] float32 or None (zero initial state)

    Returns o [B, L, Hv, V] (dtype of v; ``out`` if given, memory of its own) and, with
    ``return_state``, the final state [B, Hv, K, V] float32, which continues
    the sequence as the next call's ``h0`` or in ``linear_attention_step``.  An
    input that is not finite at some step changes no earlier output, and no
    other column of v.
    """
    (B, L, Hk, Hv, K, V), code, g = _operands(q, k, v, g, 2)
    dev = q.get_device()
    q, k, v = _steps(q), _steps(k), _steps(v)
    h0 = _state(h0, "h0", (B, Hv, K, V), dev)
    o = _out(out, v)
    h_last = None
    if return_state:
        h_last = torch.empty(B, Hv, K, V, device=v.device, dtype=_F32) if h0 is None else \
            torch.empty_like(h0)
    if B:
        nbytes = _lib.lib().tssm_linear_attention_workspace_bytes(B, L, Hk, Hv, K, V)
        on_device(dev, workspace.call, "tssm_linear_attention_forward", q, stream_handle(q),
                  nbytes, code, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), ptr(h0),
                  o.data_ptr(), ptr(h_last), B, L, Hk, Hv, K, V, *_rows(q, "q"), *_rows(k, "k"),
                  *_rows(v, "v"), *g.stride(), *_rows(o, "out"),
                  K ** -0.5 if scale is None else float(scale))
    return (o, h_last) if return_state else o


def linear_attention_backward(q, k, v, g, do, *, scale=None, h0=None, dh_last=None):
    """Gradients of ``linear_attention_forward`` for its inputs and do [B, L, Hv, V]
    (dtype of v), the gradient of o, and dh_last [B, Hv, K, V] float32 or None,
    that of the final state.

    Returns (dq, dk, dv, dg, dh0): dq, dk and dv of q's dtype, dg [B, L, Hv] and dh0
    float32 (dh0 is None without h0).  dq and dk are summed over the value heads
    that share a key head; repeated calls give identical bits.  The states are
    formed again from the inputs: nothing but the inputs needs to be kept between
    the passes.  An input or gradient that is not finite makes its chunk of 64 steps,
    and what depends on it, not finite.
    """
    (B, L, Hk, Hv, K, V), code, g = _operands(q, k, v, g, 2)
    dev = q.get_device()
    _check(do, "do", v.shape, v.dtype, dev)
    q, k, v, do = (_steps(t, chunks=True) for t in (q, k, v, do))
    h0, dh_last = _state(h0, "h0", (B, Hv, K, V), dev), \
        _state(dh_last, "dh_last", (B, Hv, K, V), dev)
    dq = torch.empty(B, L, Hk, K, device=q.device, dtype=q.dtype)
    dk, dv = torch.empty_like(dq), torch.empty(B, L, Hv, V, device=q.device, dtype=q.dtype)
    dg = torch.empty(B, L, Hv, device=q.device, dtype=_F32)
    dh0 = None if h0 is None else torch.empty(B, Hv, K, V, device=q.device, dtype=_F32)
    if B and L:
        nbytes = _lib.lib().tssm_linear_attention_backward_workspace_bytes(code, B, L, Hk, Hv, K,
                                                                          V)
        on_device(dev, workspace.call, "tssm_linear_attention_backward", q, stream_handle(q),
                  nbytes, code, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), ptr(h0),
                  do.data_ptr(), ptr(dh_last), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                  dg.data_ptr(), ptr(dh0), B, L, Hk, Hv, K, V, *_rows(q, "q"), *_rows(k, "k"),
                  *_rows(v, "v"), *g.stride(), *_rows(do, "do"),
                  K ** -0.5 if scale is None else float(scale))
    elif dh0 is not None:
        dh0.zero_() if dh_last is None else dh0.copy_(dh_last)
    return dq, dk, dv, dg, dh0


def linear_attention_step(q, k, v, g, state, *, scale=None, out=None):
    """One step of S streams, the state updated in place.

    q, k [S, Hk, K], v [S, Hv, V] of one dtype (float32 / bfloat16 / float16),
    g [S, Hv], state [S, Hv, K, V] float32 contiguous.  Returns o [S, Hv, V]
    (dtype of v; ``out`` if given, memory of its own).  The same step as
    ``linear_attention_forward`` with L = 1.
    """
    (S, Hk, Hv, K, V), code, g = _operands(q, k, v, g, 1)
    dev = q.get_device()
    _check(state, "state", (S, Hv, K, V), _F32, dev)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous")
    o = _out(out, v)
    if S:
        on_device(dev, _lib.call, "tssm_linear_attention_step", code, q.data_ptr(), k.data_ptr(),
                  v.data_ptr(), g.data_ptr(), state.data_ptr(), o.data_ptr(), S, Hk, Hv, K, V,
                  *_rows(q, "q"), *_rows(k, "k"), *_rows(v, "v"), *g.stride(), *_rows(o, "out"),
                  K ** -0.5 if scale is None else float(scale), stream_handle(q))
    return o
