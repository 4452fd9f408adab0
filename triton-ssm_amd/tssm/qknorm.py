"""Norm of queries and keys for each head and rotation by their positions, in one
pass, and its gradients (no reference counterpart).

    n = r x w          r = (mean x^2 + eps)^-1/2 ("rms"), (sum x^2 + eps)^-1/2 ("l2")
                       or 1 ("none"), over a head's K channels
    (n_a, n_b) -> amplitude (n_a cos - n_b sin, n_a sin + n_b cos)

for the R/2 pairs of the first R channels, (j, j + R/2) or, interleaved, (2 j, 2 j +
1), by the angle position * freqs[j]; the other channels stay n.  Positions are
token numbers or the times of irregular samples; angles are formed in 64 bits.
``rotary_frequencies`` gives the rates, scaled for long contexts if asked to.
What comes out is what ``linear_attention_*`` and ``gated_delta_*`` read as q and k, if
both have the same number of heads: those share key heads among value heads, not among
queries.
"""
from __future__ import annotations

import math

import torch

from . import _lib, workspace
from .launch import DTYPES, as_f32, dcode, need_gpu, on_device, ptr, stream_handle

_NORM = {"none": 0, "rms": 1, "l2": 2}
_POS = {torch.float32: 0, torch.float64: 1, torch.int32: 2, torch.int64: 3}


def rotary_frequencies(dim, base=10000.0, *, factor=1.0, how="positions", trained=None,
                       fast=32.0, slow=1.0, device=None):
    """Angular rates [dim / 2] float64 of the rotated channels: base^(-2 j / dim).

    ``factor`` > 1 stretches them for contexts ``factor`` times as long as those
    the rates were trained on:

    how="positions"  every rate is divided by it (positions come closer together)
    how="base"       the base grows so that the slowest rate is divided by it and
                     the fastest stays
    how="parts"      rates that turn more than ``fast`` times within ``trained``
                     positions stay, those that turn less than ``slow`` times are
                     divided, those between are mixed linearly; ``amplitude`` of
                     0.1 log(factor) + 1 goes with it (``rotary_amplitude``)
    """
    dim = int(dim)
    if dim <= 0 or dim % 2:
        raise ValueError(f"dim = {dim}: a positive even number of rotated channels")
    if not base > 0 or not factor >= 1:
        raise ValueError(f"base must be positive and factor at least 1, got {base} and {factor}")
    j = torch.arange(dim // 2, dtype=torch.float64)
    if how == "base":
        if dim == 2:
            raise ValueError("how='base' needs more than one rate")
        base = base * factor ** (dim / (dim - 2))
    freqs = base ** (-2.0 * j / dim)
    if how == "positions":
        freqs = freqs / factor
    elif how == "parts":
        if trained is None or not fast > slow > 0:
            raise ValueError("how='parts' needs trained (positions) and fast > slow > 0")
        turns = freqs * (trained / (2 * math.pi))
        stay = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        freqs = freqs * (stay + (1.0 - stay) / factor)
    elif how != "base":
        raise ValueError(f"how must be 'positions', 'base' or 'parts', got {how!r}")
    return freqs.to(device) if device is not None else freqs


def rotary_amplitude(factor):
    """The ``amplitude`` that goes with ``rotary_frequencies(how="parts")``."""
    return 0.1 * math.log(factor) + 1.0


def _rows(t, what):
    """Strides (b, l, h) of t [B, L, H, K] or [S, H, K]."""
    s = t.stride()
    if s[-1] != 1 and t.shape[-1] != 1:
        raise ValueError(f"{what}: innermost dimension must be contiguous")
    return s[:-1] if len(s) == 4 else (s[0], 0, s[1])


def _like(t, what, x):
    need_gpu(t, what)
    if t.shape != x.shape:
        raise ValueError(f"{what} must be {list(x.shape)}, got {list(t.shape)}")
    if t.dtype != x.dtype:
        raise TypeError(f"{what} must be {x.dtype}, got {t.dtype}")
    if t.get_device() != x.get_device():
        raise ValueError(f"{what} must be on device {x.get_device()}")
    return _rows(t, what)


def _gradient(t, what, x):
    """t checked, and its strides; copied where its rows repeat one element (the gradient
    of a sum)."""
    need_gpu(t, what)
    if t.dim() and t.stride(-1) == 0 and t.shape[-1] > 1:
        t = t.contiguous()
    return t, _like(t, what, x)


def _out(t, what, x):
    if t is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    _like(t, what, x)
    if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        raise ValueError(f"{what}: elements must not share memory")
    return t


def _apart(q, k, yq, yk):
    """Refuses an output that starts where the other input or output does, or where its own
    input does with other strides: rows would be written before they are read."""
    at, back = (q.data_ptr(), k.data_ptr()), (yq.data_ptr(), yk.data_ptr())
    other = [a == b and any(n > 1 and s != z for n, s, z in zip(x.shape, x.stride(), y.stride()))
             for a, b, x, y in zip(at, back, (q, k), (yq, yk))]
    if at[0] == back[1] or at[1] == back[0] or back[0] == back[1] or any(other):
        raise ValueError("out_q may be q and out_k may be k; outputs must not overlap otherwise")


def _weight(t, what, K, device):
    if t is None:
        return None
    need_gpu(t, what)
    if t.shape != (K,):
        raise ValueError(f"{what} must be [{K}], got {list(t.shape)}")
    if t.get_device() != device:
        raise ValueError(f"{what} must be on device {device}")
    return t if t.dtype == torch.float32 and t.is_contiguous() else as_f32(t, what).contiguous()


def _operands(q, k, positions, freqs, weight_q, weight_k, norm):
    """Checks; returns (dtype code, norm code, sizes, positions' pointer, type and
    strides, freqs, weights).  Decoding calls pay for every check, so what is right
    passes in one expression, and _explain() names what is not."""
    R, pos = 0, (None, 0, 0, 0)
    try:
        dev, dtype, sq, sk = q.get_device(), q.dtype, q.shape, k.shape
        lead, K = sq[:-2], sq[-1]
        right = (dev >= 0 and 3 <= len(sq) <= 4 and sk[:-2] == lead and sk[-1] == K
                 and dtype == k.dtype and dtype in DTYPES and k.get_device() == dev
                 and sq[-2] and sk[-2] and (1 < K <= 256 or K == 1 and norm == "none")
                 and norm in _NORM)
        if right and freqs is not None:
            R = 2 * freqs.shape[0]
            right = (freqs.dim() == 1 and freqs.dtype == torch.float64 and R <= K
                     and freqs.is_contiguous() and positions.shape == lead
                     and positions.dtype in _POS and freqs.get_device() == dev
                     and positions.get_device() == dev)
        elif positions is not None:
            right = False
        for w in (weight_q, weight_k):
            if w is not None and not (w.shape == (K,) and w.dtype == torch.float32
                                      and w.get_device() == dev and w.is_contiguous()):
                right = False
    except (AttributeError, TypeError, IndexError):
        right = False
    if not right:
        R, positions, freqs, weight_q, weight_k = _explain(q, k, positions, freqs, weight_q,
                                                           weight_k, norm)
        dtype, sq, sk, lead, K = q.dtype, q.shape, k.shape, q.shape[:-2], q.shape[-1]
    if R:
        st = positions.stride()
        st = st if len(st) == 2 else ((0, st[0]) if len(lead) == 2 else (st[0], 0))
        pos = (positions.data_ptr(), _POS[positions.dtype], *st)
    return (DTYPES[dtype], _NORM[norm], (lead[0], lead[1] if len(lead) == 2 else 1, sq[-2],
                                         sk[-2], K, R), pos, freqs, weight_q, weight_k)


def _explain(q, k, positions, freqs, weight_q, weight_k, norm):
    """Raises what is wrong with the operands; returns R and the operands that
    kernels read, converted where that is all."""
    need_gpu(q, "q")
    need_gpu(k, "k")
    if q.dim() not in (3, 4) or k.dim() != q.dim():
        raise ValueError("expected q [B, L, Hq, K] and k [B, L, Hk, K], or [S, H, K]")
    lead, K, dev = q.shape[:-2], q.shape[-1], q.get_device()
    if k.shape[:-2] != lead or k.shape[-1] != K:
        raise ValueError(f"k must be [{', '.join(map(str, lead))}, Hk, {K}], got {list(k.shape)}")
    if k.get_device() != dev:
        raise ValueError(f"k must be on device {dev}")
    dcode(q, "q")
    if k.dtype != q.dtype:
        raise TypeError(f"k must be {q.dtype}, got {k.dtype}")
    if norm not in _NORM:
        raise ValueError(f"norm must be 'rms', 'l2' or 'none', got {norm!r}")
    Hq, Hk = q.shape[-2], k.shape[-2]
    if not (Hq and Hk and K):
        raise ValueError(f"sizes must be positive: Hq = {Hq}, Hk = {Hk}, K = {K}")
    if K > 256:
        raise ValueError(f"K = {K}: a head may have at most 256 channels")
    if K == 1 and norm != "none":
        raise ValueError("K = 1: the norm of one channel is its sign")
    if (positions is None) != (freqs is None):
        raise ValueError("positions and freqs go together")
    R = 0
    if freqs is not None:
        need_gpu(freqs, "freqs")
        need_gpu(positions, "positions")
        if freqs.dim() != 1 or not freqs.is_floating_point():
            raise ValueError("freqs must be a float tensor [R / 2]")
        R = 2 * freqs.shape[0]
        if R > K:
            raise ValueError(f"{freqs.shape[0]} freqs rotate {R} channels of {K}")
        if positions.dtype not in _POS:
            raise TypeError(f"positions: unsupported dtype {positions.dtype}")
        if positions.shape != lead and not (len(lead) == 2 and positions.shape == lead[1:]):
            raise ValueError(f"positions must be {list(lead)}"
                             + (f" or {list(lead[1:])}" if len(lead) == 2 else "")
                             + f", got {list(positions.shape)}")
        for t, what in ((freqs, "freqs"), (positions, "positions")):
            if t.get_device() != dev:
                raise ValueError(f"{what} must be on device {dev}")
        freqs = freqs.to(torch.float64).contiguous()
    return (R, positions, freqs, _weight(weight_q, "weight_q", K, dev),
            _weight(weight_k, "weight_k", K, dev))


def qk_norm_rotary_forward(q, k, positions=None, freqs=None, weight_q=None, weight_k=None, *,
                           norm="rms", eps=1e-6, interleaved=False, amplitude=1.0, out_q=None,
                           out_k=None):
    """Norm and rotation of every head's row of q [B, L, Hq, K] and k [B, L, Hk, K]
    (or [S, H, K], one token of S streams), of one dtype (float32 / bfloat16 /
    float16), K <= 256 (and K > 1 with a norm).

    positions  [B, L], [L] or [S]: int32, int64, float32 or float64
    freqs      [R / 2] angular rates (float64; others are converted), R <= K;
               None, with positions: no rotation
    weight_q, weight_k  [K] (read as float32) or None

    Returns (q', k') of q's dtype, new or in ``out_q``, which may be q, and ``out_k``, which
    may be k; neither overlaps anything else.
    """
    code, norm_, sizes, pos, freqs, wq, wk = _operands(q, k, positions, freqs, weight_q,
                                                       weight_k, norm)
    yq, yk = _out(out_q, "out_q", q), _out(out_k, "out_k", k)
    if q.numel():
        if out_q is not None or out_k is not None:
            _apart(q, k, yq, yk)
        on_device(q.get_device(), _lib.call, "tssm_qk_norm_rotary_fwd", code, norm_,
                  int(bool(interleaved)), q.data_ptr(), k.data_ptr(), pos[0], pos[1], ptr(freqs),
                  ptr(wq), ptr(wk), yq.data_ptr(), yk.data_ptr(), *sizes, *_rows(q, "q"),
                  *_rows(k, "k"), *pos[2:], *_rows(yq, "out_q"), *_rows(yk, "out_k"), float(eps),
                  float(amplitude), stream_handle(q))
    return yq, yk


def qk_norm_rotary_backward(dq_out, dk_out, q, k, positions=None, freqs=None, weight_q=None,
                            weight_k=None, *, norm="rms", eps=1e-6, interleaved=False,
                            amplitude=1.0):
    """Gradients of ``qk_norm_rotary_forward`` for its inputs and the gradients
    dq_out and dk_out (shapes and dtype of q and k) of its outputs.

    Returns (dq, dk, dweight_q, dweight_k): dq and dk contiguous, of q's dtype, the
    weights' [K] float32 (None without that weight), summed in a fixed order.
    """
    code, norm_, sizes, pos, freqs, wq, wk = _operands(q, k, positions, freqs, weight_q,
                                                       weight_k, norm)
    dq_out, sdq = _gradient(dq_out, "dq_out", q)
    dk_out, sdk = _gradient(dk_out, "dk_out", k)
    dq, dk = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k))
    dwq, dwk = (None if w is None else torch.empty(sizes[4], device=q.device, dtype=torch.float32)
                for w in (wq, wk))
    weights = dwq is not None or dwk is not None
    if q.numel() or weights:
        nbytes = _lib.lib().tssm_qk_norm_rotary_workspace_bytes(sizes[4]) if weights else 0
        on_device(q.get_device(), workspace.call, "tssm_qk_norm_rotary_bwd", q, stream_handle(q),
                  nbytes, code, norm_, int(bool(interleaved)), dq_out.data_ptr(),
                  dk_out.data_ptr(), q.data_ptr(), k.data_ptr(), pos[0], pos[1], ptr(freqs),
                  ptr(wq), ptr(wk), dq.data_ptr(), dk.data_ptr(), ptr(dwq), ptr(dwk), *sizes,
                  *sdq, *sdk, *_rows(q, "q"), *_rows(k, "k"), *pos[2:], *_rows(dq, "dq"),
                  *_rows(dk, "dk"), float(eps), float(amplitude))
    return dq, dk, dwq, dwk
