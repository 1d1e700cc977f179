"""What stands next to the attention of a transformer block, on CUDA torch tensors: rotary positions of queries and
keys, alone or behind an RMS norm of every head, with their gradients.

The functions are thin: they check their arguments (``ValueError`` / ``TypeError``), allocate outputs with torch, and
make one call of the C ABI (``include/asc_cuda.h``) on torch's current stream of the tensors' device.  They return
without waiting for the GPU and record no autograd history; every operator's gradient is a function of its own.  A
status other than 0 raises ``RuntimeError`` (:func:`pyasc_b200.capi.call`).

Tensors are [batch, sequence, heads, head_dim] with any strides, as long as the last dimension is contiguous: slices of
a packed projection, or ``x.transpose(1, 2)`` of a [batch, heads, sequence, head_dim] tensor.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
from typing import Optional, Sequence, Tuple

import torch

from . import capi

_DTYPE_CODE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


# --------------------------------------------------------------------------------------------------
# Arguments
# --------------------------------------------------------------------------------------------------
def _check_tensor(name: str, t: torch.Tensor, dtypes: Sequence[torch.dtype], device: Optional[torch.device],
                  shape: Optional[Sequence[int]] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _check_rows(name: str, t: torch.Tensor) -> None:
    if t.dim() != 4:
        raise ValueError(f"{name} must be [batch, sequence, heads, head_dim], got {t.dim()} dimensions")
    if t.shape[3] > 1 and t.stride(3) != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")


def _check_output(name: str, t: torch.Tensor, like: torch.Tensor, shape: Sequence[int]) -> None:
    _check_tensor(name, t, (like.dtype, ), like.device, shape)
    _check_rows(name, t)
    if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{name} repeats memory (a stride of 0): it cannot be written")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _int64s(*values: int):
    return (ctypes.c_int64 * len(values))(*values)


def _call(fn_name: str, device: torch.device, *args) -> None:
    """One C-ABI call with ``device`` current, on its current torch stream."""
    index = device.index
    with contextlib.nullcontext() if index == torch.cuda.current_device() else torch.cuda.device(index):
        capi.call(fn_name, *args, torch.cuda.current_stream(index).cuda_stream)


# --------------------------------------------------------------------------------------------------
# Rotary positions
# --------------------------------------------------------------------------------------------------
def rotary_frequencies(rotated: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original_context: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """Angles per position of the ``rotated / 2`` pairs of a head (float64), and the factor of their cosines and sines.

    ``scaling`` stretches the context by ``factor``: ``"linear"`` divides every frequency; ``"ntk"`` raises the base, so
    that fast pairs keep their frequency and the slowest is divided by ``factor``; ``"yarn"`` (Peng et al., 2023) divides
    the pairs that turn less than ``beta_slow`` times within ``original_context``, keeps those that turn more than
    ``beta_fast`` times, blends in between, and scales cosines and sines by ``0.1 ln(factor) + 1``.
    """
    if rotated < 0 or rotated % 2:
        raise ValueError(f"the rotated part of a head must be even, got {rotated}")
    if base <= 1.0 or factor < 1.0:
        raise ValueError("rotary positions need a base above 1 and a factor of at least 1")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if scaling == "ntk" and rotated > 2:
        base = base * factor**(rotated / (rotated - 2))
    i = torch.arange(rotated // 2, dtype=torch.float64)
    frequencies = base**(-2.0 * i / max(rotated, 1))
    scale = 1.0
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "yarn":
        if original_context <= 0:
            raise ValueError("yarn scaling needs the original context length")

        def pair_that_turns(times: float) -> float:
            return rotated * math.log(original_context / (2 * math.pi * times)) / (2 * math.log(base))

        low = max(math.floor(pair_that_turns(beta_fast)), 0)
        high = min(math.ceil(pair_that_turns(beta_slow)), rotated - 1)
        slow = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        frequencies = frequencies * (slow / factor + (1 - slow))
        scale = 0.1 * math.log(factor) + 1.0
    return frequencies.to(device), scale


def _rotary_arguments(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor):
    """Checks what all four functions share; dims, strides of the positions and the flag of their type."""
    _check_tensor("q", q, tuple(_DTYPE_CODE), None)
    _check_rows("q", q)
    batch, seq, heads, head_dim = q.shape
    kv_heads = 0
    if k is not None:
        _check_tensor("k", k, (q.dtype, ), q.device)
        _check_rows("k", k)
        kv_heads = k.shape[2]
        if k.shape != (batch, seq, kv_heads, head_dim):
            raise ValueError(f"k has shape {tuple(k.shape)}, q {tuple(q.shape)}: only the heads may differ")
    _check_tensor("positions", positions, (torch.int64, torch.int32), q.device)
    if positions.dim() not in (1, 2) or positions.shape[-1] != seq or (positions.dim() == 2 and
                                                                       positions.shape[0] not in (1, batch)):
        raise ValueError(f"positions must be [sequence] or [batch, sequence], got {tuple(positions.shape)}")
    _check_tensor("frequencies", frequencies, (torch.float64, ), q.device)
    if frequencies.dim() != 1 or (frequencies.numel() > 1 and frequencies.stride(0) != 1):
        raise ValueError("frequencies must be one contiguous row")
    rotated = 2 * frequencies.numel()
    if rotated > head_dim:
        raise ValueError(f"{frequencies.numel()} frequencies turn {rotated} elements of a head of {head_dim}")
    batch_stride = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    flags = 4 if positions.dtype == torch.int32 else 0
    return (batch, seq, heads, kv_heads, head_dim, rotated), (batch_stride, positions.stride(-1)), flags


def _strides(t: Optional[torch.Tensor]) -> Tuple[int, int, int]:
    return (0, 0, 0) if t is None else t.stride()[:3]


def _gammas(q: torch.Tensor, k: Optional[torch.Tensor], q_gamma: Optional[torch.Tensor],
            k_gamma: Optional[torch.Tensor]) -> int:
    code = None
    for name, g in (("q_gamma", q_gamma), ("k_gamma", k_gamma)):
        if g is None:
            continue
        _check_tensor(name, g, tuple(_DTYPE_CODE), q.device, (q.shape[3], ))
        if g.numel() > 1 and g.stride(0) != 1:
            raise ValueError(f"{name} must be contiguous")
        if code is not None and code != _DTYPE_CODE[g.dtype]:
            raise TypeError("q_gamma and k_gamma must have one type")
        code = _DTYPE_CODE[g.dtype]
    return code or 0


def _rotate(q, k, q_gamma, k_gamma, positions, frequencies, eps, scale, interleaved, flags, q_out, k_out):
    dims, pos_strides, pos_flag = _rotary_arguments(q, k, positions, frequencies)
    gamma_code = _gammas(q, k, q_gamma, k_gamma)
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check_output("q_out", q_out, q, q.shape)
    if k is None:
        if k_out is not None:
            raise ValueError("k_out without k")
    elif k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    else:
        _check_output("k_out", k_out, k, k.shape)
    _call("asc_cuda_norm_rotary", q.device, _ptr(q), _ptr(k), _ptr(q_out), _ptr(k_out), _ptr(q_gamma), _ptr(k_gamma),
          _ptr(positions), _ptr(frequencies), _int64s(*dims),
          _int64s(*_strides(q), *_strides(k), *_strides(q_out), *_strides(k_out), *pos_strides), eps, scale,
          _DTYPE_CODE[q.dtype], gamma_code, flags | pos_flag | bool(interleaved))
    return q_out, k_out


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, *,
           scale: float = 1.0, interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
           k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Queries [B, S, Hq, D] and keys [B, S, Hk, D] (``k`` may be None) turned by ``positions`` ([S] or [B, S], int64 or
    int32) times ``frequencies`` (float64, half as many as elements are turned; the rest of a head passes).  Pairs are
    (i, i + r / 2), or (2 i, 2 i + 1) with ``interleaved``.  ``scale`` multiplies cosines and sines (see
    :func:`rotary_frequencies`).  float16, bfloat16 or float32.  ``q_out=q, k_out=k`` turns in place."""
    return _rotate(q, k, None, None, positions, frequencies, 0.0, scale, interleaved, 0, q_out, k_out)


def rotary_backward(dq_out: torch.Tensor, dk_out: Optional[torch.Tensor], positions: torch.Tensor,
                    frequencies: torch.Tensor, *, scale: float = 1.0, interleaved: bool = False,
                    dq: Optional[torch.Tensor] = None,
                    dk: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of :func:`rotary`'s q and k from those of its outputs: the rotation turned back."""
    return _rotate(dq_out, dk_out, None, None, positions, frequencies, 0.0, scale, interleaved, 8, dq, dk)


def norm_rotary(q: torch.Tensor, k: Optional[torch.Tensor], q_gamma: Optional[torch.Tensor],
                k_gamma: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, *, eps: float = 1e-6,
                scale: float = 1.0, interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """:func:`rotary` of ``x / sqrt(mean(x^2) + eps) * gamma`` of every head, in the same pass.  The gammas hold
    head_dim values of one type (float16, bfloat16 or float32; None: ones)."""
    return _rotate(q, k, q_gamma, k_gamma, positions, frequencies, eps, scale, interleaved, 2, q_out, k_out)


def norm_rotary_backward(dq_out: torch.Tensor, dk_out: Optional[torch.Tensor], q: torch.Tensor, k: Optional[torch.Tensor],
                         q_gamma: Optional[torch.Tensor], k_gamma: Optional[torch.Tensor], positions: torch.Tensor,
                         frequencies: torch.Tensor, *, eps: float = 1e-6, scale: float = 1.0, interleaved: bool = False,
                         dq: Optional[torch.Tensor] = None, dk: Optional[torch.Tensor] = None):
    """Gradients ``(dq, dk, dq_gamma, dk_gamma)`` of :func:`norm_rotary` from those of its outputs and its inputs.  The
    gammas' gradients are float32 sums over all rows in a fixed order (None where there is no gamma).  ``dq`` may be
    ``dq_out`` or ``q``, ``dk`` likewise."""
    dims, pos_strides, pos_flag = _rotary_arguments(q, k, positions, frequencies)
    gamma_code = _gammas(q, k, q_gamma, k_gamma)
    _check_tensor("dq_out", dq_out, (q.dtype, ), q.device, q.shape)
    _check_rows("dq_out", dq_out)
    if (k is None) != (dk_out is None):
        raise ValueError("k and dk_out go together")
    if dq is None:
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check_output("dq", dq, q, q.shape)
    if k is None:
        if dk is not None or k_gamma is not None:
            raise ValueError("dk or k_gamma without k")
    else:
        _check_tensor("dk_out", dk_out, (k.dtype, ), k.device, k.shape)
        _check_rows("dk_out", dk_out)
        if dk is None:
            dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        else:
            _check_output("dk", dk, k, k.shape)
    dq_gamma, dk_gamma = (None if g is None else torch.empty(q.shape[3], dtype=torch.float32, device=q.device)
                          for g in (q_gamma, k_gamma))
    _call("asc_cuda_norm_rotary_bwd", q.device, _ptr(dq_out), _ptr(dk_out), _ptr(q), _ptr(k), _ptr(dq), _ptr(dk),
          _ptr(q_gamma), _ptr(k_gamma), _ptr(dq_gamma), _ptr(dk_gamma), _ptr(positions), _ptr(frequencies),
          _int64s(*dims),
          _int64s(*_strides(dq_out), *_strides(dk_out), *_strides(q), *_strides(k), *_strides(dq), *_strides(dk),
                  *pos_strides), eps, scale, _DTYPE_CODE[q.dtype], gamma_code, 2 | pos_flag | bool(interleaved))
    return dq, dk, dq_gamma, dk_gamma
