"""What stands next to the self-attention of a transformer block, on CUDA torch tensors: rotary positions of queries and
keys, alone or behind an RMS norm of every head, and attention to the states of another sequence, with their gradients.

The functions are thin: they check their arguments (``ValueError`` / ``TypeError``), allocate outputs with torch, and
make one call of the C ABI (``include/asc_cuda.h``) on torch's current stream of the tensors' device.  They return
without waiting for the GPU and record no autograd history; every operator's gradient is a function of its own.  A
status other than 0 raises ``RuntimeError`` (:func:`pyasc_b200.capi.call`); a device-side wait that ran out shows at the
next :func:`pyasc_b200.capi.check_device_status`.  Calls may be captured into CUDA graphs, the first ones too; workspaces
belong to a call, so calls and graphs may run at the same time on several streams.

Tensors are [batch, sequence, heads, head_dim] with any strides, as long as the last dimension is contiguous: slices of
a packed projection, or ``x.transpose(1, 2)`` of a [batch, heads, sequence, head_dim] tensor.
"""
from __future__ import annotations

import math
import struct
from typing import Dict, Optional, Sequence, Tuple

import torch

from . import capi

_DTYPE_CODE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


# --------------------------------------------------------------------------------------------------
# Arguments
# --------------------------------------------------------------------------------------------------
# A call's host time is most of the smallest launches, and a program makes the same call over and over: what the checks
# allow, and the sizes and strides they pack for the C ABI, are kept by the arguments' layouts (shapes, strides, types,
# device; never addresses or contents).
_layouts: Dict[tuple, tuple] = {}
_MAX_LAYOUTS = 1024


def _layout(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _remember(key: tuple, plan: tuple) -> tuple:
    if len(_layouts) >= _MAX_LAYOUTS:
        _layouts.clear()
    _layouts[key] = plan
    return plan


def _device_of(name: str, t: torch.Tensor) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _check_rows(name: str, t: torch.Tensor, dtype: torch.dtype, device: int) -> Tuple[int, ...]:
    """Shape of a [batch, sequence, heads, head_dim] tensor of this type and device."""
    if _device_of(name, t) != device:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} has type {t.dtype}, expected {dtype}")
    shape = t.shape
    if len(shape) != 4:
        raise ValueError(f"{name} must be [batch, sequence, heads, head_dim], got {len(shape)} dimensions")
    if shape[3] > 1 and t.stride(3) != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    return shape


def _check_shape(name: str, shape: Sequence[int], expected: Sequence[int]) -> None:
    if shape != expected:
        raise ValueError(f"{name} has shape {tuple(shape)}, expected {tuple(expected)}")


def _check_vector(name: str, t: torch.Tensor, dtypes, device: int) -> None:
    """A tensor of one of these types on this device."""
    if _device_of(name, t) != device:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")


def _output(name: str, given: Optional[torch.Tensor], like: torch.Tensor, shape: Sequence[int], device: int) -> torch.Tensor:
    """The given output, checked, or a new one (in the order of ``like``'s dimensions)."""
    if given is None:
        return torch.empty_like(like)
    _check_shape(name, _check_rows(name, given, like.dtype, device), shape)
    if any(n > 1 and s == 0 for n, s in zip(given.shape, given.stride())):
        raise ValueError(f"{name} repeats memory (a stride of 0): it cannot be written")
    return given


_PACK = {n: struct.Struct(f"{n}q").pack for n in (6, 12, 14, 20, 24)}     # host int64 arrays of the C ABI
_NO_STRIDES = (0, 0, 0)


def _call(fn_name: str, device: int, *args) -> None:
    """One C-ABI call with ``device`` current, on its current torch stream."""
    stream = torch._C._cuda_getCurrentRawStream(device)
    if device == torch._C._cuda_getDevice():
        capi.call(fn_name, *args, stream)
    else:
        with torch.cuda.device(device):
            capi.call(fn_name, *args, stream)


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
    """Checks what all four functions share: device, shapes, the C ABI's dims, strides and type flag of the positions."""
    device = _device_of("q", q)
    dtype = q.dtype
    if dtype not in _DTYPE_CODE:
        raise TypeError(f"q has type {dtype}, expected float16, bfloat16 or float32")
    q_shape = _check_rows("q", q, dtype, device)
    batch, seq, heads, head_dim = q_shape
    kv_heads, k_shape = 0, None
    if k is not None:
        k_shape = _check_rows("k", k, dtype, device)
        kv_heads = k_shape[2]
        _check_shape("k", k_shape, (batch, seq, kv_heads, head_dim))
    _check_vector("positions", positions, _POSITION_TYPES, device)
    shape, pos_strides = positions.shape, positions.stride()
    if len(shape) == 1 and shape[0] == seq:
        pos_strides = (0, pos_strides[0])
    elif len(shape) == 2 and shape[1] == seq and shape[0] in (1, batch):
        if shape[0] == 1:
            pos_strides = (0, pos_strides[1])
    else:
        raise ValueError(f"positions must be [sequence] or [batch, sequence], got {tuple(shape)}")
    _check_vector("frequencies", frequencies, _FREQUENCY_TYPES, device)
    if frequencies.dim() != 1 or not frequencies.is_contiguous():
        raise ValueError("frequencies must be one contiguous row")
    rotated = 2 * frequencies.numel()
    if rotated > head_dim:
        raise ValueError(f"{frequencies.numel()} frequencies turn {rotated} elements of a head of {head_dim}")
    flags = 4 if positions.dtype == torch.int32 else 0
    return device, q_shape, k_shape, _PACK[6](batch, seq, heads, kv_heads, head_dim, rotated), pos_strides, flags


_POSITION_TYPES = (torch.int64, torch.int32)
_FREQUENCY_TYPES = (torch.float64, )


def _strides(t: Optional[torch.Tensor]) -> Tuple[int, ...]:
    return _NO_STRIDES if t is None else t.stride()[:3]


def _gammas(device: int, head_dim: int, q_gamma: Optional[torch.Tensor], k_gamma: Optional[torch.Tensor]) -> int:
    code = None
    for name, g in (("q_gamma", q_gamma), ("k_gamma", k_gamma)):
        if g is None:
            continue
        _check_vector(name, g, _DTYPE_CODE, device)
        _check_shape(name, g.shape, (head_dim, ))
        if not g.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if code is not None and code != _DTYPE_CODE[g.dtype]:
            raise TypeError("q_gamma and k_gamma must have one type")
        code = _DTYPE_CODE[g.dtype]
    return code or 0


def _rotary_plan(tensors, interleaved, flags):
    """Checks of a forward call: device, dims, strides, codes of the types, flags."""
    q, k, q_gamma, k_gamma, positions, frequencies, q_out, k_out = tensors
    device, q_shape, k_shape, dims, pos_strides, pos_flag = _rotary_arguments(q, k, positions, frequencies)
    if k is None and (k_out is not None or k_gamma is not None):
        raise ValueError("an output or a gamma of k without k")
    gamma_code = _gammas(device, q_shape[3], q_gamma, k_gamma)
    q_out = _output("the output of q", q_out, q, q_shape, device)
    k_out = None if k is None else _output("the output of k", k_out, k, k_shape, device)
    strides = _PACK[14](*_strides(q), *_strides(k), *_strides(q_out), *_strides(k_out), *pos_strides)
    return device, dims, strides, _DTYPE_CODE[q.dtype], gamma_code, flags | pos_flag | bool(interleaved)


def _rotate(q, k, q_gamma, k_gamma, positions, frequencies, eps, scale, interleaved, flags, q_out, k_out):
    tensors = (q, k, q_gamma, k_gamma, positions, frequencies, q_out, k_out)
    try:
        key = (flags, interleaved, *map(_layout, tensors))
        plan = _layouts.get(key)
    except AttributeError:               # not tensors: the checks say which
        key = plan = None
    if plan is None:
        plan = _remember(key, _rotary_plan(tensors, interleaved, flags))
    device, dims, strides, code, gamma_code, flags = plan
    if q_out is None:
        q_out = torch.empty_like(q)
    if k_out is None and k is not None:
        k_out = torch.empty_like(k)
    _call("asc_cuda_norm_rotary", device, q.data_ptr(), _ptr(k), q_out.data_ptr(), _ptr(k_out), _ptr(q_gamma),
          _ptr(k_gamma), positions.data_ptr(), frequencies.data_ptr(), dims, strides, eps, scale, code, gamma_code, flags)
    return q_out, k_out


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


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


def _rotary_backward_plan(tensors, interleaved):
    dq_out, dk_out, q, k, q_gamma, k_gamma, positions, frequencies, dq, dk = tensors
    device, q_shape, k_shape, dims, pos_strides, pos_flag = _rotary_arguments(q, k, positions, frequencies)
    if (k is None) != (dk_out is None):
        raise ValueError("k and dk_out go together")
    if k is None and (dk is not None or k_gamma is not None):
        raise ValueError("an output or a gamma of k without k")
    gamma_code = _gammas(device, q_shape[3], q_gamma, k_gamma)
    _check_shape("dq_out", _check_rows("dq_out", dq_out, q.dtype, device), q_shape)
    dq = _output("dq", dq, q, q_shape, device)
    if k is not None:
        _check_shape("dk_out", _check_rows("dk_out", dk_out, q.dtype, device), k_shape)
        dk = _output("dk", dk, k, k_shape, device)
    strides = _PACK[20](*_strides(dq_out), *_strides(dk_out), *_strides(q), *_strides(k), *_strides(dq), *_strides(dk),
                        *pos_strides)
    return device, dims, strides, _DTYPE_CODE[q.dtype], gamma_code, 2 | pos_flag | bool(interleaved)


def norm_rotary_backward(dq_out: torch.Tensor, dk_out: Optional[torch.Tensor], q: torch.Tensor, k: Optional[torch.Tensor],
                         q_gamma: Optional[torch.Tensor], k_gamma: Optional[torch.Tensor], positions: torch.Tensor,
                         frequencies: torch.Tensor, *, eps: float = 1e-6, scale: float = 1.0, interleaved: bool = False,
                         dq: Optional[torch.Tensor] = None, dk: Optional[torch.Tensor] = None):
    """Gradients ``(dq, dk, dq_gamma, dk_gamma)`` of :func:`norm_rotary` from those of its outputs and its inputs.  The
    gammas' gradients are float32 sums over all rows in a fixed order (None where there is no gamma).  ``dq`` may be
    ``dq_out`` or ``q``, ``dk`` likewise."""
    tensors = (dq_out, dk_out, q, k, q_gamma, k_gamma, positions, frequencies, dq, dk)
    try:
        key = ("norm_rotary_backward", interleaved, *map(_layout, tensors))
        plan = _layouts.get(key)
    except AttributeError:
        key = plan = None
    if plan is None:
        plan = _remember(key, _rotary_backward_plan(tensors, interleaved))
    device, dims, strides, code, gamma_code, flags = plan
    if dq is None:
        dq = torch.empty_like(q)
    if dk is None and k is not None:
        dk = torch.empty_like(k)
    dq_gamma, dk_gamma = (None if g is None else torch.empty_like(g, dtype=torch.float32) for g in (q_gamma, k_gamma))
    _call("asc_cuda_norm_rotary_bwd", device, dq_out.data_ptr(), _ptr(dk_out), q.data_ptr(), _ptr(k), dq.data_ptr(),
          _ptr(dk), _ptr(q_gamma), _ptr(k_gamma), _ptr(dq_gamma), _ptr(dk_gamma), positions.data_ptr(),
          frequencies.data_ptr(), dims, strides, eps, scale, code, gamma_code, flags)
    return dq, dk, dq_gamma, dk_gamma


# --------------------------------------------------------------------------------------------------
# Attention to another sequence
# --------------------------------------------------------------------------------------------------
def _cross_arguments(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_lengths: Optional[torch.Tensor]):
    """Checks what both directions share: device, shapes and the C ABI's dims."""
    device = _device_of("q", q)
    dtype = q.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"q has type {dtype}, expected float16 or bfloat16")
    q_shape, k_shape = _check_rows("q", q, dtype, device), _check_rows("k", k, dtype, device)
    batch, seq, heads, head_dim = q_shape
    kv_seq, kv_heads = k_shape[1], k_shape[2]
    _check_shape("k", k_shape, (batch, kv_seq, kv_heads, head_dim))
    _check_shape("v", _check_rows("v", v, dtype, device), k_shape)
    if heads % kv_heads if kv_heads else heads:
        raise ValueError(f"{heads} query heads are not a multiple of {kv_heads} key heads")
    if kv_lengths is not None:
        _check_vector("kv_lengths", kv_lengths, (torch.int32, ), device)
        _check_shape("kv_lengths", kv_lengths.shape, (batch, ))
        if not kv_lengths.is_contiguous():
            raise ValueError("kv_lengths must be contiguous")
    return device, q_shape, k_shape, _PACK[6](batch, seq, kv_seq, heads, kv_heads, head_dim)


def _default_scale(q: torch.Tensor) -> float:
    return q.shape[3]**-0.5 if q.shape[3] else 0.0


def _cross_plan(tensors):
    q, k, v, kv_lengths, out = tensors
    device, q_shape, _, dims = _cross_arguments(q, k, v, kv_lengths)
    out = _output("out", out, q, q_shape, device)
    strides = _PACK[12](*_strides(q), *_strides(k), *_strides(v), *_strides(out))
    return device, dims, strides, _DTYPE_CODE[q.dtype], (q_shape[0], q_shape[2], q_shape[1])


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, kv_lengths: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """``softmax(scale q k^T) v`` of queries [B, S, Hq, D] and keys and values [B, T, Hkv, D] of another sequence.

    float16 or bfloat16; D a multiple of 8 up to 128; Hq a multiple of Hkv (grouped heads).  ``kv_lengths`` (int32 [B]):
    keys from there on do not take part, whatever they hold.  ``scale`` is ``D ** -0.5`` unless given.  k and v may repeat
    one state (``expand``) over batch or heads.  S = 1 is the form for generated tokens: few rows are cut along the keys
    and joined.  ``return_lse`` adds the float32 [B, Hq, S] logarithms of the softmax sums, which the gradient needs; a
    query without keys gives 0 and -inf.  ``out`` may be ``q`` and must not overlap k or v.  Returns ``out`` or
    ``(out, lse)``."""
    tensors = (q, k, v, kv_lengths, out)
    try:
        key = ("cross_attention", *map(_layout, tensors))
        plan = _layouts.get(key)
    except AttributeError:
        key = plan = None
    if plan is None:
        plan = _remember(key, _cross_plan(tensors))
    device, dims, strides, code, lse_shape = plan
    if out is None:
        out = torch.empty_like(q)
    lse = torch.empty(lse_shape, dtype=torch.float32, device=q.device) if return_lse else None
    _call("asc_cuda_cross_attn_fwd_f16", device, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse),
          _ptr(kv_lengths), dims, strides, _default_scale(q) if scale is None else scale, code)
    return (out, lse) if return_lse else out


def _cross_backward_plan(tensors):
    dout, q, k, v, out, lse, kv_lengths, dq, dk, dv = tensors
    device, q_shape, k_shape, dims = _cross_arguments(q, k, v, kv_lengths)
    dtype = q.dtype
    _check_shape("dout", _check_rows("dout", dout, dtype, device), q_shape)
    _check_shape("out", _check_rows("out", out, dtype, device), q_shape)
    _check_vector("lse", lse, (torch.float32, ), device)
    _check_shape("lse", lse.shape, (q_shape[0], q_shape[2], q_shape[1]))
    if not lse.is_contiguous():
        raise ValueError("lse must be contiguous")
    dq = _output("dq", dq, q, q_shape, device)
    dk, dv = _output("dk", dk, k, k_shape, device), _output("dv", dv, v, k_shape, device)
    strides = _PACK[24](*_strides(dout), *_strides(q), *_strides(k), *_strides(v), *_strides(out), *_strides(dq),
                        *_strides(dk), *_strides(dv))
    return device, dims, strides, _DTYPE_CODE[dtype]


def cross_attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                             lse: torch.Tensor, *, kv_lengths: Optional[torch.Tensor] = None,
                             scale: Optional[float] = None, dq: Optional[torch.Tensor] = None,
                             dk: Optional[torch.Tensor] = None, dv: Optional[torch.Tensor] = None):
    """Gradients ``(dq, dk, dv)`` of :func:`cross_attention`'s output from its gradient, its inputs, ``out`` and ``lse``
    (of the same lengths and scale).  Keys that do not take part get 0; where k or v repeat one state over batch or heads,
    dk and dv hold one gradient for each entry.  Every sum is taken in a fixed order.  The outputs must not overlap the
    inputs."""
    tensors = (dout, q, k, v, out, lse, kv_lengths, dq, dk, dv)
    try:
        key = ("cross_attention_backward", *map(_layout, tensors))
        plan = _layouts.get(key)
    except AttributeError:
        key = plan = None
    if plan is None:
        plan = _remember(key, _cross_backward_plan(tensors))
    device, dims, strides, code = plan
    dq = torch.empty_like(q) if dq is None else dq
    dk = torch.empty_like(k) if dk is None else dk
    dv = torch.empty_like(v) if dv is None else dv
    _call("asc_cuda_cross_attn_bwd_f16", device, dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
          lse.data_ptr(), _ptr(kv_lengths), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dims, strides,
          _default_scale(q) if scale is None else scale, code)
    return dq, dk, dv
