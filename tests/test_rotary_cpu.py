"""Rotary positions without a GPU: frequencies, refusals of the Python functions and status codes of the C ABI."""
import ctypes
import math

import pytest
import torch

from oracle import transformer as R
from pyasc_b200 import attention as A
from pyasc_b200 import capi


def test_frequencies():
    f, scale = A.rotary_frequencies(8, 10000.0)
    assert f.dtype == torch.float64 and scale == 1.0
    torch.testing.assert_close(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    torch.testing.assert_close(A.rotary_frequencies(8, scaling="linear", factor=4.0)[0], f / 4)
    ntk = A.rotary_frequencies(8, scaling="ntk", factor=4.0)[0]
    assert ntk[0] == f[0]
    torch.testing.assert_close(ntk[-1], f[-1] / 4)
    assert A.rotary_frequencies(0)[0].numel() == 0


def test_yarn_frequencies():
    f = A.rotary_frequencies(128)[0]
    y, scale = A.rotary_frequencies(128, scaling="yarn", factor=8.0, original_context=4096)
    assert scale == 0.1 * math.log(8.0) + 1
    turns = 4096 * f / (2 * math.pi)                     # turns of each pair within the original context
    assert torch.equal(y[turns > 40], f[turns > 40])
    torch.testing.assert_close(y[turns < 0.8], f[turns < 0.8] / 8)
    assert ((y <= f) & (y >= f / 8 * (1 - 1e-12))).all()


@pytest.mark.parametrize("args, kwargs", [((7, ), {}), ((8, 1.0), {}), ((8, ), {"scaling": "other"}), ((-2, ), {}),
                                          ((8, ), {"scaling": "yarn", "factor": 2.0}), ((8, ), {"factor": 0.5})])
def test_frequencies_refuse(args, kwargs):
    with pytest.raises(ValueError):
        A.rotary_frequencies(*args, **kwargs)


def test_host_tensors_are_refused():
    q, pos = torch.zeros(1, 4, 2, 64), torch.arange(4)
    f, _ = A.rotary_frequencies(64)
    for call in (lambda: A.rotary(q, None, pos, f), lambda: A.rotary_backward(q, None, pos, f),
                 lambda: A.norm_rotary(q, None, None, None, pos, f),
                 lambda: A.norm_rotary_backward(q, None, q, None, None, None, pos, f)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        A.rotary([1.0], None, pos, f)


def _call(fn, dims, strides, flags=0, dtype=0, gamma_dtype=0, off=0, out_null=False):
    buf = (ctypes.c_double * 64)()
    p = ctypes.addressof(buf)
    lib = capi.load()
    d, s = (ctypes.c_int64 * len(dims))(*dims), (ctypes.c_int64 * len(strides))(*strides)
    out = None if out_null else p
    if fn == "fwd":
        return lib.asc_cuda_norm_rotary(p + off, p, out, out, p, p, p, p, d, s, 1e-6, 1.0, dtype, gamma_dtype, flags, None)
    return lib.asc_cuda_norm_rotary_bwd(p + off, p, p, p, out, out, p, p, None, None, p, p, d, s, 1e-6, 1.0, dtype,
                                        gamma_dtype, flags, None)


@pytest.mark.parametrize("fn, n, flags", [("fwd", 14, 0), ("bwd", 20, 2)])
def test_status_codes(fn, n, flags):
    one = [64] * n
    good = [2, 2, 2, 2, 8, 8]
    assert _call(fn, [0, 2, 2, 2, 8, 8], one, flags) == 0              # nothing to do
    assert _call(fn, [2, 2, 0, 0, 8, 8], one, flags) == 0
    assert _call(fn, [2, 2, 2, 2, 8, 7], one, flags) == 1              # odd
    assert _call(fn, [2, 2, 2, 2, 8, 10], one, flags) == 1             # more than the head
    assert _call(fn, [2, 2, -1, 2, 8, 8], one, flags) == 1
    assert _call(fn, [2, 2, 2, 2, 1026, 8], one, flags) == 6
    assert _call(fn, [1 << 20, 1 << 20, 2, 2, 8, 8], one, flags) == 6
    assert _call(fn, good, one, flags, dtype=3) == 1
    assert _call(fn, good, one, flags, gamma_dtype=-1) == 1
    assert _call(fn, good, one, flags | 16) == 1
    assert _call(fn, good, one, flags, out_null=True) == 1
    assert _call(fn, good, one, flags, off=1) == 2
    assert _call(fn, good, one, flags, dtype=2, off=2) == 2
    assert _call(fn, good, [0] * n, flags) == 1                        # outputs that share memory
    if fn == "bwd":
        assert _call(fn, good, one, 0) == 1                            # without the norm it is the forward, turned back
        assert _call(fn, good, one, 10) == 1


def test_the_gradient_of_the_definition():
    """The formulas of the 64-bit definition against autograd."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 2, 16, generator=g, dtype=torch.float64, requires_grad=True)
    gamma = torch.randn(16, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(2, 3, 2, 16, generator=g, dtype=torch.float64)
    f, pos = A.rotary_frequencies(8)[0], torch.arange(3) + 5
    for interleaved in (False, True):
        y = R.norm_rotary(x, gamma, pos, f, 1e-3, 1.2, interleaved)
        want = torch.autograd.grad(y, (x, gamma), dy)
        dx, dgamma, _, _ = R.norm_rotary_backward(dy, x.detach(), gamma.detach(), pos, f, 1e-3, 1.2, interleaved)
        torch.testing.assert_close(dx, want[0])
        torch.testing.assert_close(dgamma, want[1])


@pytest.mark.parametrize("grouped", [1, 3])
def test_the_gradient_of_attention(grouped):
    g = torch.Generator().manual_seed(2)
    q = torch.randn(2, 4, 2 * grouped, 8, generator=g, dtype=torch.float64, requires_grad=True)
    k = torch.randn(2, 5, 2, 8, generator=g, dtype=torch.float64, requires_grad=True)
    v = torch.randn(2, 5, 2, 8, generator=g, dtype=torch.float64, requires_grad=True)
    do = torch.randn(2, 4, 2 * grouped, 8, generator=g, dtype=torch.float64)
    for lengths in (None, torch.tensor([5, 2]), torch.tensor([0, 3])):
        out, _ = R.cross_attention(q, k, v, lengths)
        want = torch.autograd.grad(out, (q, k, v), do)
        got = R.cross_attention_backward(do, q.detach(), k.detach(), v.detach(), lengths)
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b)
