"""Attention to another sequence without a GPU: status codes of the C ABI and refusals of host tensors."""
import ctypes

import pytest
import torch

from pyasc_b200 import attention as A
from pyasc_b200 import capi


def forward(dims, strides=(64, ) * 12, scale=1.0, dtype=0, q_off=0, k_null=False, lse_off=None):
    buf = (ctypes.c_double * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    return capi.load().asc_cuda_cross_attn_fwd_f16(p + q_off, None if k_null else p, p, p, None if lse_off is None else p + lse_off,
                                                   None, (ctypes.c_int64 * 6)(*dims), (ctypes.c_int64 * 12)(*strides), scale,
                                                   dtype, None)


GOOD = (2, 3, 4, 2, 2, 64)


def changed(i, value, base=GOOD):
    return tuple(value if j == i else x for j, x in enumerate(base))


def test_nothing_to_do():
    for i in (0, 1):
        assert forward(changed(i, 0)) == 0
    assert forward((2, 3, 4, 0, 0, 64)) == 0


def test_status_codes():
    for i in range(6):
        assert forward(changed(i, -1)) == 1
    assert forward((2, 3, 4, 3, 2, 64)) == 1           # heads that do not group
    assert forward((2, 3, 4, 3, 0, 64)) == 1
    assert forward(changed(5, 60)) == 3
    assert forward(changed(5, 136)) == 3
    assert forward(GOOD, dtype=2) == 1
    assert forward(GOOD, scale=-0.5) == 1
    assert forward(GOOD, scale=float("nan")) == 1
    assert forward(GOOD, scale=float("inf")) == 1
    assert forward(GOOD, q_off=2) == 2
    assert forward(GOOD, k_null=True) == 1
    assert forward(GOOD, lse_off=2) == 2
    for i in range(12):
        assert forward(GOOD, strides=changed(i, 60, (64, ) * 12)) == 2
        assert forward(GOOD, strides=changed(i, -64, (64, ) * 12)) == 1
    for i in (0, 2, 1, 4, 7, 9, 10, 11):               # a stride of 0 only over batch and heads of k and v
        assert forward(GOOD, strides=changed(i, 0, (64, ) * 12)) == 1
    assert forward(GOOD, strides=changed(3, 1 << 39, (64, ) * 12)) == 6
    assert forward(changed(0, 1 << 25)) == 6


def test_host_tensors_are_refused():
    q = torch.zeros(1, 2, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        A.cross_attention(q, q, q)
    with pytest.raises(TypeError):
        A.cross_attention(None, q, q)


def test_a_call_runs_on_its_tensors_device(monkeypatch):
    """With another device current, the tensors' device is made current for the call, and its stream is used."""
    seen = []

    class Current:
        device = 0

        def __init__(self, device):
            self.to = device

        def __enter__(self):
            self.back, Current.device = Current.device, self.to

        def __exit__(self, *_):
            Current.device = self.back

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: Current.device, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 100 + device, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Current)
    monkeypatch.setattr(capi, "call", lambda name, *args: seen.append((Current.device, name, args)))
    A._call("f", 1, 7)
    A._call("g", 0, 8)
    assert seen == [(1, "f", (7, 101)), (0, "g", (8, 100))] and Current.device == 0


def test_layouts_that_are_kept_are_bounded():
    before = dict(A._layouts)
    try:
        for i in range(A._MAX_LAYOUTS + 10):
            A._remember(("test", i), (i, ))
        assert len(A._layouts) <= A._MAX_LAYOUTS
    finally:
        A._layouts.clear()
        A._layouts.update(before)
