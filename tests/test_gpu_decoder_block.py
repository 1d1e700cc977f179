"""The attention part of an encoder-decoder block as it is used: per-head norms and rotary positions of packed queries and
keys, causal self-attention, attention to padded encoder states, and back through both; in prompts and token by token."""
import os
import subprocess
import sys

import pytest
import torch

from oracle import golden as G
from oracle import transformer as R
from pyasc_b200 import attention as A
from pyasc_b200 import capi
from pyasc_b200 import tutorials as T

pytestmark = pytest.mark.gpu
DT = torch.float16


def normal(shape, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(DT)


def setup(b, s, h, hk, t, d):
    packed = normal((b, s, (h + 2 * hk) * d), 1)
    q, k, v = (packed[..., i * d:j * d].unflatten(-1, (j - i, d)) for i, j in ((0, h), (h, h + hk), (h + hk, h + 2 * hk)))
    states = normal((b, t, 2, hk, d), 2)
    gammas = [(1 + 0.2 * normal((d, ), i).float()).to(DT) for i in (3, 4)]
    frequencies, scale = A.rotary_frequencies(d, scaling="yarn", factor=4.0, original_context=2048, device="cuda")
    return q, k, v, states, gammas, frequencies, scale


def test_block_and_its_gradients():
    b, s, h, t, d = 2, 200, 4, 333, 128
    q, k, v, states, (qg, kg), freq, scale = setup(b, s, h, h, t, d)
    pos = torch.arange(s, device="cuda") + 5000
    lengths = torch.tensor([333, 100], dtype=torch.int32, device="cuda")
    # the norm lays its results out as the self-attention kernel reads them
    qr, kr = (torch.empty(b, h, s, d, dtype=DT, device="cuda") for _ in range(2))
    A.norm_rotary(q, k, qg, kg, pos, freq, scale=scale, q_out=qr.transpose(1, 2), k_out=kr.transpose(1, 2))
    vr, o = v.transpose(1, 2).contiguous(), torch.empty_like(qr)
    T.attention_launch(qr, kr, vr, o, causal=True, q_tile=100)     # (query tiles divide the sequence)
    x = o.transpose(1, 2)                                   # [B, S, H, D] again, strided
    y, lse = A.cross_attention(x, states[:, :, 0], states[:, :, 1], kv_lengths=lengths, return_lse=True)
    dy = normal(y.shape, 9)
    dx, dk, dv = A.cross_attention_backward(dy, x, states[:, :, 0], states[:, :, 1], y, lse, kv_lengths=lengths)
    capi.check_device_status(None)

    # each stage against 64 bits of its own inputs, as the parity tests of the stages do
    for got, src, g in ((qr, q, qg), (kr, k, kg)):
        want = R.norm_rotary(src, g, pos, freq, 1e-6, scale, False)
        size = R.partner_sum(R.norm(src, g, 1e-6), d, False) * scale
        assert ((got.transpose(1, 2).double() - want).abs() <= want.abs() * 2.0**-11 + size * 2.0**-18 + 2.0**-25).all()
    G.assert_half_close(o, G.attention(qr.cpu(), kr.cpu(), vr.cpu(), True))
    want, _ = R.cross_attention(x, states[:, :, 0], states[:, :, 1], lengths)
    G.assert_half_close(y, want.float().cpu())
    bounds = R.cross_attention_backward_bounds(dy, x, states[:, :, 0], states[:, :, 1], lengths, d**-0.5, 2.0**-11 * 1.001,
                                               2.0**-25)
    for got, want, bound in zip((dx, dk, dv), R.cross_attention_backward(dy, x, states[:, :, 0], states[:, :, 1], lengths),
                                bounds):
        assert ((got.double() - want).abs() <= bound).all()


def test_tokens_one_by_one_are_the_prompt():
    """A token at a time gives what the whole prompt gives: rotary bit by bit, attention within its roundings."""
    b, s, h, hk, t, d = 2, 9, 8, 2, 500, 64
    q, k, _, states, (qg, kg), freq, scale = setup(b, s, h, hk, t, d)
    pos = torch.arange(s, device="cuda")[None] + torch.tensor([[0], [70]], device="cuda")
    lengths = torch.tensor([17, 500], dtype=torch.int32, device="cuda")
    whole = A.norm_rotary(q, k, qg, kg, pos, freq, scale=scale)
    out = A.cross_attention(whole[0], states[:, :, 0], states[:, :, 1], kv_lengths=lengths)
    for i in range(s):
        one = A.norm_rotary(q[:, i:i + 1], k[:, i:i + 1], qg, kg, pos[:, i:i + 1], freq, scale=scale)
        assert torch.equal(one[0], whole[0][:, i:i + 1]) and torch.equal(one[1], whole[1][:, i:i + 1])
        token = A.cross_attention(one[0], states[:, :, 0], states[:, :, 1], kv_lengths=lengths)
        torch.testing.assert_close(token, out[:, i:i + 1], atol=2e-3, rtol=2e-3)


@pytest.mark.parametrize("b, h, hk, s, t, d", [(2, 4, 2, 128, 333, 128), (1, 6, 1, 1, 900, 64), (2, 3, 3, 96, 96, 80)])
def test_script_form(b, h, hk, s, t, d):
    """The asc2 script, with device tensors and with host tensors."""
    q, k, v = (torch.randn(n, generator=G.gen()).to(DT) for n in ((b, h, s, d), (b, hk, t, d), (b, hk, t, d)))
    want, _ = R.cross_attention(*(x.transpose(1, 2) for x in (q, k, v)))
    want = want.transpose(1, 2).float()
    o = torch.empty_like(q)
    T.cross_attention_launch(q, k, v, o)
    G.assert_half_close(o, want)
    od = torch.empty_like(q, device="cuda")
    T.cross_attention_launch(q.cuda(), k.cuda(), v.cuda(), od)
    assert torch.equal(od.cpu(), o)


def test_output_over_its_queries():
    """out may be q: whoever reads a query reads it before its result is stored."""
    for b, s, h, hk, t, d in ((2, 1, 8, 2, 3000, 128), (2, 40, 6, 3, 700, 64), (1, 700, 2, 2, 5000, 128)):
        q, _, _, states, _, _, _ = setup(b, s, h, hk, t, d)
        q = q.contiguous()
        want = A.cross_attention(q, states[:, :, 0], states[:, :, 1])
        assert torch.equal(A.cross_attention(q, states[:, :, 0], states[:, :, 1], out=q), want)


def test_calls_on_two_streams_at_once():
    """Launches that overlap use workspaces of their own."""
    b, s, h, t, d = 1, 3, 4, 6000, 128
    q, _, _, states, _, _, _ = setup(b, s, h, h, t, d)
    want = A.cross_attention(q, states[:, :, 0], states[:, :, 1], return_lse=True)
    dy = normal(q.shape, 5)
    grads = A.cross_attention_backward(dy, q, states[:, :, 0], states[:, :, 1], *want)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(4)], []
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                y = A.cross_attention(q, states[:, :, 0], states[:, :, 1], return_lse=True)
                got.append((*y, *A.cross_attention_backward(dy, q, states[:, :, 0], states[:, :, 1], *y)))
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(a, b) for a, b in zip(x, (*want, *grads)))


FIRST_CALLS_IN_A_CAPTURE = """
import torch
from pyasc_b200 import attention as A
q, k, p = (torch.randn(2, n, h, 64, device="cuda").half() for n, h in ((1, 4), (3000, 2), (300, 4)))
frequencies, _ = A.rotary_frequencies(64, device="cuda")
positions, gamma = torch.arange(300, device="cuda"), torch.ones(64, device="cuda")

def step():
    x, _ = A.norm_rotary(p, None, gamma, None, positions, frequencies)
    y, lse = A.cross_attention(x, k, k, return_lse=True)
    return (x, y, *A.cross_attention_backward(p, x, k, k, y, lse), A.cross_attention(q, k, k),
            A.norm_rotary_backward(p, None, p, None, gamma, None, positions, frequencies)[2])

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
"""


def test_first_calls_inside_a_capture():
    """A process whose first calls are captured: what the library sets up on first use does not break the capture."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS_IN_A_CAPTURE], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
