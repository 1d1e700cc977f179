"""Rotary positions and per-head norms (pyasc_b200/attention.py) against their definition in 64 bits.

Tolerances, in units u = 2^-24 of fp32 rounding.  Forward: the mean of squares sums at most 32 values in a lane and 5
shuffle steps (37 u, halved by the root), root, division, two factors (4 u), sine and cosine with their angle's rounding
(4 u of the pair's size), scale, products and sum (3 u): under 32 u of |lo| + |hi|.  Backward: the same again for the
second sum, 64 u of the magnitudes that are added.  A gamma's gradient adds the terms of a lane and of the groups of a
CTA one after another, at most 64 each at these sizes: 192 u of the sum of magnitudes.  On top half a step of the
output type, and for float16 half of its smallest step.
"""
import pytest
import torch

from oracle import transformer as R
from pyasc_b200 import attention as A
from pyasc_b200 import capi

pytestmark = pytest.mark.gpu
U = 2.0**-24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=gen(seed), device="cuda").to(dtype)


def assert_near(got, want, size, units):
    step = torch.finfo(got.dtype).eps / 2
    least = 2.0**-25 if got.dtype == torch.float16 else 1e-38
    bound = want.abs() * step + size * units * U * (1 + step) + least
    off = (got.double() - want).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1, f"{worst:.3g} times the bound, at {(off / bound).argmax().item()}"


def positions_of(batch, seq, first=0):
    return first + torch.randint(0, 50, (batch, 1), generator=gen(9), device="cuda") + torch.arange(seq, device="cuda")


def check_forward(q, k, qg, kg, pos, freq, eps, scale, interleaved, normed, **out):
    if normed:
        got = A.norm_rotary(q, k, qg, kg, pos, freq, eps=eps, scale=scale, interleaved=interleaved, **out)
    else:
        got = A.rotary(q, k, pos, freq, scale=scale, interleaved=interleaved, **out)
    capi.check_device_status(None)
    for y, x, g in zip(got, (q, k), (qg, kg)):
        if x is None:
            assert y is None
            continue
        want = R.norm_rotary(x, g, pos, freq, eps, scale, interleaved, normed)
        n = R.norm(x, g, eps) if normed else x.double()
        assert y.dtype == x.dtype and y.shape == x.shape
        assert_near(y, want, R.partner_sum(n, 2 * freq.numel(), interleaved) * max(scale, 1.0), 32)
    return got


CASES = [
    # B, S, Hq, Hk, D, rotated
    (1, 1, 1, 1, 128, 128),
    (1, 1, 32, 8, 128, 128),
    (64, 1, 8, 2, 64, 64),
    (2, 37, 3, 1, 128, 64),
    (3, 130, 4, 4, 96, 96),
    (2, 33, 5, 1, 80, 40),
    (2, 33, 2, 2, 80, 16),
    (1, 700, 2, 1, 256, 256),
    (1, 19, 2, 1, 512, 512),
    (2, 9, 3, 2, 20, 10),
    (1, 11, 1, 1, 1024, 1000),
    (1, 5, 2, 1, 7, 6),
    (2, 6, 2, 1, 64, 0),
    (1, 3000, 6, 1, 16, 16),
    (2, 12, 2, 1, 1, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b, s, h, hk, d, r", CASES)
def test_forward(b, s, h, hk, d, r, interleaved, dtype):
    packed = normal((b, s, (h + 2 * hk) * d), dtype, d + s)
    q = packed[..., :h * d].unflatten(-1, (h, d))
    k = packed[..., h * d:(h + hk) * d].unflatten(-1, (hk, d))
    freq, _ = A.rotary_frequencies(r, device="cuda")
    pos = positions_of(b, s)
    qg, kg = (1 + 0.2 * normal((d, ), torch.float32, i) for i in (1, 2))
    check_forward(q, k, qg.to(dtype), kg.to(dtype), pos, freq, 1e-6, 1.0, interleaved, True)
    check_forward(q, k, None, None, pos, freq, 0.0, 1.25, interleaved, False)
    y = A.rotary_backward(*A.rotary(q, k, pos, freq, interleaved=interleaved), pos, freq, interleaved=interleaved)
    for a, x in zip(y, (q, k)):           # there and back: two roundings, of values up to sqrt(2) times the pair's
        step = torch.finfo(dtype).eps / 2
        assert ((a.double() - x.double()).abs() <= (4 * step + 64 * U) * R.partner_sum(x.double(), r, interleaved) + 1e-7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b, s, h, hk, d, r", CASES)
def test_backward(b, s, h, hk, d, r, interleaved, dtype):
    q, k = normal((b, s, h, d), dtype, 3), normal((b, s, hk, d), dtype, 4)
    dq_out, dk_out = normal((b, h, s, d), dtype, 5).transpose(1, 2), normal((b, s, hk, d), dtype, 6)
    freq, scale = A.rotary_frequencies(r, scaling="yarn", factor=4.0, original_context=64, device="cuda")
    pos = positions_of(b, s, 100000)
    qg, kg = ((1 + 0.2 * normal((d, ), torch.float32, i)).to(dtype) for i in (1, 2))
    got = A.norm_rotary_backward(dq_out, dk_out, q, k, qg, kg, pos, freq, eps=1e-5, scale=scale, interleaved=interleaved)
    again = A.norm_rotary_backward(dq_out, dk_out, q, k, qg, kg, pos, freq, eps=1e-5, scale=scale, interleaved=interleaved)
    assert all(torch.equal(x, y) for x, y in zip(got, again))        # sums in a fixed order
    for dx, dg, dy, x, g in ((got[0], got[2], dq_out, q, qg), (got[1], got[3], dk_out, k, kg)):
        want, want_g, size, size_g = R.norm_rotary_backward(dy, x, g, pos, freq, 1e-5, scale, interleaved)
        assert_near(dx, want, size, 64)
        assert dg.dtype == torch.float32
        assert_near(dg, want_g, size_g, 192)


def test_backward_against_differences():
    """dx and dgamma against central differences of the 64-bit forward, along a direction."""
    b, s, h, d = 2, 5, 3, 64
    x, dy, g = normal((b, s, h, d), torch.float32, 1), normal((b, s, h, d), torch.float32, 2), normal((d, ), torch.float32, 3)
    freq, _ = A.rotary_frequencies(32, device="cuda")
    pos = torch.arange(s, device="cuda")
    dx, _, dg, _ = A.norm_rotary_backward(dy, None, x, None, g, None, pos, freq, eps=1e-3)
    vx, vg, e = normal(x.shape, torch.float64, 4), normal(g.shape, torch.float64, 5), 1e-5

    def f(t):
        y = R.norm_rotary(x.double() + t * vx, g.double() + t * vg, pos, freq, 1e-3, 1.0, False)
        return (y * dy.double()).sum()

    want = (f(e) - f(-e)) / (2 * e)
    got = (dx.double() * vx).sum() + (dg.double() * vg).sum()
    # the difference is off by e^2 / 6 times a third derivative of order 1e3, and rounding of 1e-13 / e
    assert abs(got - want) <= 1e-6 * ((dx.double() * vx).abs().sum() + (dg.double() * vg).abs().sum())


@pytest.mark.parametrize("how", ["misaligned", "eight_bytes", "odd_pitch", "transposed", "in_place", "expanded"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts(how, dtype):
    b, s, h, hk, d, r = 2, 21, 4, 2, 64, 64
    freq, _ = A.rotary_frequencies(r, device="cuda")
    pos = positions_of(b, s)
    qg, kg = normal((d, ), dtype, 1), normal((d, ), dtype, 2)
    out = {}
    if how == "misaligned":
        q, k = (normal((b * s * n * d + 1, ), dtype, n)[1:].view(b, s, n, d) for n in (h, hk))
    elif how == "eight_bytes":
        q, k = (normal((b * s * n * d + 4, ), dtype, n)[4:].view(b, s, n, d) for n in (h, hk))
    elif how == "odd_pitch":
        q, k = (normal((b, s, n, d + 3), dtype, n)[..., :d] for n in (h, hk))
        out = {"q_out": torch.empty(b, s, h, d + 1, dtype=dtype, device="cuda")[..., :d]}
    elif how == "transposed":
        q, k = (normal((b, n, s, d), dtype, n).transpose(1, 2) for n in (h, hk))
        out = {"q_out": torch.empty(b, h, s, d, dtype=dtype, device="cuda").transpose(1, 2),
               "k_out": torch.empty(s, b, hk, d, dtype=dtype, device="cuda").transpose(0, 1)}
    elif how == "expanded":
        q, k = normal((1, s, h, d), dtype, 1).expand(b, -1, -1, -1), normal((b, s, 1, d), dtype, 2).expand(-1, -1, hk, -1)
    else:
        packed = normal((b, s, (h + hk) * d), dtype, 7)
        q, k = packed[..., :h * d].unflatten(-1, (h, d)), packed[..., h * d:].unflatten(-1, (hk, d))
    for normed in (False, True):
        q0, k0 = q.clone(), k.clone()
        if how == "in_place":
            got = A.norm_rotary(q, k, qg, kg, pos, freq, q_out=q, k_out=k) if normed else A.rotary(q, k, pos, freq,
                                                                                                   q_out=q, k_out=k)
            assert got[0] is q and got[1] is k
            want = check_forward(q0, k0, qg, kg, pos, freq, 1e-6, 1.0, False, normed)
            assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        else:
            got = check_forward(q, k, qg, kg, pos, freq, 1e-6, 1.0, False, normed, **out)
            assert torch.equal(q, q0) and torch.equal(k, k0)
            for name, y in zip(("q_out", "k_out"), got):
                assert name not in out or y is out[name]
    dq, dk = normal(q.shape, dtype, 11), normal(k.shape, dtype, 12)
    plain = A.norm_rotary_backward(dq, dk, q.contiguous(), k.contiguous(), qg, kg, pos, freq)
    other = A.norm_rotary_backward(dq, dk, q, k, qg, kg, pos, freq)
    for x, y in zip(plain, other):        # the kernels for odd strides add in another order
        torch.testing.assert_close(x, y, rtol=2 * torch.finfo(x.dtype).eps, atol=2e-5)


def test_nothing_is_written_outside():
    b, s, h, d = 2, 7, 3, 40
    whole = torch.full((b, s + 2, h + 1, d + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    q = normal((b, s, h, d), torch.bfloat16, 1)
    freq, _ = A.rotary_frequencies(32, device="cuda")
    A.rotary(q, None, torch.arange(s, device="cuda"), freq, q_out=whole[:, 1:-1, :h, :d])
    inner = whole[:, 1:-1, :h, :d].clone()
    whole[:, 1:-1, :h, :d] = 7.0
    assert (whole == 7).all() and not (inner == 7).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_non_finite_values_stay_in_their_pair(interleaved):
    q = normal((1, 2, 2, 64), torch.float32, 1)
    q[0, 0, 0, 40] = float("inf")        # in the part that passes
    q[0, 1, 1, 3] = float("nan")
    freq, _ = A.rotary_frequencies(32, device="cuda")
    y, _ = A.rotary(q, None, torch.arange(2, device="cuda") + 1, freq, interleaved=interleaved)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[0, 0, 0, 40] = True
    for i in (2, 3) if interleaved else (3, 19):
        want[0, 1, 1, i] = True
    assert torch.equal(bad, want)
    assert y[0, 0, 0, 40] == float("inf")


def test_position_types_and_shapes():
    b, s = 3, 17
    q = normal((b, s, 2, 128), torch.bfloat16, 1)
    freq, _ = A.rotary_frequencies(128, device="cuda")
    row = torch.arange(s, device="cuda") + 123456
    base, _ = A.rotary(q, None, row, freq)
    both = torch.stack([row] * b)
    wide = torch.zeros(b, 2 * s, dtype=torch.int64, device="cuda")
    wide[:, ::2] = both
    for pos in (row.int(), row[None], row.expand(b, s), both, both.int(), wide[:, ::2]):
        assert torch.equal(A.rotary(q, None, pos, freq)[0], base)
    back, _ = A.rotary(q, None, -row, freq)                # negative positions turn the other way
    assert torch.equal(back, A.rotary_backward(q, None, row, freq)[0])


def test_far_positions_keep_their_angle():
    s = 64
    q = normal((1, s, 2, 128), torch.float32, 1)
    freq, _ = A.rotary_frequencies(128, device="cuda")
    check_forward(q, None, None, None, torch.arange(s, device="cuda") + (1 << 40), freq, 0.0, 1.0, False, False)


def test_gamma_types_and_absence():
    q, k = normal((2, 9, 4, 64), torch.float16, 1), normal((2, 9, 2, 64), torch.float16, 2)
    freq, _ = A.rotary_frequencies(64, device="cuda")
    pos = torch.arange(9, device="cuda")
    for t in (torch.float32, torch.bfloat16, torch.float16):
        check_forward(q, k, normal((64, ), t, 3), normal((64, ), t, 4), pos, freq, 1e-6, 1.0, False, True)
    check_forward(q, k, None, normal((64, ), torch.float32, 4), pos, freq, 1e-6, 1.0, True, True)
    dq, dk, gq, gk = A.norm_rotary_backward(q, k, q, k, None, normal((64, ), torch.float32, 4), pos, freq)
    assert gq is None and gk.shape == (64, )
    want, _, size, _ = R.norm_rotary_backward(q, q, None, pos, freq, 1e-6, 1.0, False)
    assert_near(dq, want, size, 64)


def test_empty():
    freq, _ = A.rotary_frequencies(64, device="cuda")
    g = torch.ones(64, device="cuda")
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64)):
        q, pos = torch.empty(shape, device="cuda"), torch.arange(shape[1], device="cuda")
        assert A.rotary(q, None, pos, freq)[0].shape == shape
        dq, _, dg, _ = A.norm_rotary_backward(q, None, q, None, g, None, pos, freq)
        assert dq.shape == shape and (dg == 0).all()
    k = normal((2, 4, 1, 64), torch.float32, 1)            # keys without queries
    y = A.rotary(torch.empty(2, 4, 0, 64, device="cuda"), k, torch.arange(4, device="cuda"), freq)[1]
    assert torch.equal(y, A.rotary(k, None, torch.arange(4, device="cuda"), freq)[0])


def test_offsets_past_32_bits():
    free, _ = torch.cuda.mem_get_info()
    assert free > 30 << 30
    stride = (1 << 32) + 256
    buf = torch.empty(stride + 4096, dtype=torch.bfloat16, device="cuda")
    q = buf.as_strided((2, 8, 4, 64), (stride, 256, 64, 1))
    q.copy_(normal((2, 8, 4, 64), torch.bfloat16, 1))
    freq, _ = A.rotary_frequencies(64, device="cuda")
    pos = torch.arange(8, device="cuda")
    want, _ = A.rotary(q.contiguous(), None, pos, freq)
    assert torch.equal(A.rotary(q, None, pos, freq)[0], want)
    A.rotary(q, None, pos, freq, q_out=q)
    assert torch.equal(q, want)


def test_streams_and_graphs():
    q, k = normal((2, 65, 4, 128), torch.bfloat16, 1), normal((2, 65, 2, 128), torch.bfloat16, 2)
    g = normal((128, ), torch.bfloat16, 3)
    freq, _ = A.rotary_frequencies(128, device="cuda")
    pos = positions_of(2, 65)

    def step():
        y = A.norm_rotary(q, k, g, g, pos, freq)
        return (*y, *A.norm_rotary_backward(*y, q, k, g, g, pos, freq))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):                    # two graphs, each with its own workspace, replayed at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    q.copy_(normal(q.shape, torch.bfloat16, 8))
    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_in_place_backward():
    q, k = normal((2, 33, 4, 64), torch.float16, 1), normal((2, 33, 2, 64), torch.float16, 2)
    dq, dk = normal(q.shape, torch.float16, 3), normal(k.shape, torch.float16, 4)
    freq, _ = A.rotary_frequencies(64, device="cuda")
    pos, g = torch.arange(33, device="cuda"), normal((64, ), torch.float16, 5)
    want = A.norm_rotary_backward(dq, dk, q, k, g, g, pos, freq)
    a, b = dq.clone(), k.clone()
    got = A.norm_rotary_backward(a, dk, q, b, g, g, pos, freq, dq=a, dk=b)
    assert got[0] is a and got[1] is b
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_refusals():
    q, k = normal((2, 4, 4, 64), torch.float16, 1), normal((2, 4, 2, 64), torch.float16, 2)
    pos, g = torch.arange(4, device="cuda"), torch.ones(64, device="cuda")
    freq, _ = A.rotary_frequencies(64, device="cuda")
    wide, _ = A.rotary_frequencies(66, device="cuda")
    calls = [
        (ValueError, lambda: A.rotary(q, k[:1], pos, freq)),
        (ValueError, lambda: A.rotary(q, k[:, :3], pos, freq)),
        (ValueError, lambda: A.rotary(q, k[..., :32], pos, freq)),
        (ValueError, lambda: A.rotary(q[0], None, pos, freq)),
        (ValueError, lambda: A.rotary(q.transpose(2, 3), None, pos, freq)),
        (ValueError, lambda: A.rotary(q, k.cpu(), pos, freq)),
        (TypeError, lambda: A.rotary(q, k.float(), pos, freq)),
        (TypeError, lambda: A.rotary(q.double(), None, pos, freq)),
        (TypeError, lambda: A.rotary(q, k, pos.float(), freq)),
        (ValueError, lambda: A.rotary(q, k, pos[:3], freq)),
        (ValueError, lambda: A.rotary(q, k, pos.expand(3, 4), freq)),
        (TypeError, lambda: A.rotary(q, k, pos, freq.float())),
        (ValueError, lambda: A.rotary(q, k, pos, wide)),
        (ValueError, lambda: A.rotary(q, k, pos, freq.expand(2, -1))),
        (ValueError, lambda: A.rotary(q, k, pos, freq, q_out=torch.empty_like(k))),
        (ValueError, lambda: A.rotary(q, k, pos, freq, q_out=q[:1].expand(2, -1, -1, -1))),
        (ValueError, lambda: A.rotary(q, None, pos, freq, k_out=k)),
        (ValueError, lambda: A.norm_rotary(q, k, g[:32], g, pos, freq)),
        (TypeError, lambda: A.norm_rotary(q, k, g, g.half(), pos, freq)),
        (ValueError, lambda: A.norm_rotary(q, None, g, g, pos, freq)),
        (ValueError, lambda: A.norm_rotary_backward(q, None, q, k, g, g, pos, freq)),
        (ValueError, lambda: A.norm_rotary_backward(q[:, :3], k, q, k, g, g, pos, freq)),
        (ValueError, lambda: A.norm_rotary_backward(q, k, q, k, g, g, pos, freq, dk=q)),
        (RuntimeError, lambda: A.rotary(q.repeat(1, 1, 1, 17), None, pos, freq)),       # a head of 1088
    ]
    A.rotary(q, k, pos, freq)                      # (an allowed call does not let a refused one through)
    for error, call in calls:
        with pytest.raises(error):
            call()
