"""Gradients of attention to another sequence against their formulas in 64 bits; the bounds count the roundings of P, dS,
out and the results, see ``oracle.transformer.cross_attention_backward_bounds``."""
import pytest
import torch

from oracle import transformer as R
from pyasc_b200 import attention as A
from pyasc_b200 import capi

pytestmark = pytest.mark.gpu


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def check(q, k, v, do, lengths=None, scale=None, **kw):
    out, lse = A.cross_attention(q, k, v, kv_lengths=lengths, scale=scale, return_lse=True)
    got = A.cross_attention_backward(do, q, k, v, out, lse, kv_lengths=lengths, scale=scale, **kw)
    capi.check_device_status(None)
    scale = q.shape[-1]**-0.5 if scale is None else scale
    want = R.cross_attention_backward(do, q, k, v, lengths, scale)
    step = torch.finfo(q.dtype).eps / 2
    bounds = R.cross_attention_backward_bounds(do, q, k, v, lengths, scale, step * (1 + step),
                                               2.0**-25 if q.dtype == torch.float16 else 1e-38)
    for name, a, b, bound in zip(("dq", "dk", "dv"), got, want, bounds):
        assert a.shape == b.shape and a.dtype == q.dtype
        off = (a.double() - b).abs()
        assert torch.isfinite(a).all(), name
        assert (off <= bound).all(), f"{name}: {(off / bound).max().item():.3g} times the bound"
    again = A.cross_attention_backward(do, q, k, v, out, lse, kv_lengths=lengths, scale=scale)
    assert all(torch.equal(a, b) for a, b in zip(got, again))        # a fixed order of all sums
    return got


SIZES = [
    # B, S, T, Hq, Hkv, D
    (1, 1, 1, 1, 1, 64),
    (1, 128, 64, 1, 1, 128),
    (1, 64, 128, 1, 1, 64),
    (2, 1, 300, 8, 2, 128),
    (1, 5, 129, 12, 2, 64),
    (1, 16, 100, 20, 1, 96),
    (2, 17, 77, 6, 3, 128),
    (1, 32, 65, 4, 1, 80),
    (1, 33, 200, 6, 2, 128),
    (2, 100, 63, 9, 3, 64),
    (1, 257, 190, 2, 1, 72),
    (2, 333, 77, 3, 3, 40),
    (1, 700, 1025, 4, 2, 128),
    (3, 513, 321, 4, 4, 64),
    (1, 40, 5000, 2, 1, 128),
    (1, 5000, 40, 2, 1, 128),
    (1, 300, 1, 2, 2, 8),
    (1, 1, 700, 64, 1, 128),
    (2, 3, 130, 17, 1, 64),
    (40, 130, 260, 4, 4, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b, s, t, h, hk, d", SIZES)
def test_gradients(b, s, t, h, hk, d, dtype):
    q, packed, do = normal((b, s, h, d), dtype, 1), normal((b, t, 2, hk, d), dtype, 2), normal((b, s, h, d), dtype, 3)
    check(q, packed[:, :, 0], packed[:, :, 1], do)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("s", [1, 20, 200])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("fill", [0.0, float("nan"), float("-inf")])
def test_lengths(s, d, fill, dtype):
    t = 400
    lengths = torch.tensor([0, 1, 63, 64, 65, 127, 128, 129, 399, 400], dtype=torch.int32, device="cuda")
    b = lengths.numel()
    q, k, v = normal((b, s, 4, d), dtype, 1), normal((b, t, 2, d), dtype, 2), normal((b, t, 2, d), dtype, 3)
    do = normal((b, s, 4, d), dtype, 4)
    want = check(q, k, v, do, lengths)
    gone = torch.arange(t, device="cuda")[None] >= lengths[:, None]
    k[gone], v[gone] = fill, fill
    got = check(q, k, v, do, lengths)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert (got[1][gone] == 0).all() and (got[2][gone] == 0).all() and (got[0][0] == 0).all()


@pytest.mark.parametrize("s", [3, 150])
def test_layouts(s):
    b, t, h, hk, d, dt = 2, 200, 4, 2, 64, torch.bfloat16
    q, k, v, do = normal((b, s, h, d), dt, 1), normal((b, t, hk, d), dt, 2), normal((b, t, hk, d), dt, 3), normal((b, s, h, d), dt, 4)
    want = check(q, k, v, do)

    def transposed(x):
        return x.transpose(1, 2).contiguous().transpose(1, 2)

    whole = torch.full((b, t, 3, hk, d), 7.0, dtype=dt, device="cuda")
    dq = torch.full((b, s + 1, h, d + 8), 7.0, dtype=dt, device="cuda")
    out, lse = A.cross_attention(q, k, v, return_lse=True)
    got = A.cross_attention_backward(transposed(do), transposed(q), transposed(k), v, transposed(out), lse,
                                     dq=dq[:, :s, :, :d], dk=whole[:, :, 0], dv=whole[:, :, 2])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert (whole[:, :, 1] == 7).all() and (dq[:, s] == 7).all() and (dq[..., d:] == 7).all()
    # one state for the batch: a gradient for each entry
    got = check(q, k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1), do)
    same = check(q, k[:1].repeat(b, 1, 1, 1), v[:1].repeat(b, 1, 1, 1), do)
    assert all(torch.equal(a, b) for a, b in zip(got, same))
    got = check(q, k[:, :, :1].expand(-1, -1, hk, -1), v, do)
    same = check(q, k[:, :, :1].repeat(1, 1, hk, 1), v, do)
    assert all(torch.equal(a, b) for a, b in zip(got, same))


def test_against_differences():
    """The gradients along a direction against central differences of the 64-bit forward."""
    b, s, t, h, hk, d = 1, 20, 30, 4, 2, 64
    x = [normal(n, torch.float16, i) for i, n in enumerate(((b, s, h, d), (b, t, hk, d), (b, t, hk, d)))]
    do = normal((b, s, h, d), torch.float16, 5)
    out, lse = A.cross_attention(*x, return_lse=True)
    got = A.cross_attention_backward(do, *x, out, lse)
    bounds = R.cross_attention_backward_bounds(do, *x, None, d**-0.5, 2.0**-11, 2.0**-25)
    e = 1e-5
    for i in range(3):
        w = normal(x[i].shape, torch.float64, 7 + i)

        def f(step):
            y = [a.double() for a in x]
            y[i] = y[i] + step * w
            return (R.cross_attention(*y)[0] * do.double()).sum()

        want = (f(e) - f(-e)) / (2 * e)
        # truncation of the difference: e^2 times a third derivative far below 1e4; rounding 1e-12 / e
        assert abs((got[i].double() * w).sum() - want) <= (bounds[i] * w.abs()).sum() + 2e-6


def test_empty():
    def z(*shape):
        return torch.randn(shape, device="cuda").half()

    def back(q, k):
        out, lse = A.cross_attention(q, k, k, return_lse=True)
        return A.cross_attention_backward(q, q, k, k, out, lse)

    for b, s, t in ((0, 3, 5), (2, 0, 5), (2, 3, 0), (2, 200, 0)):
        dq, dk, dv = back(z(b, s, 4, 64), z(b, t, 2, 64))
        assert dq.shape == (b, s, 4, 64) and dk.shape == dv.shape == (b, t, 2, 64)
        assert (dq == 0).all() and (dk == 0).all() and (dv == 0).all()


def test_scale_zero_and_other():
    q, k, v, do = (normal((1, n, 2, 64), torch.bfloat16, n) for n in (70, 90, 90, 70))
    dq, dk, _ = check(q, k, v, do, scale=0.0)
    assert (dq == 0).all() and (dk == 0).all()
    check(q, k, v, do, scale=0.5)


def test_refusals():
    q, k = (torch.zeros(2, 4, n, 64, dtype=torch.float16, device="cuda") for n in (4, 2))
    out, lse = A.cross_attention(q, k, k, return_lse=True)
    good = [q, q, k, k, out, lse]
    for i, error, bad in ((0, ValueError, q[:1]), (0, TypeError, q.float()), (0, ValueError, q.cpu()),
                          (0, RuntimeError, q[:1].expand(2, -1, -1, -1)), (1, ValueError, q[:, :3]),
                          (4, ValueError, out[:, :, :2]), (5, TypeError, lse.half()), (5, ValueError, lse[:, :2]),
                          (5, ValueError, lse.transpose(1, 2).contiguous().transpose(1, 2))):
        args = list(good)
        args[i] = bad
        with pytest.raises(error):
            A.cross_attention_backward(*args)
    with pytest.raises(ValueError):
        A.cross_attention_backward(*good, dk=k[:1].expand(2, -1, -1, -1))


@pytest.mark.parametrize("s, t", [(5, 2000), (700, 40), (200, 200)])
def test_streams_and_graphs(s, t):
    q, k, v, do = (normal((2, n, 2, 128), torch.bfloat16, i) for i, n in enumerate((s, t, t, s)))
    lengths = torch.tensor([t, t // 2], dtype=torch.int32, device="cuda")

    def step():
        out, lse = A.cross_attention(q, k, v, kv_lengths=lengths, return_lse=True)
        return A.cross_attention_backward(do, q, k, v, out, lse, kv_lengths=lengths)

    step()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    do.copy_(normal(do.shape, torch.bfloat16, 9))
    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    with torch.cuda.stream(streams[0]):
        eager = step()
    torch.cuda.synchronize()
    for got in (*outs, eager):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    stride, t, s = (1 << 32) + 256, 150, 100
    buf = torch.zeros(stride + 200 * 512, dtype=torch.bfloat16, device="cuda")
    k = buf.as_strided((2, t, 2, 128), (stride, 256, 128, 1))
    k.copy_(normal((2, t, 2, 128), torch.bfloat16, 1))
    q, do = normal((2, s, 4, 128), torch.bfloat16, 2), normal((2, s, 4, 128), torch.bfloat16, 3)
    out, lse = A.cross_attention(q, k, k, return_lse=True)
    kc = k.contiguous()
    want = A.cross_attention_backward(do, q, kc, kc, out, lse)
    got = A.cross_attention_backward(do, q, k, k, out, lse)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    A.cross_attention_backward(do, q, kc, kc, out, lse, dv=k)
    assert torch.equal(k, want[2])
