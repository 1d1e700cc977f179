"""Attention to another sequence (pyasc_b200/attention.py) against its definition in 64 bits.

Tolerances.  With u half a step of the 16-bit type and |V| the largest value an output can be made of: P is rounded to
the type (u of each p, so u sum p |v| in all), the output once more (u |o|), and fp32 work on scores, exponentials and
sums stays below 2^-13 of sum p |v| at these sizes (a score of magnitude s is off by about (8 + |s|) 2^-22 from the
products' truncation and the exponent's scaling, |s| < 40, twice for numerator and sum).  lse: the score's error,
2^-15 + 2^-20 |lse|.
"""
import math

import pytest
import torch

from oracle import transformer as R
from pyasc_b200 import attention as A
from pyasc_b200 import capi

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=gen(seed), device="cuda").to(dtype)


def check(q, k, v, lengths=None, scale=None, **kw):
    got, lse = A.cross_attention(q, k, v, kv_lengths=lengths, scale=scale, return_lse=True, **kw)
    capi.check_device_status(None)
    want, want_lse = R.cross_attention(q, k, v, lengths, scale)
    size, _ = R.cross_attention(q, k, R._clean(v, lengths).abs(), lengths, scale)
    u = torch.finfo(q.dtype).eps / 2
    bound = (u + 2.0**-13) * size + u * want.abs() * 1.01 + (2.0**-24 if q.dtype == torch.float16 else 1e-38)
    off = (got.double() - want).abs()
    assert got.shape == q.shape and got.dtype == q.dtype and torch.isfinite(got).all()
    assert (off <= bound).all(), f"{(off / bound).max().item():.3g} times the bound"
    empty = want_lse == -math.inf
    assert torch.equal(empty, lse == -math.inf)
    off = torch.where(empty, 0.0, (lse.double() - want_lse).abs())
    bound = torch.where(empty, 1.0, 2.0**-15 + 2.0**-20 * want_lse.abs())
    assert (off <= bound).all(), f"lse {(off / bound).max().item():.3g} times the bound"
    assert (got.transpose(1, 2)[empty] == 0).all()
    return got, lse


SIZES = [
    # B, S, T, Hq, Hkv, D
    (1, 1, 1, 1, 1, 128),
    (1, 1, 128, 4, 1, 64),
    (2, 1, 1500, 8, 2, 128),
    (1, 1, 9000, 6, 1, 128),
    (3, 5, 77, 4, 4, 64),
    (2, 7, 129, 12, 2, 80),
    (1, 16, 1000, 20, 1, 96),
    (1, 33, 500, 9, 3, 128),
    (1, 64, 300, 6, 2, 64),
    (2, 65, 300, 6, 2, 128),
    (1, 128, 128, 2, 2, 128),
    (1, 129, 255, 2, 1, 72),
    (2, 333, 77, 3, 3, 40),
    (1, 700, 1025, 4, 2, 128),
    (2, 513, 640, 4, 4, 64),
    (1, 300, 1, 2, 2, 8),
    (1, 1, 700, 64, 1, 128),
    (2, 3, 130, 17, 1, 64),
    (60, 256, 200, 4, 4, 64),
    (40, 3, 513, 8, 8, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b, s, t, h, hk, d", SIZES)
def test_forward(b, s, t, h, hk, d, dtype):
    q, packed = normal((b, s, h, d), dtype, 1), normal((b, t, 2, hk, d), dtype, 2)
    check(q, packed[:, :, 0], packed[:, :, 1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("s", [1, 20, 200])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("fill", [0.0, float("nan"), float("inf"), -65504.0])
def test_lengths(s, d, fill, dtype):
    """Lengths of zero, one, around tile borders and the whole; padding that holds anything."""
    t = 700
    lengths = torch.tensor([0, 1, 127, 128, 129, 400, 699, 700, 5], dtype=torch.int32, device="cuda")
    b = lengths.numel()
    q, k, v = normal((b, s, 4, d), dtype, 1), normal((b, t, 2, d), dtype, 2), normal((b, t, 2, d), dtype, 3)
    want = check(q, k, v, lengths)
    gone = torch.arange(t, device="cuda")[None] >= lengths[:, None]
    k[gone], v[gone] = fill, fill
    got = check(q, k, v, lengths)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wild = lengths.clone()
    wild[0], wild[7] = -3, 1 << 30                       # clamped to 0 and to all
    assert torch.equal(A.cross_attention(q, k, v, kv_lengths=wild), got[0])


def test_all_lengths_of_one_tile():
    t = 128
    lengths = torch.arange(t + 1, dtype=torch.int32, device="cuda")
    b = t + 1
    q, k, v = (normal((b, n, 2, 64), torch.bfloat16, n) for n in (9, t, t + 0))
    k[torch.arange(t, device="cuda")[None] >= lengths[:, None]] = float("nan")
    v = normal((b, t, 2, 64), torch.bfloat16, 3)
    v[torch.arange(t, device="cuda")[None] >= lengths[:, None]] = float("nan")
    check(q, k, v, lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_scores_and_moving_maximum(dtype):
    """Keys in rising order make the running maximum move in every tile."""
    t, d = 2000, 64
    q = torch.ones(1, 140, 2, d, device="cuda", dtype=dtype)
    k = (torch.linspace(-4, 4, t, device="cuda")[None, :, None, None].expand(1, t, 2, d)).to(dtype).contiguous()
    v = normal((1, t, 2, d), dtype, 1)
    check(q, k, v)
    check(q, k.flip(1), v, torch.tensor([1999], dtype=torch.int32, device="cuda"))
    check(q, k, v, scale=0.0)


@pytest.mark.parametrize("s", [1, 130])
def test_layouts(s):
    b, t, h, hk, d, dt = 2, 300, 4, 2, 64, torch.bfloat16
    q, k, v = normal((b, s, h, d), dt, 1), normal((b, t, hk, d), dt, 2), normal((b, t, hk, d), dt, 3)
    want = A.cross_attention(q, k, v)

    def transposed(x):
        return x.transpose(1, 2).contiguous().transpose(1, 2)

    out = torch.full((b, s + 1, h, d + 8), 7.0, dtype=dt, device="cuda")
    got = A.cross_attention(transposed(q), transposed(k), v.transpose(0, 1).contiguous().transpose(0, 1),
                            out=out[:, :s, :, :d])
    assert torch.equal(got, want) and got.data_ptr() == out.data_ptr()
    inner = out[:, :s, :, :d].clone()
    out[:, :s, :, :d] = 7.0
    assert (out == 7).all() and torch.equal(inner, want)         # nothing outside the view
    # one state for the whole batch, one head for all
    got = A.cross_attention(q, k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1))
    assert torch.equal(got, A.cross_attention(q, k[:1].repeat(b, 1, 1, 1), v[:1].repeat(b, 1, 1, 1)))
    got = A.cross_attention(q, k[:, :, :1].expand(-1, -1, hk, -1), v)
    assert torch.equal(got, A.cross_attention(q, k[:, :, :1].repeat(1, 1, hk, 1), v))


def test_empty():
    def z(*shape):
        return torch.randn(shape, device="cuda", dtype=torch.float32).half()

    assert A.cross_attention(z(0, 3, 2, 64), z(0, 5, 2, 64), z(0, 5, 2, 64)).shape == (0, 3, 2, 64)
    assert A.cross_attention(z(2, 0, 2, 64), z(2, 5, 2, 64), z(2, 5, 2, 64)).shape == (2, 0, 2, 64)
    for s in (1, 200):
        out, lse = A.cross_attention(z(2, s, 2, 64), z(2, 0, 2, 64), z(2, 0, 2, 64), return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
        lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
        out, lse = A.cross_attention(z(2, s, 2, 64), z(2, 900, 2, 64), z(2, 900, 2, 64), kv_lengths=lengths, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_refusals():
    q, k = (torch.zeros(2, 4, n, 64, dtype=torch.float16, device="cuda") for n in (4, 2))
    bad = [
        (ValueError, (q, k[:, :, :1].expand(-1, -1, 3, -1).contiguous(), k), {}),
        (ValueError, (q, k[:1], k[:1]), {}),
        (ValueError, (q, k, k[:, :3]), {}),
        (TypeError, (q, k.bfloat16(), k), {}),
        (TypeError, (q.float(), k.float(), k.float()), {}),
        (ValueError, (q, k.cpu(), k), {}),
        (ValueError, (q[0], k, k), {}),
        (ValueError, (q.transpose(2, 3).contiguous().transpose(2, 3), k, k), {}),
        (TypeError, (q, k, k), {"kv_lengths": torch.zeros(2, dtype=torch.int64, device="cuda")}),
        (ValueError, (q, k, k), {"kv_lengths": torch.zeros(3, dtype=torch.int32, device="cuda")}),
        (ValueError, (q, k, k), {"out": q[:1].expand(2, -1, -1, -1)}),
        (RuntimeError, (q, k, k), {"scale": -1.0}),
        (RuntimeError, (q, k, k), {"scale": float("nan")}),
        (RuntimeError, (q[..., :60], k[..., :60], k[..., :60]), {}),                      # head size not a multiple of 8
        (RuntimeError, tuple(x.repeat(1, 1, 1, 3) for x in (q, k, k)), {}),               # beyond 128
    ]
    flat = torch.zeros(2 * 4 * 4 * 64 + 1, dtype=torch.float16, device="cuda")
    bad.append((RuntimeError, (flat[1:].view(2, 4, 4, 64), k, k), {}))                    # not 16-byte aligned
    for error, args, kwargs in bad:
        with pytest.raises(error):
            A.cross_attention(*args, **kwargs)


@pytest.mark.parametrize("s", [1, 140])
def test_streams_and_graphs(s):
    q, k, v = (normal((2, n, 2, 128), torch.bfloat16, n) for n in (s, 2901, 2901))
    lengths = torch.tensor([2901, 77], dtype=torch.int32, device="cuda")
    graphs, outs = [], []
    A.cross_attention(q, k, v, kv_lengths=lengths)
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(A.cross_attention(q, k, v, kv_lengths=lengths))
        graphs.append(graph)
    q.copy_(normal(q.shape, torch.bfloat16, 5))
    lengths.copy_(torch.tensor([5, 2899], dtype=torch.int32))
    want = A.cross_attention(q, k, v, kv_lengths=lengths)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        with torch.cuda.stream(streams[0]):              # an eager call beside the replays
            eager = A.cross_attention(q, k, v, kv_lengths=lengths)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in (*outs, eager))


def test_offsets_past_32_bits():
    stride = (1 << 32) + 256
    t = 300
    buf = torch.empty(stride + t * 256, dtype=torch.bfloat16, device="cuda")
    k = buf.as_strided((2, t, 2, 128), (stride, 256, 128, 1))
    k.copy_(normal((2, t, 2, 128), torch.bfloat16, 1))
    for s in (1, 130):
        q = normal((2, s, 4, 128), torch.bfloat16, 2)
        assert torch.equal(A.cross_attention(q, k, k), A.cross_attention(q, k.contiguous(), k.contiguous()))
        out = buf.as_strided((2, s, 4, 128), (stride, 512, 128, 1))
        want = A.cross_attention(q, k.contiguous(), k.contiguous())
        kept = k.contiguous()
        assert torch.equal(A.cross_attention(q, kept, kept, out=out), want)
        k.copy_(kept)


def test_agrees_with_self_attention():
    """Full attention through the contiguous [B, H, S, D] entry point is the same computation."""
    b, h, s, d = 2, 3, 256, 128
    q, k, v = (normal((b, h, s, d), torch.float16, i) for i in range(3))
    o = torch.empty_like(q)
    capi.call("asc_cuda_attn_fwd_f16", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), b, h, s, d, d**-0.5, 0, 0,
              torch.cuda.current_stream().cuda_stream)
    got = A.cross_attention(*(x.transpose(1, 2) for x in (q, k, v)))
    torch.testing.assert_close(got.transpose(1, 2), o, atol=2e-3, rtol=2e-3)
