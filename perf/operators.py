"""Cases of the operators around attention: rotary positions, per-head norms of queries and keys with the rotation in
the same pass (both with their gradients), and attention to the states of another sequence (forward, its form for
single tokens, gradients).

``run`` computes either the plain torch form (``own`` false) or calls ``pyasc_b200.attention`` (``own`` true).
Tensors are [batch, sequence, heads, head_dim]; queries and keys that get rotated are slices of one packed projection,
as a model has them.
"""
import math

import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# --------------------------------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------------------------------
def _rotary(name, op, batch, seq, heads, kv_heads, head_dim, rotated, interleaved, dtype, first=0, stretch=1.0):
    case = {"op": op, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "rotated": rotated, "interleaved": interleaved, "dtype": dtype, "first": first, "stretch": stretch}
    return dict(case, name=name) if name else case


def _cross(name, op, batch, seq, kv_seq, heads, kv_heads, head_dim, dtype, ragged, lse=False):
    case = {"op": op, "batch": batch, "seq": seq, "kv_seq": kv_seq, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "ragged": ragged, "lse": lse}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one generated token of one conversation: nothing but latency
        _rotary("rotary_token", "rotary", 1, 1, 32, 8, 128, 128, False, "bfloat16", first=2047),
        # prompts of a model that turns half of each head, adjacent pairs, an odd length
        _rotary("rotary_part_interleaved", "rotary", 3, 1021, 16, 16, 128, 64, True, "float16"),
        # a long document far into a stretched context
        _rotary("rotary_long", "rotary", 1, 16384, 32, 8, 128, 128, False, "bfloat16", first=1000000, stretch=8.0),
        # one token for each of many conversations
        _rotary("norm_rotary_tokens", "norm_rotary", 64, 1, 32, 8, 128, 128, False, "bfloat16", first=4095),
        # a training batch's queries and keys, and their gradients
        _rotary("norm_rotary_batch", "norm_rotary", 4, 4096, 32, 8, 128, 128, False, "bfloat16"),
        _rotary("norm_rotary_gradient", "norm_rotary_gradient", 2, 4095, 16, 4, 128, 128, False, "bfloat16"),
        # a decoder's token against the encoder's states of a few requests, padded to the longest
        _cross("cross_token", "cross", 8, 1, 1500, 32, 8, 128, "bfloat16", True),
        # the same against long documents
        _cross("cross_token_long", "cross", 16, 1, 8192, 32, 8, 128, "float16", False),
        # decoder prompts against padded encoder states, small heads, log-sum-exp kept for training
        _cross("cross_ragged", "cross", 4, 448, 1500, 20, 20, 64, "float16", True, lse=True),
        # as many queries as keys, at the sizes of the self-attention workload
        _cross("cross_full", "cross", 4, 4096, 4096, 32, 32, 128, "bfloat16", False),
        # gradients: an odd number of queries against a short text
        _cross("cross_gradient_short", "cross_gradient", 2, 333, 77, 16, 16, 64, "bfloat16", True),
        # gradients of grouped heads at training size
        _cross("cross_gradient", "cross_gradient", 2, 2048, 4096, 32, 8, 128, "bfloat16", False),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "norm_rotary", "norm_rotary_gradient", "cross", "cross_gradient"])
    most = [work(case) for case in listed() if case["op"] == op]
    while True:
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
        dtype = rng.choice(["float16", "bfloat16"])
        if op.startswith("cross"):
            seq = 1 if op == "cross" and rng.random() < 0.35 else _log_int(rng, 1, 5000)
            case = _cross(None, op, _log_int(rng, 1, 32), seq, _log_int(rng, 1, 20000), heads, kv_heads,
                          rng.choice([64, 80, 96, 128, 128]), dtype, rng.random() < 0.5,
                          lse=op == "cross" and rng.random() < 0.5)
        else:
            head_dim = rng.choice([64, 80, 96, 128, 128, 256])
            case = _rotary(None, op, _log_int(rng, 1, 64), _log_int(rng, 1, 20000), heads, kv_heads, head_dim,
                           rng.choice([head_dim, head_dim, head_dim // 2]), rng.random() < 0.5,
                           rng.choice([dtype, dtype, "float32"]), first=rng.choice([0, 1000, _log_int(rng, 1, 1000000)]),
                           stretch=rng.choice([1.0, 4.0]))
        if heads <= 64 and all(work(case)[k] <= max(w[k] for w in most) for k in ("bytes", "flops")):
            return case


def _lengths(case):
    """Keys of each batch entry: all of them, or from the longest down to half of it."""
    b, n = case["batch"], case["kv_seq"]
    return [n - (i * n) // (2 * b) if case["ragged"] else n for i in range(b)]


def work(case):
    size = _DTYPES[case["dtype"]].itemsize
    b, s, h, hk, d = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "head_dim"))
    if not case["op"].startswith("cross"):
        n = b * s * (h + hk) * d
        tensors = 3 if case["op"].endswith("gradient") else 2
        gammas = 0 if case["op"] == "rotary" else 2 * d * (size if tensors == 2 else size + 4)
        return {"bytes": tensors * n * size + 8 * b * s + 4 * case["rotated"] + gammas,
                "flops": n * {"rotary": 3, "norm_rotary": 7, "norm_rotary_gradient": 16}[case["op"]]}
    keys = sum(_lengths(case))
    queries, states, lse = b * s * h * d * size, keys * hk * d * size, 4 * b * s * h
    products = h * s * keys * d * 2
    if case["op"] == "cross":
        return {"bytes": 2 * queries + 2 * states + (lse if case["lse"] else 0), "flops": 2 * products}
    written = 2 * b * case["kv_seq"] * hk * d * size        # gradients of padded keys are written too, as zeros
    return {"bytes": 4 * queries + 2 * states + written + lse, "flops": 5 * products}


# --------------------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------------------
def _frequencies(case):
    i = torch.arange(0, case["rotated"], 2, dtype=torch.float64)
    return 10000.0 ** (-i / case["rotated"]) / case["stretch"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    b, s, h, hk, d = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "head_dim"))

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    if not case["op"].startswith("cross"):
        packed = normal(b, s, (h + 2 * hk) * d)         # queries, keys and values of one projection
        shift = torch.randint(0, 64, (b, 1), generator=g, device="cuda")
        state = {"op": case["op"], "interleaved": case["interleaved"],
                 "q": packed[..., :h * d].unflatten(-1, (h, d)),
                 "k": packed[..., h * d:(h + hk) * d].unflatten(-1, (hk, d)),
                 "positions": case["first"] + shift + torch.arange(s, device="cuda"),
                 "frequencies": _frequencies(case).cuda(),
                 "scale": 1.0 + 0.1 * math.log(case["stretch"]), "eps": 1e-6}
        if case["op"] != "rotary":
            state["q_gamma"] = (1 + 0.2 * normal(d).float()).to(dtype)
            state["k_gamma"] = (1 + 0.2 * normal(d).float()).to(dtype)
        if case["op"].endswith("gradient"):
            state["dq"], state["dk"] = normal(b, s, h, d), normal(b, s, hk, d)
        return state

    n = case["kv_seq"]
    packed = normal(b, n, 2, hk, d)                     # keys and values of one projection of the other sequence
    state = {"op": case["op"], "lse": case["lse"], "scale": d ** -0.5,
             "q": normal(b, s, h, d), "k": packed[:, :, 0], "v": packed[:, :, 1], "lengths": None}
    if case["ragged"]:
        lengths = torch.tensor(_lengths(case), dtype=torch.int32)
        order = torch.randperm(b, generator=torch.Generator().manual_seed(seed))
        state["lengths"] = lengths[order].cuda()
    if case["op"] == "cross_gradient":
        state["out"], state["saved"] = _plain_cross(state["q"], state["k"], state["v"], state["lengths"], state["scale"])
        state["dout"] = normal(b, s, h, d)
    return state


# --------------------------------------------------------------------------------------------------
# Plain forms
# --------------------------------------------------------------------------------------------------
def _angles(state, dtype):
    a = state["positions"].double()[..., None, None] * state["frequencies"]       # far positions: 64 bits
    return (a.cos() * state["scale"]).to(dtype), (a.sin() * state["scale"]).to(dtype)


def _turn(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., r:]], -1)
    a, b = x[..., :r // 2], x[..., r // 2:r]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)


def _plain_rotary(x, gamma, state, cos, sin):
    y = x.float()
    if gamma is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + state["eps"]) * gamma.float()
    return _turn(y, cos, sin, state["interleaved"]).to(x.dtype)


def _plain_rotary_gradient(dy, x, gamma, state, cos, sin):
    y, dn = x.float(), _turn(dy.float(), cos, -sin, state["interleaved"])
    rstd = torch.rsqrt((y * y).mean(-1, keepdim=True) + state["eps"])
    t = dn * gamma.float()
    dx = rstd * t - y * (rstd ** 3 * (y * t).mean(-1, keepdim=True))
    return dx.to(x.dtype), (y * rstd * dn).double().sum((0, 1, 2)).float()


def _grouped(x, heads):
    """[B, S, Hk, D] as [B, H, S, D] in 32 bits, each head of the states once for every head of its group."""
    return x.float().transpose(1, 2).repeat_interleave(heads // x.shape[2], 1)


def _masked(scores, lengths):
    if lengths is None:
        return scores
    keys = torch.arange(scores.shape[-1], device=scores.device)
    return scores.masked_fill(keys >= lengths[:, None, None, None], -math.inf)


def _plain_cross(q, k, v, lengths, scale):
    scores = _masked((_grouped(q, q.shape[2]) @ _grouped(k, q.shape[2]).transpose(-1, -2)).mul_(scale), lengths)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)                   # a row without keys
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ _grouped(v, q.shape[2])) / torch.where(total == 0, 1.0, total)
    return out.transpose(1, 2).contiguous().to(q.dtype), (top + total.log())[..., 0]


def _plain_cross_gradient(state):
    q, k, v, scale = state["q"], state["k"], state["v"], state["scale"]
    h, hk = q.shape[2], k.shape[2]
    qs, ks, vs, dos = (_grouped(x, h) for x in (q, k, v, state["dout"]))
    p = _masked((qs @ ks.transpose(-1, -2)).mul_(scale), state["lengths"])
    lse = state["saved"][..., None]
    p = p.sub_(torch.where(lse == -math.inf, 0.0, lse)).exp_()
    dv = p.transpose(-1, -2) @ dos
    ds = dos @ vs.transpose(-1, -2)
    ds = ds.sub_((dos * _grouped(state["out"], h)).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = ds @ ks, ds.transpose(-1, -2) @ qs

    def summed(x):
        return x.unflatten(1, (hk, h // hk)).sum(2).transpose(1, 2).contiguous().to(k.dtype)

    return dq.transpose(1, 2).contiguous().to(q.dtype), summed(dk), summed(dv)


# --------------------------------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if own:
        from pyasc_b200 import attention
        if op == "cross":
            return attention.cross_attention(state["q"], state["k"], state["v"], kv_lengths=state["lengths"],
                                             scale=state["scale"], return_lse=state["lse"])
        if op == "cross_gradient":
            return attention.cross_attention_backward(state["dout"], state["q"], state["k"], state["v"], state["out"],
                                                      state["saved"], kv_lengths=state["lengths"], scale=state["scale"])
        options = {"scale": state["scale"], "interleaved": state["interleaved"]}
        if op == "rotary":
            return attention.rotary(state["q"], state["k"], state["positions"], state["frequencies"], **options)
        if op == "norm_rotary":
            return attention.norm_rotary(state["q"], state["k"], state["q_gamma"], state["k_gamma"],
                                         state["positions"], state["frequencies"], eps=state["eps"], **options)
        return attention.norm_rotary_backward(state["dq"], state["dk"], state["q"], state["k"], state["q_gamma"],
                                              state["k_gamma"], state["positions"], state["frequencies"],
                                              eps=state["eps"], **options)
    if op == "cross":
        out, lse = _plain_cross(state["q"], state["k"], state["v"], state["lengths"], state["scale"])
        return (out, lse) if state["lse"] else out
    if op == "cross_gradient":
        return _plain_cross_gradient(state)
    cos, sin = _angles(state, torch.float32)
    if op == "norm_rotary_gradient":
        dq, dq_gamma = _plain_rotary_gradient(state["dq"], state["q"], state["q_gamma"], state, cos, sin)
        dk, dk_gamma = _plain_rotary_gradient(state["dk"], state["k"], state["k_gamma"], state, cos, sin)
        return dq, dk, dq_gamma, dk_gamma
    return (_plain_rotary(state["q"], state.get("q_gamma"), state, cos, sin),
            _plain_rotary(state["k"], state.get("k_gamma"), state, cos, sin))


# --------------------------------------------------------------------------------------------------
# The definition in 64 bits
# --------------------------------------------------------------------------------------------------
def _exact_rotation(case, state):
    """cos + i sin of every token's pairs, times the scale: [B, S, 1, r/2] complex."""
    angle = torch.einsum("bs,f->bsf", state["positions"].double(), state["frequencies"].double())
    return torch.polar(torch.full_like(angle, state["scale"]), angle)[:, :, None]


def _exact_turn(x, rotation, interleaved):
    r = 2 * rotation.shape[-1]
    head, rest = x[..., :r], x[..., r:]
    if interleaved:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], r // 2, 2)) * rotation
        turned = torch.view_as_real(z).reshape(head.shape)
    else:
        z = torch.complex(*head.chunk(2, -1)) * rotation
        turned = torch.cat([z.real, z.imag], -1)
    return torch.cat([turned, rest], -1)


def _exact_rotary(case, state):
    rotation = _exact_rotation(case, state)
    results, gammas = [], []
    for name in ("q", "k"):
        x = state[name].double().contiguous()
        if case["op"] == "rotary":
            results.append(_exact_turn(x, rotation, case["interleaved"]))
            continue
        gamma = state[name + "_gamma"].double()
        unit = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + state["eps"]).sqrt()
        if case["op"] == "norm_rotary":
            results.append(_exact_turn(unit * gamma, rotation, case["interleaved"]))
            continue
        back = _exact_turn(state["d" + name].double(), rotation.conj(), case["interleaved"])
        norm = (x.square().sum(-1, keepdim=True) / x.shape[-1] + state["eps"]).sqrt()
        along = (unit * back * gamma).sum(-1, keepdim=True) / x.shape[-1]
        results.append((back * gamma - unit * along) / norm)
        gammas.append((unit * back).flatten(0, 2).sum(0))
    return tuple(results + gammas)


def _exact_cross(case, state):
    b, s, h, d = state["q"].shape
    n, hk = state["k"].shape[1:3]
    lengths = [n] * b if state["lengths"] is None else state["lengths"].tolist()
    kind = {"dtype": torch.float64, "device": "cuda"}
    out, lse = torch.zeros(b, s, h, d, **kind), torch.full((b, h, s), -math.inf, **kind)
    dq, dk, dv = torch.zeros(b, s, h, d, **kind), torch.zeros(b, n, hk, d, **kind), torch.zeros(b, n, hk, d, **kind)
    for i in range(b):
        for j in range(h):
            t, m = lengths[i], j // (h // hk)
            if t == 0:
                continue
            q, k, v = state["q"][i, :, j].double(), state["k"][i, :t, m].double(), state["v"][i, :t, m].double()
            scores = torch.einsum("sd,td->st", q, k) * state["scale"]
            lse[i, j] = torch.logsumexp(scores, -1)
            p = torch.softmax(scores, -1)
            out[i, :, j] = torch.einsum("st,td->sd", p, v)
            if case["op"] == "cross_gradient":
                do = state["dout"][i, :, j].double()
                dp = torch.einsum("sd,td->st", do, v)
                ds = (dp - (dp * p).sum(-1, keepdim=True)) * p * state["scale"]
                dq[i, :, j] = torch.einsum("st,td->sd", ds, k)
                dk[i, :t, m] += torch.einsum("st,sd->td", ds, q)
                dv[i, :t, m] += torch.einsum("st,sd->td", p, do)
    if case["op"] == "cross_gradient":
        return dq, dk, dv
    return (out, lse) if case["lse"] else out


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_cross(case, state) if case["op"].startswith("cross") else _exact_rotary(case, state)
