"""The asc2 form of attention to another sequence: what the planner makes of it, and what it refuses."""
import asc
import asc2
import pytest
import torch

from pyasc_b200 import tutorials as T


@pytest.fixture(autouse=True)
def dry_run(monkeypatch):
    monkeypatch.setenv("DRY_RUN", "1")


def empty(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b, h, hk, s, t, d", [(2, 4, 4, 256, 77, 128), (1, 8, 2, 100, 300, 64), (3, 2, 1, 1, 1000, 80),
                                               (2, 3, 3, 128, 128, 64)])
def test_plan(b, h, hk, s, t, d, dtype):
    T.cross_attention_launch(empty(b, h, s, d, dtype=dtype), empty(b, hk, t, d, dtype=dtype), empty(b, hk, t, d, dtype=dtype),
                             empty(b, h, s, d, dtype=dtype), core_num=5)
    plan = T.cross_attention_kernel.last_plan
    assert [step.fn_name for step in plan.steps] == ["asc_cuda_cross_attn_fwd_f16"]
    assert plan.steps[0].note == f"{b * hk} sequences x {h // hk * s} queries x {t} keys x {d}"
    assert plan.reads == {0, 1, 2} and plan.writes == {3} and not plan.partial_writes
    assert plan.pipeline.streamed == {0: h // hk * s * d * 2, 1: t * d * 2, 2: t * d * 2, 3: h // hk * s * d * 2}


def test_self_attention_keeps_its_kernel():
    T.cross_attention_launch(empty(2, 3, 256, 128), empty(2, 3, 256, 128), empty(2, 3, 256, 128), empty(2, 3, 256, 128))
    assert [s.fn_name for s in T.cross_attention_kernel.last_plan.steps] == ["asc_cuda_attn_fwd_f16"]


def script(q_rows, k_rows, head_dim, kv_of, out="o", causal=False):
    @asc2.jit
    def attn(q_ptr: asc.GlobalAddress, k_ptr: asc.GlobalAddress, v_ptr: asc.GlobalAddress, o_ptr: asc.GlobalAddress):
        gm = {"q": asc2.tensor(q_ptr, [q_rows, head_dim]), "k": asc2.tensor(k_ptr, [k_rows, head_dim]),
              "v": asc2.tensor(v_ptr, [k_rows, head_dim]), "o": asc2.tensor(o_ptr, [q_rows, head_dim])}
        for t in range(asc2.block_idx(), q_rows // 64, asc2.block_num()):
            q = asc2.load(gm["q"], [64, head_dim], offsets=[t * 64, 0])
            k = asc2.load(gm["k"], [100, head_dim], offsets=[kv_of(t), 0])
            v = asc2.load(gm["v"], [100, head_dim], offsets=[kv_of(t), 0])
            s = asc2.matmul(q, k, trans_b=True) * 0.125
            if causal:
                s = asc2.causal_mask(s, 0, 0)
            asc2.store(asc2.matmul(asc2.softmax(s).to(asc.float16), v).to(asc.float16), gm[out], offsets=[t * 64, 0])

    attn[4](empty(q_rows, head_dim), empty(k_rows, head_dim), empty(k_rows, head_dim), empty(q_rows, head_dim))
    return attn


def test_refusals():
    assert script(256, 200, 64, lambda t: (t // 2) * 100).last_plan.pattern == "attention"
    for bad in (
            lambda: script(256, 200, 64, lambda t: (t % 2) * 100),   # keys of another head
            lambda: script(256, 200, 64, lambda t: (t // 2) * 100, causal=True),
            lambda: script(256, 300, 64, lambda t: 0),                                     # 256 queries over 3 sequences
            lambda: script(256, 200, 144, lambda t: (t // 2) * 100),
            lambda: script(256, 250, 64, lambda t: 0),
    ):
        with pytest.raises(NotImplementedError):
            bad()
    with pytest.raises((NotImplementedError, RuntimeError)):
        script(200, 200, 64, lambda t: (t // 2) * 100, out="k")
