"""Attention of a decoder's queries to an encoder's states, ``softmax(scale * Q K^T) V``, per query tile.

The script of self-attention (flash_attention.py) with two lengths and two numbers of heads: ``heads`` sequences of queries
read ``kv_heads`` sequences of keys and values, ``heads / kv_heads`` of them in a row the same one.  The platform runs it as
one call of ``asc_cuda_cross_attn_fwd_f16``; padded states, strided tensors, the log-sum-exp and the gradients are reached
through :mod:`pyasc_b200.attention`."""
import asc
import asc2


@asc2.jit
def cross_attention_kernel(q_ptr: asc.GlobalAddress, k_ptr: asc.GlobalAddress, v_ptr: asc.GlobalAddress,
                           o_ptr: asc.GlobalAddress, scale: float, heads: asc.ConstExpr[int], kv_heads: asc.ConstExpr[int],
                           q_seq: asc.ConstExpr[int], kv_seq: asc.ConstExpr[int], head_dim: asc.ConstExpr[int],
                           q_tile: asc.ConstExpr[int], dtype: asc.ConstExpr):
    q_gm = asc2.tensor(q_ptr, [heads * q_seq, head_dim])
    k_gm = asc2.tensor(k_ptr, [kv_heads * kv_seq, head_dim])
    v_gm = asc2.tensor(v_ptr, [kv_heads * kv_seq, head_dim])
    o_gm = asc2.tensor(o_ptr, [heads * q_seq, head_dim])
    tiles_per_head = q_seq // q_tile
    group = heads // kv_heads
    for t in range(asc2.block_idx(), heads * tiles_per_head, asc2.block_num()):
        head = t // tiles_per_head
        q_row = head * q_seq + (t % tiles_per_head) * q_tile
        kv_row = (head // group) * kv_seq
        q = asc2.load(q_gm, [q_tile, head_dim], offsets=[q_row, 0], location=asc2.TileLocation.L0A)
        k = asc2.load(k_gm, [kv_seq, head_dim], offsets=[kv_row, 0], location=asc2.TileLocation.L0B)
        v = asc2.load(v_gm, [kv_seq, head_dim], offsets=[kv_row, 0], location=asc2.TileLocation.L0B)
        p = asc2.softmax(asc2.matmul(q, k, trans_b=True) * scale).to(dtype)
        asc2.store(asc2.matmul(p, v).to(dtype), o_gm, offsets=[q_row, 0])


_ASC_DTYPE = {"float16": asc.float16, "bfloat16": asc.bfloat16}


def cross_attention_launch(q, k, v, o, scale=None, core_num: int = 148, q_tile: int = 128, stream=None):
    """q, o: contiguous [batch, heads, q_seq, head_dim], k, v: [batch, kv_heads, kv_seq, head_dim] fp16 / bf16 tensors; o is
    written in place."""
    batch, heads, q_seq, head_dim = q.shape
    kv_heads, kv_seq = k.shape[1], k.shape[2]
    if scale is None:
        scale = float(head_dim) ** -0.5
    q_tile = min(q_tile, q_seq)
    while q_seq % q_tile:
        q_tile -= 1
    dtype = _ASC_DTYPE[str(q.dtype).replace("torch.", "")]
    launch = cross_attention_kernel[core_num] if stream is None else cross_attention_kernel[core_num, stream]
    launch(q, k, v, o, float(scale), batch * heads, batch * kv_heads, q_seq, kv_seq, head_dim, q_tile, dtype)
    return o
