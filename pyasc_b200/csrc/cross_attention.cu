// Attention of queries to another sequence's keys and values (fp16 / bf16, head sizes up to 128), forward, for sm_100a:
//   S = scale Q K^T,  keys from the length of their batch entry on are not there,  P = softmax(S),  O = P V,
//   lse = log sum exp S (natural logarithm);  a query without any key: O = 0, lse = -inf.
//
// One pass over the keys with a running maximum and sum per query row, fp32; P is rounded to the inputs' type for the
// second product, as half-precision attention does.  Tensor-core bound for many query rows (4 Sq Skv D flops against
// (2 Sq + 2 Skv) D values), HBM-bound on K and V for single tokens.
//
// A tile is 128 query rows of one (batch, key head): 128 consecutive queries of one head, or, when queries are few, all
// queries of several heads of the group, so that a group's heads read their keys once (TMA box {64, seg, pack, 1}).  An
// item is a pair of tiles over all keys.  Where whole items would leave SMs idle some are cut along the keys
// (attention_schedule.cuh): a part writes its unnormalised fp32 sum, maximum and total to a workspace, and a second
// kernel joins the parts in order.
//   warps 0-3   softmax of tile 0, one thread per row: scores from tensor memory, P back into the same columns,
//   warps 4-7   (same for tile 1)  lazy rescaling of the accumulator, epilogue
//   warp 8      TMA producer: Q tiles, K and V tiles through two rings of kStages 128B-swizzled stages
//   warp 9      MMA issuer: S = Q K^T, O += P V (P from tensor memory), accumulators S0 S1 O0 O1 in tensor memory
// Head sizes that are not 64 or 128 are padded by the tensor maps (columns past D read as zero).  All waits are bounded.
//
// Up to 16 query rows per key head (single tokens, with the heads of a group) have nothing to fill such tiles with, and
// the chain scores - softmax - product of a 128-key step is longer than its keys take to arrive.  They go to a kernel of
// independent warps instead, see cross_few_kernel.
#include "../../include/asc_cuda.h"
#include "attention_common.cuh"
#include "attention_schedule.cuh"
#include "cross_attention.h"
#include "host_common.h"

namespace {

using namespace ascdev;
using namespace asccross;
using ascsched::Range;
using ascsched::Schedule;
using ascsched::Segment;
using ascsched::Walker;

constexpr int kTileQ = 128;    // query rows per tile (= TMEM lanes)
constexpr int kTileKV = 128;   // keys per step
constexpr int kThreads = 384;
constexpr uint32_t kColS = 0;               // S_t at columns [128 t, 128 t + 128); P_t aliases its first 64 columns
constexpr uint32_t kColO = 256;             // O_t at columns [256 + 128 t, ...)
constexpr float kRescaleThreshold = 8.0f;   // in log2 units
constexpr float kLn2 = 0.6931471805599453f;
// Register split after launch, see attention.cu: the increase may only take what the decrease releases.
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(8 * kSoftmaxRegs + 4 * kOtherRegs <= 12 * kLaunchRegs, "register split exceeds the launch allocation");

struct CrossParams {
  void* o;
  float* lse;                // [B, Hq, Sq] contiguous, may be null
  float* part_o;             // parts: [slot][rows of an item][D] unnormalised sums
  float2* part_ml;           // parts: [slot][rows of an item] (maximum in log2 units, total)
  Schedule work;
  int64_t ob, os, oh;        // strides of o in elements
  int32_t B, Sq, Skv, Hkv, group, D;
  int32_t seg, pack;         // rows per head and heads per tile
  int32_t tiles;             // query tiles per (batch, key head)
  int32_t tiles_per_head;    // pack == 1
  int32_t k_heads, k_batches, v_heads, v_batches;   // 0: that dimension of K / V has a stride of 0
  float scale_log2;          // softmax scale * log2(e)
  uint32_t* status;
};

__device__ __forceinline__ bool tile_exists(const CrossParams& p, int tile) { return tile < p.tiles; }

// first head of a tile within its group and first query
__device__ __forceinline__ void tile_origin(const CrossParams& p, int tile, int& head, int& s0) {
  if (p.pack == 1) {
    head = tile / p.tiles_per_head;
    s0 = (tile - head * p.tiles_per_head) * kTileQ;
  } else {
    head = tile * p.pack;
    s0 = 0;
  }
}

// Head and query of a tile's row; false where there is none.
__device__ __forceinline__ bool row_place(const CrossParams& p, const Segment& it, int tile, int row, int& h, int& s) {
  int head0, s0;
  tile_origin(p, tile, head0, s0);
  const int hl = head0 + row / p.seg;
  s = s0 + row % p.seg;
  h = it.hkv * p.group + hl;
  return row < p.seg * p.pack && hl < p.group && s < p.Sq;
}

template <int kStages>
struct CrossCtl {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], p_half[2], p_full[2], o_full[2];
  uint32_t tmem_base;
  uint32_t abort_flag;
};

// Softmax warpgroup of one query tile: one thread per row.
template <bool kBf16, int kHalves, int kTiles, typename Ctl>
__device__ __forceinline__ bool softmax_role(const CrossParams& p, Ctl& ctl, uint32_t tmem_base, int t, const Segment& it,
                                             int tile, uint32_t& s_it, uint32_t& o_it) {
  volatile uint32_t* abort_flag = &ctl.abort_flag;
  const int row = threadIdx.x & 127;            // row inside the tile == TMEM lane
  const uint32_t lane_base = ((threadIdx.x >> 5) & 3) * 32;
  const uint32_t t_s = tmem_base + (lane_base << 16) + kColS + t * 128;
  const uint32_t t_o = tmem_base + (lane_base << 16) + kColO + t * 128;
  const float sl2 = p.scale_log2;
  const int steps = it.n;
  float m_ref = 0.f;  // maximum (raw score units) the exponentials are taken against
  float l = 0.f;      // running sum of exp2((s - m_ref) * sl2)

  int limit = it.len - 1 - it.first * kTileKV;   // columns c <= limit are there (at least one)
  for (int j = 0; j < steps; ++j, limit -= kTileKV) {
    if (!mbar_wait(smem_u32(&ctl.s_full[t]), s_it & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_TMEM_FULL)) return false;
    ++s_it;
    tc_fence_after();
    uint32_t s[4][32];
#pragma unroll
    for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(t_s + c * 32, s[c]);
    tmem_ld_wait();

    if (limit < kTileKV - 1) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (c * 32 + i > limit) s[c][i] = 0xff800000u;  // -inf
    }
    float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      mx0 = max3(mx0, __uint_as_float(s[0][i]), __uint_as_float(s[0][i + 1]));
      mx1 = max3(mx1, __uint_as_float(s[1][i]), __uint_as_float(s[1][i + 1]));
      mx2 = max3(mx2, __uint_as_float(s[2][i]), __uint_as_float(s[2][i + 1]));
      mx3 = max3(mx3, __uint_as_float(s[3][i]), __uint_as_float(s[3][i + 1]));
    }
    const float row_max = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));

    // The reference maximum only moves when the row maximum exceeds it by more than 2^8; until then exponentials may
    // grow up to 256, well inside the range of fp16, bf16 and fp32.
    float alpha = 1.f;
    bool moved = false;
    if (j == 0) {
      m_ref = row_max;
    } else if ((row_max - m_ref) * sl2 > kRescaleThreshold) {
      alpha = ex2_approx((m_ref - row_max) * sl2);
      m_ref = row_max;
      moved = true;
    }
    if (__any_sync(0xffffffffu, moved)) {
      // O_t *= alpha for this thread's row.  The previous P V has retired: its commit is ordered before the commit that
      // published these scores.
      l *= alpha;
#pragma unroll 1
      for (int c = 0; c < 2 * kHalves; ++c) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(t_o + c * 32, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
        tmem_st_32x32b_x32(t_o + c * 32, o);
      }
    }
    const float neg_m = -m_ref * sl2;
    float l0 = 0.f, l1 = 0.f, l2 = 0.f, l3 = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t pk[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1])),
                                    make_float2(sl2, sl2), make_float2(neg_m, neg_m));
        // a quarter on the FMA pipe (measured 872 -> 854 us at [4, 4096, 32, 128]; an eighth or three eighths: less)
        const float2 e = i % 4 == 3 ? exp2_poly(x) : make_float2(ex2_approx(x.x), ex2_approx(x.y));
        const float e0 = e.x, e1 = e.y;
        if (i & 1) {
          const float2 t2 = __fadd2_rn(make_float2(l2, l3), make_float2(e0, e1));
          l2 = t2.x, l3 = t2.y;
        } else {
          const float2 t2 = __fadd2_rn(make_float2(l0, l1), make_float2(e0, e1));
          l0 = t2.x, l1 = t2.y;
        }
        pk[i] = pack2<kBf16>(e0, e1);
      }
      tmem_st_32x32b_x16(t_s + c * 16, pk);
      if (c == 1) {          // the product of the first 64 keys starts while the others are computed (850 -> 839 us)
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&ctl.p_half[t]));
      }
    }
    l += (l0 + l1) + (l2 + l3);
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&ctl.p_full[t]));
  }

  int h, s_row;
  const bool valid = row_place(p, it, tile, row, h, s_row);
  const int64_t flat = (static_cast<int64_t>(it.b) * (p.Hkv * p.group) + h) * p.Sq + s_row;   // [B, Hq, Sq]
  if (steps == 0) {
    if (!valid) return true;
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.o) + it.b * p.ob + s_row * p.os + h * p.oh;
    for (int c = 0; c < p.D; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0, 0, 0, 0);
    if (p.lse != nullptr) p.lse[flat] = -INFINITY;
    return true;
  }
  // ------------------------------ epilogue: O / l -> 16-bit -> global, or the part as it is ------------------------
  if (!mbar_wait(smem_u32(&ctl.o_full[t]), o_it & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_TMEM_FULL)) return false;
  ++o_it;
  tc_fence_after();
  if (it.slot >= 0) {
    const int64_t at = static_cast<int64_t>(it.slot) * (kTiles * kTileQ) + t * kTileQ + row;
    if (valid) p.part_ml[at] = make_float2(m_ref * sl2, l);
    float* dst = p.part_o + at * p.D;
#pragma unroll 1
    for (int c = 0; c < 2 * kHalves; ++c) {
      uint32_t o[32];
      tmem_ld_32x32b_x32(t_o + c * 32, o);
      tmem_ld_wait();
      if (valid) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c * 32 + i * 4 < p.D)
            reinterpret_cast<uint4*>(dst + c * 32)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      }
    }
  } else {
    const float inv = 1.f / l;
    if (valid && p.lse != nullptr) p.lse[flat] = (m_ref * sl2 + log2f(l)) * kLn2;
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.o) + it.b * p.ob + s_row * p.os + h * p.oh;
#pragma unroll 1
    for (int c = 0; c < 2 * kHalves; ++c) {
      uint32_t o[32];
      tmem_ld_32x32b_x32(t_o + c * 32, o);
      tmem_ld_wait();
      if (valid) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          pk[i] = pack2<kBf16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c * 32 + i * 8 < p.D)
            reinterpret_cast<uint4*>(dst + c * 32)[i] = make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
      }
    }
  }
  // O_t has been read: the first P V of the next item may overwrite it.  That MMA is issued only after this thread's
  // next p_full arrival, which follows in program order.
  tc_fence_before();
  return true;
}

// kTiles: query tiles an item holds (1: the second tile's shared memory goes into more stages of K and V)
template <bool kBf16, int kHalves, int kTiles>
__global__ void __launch_bounds__(kThreads, 1)
    cross_fwd_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                     const __grid_constant__ CUtensorMap tmap_v, const CrossParams p, const uint32_t idesc_qk,
                     const uint32_t idesc_pv) {
  constexpr uint32_t kTileBytes = kHalves * kHalfTile;
  constexpr int kStages = kHalves == 1 ? 4 : kTiles == 1 ? 3 : 2;
  constexpr uint32_t kSmemQ = 0, kSmemK = kTiles * kTileBytes, kSmemV = kSmemK + kStages * kTileBytes;
  extern __shared__ uint8_t smem_raw[];
  __shared__ CrossCtl<kStages> ctl;
  __shared__ Range range;
  __shared__ ascsched::Walk walks[8];

  const uint32_t warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  volatile uint32_t* abort_flag = &ctl.abort_flag;

  if (threadIdx.x == 0) {
    ctl.abort_flag = 0;
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctl.q_full[i]), 1);
      mbar_init(smem_u32(&ctl.q_empty[i]), 1);
      mbar_init(smem_u32(&ctl.s_full[i]), 1);
      mbar_init(smem_u32(&ctl.p_half[i]), 4);
      mbar_init(smem_u32(&ctl.p_full[i]), 4);
      mbar_init(smem_u32(&ctl.o_full[i]), 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&ctl.k_full[i]), 1);
      mbar_init(smem_u32(&ctl.k_empty[i]), 1);
      mbar_init(smem_u32(&ctl.v_full[i]), 1);
      mbar_init(smem_u32(&ctl.v_empty[i]), 1);
    }
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(&ctl.tmem_base), 512);
    tmem_relinquish();
  }
  let_next_start();
  if (warp == 10) ascsched::find_range(p.work, blockIdx.x, gridDim.x, &range);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctl.tmem_base;

  // Every role walks the same list of segments, so the use counts of the barriers advance identically in all of them.
  if (warp < 8) {
    setmaxnreg_inc<kSoftmaxRegs>();
    const int t = static_cast<int>(warp >> 2);
    uint32_t s_it = 0, o_it = 0;
    bool ok = t < kTiles;
    ascsched::Walk& walk = walks[warp];
    walk.start(p.work, range, blockIdx.x, gridDim.x);
    const Segment& it = walk.segment;
    while (ok && walk.next(p.work)) {
      const int tile = it.tile * kTiles + t;
      if (tile_exists(p, tile)) ok = softmax_role<kBf16, kHalves, kTiles>(p, ctl, tmem_base, t, it, tile, s_it, o_it);
    }
    if (ok)
      ascsched::for_empty_items(p.work, blockIdx.x, gridDim.x, [&](const Segment& e) {
        const int tile = e.tile * kTiles + t;
        if (tile_exists(p, tile)) softmax_role<kBf16, kHalves, kTiles>(p, ctl, tmem_base, t, e, tile, s_it, o_it);
      });
  } else {
    setmaxnreg_dec<kOtherRegs>();
    if (warp == 8) {
      // ------------------------------ TMA producer ------------------------------
      bool ok = true;
      uint32_t q_it[2] = {0, 0};
      Ring<kStages> k_ring, v_ring;
      const uint32_t q_bytes = static_cast<uint32_t>(p.seg * p.pack) * 128u * kHalves;
      Walker walk(p.work, range, blockIdx.x, gridDim.x);
      Segment it;
      while (ok && walk.next(p.work, it)) {
        if (it.n == 0) continue;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const int tile = it.tile * kTiles + t;
          if (!ok || !tile_exists(p, tile)) continue;
          // the previous item's Q K^T of this tile have retired
          ok = mbar_wait(smem_u32(&ctl.q_empty[t]), (q_it[t] & 1) ^ 1, abort_flag, p.status, ASC_DEV_TIMEOUT_EMPTY);
          if (!ok) continue;
          ++q_it[t];
          if (elect_one()) {
            int head0, s0;
            tile_origin(p, tile, head0, s0);
            const uint32_t bar = smem_u32(&ctl.q_full[t]);
            const uint32_t dst = smem_base + kSmemQ + t * kTileBytes;
            mbar_arrive_expect_tx(bar, q_bytes);
#pragma unroll
            for (int c = 0; c < kHalves; ++c)
              tma_load_4d(dst + c * kHalfTile, &tmap_q, bar, c * 64, s0, it.hkv * p.group + head0, it.b);
          }
          __syncwarp();
        }
        for (int j = 0; j < it.n && ok; ++j) {
          const int key = (it.first + j) * kTileKV;
          ok = mbar_wait(smem_u32(&ctl.k_empty[k_ring.stage]), k_ring.phase ^ 1, abort_flag, p.status, ASC_DEV_TIMEOUT_EMPTY);
          if (!ok) break;
          if (elect_one()) {
            const uint32_t bar = smem_u32(&ctl.k_full[k_ring.stage]);
            const uint32_t dst = smem_base + kSmemK + k_ring.stage * kTileBytes;
            mbar_arrive_expect_tx(bar, kTileBytes);
#pragma unroll
            for (int c = 0; c < kHalves; ++c)
              tma_load_4d(dst + c * kHalfTile, &tmap_k, bar, c * 64, key, it.hkv * p.k_heads, it.b * p.k_batches);
          }
          k_ring.next();
          ok = mbar_wait(smem_u32(&ctl.v_empty[v_ring.stage]), v_ring.phase ^ 1, abort_flag, p.status, ASC_DEV_TIMEOUT_EMPTY);
          if (!ok) break;
          if (elect_one()) {
            const uint32_t bar = smem_u32(&ctl.v_full[v_ring.stage]);
            const uint32_t dst = smem_base + kSmemV + v_ring.stage * kTileBytes;
            mbar_arrive_expect_tx(bar, kTileBytes);
#pragma unroll
            for (int c = 0; c < kHalves; ++c)
              tma_load_4d(dst + c * kHalfTile, &tmap_v, bar, c * 64, key, it.hkv * p.v_heads, it.b * p.v_batches);
          }
          v_ring.next();
          __syncwarp();
        }
      }
    } else if (warp == 9) {
      // ------------------------------- MMA issuer -------------------------------
      const uint64_t q_desc0 = make_smem_desc_sw128(smem_base + kSmemQ, 16, 1024);
      const uint64_t k_desc0 = make_smem_desc_sw128(smem_base + kSmemK, 16, 1024);
      const uint64_t v_desc0 = make_smem_desc_sw128(smem_base + kSmemV, kHalfTile, 1024);
      // S_t = Q_t K_j^T: both operands K-major, in halves of 64 columns
      auto issue_qk = [&](int t, uint32_t k_stage) {
        const uint64_t qd = q_desc0 + static_cast<uint64_t>(t) * (kTileBytes >> 4);
        const uint64_t kd = k_desc0 + static_cast<uint64_t>(k_stage) * (kTileBytes >> 4);
        const uint32_t d = tmem_base + kColS + t * 128;
#pragma unroll
        for (int ks = 0; ks < 4 * kHalves; ++ks) {
          const uint32_t off = ((ks >> 2) * kHalfTile + (ks & 3) * 32) >> 4;
          umma_f16_ss(d, qd + off, kd + off, idesc_qk, ks > 0 ? 1u : 0u);
        }
      };
      // O_t (+)= P_t V_j for one half of the keys: P from tensor memory (8 columns per 16 keys), V MN-major as stored
      auto issue_pv = [&](int t, uint32_t v_stage, int part, uint32_t accumulate) {
        const uint64_t vd = v_desc0 + static_cast<uint64_t>(v_stage) * (kTileBytes >> 4);
        const uint32_t d = tmem_base + kColO + t * 128;
        const uint32_t a = tmem_base + kColS + t * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ks = 4 * part + i;
          umma_f16_ts(d, a + ks * 8, vd + ((ks * 2048) >> 4), idesc_pv, (accumulate || ks > 0) ? 1u : 0u);
        }
      };
      bool ok = true;
      uint32_t q_it[2] = {0, 0}, p_it[2] = {0, 0};
      Ring<kStages> k_ring, v_ring;
      Walker walk(p.work, range, blockIdx.x, gridDim.x);
      Segment it;
      while (ok && walk.next(p.work, it)) {
        if (it.n == 0) continue;
        bool here[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) here[t] = t < kTiles && tile_exists(p, it.tile * kTiles + t);
        // first scores of the tiles
        ok = mbar_wait(smem_u32(&ctl.k_full[k_ring.stage]), k_ring.phase, abort_flag, p.status, ASC_DEV_TIMEOUT_FULL);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          if (!ok || !here[t]) continue;
          ok = mbar_wait(smem_u32(&ctl.q_full[t]), q_it[t] & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_FULL);
          if (!ok) continue;
          ++q_it[t];
          tc_fence_after();
          if (elect_one()) {
            issue_qk(t, k_ring.stage);
            umma_commit(smem_u32(&ctl.s_full[t]));
            if (it.n == 1) umma_commit(smem_u32(&ctl.q_empty[t]));   // the tile's only Q K^T
          }
          __syncwarp();
        }
        if (ok && elect_one()) umma_commit(smem_u32(&ctl.k_empty[k_ring.stage]));
        __syncwarp();
        k_ring.next();
        for (int j = 0; j < it.n && ok; ++j) {
          ok = mbar_wait(smem_u32(&ctl.v_full[v_ring.stage]), v_ring.phase, abort_flag, p.status, ASC_DEV_TIMEOUT_FULL);
          if (!ok) break;
          const int here_keys = it.len - (it.first + j) * kTileKV;
          if (here_keys < kTileKV && it.len < p.Skv) {
            // rows of V past the length may hold anything, NaN too, and P's zeros would not silence that: clear them
            const uint32_t base = smem_base + kSmemV + v_ring.stage * kTileBytes;
            for (int i = here_keys * 8 + static_cast<int>(lane); i < kTileKV * 8; i += 32)
#pragma unroll
              for (int c = 0; c < kHalves; ++c) st_shared_zero16(base + c * kHalfTile + i * 16);
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (j + 1 < it.n) {
            ok = mbar_wait(smem_u32(&ctl.k_full[k_ring.stage]), k_ring.phase, abort_flag, p.status, ASC_DEV_TIMEOUT_FULL);
            if (!ok) break;
          }
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            if (!ok || !here[t]) continue;
            ok = mbar_wait(smem_u32(&ctl.p_half[t]), p_it[t] & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_OTHER);
            if (!ok) continue;
            tc_fence_after();
            if (elect_one()) issue_pv(t, v_ring.stage, 0, j > 0 ? 1u : 0u);
            __syncwarp();
            ok = mbar_wait(smem_u32(&ctl.p_full[t]), p_it[t] & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_OTHER);
            if (!ok) continue;
            ++p_it[t];
            tc_fence_after();
            if (elect_one()) {
              issue_pv(t, v_ring.stage, 1, j > 0 ? 1u : 0u);
              if (j + 1 < it.n) {
                issue_qk(t, k_ring.stage);
                umma_commit(smem_u32(&ctl.s_full[t]));
                // the tile's last Q K^T of this item: the producer may load the next item's Q tile
                if (j + 2 == it.n) umma_commit(smem_u32(&ctl.q_empty[t]));
              } else {
                umma_commit(smem_u32(&ctl.o_full[t]));
              }
            }
            __syncwarp();
          }
          if (ok && elect_one()) {
            umma_commit(smem_u32(&ctl.v_empty[v_ring.stage]));
            if (j + 1 < it.n) umma_commit(smem_u32(&ctl.k_empty[k_ring.stage]));
          }
          __syncwarp();
          v_ring.next();
          if (j + 1 < it.n) k_ring.next();
        }
      }
    }
  }

  if (*abort_flag) {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// --------------------------------------------------------------------------------------------------------------
// Up to 16 query rows per key head.  A warp takes 16 keys at a time straight from memory to registers, in the layout of
// mma.sync m16n8k16, and no barrier stands between two loads: what bounds it is HBM.  The products may run over d in any
// order as long as both operands agree, so a lane loads 16 consecutive bytes of K (8 elements of one key) and uses them
// as the k pairs of two products; Q is laid out alike.  For P V the roles of n and d are permuted in the same way: a
// lane loads 8 elements of four keys and pairs the keys up with byte permutes.  The next 16 keys are loaded before the
// current ones are computed.  The four warps of a CTA are joined in shared memory.  CTAs that share an item are a cluster
// where its sizes fit (kCluster: each takes an equal range of the keys, and the parts meet in distributed shared memory;
// one launch and no workspace), otherwise they follow the schedule and cross_join_kernel joins them.
// --------------------------------------------------------------------------------------------------------------
constexpr int kFewRows = 16;
constexpr int kFewWarps = 4;
constexpr int kFewKeys = 16;                          // keys of a warp's step
constexpr int kFewStep = kFewWarps * kFewKeys;        // keys of a CTA's step

template <bool kBf16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 bytes that are read once
__device__ __forceinline__ uint4 load_once(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

struct FewParams {
  const uint16_t *q, *k, *v;
  Strides qs, ks, vs;
};

template <int kHalves>
struct FewTile {
  uint4 k[2][2 * kHalves];       // keys g and 8 + g, 32 columns each: 8 elements at 32 i + 8 c
  uint4 v[4][kHalves];           // keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9: 8 elements at 64 i + 8 g
};

template <int kHalves>
__device__ __forceinline__ void load_tile(const CrossParams& p, const FewParams& f, const uint16_t* k, const uint16_t* v,
                                          int key0, int len, int g, int c, FewTile<kHalves>& t) {
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int key = key0 + 8 * n + g;
#pragma unroll
    for (int i = 0; i < 2 * kHalves; ++i) {
      const int d = 32 * i + 8 * c;
      t.k[n][i] = key < len && d < p.D ? load_once(k + key * f.ks.s + d) : zero;
    }
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int key = key0 + 2 * c + (n & 1) + 8 * (n >> 1);
#pragma unroll
    for (int i = 0; i < kHalves; ++i) {
      const int d = 64 * i + 8 * g;
      t.v[n][i] = key < len && d < p.D ? load_once(v + key * f.vs.s + d) : zero;
    }
  }
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

template <bool kBf16, int kHalves, bool kCluster>
__global__ void __launch_bounds__(kFewWarps * 32, 2) cross_few_kernel(const CrossParams p, const FewParams f, const int cluster) {
  constexpr int kD = 64 * kHalves;
  constexpr int kPitch = kD + 4;                       // shared rows of fp32 sums
  extern __shared__ float few_smem[];                  // [warp][row][kPitch]
  __shared__ float2 ml[kFewWarps][kFewRows];
  __shared__ Range range;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  if (!kCluster) {
    let_next_start();
    if (warp == 0) ascsched::find_range(p.work, blockIdx.x, gridDim.x, &range);
    __syncthreads();
  }
  const int rows = p.group * p.Sq;
  const float sl2 = p.scale_log2;

  auto row_of = [&](const Segment& it, int r, int& h, int& s) {
    const int hl = r / p.Sq;
    s = r - hl * p.Sq;
    h = it.hkv * p.group + hl;
    return r < rows;
  };
  auto write_zero = [&](const Segment& it) {
    const int r = threadIdx.x >> 3;                    // 8 threads a row
    int h, s;
    if (!row_of(it, r, h, s)) return;
    uint16_t* dst = static_cast<uint16_t*>(p.o) + it.b * p.ob + s * p.os + h * p.oh;
    for (int d = (threadIdx.x & 7) * 8; d < p.D; d += 64) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
    if ((threadIdx.x & 7) == 0 && p.lse != nullptr) p.lse[(static_cast<int64_t>(it.b) * (p.Hkv * p.group) + h) * p.Sq + s] = -INFINITY;
  };

  Walker walk(p.work, kCluster ? Range{0, 0, 0, 0} : range, blockIdx.x, gridDim.x);
  Segment it;
  bool once = true;
  while (kCluster ? once : walk.next(p.work, it)) {
    if (kCluster) {          // one item per cluster, its steps in equal ranges
      once = false;
      const int item = blockIdx.x / cluster, rank = blockIdx.x - item * cluster;
      it.b = item / p.Hkv, it.hkv = item - it.b * p.Hkv, it.tile = 0;
      it.len = p.work.len_of(it.b);
      const int steps = (it.len + kFewStep - 1) / kFewStep, each = (steps + cluster - 1) / cluster;
      it.first = rank * each;
      it.n = max(0, min(each, steps - it.first));
      it.slot = 0;           // a part: it meets the others below
    } else if (it.n == 0) {
      write_zero(it);
      continue;
    }
    // Q, as the A operand of the first product
    uint32_t q[4 * kHalves][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      int h, s;
      const bool there = row_of(it, g + 8 * half, h, s);
      const uint16_t* row = f.q + it.b * f.qs.b + s * f.qs.s + h * f.qs.h;
#pragma unroll
      for (int i = 0; i < 2 * kHalves; ++i) {
        const int d = 32 * i + 8 * c;
        const uint4 x = there && d < p.D ? *reinterpret_cast<const uint4*>(row + d) : make_uint4(0, 0, 0, 0);
        q[2 * i][half] = x.x, q[2 * i][2 + half] = x.y;
        q[2 * i + 1][half] = x.z, q[2 * i + 1][2 + half] = x.w;
      }
    }
    const uint16_t* k = f.k + it.b * f.ks.b + it.hkv * f.ks.h;
    const uint16_t* v = f.v + it.b * f.vs.b + it.hkv * f.vs.h;
    const int end = min(it.len, (it.first + it.n) * kFewStep);
    int key0 = it.first * kFewStep + warp * kFewKeys;

    float o[kHalves][8][4];        // [half][j]: rows g, g + 8 at d = 64 half + 16 c + j (and + 8)
#pragma unroll
    for (int i = 0; i < kHalves; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][j][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};     // rows g, g + 8: maximum (raw), sum of this lane's keys

    FewTile<kHalves> t;
    if (key0 < end) load_tile<kHalves>(p, f, k, v, key0, end, g, c, t);
    for (; key0 < end; key0 += kFewStep) {
      float sc[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * kHalves; ++i) {
          mma_16816<kBf16>(sc[n], q[2 * i], t.k[n][i].x, t.k[n][i].y);
          mma_16816<kBf16>(sc[n], q[2 * i + 1], t.k[n][i].z, t.k[n][i].w);
        }
      }
      uint4 vv[4][kHalves];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < kHalves; ++i) vv[n][i] = t.v[n][i];
      if (key0 + kFewStep < end) load_tile<kHalves>(p, f, k, v, key0 + kFewStep, end, g, c, t);
      if (key0 + kFewKeys > end) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + 8 * n + 2 * c + (e & 1) >= end) sc[n][e] = -INFINITY;
      }
      // running maximum of the two rows, moved only when it grows by more than 2^8 (see softmax_role)
      float top[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      }
      const bool move0 = m[0] == -INFINITY || (top[0] - m[0]) * sl2 > kRescaleThreshold;
      const bool move1 = m[1] == -INFINITY || (top[1] - m[1]) * sl2 > kRescaleThreshold;
      if (__any_sync(0xffffffffu, move0 || move1)) {
        // (a first maximum: the sums are 0 and stay so)
        const float a0 = !move0 ? 1.f : m[0] == -INFINITY ? 0.f : ex2_approx((m[0] - top[0]) * sl2);
        const float a1 = !move1 ? 1.f : m[1] == -INFINITY ? 0.f : ex2_approx((m[1] - top[1]) * sl2);
        if (move0) m[0] = top[0];
        if (move1) m[1] = top[1];
        l[0] *= a0, l[1] *= a1;
#pragma unroll
        for (int i = 0; i < kHalves; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) o[i][j][0] *= a0, o[i][j][1] *= a0, o[i][j][2] *= a1, o[i][j][3] *= a1;
      }
      uint32_t pa[4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float e0 = ex2_approx((sc[n][2 * r] - m[r]) * sl2), e1 = ex2_approx((sc[n][2 * r + 1] - m[r]) * sl2);
          l[r] += e0 + e1;
          pa[2 * n + r] = pack2<kBf16>(e0, e1);
        }
#pragma unroll
      for (int i = 0; i < kHalves; ++i) {
        const uint32_t a0[4] = {vv[0][i].x, vv[0][i].y, vv[0][i].z, vv[0][i].w}, a1[4] = {vv[1][i].x, vv[1][i].y, vv[1][i].z, vv[1][i].w};
        const uint32_t b0[4] = {vv[2][i].x, vv[2][i].y, vv[2][i].z, vv[2][i].w}, b1[4] = {vv[3][i].x, vv[3][i].y, vv[3][i].z, vv[3][i].w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          mma_16816<kBf16>(o[i][2 * w], pa, __byte_perm(a0[w], a1[w], 0x5410), __byte_perm(b0[w], b1[w], 0x5410));
          mma_16816<kBf16>(o[i][2 * w + 1], pa, __byte_perm(a0[w], a1[w], 0x7632), __byte_perm(b0[w], b1[w], 0x7632));
        }
      }
    }
    // the lanes of a row, then the warps
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (c == 0) ml[warp][g + 8 * r] = make_float2(m[r] == -INFINITY ? -INFINITY : m[r] * sl2, l[r]);
    }
    float* mine = few_smem + warp * kFewRows * kPitch;
#pragma unroll
    for (int i = 0; i < kHalves; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < 8; j += 4)
          *reinterpret_cast<float4*>(mine + (g + 8 * (e >> 1)) * kPitch + 64 * i + 16 * c + 8 * (e & 1) + j) =
              make_float4(o[i][j][e], o[i][j + 1][e], o[i][j + 2][e], o[i][j + 3][e]);
    __syncthreads();
    const int r = threadIdx.x >> 3;                    // 8 threads a row, 8 columns at a time
    int h, s;
    if (row_of(it, r, h, s)) {
      float top = -INFINITY, total = 0.f, w[kFewWarps];
#pragma unroll
      for (int i = 0; i < kFewWarps; ++i) top = fmaxf(top, ml[i][r].x);
#pragma unroll
      for (int i = 0; i < kFewWarps; ++i) {
        w[i] = ml[i][r].y == 0.f ? 0.f : exp2f(ml[i][r].x - top);      // (a warp without keys)
        total += w[i] * ml[i][r].y;
      }
      const int64_t part = static_cast<int64_t>(it.slot) * kFewRows + r;
      float* joined = few_smem + kFewWarps * kFewRows * kPitch;      // kCluster: [row][kPitch], then (top, total) per row
      const float inv = 1.f / total;
      uint16_t* dst = static_cast<uint16_t*>(p.o) + it.b * p.ob + s * p.os + h * p.oh;
      for (int d = (threadIdx.x & 7) * 8; d < p.D; d += 64) {
        float sum[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = 0.f;
#pragma unroll
        for (int i = 0; i < kFewWarps; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] = fmaf(w[i], few_smem[(i * kFewRows + r) * kPitch + d + e], sum[e]);
        if (it.slot >= 0) {
          float4* to = reinterpret_cast<float4*>(kCluster ? joined + r * kPitch + d : p.part_o + part * p.D + d);
          to[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
          to[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
        } else {
          *reinterpret_cast<uint4*>(dst + d) =
              make_uint4(pack2<kBf16>(sum[0] * inv, sum[1] * inv), pack2<kBf16>(sum[2] * inv, sum[3] * inv),
                         pack2<kBf16>(sum[4] * inv, sum[5] * inv), pack2<kBf16>(sum[6] * inv, sum[7] * inv));
        }
      }
      if ((threadIdx.x & 7) == 0) {
        if (kCluster) reinterpret_cast<float2*>(joined + kFewRows * kPitch)[r] = make_float2(top, total);
        else if (it.slot >= 0) p.part_ml[part] = make_float2(top, total);
        else if (p.lse != nullptr) p.lse[(static_cast<int64_t>(it.b) * (p.Hkv * p.group) + h) * p.Sq + s] = (top + log2f(total)) * kLn2;
      }
    }
    if (!kCluster) __syncthreads();               // the sums have been read
  }
  if (!kCluster) {
    ascsched::for_empty_items(p.work, blockIdx.x, gridDim.x, write_zero);
    return;
  }
  // the parts of the cluster: rows in turn, D / 4 threads a row, CTAs in order
  cluster_sync();
  const int rank = blockIdx.x % cluster, per_row = p.D / 4, abreast = kFewWarps * 32 / per_row;
  const uint32_t joined = smem_u32(few_smem + kFewWarps * kFewRows * kPitch), joined_ml = joined + kFewRows * kPitch * 4;
  if (threadIdx.x < abreast * per_row) {
    const int col = threadIdx.x % per_row * 4;
    for (int r = rank + cluster * (threadIdx.x / per_row); r < rows; r += cluster * abreast) {
      float top = -INFINITY, total = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = 0; i < cluster; ++i) top = fmaxf(top, ld_cluster2(mapa_shared(joined_ml + r * 8, i)).x);
      for (int i = 0; i < cluster; ++i) {
        const float2 x = ld_cluster2(mapa_shared(joined_ml + r * 8, i));
        const float w = x.y == 0.f ? 0.f : exp2f(x.x - top);          // (a part without keys)
        const float4 o4 = ld_cluster4(mapa_shared(joined + (r * kPitch + col) * 4, i));
        total += w * x.y;
        acc.x += w * o4.x, acc.y += w * o4.y, acc.z += w * o4.z, acc.w += w * o4.w;
      }
      const float inv = total == 0.f ? 0.f : 1.f / total;             // no key at all: 0
      int h, s;
      row_of(it, r, h, s);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.o) + it.b * p.ob + s * p.os + h * p.oh + col) =
          make_uint2(pack2<kBf16>(acc.x * inv, acc.y * inv), pack2<kBf16>(acc.z * inv, acc.w * inv));
      if (col == 0 && p.lse != nullptr)
        p.lse[(static_cast<int64_t>(it.b) * (p.Hkv * p.group) + h) * p.Sq + s] = total == 0.f ? -INFINITY : (top + log2f(total)) * kLn2;
    }
  }
  cluster_sync();                  // no CTA leaves while its part is read
}

// Joins the parts of the items that were cut, in order: block column = border.  kTiles: query tiles of an item, 0 for
// cross_few_kernel's rows.  D / 4 threads a row; a thread's rows are loaded independently of each other.
constexpr int kJoinRows = 4;
template <bool kBf16, int kTiles>
__global__ void __launch_bounds__(256) cross_join_kernel(const CrossParams p, int ctas) {
  constexpr int kRows = kTiles == 0 ? kFewRows : kTiles * kTileQ;
  __shared__ ascsched::Cut cut;
  __shared__ int found;
  if (threadIdx.x < 32) {
    ascsched::Cut mine;
    const bool is = ascsched::find_cut(p.work, blockIdx.x + 1, ctas, mine);
    if (threadIdx.x == 0) cut = mine, found = is;
  }
  wait_for_previous();
  __syncthreads();
  if (!found) return;
  const int per_row = p.D / 4, abreast = 256 / per_row;          // rows the CTA works on side by side
  const int c = threadIdx.x % per_row * 4, r0 = blockIdx.y * abreast * kJoinRows + threadIdx.x / per_row;
  if (threadIdx.x >= abreast * per_row) return;
  int h[kJoinRows], s[kJoinRows];
  bool there[kJoinRows];
#pragma unroll
  for (int i = 0; i < kJoinRows; ++i) {
    const int r = r0 + i * abreast;
    if (kTiles == 0) {
      h[i] = r / p.Sq;
      s[i] = r - h[i] * p.Sq;
      there[i] = h[i] < p.group && r < kRows;
      h[i] += cut.item.hkv * p.group;
    } else {
      const int tile = cut.item.tile * kTiles + r / kTileQ;
      there[i] = r < kRows && tile_exists(p, tile) && row_place(p, cut.item, tile, r % kTileQ, h[i], s[i]);
    }
  }
  float m[kJoinRows], l[kJoinRows];
  float4 acc[kJoinRows];
#pragma unroll
  for (int i = 0; i < kJoinRows; ++i) m[i] = -INFINITY, l[i] = 0.f, acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  cut.parts([&](int slot) {
    float2 ml[kJoinRows];
    float4 o[kJoinRows];
#pragma unroll
    for (int i = 0; i < kJoinRows; ++i)
      if (there[i]) {
        const int64_t at = static_cast<int64_t>(slot) * kRows + r0 + i * abreast;
        ml[i] = p.part_ml[at];
        o[i] = *reinterpret_cast<const float4*>(p.part_o + at * p.D + c);
      }
#pragma unroll
    for (int i = 0; i < kJoinRows; ++i)
      if (there[i]) {
        const float top = fmaxf(m[i], ml[i].x);
        const float a = m[i] == -INFINITY ? 0.f : exp2f(m[i] - top), w = exp2f(ml[i].x - top);
        m[i] = top;
        l[i] = l[i] * a + w * ml[i].y;
        acc[i].x = acc[i].x * a + w * o[i].x, acc[i].y = acc[i].y * a + w * o[i].y;
        acc[i].z = acc[i].z * a + w * o[i].z, acc[i].w = acc[i].w * a + w * o[i].w;
      }
  });
#pragma unroll
  for (int i = 0; i < kJoinRows; ++i)
    if (there[i]) {
      const float inv = 1.f / l[i];
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.o) + cut.item.b * p.ob + s[i] * p.os + h[i] * p.oh;
      *reinterpret_cast<uint2*>(dst + c) = make_uint2(pack2<kBf16>(acc[i].x * inv, acc[i].y * inv), pack2<kBf16>(acc[i].z * inv, acc[i].w * inv));
      if (c == 0 && p.lse != nullptr)
        p.lse[(static_cast<int64_t>(cut.item.b) * (p.Hkv * p.group) + h[i]) * p.Sq + s[i]] = (m[i] + log2f(l[i])) * kLn2;
    }
}

// ------------------------------------------------ host ---------------------------------------------------------
template <bool kBf16, int kTiles>
int32_t launch_join(const CrossParams& p, int ctas, cudaStream_t stream) {
  const int rows = kTiles == 0 ? kFewRows : kTiles * kTileQ, per_cta = 256 / (p.D / 4) * kJoinRows;
  ASC_CUDA_TRY(aschost::launch_after(cross_join_kernel<kBf16, kTiles>, dim3(ctas - 1, (rows + per_cta - 1) / per_cta), dim3(256),
                                     0, stream, p, ctas));
  aschost::count_launch();
  return ASC_OK;
}

template <bool kBf16, int kHalves>
int32_t launch_few(const CrossParams& p, const FewParams& f, int grid, int cluster, cudaStream_t stream) {
  const size_t smem = kFewWarps * kFewRows * (64 * kHalves + 4) * sizeof(float);
  if (cluster > 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kFewWarps * 32);
    cfg.dynamicSmemBytes = smem + kFewRows * ((64 * kHalves + 4) * sizeof(float) + sizeof(float2));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ASC_CUDA_TRY(cudaLaunchKernelEx(&cfg, cross_few_kernel<kBf16, kHalves, true>, p, f, cluster));
    aschost::count_launch();
    return ASC_OK;
  }
  cross_few_kernel<kBf16, kHalves, false><<<grid, kFewWarps * 32, smem, stream>>>(p, f, 0);
  aschost::count_launch();
  ASC_CUDA_TRY(cudaGetLastError());
  if (p.work.cut && grid > 1) return launch_join<kBf16, 0>(p, grid, stream);
  return ASC_OK;
}

template <bool kBf16, int kHalves, int kTiles>
int32_t launch_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CrossParams& p, int grid,
                   cudaStream_t stream) {
  constexpr int kStages = kHalves == 1 ? 4 : kTiles == 1 ? 3 : 2;
  constexpr uint32_t smem = (kTiles + 2 * kStages) * kHalves * kHalfTile + 1024;
  auto kernel = cross_fwd_kernel<kBf16, kHalves, kTiles>;
  static aschost::PerDevice attr_set;
  int dev = 0;
  ASC_CUDA_TRY(cudaGetDevice(&dev));
  if (!attr_set.get(dev)) {
    aschost::SetUpInCapture relaxed;
    // refuse to launch a build whose register split would wait forever (see attention.cu)
    cudaFuncAttributes fa{};
    ASC_CUDA_TRY(cudaFuncGetAttributes(&fa, kernel));
    if (12 * fa.numRegs < 8 * kSoftmaxRegs + 4 * kOtherRegs) return ASC_ERR_UNSUPPORTED;
    ASC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_set.set(dev, 1);
  }
  const uint32_t fmt = kBf16 ? 1u : 0u;
  const uint32_t idesc_qk = make_idesc(1, fmt, fmt, 0, 0, kTileQ, kTileKV);
  const uint32_t idesc_pv = make_idesc(1, fmt, fmt, 0, 1, kTileQ, 64 * kHalves);
  kernel<<<grid, kThreads, smem, stream>>>(tq, tk, tv, p, idesc_qk, idesc_pv);
  aschost::count_launch();
  ASC_CUDA_TRY(cudaGetLastError());
  if (p.work.cut && grid > 1) return launch_join<kBf16, kTiles>(p, grid, stream);
  return ASC_OK;
}

template <bool kBf16>
int32_t launch_any(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CrossParams& p, int tiles,
                   int grid, cudaStream_t st) {
  if (p.D <= 64)
    return tiles == 1 ? launch_fwd<kBf16, 1, 1>(tq, tk, tv, p, grid, st) : launch_fwd<kBf16, 1, 2>(tq, tk, tv, p, grid, st);
  return tiles == 1 ? launch_fwd<kBf16, 2, 1>(tq, tk, tv, p, grid, st) : launch_fwd<kBf16, 2, 2>(tq, tk, tv, p, grid, st);
}

}  // namespace

extern "C" int32_t asc_cuda_cross_attn_fwd_f16(const void* q, const void* k, const void* v, void* o, float* lse,
                                               const int32_t* kv_lengths, const int64_t* dims, const int64_t* strides,
                                               float scale, int32_t dtype, void* stream) {
  int32_t rc = check_dims(dims, strides, scale, dtype);
  if (rc != ASC_OK) return rc;
  const int64_t B = dims[0], Sq = dims[1], Skv = dims[2], Hq = dims[3], Hkv = dims[4], D = dims[5];
  if (B == 0 || Sq == 0 || Hq == 0 || D == 0) return ASC_OK;
  const Strides qs = strides_of(strides, B, Sq, Hq), ks = strides_of(strides + 3, B, Skv, Hkv),
                vs = strides_of(strides + 6, B, Skv, Hkv), os = strides_of(strides + 9, B, Sq, Hq);
  if ((rc = check_operand(q, qs, B, Sq, Hq, false)) != ASC_OK) return rc;
  if ((rc = check_operand(o, os, B, Sq, Hq, true)) != ASC_OK) return rc;
  if (Skv > 0) {
    if ((rc = check_operand(k, ks, B, Skv, Hkv, false)) != ASC_OK) return rc;
    if ((rc = check_operand(v, vs, B, Skv, Hkv, false)) != ASC_OK) return rc;
  }
  if (reinterpret_cast<uintptr_t>(lse) % 4 != 0 || reinterpret_cast<uintptr_t>(kv_lengths) % 4 != 0) return ASC_ERR_MISALIGNED;
  // a query dimension that repeats memory has its own tensor-map coordinates: those are not folded
  if ((B > 1 && qs.b == 0) || (Hq > 1 && qs.h == 0)) return ASC_ERR_INVALID_ARG;

  CrossParams p{};
  p.o = o;
  p.lse = lse;
  p.ob = os.b, p.os = os.s, p.oh = os.h;
  p.B = static_cast<int32_t>(B);
  p.Sq = static_cast<int32_t>(Sq);
  p.Skv = static_cast<int32_t>(Skv);
  p.Hkv = static_cast<int32_t>(Hkv);
  p.group = static_cast<int32_t>(Hq / Hkv);
  p.D = static_cast<int32_t>(D);
  p.scale_log2 = log2_scale(scale);
  int sms = 0;
  if ((rc = aschost::sm_count(&sms)) != ASC_OK) return rc;
  if (B * Hq > 0x7fffffff) return ASC_ERR_TOO_LARGE;
  const bool bf16 = dtype == 1, few = p.group * Sq <= kFewRows;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int64_t tiles = 1;
  int tiles_per_item = 1, grid = 0, cluster = 0;
  if (few) {
    // every key is read once, so nothing is lost by streaming different heads at the same time
    p.work = {kv_lengths, p.B, p.Skv, p.Hkv, 1, 0, kFewStep, static_cast<int32_t>(B * Hkv), 0, 0};
    const int64_t steps = (Skv + kFewStep - 1) / kFewStep, items = B * Hkv, slots = 2 * sms;
    grid = ascsched::plan(p.work, steps, static_cast<int>(slots), 0, 1, 8);
    // a cluster for each item, if that is as fast: its join costs about a step, against a launch of about eight
    for (int c = 1; c <= 8 && items * c <= slots; c *= 2) cluster = c;
    const int64_t each = cluster > 0 ? (steps + cluster - 1) / cluster : 0;
    if (cluster > 0 && p.work.cut && each + 2 > (items * steps + slots - 1) / slots + 10) cluster = 0;
    if (cluster > 0) p.work.cut = 0, grid = static_cast<int>(items * cluster);
  } else {
    // Few queries: several heads of a group share a tile, each with its queries rounded up to whole swizzle atoms of 8
    // rows.  Otherwise 128 queries of one head.
    const int seg = static_cast<int>((Sq + 7) / 8 * 8 < kTileQ ? (Sq + 7) / 8 * 8 : kTileQ);
    p.pack = kTileQ / seg < p.group ? kTileQ / seg : p.group;
    p.seg = p.pack > 1 ? seg : kTileQ;
    p.tiles_per_head = static_cast<int32_t>((Sq + kTileQ - 1) / kTileQ);
    tiles = p.pack > 1 ? (p.group + p.pack - 1) / p.pack : static_cast<int64_t>(p.group) * p.tiles_per_head;
    tiles_per_item = tiles == 1 ? 1 : 2;
    const int64_t pairs = (tiles + tiles_per_item - 1) / tiles_per_item;
    if (B * Hkv * pairs > 0x7fffffff) return ASC_ERR_TOO_LARGE;
    p.tiles = static_cast<int32_t>(tiles);
    p.work = {kv_lengths, p.B, p.Skv, p.Hkv, static_cast<int32_t>(pairs), 0, kTileKV, static_cast<int32_t>(B * Hkv * pairs), 0, 0};
    // an item costs about three steps of 128 keys besides its own (its start, its epilogue); joining costs a launch and
    // writes and reads every cut row once more (measured: 16 us, or 8 steps, where 147 items of 256 rows were cut)
    const int64_t rows = tiles_per_item * static_cast<int64_t>(kTileQ) < p.group * Sq ? tiles_per_item * kTileQ : p.group * Sq;
    grid = ascsched::plan(p.work, (Skv + kTileKV - 1) / kTileKV, sms, 2 * B * Skv * Hkv * D * 2, 3, 4 + static_cast<int>(rows / 20));
  }
  void* ws = nullptr;
  if (p.work.cut) {
    const size_t rows = static_cast<size_t>(2) * grid * (few ? kFewRows : tiles_per_item * kTileQ), o_bytes = rows * D * sizeof(float);
    if ((rc = aschost::scratch_alloc(&ws, o_bytes + rows * sizeof(float2), st)) != ASC_OK) return rc;
    p.part_o = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + o_bytes);
  }
  if (few) {
    const FewParams f{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), qs, ks, vs};
    if (D <= 64) rc = bf16 ? launch_few<true, 1>(p, f, grid, cluster, st) : launch_few<false, 1>(p, f, grid, cluster, st);
    else rc = bf16 ? launch_few<true, 2>(p, f, grid, cluster, st) : launch_few<false, 2>(p, f, grid, cluster, st);
  } else {
    CUtensorMap tq, tk, tv;
    rc = aschost::device_status_word(&p.status);
    if (rc == ASC_OK) rc = encode_rows(&tq, bf16, q, B, Sq, Hq, D, qs, p.seg, p.pack, nullptr, nullptr);
    if (rc == ASC_OK && Skv > 0) rc = encode_rows(&tk, bf16, k, B, Skv, Hkv, D, ks, kTileKV, 1, &p.k_heads, &p.k_batches);
    if (rc == ASC_OK && Skv > 0) rc = encode_rows(&tv, bf16, v, B, Skv, Hkv, D, vs, kTileKV, 1, &p.v_heads, &p.v_batches);
    if (Skv == 0) tk = tv = tq;        // never read: no item has a key
    if (rc == ASC_OK)
      rc = bf16 ? launch_any<true>(tq, tk, tv, p, tiles_per_item, grid, st) : launch_any<false>(tq, tk, tv, p, tiles_per_item, grid, st);
  }
  if (ws != nullptr) {
    const int32_t freed = aschost::scratch_free(ws, st);
    if (rc == ASC_OK) rc = freed;
  }
  return rc;
}
