// Gradients of attention to another sequence (cross_attention.cu), fp16 / bf16, for sm_100a.  With P = exp(scale Q K^T -
// lse) recomputed from the saved lse, and delta = rowsum(dO o O):
//   dV = P^T dO,   dS = P o (dO V^T - delta),   dQ = scale dS K,   dK = scale dS^T Q.
//
// Two passes of one kernel (side by side in one launch, each on its share of the SMs), which differ in what stays and
// what streams:
//   dQ      keeps 128 queries (Q, dO) and streams keys (K, V):   S = Q K^T, dP = dO V^T, dQ += dS K
//   dK, dV  keeps 128 keys (K, V) and streams queries (Q, dO):   S = K Q^T, dP = V dO^T, dK += dS Q, dV += P dO
// so that every sum stays in tensor memory and is written once: no atomics, the same bits in every run.  That costs seven
// products instead of the five of a single pass; the five cannot keep all three sums on the SM, and adding dQ up across
// SMs in memory would make its bits depend on the order.  dS and P are rounded to the inputs' type for their products.
//
// The stream comes in tiles of 64 rows, double buffered in tensor memory, so the exponentials of one step overlap the
// products of its neighbours.  A step's 64 columns are halved between two warpgroups: what bounds a step is the chain
// from its scores to its sums (its instructions fill a fifth of the issue slots), and half the columns are half the chain.
//   warps 0-15   four warpgroups, (step parity) x (half of the columns): scores and dP from tensor memory, dS and P back
//                into the same columns; at the end each writes a quarter of the sums
//   warp 16      TMA producer: the kept tiles, then a ring of kStages stages (two tiles, and per query row its lse and
//                delta when queries stream)
//   warp 17      MMA issuer
// Where whole items (a kept tile and its stream) would leave SMs idle some are cut along the stream
// (attention_schedule.cuh): parts go to an fp32 workspace and are added up in order.
// A small kernel first writes -lse (in log2 units) and -delta per query row, -inf for rows that must not count.
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

constexpr int kTile = 128;      // kept rows (= TMEM lanes)
constexpr int kStep = 64;       // streamed rows per step
constexpr int kMathWarps = 16;
constexpr int kThreads = (kMathWarps + 4) * 32;   // whole warpgroups: two warps idle
// Register split after launch, see attention.cu: the increase may only take what the decrease releases.
constexpr int kLaunchRegs = 96, kMathRegs = 104, kOtherRegs = 64;
static_assert(kMathWarps * kMathRegs + 4 * kOtherRegs <= (kMathWarps + 4) * kLaunchRegs, "register split exceeds the launch allocation");
constexpr int kStages = 4;
constexpr uint32_t kHalfStep = 64 * 128;    // 64 columns of a 64-row tile: 8 KiB
constexpr uint32_t kColS = 0, kColAcc = 256;   // buffer b: S at 128 b, dP at 128 b + 64; sums at 256 and 384
struct BwdParams {
  void* out[2];              // dQ, -  or  dK, dV
  int64_t ob[2], os[2], oh[2];
  float* part;               // parts: [slot][sum][128 rows][D], unscaled
  Schedule work;
  const float* rows_l;       // [B, Hq, rows_pad] -lse log2 e, or -inf
  const float* rows_d;       // [B, Hq, rows_pad] -delta
  int32_t B, Sq, Skv, Hkv, group, D;
  int32_t rows_pad;
  int32_t seg, pack;         // queries: rows per head and heads per tile (kept: of 128, streamed: of 64)
  int32_t q_tiles_per_head;  // pack == 1
  int32_t k_heads, k_batches, v_heads, v_batches;
  float scale, scale_log2;
  uint32_t* status;
};

// first head within its group and first query of a query tile of `rows` rows
__device__ __forceinline__ void tile_origin(const BwdParams& p, int tile, int rows, int& head, int& s0) {
  if (p.pack == 1) {
    head = tile / p.q_tiles_per_head;
    s0 = (tile - head * p.q_tiles_per_head) * rows;
  } else {
    head = tile * p.pack;
    s0 = 0;
  }
}

// Sequence position and head of a kept tile's row; false where there is none.
template <bool kKeys>
__device__ __forceinline__ bool row_place(const BwdParams& p, const Segment& it, int row, int& s, int& h) {
  if (kKeys) {
    s = it.tile * kTile + row;
    h = it.hkv;
    return s < p.Skv;
  }
  int head0, s0;
  tile_origin(p, it.tile, kTile, head0, s0);
  const int hl = head0 + row / p.seg;
  s = s0 + row % p.seg;
  h = it.hkv * p.group + hl;
  return row < p.seg * p.pack && hl < p.group && s < p.Sq;
}

struct BwdCtl {
  uint64_t r_full, r_empty;                       // kept tiles
  uint64_t c_full[kStages], c_empty[kStages];     // stream
  uint64_t s_full[2], p_full[2];                  // scores and dP written / dS and P written
  uint64_t acc_full, acc_empty;
  uint32_t tmem_base;
  uint32_t abort_flag;
};

__device__ __forceinline__ void bulk_load(uint32_t dst_smem, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst_smem),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
               : "memory");
}
// Half a step: 32 scores and dP of this thread's row -> dS (and P), packed into the first 16 of the same columns.
// (neg_l, neg_d): -lse and -delta of the row, or of the columns, from shared memory, when queries stream.
template <bool kBf16, bool kKeys>
__device__ __forceinline__ void step_math(uint32_t t_s, const float* col_l, const float* col_d, float neg_l, float neg_d,
                                          float sl2, int limit) {
  uint32_t s[32], d[32];
  tmem_ld_32x32b_x32(t_s, s);
  tmem_ld_32x32b_x32(t_s + 64, d);
  tmem_ld_wait();
  if (!kKeys && limit < 31) {       // keys that are not there: whatever K and V hold, they count nothing
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i > limit) s[i] = 0xff800000u, d[i] = 0u;
  }
  const float2 sl = make_float2(sl2, sl2);
  uint32_t ds[16], pp[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float4 l = make_float4(neg_l, neg_l, neg_l, neg_l), delta = make_float4(neg_d, neg_d, neg_d, neg_d);
    if (kKeys) {
      l = reinterpret_cast<const float4*>(col_l)[i];
      delta = reinterpret_cast<const float4*>(col_d)[i];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = 4 * i + 2 * k;
      const float2 lc = k == 0 ? make_float2(l.x, l.y) : make_float2(l.z, l.w);
      const float2 dc = k == 0 ? make_float2(delta.x, delta.y) : make_float2(delta.z, delta.w);
      const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sl, lc);
      const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
      const float2 g = __fmul2_rn(e, __fadd2_rn(make_float2(__uint_as_float(d[c]), __uint_as_float(d[c + 1])), dc));
      ds[c / 2] = pack2<kBf16>(g.x, g.y);
      if (kKeys) pp[c / 2] = pack2<kBf16>(e.x, e.y);
    }
  }
  tmem_st_32x32b_x16(t_s, ds);
  if (kKeys) tmem_st_32x32b_x16(t_s + 64, pp);
}

// Writes `kCols` columns of a sum for this thread's row, or zeros: for all rows (there was no step) or for a row that is
// gone (its key is not there).
template <bool kBf16, int kCols>
__device__ __forceinline__ void write_row(const BwdParams& p, uint32_t t_acc, int which, int col0, bool valid, bool no_sum,
                                          bool gone, int b, int s, int h, float* part, float scale) {
  const bool zero = no_sum || gone;
  uint16_t* dst = static_cast<uint16_t*>(p.out[which]) + b * p.ob[which] + s * p.os[which] + h * p.oh[which];
#pragma unroll
  for (int c = 0; c < kCols; c += 16) {
    uint32_t o[16];
    if (!no_sum) {                 // warp-wide, also where the warp has rows that are gone
      tmem_ld_32x32b_x16(t_acc + c, o);
      tmem_ld_wait();
    }
    if (!valid) continue;
    if (part != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col0 + c + i * 4 < p.D)
          reinterpret_cast<uint4*>(part + col0 + c)[i] =
              zero ? make_uint4(0, 0, 0, 0) : make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    } else {
      uint32_t pk[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        pk[i] = zero ? 0u : pack2<kBf16>(__uint_as_float(o[2 * i]) * scale, __uint_as_float(o[2 * i + 1]) * scale);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (col0 + c + i * 8 < p.D)
          reinterpret_cast<uint4*>(dst + col0 + c)[i] = make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
    }
  }
}

// Tensor maps of a pass: kept tiles 1 and 2, stream 1 and 2.  Keys kept: K, V; Q, dO.  Queries kept: Q, dO; K, V.
struct Maps {
  CUtensorMap r1, r2, c1, c2;
};

template <bool kBf16, int kHalves, bool kKeys>
__device__ __forceinline__ void bwd_pass(const Maps& maps, const BwdParams& p, const int cta, const int ctas,
                                         uint8_t* smem_raw, BwdCtl& ctl, Range& range, ascsched::Walk* walks) {
  const CUtensorMap &tmap_r1 = maps.r1, &tmap_r2 = maps.r2, &tmap_c1 = maps.c1, &tmap_c2 = maps.c2;
  constexpr uint32_t kFmt = kBf16 ? 1u : 0u;
  const uint32_t idesc_s = make_idesc(1, kFmt, kFmt, 0, 0, kTile, kKeys ? p.seg * p.pack : kStep);
  constexpr uint32_t idesc_acc = make_idesc(1, kFmt, kFmt, 0, 1, kTile, 64 * kHalves);
  constexpr uint32_t kKept = kHalves * kHalfTile, kStream = kHalves * kHalfStep;
  constexpr uint32_t kSmemR = 0, kSmemC = 2 * kKept, kSmemPairs = kSmemC + kStages * 2 * kStream;
  const uint32_t warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  volatile uint32_t* abort_flag = &ctl.abort_flag;
  const int stream_rows = kKeys ? p.seg * p.pack : kStep;      // rows of a stream tile: 16, 32, 48 or 64

  if (threadIdx.x == 0) {
    ctl.abort_flag = 0;
    prefetch_tmap(&tmap_r1);
    prefetch_tmap(&tmap_r2);
    prefetch_tmap(&tmap_c1);
    prefetch_tmap(&tmap_c2);
    mbar_init(smem_u32(&ctl.r_full), 1);
    mbar_init(smem_u32(&ctl.r_empty), 1);
    mbar_init(smem_u32(&ctl.acc_full), 1);
    mbar_init(smem_u32(&ctl.acc_empty), kMathWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctl.s_full[i]), 1);
      mbar_init(smem_u32(&ctl.p_full[i]), kMathWarps / 2);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&ctl.c_full[i]), 1);
      mbar_init(smem_u32(&ctl.c_empty[i]), 1);
    }
    fence_mbar_init();
  }
  if (warp == kMathWarps + 1) {
    tmem_alloc(smem_u32(&ctl.tmem_base), 512);
    tmem_relinquish();
  }
  if (warp == kMathWarps) ascsched::find_range(p.work, cta, ctas, &range);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctl.tmem_base;

  // Every role walks the same list of segments.  `g` numbers the steps of all segments: it gives the buffer (g & 1), the
  // warpgroup and the phases; `done` counts segments with steps and gives the phases of the kept tiles and the sums.
  if (warp < kMathWarps) {
    setmaxnreg_inc<kMathRegs>();
    const int parity = static_cast<int>(warp >> 2) & 1, half = static_cast<int>(warp >> 3);
    const uint8_t* pairs = smem_raw + (smem_base - smem_u32(smem_raw)) + kSmemPairs + half * 32 * 4;
    const int row = threadIdx.x & 127;
    const uint32_t lane_base = ((threadIdx.x >> 5) & 3) * 32;
    const uint32_t t_base = tmem_base + (lane_base << 16);
    uint32_t g = 0, done = 0;
    bool ok = true;
    // writes a segment's sums, or zeros where there is no step
    auto finish = [&](const Segment& it) {
      int s, h;
      const bool valid = row_place<kKeys>(p, it, row, s, h);
      const bool gone = kKeys && s >= it.len;          // a key that is not there: its gradient is 0
      float* part = nullptr;
      if (it.slot >= 0) part = p.part + (static_cast<int64_t>(it.slot) * (kKeys ? 2 : 1) * kTile + row) * p.D;
      if (kKeys) {             // dK by the warpgroups of the first half, dV by the others; each one half of the columns
        const int col0 = parity * 32 * kHalves;
        if (part != nullptr) part += half * kTile * p.D;
        write_row<kBf16, 32 * kHalves>(p, t_base + kColAcc + half * 128 + col0, half, col0, valid, it.n == 0, gone, it.b, s, h,
                                       part, half == 0 ? p.scale : 1.f);
      } else {
        const int col0 = (half * 2 + parity) * 16 * kHalves;
        write_row<kBf16, 16 * kHalves>(p, t_base + kColAcc + col0, 0, col0, valid, it.n == 0, gone, it.b, s, h, part, p.scale);
      }
    };
    ascsched::Walk& walk = walks[warp];
    walk.start(p.work, range, cta, ctas);
    const Segment& it = walk.segment;
    while (ok && walk.next(p.work)) {
      const int steps = it.n;
      int limit = it.len - 1 - it.first * kStep - half * 32;
      int s, h;
      float neg_l = 0.f, neg_d = 0.f;
      if (!kKeys && row_place<kKeys>(p, it, row, s, h)) {
        const int64_t at = (static_cast<int64_t>(it.b) * (p.Hkv * p.group) + h) * p.rows_pad + s;
        neg_l = p.rows_l[at], neg_d = p.rows_d[at];
      }
      for (int i = 0; i < steps && ok; ++i, limit -= kStep) {
        const uint32_t step = g + i, buf = step & 1;
        if (static_cast<int>(buf) != parity) continue;
        if (kKeys) {           // the rows' lse and delta were written by the copy that this barrier counts
          ok = mbar_wait(smem_u32(&ctl.c_full[step % kStages]), (step / kStages) & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_FULL);
          if (!ok) break;
        }
        ok = mbar_wait(smem_u32(&ctl.s_full[buf]), (step >> 1) & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_TMEM_FULL);
        if (!ok) break;
        tc_fence_after();
        const float* cols = reinterpret_cast<const float*>(pairs + (step % kStages) * (kStep * 8));
        step_math<kBf16, kKeys>(t_base + kColS + buf * 128 + half * 32, cols, cols + kStep, neg_l, neg_d, p.scale_log2,
                                limit);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.p_full[buf]));
      }
      if (!ok) break;
      g += steps;
      const bool zero = steps == 0;
      if (!zero) {
        ok = mbar_wait(smem_u32(&ctl.acc_full), done & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_TMEM_FULL);
        if (!ok) break;
        ++done;
        tc_fence_after();
      }
      finish(it);
      if (!zero) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.acc_empty));
      }
    }
    if (ok) ascsched::for_empty_items(p.work, cta, ctas, finish);
  } else {
    setmaxnreg_dec<kOtherRegs>();
    if (warp == kMathWarps && elect_one()) {
      // ------------------------------ TMA producer (one thread) ------------------------------
      bool ok = true;
      uint32_t done = 0;
      Ring<kStages> ring;
      const uint32_t kept_rows = kKeys ? kTile : static_cast<uint32_t>(p.seg * p.pack);
      const uint32_t r_bytes = 2 * kept_rows * 128u * kHalves;
      const uint32_t c_bytes = 2 * static_cast<uint32_t>(stream_rows) * 128u * kHalves + (kKeys ? stream_rows * 8u : 0u);
      Walker walk(p.work, range, cta, ctas);
      Segment it;
      while (ok && walk.next(p.work, it)) {
        if (it.n == 0) continue;
        ok = mbar_wait(smem_u32(&ctl.r_empty), (done & 1) ^ 1, abort_flag, p.status, ASC_DEV_TIMEOUT_EMPTY);
        if (!ok) break;
        ++done;
        {
          const uint32_t bar = smem_u32(&ctl.r_full), dst = smem_base + kSmemR;
          mbar_arrive_expect_tx(bar, r_bytes);
          int head0 = 0, s0 = 0;
          if (!kKeys) tile_origin(p, it.tile, kTile, head0, s0);
#pragma unroll
          for (int c = 0; c < kHalves; ++c) {
            if (kKeys) {
              tma_load_4d(dst + c * kHalfTile, &tmap_r1, bar, c * 64, it.tile * kTile, it.hkv * p.k_heads, it.b * p.k_batches);
              tma_load_4d(dst + kKept + c * kHalfTile, &tmap_r2, bar, c * 64, it.tile * kTile, it.hkv * p.v_heads, it.b * p.v_batches);
            } else {
              tma_load_4d(dst + c * kHalfTile, &tmap_r1, bar, c * 64, s0, it.hkv * p.group + head0, it.b);
              tma_load_4d(dst + kKept + c * kHalfTile, &tmap_r2, bar, c * 64, s0, it.hkv * p.group + head0, it.b);
            }
          }
        }
        for (int i = 0; i < it.n && ok; ++i) {
          ok = mbar_wait(smem_u32(&ctl.c_empty[ring.stage]), ring.phase ^ 1, abort_flag, p.status, ASC_DEV_TIMEOUT_EMPTY);
          if (!ok) break;
          {
            const uint32_t bar = smem_u32(&ctl.c_full[ring.stage]);
            const uint32_t dst = smem_base + kSmemC + ring.stage * 2 * kStream;
            mbar_arrive_expect_tx(bar, c_bytes);
            int head0 = 0, s0 = (it.first + i) * kStep;
            if (kKeys) tile_origin(p, it.first + i, kStep, head0, s0);
            const int h0 = it.hkv * p.group + head0;
#pragma unroll
            for (int c = 0; c < kHalves; ++c) {
              if (kKeys) {
                tma_load_4d(dst + c * kHalfStep, &tmap_c1, bar, c * 64, s0, h0, it.b);
                tma_load_4d(dst + kStream + c * kHalfStep, &tmap_c2, bar, c * 64, s0, h0, it.b);
              } else {
                tma_load_4d(dst + c * kHalfStep, &tmap_c1, bar, c * 64, s0, it.hkv * p.k_heads, it.b * p.k_batches);
                tma_load_4d(dst + kStream + c * kHalfStep, &tmap_c2, bar, c * 64, s0, it.hkv * p.v_heads, it.b * p.v_batches);
              }
            }
            if (kKeys) {
              const int64_t at = (static_cast<int64_t>(it.b) * (p.Hkv * p.group) + h0) * p.rows_pad + s0;
              const uint32_t to = smem_base + kSmemPairs + ring.stage * (kStep * 8);
              bulk_load(to, p.rows_l + at, stream_rows * 4, bar);
              bulk_load(to + kStep * 4, p.rows_d + at, stream_rows * 4, bar);
            }
          }
          ring.next();
          }
      }
    } else if (warp == kMathWarps + 1 && elect_one()) {
      // ------------------------------- MMA issuer (one thread) -------------------------------
      const uint64_t r_desc0 = make_smem_desc_sw128(smem_base + kSmemR, 16, 1024);
      const uint64_t c_desc0 = make_smem_desc_sw128(smem_base + kSmemC, 16, 1024);             // as N x K, K-major
      const uint64_t ct_desc0 = make_smem_desc_sw128(smem_base + kSmemC, kHalfStep, 1024);     // as K x N, MN-major
      // S = R1 C1^T and dP = R2 C2^T into buffer `buf`
      auto issue_scores = [&](uint32_t buf, uint32_t stage) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const uint64_t rd = r_desc0 + ((m * kKept) >> 4);
          const uint64_t cd = c_desc0 + ((stage * 2 * kStream + m * kStream) >> 4);
          const uint32_t d = tmem_base + kColS + buf * 128 + m * 64;
#pragma unroll
          for (int ks = 0; ks < 4 * kHalves; ++ks)
            umma_f16_ss(d, rd + (((ks >> 2) * kHalfTile + (ks & 3) * 32) >> 4),
                        cd + (((ks >> 2) * kHalfStep + (ks & 3) * 32) >> 4), idesc_s, ks > 0 ? 1u : 0u);
        }
      };
      // sums += dS C1 (and P C2)
      auto issue_sums = [&](uint32_t buf, uint32_t stage, int acc_steps, bool first) {
#pragma unroll
        for (int m = 0; m < (kKeys ? 2 : 1); ++m) {
          const uint64_t cd = ct_desc0 + ((stage * 2 * kStream + m * kStream) >> 4);
          const uint32_t a = tmem_base + kColS + buf * 128 + m * 64, d = tmem_base + kColAcc + m * 128;
#pragma unroll
          for (int ks = 0; ks < kStep / 16; ++ks)
            if (ks < acc_steps) umma_f16_ts(d, a + (ks >> 1) * 32 + (ks & 1) * 8, cd + ((ks * 2048) >> 4), idesc_acc, (!first || ks > 0) ? 1u : 0u);
        }
      };
      bool ok = true;
      uint32_t g = 0, done = 0;
      Ring<kStages> s_ring, a_ring;        // stages in the order of their scores and of their sums
      Walker walk(p.work, range, cta, ctas);
      Segment it;
      while (ok && walk.next(p.work, it)) {
        if (it.n == 0) continue;
        ok = mbar_wait(smem_u32(&ctl.r_full), done & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_FULL);
        if (!ok) break;
        // Stage of step i has landed (and rows past the length are cleared).  Waited for before the wait on the math
        // warps, so that nothing but that wait stands between their arrival and the next products.
        auto landed = [&](int i) {
          ok = mbar_wait(smem_u32(&ctl.c_full[s_ring.stage]), s_ring.phase, abort_flag, p.status, ASC_DEV_TIMEOUT_FULL);
          if (!ok || kKeys) return;
          const int here = it.len - (it.first + i) * kStep;
          if (here < kStep && it.len < p.Skv) {
            // Rows of K past the length may hold anything, NaN too, and the zeros of dS would not silence that: the sums
            // leave out whole groups of 16, the rest of the last group is cleared.
            const uint32_t base = smem_base + kSmemC + s_ring.stage * 2 * kStream;
            for (int j = here * 8; j < (here + 15) / 16 * 16 * 8; ++j)
#pragma unroll
              for (int c = 0; c < kHalves; ++c) st_shared_zero16(base + c * kHalfStep + j * 16);
            fence_proxy_async_smem();
          }
        };
        auto scores = [&](int i) {
          issue_scores((g + i) & 1, s_ring.stage);
          umma_commit(smem_u32(&ctl.s_full[(g + i) & 1]));
          if (i + 1 == it.n) umma_commit(smem_u32(&ctl.r_empty));      // the kept tiles' last use as an operand
        };
        for (int i = 0; i < 2 && i < it.n && ok; ++i) {
          landed(i);
          if (!ok) break;
          tc_fence_after();
          scores(i);
          s_ring.next();
        }
        for (int i = 0; i < it.n && ok; ++i) {
          const uint32_t step = g + i, buf = step & 1;
          const bool more = i + 2 < it.n;
          if (more) landed(i + 2);
          if (ok && i == 0)        // the previous item's sums have been read
            ok = mbar_wait(smem_u32(&ctl.acc_empty), (done & 1) ^ 1, abort_flag, p.status, ASC_DEV_TIMEOUT_TMEM_EMPTY);
          if (!ok) break;
          ok = mbar_wait(smem_u32(&ctl.p_full[buf]), (step >> 1) & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_OTHER);
          if (!ok) break;
          tc_fence_after();
          const int rows = kKeys ? stream_rows : min(kStep, it.len - (it.first + i) * kStep);
          issue_sums(buf, a_ring.stage, (rows + 15) / 16, i == 0);
          umma_commit(smem_u32(&ctl.c_empty[a_ring.stage]));
          if (more) scores(i + 2);
          else if (i + 1 == it.n) umma_commit(smem_u32(&ctl.acc_full));
          a_ring.next();
          if (more) s_ring.next();
        }
        g += it.n;
        ++done;
      }
    }
  }

  if (*abort_flag) {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncwarp();       // the lanes that issued come back to the others
  tc_fence_before();
  __syncthreads();
  if (warp == kMathWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// CTAs [0, k_ctas) keep keys (dK, dV), the others queries (dQ)
template <bool kBf16, int kHalves>
__global__ void __launch_bounds__(kThreads, 1)
    cross_bwd_kernel(const __grid_constant__ Maps k_maps, const __grid_constant__ Maps q_maps,
                     const __grid_constant__ BwdParams pk, const __grid_constant__ BwdParams pq, const int k_ctas) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ BwdCtl ctl;
  __shared__ Range range;
  __shared__ ascsched::Walk walks[kMathWarps];
  const int cta = blockIdx.x;
  if (cta < k_ctas)
    bwd_pass<kBf16, kHalves, true>(k_maps, pk, cta, k_ctas, smem_raw, ctl, range, walks);
  else
    bwd_pass<kBf16, kHalves, false>(q_maps, pq, cta - k_ctas, gridDim.x - k_ctas, smem_raw, ctl, range, walks);
}

template <bool kBf16>
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b) {
  if (kBf16)
    return __uint_as_float(a << 16) * __uint_as_float(b << 16) + __uint_as_float(a & 0xffff0000u) * __uint_as_float(b & 0xffff0000u);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
  return x.x * y.x + x.y * y.y;
}

// -lse log2 e and -delta of every query row; -inf and 0 for rows past the queries and rows without keys, whose P is then
// 0.  16 lanes a row (8 elements each), four rows of a lane loaded at once: HBM-bound on O and dO.
constexpr int kRowsPerCta = 64;
template <bool kBf16>
__global__ void __launch_bounds__(256) cross_rows_kernel(const uint16_t* o, const uint16_t* dout, const float* lse,
                                                         float* rows_l, float* rows_d, int64_t n, int Sq, int rows_pad,
                                                         int Hq, int D, Strides os, Strides ds) {
  const int lane = threadIdx.x & 15;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kRowsPerCta + (threadIdx.x >> 4);
  uint4 x[4], y[4];
  float l[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t i = i0 + 16 * k;
    x[k] = y[k] = make_uint4(0, 0, 0, 0);
    l[k] = -INFINITY;
    const int64_t bh = i / rows_pad;
    const int s = static_cast<int>(i - bh * rows_pad);
    if (i >= n || s >= Sq) continue;
    const int64_t b = bh / Hq, h = bh - b * Hq;
    if (lane * 8 < D) {
      x[k] = *reinterpret_cast<const uint4*>(o + b * os.b + s * os.s + h * os.h + lane * 8);
      y[k] = *reinterpret_cast<const uint4*>(dout + b * ds.b + s * ds.s + h * ds.h + lane * 8);
    }
    l[k] = lse[bh * Sq + s];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float t = dot2<kBf16>(x[k].x, y[k].x) + dot2<kBf16>(x[k].y, y[k].y) + dot2<kBf16>(x[k].z, y[k].z) + dot2<kBf16>(x[k].w, y[k].w);
#pragma unroll
    for (int m = 8; m > 0; m >>= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
    const int64_t i = i0 + 16 * k;
    if (lane != 0 || i >= n) continue;
    rows_l[i] = -l[k] * kLog2e, rows_d[i] = -t;
    if (l[k] == -INFINITY) rows_l[i] = -INFINITY, rows_d[i] = 0.f;
  }
}

// Adds the parts of a pass's cut items, in order: block column = border, D / 4 threads a row.
template <bool kBf16, bool kKeys>
__device__ __forceinline__ void add_parts(const BwdParams& p, int ctas) {
  constexpr int kSums = kKeys ? 2 : 1, kRowsAtOnce = 4;
  __shared__ ascsched::Cut cut;
  __shared__ int found;
  if (threadIdx.x < 32) {
    ascsched::Cut mine;
    const bool is = ascsched::find_cut(p.work, blockIdx.x + 1, ctas, mine);
    if (threadIdx.x == 0) cut = mine, found = is;
  }
  __syncthreads();
  if (!found) return;
  const int per_row = p.D / 4, abreast = 256 / per_row;
  const int c = threadIdx.x % per_row * 4, r0 = blockIdx.y * abreast * kRowsAtOnce + threadIdx.x / per_row;
  if (threadIdx.x >= abreast * per_row) return;
  float4 acc[kRowsAtOnce];
#pragma unroll
  for (int i = 0; i < kRowsAtOnce; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  cut.parts([&](int slot) {
    float4 x[kRowsAtOnce];
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int r = r0 + i * abreast;              // rows that do not exist were not written: they are not stored below
      if (r < kSums * kTile)
        x[i] = *reinterpret_cast<const float4*>(p.part + (static_cast<int64_t>(slot) * kSums * kTile + r) * p.D + c);
    }
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) acc[i].x += x[i].x, acc[i].y += x[i].y, acc[i].z += x[i].z, acc[i].w += x[i].w;
  });
#pragma unroll
  for (int i = 0; i < kRowsAtOnce; ++i) {
    const int r = r0 + i * abreast, w = r / kTile;
    int s, h;
    if (r >= kSums * kTile || !row_place<kKeys>(p, cut.item, r % kTile, s, h)) continue;
    const float scale = w == 0 ? p.scale : 1.f;
    if (kKeys && s >= cut.item.len) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out[w]) + cut.item.b * p.ob[w] + s * p.os[w] + h * p.oh[w] + c) =
        make_uint2(pack2<kBf16>(acc[i].x * scale, acc[i].y * scale), pack2<kBf16>(acc[i].z * scale, acc[i].w * scale));
  }
}

template <bool kBf16>
__global__ void __launch_bounds__(256) cross_add_kernel(const BwdParams pk, const BwdParams pq, int k_ctas, int q_ctas) {
  if (blockIdx.z == 0) {
    if (pk.work.cut && blockIdx.x + 1 < k_ctas) add_parts<kBf16, true>(pk, k_ctas);
  } else {
    if (pq.work.cut && blockIdx.x + 1 < q_ctas) add_parts<kBf16, false>(pq, q_ctas);
  }
}

// Zeros for a [B, S, H, D] gradient, a warp per row
__global__ void __launch_bounds__(256) cross_zero_kernel(uint16_t* out, int64_t n, int S, int H, int D, Strides st) {
  const int c = (threadIdx.x & 31) * 4;
  const int64_t i = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (i >= n || c >= D) return;
  const int64_t h = i % H, bs = i / H;
  *reinterpret_cast<uint2*>(out + bs / S * st.b + bs % S * st.s + h * st.h + c) = make_uint2(0u, 0u);
}

// ------------------------------------------------ host ---------------------------------------------------------
template <bool kBf16, int kHalves>
int32_t launch_bwd(const Maps& k_maps, const Maps& q_maps, const BwdParams& pk, const BwdParams& pq, int k_ctas, int q_ctas,
                   cudaStream_t stream) {
  constexpr uint32_t smem = 2 * kHalves * kHalfTile + kStages * (2 * kHalves * kHalfStep + kStep * 8) + 1024;
  auto kernel = cross_bwd_kernel<kBf16, kHalves>;
  static aschost::PerDevice attr_set;
  int dev = 0;
  ASC_CUDA_TRY(cudaGetDevice(&dev));
  if (!attr_set.get(dev)) {
    aschost::SetUpInCapture relaxed;
    // refuse to launch a build whose register split would wait forever (see attention.cu)
    cudaFuncAttributes fa{};
    ASC_CUDA_TRY(cudaFuncGetAttributes(&fa, kernel));
    if ((kMathWarps + 4) * fa.numRegs < kMathWarps * kMathRegs + 4 * kOtherRegs) return ASC_ERR_UNSUPPORTED;
    ASC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_set.set(dev, 1);
  }
  kernel<<<k_ctas + q_ctas, kThreads, smem, stream>>>(k_maps, q_maps, pk, pq, k_ctas);
  aschost::count_launch();
  ASC_CUDA_TRY(cudaGetLastError());
  if (pk.work.cut || pq.work.cut) {
    const int rows = 2 * kTile, per_cta = 256 / (pk.D / 4) * 4;
    const int columns = (k_ctas > q_ctas ? k_ctas : q_ctas) - 1;
    if (columns > 0) {
      cross_add_kernel<kBf16><<<dim3(columns, (rows + per_cta - 1) / per_cta, 2), 256, 0, stream>>>(pk, pq, k_ctas, q_ctas);
      aschost::count_launch();
      ASC_CUDA_TRY(cudaGetLastError());
    }
  }
  return ASC_OK;
}

struct Call {
  const void *dout, *q, *k, *v, *o;
  const float* lse;
  void* grad[3];             // dq, dk, dv
  int64_t B, Sq, Skv, Hq, Hkv, D;
  Strides sdo, sq, sk, sv, so, sg[3];
  const int32_t* lengths;
  float scale;
  cudaStream_t stream;
};

// Both passes, on a workspace of a -lse and a -delta per query row and, where items are cut, their parts.
template <bool kBf16>
int32_t run(const Call& c) {
  int sms = 0;
  int32_t rc = aschost::sm_count(&sms);
  if (rc != ASC_OK) return rc;
  const int64_t group = c.Hq / c.Hkv;
  BwdParams p{};
  p.B = static_cast<int32_t>(c.B);
  p.Sq = static_cast<int32_t>(c.Sq);
  p.Skv = static_cast<int32_t>(c.Skv);
  p.Hkv = static_cast<int32_t>(c.Hkv);
  p.group = static_cast<int32_t>(group);
  p.D = static_cast<int32_t>(c.D);
  p.scale = c.scale;
  p.scale_log2 = log2_scale(c.scale);
  if ((rc = aschost::device_status_word(&p.status)) != ASC_OK) return rc;

  // Queries in the stream: few queries share a tile of at most 64 rows over a number of heads that divides the group,
  // each head's rows rounded up to 16 (the products' step), so that no row of a tile is undefined.
  BwdParams pk = p, pq = p;
  pk.seg = kStep, pk.pack = 1;
  if (c.Sq <= kStep / 2) {
    const int seg = static_cast<int>((c.Sq + 15) / 16 * 16);
    int pack = kStep / seg;
    while (group % pack != 0) --pack;
    if (pack > 1) pk.seg = seg, pk.pack = pack;
  }
  const int64_t rows_pad = pk.pack > 1 ? pk.seg : (c.Sq + kStep - 1) / kStep * kStep;
  pk.q_tiles_per_head = static_cast<int32_t>((c.Sq + kStep - 1) / kStep);
  const int64_t k_steps = pk.pack > 1 ? group / pk.pack : group * pk.q_tiles_per_head;
  const int64_t kv_tiles = (c.Skv + kTile - 1) / kTile;
  // Queries kept: as in the forward
  const int seg = static_cast<int>((c.Sq + 7) / 8 * 8 < kTile ? (c.Sq + 7) / 8 * 8 : kTile);
  pq.pack = static_cast<int32_t>(kTile / seg < group ? kTile / seg : group);
  pq.seg = pq.pack > 1 ? seg : kTile;
  pq.q_tiles_per_head = static_cast<int32_t>((c.Sq + kTile - 1) / kTile);
  const int64_t q_tiles = pq.pack > 1 ? (group + pq.pack - 1) / pq.pack : group * pq.q_tiles_per_head;
  if (k_steps > (1 << 30) || c.B * c.Hkv * kv_tiles > 0x7fffffff || c.B * c.Hkv * q_tiles > 0x7fffffff ||
      c.B * c.Hq > 0x7fffffff || c.B * c.Hq * rows_pad > (1ll << 33))
    return ASC_ERR_TOO_LARGE;
  pk.work = {c.lengths, p.B, p.Skv, p.Hkv, static_cast<int32_t>(kv_tiles), static_cast<int32_t>(k_steps), kTile,
             static_cast<int32_t>(c.B * c.Hkv * kv_tiles), 0, 0};
  pq.work = {c.lengths, p.B, p.Skv, p.Hkv, static_cast<int32_t>(q_tiles), 0, kStep,
             static_cast<int32_t>(c.B * c.Hkv * q_tiles), 0, 0};
  // The passes share the SMs: each item an SM of its own where that is enough, otherwise by what a step costs, four
  // products for keys against three for queries and the same chain of waits: 6 to 5 (measured at [2, 2048] on 4096, 32 / 8
  // heads of 128: 822 us; 6 to 4.7: 861, 6 to 5.3: 838).
  const int64_t q_steps = (c.Skv + kStep - 1) / kStep;
  int k_sms = 0;
  if (c.Skv > 0) {
    const int64_t k_items = pk.work.items, q_items = pq.work.items;
    const double k_cost = 6.0 * k_items * (k_steps + 5), q_cost = 5.0 * q_items * (q_steps + 5);
    if (k_items + q_items <= sms) k_sms = static_cast<int>(k_items);
    else k_sms = static_cast<int>(sms * k_cost / (k_cost + q_cost) + 0.5);
    k_sms = k_sms < 1 ? 1 : k_sms > sms - 1 ? sms - 1 : k_sms;
  }
  // an item costs about five steps of 64 rows besides its own (kept tiles, sums), adding parts up about eight
  const int k_grid = c.Skv > 0 ? ascsched::plan(pk.work, k_steps, k_sms, 2 * c.B * c.Sq * c.Hq * c.D * 2, 5, 8) : 0;
  const int q_grid = ascsched::plan(pq.work, q_steps, sms - k_sms, 2 * c.B * c.Skv * c.Hkv * c.D * 2, 5, 8);
  pk.rows_pad = pq.rows_pad = static_cast<int32_t>(rows_pad);

  Maps mk, mq;
  if ((rc = encode_rows(&mq.r1, kBf16, c.q, c.B, c.Sq, c.Hq, c.D, c.sq, pq.seg, pq.pack, nullptr, nullptr)) != ASC_OK ||
      (rc = encode_rows(&mq.r2, kBf16, c.dout, c.B, c.Sq, c.Hq, c.D, c.sdo, pq.seg, pq.pack, nullptr, nullptr)) != ASC_OK)
    return rc;
  if (c.Skv == 0) {
    mq.c1 = mq.c2 = mq.r1;        // never read: no item has a step
    mk = mq;
  } else if ((rc = encode_rows(&mk.r1, kBf16, c.k, c.B, c.Skv, c.Hkv, c.D, c.sk, kTile, 1, &pk.k_heads, &pk.k_batches)) != ASC_OK ||
             (rc = encode_rows(&mk.r2, kBf16, c.v, c.B, c.Skv, c.Hkv, c.D, c.sv, kTile, 1, &pk.v_heads, &pk.v_batches)) != ASC_OK ||
             (rc = encode_rows(&mk.c1, kBf16, c.q, c.B, c.Sq, c.Hq, c.D, c.sq, pk.seg, pk.pack, nullptr, nullptr)) != ASC_OK ||
             (rc = encode_rows(&mk.c2, kBf16, c.dout, c.B, c.Sq, c.Hq, c.D, c.sdo, pk.seg, pk.pack, nullptr, nullptr)) != ASC_OK ||
             (rc = encode_rows(&mq.c1, kBf16, c.k, c.B, c.Skv, c.Hkv, c.D, c.sk, kStep, 1, &pq.k_heads, &pq.k_batches)) != ASC_OK ||
             (rc = encode_rows(&mq.c2, kBf16, c.v, c.B, c.Skv, c.Hkv, c.D, c.sv, kStep, 1, &pq.v_heads, &pq.v_batches)) != ASC_OK) {
    return rc;
  }

  const size_t n_rows = static_cast<size_t>(c.B) * c.Hq * rows_pad;
  const size_t rows_bytes = (n_rows * 2 * sizeof(float) + 255) / 256 * 256, slot_bytes = static_cast<size_t>(kTile) * c.D * sizeof(float);
  const size_t k_bytes = pk.work.cut ? 4 * k_grid * slot_bytes : 0, q_bytes = pq.work.cut ? 2 * q_grid * slot_bytes : 0;
  void* ws = nullptr;
  if ((rc = aschost::scratch_alloc(&ws, rows_bytes + k_bytes + q_bytes, c.stream)) != ASC_OK) return rc;
  char* at = static_cast<char*>(ws);
  float* rows = reinterpret_cast<float*>(at);
  pk.rows_l = pq.rows_l = rows;
  pk.rows_d = pq.rows_d = rows + n_rows;
  pk.part = reinterpret_cast<float*>(at + rows_bytes);
  pq.part = reinterpret_cast<float*>(at + rows_bytes + k_bytes);
  for (int i = 0; i < 3; ++i) {
    BwdParams& to = i == 0 ? pq : pk;
    const int w = i == 2;
    to.out[w] = c.grad[i];
    to.ob[w] = c.sg[i].b, to.os[w] = c.sg[i].s, to.oh[w] = c.sg[i].h;
  }
  cross_rows_kernel<kBf16><<<static_cast<unsigned>((n_rows + kRowsPerCta - 1) / kRowsPerCta), 256, 0, c.stream>>>(
      static_cast<const uint16_t*>(c.o), static_cast<const uint16_t*>(c.dout), c.lse, rows, rows + n_rows,
      static_cast<int64_t>(n_rows), p.Sq, pk.rows_pad, static_cast<int>(c.Hq), p.D, c.so, c.sdo);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) aschost::count_launch();
  else rc = aschost::record_cuda_error(e, "cross_rows_kernel");
  if (rc == ASC_OK)
    rc = c.D <= 64 ? launch_bwd<kBf16, 1>(mk, mq, pk, pq, k_grid, q_grid, c.stream)
                   : launch_bwd<kBf16, 2>(mk, mq, pk, pq, k_grid, q_grid, c.stream);
  const int32_t freed = aschost::scratch_free(ws, c.stream);
  return rc == ASC_OK ? freed : rc;
}

// Without a query the gradients of k and v are sums of nothing.
int32_t no_queries(const Call& c) {
  const int64_t n = c.B * c.Skv * c.Hkv;
  if ((n + 7) / 8 > 0x7fffffff) return ASC_ERR_TOO_LARGE;
  for (int i = 1; i < 3; ++i) {
    cross_zero_kernel<<<static_cast<unsigned>((n + 7) / 8), 256, 0, c.stream>>>(
        static_cast<uint16_t*>(c.grad[i]), n, static_cast<int>(c.Skv), static_cast<int>(c.Hkv), static_cast<int>(c.D), c.sg[i]);
    ASC_CUDA_TRY(cudaGetLastError());
    aschost::count_launch();
  }
  return ASC_OK;
}

}  // namespace

extern "C" int32_t asc_cuda_cross_attn_bwd_f16(const void* d_o, const void* q, const void* k, const void* v, const void* o,
                                               const float* lse, const int32_t* kv_lengths, void* dq, void* dk, void* dv,
                                               const int64_t* dims, const int64_t* strides, float scale, int32_t dtype,
                                               void* stream) {
  int32_t rc = check_dims(dims, strides, scale, dtype);
  if (rc != ASC_OK) return rc;
  Call c{d_o, q, k, v, o, lse, {dq, dk, dv}, dims[0], dims[1], dims[2], dims[3], dims[4], dims[5], {}, {}, {}, {}, {}, {},
         kv_lengths, scale, static_cast<cudaStream_t>(stream)};
  if (c.B == 0 || c.Hkv == 0 || c.D == 0 || (c.Sq == 0 && c.Skv == 0) || (c.Hq == 0 && c.Skv == 0)) return ASC_OK;
  // strides: dO, q, k, v, o, dq, dk, dv
  c.sdo = strides_of(strides, c.B, c.Sq, c.Hq);
  c.sq = strides_of(strides + 3, c.B, c.Sq, c.Hq);
  c.sk = strides_of(strides + 6, c.B, c.Skv, c.Hkv);
  c.sv = strides_of(strides + 9, c.B, c.Skv, c.Hkv);
  c.so = strides_of(strides + 12, c.B, c.Sq, c.Hq);
  c.sg[0] = strides_of(strides + 15, c.B, c.Sq, c.Hq);
  c.sg[1] = strides_of(strides + 18, c.B, c.Skv, c.Hkv);
  c.sg[2] = strides_of(strides + 21, c.B, c.Skv, c.Hkv);
  const bool queries = c.Sq > 0 && c.Hq > 0;
  if (c.Skv > 0) {
    if ((rc = check_operand(dk, c.sg[1], c.B, c.Skv, c.Hkv, true)) != ASC_OK) return rc;
    if ((rc = check_operand(dv, c.sg[2], c.B, c.Skv, c.Hkv, true)) != ASC_OK) return rc;
    if (queries) {
      if ((rc = check_operand(k, c.sk, c.B, c.Skv, c.Hkv, false)) != ASC_OK) return rc;
      if ((rc = check_operand(v, c.sv, c.B, c.Skv, c.Hkv, false)) != ASC_OK) return rc;
    }
  }
  if (!queries) return no_queries(c);
  // (queries and their gradients must not repeat memory; see the forward)
  if ((rc = check_operand(q, c.sq, c.B, c.Sq, c.Hq, true)) != ASC_OK) return rc;
  if ((rc = check_operand(d_o, c.sdo, c.B, c.Sq, c.Hq, true)) != ASC_OK) return rc;
  if ((rc = check_operand(o, c.so, c.B, c.Sq, c.Hq, false)) != ASC_OK) return rc;
  if ((rc = check_operand(dq, c.sg[0], c.B, c.Sq, c.Hq, true)) != ASC_OK) return rc;
  if (lse == nullptr) return ASC_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(lse) % 4 != 0 || reinterpret_cast<uintptr_t>(kv_lengths) % 4 != 0) return ASC_ERR_MISALIGNED;
  return dtype == 1 ? run<true>(c) : run<false>(c);
}
