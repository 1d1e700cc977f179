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
// item is a pair of tiles over a range of the keys.  Few items are cut along the keys (`splits`): each writes its
// unnormalised fp32 sum, maximum and total to a workspace, and a second kernel joins them in order.
//   warps 0-3   softmax of tile 0, one thread per row: scores from tensor memory, P back into the same columns,
//   warps 4-7   (same for tile 1)  lazy rescaling of the accumulator, epilogue
//   warp 8      TMA producer: Q tiles, K and V tiles through two rings of kStages 128B-swizzled stages
//   warp 9      MMA issuer: S = Q K^T, O += P V (P from tensor memory), accumulators S0 S1 O0 O1 in tensor memory
// Head sizes that are not 64 or 128 are padded by the tensor maps (columns past D read as zero).  All waits are bounded.
#include "../../include/asc_cuda.h"
#include "attention_common.cuh"
#include "cross_attention.h"
#include "host_common.h"

namespace {

using namespace ascdev;
using namespace asccross;

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
  const int32_t* lengths;    // keys of each batch entry, null: Skv each
  float* part_o;             // splits > 1: [splits][B Hq Sq][D] unnormalised sums
  float2* part_ml;           // splits > 1: [splits][B Hq Sq] (maximum in log2 units, total)
  int64_t ob, os, oh;        // strides of o in elements
  int32_t B, Sq, Skv, Hkv, group, D;
  int32_t seg, pack;         // rows per head and heads per tile
  int32_t tiles;             // query tiles per (batch, key head)
  int32_t tiles_per_head;    // pack == 1
  int32_t pairs;             // query tile groups per (batch, key head): kTiles tiles each
  int32_t splits;
  int32_t items;
  int32_t k_heads, k_batches, v_heads, v_batches;   // 0: that dimension of K / V has a stride of 0
  float scale_log2;          // softmax scale * log2(e)
  uint32_t* status;
};

// K and V are read through tensor maps; a broadcast dimension (stride 0) has extent 1 there.
struct Item {
  int b, hkv, pair, split;
  int key0, n;               // first key and number of key tiles of this split
  int len;                   // keys of the batch entry
};

template <int kTiles>
__device__ __forceinline__ Item item_of(const CrossParams& p, int u) {
  Item it;
  const int per_head = p.pairs * p.splits;
  const int bh = u / per_head, r = u - bh * per_head;
  it.split = r / p.pairs;
  it.pair = r - it.split * p.pairs;
  it.b = bh / p.Hkv;
  it.hkv = bh - it.b * p.Hkv;
  int len = p.Skv;
  if (p.lengths != nullptr) {
    len = __ldg(p.lengths + it.b);
    len = len < 0 ? 0 : len > p.Skv ? p.Skv : len;
  }
  it.len = len;
  const int total = (len + kTileKV - 1) / kTileKV;
  const int per = (total + p.splits - 1) / p.splits;
  const int j0 = it.split * per;
  const int left = total - j0;
  it.key0 = j0 * kTileKV;
  it.n = left < 0 ? 0 : left < per ? left : per;
  return it;
}

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

template <int kStages>
struct CrossCtl {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint32_t tmem_base;
  uint32_t abort_flag;
};

// Softmax warpgroup of one query tile: one thread per row.
template <bool kBf16, int kHalves, typename Ctl>
__device__ __forceinline__ bool softmax_role(const CrossParams& p, Ctl& ctl, uint32_t tmem_base, int t, const Item& it,
                                             int tile, uint32_t& s_it, uint32_t& o_it) {
  volatile uint32_t* abort_flag = &ctl.abort_flag;
  const int row = threadIdx.x & 127;            // row inside the tile == TMEM lane
  const uint32_t lane_base = ((threadIdx.x >> 5) & 3) * 32;
  const uint32_t t_s = tmem_base + (lane_base << 16) + kColS + t * 128;
  const uint32_t t_o = tmem_base + (lane_base << 16) + kColO + t * 128;
  const float sl2 = p.scale_log2;
  int head0, s0;
  tile_origin(p, tile, head0, s0);
  const int hl = head0 + row / p.seg;
  const int s_row = s0 + row % p.seg;
  const bool valid = row < p.seg * p.pack && hl < p.group && s_row < p.Sq;
  const int h = it.hkv * p.group + hl;
  const int64_t flat = (static_cast<int64_t>(it.b) * (p.Hkv * p.group) + h) * p.Sq + s_row;   // [B, Hq, Sq]

  float m_ref = 0.f;  // maximum (raw score units) the exponentials are taken against
  float l = 0.f;      // running sum of exp2((s - m_ref) * sl2)

  for (int j = 0; j < it.n; ++j) {
    if (!mbar_wait(smem_u32(&ctl.s_full[t]), s_it & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_TMEM_FULL)) return false;
    ++s_it;
    tc_fence_after();
    uint32_t s[4][32];
#pragma unroll
    for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(t_s + c * 32, s[c]);
    tmem_ld_wait();

    const int limit = it.len - 1 - it.key0 - j * kTileKV;   // columns c <= limit are there (at least one)
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
        const float e0 = ex2_approx(x.x);
        const float e1 = ex2_approx(x.y);
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
    }
    l += (l0 + l1) + (l2 + l3);
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&ctl.p_full[t]));
  }

  if (it.n == 0) {
    // no key in this part: nothing to add, or (whole rows) a result of zero
    if (!valid) return true;
    if (p.splits > 1) {
      p.part_ml[static_cast<int64_t>(it.split) * p.B * p.Hkv * p.group * p.Sq + flat] = make_float2(-INFINITY, 0.f);
      return true;
    }
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.o) + it.b * p.ob + s_row * p.os + h * p.oh;
    for (int c = 0; c < p.D; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0, 0, 0, 0);
    if (p.lse != nullptr) p.lse[flat] = -INFINITY;
    return true;
  }
  // ------------------------------ epilogue: O / l -> 16-bit -> global, or the part as it is ------------------------
  if (!mbar_wait(smem_u32(&ctl.o_full[t]), o_it & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_TMEM_FULL)) return false;
  ++o_it;
  tc_fence_after();
  if (p.splits > 1) {
    const int64_t at = static_cast<int64_t>(it.split) * p.B * p.Hkv * p.group * p.Sq + flat;
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctl.tmem_base;

  // Every role walks the same list of items, so the use counts of the barriers advance identically in all of them.
  if (warp < 8) {
    setmaxnreg_inc<kSoftmaxRegs>();
    const int t = static_cast<int>(warp >> 2);
    uint32_t s_it = 0, o_it = 0;
    bool ok = t < kTiles;
    for (int u = blockIdx.x; u < p.items && ok; u += gridDim.x) {
      const Item it = item_of<kTiles>(p, u);
      const int tile = it.pair * kTiles + t;
      if (tile_exists(p, tile)) ok = softmax_role<kBf16, kHalves>(p, ctl, tmem_base, t, it, tile, s_it, o_it);
    }
  } else {
    setmaxnreg_dec<kOtherRegs>();
    if (warp == 8) {
      // ------------------------------ TMA producer ------------------------------
      bool ok = true;
      uint32_t q_it[2] = {0, 0};
      Ring<kStages> k_ring, v_ring;
      const uint32_t q_bytes = static_cast<uint32_t>(p.seg * p.pack) * 128u * kHalves;
      for (int u = blockIdx.x; u < p.items && ok; u += gridDim.x) {
        const Item it = item_of<kTiles>(p, u);
        if (it.n == 0) continue;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const int tile = it.pair * kTiles + t;
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
          const int key = it.key0 + j * kTileKV;
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
      // O_t (+)= P_t V_j: P from tensor memory (8 columns per 16 keys), V MN-major as stored
      auto issue_pv = [&](int t, uint32_t v_stage, uint32_t accumulate) {
        const uint64_t vd = v_desc0 + static_cast<uint64_t>(v_stage) * (kTileBytes >> 4);
        const uint32_t d = tmem_base + kColO + t * 128;
        const uint32_t a = tmem_base + kColS + t * 128;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          umma_f16_ts(d, a + ks * 8, vd + ((ks * 2048) >> 4), idesc_pv, (accumulate || ks > 0) ? 1u : 0u);
      };
      bool ok = true;
      uint32_t q_it[2] = {0, 0}, p_it[2] = {0, 0};
      Ring<kStages> k_ring, v_ring;
      for (int u = blockIdx.x; u < p.items && ok; u += gridDim.x) {
        const Item it = item_of<kTiles>(p, u);
        if (it.n == 0) continue;
        bool here[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) here[t] = t < kTiles && tile_exists(p, it.pair * kTiles + t);
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
          const int here_keys = it.len - it.key0 - j * kTileKV;
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
            ok = mbar_wait(smem_u32(&ctl.p_full[t]), p_it[t] & 1, abort_flag, p.status, ASC_DEV_TIMEOUT_OTHER);
            if (!ok) continue;
            ++p_it[t];
            tc_fence_after();
            if (elect_one()) {
              issue_pv(t, v_ring.stage, j > 0 ? 1u : 0u);
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

// Joins the parts of rows that were cut along the keys: a warp per row, parts in order.
template <bool kBf16>
__global__ void __launch_bounds__(256) cross_join_kernel(const CrossParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(p.B) * p.Hkv * p.group * p.Sq;
  const int64_t row = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (row >= rows) return;
  float m = -INFINITY;
  for (int i = 0; i < p.splits; ++i) m = fmaxf(m, p.part_ml[i * rows + row].x);
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
  const int c = lane * 4;
  for (int i = 0; i < p.splits; ++i) {
    const float2 ml = p.part_ml[i * rows + row];
    if (ml.y == 0.f) continue;                  // no key in this part (NaN is not 0 and is carried on)
    const float w = exp2f(ml.x - m);
    l += w * ml.y;
    if (c < p.D) {
      const float4 o = *reinterpret_cast<const float4*>(p.part_o + (i * rows + row) * p.D + c);
      acc[0] += w * o.x, acc[1] += w * o.y, acc[2] += w * o.z, acc[3] += w * o.w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int s = static_cast<int>(row % p.Sq);
  const int64_t bh = row / p.Sq;
  const int heads = p.Hkv * p.group;
  uint16_t* dst = reinterpret_cast<uint16_t*>(p.o) + bh / heads * p.ob + s * p.os + bh % heads * p.oh;
  if (c < p.D)
    *reinterpret_cast<uint2*>(dst + c) = make_uint2(pack2<kBf16>(acc[0] * inv, acc[1] * inv), pack2<kBf16>(acc[2] * inv, acc[3] * inv));
  if (lane == 0 && p.lse != nullptr) p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// ------------------------------------------------ host ---------------------------------------------------------
// Parts the keys are cut into: the count with the least time on the busiest SM, in key tiles, where an item costs about
// three tiles beyond its own (its start, its epilogue) and joining costs every row once more.
int choose_splits(int64_t items, int64_t key_tiles, int64_t sms) {
  int best = 1;
  int64_t best_cost = (items + sms - 1) / sms * (key_tiles + 3);
  for (int s = 2; s <= kMaxSplits && s <= key_tiles; ++s) {
    const int64_t cost = (items * s + sms - 1) / sms * ((key_tiles + s - 1) / s + 3) + 4;
    if (cost < best_cost) best_cost = cost, best = s;
  }
  return best;
}

template <bool kBf16, int kHalves, int kTiles>
int32_t launch_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CrossParams& p, int sms,
                   cudaStream_t stream) {
  constexpr int kStages = kHalves == 1 ? 4 : kTiles == 1 ? 3 : 2;
  constexpr uint32_t smem = (kTiles + 2 * kStages) * kHalves * kHalfTile + 1024;
  auto kernel = cross_fwd_kernel<kBf16, kHalves, kTiles>;
  static aschost::PerDevice attr_set;
  int dev = 0;
  ASC_CUDA_TRY(cudaGetDevice(&dev));
  if (!attr_set.get(dev)) {
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
  const int grid = p.items < sms ? p.items : sms;
  kernel<<<grid, kThreads, smem, stream>>>(tq, tk, tv, p, idesc_qk, idesc_pv);
  aschost::count_launch();
  ASC_CUDA_TRY(cudaGetLastError());
  return ASC_OK;
}

template <bool kBf16>
int32_t launch_any(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CrossParams& p, int tiles,
                   int sms, cudaStream_t st) {
  if (p.D <= 64)
    return tiles == 1 ? launch_fwd<kBf16, 1, 1>(tq, tk, tv, p, sms, st) : launch_fwd<kBf16, 1, 2>(tq, tk, tv, p, sms, st);
  return tiles == 1 ? launch_fwd<kBf16, 2, 1>(tq, tk, tv, p, sms, st) : launch_fwd<kBf16, 2, 2>(tq, tk, tv, p, sms, st);
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
  p.lengths = kv_lengths;
  p.ob = os.b, p.os = os.s, p.oh = os.h;
  p.B = static_cast<int32_t>(B);
  p.Sq = static_cast<int32_t>(Sq);
  p.Skv = static_cast<int32_t>(Skv);
  p.Hkv = static_cast<int32_t>(Hkv);
  p.group = static_cast<int32_t>(Hq / Hkv);
  p.D = static_cast<int32_t>(D);
  p.scale_log2 = log2_scale(scale);
  // Few queries: several heads of a group share a tile, each with its queries rounded up to whole swizzle atoms of 8
  // rows.  Otherwise 128 queries of one head.
  const int seg = static_cast<int>((Sq + 7) / 8 * 8 < kTileQ ? (Sq + 7) / 8 * 8 : kTileQ);
  p.pack = kTileQ / seg < p.group ? kTileQ / seg : p.group;
  p.seg = p.pack > 1 ? seg : kTileQ;
  p.tiles_per_head = static_cast<int32_t>((Sq + kTileQ - 1) / kTileQ);
  const int64_t tiles = p.pack > 1 ? (p.group + p.pack - 1) / p.pack : static_cast<int64_t>(p.group) * p.tiles_per_head;
  const int tiles_per_item = tiles == 1 ? 1 : 2;
  const int64_t pairs = (tiles + tiles_per_item - 1) / tiles_per_item;
  int sms = 0;
  if ((rc = aschost::sm_count(&sms)) != ASC_OK) return rc;
  const int64_t whole = B * Hkv * pairs;
  if (whole > 0x7fffffff / kMaxSplits || B * Hq > 0x7fffffff) return ASC_ERR_TOO_LARGE;
  p.tiles = static_cast<int32_t>(tiles);
  p.pairs = static_cast<int32_t>(pairs);
  p.splits = choose_splits(whole, (Skv + kTileKV - 1) / kTileKV, sms);
  p.items = static_cast<int32_t>(whole * p.splits);

  const bool bf16 = dtype == 1;
  CUtensorMap tq, tk, tv;
  if ((rc = encode_rows(&tq, bf16, q, B, Sq, Hq, D, qs, p.seg, p.pack, nullptr, nullptr)) != ASC_OK) return rc;
  if (Skv > 0) {
    if ((rc = encode_rows(&tk, bf16, k, B, Skv, Hkv, D, ks, kTileKV, 1, &p.k_heads, &p.k_batches)) != ASC_OK) return rc;
    if ((rc = encode_rows(&tv, bf16, v, B, Skv, Hkv, D, vs, kTileKV, 1, &p.v_heads, &p.v_batches)) != ASC_OK) return rc;
  } else {
    tk = tv = tq;        // never read: no item has a key
  }
  if ((rc = aschost::device_status_word(&p.status)) != ASC_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  void* ws = nullptr;
  const int64_t rows = B * Hq * Sq;
  if (p.splits > 1) {
    const size_t o_bytes = static_cast<size_t>(p.splits) * rows * D * sizeof(float);
    if ((rc = aschost::scratch_alloc(&ws, o_bytes + static_cast<size_t>(p.splits) * rows * sizeof(float2), st)) != ASC_OK)
      return rc;
    p.part_o = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + o_bytes);
  }
  rc = bf16 ? launch_any<true>(tq, tk, tv, p, tiles_per_item, sms, st) : launch_any<false>(tq, tk, tv, p, tiles_per_item, sms, st);
  if (p.splits > 1) {
    if (rc == ASC_OK) {
      const unsigned grid = static_cast<unsigned>((rows + 7) / 8);
      if (bf16) cross_join_kernel<true><<<grid, 256, 0, st>>>(p);
      else cross_join_kernel<false><<<grid, 256, 0, st>>>(p);
      const cudaError_t e = cudaGetLastError();
      if (e == cudaSuccess) aschost::count_launch();
      else rc = aschost::record_cuda_error(e, "cross_join_kernel");
    }
    const int32_t freed = aschost::scratch_free(ws, st);
    if (rc == ASC_OK) rc = freed;
  }
  return rc;
}
