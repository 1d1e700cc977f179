// What the forward and the gradient of attention to another sequence share: sizes, the ring counter of the pipelines,
// argument checks and tensor maps.
#pragma once

#include "host_common.h"

namespace asccross {

constexpr uint32_t kHalfTile = 128 * 128;   // 64 columns of a 128-row 16-bit tile: 16 KiB
constexpr float kLog2e = 1.4426950408889634f;

template <int kStages>
struct Ring {
  uint32_t stage = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == kStages) stage = 0, phase ^= 1;
  }
};

// Softmax scale in log2 units.  A scale of 0 becomes the least normal number: any finite score times it is still 0 next
// to 1, and the -inf of a key that is not there stays -inf (times 0 it would be NaN).
inline float log2_scale(float scale) {
  const float s = scale * kLog2e;
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

struct Strides {
  int64_t b, s, h;
};

// Tensor map of a [B, S, H, D] operand seen as (D, S, H, B) with boxes of 64 x rows x heads; a dimension of one element
// or with a stride of 0 becomes extent 1.  `heads` / `batches`: what to multiply coordinates with.
inline int32_t encode_rows(CUtensorMap* map, bool bf16, const void* base, int64_t B, int64_t S, int64_t H, int64_t D,
                    const Strides& st, uint32_t rows, uint32_t box_heads, int32_t* heads, int32_t* batches) {
  const bool one_h = H == 1 || st.h == 0, one_b = B == 1 || st.b == 0;
  if (heads != nullptr) *heads = !one_h;
  if (batches != nullptr) *batches = !one_b;
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(S), one_h ? 1ull : static_cast<uint64_t>(H),
                            one_b ? 1ull : static_cast<uint64_t>(B)};
  const uint64_t any = 16;        // the stride of a dimension of one element is not used
  const uint64_t strides[3] = {S == 1 ? any : static_cast<uint64_t>(st.s) * 2, one_h ? any : static_cast<uint64_t>(st.h) * 2,
                               one_b ? any : static_cast<uint64_t>(st.b) * 2};
  const uint32_t box[4] = {64, rows, box_heads, 1};
  return aschost::encode_tmap(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims,
                              strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

// What forward and backward check alike.  strides: q, k, v, then the others, three (batch, sequence, head) each.
inline int32_t check_dims(const int64_t* dims, const int64_t* strides, float scale, int32_t dtype) {
  if (dims == nullptr || strides == nullptr) return ASC_ERR_INVALID_ARG;
  for (int i = 0; i < 6; ++i)
    if (dims[i] < 0) return ASC_ERR_INVALID_ARG;
  const int64_t B = dims[0], Sq = dims[1], Skv = dims[2], Hq = dims[3], Hkv = dims[4], D = dims[5];
  if (dtype < 0 || dtype > 1 || !(scale >= 0.f) || scale > 3.0e38f) return ASC_ERR_INVALID_ARG;
  if (Hkv == 0 ? Hq != 0 : Hq % Hkv != 0) return ASC_ERR_INVALID_ARG;
  if (D > 128 || D % 8 != 0) return ASC_ERR_UNSUPPORTED;
  if (B > (1 << 24) || Sq > (1 << 30) || Skv > (1 << 30) || Hq > (1 << 16)) return ASC_ERR_TOO_LARGE;
  return ASC_OK;
}

inline Strides strides_of(const int64_t* s, int64_t B, int64_t S, int64_t H) {
  return {B > 1 ? s[0] : 0, S > 1 ? s[1] : 0, H > 1 ? s[2] : 0};
}

// An operand that TMA reads or 16-byte vectors write.
inline int32_t check_operand(const void* p, const Strides& s, int64_t B, int64_t S, int64_t H, bool written) {
  if (p == nullptr) return ASC_ERR_INVALID_ARG;
  if (!aschost::aligned16(p) || s.b % 8 != 0 || s.s % 8 != 0 || s.h % 8 != 0) return ASC_ERR_MISALIGNED;
  if (s.b < 0 || s.s < 0 || s.h < 0) return ASC_ERR_INVALID_ARG;
  if (s.b >= (1ll << 38) || s.s >= (1ll << 38) || s.h >= (1ll << 38)) return ASC_ERR_TOO_LARGE;
  if (S > 1 && s.s == 0) return ASC_ERR_INVALID_ARG;
  if (written && ((B > 1 && s.b == 0) || (H > 1 && s.h == 0))) return ASC_ERR_INVALID_ARG;
  return ASC_OK;
}

}  // namespace asccross
