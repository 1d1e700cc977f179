// How the gradient and the forward of attention to another sequence hand out their work.
//
// An item is a kept tile of one (batch, key head) and its steps along the streamed axis.  Items differ in length when the
// batch entries do, and there are seldom a whole multiple of the SMs of them.  The first `whole` items go round the CTAs
// one by one (neighbouring CTAs then stream the same rows through L2).  The steps of the others, in order, are divided
// evenly: CTA c takes positions [first + c W / G, first + (c + 1) W / G).  An item that a border falls into is computed in
// parts, each into a slot of a workspace, and a second kernel adds the parts up in order; with `cut` 0 the borders are
// moved to the nearest start of an item, and there are no parts.
#pragma once

#include "host_common.h"

namespace ascsched {

struct Schedule {
  const int32_t* lengths;    // keys of each batch entry, null: Skv each
  int32_t B, Skv, heads;     // heads: key heads
  int32_t tiles;             // kept tiles per (batch, head); keys kept: of an entry of Skv keys
  int32_t steps;             // keys kept: steps of an item; 0: queries are kept, steps follow from the length
  int32_t key_rows;          // keys per step (queries kept) or per tile (keys kept)
  int32_t items;             // B * heads * tiles
  int32_t whole, cut;

  __host__ __device__ int tiles_of(int len) const { return steps > 0 ? (len + key_rows - 1) / key_rows : tiles; }
  __host__ __device__ int steps_of(int len) const { return steps > 0 ? steps : (len + key_rows - 1) / key_rows; }
#ifdef __CUDACC__
  __device__ int len_of(int b) const {
    if (lengths == nullptr) return Skv;
    const int n = __ldg(lengths + b);
    return n < 0 ? 0 : n > Skv ? Skv : n;
  }
  __device__ int work_of(int b) const {
    const int len = len_of(b);
    return heads * tiles_of(len) * steps_of(len);
  }
#endif
};

#ifdef __CUDACC__

// A position of the divided steps: the batch entry it lies in and the steps before that entry.
struct Position {
  int pos, b, base;
};

// All steps, and the entry that position `pos` (below the total) lies in.  Called by a whole warp.
__device__ __forceinline__ int total_steps(const Schedule& s) {
  if (s.lengths == nullptr) return s.B * s.work_of(0);
  int t = 0;
  for (int b = threadIdx.x & 31; b < s.B; b += 32) t += s.work_of(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}
__device__ __forceinline__ Position locate(const Schedule& s, int pos) {
  if (s.lengths == nullptr) {
    const int w = s.work_of(0);
    return {pos, pos / w, pos / w * w};
  }
  int base = 0;
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < s.B; b0 += 32) {
    int w = b0 + lane < s.B ? s.work_of(b0 + lane) : 0;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {                 // inclusive prefix sums
      const int up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + w > pos);
    if (past != 0) {
      const int at = __ffs(past) - 1;
      const int before = __shfl_sync(0xffffffffu, w, at > 0 ? at - 1 : 0);
      return {pos, b0 + at, base + (at > 0 ? before : 0)};
    }
    base += __shfl_sync(0xffffffffu, w, 31);
  }
  return {pos, s.B, base};                            // pos is the total
}

// Border c of `ctas` (0 ... ctas) as a position; moved to an item's start where items are not cut.
__device__ __forceinline__ Position border(const Schedule& s, int total, int c, int ctas) {
  const int first = s.whole > 0 ? static_cast<int>(static_cast<int64_t>(total) / s.items * s.whole) : 0;
  Position p = locate(s, first + static_cast<int>(static_cast<int64_t>(total - first) * c / ctas));
  if (s.cut == 0 && p.b < s.B) {
    const int n = s.steps_of(s.len_of(p.b));
    const int in = (p.pos - p.base) % n;
    p.pos += 2 * in < n ? -in : n - in;
  }
  return p;
}

struct Segment {
  int b, hkv, tile;
  int first, n;              // steps [first, first + n)
  int len;                   // keys of the batch entry
  int slot;                  // workspace slot of a part, -1: the whole item
};

// The range of a CTA, written to shared memory by one warp before the roles part.
struct Range {
  int pos, end, b, base;
};
__device__ __forceinline__ void find_range(const Schedule& s, int cta, int ctas, Range* out) {
  Range r{0, 0, 0, 0};
  if (s.whole < s.items) {
    const int total = total_steps(s);
    const Position from = border(s, total, cta, ctas), to = border(s, total, cta + 1, ctas);
    r = {from.pos, to.pos, from.b, from.base};
  }
  if ((threadIdx.x & 31) == 0) *out = r;
}

// The segments of a CTA, in the same order for every role.
struct Walker {
  int cta, ctas, u, pos, end, start, b, base, tiles, steps, len;

  Walker() = default;
  __device__ Walker(const Schedule& s, const Range& r, int cta_, int ctas_)
      : cta(cta_), ctas(ctas_), u(cta_), pos(r.pos), end(r.end), start(r.pos), b(r.b), base(r.base) {
    if (pos < end) load(s);
  }
  __device__ void load(const Schedule& s) {
    len = s.len_of(b);
    tiles = s.tiles_of(len), steps = s.steps_of(len);
  }
  __device__ bool next(const Schedule& s, Segment& g) {
    if (u < s.whole) {
      const int bh = u / s.tiles;
      g.tile = u - bh * s.tiles;
      g.b = bh / s.heads;
      g.hkv = bh - g.b * s.heads;
      g.len = s.len_of(g.b);
      g.first = 0;
      g.n = g.tile < s.tiles_of(g.len) ? s.steps_of(g.len) : 0;
      g.slot = -1;
      u += ctas;
      return true;
    }
    if (pos >= end) return false;
    while (b + 1 < s.B && pos - base >= s.heads * tiles * steps) {
      base += s.heads * tiles * steps;
      ++b;
      load(s);
    }
    const int r = pos - base, i = r / steps;
    g.b = b;
    g.hkv = i / tiles;
    g.tile = i - g.hkv * tiles;
    g.len = len;
    g.first = r - i * steps;
    g.n = min(steps - g.first, end - pos);
    g.slot = g.n == steps ? -1 : 2 * cta + (pos != start);
    pos += g.n;
    return true;
  }
};

// A warp's walk kept in shared memory, for the warps whose registers are full of scores: `next` puts the segment there
// too.  Called by whole warps, each with a Walk of its own.
struct Walk {
  Walker walker;
  Segment segment;

  __device__ void start(const Schedule& s, const Range& r, int cta, int ctas) {
    const Walker w(s, r, cta, ctas);
    if ((threadIdx.x & 31) == 0) walker = w;
    __syncwarp();
  }
  __device__ bool next(const Schedule& s) {
    Walker w = walker;
    Segment g;
    const bool more = w.next(s, g);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      walker = w;
      if (more) segment = g;
    }
    __syncwarp();
    return more;
  }
};

// Items without steps among the divided ones (an entry without keys, a tile of keys past the length): their results are
// zeros, which the CTAs write in turn.  `f(segment)` is called for each.
template <typename F>
__device__ __forceinline__ void for_empty_items(const Schedule& s, int cta, int ctas, F&& f) {
  if (s.lengths == nullptr) return;
  for (int u = s.whole + cta; u < s.items; u += ctas) {
    Segment g;
    const int bh = u / s.tiles;
    g.tile = u - bh * s.tiles;
    g.b = bh / s.heads;
    g.hkv = bh - g.b * s.heads;
    g.len = s.len_of(g.b);
    if (g.tile < s.tiles_of(g.len) && s.steps_of(g.len) > 0) continue;
    g.first = g.n = 0;
    g.slot = -1;
    f(g);
  }
}

// For the kernel that adds parts up, block column c = 1 ... ctas - 1: the item that border c cuts, if no earlier border
// cuts it.  Its parts are `first_slot` and those of the CTAs from c on whose range is not empty and begins in the item.
struct Cut {
  Segment item;
  int first_slot, c, end, first, work, ctas;
  __device__ int at(int k) const { return first + static_cast<int>(static_cast<int64_t>(work) * k / ctas); }
  // f(slot) for every part in order
  template <typename F>
  __device__ void parts(F&& f) const {
    f(first_slot);
    for (int k = c; k < ctas && at(k) < end; ++k)
      if (at(k + 1) > at(k)) f(2 * k);
  }
};
__device__ __forceinline__ bool find_cut(const Schedule& s, int c, int ctas, Cut& cut) {
  const int total = total_steps(s);
  const Position p = border(s, total, c, ctas);
  if (p.b >= s.B) return false;
  const int len = s.len_of(p.b), tiles = s.tiles_of(len), steps = s.steps_of(len);
  const int i = (p.pos - p.base) / steps;
  const int begin = p.base + i * steps;
  cut.first = s.whole > 0 ? static_cast<int>(static_cast<int64_t>(total) / s.items * s.whole) : 0;
  cut.work = total - cut.first, cut.ctas = ctas, cut.c = c, cut.end = begin + steps;
  const int before = cut.at(c - 1);
  if (p.pos == begin || before > begin) return false;
  cut.item.b = p.b, cut.item.hkv = i / tiles, cut.item.tile = i % tiles, cut.item.len = len;
  cut.item.first = 0, cut.item.n = steps, cut.item.slot = -1;
  cut.first_slot = 2 * (c - 1) + (before != begin);
  return true;
}

#endif  // __CUDACC__

// Chooses `whole` and `cut` and the grid.  One step costs about as much as a unit; an item costs `item_cost` of them
// besides, adding parts up `join_cost` in all.
//   - Work that is streamed from L2 anyway (`streamed_bytes` small) is divided as a whole; otherwise only the remainder
//     after whole rounds over the SMs, because CTAs that stream different heads at the same time miss L2.
//   - With lengths given the rounds cannot be counted on the host: all or nothing is divided.
inline int plan(Schedule& s, int64_t steps_per_item, int sms, int64_t streamed_bytes, int item_cost, int join_cost) {
  const int64_t items = s.items;
  const bool fits_l2 = streamed_bytes <= (64ll << 20);
  const int64_t rounds = (items + sms - 1) / sms;
  const int64_t cost_whole = rounds * (steps_per_item + item_cost);
  s.whole = s.items;
  s.cut = 0;
  if (steps_per_item == 0 || items * steps_per_item >= (1ll << 30)) return s.items < sms ? s.items : sms;
  if (s.lengths == nullptr) {
    const int64_t full = fits_l2 && items < 4ll * sms ? 0 : items / sms;
    const int64_t rest = items - full * sms;
    const int64_t work = rest * steps_per_item;
    const int64_t ctas = work < sms ? work : sms;
    const int64_t cost_cut = full * (steps_per_item + item_cost) + (work + sms - 1) / sms + 2 * item_cost + join_cost;
    if (rest > 0 && cost_cut < cost_whole) {
      s.whole = static_cast<int32_t>(full * sms);
      s.cut = 1;
      return full > 0 ? sms : static_cast<int>(ctas);
    }
  } else if (fits_l2 || items <= sms) {
    const int64_t work = items * steps_per_item;
    s.cut = (work + sms - 1) / sms + 2 * item_cost + join_cost < cost_whole;
    if (!s.cut && items <= sms) return s.items;       // one item each
    s.whole = 0;
    const int64_t most = s.cut ? work : items;
    return static_cast<int>(most < sms ? most : sms);
  }
  return s.items < sms ? s.items : sms;
}

}  // namespace ascsched
