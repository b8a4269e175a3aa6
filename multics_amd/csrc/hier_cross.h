// Shared parts of the cross attention kernels: rows, key tiles and their masks.
//
// The query heads that share a key head are rows of one product: row r of
// (stream b, key head) is query r / G of head G * hk + r % G, so a tile of 128
// rows is full with few queries and many heads too, and a key head's gradients are
// sums over its rows.  Keys come in tiles of 64, contiguous in memory, by buffer
// loads into LDS (the layouts of hier_tile.h): a key past the stream's length or
// masked is an out-of-range row, which the load writes as zeros, so whatever such
// rows hold is never read.
#pragma once

#include "hier_gemm.h"
#include "hier_tile.h"

namespace hier {
namespace cross {

using gemm::f32x16;
using gemm::u32x4;
using tile::Geo;
using tile::kBothRead;
using tile::kRowRead;
using tile::kSlab;
using tile::kTrRead;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 128;           // rows of a work item (forward, dQ), keys of one (dK, dV)

// Rows of 64 to a tile of LDS, S the read pattern's swizzle: the lane's offsets
// from the tile's first row.
template <int D, int S>
struct Rows64 {
  uint32_t voff[Geo<D>::NI];
  int first;                         // the lane's first row of the tile
  __device__ __forceinline__ void init(int wave, int lane, int64_t ss) {
    tile::Copier<D, S> c;
    c.init(wave, lane);
    first = c.idx_off;
#pragma unroll
    for (int e = 0; e < Geo<D>::NI; ++e) voff[e] = (uint32_t)((first + e) * (int)(2 * ss)) + c.add(e);
  }
  // Rows of the tile (of SPAN) at byte address `base`, `rows` of them (or fewer) in
  // range; with MASK only those whose bit of `seen` is set.
  template <bool MASK, int SPAN = kSlab>
  __device__ __forceinline__ void copy(uint64_t base, int64_t rows, int64_t ss, uint64_t seen, const char* slot,
                                       int wave) const {
    const int64_t left = rows <= 0 ? 0 : rows >= SPAN ? 0x7fffffff : 2 * ((rows - 1) * ss + D);
    const u32x4 srd = {(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu, (uint32_t)left, 0x00020000u};
    const uint32_t bits = MASK ? (uint32_t)(seen >> first) : 0u;
#pragma unroll
    for (int e = 0; e < Geo<D>::NI; ++e) {
      const uint32_t v = !MASK || (bits >> e & 1u) ? voff[e] : gemm::kOut;
      gemm::dma(srd, v, (uint32_t)(uintptr_t)(slot + (16 * wave + Geo<D>::NR * e) * Geo<D>::ROWB));
    }
  }
};

template <typename T>
__device__ __forceinline__ u32x4 row_operand(const char* base, int off) {
  return *reinterpret_cast<const u32x4*>(base + off);
}
__device__ __forceinline__ u32x4 tr_operand(const char* lo, const char* hi) {
  return __builtin_bit_cast(u32x4, tile::tr_read(lo, hi));
}

// A lane's row of D channels as MFMA operands: chunk c holds channels 16 c + 8 (lane / 32) .. + 8.
template <int D>
__device__ __forceinline__ void load_row(u32x4* dst, const uint16_t* row, int lane) {
  const uint16_t* p = row + 8 * (lane >> 5);
#pragma unroll
  for (int c = 0; c < Geo<D>::NC; ++c) dst[c] = *reinterpret_cast<const u32x4*>(p + 16 * c);
}

// Which keys of tile t are seen, of a stream of `len` keys.  `byte`: the lane's key's
// mask byte, loaded before (MASK).
template <bool MASK>
__device__ __forceinline__ uint64_t seen_keys(int64_t len, int t, uint32_t byte) {
  const int64_t left = len - (int64_t)t * kSlab;
  const uint64_t in = left >= kSlab ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
  if constexpr (MASK) return in & __ballot(byte != 0);
  else return in;
}

// Element i of a 32 x 32 result's key: 8 (i / 4) + 4 (lane / 32) + i % 4 of 32.
__device__ __forceinline__ bool key_bit(uint32_t bits, int i, int lane) {
  return bits >> (8 * (i >> 2) + (i & 3) + 4 * (lane >> 5)) & 1u;
}

// HIER_OK, or what is wrong with the sizes, types and views (hier_cross_fwd.hip).
int check(const HierCrossArgs& a);

// Parts of the tiles that an item goes over, by a model of the time in us: of the `slots`
// workgroups that run at once each takes `full` a tile where all of them work, `least` at
// best, `start` tiles' time to start and end, and the parts' fp32 sums (`bytes` of
// one part of all items) are written and read at 5 TB/s by a launch more.
struct SplitModel {
  int slots;
  double full, least, start;
  int tiles;                         // of a part, at least
};
inline int best_splits(const SplitModel& m, int64_t items, int64_t tiles, double bytes, int most) {
  int best = 1;
  double time = 1e30;
  for (int64_t n = 1; n <= most && (n == 1 || n * m.tiles <= tiles); ++n) {
    const double each = (double)((tiles + n - 1) / n) + m.start;
    const int64_t whole = items * n / m.slots;
    const double rest = (double)(items * n % m.slots) / m.slots;
    double t = each * (m.full * (double)whole + (rest > 0 ? (m.least > m.full * rest ? m.least : m.full * rest) : 0.0));
    if (n > 1) t += 4 + 2 * (double)n * bytes / 5e6;
    if (t < time) {
      time = t;
      best = (int)n;
    }
  }
  return best;
}

inline int64_t row_tiles(int64_t rows) { return (rows + kRows - 1) / kRows; }

}  // namespace cross
}  // namespace hier
