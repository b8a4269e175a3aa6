// The 16-bit types of the block's operators (norms, products, cross attention)
// and their conversions; sums of partial rows in a fixed order.
#pragma once

#include "hier_common.h"

namespace hier {

typedef uint32_t w32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Eight values of a 16-byte word.
template <typename T>
struct Eight {
  typedef T type __attribute__((ext_vector_type(8)));
};
template <typename T>
using vec8 = typename Eight<T>::type;

template <typename T>
__device__ __forceinline__ void widen(const w32x4& w, float* f) {
  const vec8<T> v = __builtin_bit_cast(vec8<T>, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
}
// Round to nearest even, the only rounding to 16 bits of a result.
template <typename T>
__device__ __forceinline__ w32x4 narrow(const float* f) {
  vec8<T> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (T)f[i];
  return __builtin_bit_cast(w32x4, v);
}

// Division of row numbers below 2^31 by g, 1 <= g < 2^31:
// r / g = (r * mul) >> (32 + shift), mul = floor(2^(32 + shift) / g) + 1 with
// shift = ceil(log2 g) - 1; g = 1 needs none.
struct Div {
  uint32_t g, mul, shift;
};
inline Div make_div(uint32_t g) {
  Div d = {g, 0u, 0u};
  if (g == 1) return d;
  while ((1ull << (d.shift + 1)) < g) ++d.shift;
  d.mul = (uint32_t)((1ull << (32 + d.shift)) / g + 1);
  return d;
}
__device__ __forceinline__ uint32_t quotient(uint32_t r, const Div& d) {
  return d.g == 1 ? r : __umulhi(r, d.mul) >> d.shift;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// out[g][c] = sum of the rows g * rows .. + rows of partial [groups * rows][C], in
// a fixed order: 32 threads a column add every 32nd row, then a tree joins them.
// type: the output's (HIER_BF16, HIER_FP16, HIER_FP32).
int sum_rows(const float* partial, int64_t rows, int64_t groups, int64_t C, void* out, int type,
             hipStream_t stream);

}  // namespace hier
