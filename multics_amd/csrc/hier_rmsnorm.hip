// Root-mean-square norm over the model's channels, with the addition of a
// residual before it, and its gradient:
//   h = x + r,  s = 1 / sqrt(mean(h^2) + eps),  y = h s w
//   dx = dr = s (dy w - h s mean(dy w h s)) + dh,   dw = sum over rows of dy h s
// All in fp32; y, h and dx are rounded once.  The norm (and its gradient) takes the
// sum before its rounding to h, so that dw, which is fp32, is fp32 throughout.
//
// Bound by memory: every element is read and written once (the gradient reads
// x and r again rather than a saved h).  A row stays in the registers of the
// 1, 4 or 16 waves that own it (WPR; at most 4 chunks of 8 channels a lane), so
// its mean of squares and its output need one read.  Rows that no 16-byte
// access fits (an odd number of channels, an odd stride) go through the same
// code with 2-byte accesses that neighbouring lanes make side by side (VEC 1).
// The gain's gradient is summed over the rows of a workgroup in registers,
// over its waves in LDS, and over the workgroups by sum_rows: a fixed order.
//
// Measured, bf16: 18,816 x 1,536 with residual 41 us (231 MB, 5.6 TB/s; a copy of as
// much reaches 5.1), its gradient 59 + 4 of sum_rows (289 MB, 4.9 TB/s); with a row's
// loads one after the other, each waited for by its conversion, 70 and 90.  At an odd
// address (2-byte accesses) 45 and 65, 24 for 20 without residual: whole lines all the same, but
// eight instructions for one; 1,537 channels, a fourth chunk, 57 and 78.  2 x 1,536: 2.6,
// a launch.  512 workgroups of the gradient: each sum is one row to read again.
#include "hier_launch.h"
#include "hier_types.h"

#include <algorithm>

namespace hier {
namespace {

// ---- sums of partial rows ----------------------------------------------------

constexpr int kCols = 32, kLines = 32;

__global__ __launch_bounds__(kCols * kLines) void sum_rows_kernel(const float* partial, int64_t rows, int64_t groups,
                                                                  int64_t C, void* out, int type) {
  __shared__ float part[kLines][kCols + 1];
  const int col = threadIdx.x % kCols, line = threadIdx.x / kCols;
  const int64_t c = (int64_t)blockIdx.x * kCols + col;
  for (int64_t g = blockIdx.y; g < groups; g += gridDim.y) {
    const float* p = partial + g * rows * C + c;
    float s = 0.f;
    if (c < C) {
      int64_t r = line;
      for (; r + 7 * kLines < rows; r += 8 * kLines) {   // eight loads in flight
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[(r + i * kLines) * C];
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
      }
      for (; r < rows; r += kLines) s += p[r * C];
    }
    part[line][col] = s;
    __syncthreads();
#pragma unroll
    for (int n = kLines / 2; n > 0; n /= 2) {
      if (line < n) part[line][col] += part[line + n][col];
      __syncthreads();
    }
    if (line == 0 && c < C) {
      const int64_t at = g * C + c;
      const float v = part[0][col];
      if (type == HIER_FP32) static_cast<float*>(out)[at] = v;
      else if (type == HIER_BF16) static_cast<__bf16*>(out)[at] = (__bf16)v;
      else static_cast<_Float16*>(out)[at] = (_Float16)v;
    }
  }
}

// ---- rows in registers -------------------------------------------------------

// A lane's channels of a row: chunk i of eight, i < NCH.  VEC 8: eight
// neighbouring channels; VEC 1: every (64 * WPR)-th.
template <int VEC, int WPR>
__device__ __forceinline__ int channel(int i, int j, int t) {
  return VEC == 8 ? 8 * (i * 64 * WPR + t) + j : (8 * i + j) * 64 * WPR + t;
}

// Chunk i of a row as it lies in memory.  Lanes past the last channel read the
// row's end and get zeros in `values`: without a branch around them all of a
// row's loads leave together.
template <typename T, int VEC>
struct Raw {
  w32x4 w;
};
template <typename T>
struct Raw<T, 1> {
  T v[8];
};
template <typename T, int VEC, int WPR>
__device__ __forceinline__ Raw<T, VEC> fetch(const T* row, int i, int t, int C) {
  Raw<T, VEC> r;
  if constexpr (VEC == 8) {
    r.w = *reinterpret_cast<const w32x4*>(row + min(channel<8, WPR>(i, 0, t), C - 8));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = row[min(channel<1, WPR>(i, j, t), C - 1)];
  }
  return r;
}
template <typename T, int VEC, int WPR>
__device__ __forceinline__ void values(const Raw<T, VEC>& r, int i, int t, int C, float* f) {
  if constexpr (VEC == 8) {
    widen<T>(r.w, f);
    const bool in = channel<8, WPR>(i, 0, t) < C;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = in ? f[j] : 0.f;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = channel<1, WPR>(i, j, t) < C ? (float)r.v[j] : 0.f;
  }
}
template <typename T, int VEC, int WPR>
__device__ __forceinline__ void load8(const T* row, int i, int t, int C, float* f) {
  values<T, VEC, WPR>(fetch<T, VEC, WPR>(row, i, t, C), i, t, C, f);
}

template <typename T, int VEC, int WPR>
__device__ __forceinline__ void store8(T* row, int i, int t, int C, const float* f) {
  if constexpr (VEC == 8) {
    const int c = channel<8, WPR>(i, 0, t);
    if (c < C) *reinterpret_cast<w32x4*>(row + c) = narrow<T>(f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = channel<1, WPR>(i, j, t);
      if (c < C) row[c] = (T)f[j];
    }
  }
}

// The gain's values (any of the three types; 0 past the last channel).
template <int VEC, int WPR>
__device__ __forceinline__ void load_gain(const void* w, int type, int i, int t, int C, float* f) {
  if (type == HIER_FP32) {
    const float* p = static_cast<const float*>(w);
    if constexpr (VEC == 8) {
      const int c = channel<8, WPR>(i, 0, t), at = min(c, C - 8);
      const f32x4 lo = *reinterpret_cast<const f32x4*>(p + at), hi = *reinterpret_cast<const f32x4*>(p + at + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[j] = c < C ? lo[j] : 0.f;
        f[4 + j] = c < C ? hi[j] : 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = channel<1, WPR>(i, j, t);
        f[j] = c < C ? p[min(c, C - 1)] : 0.f;
      }
    }
  } else if (type == HIER_BF16) {
    load8<__bf16, VEC, WPR>(static_cast<const __bf16*>(w), i, t, C, f);
  } else {
    load8<_Float16, VEC, WPR>(static_cast<const _Float16*>(w), i, t, C, f);
  }
}

// Sum over the WPR waves that share a row (every lane gets it).
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* lds) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d, 64);
  if constexpr (WPR > 1) {
    const int wave = threadIdx.x / 64;
    __syncthreads();                     // the last sum has been read
    if (threadIdx.x % 64 == 0) lds[wave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) v += lds[i];
  }
  return v;
}

template <int WPR>
constexpr int threads_of() { return WPR == 16 ? 1024 : 256; }

template <typename T, int VEC, int WPR, int NCH>
__global__ __launch_bounds__(threads_of<WPR>()) void norm_kernel(HierRmsNormArgs a) {
  __shared__ float lds[16];
  const int t = threadIdx.x % (64 * WPR);
  const int64_t group = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;      // (launch_grid)
  const int64_t row = WPR == 1 ? group * 4 + threadIdx.x / 64 : group;
  if (row >= a.M) return;                // (WPR > 1: the whole workgroup or none of it)
  float h[NCH][8], w[NCH][8];
  float sq = 0.f;
  Raw<T, VEC> xr[NCH], rr[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) xr[i] = fetch<T, VEC, WPR>(static_cast<const T*>(a.x) + row * a.x_ss, i, t, a.C);
  if (a.r)
#pragma unroll
    for (int i = 0; i < NCH; ++i) rr[i] = fetch<T, VEC, WPR>(static_cast<const T*>(a.r) + row * a.r_ss, i, t, a.C);
#pragma unroll
  for (int i = 0; i < NCH; ++i) load_gain<VEC, WPR>(a.w, a.gain_type, i, t, a.C, w[i]);
#pragma unroll
  for (int i = 0; i < NCH; ++i) values<T, VEC, WPR>(xr[i], i, t, a.C, h[i]);
  if (a.r) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float r[8];
      values<T, VEC, WPR>(rr[i], i, t, a.C, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] += r[j];
      store8<T, VEC, WPR>(static_cast<T*>(a.h) + row * a.h_ss, i, t, a.C, h[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) sq = fmaf(h[i][j], h[i][j], sq);
  const float s = 1.f / sqrtf(row_sum<WPR>(sq, lds) / (float)a.C + a.eps);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = h[i][j] * s * w[i][j];
    store8<T, VEC, WPR>(static_cast<T*>(a.y) + row * a.y_ss, i, t, a.C, y);
  }
}

template <typename T, int VEC, int WPR, int NCH>
__global__ __launch_bounds__(threads_of<WPR>()) void norm_bwd_kernel(HierRmsNormBwdArgs a) {
  constexpr int ROWS = WPR == 1 ? 4 : 1;          // rows that a workgroup has in hand
  __shared__ float lds[16];
  __shared__ float sums[WPR == 1 ? 4 * NCH * 512 : 1];
  const int t = threadIdx.x % (64 * WPR);
  float w[NCH][8], dw[NCH][8];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    load_gain<VEC, WPR>(a.w, a.gain_type, i, t, a.C, w[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.f;
  }
  const int64_t first = (int64_t)blockIdx.x * ROWS + (WPR == 1 ? threadIdx.x / 64 : 0);
  for (int64_t row = first; row < a.M; row += (int64_t)gridDim.x * ROWS) {
    float h[NCH][8], g[NCH][8];
    float sq = 0.f, dot = 0.f;
    Raw<T, VEC> xr[NCH], rr[NCH], gr[NCH], dr[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      xr[i] = fetch<T, VEC, WPR>(static_cast<const T*>(a.x) + row * a.x_ss, i, t, a.C);
      gr[i] = fetch<T, VEC, WPR>(static_cast<const T*>(a.dy) + row * a.dy_ss, i, t, a.C);
    }
    if (a.r)
#pragma unroll
      for (int i = 0; i < NCH; ++i) rr[i] = fetch<T, VEC, WPR>(static_cast<const T*>(a.r) + row * a.r_ss, i, t, a.C);
    if (a.dh)
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        dr[i] = fetch<T, VEC, WPR>(static_cast<const T*>(a.dh) + row * a.dh_ss, i, t, a.C);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      values<T, VEC, WPR>(xr[i], i, t, a.C, h[i]);
      values<T, VEC, WPR>(gr[i], i, t, a.C, g[i]);
    }
    if (a.r)
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        float r[8];
        values<T, VEC, WPR>(rr[i], i, t, a.C, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] += r[j];
      }
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(h[i][j], h[i][j], sq);
    const float s = 1.f / sqrtf(row_sum<WPR>(sq, lds) / (float)a.C + a.eps);
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] *= s;
        dw[i][j] = fmaf(g[i][j], h[i][j], dw[i][j]);
        g[i][j] *= w[i][j];
        dot = fmaf(g[i][j], h[i][j], dot);
      }
    const float mean = row_sum<WPR>(dot, lds) / (float)a.C;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float d[8] = {};
      if (a.dh) values<T, VEC, WPR>(dr[i], i, t, a.C, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = fmaf(s, fmaf(-h[i][j], mean, g[i][j]), d[j]);
      store8<T, VEC, WPR>(static_cast<T*>(a.dx) + row * a.dx_ss, i, t, a.C, d);
    }
  }
  float* out = a.partial + (int64_t)blockIdx.x * a.C;
  if constexpr (WPR == 1) {
    float* mine = sums + (threadIdx.x / 64) * NCH * 512;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) mine[(8 * i + j) * 64 + t] = dw[i][j];
    __syncthreads();
    for (int e = threadIdx.x; e < NCH * 512; e += 256) {
      const int c = channel<VEC, 1>(e / 512, e / 64 % 8, e % 64);
      if (c < a.C)
        out[c] = (sums[e] + sums[NCH * 512 + e]) + (sums[2 * NCH * 512 + e] + sums[3 * NCH * 512 + e]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = channel<VEC, WPR>(i, j, t);
        if (c < a.C) out[c] = dw[i][j];
      }
  }
}

// Workgroups of the gradient: eight waves a CU read and write at the rate of
// memory, and each leaves one row of sums.
constexpr int64_t kBwdGroups = 512;

int64_t bwd_groups(int64_t M, int64_t C) {
  return std::min(C <= 2048 ? (M + 3) / 4 : M, kBwdGroups);
}

template <typename T, int VEC, int WPR, int NCH>
int launch(const HierRmsNormArgs& a, hipStream_t st) {
  const Grid grid = launch_grid(WPR == 1 ? (a.M + 3) / 4 : a.M, threads_of<WPR>());
  HIER_REQUIRE(grid.x > 0, HIER_EUNSUPPORTED, "rms_norm: too many rows");
  hipLaunchKernelGGL((norm_kernel<T, VEC, WPR, NCH>), dim3(grid.x, grid.y), dim3(threads_of<WPR>()), 0, st, a);
  return check_launch("norm_kernel");
}
template <typename T, int VEC, int WPR, int NCH>
int launch(const HierRmsNormBwdArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, WPR, NCH>), dim3((unsigned)bwd_groups(a.M, a.C)),
                     dim3(threads_of<WPR>()), 0, st, a);
  return check_launch("norm_bwd_kernel");
}

template <typename T, int VEC, typename A>
int by_channels(const A& a, hipStream_t st) {
  if (a.C <= 512) return launch<T, VEC, 1, 1>(a, st);
  if (a.C <= 1024) return launch<T, VEC, 1, 2>(a, st);
  if (a.C <= 1536) return launch<T, VEC, 1, 3>(a, st);
  if (a.C <= 2048) return launch<T, VEC, 1, 4>(a, st);
  if (a.C <= 4096) return launch<T, VEC, 4, 2>(a, st);
  if (a.C <= 6144) return launch<T, VEC, 4, 3>(a, st);
  if (a.C <= 8192) return launch<T, VEC, 4, 4>(a, st);
  return launch<T, VEC, 16, 2>(a, st);
}

template <typename A>
int by_type(const A& a, bool vec, hipStream_t st) {
  if (a.type == HIER_BF16) return vec ? by_channels<__bf16, 8>(a, st) : by_channels<__bf16, 1>(a, st);
  return vec ? by_channels<_Float16, 8>(a, st) : by_channels<_Float16, 1>(a, st);
}

template <typename A>
int check_common(const A& a, const char* who) {
  HIER_REQUIRE(a.M >= 0 && a.C >= 1, HIER_EINVAL, "%s: invalid M=%lld C=%d", who, (long long)a.M, a.C);
  HIER_REQUIRE(a.C <= 16384, HIER_EUNSUPPORTED, "%s: at most 16384 channels, got %d", who, a.C);
  HIER_REQUIRE(a.M < (1ll << 31), HIER_EUNSUPPORTED, "%s: too many rows", who);
  HIER_REQUIRE(a.type == HIER_BF16 || a.type == HIER_FP16, HIER_EUNSUPPORTED, "%s: bf16 or fp16 rows",
               who);
  HIER_REQUIRE(a.gain_type == HIER_BF16 || a.gain_type == HIER_FP16 || a.gain_type == HIER_FP32,
               HIER_EUNSUPPORTED, "%s: bf16, fp16 or fp32 gain", who);
  HIER_REQUIRE(number_in(a.eps, 0.f, 3.4e38f), HIER_EINVAL, "%s: eps must be a number of at least 0",
               who);
  return HIER_OK;
}

bool rows16(const void* p, int64_t ss) { return aligned16(p) && ss % 8 == 0; }

}  // namespace

int sum_rows(const float* partial, int64_t rows, int64_t groups, int64_t C, void* out, int type,
             hipStream_t stream) {
  hipLaunchKernelGGL(sum_rows_kernel,
                     dim3((unsigned)((C + kCols - 1) / kCols), (unsigned)std::min<int64_t>(groups, 65535)),
                     dim3(kCols * kLines), 0, stream, partial, rows, groups, C, out, type);
  return check_launch("sum_rows_kernel");
}

}  // namespace hier

using namespace hier;

extern "C" int hier_rms_norm(const HierRmsNormArgs* args, void* stream) {
  clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  const HierRmsNormArgs& a = *args;
  if (int rc = check_common(a, "rms_norm")) return rc;
  if (a.M == 0) return HIER_OK;
  HIER_REQUIRE(a.x && a.w && a.y && (!a.r || a.h), HIER_EINVAL, "rms_norm: NULL pointer");
  HIER_REQUIRE(a.x_ss >= 0 && a.y_ss >= a.C && (!a.r || (a.r_ss >= 0 && a.h_ss >= a.C)), HIER_EINVAL,
               "rms_norm: invalid row stride");
  const bool vec = a.C % 8 == 0 && aligned16(a.w) && rows16(a.x, a.x_ss) && rows16(a.y, a.y_ss) &&
                   (!a.r || (rows16(a.r, a.r_ss) && rows16(a.h, a.h_ss)));
  return by_type(a, vec, (hipStream_t)stream);
}

extern "C" int64_t hier_rms_norm_bwd_rows(const HierRmsNormBwdArgs* a) {
  return a ? bwd_groups(a->M, a->C) : -1;
}

extern "C" int hier_rms_norm_bwd(const HierRmsNormBwdArgs* args, void* stream) {
  clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  HierRmsNormBwdArgs a = *args;
  if (int rc = check_common(a, "rms_norm_bwd")) return rc;
  HIER_REQUIRE(a.M >= 1, HIER_EINVAL, "rms_norm_bwd: no rows");
  HIER_REQUIRE(a.x && a.w && a.dy && a.dx && a.dw && a.partial, HIER_EINVAL, "rms_norm_bwd: NULL pointer");
  HIER_REQUIRE(a.x_ss >= 0 && a.dy_ss >= 0 && a.dx_ss >= a.C && (!a.r || a.r_ss >= 0) &&
                   (!a.dh || a.dh_ss >= 0),
               HIER_EINVAL, "rms_norm_bwd: invalid row stride");
  HIER_REQUIRE(a.partial_rows >= bwd_groups(a.M, a.C), HIER_EINVAL,
               "rms_norm_bwd: partial holds %lld rows, needs %lld", (long long)a.partial_rows,
               (long long)bwd_groups(a.M, a.C));
  const bool vec = a.C % 8 == 0 && aligned16(a.w) && rows16(a.x, a.x_ss) && rows16(a.dy, a.dy_ss) &&
                   rows16(a.dx, a.dx_ss) && (!a.r || rows16(a.r, a.r_ss)) &&
                   (!a.dh || rows16(a.dh, a.dh_ss));
  const bool one = bwd_groups(a.M, a.C) == 1;        // its row of sums is dw
  if (one) a.partial = a.dw;
  if (int rc = by_type(a, vec, (hipStream_t)stream)) return rc;
  return one ? HIER_OK : sum_rows(a.partial, bwd_groups(a.M, a.C), 1, a.C, a.dw, HIER_FP32, (hipStream_t)stream);
}
