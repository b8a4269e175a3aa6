// Append to a paged KV cache held in 8 bits: K and V rows of a cached block to
// e4m3 codes in their pool rows, with one power-of-two scale for each block of
// 16 rows and head (the definition stands in hierattn.h).
//
//   e = min { e >= -100 : max|x| <= 448 * 2^e },   code = e4m3(x * 2^-e)
//
// x * 2^-e is exact, so a code is one rounding (to nearest even, at most half
// a step, 2^-4 of the value) away from the bf16 input, and code * 2^e is exact
// in bf16 again.  One pass: a wave holds a block of one head, K and V, in
// registers (16 rows x D x 2 B each), takes the two maxima and writes 1 byte a
// value.  Bound by HBM: 6,678 rows of 24 heads of 128 (82 MB read, 41 written):
// 26 us, 4.7 TB/s, what a large copy reaches.
#include "hier_common.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kBlock = HIER_FP8_BLOCK;

// Largest of the packed 15-bit magnitudes (the order of the values'
// magnitudes; 0x7f80 and above is not finite).
__device__ __forceinline__ uint32_t max_mag(uint32_t m, uint32_t w) {
  const uint32_t lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
  return max(m, max(lo, hi));
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d, 64));
  return v;
}

// Exponent + 127 of the scale of a block whose largest magnitude has these
// bits: 448 = 1.75 * 2^8, so bf16 1.m * 2^E needs E - 8, or one more when
// 1.m > 1.75.
__device__ __forceinline__ uint32_t scale_byte(uint32_t mag) {
  const int e = (int)(mag >> 7) - 127 - 8 + ((mag & 0x7fu) > 0x60u ? 1 : 0);
  return mag == 0 ? 127u : (uint32_t)(max(e, -100) + 127);
}

// Eight bf16 values over the scale 2^(byte - 127) as e4m3 codes.
__device__ __forceinline__ u32x2 codes(const u32x4& w, uint32_t byte) {
  const float scale = __uint_as_float(byte << 23);
  u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // (copies: a bit cast of a vector's element takes the whole vector's bits)
    const uint32_t w0 = w[2 * i], w1 = w[2 * i + 1];
    s16x2 c = {0, 0};
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, w0), scale, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, w1), scale, true);
    r[i] = __builtin_bit_cast(uint32_t, c);
  }
  return r;
}

template <int D>
__global__ __launch_bounds__(kThreads) void append_fp8_kernel(HierPageFp8Args a) {
  constexpr int LPR = D / 8;              // lanes of a row
  constexpr int RPS = 64 / LPR;           // rows of a step
  constexpr int STEPS = kBlock / RPS;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int groups = (a.H + kWaves - 1) / kWaves;
  const int b = blockIdx.x / groups, h = (blockIdx.x - b * groups) * kWaves + wave;
  if (h >= a.H) return;
  const int src = a.blocks[3 * (int64_t)b], dst = a.blocks[3 * (int64_t)b + 1],
            count = a.blocks[3 * (int64_t)b + 2];
  if (src < 0 || count < 1 || count > kBlock || src > a.n_rows - count || dst < 0 ||
      dst % kBlock != 0 || dst > a.pool_rows - kBlock)
    return;
  const int row = lane / LPR, d = 8 * (lane % LPR);
  const uint16_t* ks = a.k_src + src * a.k_src_ss + h * a.k_src_sh + d;
  const uint16_t* vs = a.v_src + src * a.v_src_ss + h * a.v_src_sh + d;
  u32x4 k[STEPS], v[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int r = i * RPS + row;
    k[i] = v[i] = u32x4{0, 0, 0, 0};
    if (r < count) {
      k[i] = *reinterpret_cast<const u32x4*>(ks + r * a.k_src_ss);
      v[i] = *reinterpret_cast<const u32x4*>(vs + r * a.v_src_ss);
    }
  }
  uint32_t mk = 0, mv = 0;
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) mk = max_mag(mk, k[i][j]), mv = max_mag(mv, v[i][j]);
  uint32_t bad = 0;                       // bit i: the lane's row of step i is not a number
  if (__ballot(max(mk, mv) >= 0x7f80u)) {
    mk = mv = 0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) m = max_mag(max_mag(m, k[i][j]), v[i][j]);
      const uint64_t rows = __ballot(m >= 0x7f80u) >> (row * LPR);
      if (rows & ((1ull << LPR) - 1)) {
        bad |= 1u << i;
        k[i] = v[i] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) mk = max_mag(mk, k[i][j]), mv = max_mag(mv, v[i][j]);
    }
  }
  const uint32_t ek = scale_byte(wave_max(mk)), ev = scale_byte(wave_max(mv));
  uint8_t* kd = a.k_pool + dst * a.pool_ss + h * a.pool_sh + d;
  uint8_t* vd = a.v_pool + dst * a.pool_ss + h * a.pool_sh + d;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int r = i * RPS + row;
    if (r >= count) continue;
    u32x2 kc = codes(k[i], ek);
    if (bad >> i & 1) kc = u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
    *reinterpret_cast<u32x2*>(kd + r * a.pool_ss) = kc;
    *reinterpret_cast<u32x2*>(vd + r * a.pool_ss) = codes(v[i], ev);
  }
  if (lane == 0) {
    const int64_t at = dst / kBlock * a.scale_ss + h * a.scale_sh;
    a.k_scale[at] = (uint8_t)ek;
    a.v_scale[at] = (uint8_t)ev;
  }
}

}  // namespace

extern "C" int hier_kv_append_fp8(const HierPageFp8Args* args, void* stream) {
  hier::clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  const HierPageFp8Args& a = *args;
  HIER_REQUIRE(a.D == 128 || a.D == 64, HIER_EUNSUPPORTED, "head_dim must be 64 or 128, got %d", a.D);
  HIER_REQUIRE(a.H >= 1 && a.n_blocks >= 0 && a.n_rows >= 0 && a.pool_rows >= 0 &&
                   a.pool_rows % kBlock == 0,
               HIER_EINVAL, "invalid H=%d n_blocks=%d n_rows=%d pool_rows=%lld", a.H, a.n_blocks,
               a.n_rows, (long long)a.pool_rows);
  if (a.n_blocks == 0) return HIER_OK;
  HIER_REQUIRE(a.k_src && a.v_src && a.blocks && a.k_pool && a.v_pool && a.k_scale && a.v_scale,
               HIER_EINVAL, "NULL pointer");
  auto aligned = [](const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; };
  HIER_REQUIRE(aligned(a.k_src, 16) && aligned(a.v_src, 16) && aligned(a.k_pool, 16) &&
                   aligned(a.v_pool, 16),
               HIER_EINVAL, "K/V rows must be 16-byte aligned");
  HIER_REQUIRE(a.k_src_ss % 8 == 0 && a.k_src_sh % 8 == 0 && a.v_src_ss % 8 == 0 &&
                   a.v_src_sh % 8 == 0 && a.pool_ss % 16 == 0 && a.pool_sh % 16 == 0,
               HIER_EINVAL, "strides must keep 16-byte rows aligned");
  const int64_t grid = (int64_t)a.n_blocks * (((int64_t)a.H + kWaves - 1) / kWaves);
  HIER_REQUIRE(grid < (1ll << 24), HIER_EUNSUPPORTED, "too many blocks of rows");
  if (a.D == 128)
    hipLaunchKernelGGL(append_fp8_kernel<128>, dim3((unsigned)grid), dim3(kThreads), 0,
                       (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(append_fp8_kernel<64>, dim3((unsigned)grid), dim3(kThreads), 0,
                       (hipStream_t)stream, a);
  return hier::check_launch("append_fp8_kernel");
}
