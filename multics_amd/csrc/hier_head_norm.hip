// RMSNorm of queries and keys for each head, gain and position rotation in one
// pass, and its gradient.
//
//   r = 1 / sqrt(mean_d(x_d^2) + eps)          over one head's D channels
//   y_d = x_d r w_d                            gain w[D], shared by the heads
//   (y_2i, y_2i+1) -> (y_2i c_i - y_2i+1 s_i,  y_2i s_i + y_2i+1 c_i)
//
// and backwards, from the inputs (nothing is kept by the forward):
//   dn = the inverse rotation of dy;  dw_d = sum over tokens and heads of dn_d x_d r
//   dh = dn w;  dx = r (dh - x r mean_d(dh x r))
// All of it in fp32, one rounding to bf16 at the store.
//
// Both are bound by HBM: every input is read once and every output written
// once, a lane holding eight neighbouring channels (16 bytes, four rotated
// pairs), a head 8 or 16 lanes, so that its sums are DPP adds and nothing goes
// through LDS.  6,678 tokens of 24 + 24 heads of 128 (167 MB): 36.6 us,
// 4.6 TB/s; the gradient of 18,816 such tokens (703 MB): 149 us, 4.7 TB/s; a
// large copy reaches 4.8 to 5.0.
#include "hier_common.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
// Groups of heads (64 lanes x 8 channels) that a wave of the forward takes.
constexpr int kGroups = 6;

template <int D>
struct Lanes {
  static constexpr int PER_HEAD = D / 8;          // lanes of one head, 8 channels each
  static constexpr int HEADS = 64 / PER_HEAD;     // heads of one 64-lane group
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
// Sum over the lanes of a head (8 or 16 neighbours), left in each of them.
template <int D>
__device__ __forceinline__ float head_sum(float v) {
  v = dpp_add<0xB1>(v);               // quad_perm [1,0,3,2]
  v = dpp_add<0x4E>(v);               // quad_perm [2,3,0,1]
  if constexpr (D == 128) {
    v = dpp_add<0x124>(v);            // row_ror:4
    return dpp_add<0x128>(v);         // row_ror:8
  }
  return dpp_add<0x141>(v);           // row_half_mirror: the other quad of 8
}

__device__ __forceinline__ void unpack(const u32x4& w, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ u32x4 pack(const float* x) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 v = {x[2 * i], x[2 * i + 1]};
    w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  }
  return w;
}

__device__ __forceinline__ void load8(const float* p, float* x) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}

// The gain of channels [d, d + 8).
__device__ __forceinline__ void load_gain(const void* w, int bf16, int d, float* x) {
  if (bf16)
    unpack(*reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(w) + d), x);
  else
    load8(static_cast<const float*>(w) + d, x);
}

template <int D>
__device__ __forceinline__ float inv_rms(const float* x, float eps) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
  return 1.f / sqrtf(fmaf(head_sum<D>(ss), 1.f / D, eps));
}

// One wave per token, tensor and kGroups groups of heads (24 heads of 128 or 48
// of 64): the groups' loads are all in flight at once, and cos, sin and the gain
// stay in registers over them.
template <int D>
__global__ __launch_bounds__(kThreads) void head_norm_kernel(HierHeadNormArgs a, int units_q,
                                                             int units, int64_t waves) {
  using L = Lanes<D>;
  const int64_t wave = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave >= waves) return;
  const int64_t t = wave / units;
  int u = (int)(wave - t * units);
  const bool is_k = u >= units_q;
  if (is_k) u -= units_q;
  const int lane = threadIdx.x & 63, sub = lane % L::PER_HEAD, d = 8 * sub;
  const int H = is_k ? a.Hk : a.Hq;
  const uint16_t* x = (is_k ? a.kx + t * a.kx_ss : a.qx + t * a.qx_ss) + d;
  uint16_t* y = (is_k ? a.k_out + t * a.k_ss : a.q_out + t * a.q_ss) + d;
  const int64_t y_sh = is_k ? a.k_sh : a.q_sh;
  const int h0 = u * kGroups * L::HEADS + lane / L::PER_HEAD;
  u32x4 xw[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int h = h0 + g * L::HEADS;
    xw[g] = h < H ? *reinterpret_cast<const u32x4*>(x + (int64_t)h * D) : u32x4{0, 0, 0, 0};
  }
  float w[8];
  load_gain(is_k ? a.norm_k_w : a.norm_q_w, a.gain_bf16, d, w);
  const f32x4 c = *reinterpret_cast<const f32x4*>(a.rope_cos + t * (D / 2) + 4 * sub);
  const f32x4 s = *reinterpret_cast<const f32x4*>(a.rope_sin + t * (D / 2) + 4 * sub);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int h = h0 + g * L::HEADS;
    float v[8], o[8];
    unpack(xw[g], v);
    const float r = inv_rms<D>(v, a.eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = v[2 * i] * r * w[2 * i], q = v[2 * i + 1] * r * w[2 * i + 1];
      o[2 * i] = p * c[i] - q * s[i];
      o[2 * i + 1] = p * s[i] + q * c[i];
    }
    if (h < H) *reinterpret_cast<u32x4*>(y + (int64_t)h * y_sh) = pack(o);
  }
}

// Workgroups [0, rows_q) take runs of q's tokens, [rows_q, rows) of k's; the
// waves of a workgroup take the tokens of its run in turn and keep the gain's
// sums of their 8 channels.  Each workgroup writes one fp32 row of sums, and
// gain_sum_kernel adds the rows in their order: the same sums every time.
template <int D>
__global__ __launch_bounds__(kThreads) void head_norm_bwd_kernel(HierHeadNormBwdArgs a, int rows_q,
                                                                 int rows_k) {
  using L = Lanes<D>;
  __shared__ float lds[kWaves][D];
  const bool is_k = (int)blockIdx.x >= rows_q;
  const int row = is_k ? blockIdx.x - rows_q : blockIdx.x, rows = is_k ? rows_k : rows_q;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sub = lane % L::PER_HEAD, d = 8 * sub;
  const int H = is_k ? a.Hk : a.Hq;
  const uint16_t* xb = (is_k ? a.kx : a.qx) + d;
  const uint16_t* gb = (is_k ? a.dk : a.dq) + d;
  uint16_t* ob = (is_k ? a.dkx : a.dqx) + d;
  const int64_t x_ss = is_k ? a.kx_ss : a.qx_ss, g_ss = is_k ? a.dk_ss : a.dq_ss,
                g_sh = is_k ? a.dk_sh : a.dq_sh, o_ss = (int64_t)H * D;
  float w[8], dw[8] = {};
  load_gain(is_k ? a.norm_k_w : a.norm_q_w, a.gain_bf16, d, w);
  const int64_t t1 = (int64_t)(row + 1) * a.S / rows;
  for (int64_t t = (int64_t)row * a.S / rows + wave; t < t1; t += kWaves) {
    const f32x4 c = *reinterpret_cast<const f32x4*>(a.rope_cos + t * (D / 2) + 4 * sub);
    const f32x4 s = *reinterpret_cast<const f32x4*>(a.rope_sin + t * (D / 2) + 4 * sub);
    for (int h0 = 0; h0 < H; h0 += L::HEADS) {
      const int h = h0 + lane / L::PER_HEAD;
      const bool in = h < H;
      u32x4 xw = {}, gw = {};
      if (in) {
        xw = *reinterpret_cast<const u32x4*>(xb + t * x_ss + (int64_t)h * D);
        gw = *reinterpret_cast<const u32x4*>(gb + t * g_ss + h * g_sh);
      }
      float x[8], g[8], dn[8], dot = 0.f;
      unpack(xw, x);
      unpack(gw, g);
      // (a lane without a head holds zeros: with eps = 0 their 0 * inf would
      // reach the gain's sums)
      const float rms = inv_rms<D>(x, a.eps), r = in ? rms : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dn[2 * i] = g[2 * i] * c[i] + g[2 * i + 1] * s[i];
        dn[2 * i + 1] = g[2 * i + 1] * c[i] - g[2 * i] * s[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= r;
        dw[i] = fmaf(dn[i], x[i], dw[i]);
        dn[i] *= w[i];
        dot = fmaf(dn[i], x[i], dot);
      }
      dot = head_sum<D>(dot) * (1.f / D);
#pragma unroll
      for (int i = 0; i < 8; ++i) dn[i] = r * (dn[i] - x[i] * dot);
      if (in) *reinterpret_cast<u32x4*>(ob + t * o_ss + (int64_t)h * D) = pack(dn);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int m = L::PER_HEAD; m < 64; m *= 2) dw[i] += __shfl_xor(dw[i], m, 64);
    if (lane < L::PER_HEAD) lds[wave][d + i] = dw[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < kWaves; ++j) v += lds[j][i];
    a.partial[(int64_t)blockIdx.x * D + i] = v;
  }
}

// dw[tensor][d] = the sum of its workgroups' rows: blockIdx.y the tensor, 16
// channels a workgroup, 16 threads a channel.
constexpr int kBatch = 16;
__global__ __launch_bounds__(kThreads) void gain_sum_kernel(HierHeadNormBwdArgs a, int rows_q,
                                                            int rows_k) {
  __shared__ float lds[16][17];
  const bool is_k = blockIdx.y != 0;
  const int rows = is_k ? rows_k : rows_q, col = threadIdx.x & 15, part = threadIdx.x >> 4;
  const float* p = a.partial + (is_k ? (int64_t)rows_q * a.D : 0) + blockIdx.x * 16 + col;
  float v = 0.f;
  int r = part;
  for (; r + 16 * (kBatch - 1) < rows; r += 16 * kBatch) {   // (loads of kBatch rows at once)
    float x[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) x[i] = p[(int64_t)(r + 16 * i) * a.D];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) v += x[i];
  }
  for (; r < rows; r += 16) v += p[(int64_t)r * a.D];
  lds[part][col] = v;
  __syncthreads();
  if (part != 0) return;
#pragma unroll
  for (int j = 1; j < 16; ++j) v += lds[j][col];
  (is_k ? a.dnorm_k : a.dnorm_q)[blockIdx.x * 16 + col] = v;
}

// Workgroups of the gradient for one tensor: at most eight tokens each until
// there are 1,024 over both tensors, four to a CU (18,816 tokens of 24 + 24 heads of 128:
// 149.7 us; 150.7 with 512, 155.1 with 2,048, whose rows of sums take longer to
// add up).
constexpr int kRowsAll = 1024;
int bwd_rows(int64_t S, int H, int H_all) {
  const int64_t most = (int64_t)kRowsAll * H / H_all, need = (S + 7) / 8;
  const int64_t rows = need < most ? need : most;
  return rows > 0 ? (int)rows : 1;
}

bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace

extern "C" int hier_head_prologue(const HierHeadNormArgs* args, void* stream) {
  hier::clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  const HierHeadNormArgs& a = *args;
  HIER_REQUIRE(a.D == 128 || a.D == 64, HIER_EUNSUPPORTED, "head_dim must be 64 or 128, got %d", a.D);
  HIER_REQUIRE(a.S >= 0 && a.Hq >= 1 && a.Hk >= 1, HIER_EINVAL, "invalid S=%lld Hq=%d Hk=%d",
               (long long)a.S, a.Hq, a.Hk);
  HIER_REQUIRE(hier::number_in(a.eps, 0.f, 3.4e38f), HIER_EINVAL,
               "eps must be a number of at least 0, got %g", (double)a.eps);
  if (a.S == 0) return HIER_OK;
  HIER_REQUIRE(a.qx && a.kx && a.norm_q_w && a.norm_k_w && a.rope_cos && a.rope_sin && a.q_out &&
                   a.k_out,
               HIER_EINVAL, "NULL tensor pointer");
  HIER_REQUIRE(al16(a.qx) && al16(a.kx) && al16(a.norm_q_w) && al16(a.norm_k_w) &&
                   al16(a.rope_cos) && al16(a.rope_sin) && al16(a.q_out) && al16(a.k_out),
               HIER_EINVAL, "tensors must be 16-byte aligned");
  HIER_REQUIRE(a.qx_ss % 8 == 0 && a.kx_ss % 8 == 0 && a.q_ss % 8 == 0 && a.q_sh % 8 == 0 &&
                   a.k_ss % 8 == 0 && a.k_sh % 8 == 0,
               HIER_EINVAL, "strides must keep 16-byte rows aligned");
  const int per_wave = kGroups * (a.D == 128 ? Lanes<128>::HEADS : Lanes<64>::HEADS);
  const int units_q = (int)(((int64_t)a.Hq + per_wave - 1) / per_wave);
  const int units_k = (int)(((int64_t)a.Hk + per_wave - 1) / per_wave);
  const int64_t waves = a.S * ((int64_t)units_q + units_k);
  const int64_t blocks = (waves + kWaves - 1) / kWaves;
  HIER_REQUIRE(a.S <= (1ll << 31) && blocks < (1ll << 24), HIER_EUNSUPPORTED, "too many tokens");
  if (a.D == 128)
    hipLaunchKernelGGL(head_norm_kernel<128>, dim3((unsigned)blocks), dim3(kThreads), 0,
                       (hipStream_t)stream, a, units_q, units_q + units_k, waves);
  else
    hipLaunchKernelGGL(head_norm_kernel<64>, dim3((unsigned)blocks), dim3(kThreads), 0,
                       (hipStream_t)stream, a, units_q, units_q + units_k, waves);
  return hier::check_launch("head_norm_kernel");
}

extern "C" int hier_head_prologue_bwd(const HierHeadNormBwdArgs* args, void* stream) {
  hier::clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  const HierHeadNormBwdArgs& a = *args;
  HIER_REQUIRE(a.D == 128 || a.D == 64, HIER_EUNSUPPORTED, "head_dim must be 64 or 128, got %d", a.D);
  HIER_REQUIRE(a.S >= 1 && a.Hq >= 1 && a.Hk >= 1 && (int64_t)a.Hq + a.Hk <= (1 << 30), HIER_EINVAL,
               "invalid S=%lld Hq=%d Hk=%d", (long long)a.S, a.Hq, a.Hk);
  HIER_REQUIRE(hier::number_in(a.eps, 0.f, 3.4e38f), HIER_EINVAL,
               "eps must be a number of at least 0, got %g", (double)a.eps);
  HIER_REQUIRE(a.qx && a.kx && a.norm_q_w && a.norm_k_w && a.rope_cos && a.rope_sin && a.dq &&
                   a.dk && a.dqx && a.dkx && a.dnorm_q && a.dnorm_k && a.partial,
               HIER_EINVAL, "NULL tensor pointer");
  HIER_REQUIRE(al16(a.qx) && al16(a.kx) && al16(a.norm_q_w) && al16(a.norm_k_w) &&
                   al16(a.rope_cos) && al16(a.rope_sin) && al16(a.dq) && al16(a.dk) &&
                   al16(a.dqx) && al16(a.dkx),
               HIER_EINVAL, "tensors must be 16-byte aligned");
  HIER_REQUIRE(a.qx_ss % 8 == 0 && a.kx_ss % 8 == 0 && a.dq_ss % 8 == 0 && a.dq_sh % 8 == 0 &&
                   a.dk_ss % 8 == 0 && a.dk_sh % 8 == 0,
               HIER_EINVAL, "strides must keep 16-byte rows aligned");
  HIER_REQUIRE(a.S <= (1ll << 31), HIER_EUNSUPPORTED, "too many tokens");
  const int rows_q = bwd_rows(a.S, a.Hq, a.Hq + a.Hk), rows_k = bwd_rows(a.S, a.Hk, a.Hq + a.Hk);
  HIER_REQUIRE(a.partial_rows >= (int64_t)rows_q + rows_k, HIER_EINVAL, "partial has %lld rows, needs %d",
               (long long)a.partial_rows, rows_q + rows_k);
  if (a.D == 128)
    hipLaunchKernelGGL(head_norm_bwd_kernel<128>, dim3(rows_q + rows_k), dim3(kThreads), 0,
                       (hipStream_t)stream, a, rows_q, rows_k);
  else
    hipLaunchKernelGGL(head_norm_bwd_kernel<64>, dim3(rows_q + rows_k), dim3(kThreads), 0,
                       (hipStream_t)stream, a, rows_q, rows_k);
  const int rc = hier::check_launch("head_norm_bwd_kernel");
  if (rc != HIER_OK) return rc;
  hipLaunchKernelGGL(gain_sum_kernel, dim3(a.D / 16, 2), dim3(kThreads), 0, (hipStream_t)stream, a,
                     rows_q, rows_k);
  return hier::check_launch("gain_sum_kernel");
}
