// Block-sparse, frame-causal attention forward over a paged KV cache held in
// 8 bits (e4m3 codes, a power-of-two scale for 16 pool rows and a head; see
// hierattn.h), for gfx950.
//
//   S = (Q K8^T) 2^ek / sqrt(D),  O = softmax(S masked) (V8 2^ev)
//
// Work items, key lists and row addressing are those of hier_attn_fwd.hip: up
// to 128 query rows of one stream and head against the stream's key list, 64
// keys at a time through LDS; rows that see no key give 0.
//
// Q K^T runs on v_mfma_scale_f32_32x32x64_f8f6f4 straight from the codes, the
// key's scale as the instruction's block scale.  A bf16 query has 8
// significant bits and an e4m3 code 4, so a row of Q enters as two codes,
// q = hi + lo, both over powers of two: the rest q - hi is at most half a step
// of hi (8 of the 16 units that q resolves there), an integer below 16 units
// and so a code itself.  The split is exact for every element down to 2^-14
// of its row's largest; below that the error is at most 2^-22 of that
// largest.  Two 8-bit products cost what one in bf16 does, and K needs no
// conversion.
//
// V is converted when its tile is staged (v_cvt_scalef32_pk_bf16_fp8, exact:
// code and scale fit a bf16) and P V runs on v_mfma_f32_32x32x16_bf16 with P
// rounded to bf16; the row sum adds the rounded weights, so a weight's
// rounding (at most 2^-8 of it) reaches the result only as the spread of such
// roundings over the keys.  m, l and O are fp32.
#include "hier_common.h"
#include "hier_launch.h"
#include "hier_tile.h"

namespace {

using namespace hier::tile;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
// As in the bf16 forward: a lane's sum of a block above kSumMax refreshes the
// running max.  Maxima are held in exp2 units (score * scale * log2 e), so that
// no scale takes kNoMax, the max of a row that has seen no key, past fp32.
constexpr float kSumMax = 16.f * 256.f;
constexpr float kNoMax = -1e30f;
constexpr float kLn2 = 0.6931471805599453f;

template <int D>
struct Geo8 {
  static constexpr int NS = D / 64;          // 64-wide d-steps of Q K^T
  static constexpr int CPR = D / 16;         // 16-byte chunks of a row of codes
  static constexpr int NL = kSlab * CPR / kThreads;   // chunks of a thread per tile
  static constexpr int KTILEB = kSlab * D;
};

// XOR mask on the 16-byte chunk index of row `row` of a K tile: 8 consecutive
// rows at one chunk column fall into different banks.
template <int D>
__device__ __forceinline__ int kswz(int row) {
  return D == 128 ? (row & 7) : ((row >> 1) & 3);
}

__device__ __forceinline__ float pow2_of(uint32_t byte) { return __uint_as_float(byte << 23); }

__device__ __forceinline__ uint32_t max_mag(uint32_t m, uint32_t w) {
  return max(m, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
}

template <int D>
struct Rows {
  i32x8 hi[Geo8<D>::NS], lo[Geo8<D>::NS];    // the row's codes, this lane's d
  int e_hi, e_lo;                            // their scales (exponent + 127)
  f32x16 o[Geo<D>::NDB];
  float m, l, alpha;                         // m in exp2 units
  int qtok, qframe;
  bool valid;
  uint32_t bits;   // OR over the sub-block's valid rows of 1 << query frame
};

// A lane's row of the item: its token, query frame and whether there is one.
template <class R>
__device__ __forceinline__ void row_of(R& r, const HierFwdFp8Args& a, const int32_t* it, int rel) {
  const int qbase = it[0], qstride = it[1], qlen = it[2], row_start = it[3], row_count = it[4];
  r.valid = rel < row_count;
  const int ri = row_start + (r.valid ? rel : 0);
  if (qstride < 0) {            // rows from the row table: (token, mask bit) pairs
    r.valid = r.valid && a.row_table != nullptr;
    const int2 tb = r.valid ? reinterpret_cast<const int2*>(a.row_table)[qbase + ri] : int2{0, 0};
    r.qtok = tb.x;
    r.qframe = tb.y;
  } else {
    r.qframe = ri / qlen;
    r.qtok = qbase + r.qframe * qstride + (ri - r.qframe * qlen);
  }
}

template <int D>
__device__ __forceinline__ void rows_init(Rows<D>& R, const HierFwdFp8Args& a, const int32_t* it,
                                          int head, int rrel, int lane) {
  row_of(R, a, it, rrel + (lane & 31));
  R.bits = wave_or(R.valid ? (1u << R.qframe) : 0u);
  const uint16_t* qp = a.q + (int64_t)R.qtok * a.q_ss + (int64_t)head * a.q_sh + 32 * (lane >> 5);
  u32x4 w[Geo8<D>::NS][4];
  uint32_t mag = 0;
#pragma unroll
  for (int s = 0; s < Geo8<D>::NS; ++s)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      w[s][c] = *reinterpret_cast<const u32x4*>(qp + 64 * s + 8 * c);
#pragma unroll
      for (int j = 0; j < 4; ++j) mag = max_mag(mag, w[s][c][j]);
    }
  const auto sw = __builtin_amdgcn_permlane32_swap(mag, mag, false, false);
  mag = max(sw[0], sw[1]);
  // the smallest power of two that takes the row's largest to at most 448
  int e = (int)(mag >> 7) - 127 - 8 + ((mag & 0x7fu) > 0x60u ? 1 : 0);
  e = max(e, -100);
  R.e_hi = e + 127;
  R.e_lo = e + 127 - 4;         // the rest is at most 16 (half a step at 448)
  const float up = pow2_of((uint32_t)R.e_hi), up_lo = pow2_of((uint32_t)R.e_lo);
#pragma unroll
  for (int s = 0; s < Geo8<D>::NS; ++s)
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int p = 0; p < 2; ++p) {            // four values: one dword of codes
        s16x2 h = {0, 0}, l = {0, 0};
        const uint32_t w0 = w[s][c][2 * p], w1 = w[s][c][2 * p + 1];
        h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(bf16x2, w0), up, false);
        h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(bf16x2, w1), up, true);
        const int hw = __builtin_bit_cast(int, h);
        const auto h0 = __builtin_amdgcn_cvt_pk_f32_fp8(hw, false);
        const auto h1 = __builtin_amdgcn_cvt_pk_f32_fp8(hw, true);
        l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(
            l, __uint_as_float(w0 << 16) - h0[0] * up,
            __uint_as_float(w0 & 0xffff0000u) - h0[1] * up, up_lo, false);
        l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(
            l, __uint_as_float(w1 << 16) - h1[0] * up,
            __uint_as_float(w1 & 0xffff0000u) - h1[1] * up, up_lo, true);
        R.hi[s][2 * c + p] = hw;
        R.lo[s][2 * c + p] = __builtin_bit_cast(int, l);
      }
#pragma unroll
  for (int db = 0; db < Geo<D>::NDB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) R.o[db][i] = 0.f;
  R.m = kNoMax;
  R.l = 0.f;
  R.alpha = 1.f;
}

// S^T of 32-key block kb: lane l holds key 32 kb + l % 32, d 64 s + 32 (l / 32) .. + 32.
template <int D>
__device__ __forceinline__ f32x16 qk_block(const Rows<D>& R, const char* ktile, const int* kscale,
                                           int kb, int lane) {
  const int key = kb * 32 + (lane & 31);
  const char* row = ktile + key * D;
  const int sw = kswz<D>(key), sk = kscale[key];
  f32x16 acc = {};
#pragma unroll
  for (int s = 0; s < Geo8<D>::NS; ++s) {
    const int c = 4 * s + 2 * (lane >> 5);
    const u32x4 x = *reinterpret_cast<const u32x4*>(row + 16 * (c ^ sw));
    const u32x4 y = *reinterpret_cast<const u32x4*>(row + 16 * ((c + 1) ^ sw));
    const i32x8 k = {(int)x[0], (int)x[1], (int)x[2], (int)x[3],
                     (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, R.hi[s], acc, 0, 0, 0, sk, 0, R.e_hi);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, R.lo[s], acc, 0, 0, 0, sk, 0, R.e_lo);
  }
  return acc;
}

// Set the scores of block kb that the lane's query frame may not see to -inf.
__device__ __forceinline__ void mask_block(f32x16& s, const uint32_t* mk, int kb, int qframe,
                                           int lane) {
#pragma unroll
  for (int g4 = 0; g4 < 4; ++g4) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(&mk[kb * 32 + 8 * g4 + 4 * (lane >> 5)]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t sel = (uint32_t)__builtin_amdgcn_sbfe((int)w[e], qframe, 1);
      const uint32_t x = __float_as_uint(s[4 * g4 + e]);
      s[4 * g4 + e] = __uint_as_float((x & sel) | (0xff800000u & ~sel));
    }
  }
}

// P of one 32-key block: exp2(s * c2 + nb) rounded to bf16, as the two P^T
// operands of the block; returns the lane's sum of the rounded P.
__device__ __forceinline__ float p_block(const f32x16& s, bf16x8* p, float c2, float nb) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    p[i >> 3][i & 7] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[i], c2, nb));
  const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
  float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    ps0 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p[c], p[c], 0, 1), one, ps0, false);
    ps1 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p[c], p[c], 2, 3), one, ps1, false);
    ps0 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p[c], p[c], 4, 5), one, ps0, false);
    ps1 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p[c], p[c], 6, 7), one, ps1, false);
  }
  return ps0 + ps1;
}

// Online softmax of one block with the lazily refreshed running max; true:
// O is to be scaled by R.alpha before the block's P V.
template <int D>
__device__ __forceinline__ bool softmax_block(Rows<D>& R, const f32x16& s, bf16x8* p, float c2) {
  const float ps = p_block(s, p, c2, -R.m);
  if (__ballot(!(ps <= kSumMax)) == 0) {
    R.l += ps;
    R.alpha = 1.f;
    return false;
  }
  float mx = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
  mx = pair_max(mx);
  const float m_new = fmaxf(R.m, mx * c2);
  R.alpha = __builtin_amdgcn_exp2f(R.m - m_new);
  R.m = m_new;
  R.l = R.l * R.alpha + p_block(s, p, c2, -m_new);
  return true;
}

template <int D>
__device__ __forceinline__ void rescale(Rows<D>& R) {
#pragma unroll
  for (int db = 0; db < Geo<D>::NDB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) R.o[db][i] *= R.alpha;
}

// O^T += V^T P^T over the two 16-key chunks of block kb.
template <int D>
__device__ __forceinline__ void pv_block(Rows<D>& R, const bf16x8* p, const char* vtile, int kb,
                                         int lane) {
  constexpr int HALF = (8 / Geo<D>::NI) * Geo<D>::ROWB;   // rows of keys +8
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int db = 0; db < Geo<D>::NDB; ++db) {
      const char* p0 = vtile + (2 * kb + j) * 16 * Geo<D>::ROWB + tr_read_off<D, kTrRead>(lane, db, 0);
      R.o[db] = mfma(tr_read(p0, p0 + HALF), p[j], R.o[db]);
    }
}

template <int D>
__device__ __forceinline__ void store_rows(const Rows<D>& R, const HierFwdFp8Args& a, int head,
                                           int split, int lane) {
  const float l = pair_sum(R.l);
  if (!R.valid) return;
  const int half = lane >> 5;
  if (a.splits > 1) {
    const int64_t at = ((int64_t)split * a.H + head) * a.q_rows + R.qtok;
    float* op = a.part_o + at * D;
#pragma unroll
    for (int db = 0; db < Geo<D>::NDB; ++db)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<f32x4*>(op + db * 32 + 8 * g4 + 4 * half) =
            f32x4{R.o[db][4 * g4], R.o[db][4 * g4 + 1], R.o[db][4 * g4 + 2], R.o[db][4 * g4 + 3]};
    if (half == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = float2{R.m, l};
    return;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint16_t* op = a.o + (int64_t)R.qtok * a.o_ss + (int64_t)head * a.o_sh;
#pragma unroll
  for (int db = 0; db < Geo<D>::NDB; ++db)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      u32x2 w;
      w[0] = (uint32_t)f2bf(R.o[db][4 * g4 + 0] * inv) | ((uint32_t)f2bf(R.o[db][4 * g4 + 1] * inv) << 16);
      w[1] = (uint32_t)f2bf(R.o[db][4 * g4 + 2] * inv) | ((uint32_t)f2bf(R.o[db][4 * g4 + 3] * inv) << 16);
      *reinterpret_cast<u32x2*>(op + db * 32 + 8 * g4 + 4 * half) = w;
    }
  if (a.lse && half == 0)
    a.lse[(int64_t)head * a.lse_stride_h + R.qtok] = l > 0.f ? fmaf(R.m, kLn2, __logf(l)) : -INFINITY;
}

template <int D>
__global__ __launch_bounds__(kThreads, 2) void attn_fp8_kernel(HierFwdFp8Args a, int total) {
  using G = Geo8<D>;
  __shared__ __align__(16) char lds_k[G::KTILEB];
  __shared__ __align__(16) char lds_v[Geo<D>::TILEB];
  __shared__ __align__(16) uint32_t lds_m[kSlab];
  __shared__ int lds_s[kSlab];
  const int logical = hier::xcd_logical(blockIdx.x, gridDim.x);
  if (logical >= total) return;
  const int per_head = a.n_items * a.splits;
  const int head = logical / per_head, rest = logical - head * per_head;
  const int item = rest / a.splits, split = rest - item * a.splits;
  const int32_t* it = a.tile_items + (int64_t)item * 8;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kv_off = it[5], nt = it[6] / kSlab;
  const int t0 = (int)((int64_t)nt * split / a.splits), t1 = (int)((int64_t)nt * (split + 1) / a.splits);
  const bool active = wave * 32 < it[4];
  const int kh = head / (a.H / a.Hk);
  const uint8_t* kp = a.k + kh * a.kv_sh;
  const uint8_t* vp = a.v + kh * a.kv_sh;
  const uint8_t* ksp = a.k_scale + kh * a.scale_sh;
  const uint8_t* vsp = a.v_scale + kh * a.scale_sh;
  const int32_t* idx = a.tile_kv_idx + kv_off;
  const uint32_t* masks = a.tile_kv_mask + kv_off;
  const uint32_t* blk = a.tile_blk_and + kv_off / kSlab;
  const float c2 = a.scale * 1.4426950408889634f;
  Rows<D> R;
  rows_init<D>(R, a, it, head, wave * 32, lane);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < G::NL; ++e) {
      const int ci = e * kThreads + tid, j = ci / G::CPR, c = ci % G::CPR;
      const int64_t row = idx[t * kSlab + j];
      const u32x4 kw = *reinterpret_cast<const u32x4*>(kp + row * a.kv_ss + 16 * c);
      const u32x4 vw = *reinterpret_cast<const u32x4*>(vp + row * a.kv_ss + 16 * c);
      const float sv = pow2_of(vsp[row / HIER_FP8_BLOCK * a.scale_ss]);
      *reinterpret_cast<u32x4*>(lds_k + j * D + 16 * (c ^ kswz<D>(j))) = kw;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        u32x4 b;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          b[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vw[2 * p + i], sv, false));
          b[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vw[2 * p + i], sv, true));
        }
        *reinterpret_cast<u32x4*>(lds_v + prow<D>(j) * Geo<D>::ROWB +
                                  16 * ((2 * c + p) ^ swz<D, kTrRead>(j))) = b;
      }
    }
    if (tid < kSlab) {
      const int64_t row = idx[t * kSlab + tid];
      lds_s[tid] = ksp[row / HIER_FP8_BLOCK * a.scale_ss];
      lds_m[tid] = masks[t * kSlab + tid];
    }
    __syncthreads();
    if (!active) continue;
    const bool masked = (blk[t] & R.bits) != R.bits;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f32x16 s = qk_block<D>(R, lds_k, lds_s, kb, lane);
      if (masked) mask_block(s, lds_m, kb, R.qframe, lane);
      bf16x8 p[2];
      if (softmax_block<D>(R, s, p, c2)) rescale<D>(R);
      pv_block<D>(R, p, lds_v, kb, lane);
    }
  }
  if (active) store_rows<D>(R, a, head, split, lane);
}

// Joins the splits of one item and head: rows in turn, D / 4 lanes a row.
template <int D>
__global__ __launch_bounds__(kThreads) void join_fp8_kernel(HierFwdFp8Args a) {
  constexpr int LPR = D / 4;
  struct { int qtok, qframe; bool valid; } r;
  const int head = blockIdx.x / a.n_items, item = blockIdx.x - head * a.n_items;
  const int32_t* it = a.tile_items + (int64_t)item * 8;
  const int d = 4 * (threadIdx.x % LPR);
  const int64_t step = (int64_t)a.H * a.q_rows;
  for (int rel = threadIdx.x / LPR; rel < it[4]; rel += kThreads / LPR) {
    row_of(r, a, it, rel);
    if (!r.valid) continue;
    const int64_t at = (int64_t)head * a.q_rows + r.qtok;
    float m = kNoMax;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[2 * (at + s * step)]);
    float l = 0.f;
    f32x4 o = {};
    for (int s = 0; s < a.splits; ++s) {
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (at + s * step));
      const float w = __builtin_amdgcn_exp2f(ml.x - m);
      const f32x4 p = *reinterpret_cast<const f32x4*>(a.part_o + (at + s * step) * D + d);
      l = fmaf(ml.y, w, l);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(p[i], w, o[i]);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    u32x2 w;
    w[0] = (uint32_t)f2bf(o[0] * inv) | ((uint32_t)f2bf(o[1] * inv) << 16);
    w[1] = (uint32_t)f2bf(o[2] * inv) | ((uint32_t)f2bf(o[3] * inv) << 16);
    *reinterpret_cast<u32x2*>(a.o + (int64_t)r.qtok * a.o_ss + (int64_t)head * a.o_sh + d) = w;
    if (a.lse && d == 0)
      a.lse[(int64_t)head * a.lse_stride_h + r.qtok] = l > 0.f ? fmaf(m, kLn2, __logf(l)) : -INFINITY;
  }
}

template <int D>
int launch(const HierFwdFp8Args& a, int64_t total, hipStream_t stream) {
  hipLaunchKernelGGL(attn_fp8_kernel<D>, dim3((unsigned)hier::xcd_grid(total)), dim3(kThreads), 0,
                     stream, a, (int)total);
  const int rc = hier::check_launch("attn_fp8_kernel");
  if (rc != HIER_OK || a.splits == 1) return rc;
  hipLaunchKernelGGL(join_fp8_kernel<D>, dim3((unsigned)(a.n_items * a.H)), dim3(kThreads), 0, stream,
                     a);
  return hier::check_launch("join_fp8_kernel");
}

}  // namespace

extern "C" int hier_attn_fwd_fp8(const HierFwdFp8Args* args, void* stream) {
  hier::clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  const HierFwdFp8Args& a = *args;
  HIER_REQUIRE(a.D == 128 || a.D == 64, HIER_EUNSUPPORTED, "head_dim must be 64 or 128, got %d", a.D);
  HIER_REQUIRE(a.H >= 1 && a.Hk >= 1 && a.H % a.Hk == 0, HIER_EINVAL,
               "H=%d must be a multiple of Hk=%d", a.H, a.Hk);
  HIER_REQUIRE(a.n_items >= 0 && a.kv_rows >= 0 && a.q_rows >= 0 && a.splits >= 1, HIER_EINVAL,
               "invalid n_items=%d kv_rows=%lld q_rows=%lld splits=%d", a.n_items,
               (long long)a.kv_rows, (long long)a.q_rows, a.splits);
  if (a.n_items == 0) return HIER_OK;
  HIER_REQUIRE(a.scale > 0.f && a.scale <= 1e30f, HIER_EINVAL, "the softmax scale must be positive, got %g",
               (double)a.scale);
  HIER_REQUIRE(a.q && a.k && a.v && a.k_scale && a.v_scale && a.o && a.tile_items && a.tile_kv_idx &&
                   a.tile_kv_mask && a.tile_blk_and,
               HIER_EINVAL, "NULL tensor pointer");
  HIER_REQUIRE(a.splits == 1 || (a.part_o && a.part_ml), HIER_EINVAL, "splits need part_o and part_ml");
  auto al16 = [](const void* p) { return ((uintptr_t)p & 15u) == 0; };
  HIER_REQUIRE(al16(a.q) && al16(a.k) && al16(a.v) && al16(a.o) && al16(a.tile_kv_idx) &&
                   al16(a.part_o) && al16(a.part_ml),
               HIER_EINVAL, "q/k/v/o, the key index list and the workspace must be 16-byte aligned");
  HIER_REQUIRE(a.q_ss % 8 == 0 && a.q_sh % 8 == 0 && a.kv_ss % 16 == 0 && a.kv_sh % 16 == 0 &&
                   a.o_ss % 4 == 0 && a.o_sh % 4 == 0,
               HIER_EINVAL, "strides must keep 16-byte rows aligned");
  const int64_t total = (int64_t)a.n_items * a.splits * a.H;
  HIER_REQUIRE((int64_t)a.n_items * a.splits < (1ll << 31) && total < (1ll << 24), HIER_EUNSUPPORTED,
               "too many work items");
  return a.D == 128 ? launch<128>(a, total, (hipStream_t)stream)
                    : launch<64>(a, total, (hipStream_t)stream);
}
