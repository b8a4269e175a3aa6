// Gradients of the cross attention (hier_cross_fwd.hip).  With P = exp(scale Q K^T - lse),
// dP = dO V^T, delta = rowsum(dO * O) and dS = P * (dP - delta):
//   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO,
// dK and dV summed over the query heads that share a key head (they are rows of one
// product, hier_cross.h).  The two kernels are laid out like the hierarchical
// backward's (hier_attn_bwd.hip), each gradient row written by one workgroup:
//
// dq      128 rows an item, four waves: K and V tiles through LDS, per 32-key block
//         S, dP, dQ.  Also writes -delta and lse log2(e) - 15 of every row, in the
//         order of the rows, for dkv.
// dkv     128 keys an item, eight waves: wave w makes S, P and dV of its 32 keys,
//         wave w + 4 of the same keys dP, dS and dK, P handed over through LDS as
//         fp16.  P is 2^15 times the weight throughout (hence the 15 above; dK and dV
//         are scaled back at the end): a weight is at most 1, and down to 2^-29 it keeps
//         fp16's eleven bits, as many keys as a call may have, while fp32 holds the sums
//         of gradients up to 10^33.  (lse in fp32 leaves a weight's
//         exponent off by 2^-23 of the score: past scores of 5 million one may come out
//         as 2, which fp16 does not hold.)  Items are few where the keys are
//         (an encoder's 512 are four a head): the rows may then be cut into splits, whose
//         fp32 sums a third kernel adds in their order.
// dP starts from -delta, as S does from -m in the forward: the subtraction is the
// matrix product's.
//
// Rounded to 16 bits: P (for dV) and dS, as the MFMAs' operands; and through the forward,
// O (delta is taken of it as it is given) and the weights whose sum lse is.  A result's
// relative error is that of its own rounding and dS's, 0.0024, where the others average out
// over some 200 keys, up to 0.0039 over a handful.
//
// Measured, bf16, D 128: four streams of 4,620 rows x 12 heads against 512 keys dq 124 us
// (three products, 703 TFLOP/s; MFMA busy 30 % of the time), dkv 141 (four, 824; 36 %); 8,192 x 8,192 x 16 heads both 1,670
// (823 TFLOP/s, counting five products).  No bank conflicts.
#include "hier_cross.h"

#include <algorithm>
#include <type_traits>

namespace hier {
namespace {

using namespace cross;
typedef __bf16 T;
constexpr float kUpLog2 = 15.f, kDown = 1.f / 32768.f;   // of dkv's P
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Launch {
  HierCrossBwdArgs a;
  Div div;
  int32_t row_tiles, key_tiles, splits, total, dq_splits;
  float* lse2;         // [B * Hk][row_tiles * 128], less kUpLog2
  float* delta;        // minus it
  float* part;         // [splits][dk, dv][B * Hk][Sk][D]; before that dQ's [dq_splits][B * Hk][rows][D]
};

template <int N, int R, int V>
__device__ __forceinline__ void sched_phase() {
  __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    if (V > 0) __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
  }
}

// 32 rows of a tile, from `s` on.
template <int D>
__device__ __forceinline__ f32x16 rows_mfma(f32x16 s, const u32x4* b, const char* tile, const int* off, int blk) {
  const char* base = tile + blk * 32 * Geo<D>::ROWB;
#pragma unroll
  for (int c = 0; c < Geo<D>::NC; ++c) s = gemm::mfma<T>(row_operand<T>(base, off[c]), b[c], s);
  return s;
}
// acc[d] += A^T p over the 32 rows of block blk of a tile.
template <int D>
__device__ __forceinline__ void tr_mfma(f32x16* acc, const u32x4* p, const char* tile, const int (*tr)[2], int blk) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int d = 0; d < Geo<D>::NDB; ++d) {
      const char* base = tile + (2 * blk + j) * 16 * Geo<D>::ROWB;
      acc[d] = gemm::mfma<T>(tr_operand(base + tr[d][0], base + tr[d][1]), p[j], acc[d]);
    }
}

template <int D>
__device__ __forceinline__ void store_acc(uint16_t* row, const f32x16* acc, float mul, int lane) {
  const int half = lane >> 5;
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      typedef T quad __attribute__((ext_vector_type(4)));
      quad v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)(acc[d][4 * g + e] * mul);
      *reinterpret_cast<u32x2*>(row + d * 32 + 8 * g + 4 * half) = __builtin_bit_cast(u32x2, v);
    }
}

template <int D>
__device__ __forceinline__ void store_part(float* row, const f32x16* acc, int lane) {
  const int half = lane >> 5;
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(row + d * 32 + 8 * g + 4 * half) =
          f32x4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
}

// ---- dQ ----------------------------------------------------------------------------

struct Stages {
  char* k[2];
  char* v[2];
};

template <int D>
struct QWork {
  u32x4 q[Geo<D>::NC], dov[Geo<D>::NC];
  f32x16 dq[Geo<D>::NDB];
  float lse2, ndelta, c2;
  int krow[Geo<D>::NC], vrow[Geo<D>::NC], ktr[Geo<D>::NDB][2];
  Rows64<D, kBothRead> ck;
  Rows64<D, kRowRead> cv;
  uint64_t kbase, vbase;
  int64_t k_ss, v_ss, len;
  const uint8_t* mask;
  int nt, wave, lane;
  bool active;
};

// P of a block in place of its scores; with MASKED, 0 for keys that are not seen.
template <bool MASKED>
__device__ __forceinline__ void p_exp(f32x16& s, float c2, float lse2, uint32_t bits, int lane) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float x = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -lse2));
    s[i] = !MASKED || key_bit(bits, i, lane) ? x : 0.f;
  }
}
__device__ __forceinline__ void ds_block(const f32x16& p, const f32x16& dp, u32x4* out) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    vec8<T> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (T)(p[8 * c + i] * dp[8 * c + i]);
    out[c] = __builtin_bit_cast(u32x4, v);
  }
}

template <bool MASK, int D>
__device__ __forceinline__ uint32_t mask_byte(const QWork<D>& w, int t) {
  if constexpr (MASK) return (int64_t)t * kSlab + w.lane < w.len ? w.mask[(int64_t)t * kSlab] : 0u;
  else return 0u;
}

// Tile t in stage PAR; tile t + 1 on its way into the other.
template <int D, bool MASK, bool MASKED, int PAR>
__device__ __forceinline__ void dq_tile(QWork<D>& w, int t, uint64_t seen, uint64_t next, const Stages& st) {
  const bool more = t + 1 < w.nt;
  const int64_t k1 = (int64_t)(t + 1) * kSlab;
  if (more)
    w.ck.template copy<MASK>(w.kbase + (uint64_t)(k1 * 2 * w.k_ss), w.len - k1, w.k_ss, next, st.k[PAR ^ 1], w.wave);
  const char* ks = st.k[PAR];
  const char* vs = st.v[PAR];
  constexpr int NC = Geo<D>::NC, NDB = Geo<D>::NDB;
  const f32x16 zero = {};
  f32x16 nd;
#pragma unroll
  for (int i = 0; i < 16; ++i) nd[i] = w.ndelta;
  f32x16 s0, dp0;
  if (w.active) {
    s0 = rows_mfma<D>(zero, w.q, ks, w.krow, 0);
    dp0 = rows_mfma<D>(nd, w.dov, vs, w.vrow, 0);
    p_exp<MASKED>(s0, w.c2, w.lse2, (uint32_t)seen, w.lane);
    sched_phase<NC, 1, 0>();
    sched_phase<NC, 1, 4>();
  }
  if (more)
    w.cv.template copy<MASK>(w.vbase + (uint64_t)(k1 * 2 * w.v_ss), w.len - k1, w.v_ss, next, st.v[PAR ^ 1], w.wave);
  if (w.active) {
    f32x16 s1 = rows_mfma<D>(zero, w.q, ks, w.krow, 1);
    u32x4 ds0[2], ds1[2];
    ds_block(s0, dp0, ds0);
    const f32x16 dp1 = rows_mfma<D>(nd, w.dov, vs, w.vrow, 1);
    p_exp<MASKED>(s1, w.c2, w.lse2, (uint32_t)(seen >> 32), w.lane);
    tr_mfma<D>(w.dq, ds0, ks, w.ktr, 0);
    ds_block(s1, dp1, ds1);
    tr_mfma<D>(w.dq, ds1, ks, w.ktr, 1);
    sched_phase<NC, 1, 7>();
    sched_phase<NC, 1, 4>();
    sched_phase<2 * NDB, 2, 7>();
    sched_phase<2 * NDB, 2, 0>();
  }
  tile::wait_copies();
  __syncthreads();
}

template <int D, bool MASK>
__global__ __launch_bounds__(256, 2) void cross_dq_kernel(Launch p) {
  __shared__ __align__(16) char k0[Geo<D>::TILEB], k1[Geo<D>::TILEB];
  __shared__ __align__(16) char v0[Geo<D>::TILEB], v1[Geo<D>::TILEB];
  const Stages st = {{k0, k1}, {v0, v1}};
  const int logical = xcd_logical(blockIdx.x, gridDim.x);
  const HierCrossArgs& a = p.a.f;
  const int per = p.row_tiles * p.dq_splits;
  if (logical >= a.B * a.Hk * per) return;
  const int hb = logical / per, in = logical - hb * per;
  const int split = in / p.row_tiles, rt = in - split * p.row_tiles;
  const int hk = hb / a.B, b = hb - hk * a.B, bh = b * a.Hk + hk;      // (as the forward's)
  QWork<D> w;
  w.lane = threadIdx.x & 63;
  w.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  w.len = a.Sk;
  if (a.kv_lens) w.len = min(max((int64_t)a.kv_lens[b], (int64_t)0), a.Sk);
  const int tiles = (int)((w.len + kSlab - 1) / kSlab);
  const int each = (tiles + p.dq_splits - 1) / p.dq_splits;
  const int t0 = min(split * each, tiles);
  w.nt = min(each, tiles - t0);
  const int64_t key0 = (int64_t)t0 * kSlab;
  w.len = min(w.len - key0, (int64_t)w.nt * kSlab);
  w.k_ss = a.k_ss;
  w.v_ss = a.v_ss;
  w.kbase = (uint64_t)a.k + 2 * (b * a.k_sb + hk * a.k_sh + key0 * a.k_ss);
  w.vbase = (uint64_t)a.v + 2 * (b * a.v_sb + hk * a.v_sh + key0 * a.v_ss);
  w.mask = MASK ? a.key_mask + b * a.mask_sb + key0 + w.lane : nullptr;
  w.ck.init(w.wave, w.lane, a.k_ss);
  w.cv.init(w.wave, w.lane, a.v_ss);
#pragma unroll
  for (int c = 0; c < Geo<D>::NC; ++c) {
    w.krow[c] = tile::row_read_off<D, kBothRead>(w.lane, c);
    w.vrow[c] = tile::row_read_off<D, kRowRead>(w.lane, c);
  }
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d) {
    w.ktr[d][0] = tile::tr_read_off<D, kBothRead>(w.lane, d, 0);
    w.ktr[d][1] = tile::tr_read_off<D, kBothRead>(w.lane, d, 1);
  }
  const uint32_t R = (uint32_t)(a.Sq * p.div.g);
  const uint32_t r0 = (uint32_t)rt * kRows + w.wave * 32;
  w.active = r0 < R;
  const bool valid = r0 + (w.lane & 31) < R;
  const uint32_t r = min(r0 + (w.lane & 31), R - 1);
  const uint32_t q = quotient(r, p.div);
  const int head = hk * (int)p.div.g + (int)(r - q * p.div.g);
  load_row<D>(w.q, static_cast<const uint16_t*>(a.q) + b * a.q_sb + (int64_t)q * a.q_ss + head * a.q_sh, w.lane);
  load_row<D>(w.dov,
              static_cast<const uint16_t*>(p.a.dout) + b * p.a.do_sb + (int64_t)q * p.a.do_ss + head * p.a.do_sh,
              w.lane);
  {
    u32x4 o[Geo<D>::NC];
    load_row<D>(o, static_cast<const uint16_t*>(a.o) + b * a.o_sb + (int64_t)q * a.o_ss + head * a.o_sh, w.lane);
    float d0 = 0.f, d1 = 0.f;
#pragma unroll
    for (int c = 0; c < Geo<D>::NC; ++c) {
      const vec8<T> x = __builtin_bit_cast(vec8<T>, w.dov[c]), y = __builtin_bit_cast(vec8<T>, o[c]);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        d0 = fmaf((float)x[e], (float)y[e], d0);
        d1 = fmaf((float)x[e + 1], (float)y[e + 1], d1);
      }
    }
    w.ndelta = -tile::pair_sum(d0 + d1);
  }
  const float lse = a.lse[((int64_t)b * a.Hq + head) * a.Sq + q];
  w.lse2 = lse == -INFINITY ? INFINITY : lse * kLog2e;
  w.c2 = a.scale * kLog2e;
  if (split == 0 && w.lane < 32) {       // rows past the last: P = 0, whatever dkv reads there
    const int64_t at = (int64_t)bh * p.row_tiles * kRows + r0 + w.lane;
    p.lse2[at] = valid ? w.lse2 - kUpLog2 : INFINITY;
    p.delta[at] = valid ? w.ndelta : 0.f;
  }
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.dq[d][i] = 0.f;
  if (w.nt > 0) {
    uint64_t seen = seen_keys<MASK>(w.len, 0, mask_byte<MASK>(w, 0));
    uint64_t next = seen_keys<MASK>(w.len, 1, mask_byte<MASK>(w, 1));
    uint32_t mb = mask_byte<MASK>(w, 2);
    w.ck.template copy<MASK>(w.kbase, w.len, w.k_ss, seen, k0, w.wave);
    w.cv.template copy<MASK>(w.vbase, w.len, w.v_ss, seen, v0, w.wave);
    tile::wait_copies();
    __syncthreads();
    auto after = [&](int t) {
      seen = next;
      next = seen_keys<MASK>(w.len, t + 2, mb);
      mb = mask_byte<MASK>(w, t + 3);
    };
    // whole tiles without masks, then the last (or all of them, with a mask)
    const int whole = MASK ? 0 : (int)(w.len / kSlab);
    int t = 0;
    for (; t + 1 < whole; t += 2) {
      dq_tile<D, MASK, false, 0>(w, t, seen, next, st);
      after(t);
      dq_tile<D, MASK, false, 1>(w, t + 1, seen, next, st);
      after(t + 1);
    }
    for (; t + 1 < w.nt; t += 2) {
      dq_tile<D, MASK, true, 0>(w, t, seen, next, st);
      after(t);
      dq_tile<D, MASK, true, 1>(w, t + 1, seen, next, st);
      after(t + 1);
    }
    if (t < w.nt) dq_tile<D, MASK, true, 0>(w, t, seen, next, st);
  }
  if (!w.active || !valid) return;
  if (p.dq_splits > 1)
    store_part<D>(p.part + ((int64_t)(split * a.B * a.Hk + bh) * R + r) * D, w.dq, w.lane);
  else
    store_acc<D>(static_cast<uint16_t*>(p.a.dq) + b * p.a.dq_sb + (int64_t)q * p.a.dq_ss + head * p.a.dq_sh, w.dq,
                 a.scale, w.lane);
}

// ---- dK, dV ------------------------------------------------------------------------

template <int D>
struct KWork {
  u32x4 kt[Geo<D>::NC];          // the lane's key's K (waves 0-3) or V (4-7)
  f32x16 acc[Geo<D>::NDB];       // dV or dK, transposed
  int row[Geo<D>::NC], tr[Geo<D>::NDB][2];
  uint32_t add[Geo<D>::NI];      // the lane's chunk in its rows
  int first;
  float c2;
  uint32_t R;
  int nt, wave, lane;
  bool active;
};

template <int D>
__global__ __launch_bounds__(512, 1) void cross_dkv_kernel(Launch p) {
  __shared__ __align__(16) char lds_q[3][Geo<D>::TILEB];
  __shared__ __align__(16) char lds_d[3][Geo<D>::TILEB];
  __shared__ __align__(16) char lds_w[3][2 * Geo<D>::MBYTES];
  __shared__ __align__(16) f16x8 lds_p[2 * 2 * 4 * 2 * 64];   // [tile parity][block][wave][half][lane]
  const int logical = xcd_logical(blockIdx.x, gridDim.x);
  if (logical >= p.total) return;
  const HierCrossArgs& a = p.a.f;
  const int per = p.key_tiles * p.splits;
  const int hb = logical / per, in = logical - hb * per;
  const int split = in / p.key_tiles, kt = in - split * p.key_tiles;
  const int hk = hb / a.B, b = hb - hk * a.B, bh = b * a.Hk + hk;
  KWork<D> w;
  w.lane = threadIdx.x & 63;
  const int wave8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool role_b = wave8 >= 4;
  w.wave = wave8 & 3;
  int64_t len = a.Sk;
  if (a.kv_lens) len = min(max((int64_t)a.kv_lens[b], (int64_t)0), a.Sk);
  const int64_t key0 = (int64_t)kt * kRows;
  const int64_t key = key0 + w.wave * 32 + (w.lane & 31);
  const bool exists = key < a.Sk;
  bool seen = key < len;
  if (a.key_mask && seen) seen = a.key_mask[b * a.mask_sb + key] != 0;
  w.R = (uint32_t)(a.Sq * p.div.g);
  const int tiles = (int)((w.R + kSlab - 1) / kSlab);
  const int each = (tiles + p.splits - 1) / p.splits;
  const int t0 = min(split * each, tiles);
  // (keys that nothing sees: zeros, without a pass over the rows)
  w.nt = key0 < len ? min(each, tiles - t0) : 0;
  w.active = key0 + w.wave * 32 < len;
  w.c2 = a.scale * kLog2e;
#pragma unroll
  for (int c = 0; c < Geo<D>::NC; ++c) {
    w.row[c] = tile::row_read_off<D, kBothRead>(w.lane, c);
    w.kt[c] = u32x4{0u, 0u, 0u, 0u};
  }
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d) {
    w.tr[d][0] = tile::tr_read_off<D, kBothRead>(w.lane, d, 0);
    w.tr[d][1] = tile::tr_read_off<D, kBothRead>(w.lane, d, 1);
#pragma unroll
    for (int i = 0; i < 16; ++i) w.acc[d][i] = 0.f;
  }
  if (seen) {
    if (role_b) load_row<D>(w.kt, static_cast<const uint16_t*>(a.v) + b * a.v_sb + key * a.v_ss + hk * a.v_sh, w.lane);
    else load_row<D>(w.kt, static_cast<const uint16_t*>(a.k) + b * a.k_sb + key * a.k_ss + hk * a.k_sh, w.lane);
  }
  {
    tile::Copier<D, kBothRead> c;
    c.init(w.wave, w.lane);
    w.first = c.idx_off;
#pragma unroll
    for (int e = 0; e < Geo<D>::NI; ++e) w.add[e] = c.add(e);
  }
  const float* lse2 = p.lse2 + (int64_t)bh * p.row_tiles * kRows;
  const float* delta = p.delta + (int64_t)bh * p.row_tiles * kRows;
  // rows of tile t: Q (waves 0-3) or dO (4-7), from the tile's first query on
  auto copy_rows = [&](auto rb, int t, int sg) {
    constexpr bool RB = decltype(rb)::value;
    const int64_t ss = RB ? p.a.do_ss : a.q_ss, sh = RB ? p.a.do_sh : a.q_sh;
    const uint32_t r0 = (uint32_t)(t0 + t) * kSlab;
    const uint32_t q0 = quotient(r0, p.div);
    const uint64_t base = (RB ? (uint64_t)p.a.dout + 2 * b * p.a.do_sb : (uint64_t)a.q + 2 * b * a.q_sb) +
                          2 * (hk * (int64_t)p.div.g * sh + (int64_t)q0 * ss);
    const u32x4 srd = {(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu, 0x7fffffffu, 0x00020000u};
    char* slot = RB ? lds_d[sg] : lds_q[sg];
#pragma unroll
    for (int e = 0; e < Geo<D>::NI; ++e) {
      const uint32_t r = r0 + w.first + e, q = quotient(r, p.div);
      const uint32_t v = (q - q0) * (uint32_t)(2 * ss) + (r - q * p.div.g) * (uint32_t)(2 * sh) + w.add[e];
      gemm::dma(srd, r < w.R ? v : gemm::kOut,
                (uint32_t)(uintptr_t)(slot + (16 * w.wave + Geo<D>::NR * e) * Geo<D>::ROWB));
    }
    if (!RB && w.wave == 0) tile::dma4(lse2 + r0, 4u * w.lane, lds_w[sg]);
    if (!RB && w.wave == 1) tile::dma4(delta + r0, 4u * w.lane, lds_w[sg] + Geo<D>::MBYTES);
  };
  f16x8* const pslot = lds_p + w.wave * 2 * 64 + w.lane;   // + parity * 1024 + block * 512 + half * 64

  // waves 0-3: S and P (2^15 times it) of a block of the tile in stage sg, kept as dV's
  // operand and handed over
  auto a_block = [&](int sg, int par, int qb, u32x4* pb) {
    const float* l2 = reinterpret_cast<const float*>(lds_w[sg]);
    const f32x16 zero = {};
    f32x16 x = rows_mfma<D>(zero, w.kt, lds_q[sg], w.row, qb);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 lw = *reinterpret_cast<const f32x4*>(&l2[qb * 32 + 8 * g + 4 * (w.lane >> 5)]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * g + e] = __builtin_amdgcn_exp2f(fmaf(x[4 * g + e], w.c2, -lw[e]));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      vec8<T> v;
      f16x8 ph;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = (T)x[8 * h + e];
        ph[e] = (_Float16)x[8 * h + e];
      }
      pb[h] = __builtin_bit_cast(u32x4, v);
      pslot[par * 1024 + qb * 512 + h * 64] = ph;
    }
  };
  // waves 4-7: dP - delta of a block; dS from the P handed over, dK
  auto b_dp = [&](int sg, int qb) {
    const float* dl = reinterpret_cast<const float*>(lds_w[sg] + Geo<D>::MBYTES);
    f32x16 init;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 dw = *reinterpret_cast<const f32x4*>(&dl[qb * 32 + 8 * g + 4 * (w.lane >> 5)]);
#pragma unroll
      for (int e = 0; e < 4; ++e) init[4 * g + e] = dw[e];
    }
    return rows_mfma<D>(init, w.kt, lds_d[sg], w.row, qb);
  };
  auto b_block = [&](int sg, int par, int qb, const f32x16& dp) {
    u32x4 ob[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f16x8 ph = pslot[par * 1024 + qb * 512 + h * 64];
      vec8<T> v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)((float)ph[e] * dp[8 * h + e]);
      ob[h] = __builtin_bit_cast(u32x4, v);
    }
    tr_mfma<D>(w.acc, ob, lds_q[sg], w.tr, qb);
  };

  auto run = [&](auto rb) {
    constexpr bool RB = decltype(rb)::value;
    const int nt = w.nt;
    copy_rows(rb, 0, 0);
    if (nt > 1) copy_rows(rb, 1, 1);
    tile::wait_copies();
    __syncthreads();
    u32x4 pb[2][2];
    f32x16 dp[2];
    if (w.active) {
      if constexpr (!RB) {
        a_block(0, 0, 0, pb[0]);
        a_block(0, 0, 1, pb[1]);
      } else {
        dp[0] = b_dp(0, 0);
        dp[1] = b_dp(0, 1);
      }
    }
    barrier_lds();        // P of tile 0 is there
    int s0 = 0, s1 = 1, s2 = 2;
    auto step = [&](int t, bool next) {
      if (t + 2 < nt) copy_rows(rb, t + 2, s2);
      if (w.active) {
        if constexpr (!RB) {
          u32x4 pn[2][2];
          if (next) {
            a_block(s1, (t + 1) & 1, 0, pn[0]);
            a_block(s1, (t + 1) & 1, 1, pn[1]);
          }
          tr_mfma<D>(w.acc, pb[0], lds_d[s0], w.tr, 0);      // dV^T += dO^T P
          tr_mfma<D>(w.acc, pb[1], lds_d[s0], w.tr, 1);
          if (next) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              pb[i][0] = pn[i][0];
              pb[i][1] = pn[i][1];
            }
          }
        } else {
          f32x16 dn[2];
          if (next) {
            dn[0] = b_dp(s1, 0);
            dn[1] = b_dp(s1, 1);
          }
          b_block(s0, t & 1, 0, dp[0]);                      // dK^T += Q^T dS
          b_block(s0, t & 1, 1, dp[1]);
          if (next) {
            dp[0] = dn[0];
            dp[1] = dn[1];
          }
        }
      }
      tile::wait_copies();
      __syncthreads();
      const int sx = s0;
      s0 = s1;
      s1 = s2;
      s2 = sx;
    };
    int t = 0;
    for (; t + 1 < nt; ++t) step(t, true);
    step(t, false);
  };
  if (w.nt > 0) {
    if (role_b) run(std::true_type{});
    else run(std::false_type{});
  }
  if (!exists) return;
  if (!seen) {            // whatever its column holds
#pragma unroll
    for (int d = 0; d < Geo<D>::NDB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) w.acc[d][i] = 0.f;
  }
  if (p.splits > 1) {
    store_part<D>(p.part + ((((int64_t)split * 2 + (role_b ? 0 : 1)) * a.B * a.Hk + bh) * a.Sk + key) * D, w.acc, w.lane);
  } else if (role_b) {
    store_acc<D>(static_cast<uint16_t*>(p.a.dk) + b * p.a.dk_sb + key * p.a.dk_ss + hk * p.a.dk_sh, w.acc,
                 a.scale * kDown, w.lane);
  } else {
    store_acc<D>(static_cast<uint16_t*>(p.a.dv) + b * p.a.dv_sb + key * p.a.dv_ss + hk * p.a.dv_sh, w.acc, kDown,
                 w.lane);
  }
}

// The splits' sums, in their order: four channels a thread of dK and dV (DQ: of dQ).
// Four splits' loads leave together, the last split's again past the end.
template <int D, bool DQ>
__global__ __launch_bounds__(256) void cross_grad_join_kernel(Launch p) {
  const HierCrossArgs& a = p.a.f;
  const int64_t rows = DQ ? (int64_t)a.B * a.Hq * a.Sq : (int64_t)a.B * a.Hk * a.Sk, n = rows * (D / 4);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (DQ ? n : 2 * n)) return;
  const bool dv = !DQ && i >= n;
  const int64_t j = dv ? i - n : i, row = j / (D / 4);
  const int d = 4 * (int)(j - row * (D / 4)), splits = DQ ? p.dq_splits : p.splits;
  const int64_t step = (DQ ? rows : 2 * rows) * D;
  const float* src = p.part + ((dv ? rows : 0) + row) * D + d;
  f32x4 s = {};
  for (int k = 0; k < splits; k += 4) {
    f32x4 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const f32x4*>(src + min(k + e, splits - 1) * step);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + e < splits) s += x[e];
  }
  const int64_t per = DQ ? (int64_t)a.Sq * p.div.g : a.Sk, bh = row / per, r = row - bh * per;
  const int b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  uint16_t* out;
  if constexpr (DQ) {
    const uint32_t q = quotient((uint32_t)r, p.div);
    const int head = hk * (int)p.div.g + (int)((uint32_t)r - q * p.div.g);
    out = static_cast<uint16_t*>(p.a.dq) + b * p.a.dq_sb + (int64_t)q * p.a.dq_ss + head * p.a.dq_sh;
  } else {
    out = dv ? static_cast<uint16_t*>(p.a.dv) + b * p.a.dv_sb + r * p.a.dv_ss + hk * p.a.dv_sh
             : static_cast<uint16_t*>(p.a.dk) + b * p.a.dk_sb + r * p.a.dk_ss + hk * p.a.dk_sh;
  }
  const float mul = DQ ? a.scale : dv ? kDown : a.scale * kDown;
  typedef T quad __attribute__((ext_vector_type(4)));
  quad v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (T)(s[e] * mul);
  *reinterpret_cast<u32x2*>(out + d) = __builtin_bit_cast(u32x2, v);
}

// Parts (SplitModel).  dK, dV, of the rows: 192 items of 73 tiles 132 us in one part, 152 in
// four (three whole rounds of workgroups, but every part starts, ends and leaves 128 KB of
// fp32 sums to join: the fourth of the CUs that is idle in one part is not worth that); 32 items of 128 tiles, D 64, 147 us with dq in one, 54
// in eight, 58 in sixteen.  dQ, of the keys: 12 items of 128
// tiles (one row each) 238 us with dK and dV in one part, 57 in 26.
int dkv_splits(const HierCrossArgs& a) {
  const double size = a.D == 128 ? 1.0 : 0.6;
  const int64_t items = (int64_t)a.B * a.Hk * row_tiles(a.Sk);
  const int64_t tiles = (a.Sq * (a.Hq / a.Hk) + kSlab - 1) / kSlab;
  return best_splits({256, 2.4 * size, 1.8 * size, 3, 8}, items, tiles, 8.0 * a.B * a.Hk * (double)a.Sk * a.D, 64);
}
int dq_splits(const HierCrossArgs& a) {
  const double size = a.D == 128 ? 1.0 : 0.6;
  const int64_t items = (int64_t)a.B * a.Hk * row_tiles(a.Sq * (a.Hq / a.Hk));
  return best_splits({512, 3.0 * size, 1.8 * size, 3.5, 2}, items, (a.Sk + kSlab - 1) / kSlab,
                     4.0 * a.B * a.Hq * (double)a.Sq * a.D, 64);
}

int64_t rows_bytes(const HierCrossArgs& a) {
  return (int64_t)a.B * a.Hk * row_tiles(a.Sq * (a.Hq / a.Hk)) * kRows * 4;
}

int64_t work_bytes(const HierCrossArgs& a) {
  const int sk = dkv_splits(a), sq = dq_splits(a);     // (dQ's parts are joined before the others are made)
  return 2 * rows_bytes(a) + std::max(sk > 1 ? (int64_t)sk * 2 * a.B * a.Hk * a.Sk * a.D * 4 : 0,
                                      sq > 1 ? (int64_t)sq * a.B * a.Hq * a.Sq * a.D * 4 : 0);
}

template <int D>
int launch(const Launch& p, hipStream_t st) {
  const HierCrossArgs& a = p.a.f;
  const int64_t items = (int64_t)a.B * a.Hk * p.row_tiles * p.dq_splits;
  auto join = [&](auto dq, int64_t rows) {
    const int64_t n = rows * (D / 4);
    hipLaunchKernelGGL((cross_grad_join_kernel<D, decltype(dq)::value>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0,
                       st, p);
    return check_launch("cross_grad_join_kernel");
  };
  if (items > 0) {
    const dim3 grid((unsigned)xcd_grid(items));
    if (a.key_mask) hipLaunchKernelGGL((cross_dq_kernel<D, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((cross_dq_kernel<D, false>), grid, dim3(256), 0, st, p);
    if (int rc = check_launch("cross_dq_kernel")) return rc;
    if (p.dq_splits > 1)
      if (int rc = join(std::true_type{}, (int64_t)a.B * a.Hq * a.Sq)) return rc;
  }
  if (p.total == 0) return HIER_OK;
  hipLaunchKernelGGL(cross_dkv_kernel<D>, dim3((unsigned)xcd_grid(p.total)), dim3(512), 0, st, p);
  if (int rc = check_launch("cross_dkv_kernel")) return rc;
  return p.splits == 1 ? HIER_OK : join(std::false_type{}, 2 * (int64_t)a.B * a.Hk * a.Sk);
}

}  // namespace
}  // namespace hier

using namespace hier;

extern "C" int64_t hier_cross_bwd_workspace(const HierCrossArgs* a) {
  clear_error();
  if (!a || a->D < 1 || a->Hk < 1 || a->Hq < a->Hk || a->B < 0 || a->Sq < 0 || a->Sk < 0) {
    fail(HIER_EINVAL, "cross attention: invalid sizes");
    return -1;
  }
  return work_bytes(*a);
}

extern "C" int hier_cross_attn_bwd(const HierCrossBwdArgs* args, void* stream) {
  clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  if (int rc = cross::check(args->f)) return rc;
  Launch p = {};
  p.a = *args;
  const HierCrossArgs& a = p.a.f;
  HIER_REQUIRE(a.type == HIER_BF16, HIER_EUNSUPPORTED, "cross attention: gradients are bf16 only");
  if (a.B == 0 || (a.Sq == 0 && a.Sk == 0)) return HIER_OK;
  HIER_REQUIRE(a.Sq == 0 || (a.lse && p.a.dout && p.a.dq), HIER_EINVAL, "cross attention: NULL pointer");
  HIER_REQUIRE(a.Sk == 0 || (p.a.dk && p.a.dv), HIER_EINVAL, "cross attention: NULL pointer");
  HIER_REQUIRE(aligned16(p.a.dout) && aligned16(p.a.dq) && aligned16(p.a.dk) && aligned16(p.a.dv), HIER_EINVAL,
               "cross attention: gradients must be 16-byte aligned");
  const int64_t ss[] = {p.a.do_sb, p.a.do_ss, p.a.do_sh, p.a.dq_sb, p.a.dq_ss, p.a.dq_sh,
                        p.a.dk_sb, p.a.dk_ss, p.a.dk_sh, p.a.dv_sb, p.a.dv_ss, p.a.dv_sh};
  for (int64_t s : ss)
    HIER_REQUIRE(s >= 0 && s % 8 == 0, HIER_EINVAL, "cross attention: strides must keep 16-byte rows");
  HIER_REQUIRE((p.a.dq_ss >= a.D || a.Sq <= 1) && (p.a.dq_sh >= a.D || a.Hq == 1) &&
                   (p.a.dk_ss >= a.D || a.Sk <= 1) && (p.a.dk_sh >= a.D || a.Hk == 1) &&
                   (p.a.dv_ss >= a.D || a.Sk <= 1) && (p.a.dv_sh >= a.D || a.Hk == 1) &&
                   (a.B == 1 || (p.a.dq_sb >= a.D && p.a.dk_sb >= a.D && p.a.dv_sb >= a.D)),
               HIER_EINVAL, "cross attention: gradients need rows of their own");
  const int64_t G = a.Hq / a.Hk;
  // a tile's rows within 31 bits of bytes
  HIER_REQUIRE(2 * (65 * a.q_ss + G * a.q_sh) < (1ll << 31) && 2 * (65 * p.a.do_ss + G * p.a.do_sh) < (1ll << 31),
               HIER_EUNSUPPORTED, "cross attention: strides of q or dout too large");
  p.div = make_div((uint32_t)G);
  p.row_tiles = (int)row_tiles(a.Sq * G);
  p.key_tiles = (int)row_tiles(a.Sk);
  p.splits = dkv_splits(a);
  p.dq_splits = dq_splits(a);
  p.total = a.B * a.Hk * p.key_tiles * p.splits;
  // fewer than 2^32 threads a launch, of 256 and of 512
  HIER_REQUIRE(xcd_grid((int64_t)a.B * a.Hk * p.row_tiles * p.dq_splits) < (1 << 24) && xcd_grid(p.total) < (1 << 23),
               HIER_EUNSUPPORTED, "cross attention: too many work items");
  const int64_t need = work_bytes(a);
  HIER_REQUIRE(need == 0 || (a.workspace && aligned16(a.workspace) && a.workspace_bytes >= need), HIER_EINVAL,
               "cross attention: workspace of %lld bytes needed", (long long)need);
  p.lse2 = static_cast<float*>(a.workspace);
  p.delta = p.lse2 + rows_bytes(a) / 4;
  p.part = p.delta + rows_bytes(a) / 4;
  return a.D == 128 ? launch<128>(p, (hipStream_t)stream) : launch<64>(p, (hipStream_t)stream);
}
