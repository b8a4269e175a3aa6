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
// and so a code itself.  hi's power of two takes the row's largest to 224 .. 448,
// lo's is 2^-4 of it, whose smallest step is 2^-13: the split is exact for every
// element down to 2^-6, which is below 2^-13 of the row's largest; what is smaller
// errs by at most 2^-14, below 2^-21 of the largest (a row whose largest is below
// 448 * 2^-100 is held over 2^-100: by at most 2^-114).  Two 8-bit products cost
// what one in bf16 does, and K needs no conversion.
//
// V is converted when its tile is staged (v_cvt_scalef32_pk_bf16_fp8, exact:
// code and scale fit a bf16) and P V runs on v_mfma_f32_32x32x16_bf16 with P
// rounded to bf16; the row sum adds the rounded weights, so a weight's
// rounding (at most 2^-8 of it) reaches the result only as the spread of such
// roundings over the keys.  m, l and O are fp32.
//
// A workgroup is four waves of 32 rows, two workgroups a CU: with 128 rows a
// tile's K and V are staged (V converted) once for four waves' products, and
// 32 rows a wave leave room for S, P, O and the query's codes without spills
// (three waves a SIMD spill: twice the time).  Full items are bound by the
// matrix units and the softmax beside them at the card's power limit: 6,678
// rows against their windows (24 heads of 128, 507 GFLOP) 530 us, 957 TFLOP/s
// of what rows see, where the bf16 kernel takes 626 over the same lists; the
// same instructions on queries of zeros, which draw less power, take 455.
// Few items are cut into parts (the caller's ``splits``; parts and their join
// below), items of at most 32 rows shared by the four waves (few_rows).
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
// running max.  Maxima are held in exp2 units (score * scale * log2 e); kNoMax,
// the max of a row that has seen no key, is below every score, so that a row's
// first visible key refreshes it whatever its score.
constexpr float kSumMax = 16.f * 256.f;
constexpr float kNoMax = -3.4028235e38f;
// The running max m is a rounded product, off by up to 2^-25 of it, and the
// weights exp2(s * c2 - m) of one rounding (an fma) carry that as a common
// factor, which the row sum takes out again: at most 2^(1/2) where |m| < kFar =
// 2^24, past fp32 from 2^32 on.  So from kFar on every block is refreshed
// (Rows::lim is below any sum) and its products are rounded as m was: the
// largest key's weight is 1 then.
constexpr float kFar = 16777216.f;
constexpr float kLn2 = 0.6931471805599453f;

template <int D>
struct Geo8 {
  static constexpr int NS = D / 64;          // 64-wide d-steps of Q K^T
  static constexpr int CPR = D / 16;         // 16-byte chunks of a row of codes
  static constexpr int RPC = 64 / CPR;       // rows of a wave's copy instruction
  static constexpr int NL = 16 / RPC;        // copies of a wave (its 16 rows) per tile
  static constexpr int KTILEB = kSlab * D;
};

// LDS stages of a workgroup: codes of K, V in bf16, masks and K scales (one
// dword a key), two of each, every one its own array (the copies into one
// stage then never make the compiler wait before it reads another).
struct Stages {
  char* k[2];
  char* v[2];
  char* m[2];
  int* s[2];
};

// Where the 16-byte chunks of a row stand in its tile.
// K tile (D bytes a row): XOR mask on the chunk index, so that 16 consecutive
// rows at one chunk column fall into different banks of a read (256 bytes).
template <int D>
__device__ __forceinline__ constexpr int kswz(int row) {
  return D == 128 ? ((row >> 1) & 7) : ((row >> 2) & 3);
}
// V tile: the swizzle of the transposed reads, and the lowest bit turned in the
// upper half of a row (D = 64: in odd rows), so that the even chunks that eight
// lanes write at once fall into different banks of a write (128 bytes); a read
// takes whole groups of four chunks and does not see it.
template <int D>
__device__ __forceinline__ constexpr int v_chunk(int row, int chunk) {
  return chunk ^ swz<D, kTrRead>(row) ^ (D == 128 ? (chunk >> 3) & 1 : row & 1);
}
// tr_read_off over it.
template <int D>
__device__ __forceinline__ int v_read_off(int lane, int db) {
  const int i = lane & 15, row = 4 * (lane >> 5) + (i >> 2);
  const int q = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
  return prow<D>(row) * Geo<D>::ROWB + 16 * v_chunk<D>(row, 4 * db + q) + 8 * (i & 1);
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
  float lim;                                 // sum of a block's P that refreshes m
  int qtok, qframe, head;
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

// ``pack`` > 1: the sub-block holds that many query heads, from ``head`` on, of
// every row (they share a key head); R.head is the lane's.
template <int D>
__device__ __forceinline__ void rows_init(Rows<D>& R, const HierFwdFp8Args& a, const int32_t* it,
                                          int head, int rrel, int lane, int pack = 1) {
  const int rel = rrel + (lane & 31);
  row_of(R, a, it, pack == 1 ? rel : rel / pack);
  R.head = head + (pack == 1 ? 0 : rel % pack);
  R.bits = __builtin_amdgcn_readfirstlane(wave_or(R.valid ? (1u << R.qframe) : 0u));
  const uint16_t* qp = a.q + (int64_t)R.qtok * a.q_ss + (int64_t)R.head * a.q_sh + 32 * (lane >> 5);
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
  R.lim = kSumMax;
}

// Per-lane LDS byte offsets of the MFMA operand reads (tile-relative).
template <int D>
struct ReadAddr {
  int k[2 * Geo8<D>::NS];   // codes of key lane % 32, d 64 s + 32 (lane / 32) .. + 32: two chunks
  int v[Geo<D>::NDB];       // first transposed V read of d-block db, key chunk 0
  __device__ __forceinline__ void init(int lane) {
    const int key = lane & 31;
#pragma unroll
    for (int i = 0; i < 2 * Geo8<D>::NS; ++i)
      k[i] = key * D + 16 * ((4 * (i >> 1) + 2 * (lane >> 5) + (i & 1)) ^ kswz<D>(key));
#pragma unroll
    for (int db = 0; db < Geo<D>::NDB; ++db) v[db] = v_read_off<D>(lane, db);
  }
};

// S^T of 32-key block kb of a tile.
template <int D>
__device__ __forceinline__ f32x16 qk_block(const Rows<D>& R, const char* kslot, const int* kscale,
                                           const ReadAddr<D>& ra, int kb, int lane) {
  const char* base = kslot + kb * 32 * D;
  const int sk = kscale[kb * 32 + (lane & 31)];
  f32x16 acc = {};
#pragma unroll
  for (int s = 0; s < Geo8<D>::NS; ++s) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(base + ra.k[2 * s]);
    const u32x4 y = *reinterpret_cast<const u32x4*>(base + ra.k[2 * s + 1]);
    const i32x8 k = {(int)x[0], (int)x[1], (int)x[2], (int)x[3],
                     (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, R.hi[s], acc, 0, 0, 0, sk, 0, R.e_hi);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, R.lo[s], acc, 0, 0, 0, sk, 0, R.e_lo);
  }
  return acc;
}

// Set the scores that the lane's query frame may not see to -inf: w, the masks
// of keys 8 g4 + 4 (lane / 32) .. + 4.
__device__ __forceinline__ void mask_four(f32x16& s, int g4, const u32x4& w, int qframe) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t sel = (uint32_t)__builtin_amdgcn_sbfe((int)w[e], qframe, 1);
    const uint32_t x = __float_as_uint(s[4 * g4 + e]);
    s[4 * g4 + e] = __uint_as_float((x & sel) | (0xff800000u & ~sel));
  }
}
// The same of block kb of a tile.
__device__ __forceinline__ void mask_block(f32x16& s, const char* mslot, int kb, int qframe,
                                           int lane) {
  const uint32_t* mk = reinterpret_cast<const uint32_t*>(mslot);
#pragma unroll
  for (int g4 = 0; g4 < 4; ++g4)
    mask_four(s, g4, *reinterpret_cast<const u32x4*>(&mk[kb * 32 + 8 * g4 + 4 * (lane >> 5)]), qframe);
}

// P of one 32-key block: exp2(s * c2 + nb) rounded to bf16, as the two P^T
// operands of the block; returns the lane's sum of the rounded P.  With ``far``
// the product is rounded by itself.
template <bool FAR = false>
__device__ __forceinline__ float p_block(const f32x16& s, bf16x8* p, float c2, float nb,
                                         bool far = false) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float x = fmaf(s[i], c2, nb);
    if constexpr (FAR) {
      float y = s[i] * c2;
      asm("" : "+v"(y));        // (a product of its own: not contracted to an fma)
      x = far ? y + nb : x;
    }
    p[i >> 3][i & 7] = (__bf16)__builtin_amdgcn_exp2f(x);
  }
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

// x = y in x's own register: the rare path writes into the registers of the
// common one, so that no copies are needed where the two meet.  (s_nop 1: the
// wait states that an exp's result and an MFMA's operand need, which the
// compiler does not add around assembly.)
__device__ __forceinline__ void put(float& x, float y) {
  asm volatile("s_nop 1\n\tv_mov_b32 %0, %2\n\ts_nop 1" : "=v"(x) : "0"(x), "v"(y));
}
__device__ __forceinline__ void put(bf16x8& x, const bf16x8& y) {
  u32x4 u = __builtin_bit_cast(u32x4, x);
  const u32x4 w = __builtin_bit_cast(u32x4, y);
  asm volatile("s_nop 1\n\tv_mov_b32 %0, %8\n\tv_mov_b32 %1, %9\n\tv_mov_b32 %2, %10\n\tv_mov_b32 %3, %11\n\ts_nop 1"
               : "=&v"(u[0]), "=&v"(u[1]), "=&v"(u[2]), "=&v"(u[3])
               : "0"(u[0]), "1"(u[1]), "2"(u[2]), "3"(u[3]), "v"(w[0]), "v"(w[1]), "v"(w[2]), "v"(w[3]));
  x = __builtin_bit_cast(bf16x8, u);
}

// Online softmax, second half: ps is the lane's sum of a block's P taken
// against the running max.  True: the max was refreshed and P recomputed; O is
// to be scaled by R.alpha before the block's P V.
template <int D>
__device__ __forceinline__ bool softmax_fix(Rows<D>& R, const f32x16& s, bf16x8* p, float c2,
                                            float ps) {
  float alpha = 1.f;
  const bool refresh = __ballot(!(ps <= R.lim)) != 0;
  if (__builtin_expect(refresh, 0)) {
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = pair_max(mx);
    const float m = fmaxf(R.m, mx * c2);
    const bool far = fabsf(m) >= kFar && m != kNoMax;
    bf16x8 q[2];
    put(ps, p_block<true>(s, q, c2, -m, far));
    put(p[0], q[0]);
    put(p[1], q[1]);
    put(alpha, __builtin_amdgcn_exp2f(R.m - m));
    put(R.m, m);
    put(R.lim, far ? -1.f : kSumMax);
  }
  R.l = fmaf(R.l, alpha, ps);
  R.alpha = alpha;
  return refresh;
}

template <int D>
__device__ __forceinline__ bool softmax_block(Rows<D>& R, const f32x16& s, bf16x8* p, float c2) {
  return softmax_fix<D>(R, s, p, c2, p_block(s, p, c2, -R.m));
}

template <int D>
__device__ __forceinline__ void rescale(Rows<D>& R, float alpha) {
#pragma unroll
  for (int db = 0; db < Geo<D>::NDB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) R.o[db][i] *= alpha;
}

// O^T += V^T P^T over the two 16-key chunks of block kb.
template <int D>
__device__ __forceinline__ void pv_block(Rows<D>& R, const bf16x8* p, const char* vslot,
                                         const ReadAddr<D>& ra, int kb) {
  constexpr int HALF = (8 / Geo<D>::NI) * Geo<D>::ROWB;   // rows of keys +8
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int db = 0; db < Geo<D>::NDB; ++db) {
      const char* p0 = vslot + (2 * kb + j) * 16 * Geo<D>::ROWB + ra.v[db];
      R.o[db] = mfma(tr_read(p0, p0 + HALF), p[j], R.o[db]);
    }
}

// Natural log of a row's sum l over its running max m (exp2 units): -inf for a
// row that sees no key, not a number where l is not one (l = 0 is told by its
// bits: the compiler takes it that there are no NaN).
__device__ __forceinline__ float normaliser(float m, float l) {
  return __float_as_uint(l) == 0u ? -INFINITY : fmaf(m, kLn2, __logf(l));
}

template <int D>
__device__ __forceinline__ void store_rows(const Rows<D>& R, const HierFwdFp8Args& a, int split,
                                           int lane) {
  const float l = pair_sum(R.l);
  if (!R.valid) return;
  const int head = R.head;
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
    a.lse[(int64_t)head * a.lse_stride_h + R.qtok] = normaliser(R.m, l);
}

// ---- staging ------------------------------------------------------------------
//
// A wave stages rows 16 w .. + 16 of a tile: lane l chunk l % CPR of rows
// 16 w + RPC e + l / CPR.  K's codes are copied to LDS as they are; V's go
// through registers (loaded while the tile before is multiplied, converted and
// written at the end of it).

template <int D>
struct Ctx {
  const char* gk;            // the head's codes
  const char* gv;
  const uint8_t* sk;         // the head's scales
  const uint8_t* sv;
  const int32_t* kv_idx;     // of the part's first tile
  const uint32_t* kv_mask;
  const uint32_t* blk;
  uint32_t ss_b, scale_b;    // bytes between rows of codes, between scales
  float c2;
  int nt, wave, lane;
  bool active;
  int row0;                  // the lane's first row of a tile
  uint32_t k16[Geo8<D>::NL], v16;   // byte offsets of its chunk in a row: K's swizzled source, V's
  int vst[2 * Geo8<D>::NL];  // where its chunks of V go
  ReadAddr<D> ra;
};

template <int D>
struct Row {
  int v[Geo8<D>::NL];
};
template <int D>
struct VRegs {
  u32x4 w[Geo8<D>::NL];
  uint32_t s[Geo8<D>::NL];
};

template <int D>
__device__ __forceinline__ Row<D> load_rows(const Ctx<D>& c, int tile) {
  Row<D> r;
  const int32_t* p = c.kv_idx + tile * kSlab;
#pragma unroll
  for (int e = 0; e < Geo8<D>::NL; ++e) r.v[e] = p[(uint32_t)c.row0 + Geo8<D>::RPC * e];
  return r;
}

template <int D>
__device__ __forceinline__ void copy_k(const Ctx<D>& c, const Row<D>& r, char* slot) {
#pragma unroll
  for (int e = 0; e < Geo8<D>::NL; ++e)
    dma16(c.gk, __umul24((uint32_t)r.v[e], c.ss_b) + c.k16[e],
          slot + (16 * c.wave + Geo8<D>::RPC * e) * D);
}

template <int D>
__device__ __forceinline__ void load_scales(const Ctx<D>& c, const uint8_t* sc, const Row<D>& r,
                                            uint32_t* s) {
#pragma unroll
  for (int e = 0; e < Geo8<D>::NL; ++e)
    s[e] = sc[(uint32_t)__umul24((uint32_t)r.v[e] / HIER_FP8_BLOCK, c.scale_b)];
}

template <int D>
__device__ __forceinline__ void store_scales(const Ctx<D>& c, const uint32_t* s, int* slot) {
  if (c.lane % Geo8<D>::CPR == 0)
#pragma unroll
    for (int e = 0; e < Geo8<D>::NL; ++e) slot[c.row0 + Geo8<D>::RPC * e] = (int)s[e];
}

template <int D>
__device__ __forceinline__ void load_v(const Ctx<D>& c, const Row<D>& r, VRegs<D>& v) {
#pragma unroll
  for (int e = 0; e < Geo8<D>::NL; ++e)
    v.w[e] = *reinterpret_cast<const u32x4*>(c.gv + (__umul24((uint32_t)r.v[e], c.ss_b) + c.v16));
  load_scales<D>(c, c.sv, r, v.s);
}

// Codes 8 p .. 8 p + 7 of a chunk as bf16 (exact).
__device__ __forceinline__ u32x4 wide_codes(const u32x4& v, int p, float scale) {
  u32x4 b;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w = v[2 * p + i];
    b[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
    b[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
  }
  return b;
}

template <int D>
__device__ __forceinline__ void store_v(const Ctx<D>& c, const VRegs<D>& v, char* slot) {
#pragma unroll
  for (int e = 0; e < Geo8<D>::NL; ++e) {
    const float sv = pow2_of(v.s[e]);
#pragma unroll
    for (int p = 0; p < 2; ++p)
      *reinterpret_cast<u32x4*>(slot + c.vst[2 * e + p]) = wide_codes(v.w[e], p, sv);
  }
}

// The lane's offsets, the part's key list and the first tiles: K(0), K(1) with
// masks and scales, V(0) resident; the rows of tiles 1 and 2 and the flags of
// tile 1 loaded (nt >= 1).
template <int D>
__device__ __forceinline__ void setup(Ctx<D>& c, const HierFwdFp8Args& a, const int32_t* it, int head,
                                      int split, int tid) {
  using G = Geo8<D>;
  c.lane = tid & 63;
  c.wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = it[6] / kSlab;
  const int t0 = (int)((int64_t)nt * split / a.splits), t1 = (int)((int64_t)nt * (split + 1) / a.splits);
  c.nt = t1 - t0;
  const int64_t off = (int64_t)it[5] + (int64_t)t0 * kSlab;
  const int kh = head / (a.H / a.Hk);
  c.gk = reinterpret_cast<const char*>(a.k + kh * a.kv_sh);
  c.gv = reinterpret_cast<const char*>(a.v + kh * a.kv_sh);
  c.sk = a.k_scale + kh * a.scale_sh;
  c.sv = a.v_scale + kh * a.scale_sh;
  c.kv_idx = a.tile_kv_idx + off;
  c.kv_mask = a.tile_kv_mask + off;
  c.blk = a.tile_blk_and + off / kSlab;
  c.ss_b = (uint32_t)a.kv_ss;
  c.scale_b = (uint32_t)a.scale_ss;
  c.c2 = a.scale * 1.4426950408889634f;
  const int chunk = c.lane % G::CPR;
  c.row0 = 16 * c.wave + c.lane / G::CPR;
  c.v16 = 16u * (uint32_t)chunk;
#pragma unroll
  for (int e = 0; e < G::NL; ++e) {
    const int row = c.row0 + G::RPC * e;
    c.k16[e] = 16u * (uint32_t)(chunk ^ kswz<D>(row));
#pragma unroll
    for (int p = 0; p < 2; ++p)
      c.vst[2 * e + p] = prow<D>(row) * Geo<D>::ROWB + 16 * v_chunk<D>(row, 2 * chunk + p);
  }
  c.ra.init(c.lane);
}

template <int D>
__device__ __forceinline__ void first_tiles(Ctx<D>& c, Row<D>& ik, Row<D>& iv, uint32_t& blk,
                                            const Stages& st) {
  const Row<D> r0 = load_rows<D>(c, 0);
  iv = load_rows<D>(c, min(1, c.nt - 1));
  ik = load_rows<D>(c, min(2, c.nt - 1));
  blk = __builtin_amdgcn_readfirstlane(c.blk[min(1, c.nt - 1)]);
  uint32_t s[Geo8<D>::NL];
  VRegs<D> v;
  copy_k<D>(c, r0, st.k[0]);
  if (c.wave == 0) copy_dwords(c.kv_mask, st.m[0], c.lane);
  load_scales<D>(c, c.sk, r0, s);
  load_v<D>(c, r0, v);
  store_scales<D>(c, s, st.s[0]);
  if (c.nt > 1) {
    copy_k<D>(c, iv, st.k[1]);
    if (c.wave == 0) copy_dwords(c.kv_mask + kSlab, st.m[1], c.lane);
    load_scales<D>(c, c.sk, iv, s);
    store_scales<D>(c, s, st.s[1]);
  }
  store_v<D>(c, v, st.v[0]);
  wait_copies();
  __syncthreads();
}

// ---- the kernel ---------------------------------------------------------------

// Half-step j = 2t + B of the pipeline: QK of block B of tile t+1 into sq,
// softmax of block j+1 (sc) into pn, P V of block B of tile t with pv; then the
// masks of sq (blk_cur: visibility flags of tile t+1).  The three are
// independent, so one scheduling region interleaves them.  PAR = t & 1: K(t+1),
// its masks and scales in stage PAR^1, V(t) in PAR.
template <int D, int PAR, int B>
__device__ __forceinline__ void half_step(Ctx<D>& c, Rows<D>& R, f32x16& sq, const f32x16& sc,
                                          const bf16x8* pv, bf16x8* pn, bool& resc,
                                          float& alpha_pend, uint32_t blk_cur, const Stages& st) {
  if (resc) rescale<D>(R, alpha_pend);
  sq = qk_block<D>(R, st.k[PAR ^ 1], st.s[PAR ^ 1], c.ra, B, c.lane);
  float ps = p_block(sc, pn, c.c2, -R.m);
  pv_block<D>(R, pv, st.v[PAR], c.ra, B);
  // keep S and the softmax results in this region (otherwise they sink past the
  // branches below, away from what they are meant to overlap)
  asm volatile("" : "+v"(sq));
  asm volatile("" : "+v"(pn[0]), "+v"(pn[1]), "+v"(ps));
  resc = softmax_fix<D>(R, sc, pn, c.c2, ps);
  alpha_pend = R.alpha;
  if ((blk_cur & R.bits) != R.bits) mask_block(sq, st.m[PAR ^ 1], B, R.qframe, c.lane);
}

// Tile iteration t (t + 1 < nt): K(t+2) with masks and scales on its way into
// stage PAR and V(t+1) into registers, half-steps 2t and 2t+1, V(t+1)
// converted into stage PAR^1.  On entry K(t+1) and V(t) are resident, S(2t+1)
// (sb) is masked, P(2t) (pa) ready with its rescale pending; ik / iv are the
// rows of tiles min(t+2, nt-1) / t+1, blk the flags of tile t+1.
template <int D, int PAR>
__device__ __forceinline__ void tile_iter(Ctx<D>& c, Rows<D>& R, int t, f32x16& sa, f32x16& sb,
                                          bf16x8* pa, bf16x8* pb, bool& resc, float& alpha_pend,
                                          Row<D>& ik, Row<D>& iv, uint32_t& blk, const Stages& st) {
  const bool more = t + 2 < c.nt;
  uint32_t s[Geo8<D>::NL];
  VRegs<D> v;
  load_v<D>(c, iv, v);
  if (more) {
    copy_k<D>(c, ik, st.k[PAR]);
    if (c.wave == 0) copy_dwords(c.kv_mask + (t + 2) * kSlab, st.m[PAR], c.lane);
  }
  load_scales<D>(c, c.sk, ik, s);
  iv = ik;
  ik = load_rows<D>(c, min(t + 3, c.nt - 1));
  const uint32_t blk_pre = c.blk[min(t + 2, c.nt - 1)];
  if (c.active) {
    half_step<D, PAR, 0>(c, R, sa, sb, pa, pb, resc, alpha_pend, blk, st);
    half_step<D, PAR, 1>(c, R, sb, sa, pb, pa, resc, alpha_pend, blk, st);
  }
  store_v<D>(c, v, st.v[PAR ^ 1]);
  if (more) store_scales<D>(c, s, st.s[PAR]);
  wait_copies();
  __syncthreads();
  blk = __builtin_amdgcn_readfirstlane(blk_pre);   // (not before: it waits for the load)
}

// Last tile (t = nt - 1): softmax of its block 1 (sb) into pb, P V of both.
template <int D, int PAR>
__device__ __forceinline__ void last_tile(Ctx<D>& c, Rows<D>& R, const f32x16& sb, const bf16x8* pa,
                                          bf16x8* pb, bool resc, float alpha_pend,
                                          const Stages& st) {
  if (resc) rescale<D>(R, alpha_pend);
  resc = softmax_block<D>(R, sb, pb, c.c2);
  alpha_pend = R.alpha;
  pv_block<D>(R, pa, st.v[PAR], c.ra, 0);
  if (resc) rescale<D>(R, alpha_pend);
  pv_block<D>(R, pb, st.v[PAR], c.ra, 1);
}

// ---- items of at most 32 rows --------------------------------------------------
//
// A hub's rows, a player's last rows or a single token fill one 32-row
// sub-block.  All four waves take it, each on every fourth tile of the list
// with a softmax state of its own, and nothing to wait for in the others: K
// goes from memory straight into the MFMA operand (a lane holds 32 codes of
// one key twice), V through 32 rows of LDS that are the wave's own.  The next
// block's loads are in flight while one is multiplied (two blocks ahead: the
// same time).  The four states are joined through LDS.  Query heads that share
// a key head are packed into the sub-block when they fit, so that its K and V
// are read once.  One token of 32 heads of 128 over 8 key heads, 4,096 cached
// frames: 20.8 us (99 as an item whose waves share each tile), of it the join of
// its eight parts 4.  A wave takes 12 blocks here, 0.6 us each by the latency of
// its loads (25.9 us this kernel with four parts, 24 blocks a wave; 18.5 with
// eight); about 11 do not depend on them (17.8 with sixteen parts): the loads of
// item, query and first rows, the join in LDS, and the workgroups of packed
// heads, which read their item and leave.

template <int D>
struct Block {               // what a wave loads of a 32-key block
  static constexpr int NV = 32 / Geo8<D>::RPC;   // 16-byte loads of V
  u32x4 k[2 * Geo8<D>::NS];
  u32x4 v[NV];
  uint32_t sk, sv[NV];
  u32x4 m[4];                // masks of the lane's 16 keys, where the block needs them
};
template <int D>
struct BlockRow {
  int k, v[Block<D>::NV];    // pool rows: of the lane's key, of its chunks of V
  uint32_t flags;            // of the block's tile
};

template <int D>
__device__ __forceinline__ BlockRow<D> block_rows(const Ctx<D>& c, int b) {
  BlockRow<D> r;
  const int32_t* p = c.kv_idx + b * 32;
  r.k = p[c.lane & 31];
#pragma unroll
  for (int e = 0; e < Block<D>::NV; ++e) r.v[e] = p[Geo8<D>::RPC * e + c.lane / Geo8<D>::CPR];
  r.flags = c.blk[b >> 1];
  return r;
}

template <int D>
__device__ __forceinline__ bool block_masked(const BlockRow<D>& r, uint32_t bits) {
  return ((uint32_t)__builtin_amdgcn_readfirstlane(r.flags) & bits) != bits;
}

// Loads of block b (rows r), with its masks if it is ``masked``.
template <int D>
__device__ __forceinline__ void block_load(const Ctx<D>& c, int b, const BlockRow<D>& r, bool masked,
                                           Block<D>& x) {
  const char* k = c.gk + (__umul24((uint32_t)r.k, c.ss_b) + 32u * (uint32_t)(c.lane >> 5));
#pragma unroll
  for (int i = 0; i < 2 * Geo8<D>::NS; ++i)
    x.k[i] = *reinterpret_cast<const u32x4*>(k + 64 * (i >> 1) + 16 * (i & 1));
#pragma unroll
  for (int e = 0; e < Block<D>::NV; ++e)
    x.v[e] = *reinterpret_cast<const u32x4*>(c.gv + (__umul24((uint32_t)r.v[e], c.ss_b) + c.v16));
  x.sk = c.sk[(uint32_t)__umul24((uint32_t)r.k / HIER_FP8_BLOCK, c.scale_b)];
#pragma unroll
  for (int e = 0; e < Block<D>::NV; ++e)
    x.sv[e] = c.sv[(uint32_t)__umul24((uint32_t)r.v[e] / HIER_FP8_BLOCK, c.scale_b)];
  if (masked) {
    const uint32_t* m = c.kv_mask + b * 32;
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4)
      x.m[g4] = *reinterpret_cast<const u32x4*>(m + (8 * g4 + 4 * (uint32_t)(c.lane >> 5)));
  }
}

template <int D>
__device__ __forceinline__ void few_rows(const HierFwdFp8Args& a, const int32_t* it, Ctx<D>& c,
                                         int head, int pack, int split, const Stages& st) {
  using B = Block<D>;
  Rows<D> R;
  rows_init<D>(R, a, it, head, 0, c.lane, pack);
  char* const vslot = (c.wave < 2 ? st.v[0] : st.v[1]) + (c.wave & 1) * 32 * Geo<D>::ROWB;
  int vst[2 * B::NV];
#pragma unroll
  for (int e = 0; e < B::NV; ++e)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int row = Geo8<D>::RPC * e + c.lane / Geo8<D>::CPR;
      vst[2 * e + p] = prow<D>(row) * Geo<D>::ROWB +
                       16 * v_chunk<D>(row, 2 * (c.lane % Geo8<D>::CPR) + p);
    }
  // block b of the wave: 32-key block b & 1 of tile wave + 4 (b >> 1)
  const int mine = c.nt > c.wave ? 2 * ((c.nt - c.wave + kWaves - 1) / kWaves) : 0;
  const auto at = [&](int b) { return 2 * (c.wave + kWaves * (b >> 1)) + (b & 1); };
  if (mine > 0) {
    B x;
    const BlockRow<D> first = block_rows<D>(c, at(0));
    bool masked = block_masked<D>(first, R.bits);
    block_load<D>(c, at(0), first, masked, x);
    BlockRow<D> next = block_rows<D>(c, at(min(1, mine - 1)));
    for (int b = 0; b < mine; ++b) {
      // S^T
      f32x16 s = {};
#pragma unroll
      for (int j = 0; j < Geo8<D>::NS; ++j) {
        const u32x4 u = x.k[2 * j], w = x.k[2 * j + 1];
        const i32x8 k = {(int)u[0], (int)u[1], (int)u[2], (int)u[3],
                         (int)w[0], (int)w[1], (int)w[2], (int)w[3]};
        s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, R.hi[j], s, 0, 0, 0, (int)x.sk, 0, R.e_hi);
        s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, R.lo[j], s, 0, 0, 0, (int)x.sk, 0, R.e_lo);
      }
      // V to LDS in bf16
#pragma unroll
      for (int e = 0; e < B::NV; ++e) {
        const float sv = pow2_of(x.sv[e]);
#pragma unroll
        for (int p = 0; p < 2; ++p)
          *reinterpret_cast<u32x4*>(vslot + vst[2 * e + p]) = wide_codes(x.v[e], p, sv);
      }
      if (masked)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) mask_four(s, g4, x.m[g4], R.qframe);
      // the next block's loads, and the rows of the one after it (past the last: the last)
      masked = block_masked<D>(next, R.bits);
      block_load<D>(c, at(min(b + 1, mine - 1)), next, masked, x);
      next = block_rows<D>(c, at(min(b + 2, mine - 1)));
      bf16x8 p[2];
      if (softmax_block<D>(R, s, p, c.c2)) rescale<D>(R, R.alpha);
      pv_block<D>(R, p, vslot, c.ra, 0);
    }
  }
  // join: waves 2, 3 into 0, 1, then 1 into 0 (O^T as fp32 [element][lane] in
  // the V stages, m and l in the mask stages)
  float* const ml = reinterpret_cast<float*>(st.m[0]);     // [64 lanes]: m, and
  float* const ll = reinterpret_cast<float*>(st.m[1]);     // l, of one wave
#pragma unroll
  for (int half = 2; half >= 1; half >>= 1) {
    __syncthreads();
    if (c.wave >= half && c.wave < 2 * half) {
      float* o = reinterpret_cast<float*>(c.wave == half ? st.v[0] : st.v[1]);
#pragma unroll
      for (int db = 0; db < Geo<D>::NDB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[(db * 16 + e) * 64 + c.lane] = R.o[db][e];
      // both halves of a row's lanes hold the same m; each its part of l
      st.s[0][(c.wave - half) * 32 + (c.lane & 31)] = __float_as_int(R.m);
      (c.wave == half ? ml : ll)[c.lane] = R.l;
    }
    __syncthreads();
    if (c.wave < half) {
      const float* o = reinterpret_cast<const float*>(c.wave == 0 ? st.v[0] : st.v[1]);
      const float m2 = __int_as_float(st.s[0][c.wave * 32 + (c.lane & 31)]);
      const float m = fmaxf(R.m, m2);
      const float w1 = __builtin_amdgcn_exp2f(R.m - m), w2 = __builtin_amdgcn_exp2f(m2 - m);
      R.l = R.l * w1 + (c.wave == 0 ? ml : ll)[c.lane] * w2;
      R.m = m;
#pragma unroll
      for (int db = 0; db < Geo<D>::NDB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          R.o[db][e] = R.o[db][e] * w1 + o[(db * 16 + e) * 64 + c.lane] * w2;
    }
  }
  if (c.wave == 0) store_rows<D>(R, a, split, c.lane);
}

template <int D>
__global__ __launch_bounds__(kThreads, 2) void attn_fp8_kernel(HierFwdFp8Args a, int total) {
  __shared__ __align__(16) char lds_k0[Geo8<D>::KTILEB], lds_k1[Geo8<D>::KTILEB];
  __shared__ __align__(16) char lds_v0[Geo<D>::TILEB], lds_v1[Geo<D>::TILEB];
  __shared__ __align__(16) char lds_m0[Geo<D>::MBYTES], lds_m1[Geo<D>::MBYTES];
  __shared__ int lds_s0[kSlab], lds_s1[kSlab];
  const Stages st = {{lds_k0, lds_k1}, {lds_v0, lds_v1}, {lds_m0, lds_m1}, {lds_s0, lds_s1}};
  const int logical = hier::xcd_logical(blockIdx.x, gridDim.x);
  if (logical >= total) return;
  const int per_head = a.n_items * a.splits;
  const int head = logical / per_head, rest = logical - head * per_head;
  const int item = rest / a.splits, split = rest - item * a.splits;
  const int32_t* it = a.tile_items + (int64_t)item * 8;
  Ctx<D> c;
  setup<D>(c, a, it, head, split, threadIdx.x);
  if (it[4] <= 32) {
    const int group = a.H / a.Hk, pack = group * it[4] <= 32 ? group : 1;
    if (head % pack == 0) few_rows<D>(a, it, c, head, pack, split, st);
    return;
  }
  c.active = c.wave * 32 < it[4];
  Rows<D> R;
  rows_init<D>(R, a, it, head, c.wave * 32, c.lane);
  const int nt = c.nt;
  if (nt == 0) {
    if (c.active) store_rows<D>(R, a, split, c.lane);
    return;
  }
  Row<D> ik, iv;
  uint32_t blk;
  first_tiles<D>(c, ik, iv, blk, st);
  // S of both blocks of tile 0 computed and masked; P of block 0
  f32x16 sa, sb;
  bf16x8 pa[2], pb[2];
  bool resc = false;
  float alpha_pend = 1.f;
  if (c.active) {
    sa = qk_block<D>(R, st.k[0], st.s[0], c.ra, 0, c.lane);
    sb = qk_block<D>(R, st.k[0], st.s[0], c.ra, 1, c.lane);
    if ((c.blk[0] & R.bits) != R.bits) {
      mask_block(sa, st.m[0], 0, R.qframe, c.lane);
      mask_block(sb, st.m[0], 1, R.qframe, c.lane);
    }
    resc = softmax_block<D>(R, sa, pa, c.c2);
    alpha_pend = R.alpha;
  }
  __syncthreads();   // every wave has read stage 0 of K, masks and scales
  // two tile iterations per trip, so that every stage is a compile-time constant
  int t = 0;
  for (; t + 2 < nt; t += 2) {
    tile_iter<D, 0>(c, R, t, sa, sb, pa, pb, resc, alpha_pend, ik, iv, blk, st);
    tile_iter<D, 1>(c, R, t + 1, sa, sb, pa, pb, resc, alpha_pend, ik, iv, blk, st);
  }
  if (t + 1 < nt) {
    tile_iter<D, 0>(c, R, t, sa, sb, pa, pb, resc, alpha_pend, ik, iv, blk, st);
    if (c.active) last_tile<D, 1>(c, R, sb, pa, pb, resc, alpha_pend, st);
  } else if (c.active) {
    last_tile<D, 0>(c, R, sb, pa, pb, resc, alpha_pend, st);
  }
  if (c.active) store_rows<D>(R, a, split, c.lane);
}

// Joins the parts of one item and head, kJoinRows rows a workgroup, D / 4 lanes
// a row: the parts' maxima and sums are read at once, one or two a lane (at
// most 32 parts), and their O's eight at a time, so that a row costs a few
// memory latencies and not one a part.  324 items of three parts: 13 of the
// call's 133 us.
constexpr int kMaxSplits = 32;
template <int D>
__global__ __launch_bounds__(kThreads) void join_fp8_kernel(HierFwdFp8Args a) {
  constexpr int LPR = D / 4, ROWS = kThreads / LPR, PER = kMaxSplits / LPR;
  struct { int qtok, qframe; bool valid; } r;
  const int head = blockIdx.x / a.n_items, item = blockIdx.x - head * a.n_items;
  const int32_t* it = a.tile_items + (int64_t)item * 8;
  const int rel = blockIdx.y * ROWS + threadIdx.x / LPR, sub = threadIdx.x % LPR;
  if (blockIdx.y * ROWS >= it[4]) return;
  row_of(r, a, it, rel);
  const int64_t at = (int64_t)head * a.q_rows + r.qtok, step = (int64_t)a.H * a.q_rows;
  float ms[PER], ls[PER], m = kNoMax;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = sub + i * LPR;
    ms[i] = kNoMax, ls[i] = 0.f;
    if (r.valid && s < a.splits) {
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (at + s * step));
      ms[i] = ml.x, ls[i] = ml.y;
    }
    m = fmaxf(m, ms[i]);
  }
#pragma unroll
  for (int d = 1; d < LPR; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, LPR));
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    ms[i] = __builtin_amdgcn_exp2f(ms[i] - m);       // a part's weight
    l = fmaf(ls[i], ms[i], l);
  }
#pragma unroll
  for (int d = 1; d < LPR; d <<= 1) l += __shfl_xor(l, d, LPR);
  f32x4 o = {};
  const float* p = a.part_o + at * D + 4 * sub;
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    f32x4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = f32x4{};
      if (r.valid && s0 + i < a.splits) x[i] = *reinterpret_cast<const f32x4*>(p + (s0 + i) * step * D);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // (a row's lanes hold parts sub and sub + LPR)
      const float w = __shfl(PER == 2 && s0 + i >= LPR ? ms[PER - 1] : ms[0], (s0 + i) % LPR, LPR);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = s0 + i < a.splits ? fmaf(x[i][j], w, o[j]) : o[j];
    }
  }
  if (!r.valid) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  u32x2 w;
  w[0] = (uint32_t)f2bf(o[0] * inv) | ((uint32_t)f2bf(o[1] * inv) << 16);
  w[1] = (uint32_t)f2bf(o[2] * inv) | ((uint32_t)f2bf(o[3] * inv) << 16);
  *reinterpret_cast<u32x2*>(a.o + (int64_t)r.qtok * a.o_ss + (int64_t)head * a.o_sh + 4 * sub) = w;
  if (a.lse && sub == 0)
    a.lse[(int64_t)head * a.lse_stride_h + r.qtok] = normaliser(m, l);
}

template <int D>
int launch(const HierFwdFp8Args& a, int64_t total, hipStream_t stream) {
  hipLaunchKernelGGL(attn_fp8_kernel<D>, dim3((unsigned)hier::xcd_grid(total)), dim3(kThreads), 0,
                     stream, a, (int)total);
  const int rc = hier::check_launch("attn_fp8_kernel");
  if (rc != HIER_OK || a.splits == 1) return rc;
  hipLaunchKernelGGL(join_fp8_kernel<D>, dim3((unsigned)(a.n_items * a.H), 128 * (D / 4) / kThreads),
                     dim3(kThreads), 0, stream, a);
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
  HIER_REQUIRE(a.n_items >= 0 && a.kv_rows >= 0 && a.q_rows >= 0 && a.splits >= 1 &&
                   a.splits <= kMaxSplits,
               HIER_EINVAL,
               "invalid n_items=%d kv_rows=%lld q_rows=%lld splits=%d", a.n_items,
               (long long)a.kv_rows, (long long)a.q_rows, a.splits);
  if (a.n_items == 0) return HIER_OK;
  HIER_REQUIRE(a.scale > 0.f && hier::number_in(a.scale, 0.f, 1e30f), HIER_EINVAL,
               "the softmax scale must be positive, got %g", (double)a.scale);
  HIER_REQUIRE(a.q && a.k && a.v && a.k_scale && a.v_scale && a.o && a.tile_items && a.tile_kv_idx &&
                   a.tile_kv_mask && a.tile_blk_and,
               HIER_EINVAL, "NULL tensor pointer");
  HIER_REQUIRE(a.splits == 1 || (a.part_o && a.part_ml), HIER_EINVAL, "splits need part_o and part_ml");
  auto al16 = [](const void* p) { return ((uintptr_t)p & 15u) == 0; };
  // (masks are read four keys at a time, row-table entries whole)
  HIER_REQUIRE(al16(a.q) && al16(a.k) && al16(a.v) && al16(a.o) && al16(a.tile_kv_mask) &&
                   al16(a.part_o) && al16(a.part_ml) && ((uintptr_t)a.row_table & 7u) == 0,
               HIER_EINVAL,
               "q/k/v/o, the key mask list and the workspace must be 16-byte aligned, the row table 8");
  HIER_REQUIRE(a.q_ss % 8 == 0 && a.q_sh % 8 == 0 && a.kv_ss % 16 == 0 && a.kv_sh % 16 == 0 &&
                   a.o_ss % 4 == 0 && a.o_sh % 4 == 0,
               HIER_EINVAL, "strides must keep 16-byte rows aligned");
  // rows of codes are addressed with 32-bit byte offsets from their head's
  // first (one 24 x 24-bit multiply)
  HIER_REQUIRE(a.kv_ss >= 0 && a.scale_ss >= 0 && a.kv_rows <= (1ll << 24) && a.kv_ss < (1ll << 24) &&
                   a.scale_ss < (1ll << 24) && a.kv_rows * a.kv_ss <= (1ll << 32) &&
                   a.kv_rows / HIER_FP8_BLOCK * a.scale_ss <= (1ll << 32),
               HIER_EUNSUPPORTED,
               "a head's codes and scales must span at most 4 GiB, of 2^24 rows and strides below 2^24");
  const int64_t total = (int64_t)a.n_items * a.splits * a.H;
  // (fewer than 2^32 threads a launch)
  HIER_REQUIRE((int64_t)a.n_items * a.splits < (1ll << 31) && hier::xcd_grid(total) < (1ll << 24),
               HIER_EUNSUPPORTED, "too many work items");
  return a.D == 128 ? launch<128>(a, total, (hipStream_t)stream)
                    : launch<64>(a, total, (hipStream_t)stream);
}
