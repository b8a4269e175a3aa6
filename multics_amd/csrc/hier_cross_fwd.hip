// Attention of Sq queries to Sk keys of another sequence (an encoder's states),
// streams of unlike key counts and masked keys, shared key heads:
//   O = softmax(scale Q K^T over the seen keys) V,  lse = ln sum exp(scale q k)
//
// The products and their layouts are the hierarchical forward's (hier_attn_fwd.hip):
// four waves of 32 rows, S^T = K Q^T, O^T += V^T P^T with v_mfma_f32_32x32x16, keys
// in 64-key tiles through LDS, two workgroups a CU (three at D 64), and a three-stage pipeline over
// 32-key blocks (S of block j + 2, softmax of j + 1, PV of j).  What differs:
//
// The running maximum is subtracted by the matrix product itself: S starts from -m
// (16 registers that hold it) in place of 0, so a weight is exp2(S c2), one
// multiplication and one exp, exact however large the scores are.  m is that of
// the blocks when it was last refreshed: while no lane's sum of a block's
// 16 weights passes 2^12 the block is taken as it is.  Otherwise, and while a row
// has seen no key, the wave takes the block's maximum, and the block after it, on
// its way already, is shifted too.
//
// Rows are few where a token asks: the keys are then cut into splits, whose
// fp32 sums and maxima a second kernel joins in their order.
//
// Measured, bf16, D 128: 8,192 x 8,192 x 16 heads 540 us (1,017 TFLOP/s; MFMA busy 47 % of
// the time, counted in a launch alone, the vector units 34 %); four streams of
// 4,620 rows x 12 heads against 512 keys 95 (612; MFMA 25 %: eight tiles an item, whose first
// loads and last stores are a third of its time; 3.5 rounds of workgroups).  Workgroups that
// stay and ask for the next item's first tiles under the present one's last: no faster there, and
// ten streams of 660 rows 40 for 36 (registers spilled), not kept.
#include "hier_cross.h"

#include <algorithm>
#include <type_traits>

namespace hier {
namespace {

using namespace cross;

constexpr int kThreads = 256;
constexpr float kSumMax = 4096.f;
constexpr int kValuPerMfma = 3;

struct Launch {
  HierCrossArgs a;
  Div div;
  int32_t row_tiles, splits, total;
  float* part_o;       // [splits][B * Hk][R][D]
  float* part_ml;      // [splits][B * Hk][R][2]
};

struct Stages {
  char* k[2];
  char* v[2];
};

template <typename T, int D>
struct Work {
  u32x4 q[Geo<D>::NC];
  f32x16 o[Geo<D>::NDB];
  f32x16 negm;
  float m, l, c2;
  int krd[Geo<D>::NC], vrd[Geo<D>::NDB];
  Rows64<D, kRowRead> ck;
  Rows64<D, kTrRead> cv;
  uint64_t kbase, vbase;         // of the item's tile 0
  int64_t k_ss, v_ss, len;       // len: keys from the item's tile 0 on
  const uint8_t* mask;           // of the lane's key of tile 0
  int nt, wave, lane;
};

template <typename T>
__device__ __forceinline__ float sum16(const u32x4* p) {
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const uint32_t x = p[c][e], y = p[c][e + 1];   // (a bit cast of an element reads the first)
      if constexpr (__is_same(T, __bf16)) {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        const pair one = {(__bf16)1.f, (__bf16)1.f};
        s0 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, x), one, s0, false);
        s1 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, y), one, s1, false);
      } else {
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        const pair one = {(_Float16)1.f, (_Float16)1.f};
        s0 = __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, x), one, s0, false);
        s1 = __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, y), one, s1, false);
      }
    }
  return s0 + s1;
}

// Weights of a block, rounded to the type of V (as PV's operand; fp32 would halve
// the products' rate), and the lane's sum of the rounded ones, exactly what
// multiplies V.
template <typename T>
__device__ __forceinline__ float weights(const f32x16& s, u32x4* p, float c2) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    vec8<T> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (T)__builtin_amdgcn_exp2f(s[8 * c + i] * c2);
    p[c] = __builtin_bit_cast(u32x4, v);
  }
  return sum16<T>(p);
}

template <typename T, int D>
__device__ __forceinline__ f32x16 scores(const Work<T, D>& w, const char* kslot, int kb) {
  const char* base = kslot + kb * 32 * Geo<D>::ROWB;
  f32x16 s = gemm::mfma<T>(row_operand<T>(base, w.krd[0]), w.q[0], w.negm);
#pragma unroll
  for (int c = 1; c < Geo<D>::NC; ++c) s = gemm::mfma<T>(row_operand<T>(base, w.krd[c]), w.q[c], s);
  return s;
}

__device__ __forceinline__ void mask_scores(f32x16& s, uint32_t bits, int lane) {
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = key_bit(bits, i, lane) ? s[i] : -INFINITY;
}

// The block's sum ps is taken, or the running maximum refreshed and the
// weights made anew; `next` is the block whose scores are made already.
// Returns whether O is to be multiplied by alpha before the block's PV.
template <typename T, int D>
__device__ __forceinline__ bool settle(Work<T, D>& w, f32x16& s, f32x16& next, u32x4* p, float ps, float& alpha) {
  if (__ballot(ps > kSumMax || w.l == 0.f) == 0) {
    w.l += ps;
    return false;
  }
  float mx = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
  mx = tile::pair_max(mx);
  const bool first = tile::pair_sum(w.l) == 0.f;
  const float up = mx == -INFINITY ? 0.f : first ? mx : fmaxf(mx, 0.f);
  const float m = w.m + up, shift = m - w.m;
  w.m = m;
  alpha = first ? 1.f : __builtin_amdgcn_exp2f(-shift * w.c2);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    w.negm[i] = -m;
    s[i] -= shift;
    next[i] -= shift;
  }
  w.l = w.l * alpha + weights<T>(s, p, w.c2);
  return true;
}

template <typename T, int D>
__device__ __forceinline__ void rescale(Work<T, D>& w, float alpha) {
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.o[d][i] *= alpha;
}

template <typename T, int D>
__device__ __forceinline__ void weigh(Work<T, D>& w, const u32x4* p, const char* vslot, int kb) {
  constexpr int HALF = (8 / Geo<D>::NI) * Geo<D>::ROWB;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int d = 0; d < Geo<D>::NDB; ++d) {
      const char* at = vslot + (2 * kb + j) * 16 * Geo<D>::ROWB + w.vrd[d];
      w.o[d] = gemm::mfma<T>(tr_operand(at, at + HALF), p[j], w.o[d]);
    }
}

template <typename T, int D, bool MASK>
__device__ __forceinline__ void copy_k(const Work<T, D>& w, int t, uint64_t seen, char* slot) {
  w.ck.template copy<MASK>(w.kbase + (uint64_t)((int64_t)t * kSlab * 2 * w.k_ss), w.len - (int64_t)t * kSlab, w.k_ss,
                           seen, slot, w.wave);
}
template <typename T, int D, bool MASK>
__device__ __forceinline__ void copy_v(const Work<T, D>& w, int t, uint64_t seen, char* slot) {
  w.cv.template copy<MASK>(w.vbase + (uint64_t)((int64_t)t * kSlab * 2 * w.v_ss), w.len - (int64_t)t * kSlab, w.v_ss,
                           seen, slot, w.wave);
}
template <bool MASK, typename T, int D>
__device__ __forceinline__ uint32_t mask_byte(const Work<T, D>& w, int t) {
  if constexpr (MASK) {
    const int64_t key = (int64_t)t * kSlab + w.lane;
    return key < w.len ? w.mask[(int64_t)t * kSlab] : 0u;
  } else {
    return 0u;
  }
}

// Half-step 2t + B: scores of block B of tile t + 1 (into sq), softmax of the next
// block (sc, into pn), PV of block B of tile t (pv).  PAR = t % 2: K(t + 1) in
// stage PAR ^ 1, V(t) in PAR.
template <typename T, int D, int PAR, int B>
__device__ __forceinline__ void half_step(Work<T, D>& w, f32x16& sq, f32x16& sc, const u32x4* pv, u32x4* pn,
                                          bool& resc, float& alpha, uint32_t bits, const Stages& st) {
  if (resc) rescale<T, D>(w, alpha);
  sq = scores<T, D>(w, st.k[PAR ^ 1], B);
  float ps = weights<T>(sc, pn, w.c2);
  weigh<T, D>(w, pv, st.v[PAR], B);
  constexpr int NM = Geo<D>::NC + 2 * Geo<D>::NDB;
  __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
  for (int i = 0; i < NM; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (i % 2 == 0) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, kValuPerMfma, 0);
  }
  // the softmax stays in this region, under the MFMAs
  asm volatile("" : "+v"(pn[0]), "+v"(pn[1]), "+v"(ps));
  resc = settle<T, D>(w, sc, sq, pn, ps, alpha);
  if (bits != ~0u) mask_scores(sq, bits, w.lane);
}

// Tile t, t + 1 < nt.  On entry K(t + 1) and V(t) are in LDS, sb holds the scores of
// block 1 of tile t, pa the weights of block 0; s1 / s2 say which keys of tiles t + 1 / t + 2 are
// seen.  The mask bytes of tile t + 3 are read here and taken where the copies are waited for.
template <typename T, int D, bool MASK, int PAR>
__device__ __forceinline__ void tile_step(Work<T, D>& w, int t, f32x16& sa, f32x16& sb, u32x4* pa, u32x4* pb,
                                          bool& resc, float& alpha, uint64_t& s1, uint64_t& s2, bool active,
                                          const Stages& st) {
  const uint32_t mb = mask_byte<MASK>(w, t + 3);
  if (t + 2 < w.nt) copy_k<T, D, MASK>(w, t + 2, s2, st.k[PAR]);
  if (active) half_step<T, D, PAR, 0>(w, sa, sb, pa, pb, resc, alpha, (uint32_t)s1, st);
  copy_v<T, D, MASK>(w, t + 1, s1, st.v[PAR ^ 1]);
  if (active) half_step<T, D, PAR, 1>(w, sb, sa, pb, pa, resc, alpha, (uint32_t)(s1 >> 32), st);
  tile::wait_copies();
  s1 = s2;
  s2 = seen_keys<MASK>(w.len, t + 3, mb);
  __syncthreads();
}

template <typename T, int D>
__device__ __forceinline__ void store_row(const Launch& p, const Work<T, D>& w, bool valid, int64_t q, int head,
                                          int b, int64_t prow, int split) {
  const HierCrossArgs& a = p.a;
  const float l = tile::pair_sum(w.l);
  const int half = w.lane >> 5;
  if (!valid) return;
  if (p.splits > 1) {
    const int64_t at = (int64_t)split * a.B * a.Hk * a.Sq * p.div.g + prow;
#pragma unroll
    for (int d = 0; d < Geo<D>::NDB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(p.part_o + at * D + d * 32 + 8 * g + 4 * half) =
            f32x4{w.o[d][4 * g], w.o[d][4 * g + 1], w.o[d][4 * g + 2], w.o[d][4 * g + 3]};
    if (half == 0) {
      p.part_ml[2 * at] = w.m;
      p.part_ml[2 * at + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* op = static_cast<T*>(a.o) + b * a.o_sb + q * a.o_ss + head * a.o_sh;
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      typedef T quad __attribute__((ext_vector_type(4)));
      quad v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)(w.o[d][4 * g + e] * inv);
      *reinterpret_cast<u32x2*>(op + d * 32 + 8 * g + 4 * half) = __builtin_bit_cast(u32x2, v);
    }
  if (a.lse && half == 0)
    a.lse[((int64_t)b * a.Hq + head) * a.Sq + q] = l == 0.f ? -INFINITY : w.m * a.scale + __logf(l);
}

// (D 64: three workgroups a CU.  With a mask the registers have to be asked to fit: four
// streams of 4,620 rows x 12 heads against 512 keys 57 -> 49 us, 46 without a mask.)
template <typename T, int D, bool MASK>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 2) void cross_fwd_kernel(Launch p) {
  __shared__ __align__(16) char k0[Geo<D>::TILEB], k1[Geo<D>::TILEB];
  __shared__ __align__(16) char v0[Geo<D>::TILEB], v1[Geo<D>::TILEB];
  const Stages st = {{k0, k1}, {v0, v1}};
  const int logical = xcd_logical(blockIdx.x, gridDim.x);
  if (logical >= p.total) return;
  const HierCrossArgs& a = p.a;
  // items of one (stream, key head) are neighbours: they share its keys in one L2.
  // Streams take turns, so that one of few keys leaves no XCD without work (ten
  // streams of 660 queries, of 512 keys or fewer: 43 -> 36 us)
  const int per = p.row_tiles * p.splits;
  const int hb = logical / per, in = logical - hb * per;
  const int split = in / p.row_tiles, rt = in - split * p.row_tiles;
  const int hk = hb / a.B, b = hb - hk * a.B, bh = b * a.Hk + hk;
  Work<T, D> w;
  w.lane = threadIdx.x & 63;
  w.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t len = a.Sk;
  if (a.kv_lens) len = min(max((int64_t)a.kv_lens[b], (int64_t)0), a.Sk);
  const int tiles = (int)((len + kSlab - 1) / kSlab);
  const int each = (tiles + p.splits - 1) / p.splits;
  const int t0 = min(split * each, tiles);
  w.nt = min(each, tiles - t0);
  const int64_t key0 = (int64_t)t0 * kSlab;
  w.len = min(len - key0, (int64_t)w.nt * kSlab);
  w.k_ss = a.k_ss;
  w.v_ss = a.v_ss;
  w.kbase = (uint64_t)a.k + 2 * (b * a.k_sb + hk * a.k_sh + key0 * a.k_ss);
  w.vbase = (uint64_t)a.v + 2 * (b * a.v_sb + hk * a.v_sh + key0 * a.v_ss);
  w.mask = MASK ? a.key_mask + b * a.mask_sb + key0 + w.lane : nullptr;
  w.ck.init(w.wave, w.lane, a.k_ss);
  w.cv.init(w.wave, w.lane, a.v_ss);
#pragma unroll
  for (int c = 0; c < Geo<D>::NC; ++c) w.krd[c] = tile::row_read_off<D, kRowRead>(w.lane, c);
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d) w.vrd[d] = tile::tr_read_off<D, kTrRead>(w.lane, d, 0);
  // the lane's row (the last one where there is none)
  const uint32_t R = (uint32_t)(a.Sq * p.div.g);
  const uint32_t r0 = (uint32_t)rt * kRows + w.wave * 32;
  const bool active = r0 < R;
  const bool valid = r0 + (w.lane & 31) < R;
  const uint32_t r = min(r0 + (w.lane & 31), R - 1);
  const uint32_t q = quotient(r, p.div);
  const int head = hk * (int)p.div.g + (int)(r - q * p.div.g);
  const int64_t prow = (int64_t)bh * R + r;
  load_row<D>(w.q, static_cast<const uint16_t*>(a.q) + b * a.q_sb + (int64_t)q * a.q_ss + head * a.q_sh, w.lane);
  w.m = 0.f;
  w.l = 0.f;
  w.c2 = a.scale * kLog2e;
#pragma unroll
  for (int i = 0; i < 16; ++i) w.negm[i] = 0.f;
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.o[d][i] = 0.f;
  if (w.nt <= 0) {
    if (active) store_row<T, D>(p, w, valid, q, head, b, prow, split);
    return;
  }

  const uint64_t s0 = seen_keys<MASK>(w.len, 0, mask_byte<MASK>(w, 0));
  uint64_t s1 = seen_keys<MASK>(w.len, 1, mask_byte<MASK>(w, 1));
  uint64_t s2 = seen_keys<MASK>(w.len, 2, mask_byte<MASK>(w, 2));
  copy_k<T, D, MASK>(w, 0, s0, k0);
  copy_v<T, D, MASK>(w, 0, s0, v0);
  if (w.nt > 1) copy_k<T, D, MASK>(w, 1, s1, k1);
  tile::wait_copies();
  __syncthreads();
  f32x16 sa, sb;
  u32x4 pa[2], pb[2];
  bool resc = false;
  float alpha = 1.f;
  if (active) {
    sa = scores<T, D>(w, k0, 0);
    sb = scores<T, D>(w, k0, 1);
    mask_scores(sa, (uint32_t)s0, w.lane);
    mask_scores(sb, (uint32_t)(s0 >> 32), w.lane);
    resc = settle<T, D>(w, sa, sb, pa, weights<T>(sa, pa, w.c2), alpha);
  }
  __syncthreads();          // K stage 0 has been read
  int t = 0;
  for (; t + 2 < w.nt; t += 2) {
    tile_step<T, D, MASK, 0>(w, t, sa, sb, pa, pb, resc, alpha, s1, s2, active, st);
    tile_step<T, D, MASK, 1>(w, t + 1, sa, sb, pa, pb, resc, alpha, s1, s2, active, st);
  }
  const char* vs = v0;
  if (t + 1 < w.nt) {
    tile_step<T, D, MASK, 0>(w, t, sa, sb, pa, pb, resc, alpha, s1, s2, active, st);
    vs = v1;
  }
  if (!active) return;
  // the last tile: softmax of its block 1, PV of both
  if (resc) rescale<T, D>(w, alpha);
  resc = settle<T, D>(w, sb, sa, pb, weights<T>(sb, pb, w.c2), alpha);
  weigh<T, D>(w, pa, vs, 0);
  if (resc) rescale<T, D>(w, alpha);
  weigh<T, D>(w, pb, vs, 1);
  store_row<T, D>(p, w, valid, q, head, b, prow, split);
}

// ---- few rows --------------------------------------------------------------------
//
// At most 32 rows of a key head (a token of a few query heads): the keys are what is
// read, each once, and nothing is shared by the waves.  Each takes every fourth 64-key
// tile of the item through an LDS tile of its own, with its own waits and no barrier:
// K's next tile leaves as soon as the scores are made, V's after PV.  The four waves'
// O, maximum and sum meet in LDS.  Bound by memory, and by the start and the join where
// the keys are few: four streams of 8 heads and 4,096 keys (67 MB) 17.3 us with the join
// (3.9 TB/s; the 128-row kernel, whose waves wait for one another's tiles, 27.8), one of
// 8 and 8,192 keys 14.6 (29.3), 64 of 12 and 512 keys (201 MB) 42 (44; 4.8 TB/s).

constexpr int kFewRows = 32;

template <int N>
__device__ __forceinline__ void wait_own() {     // at most N of the wave's copies in flight, its LDS reads done
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "i"(N) : "memory");
}

template <typename T, int D, int WAVES, bool MASK>
__global__ __launch_bounds__(64 * WAVES, 1) void cross_few_kernel(Launch p) {
  constexpr int COPIES = 4 * Geo<D>::NI;         // instructions of a tile
  constexpr int Q4 = D / 4;                      // 16-byte pieces of a row of O
  __shared__ __align__(16) char lds[WAVES][2][Geo<D>::TILEB];
  __shared__ float stat[WAVES][2][kFewRows];
  static_assert(kFewRows * D * 4 <= 2 * Geo<D>::TILEB, "a wave's O fits its tiles");
  const int logical = xcd_logical(blockIdx.x, gridDim.x);
  if (logical >= p.total) return;
  const HierCrossArgs& a = p.a;
  const int hb = logical / p.splits, split = logical - hb * p.splits;
  const int hk = hb / a.B, b = hb - hk * a.B, bh = b * a.Hk + hk;       // (as above)
  Work<T, D> w;
  w.lane = threadIdx.x & 63;
  w.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t len = a.Sk;
  if (a.kv_lens) len = min(max((int64_t)a.kv_lens[b], (int64_t)0), a.Sk);
  const int tiles = (int)((len + kSlab - 1) / kSlab);
  const int each = (tiles + p.splits - 1) / p.splits;
  const int first = min(split * each, tiles) + w.wave, end = min((split + 1) * each, tiles);
  const uint64_t kbase = (uint64_t)a.k + 2 * (b * a.k_sb + hk * a.k_sh);
  const uint64_t vbase = (uint64_t)a.v + 2 * (b * a.v_sb + hk * a.v_sh);
  const uint8_t* mask = MASK ? a.key_mask + b * a.mask_sb + w.lane : nullptr;
  w.ck.init(0, w.lane, a.k_ss);
  w.cv.init(0, w.lane, a.v_ss);
#pragma unroll
  for (int c = 0; c < Geo<D>::NC; ++c) w.krd[c] = tile::row_read_off<D, kRowRead>(w.lane, c);
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d) w.vrd[d] = tile::tr_read_off<D, kTrRead>(w.lane, d, 0);
  const uint32_t R = (uint32_t)(a.Sq * p.div.g);
  {
    const uint32_t r = min((uint32_t)w.lane & 31, R - 1), q = quotient(r, p.div);
    const int head = hk * (int)p.div.g + (int)(r - q * p.div.g);
    load_row<D>(w.q, static_cast<const uint16_t*>(a.q) + b * a.q_sb + (int64_t)q * a.q_ss + head * a.q_sh, w.lane);
  }
  w.m = 0.f;
  w.l = 0.f;
  w.c2 = a.scale * kLog2e;
#pragma unroll
  for (int i = 0; i < 16; ++i) w.negm[i] = 0.f;
#pragma unroll
  for (int d = 0; d < Geo<D>::NDB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.o[d][i] = 0.f;
  char* const ks = lds[w.wave][0];
  char* const vs = lds[w.wave][1];
  auto byte_of = [&](int t) -> uint32_t {
    if constexpr (MASK) return (int64_t)t * kSlab + w.lane < len ? mask[(int64_t)t * kSlab] : 0u;
    else return 0u;
  };
  // rows 16 i .. + 16 of a tile are the copies of a workgroup's wave i
  auto copy = [&](const auto& c, uint64_t base, int64_t ss, int t, uint64_t seen, char* slot) {
    const int64_t key0 = (int64_t)t * kSlab;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c.template copy<MASK, 16>(base + (uint64_t)((key0 + 16 * i) * 2 * ss), len - key0 - 16 * i, ss, seen >> (16 * i),
                                slot, i);
  };
  if (first < end) {
    uint64_t seen = seen_keys<MASK>(len, first, byte_of(first));
    copy(w.ck, kbase, a.k_ss, first, seen, ks);
    copy(w.cv, vbase, a.v_ss, first, seen, vs);
    // Q too, here: the compiler, which does not see the copies, would wait for all of them in the loop
#pragma unroll
    for (int c = 0; c < Geo<D>::NC; ++c) asm volatile("" : "+v"(w.q[c]));
    for (int t = first; t < end; t += WAVES) {
      const bool more = t + WAVES < end;
      const uint32_t mb = more ? byte_of(t + WAVES) : 0u;
      wait_own<COPIES>();                        // K is there
      f32x16 sa = scores<T, D>(w, ks, 0), sb = scores<T, D>(w, ks, 1);
      const uint64_t now = seen;
      seen = seen_keys<MASK>(len, t + WAVES, mb);
      wait_own<COPIES>();                        // (its LDS reads)
      if (more) copy(w.ck, kbase, a.k_ss, t + WAVES, seen, ks);
      if (now != ~0ull) {
        mask_scores(sa, (uint32_t)now, w.lane);
        mask_scores(sb, (uint32_t)(now >> 32), w.lane);
      }
      u32x4 pa[2], pb[2];
      float alpha = 1.f;
      bool resc = settle<T, D>(w, sa, sb, pa, weights<T>(sa, pa, w.c2), alpha);
      if (resc) rescale<T, D>(w, alpha);
      resc = settle<T, D>(w, sb, sa, pb, weights<T>(sb, pb, w.c2), alpha);
      if (more) wait_own<COPIES>();              // V is there
      else wait_own<0>();
      weigh<T, D>(w, pa, vs, 0);
      if (resc) rescale<T, D>(w, alpha);
      weigh<T, D>(w, pb, vs, 1);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) copy(w.cv, vbase, a.v_ss, t + WAVES, seen, vs);
    }
  }
  // the waves' results, 16-byte pieces of a row swizzled by the row
  const int row = w.lane & 31, half = w.lane >> 5;
  {
    const float l = tile::pair_sum(w.l);
    if (half == 0) {
      stat[w.wave][0][row] = w.m;
      stat[w.wave][1][row] = l;
    }
    f32x4* const mine = reinterpret_cast<f32x4*>(ks) + row * Q4;
#pragma unroll
    for (int d = 0; d < Geo<D>::NDB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        mine[(8 * d + 2 * g + half) ^ (row & (Q4 - 1))] =
            f32x4{w.o[d][4 * g], w.o[d][4 * g + 1], w.o[d][4 * g + 2], w.o[d][4 * g + 3]};
  }
  __syncthreads();
  for (int i = threadIdx.x; i < (int)R * Q4; i += 64 * WAVES) {
    const uint32_t r = i / Q4, c = i % Q4;
    float top = -INFINITY, l = 0.f, wt[WAVES];
#pragma unroll
    for (int j = 0; j < WAVES; ++j) {
      wt[j] = stat[j][1][r] == 0.f ? -INFINITY : stat[j][0][r];
      top = fmaxf(top, wt[j]);
    }
    f32x4 o = {};
#pragma unroll
    for (int j = 0; j < WAVES; ++j) {
      const float lj = stat[j][1][r];
      wt[j] = lj == 0.f ? 0.f : __builtin_amdgcn_exp2f((wt[j] - top) * w.c2);
      l += lj * wt[j];
      const f32x4 x = reinterpret_cast<const f32x4*>(lds[j][0])[r * Q4 + (c ^ (r & (Q4 - 1)))];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], wt[j], o[e]);
    }
    if (p.splits > 1) {
      const int64_t at = ((int64_t)split * a.B * a.Hk + bh) * R + r;
      *reinterpret_cast<f32x4*>(p.part_o + at * D + 4 * c) = o;
      if (c == 0) {
        p.part_ml[2 * at] = top;
        p.part_ml[2 * at + 1] = l;
      }
      continue;
    }
    const uint32_t q = quotient(r, p.div);
    const int head = hk * (int)p.div.g + (int)(r - q * p.div.g);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    typedef T quad __attribute__((ext_vector_type(4)));
    quad v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (T)(o[e] * inv);
    *reinterpret_cast<u32x2*>(static_cast<T*>(a.o) + b * a.o_sb + (int64_t)q * a.o_ss + head * a.o_sh + 4 * c) =
        __builtin_bit_cast(u32x2, v);
    if (a.lse && c == 0)
      a.lse[((int64_t)b * a.Hq + head) * a.Sq + q] = l == 0.f ? -INFINITY : top * a.scale + __logf(l);
  }
}

// ---- the splits' join ------------------------------------------------------------

constexpr int kMaxSplits = 64;      // a lane of the join each

// A wave a row: lane s holds split s's maximum and sum.
template <typename T, int D>
__global__ __launch_bounds__(256) void cross_join_kernel(Launch p) {
  const HierCrossArgs& a = p.a;
  const int64_t rows = (int64_t)a.B * a.Hk * a.Sq * p.div.g;
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const int lane = threadIdx.x & 63;
  if (row >= rows) return;
  float m = -INFINITY, l = 0.f;
  if (lane < p.splits) {
    const float* ml = p.part_ml + 2 * ((int64_t)lane * rows + row);
    l = ml[1];
    m = l == 0.f ? -INFINITY : ml[0];
  }
  float top = m;
#pragma unroll
  for (int d = 32; d > 0; d /= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
  // (a split that is not a number: its sum is, and the row becomes it)
  const float weight = l == 0.f ? 0.f : __builtin_amdgcn_exp2f((m - top) * (a.scale * kLog2e));
  float total = l * weight;
#pragma unroll
  for (int d = 32; d > 0; d /= 2) total += __shfl_xor(total, d, 64);
  constexpr int E = D / 64;
  float o[E] = {};
  // (eight splits' loads leave together, the last split's again past the end)
  for (int s0 = 0; s0 < p.splits; s0 += 8) {
    float x[8][E];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e)
        x[i][e] = p.part_o[((int64_t)min(s0 + i, p.splits - 1) * rows + row) * D + E * lane + e];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float ws = __shfl(weight, (s0 + i) & 63, 64);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (s0 + i < p.splits) o[e] = fmaf(x[i][e], ws, o[e]);
    }
  }
  const int R = (int)(a.Sq * p.div.g);
  const int bh = (int)(row / R);
  const uint32_t r = (uint32_t)(row - (int64_t)bh * R), q = quotient(r, p.div);
  const int b = bh / a.Hk, head = (bh - b * a.Hk) * (int)p.div.g + (int)(r - q * p.div.g);
  const float inv = total == 0.f ? 0.f : 1.f / total;
  T* op = static_cast<T*>(a.o) + b * a.o_sb + (int64_t)q * a.o_ss + head * a.o_sh + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = (T)(o[e] * inv);
  if (a.lse && lane == 0)
    a.lse[((int64_t)b * a.Hq + head) * a.Sq + q] = total == 0.f ? -INFINITY : top * a.scale + __logf(total);
}

// Parts of every key list (SplitModel).  444 items of 8 tiles 27 us in one part, 58 in
// two; 16 items of 64 tiles 20.7 in 16, 25 in 32.
// Few rows: workgroups for the 256 CUs, of a tile a wave at least.
bool few_rows(const HierCrossArgs& a) { return a.Sq * (a.Hq / a.Hk) <= kFewRows; }

// Waves of a few-row workgroup: two (and two workgroups a CU) where the items need no
// splits, so that streams of unlike lengths and of two tiles leave fewer waves without
// work, else four (less to join).  64 streams of 8 heads and 77 keys 8.4 us with two,
// 11.9 with four; 64 of 12 and 512 keys or fewer 27 / 31; 16 of 12 and 512 15 / 11.7;
// one of 8 and 8,192 17 / 14.6.
int few_waves(const HierCrossArgs& a) { return (int64_t)a.B * a.Hk >= 512 ? 2 : 4; }

int splits_of(const HierCrossArgs& a) {
  const int64_t items = (int64_t)a.B * a.Hk * row_tiles(a.Sq * (a.Hq / a.Hk));
  const int64_t tiles = (a.Sk + kSlab - 1) / kSlab;
  if (few_rows(a) && items > 0) {
    const int waves = few_waves(a);
    return (int)std::max<int64_t>(1, std::min<int64_t>({1024 / waves / items, (tiles + waves - 1) / waves, kMaxSplits}));
  }
  const double size = a.D == 128 ? 1.0 : 0.6;
  return best_splits({512, 2.1 * size, 1.4 * size, 3.5, 2}, items, tiles, 4.0 * a.B * a.Hq * (double)a.Sq * a.D, kMaxSplits);
}

int64_t part_bytes(const HierCrossArgs& a, int splits, int D) {
  return splits == 1 ? 0 : (int64_t)splits * a.B * a.Hq * a.Sq * (D + 2) * 4;
}

template <typename T, int D>
int launch(const Launch& p, hipStream_t st) {
  const dim3 grid((unsigned)xcd_grid(p.total));
  if (few_rows(p.a)) {
    auto few = [&](auto waves, auto mask) {
      constexpr int W = decltype(waves)::value;
      hipLaunchKernelGGL((cross_few_kernel<T, D, W, decltype(mask)::value>), grid, dim3(64 * W), 0, st, p);
    };
    const bool two = few_waves(p.a) == 2;
    typedef std::integral_constant<int, 2> Two;
    typedef std::integral_constant<int, 4> Four;
    if (p.a.key_mask) two ? few(Two{}, std::true_type{}) : few(Four{}, std::true_type{});
    else two ? few(Two{}, std::false_type{}) : few(Four{}, std::false_type{});
  }
  else if (p.a.key_mask)
    hipLaunchKernelGGL((cross_fwd_kernel<T, D, true>), grid, dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL((cross_fwd_kernel<T, D, false>), grid, dim3(kThreads), 0, st, p);
  if (int rc = check_launch("cross_fwd_kernel")) return rc;
  if (p.splits == 1) return HIER_OK;
  const int64_t rows = (int64_t)p.a.B * p.a.Hq * p.a.Sq;
  hipLaunchKernelGGL((cross_join_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p);
  return check_launch("cross_join_kernel");
}

}  // namespace

// Shared by the forward and the gradient.
int cross::check(const HierCrossArgs& a) {
  HIER_REQUIRE(a.D == 128 || a.D == 64, HIER_EUNSUPPORTED, "cross attention: head_dim must be 64 or 128, got %d", a.D);
  HIER_REQUIRE(a.B >= 0 && a.Sq >= 0 && a.Sk >= 0 && a.Hq >= 1 && a.Hk >= 1 && a.Hq % a.Hk == 0, HIER_EINVAL,
               "cross attention: invalid B=%d Sq=%lld Sk=%lld Hq=%d Hk=%d", a.B, (long long)a.Sq, (long long)a.Sk,
               a.Hq, a.Hk);
  HIER_REQUIRE(a.type == HIER_BF16 || a.type == HIER_FP16, HIER_EUNSUPPORTED, "cross attention: bf16 or fp16");
  HIER_REQUIRE(number_in(a.scale, 1e-30f, 1e30f), HIER_EINVAL, "cross attention: the scale must be positive");
  const int64_t G = a.Hq / a.Hk;
  HIER_REQUIRE(a.Sq * G < (1ll << 30) && a.Sk < (1ll << 30), HIER_EUNSUPPORTED, "cross attention: too many rows");
  HIER_REQUIRE((int64_t)a.B * a.Hk * row_tiles(a.Sq * G) <= (1 << 23) && (int64_t)a.B * a.Hk <= (1 << 23) &&
                   (int64_t)a.B * a.Hk * row_tiles(a.Sk) <= (1 << 23),
               HIER_EUNSUPPORTED, "cross attention: too many work items");
  if (a.B == 0 || a.Sq == 0) return HIER_OK;
  HIER_REQUIRE(a.q && a.o && (a.Sk == 0 || (a.k && a.v)), HIER_EINVAL, "cross attention: NULL pointer");
  HIER_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.o), HIER_EINVAL,
               "cross attention: q, k, v and o must be 16-byte aligned");
  const int64_t ss[] = {a.q_sb, a.q_ss, a.q_sh, a.k_sb, a.k_ss, a.k_sh, a.v_sb, a.v_ss, a.v_sh, a.o_sb, a.o_ss, a.o_sh};
  for (int64_t s : ss)
    HIER_REQUIRE(s >= 0 && s % 8 == 0, HIER_EINVAL, "cross attention: strides must keep 16-byte rows");
  HIER_REQUIRE((a.k_ss >= a.D && a.v_ss >= a.D) || a.Sk <= 1, HIER_EINVAL, "cross attention: keys must not overlap");
  HIER_REQUIRE(a.k_ss < (1ll << 23) && a.v_ss < (1ll << 23), HIER_EUNSUPPORTED,
               "cross attention: K/V row stride of 8M elements or more");
  return HIER_OK;
}

}  // namespace hier

using namespace hier;

extern "C" int64_t hier_cross_workspace(const HierCrossArgs* a) {
  clear_error();
  if (!a || a->D < 1 || a->Hk < 1 || a->Hq < a->Hk || a->B < 0 || a->Sq < 0 || a->Sk < 0) {
    fail(HIER_EINVAL, "cross attention: invalid sizes");
    return -1;
  }
  return part_bytes(*a, splits_of(*a), a->D);
}

extern "C" int hier_cross_attn(const HierCrossArgs* args, void* stream) {
  clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  if (int rc = cross::check(*args)) return rc;
  Launch p = {};
  p.a = *args;
  const HierCrossArgs& a = p.a;
  if (a.B == 0 || a.Sq == 0) return HIER_OK;
  HIER_REQUIRE((a.o_ss >= a.D || a.Sq == 1) && (a.o_sh >= a.D || a.Hq == 1) && (a.o_sb >= a.D || a.B == 1),
               HIER_EINVAL, "cross attention: o needs rows of its own");
  p.div = make_div((uint32_t)(a.Hq / a.Hk));
  p.row_tiles = (int)row_tiles(a.Sq * p.div.g);
  p.splits = splits_of(a);
  p.total = a.B * a.Hk * p.row_tiles * p.splits;
  const int64_t need = part_bytes(a, p.splits, a.D);
  HIER_REQUIRE(need == 0 || (a.workspace && aligned16(a.workspace) && a.workspace_bytes >= need), HIER_EINVAL,
               "cross attention: workspace of %lld bytes needed", (long long)need);
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = p.part_o + (int64_t)p.splits * a.B * a.Hq * a.Sq * a.D;
  const hipStream_t st = (hipStream_t)stream;
  if (a.type == HIER_BF16) return a.D == 128 ? launch<__bf16, 128>(p, st) : launch<__bf16, 64>(p, st);
  return a.D == 128 ? launch<_Float16, 128>(p, st) : launch<_Float16, 64>(p, st);
}
