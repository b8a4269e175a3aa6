// Matrix product out of LDS tiles for gfx950: C[m][n] = sum_k A(m, k) B(n, k),
// fp32 accumulation, 16-bit operands, each in either of two layouts:
//   rows        A[m][k], k contiguous (activations, and weights [out][in])
//   transposed  A[k][m], m contiguous (weights in dx = dz W, both operands of
//               dW = dz^T x)
//
// Workgroup = 4 waves, one per SIMD, in a 2 x 2 grid over a BM x BN tile; a wave
// owns BM/2 x BN/2 of it in accumulators (256 of its 512 registers at 256 x
// 256).  A product step is 16 deep (v_mfma_f32_32x32x16): BM/64 + BN/64 operand
// reads from LDS feed (BM/64)(BN/64) MFMAs, so the larger the wave's part the
// fewer bytes LDS has to deliver for an MFMA.
//
// K tiles of BK go HBM/L2 -> LDS with buffer_load_dwordx4 ... lds, S stages.
// A buffer load out of its range writes zeros: rows past the end, the ragged
// last K tile and tiles past the end need no other handling, and nothing past a
// view's last element is read.  The operands of step k+1 are read while the
// MFMAs of step k run.  One barrier a tile, before its last step: by then every
// wave has read the tile to its end, and the next tile has landed, so the last
// step starts on the next tile and its stage is filled anew.
//
// LDS layouts (16-byte chunks, XOR-swizzled so that no 16 lanes of a read meet
// in a bank; a global read of a wave is whole lines all the same):
//   rows        row r of BK/8 chunks, chunk c at position c ^ (r / (128/BK) % (BK/8))
//   transposed  k-row r of R/8 chunks, chunk c at position c ^ 4 (r % 4)
#pragma once

#include "hier_launch.h"
#include "hier_types.h"

namespace hier {
namespace gemm {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename T>
__device__ __forceinline__ f32x16 mfma(const u32x4& a, const u32x4& b, const f32x16& c) {
  const vec8<T> x = __builtin_bit_cast(vec8<T>, a), y = __builtin_bit_cast(vec8<T>, b);
  if constexpr (sizeof(T) == 2 && __is_same(T, __bf16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
}

constexpr uint32_t kOut = 0x80000000u;   // an offset past any view's range

// 64 lanes x 16 bytes into LDS at l (wave-uniform).  The copies are in assembly
// so that the compiler does not wait for them at every LDS read; they are
// waited for by wait_vm and a barrier.
__device__ __forceinline__ void dma(const u32x4& srd, uint32_t voff, uint32_t l) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :: "v"(voff), "s"(srd), "{m0}"(l) : "memory");
}

// This wave's LDS reads done and at most N of its copies in flight, then the
// workgroup's barrier.
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "i"(N) : "memory");
}

// One operand of a workgroup: R rows (of m or n) of a K tile.
template <bool TR, int R, int BK>
struct Operand {
  static constexpr int BYTES = R * BK * 2;
  static constexpr int COPIES = BYTES / 4096;                     // a wave's, per tile
  static constexpr int CPR = TR ? R / 8 : BK / 8;                 // chunks per LDS row
  static constexpr int LPC = 64 / CPR;                            // LDS rows per copy
  static constexpr int KK = BK / 16;
  static constexpr int MI = R / 64;                               // 32-row blocks of a wave
  uint64_t base;       // first byte of the present tile to copy
  int64_t left;        // bytes of the view from there
  int64_t step;        // bytes to the next tile
  uint32_t voff, sstep;
  int k8;              // rows: the lane's first k of a tile
  int rd[TR ? MI : KK];

  // rows: view of `rows` x K, ld elements apart, from row `first`, k0 on.
  // transposed: view of K x `rows`.
  __device__ __forceinline__ void init(const void* p, int64_t ld, int64_t rows, int64_t first, int64_t k0,
                                       int64_t kend, int wave, int part, int lane) {
    const int line = lane / CPR, pos = lane % CPR;
    if constexpr (TR) {
      rows = (rows + 7) / 8 * 8;         // (a view's rows of k are whole chunks)
      const int chunk = pos ^ (4 * ((LPC * wave + line) & 3));
      base = (uint64_t)p + 2 * (k0 * ld + first);
      left = 2 * ((kend - k0 - 1) * ld + rows - first);
      step = 2 * BK * ld;
      voff = (uint32_t)((LPC * wave + line) * (int)(2 * ld) + 16 * chunk);
      if (first + 8 * chunk >= rows) voff = kOut;
      k8 = 0;
#pragma unroll
      for (int b = 0; b < MI; ++b) {
        const int i = lane & 15, r = 8 * (lane >> 5) + (i >> 2);
        const int q = 4 * (part * MI + b) + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
        rd[b] = r * (2 * R) + 16 * (q ^ (4 * (r & 3))) + 8 * (i & 1);
      }
    } else {
      kend = (kend + 7) / 8 * 8;
      const int row = LPC * wave + line;
      const int chunk = pos ^ (row / (128 / BK) % CPR);
      base = (uint64_t)p + 2 * (first * ld + k0);
      left = 2 * ((rows - first - 1) * ld + kend - k0);
      step = 2 * BK;
      voff = (uint32_t)(row * (int)(2 * ld) + 16 * chunk);
      k8 = 8 * chunk;
      const int r = lane & 31;
#pragma unroll
      for (int k = 0; k < KK; ++k)
        rd[k] = (part * 32 * MI + r) * (2 * BK) + 16 * ((2 * k + (lane >> 5)) ^ (r / (128 / BK) % CPR));
    }
    sstep = (uint32_t)(4 * LPC * (2 * ld));
  }

  // Copy j of the wave's for the tile that `base` is at; kleft = its K.
  __device__ __forceinline__ void copy(int j, int kleft, uint32_t lds, int wave) const {
    const uint32_t n = left <= 0 ? 0u : (left < 0x7fffffff ? (uint32_t)left : 0x7fffffffu);
    const u32x4 srd = {(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu, n, 0x00020000u};
    const uint32_t v = TR ? voff : (k8 < kleft ? voff : kOut);
    // (the whole offset in the lane's register: it is what the range check sees;
    // kOut plus the copies' rows, under 2^30, stays past every range)
    dma(srd, v + j * sstep, lds + 1024 * (wave + 4 * j));
  }
  __device__ __forceinline__ void next() {
    base += step;
    left -= step;
  }
  // No more tiles: the copies write zeros.
  __device__ __forceinline__ void end() {
    left = 0;
    step = 0;
  }

  // Operand of block b and step k from the tile at `t`: lane l holds row
  // 32 b + l % 32, k = 16 k + 8 (l / 32) .. + 8.
  __device__ __forceinline__ u32x4 read(const char* t, int b, int k) const {
    if constexpr (TR) {
      const char* p = t + rd[b] + k * 16 * 2 * R;
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * 2 * R));
      return __builtin_bit_cast(u32x4, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      return *reinterpret_cast<const u32x4*>(t + rd[k] + b * 32 * 2 * BK);
    }
  }
};

// acc[ni][mi]: 32 x 32 blocks, lane l holds row m = 32 mi + l % 32 and
// n = 32 ni + 8 (r / 4) + 4 (l / 32) + r % 4 of the wave's part.
//
// The K tiles of a workgroup's work items are one stream: while an item is
// multiplied, and while its results go out, the copies run ahead into the next
// (`Next` sets the operands to it), so only the first one waits for memory.
template <typename T, bool ATR, bool BTR, int BM, int BN, int BK, int S>
struct Product {
  typedef Operand<ATR, BM, BK> A;
  typedef Operand<BTR, BN, BK> B;
  static constexpr int MI = A::MI, NI = B::MI, KK = BK / 16;
  static constexpr int STAGE = A::BYTES + B::BYTES;
  static constexpr int LDS = S * STAGE;
  static constexpr int COPIES = A::COPIES + B::COPIES;
  static constexpr int READS = MI + NI, NM = NI * MI;
  // A tile's copies are made in the first SPREAD steps after its stage is free
  // (the last step of one tile, the first of the next ..): the workgroup's copies
  // leave at about the rate that the CU's address unit takes them (one 1 KiB copy in
  // 16 cycles), and land before the tile after next needs them.  8192^3: in one
  // step 1,184 TFLOP/s, in two 1,234, in three 1,189, in all four 1,118.
  static constexpr int SPREAD = 2;
  static constexpr int FIRST = (COPIES + SPREAD - 1) / SPREAD;
  static_assert(KK % 2 == 0 && S >= 2, "");

  A a;
  B b;
  int64_t kall;           // K left of the item that is being copied
  int kleft;              // the same, at most 2^30
  uint32_t l0, fill;      // LDS address, stage that the next tile goes to
  const char* lds;
  const char* cur;        // stage of the present tile
  int wave;
  u32x4 fa[2][MI], fb[2][NI];

  __device__ __forceinline__ void item(int64_t K) {
    kall = K;
    kleft = (int)(K < (1 << 30) ? K : (1 << 30));
  }
  __device__ __forceinline__ void copy_one(int j) {
    if (j < A::COPIES) a.copy(j, kleft, l0 + fill, wave);
    else b.copy(j - A::COPIES, kleft, l0 + fill + A::BYTES, wave);
  }
  template <typename Next>
  __device__ __forceinline__ void copied(Next& next) {
    a.next();
    b.next();
    fill = fill + STAGE == LDS ? 0 : fill + STAGE;
    item(kall - BK);
    if (kall <= 0) next();
  }
  __device__ __forceinline__ void read_one(const char* t, int k, int par, int i) {
    if (i < NI) fb[par][i] = b.read(t + A::BYTES, i, k);
    else fa[par][i - NI] = a.read(t, i - NI, k);
  }

  // a, b and the first item set: the first tiles on their way, the first one's
  // first operands read.
  template <typename Next>
  __device__ __forceinline__ void start(char* base, int w, Next& next) {
    lds = cur = base;
    l0 = (uint32_t)(uintptr_t)base;
    fill = 0;
    wave = w;
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int j = 0; j < (s < S - 1 ? COPIES : FIRST); ++j) copy_one(j);
      if (SPREAD == 1 || s < S - 1) copied(next);
    }
    wait_barrier<(S - 2) * COPIES + FIRST>();
#pragma unroll
    for (int i = 0; i < READS; ++i) read_one(cur, 0, 0, i);
  }

  // acc += the item's product, nt tiles of K.
  template <typename Next>
  __device__ __forceinline__ void run(f32x16 (&acc)[NI][MI], int nt, Next& next) {
    for (int t = 0; t < nt; ++t) {
#pragma unroll
      for (int k = 0; k < KK; ++k) {
        const bool last = k == KK - 1;
        const char* from = cur;
        if (last) {
          wait_barrier<(S - 2) * COPIES>();
          cur = cur + STAGE == lds + LDS ? lds : cur + STAGE;
          from = cur;
        }
        const int kn = last ? 0 : k + 1, part = last ? 0 : k + 1;
        int reads = 0, copies = min(part * FIRST, COPIES);
#pragma unroll
        for (int i = 0; i < NM; ++i) {
          // the next step's reads and the copies spread between the MFMAs
          const int want_r = ((i + 1) * READS + NM - 1) / NM;
#pragma unroll
          for (; reads < want_r; ++reads) read_one(from, kn, (k + 1) & 1, reads);
          if (part < SPREAD) {
            const int want_c = min(COPIES, part * FIRST + ((i + 1) * FIRST + NM - 1) / NM);
#pragma unroll
            for (; copies < want_c; ++copies) copy_one(copies);
          }
          const int n = i / MI, m = i % MI;
          acc[n][m] = mfma<T>(fb[k & 1][n], fa[k & 1][m], acc[n][m]);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (part == SPREAD - 1) copied(next);
      }
    }
  }
};

// Work item of a launch: XCDs take runs of neighbouring tiles, in groups of
// eight tile rows, so that the tiles that run at once share rows and columns.
__device__ __forceinline__ void tile_of(int idx, int tm, int tn, int& m, int& n) {
  constexpr int GROUP = 8;
  const int per = GROUP * tn, g = idx / per, in = idx - g * per;
  const int rows = min(GROUP, tm - g * GROUP);
  n = in / rows;
  m = g * GROUP + (in - n * rows);
}

}  // namespace gemm
}  // namespace hier
