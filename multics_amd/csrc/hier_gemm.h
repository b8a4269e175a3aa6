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
// K tiles of 64 go HBM/L2 -> LDS with buffer_load_dwordx4 ... lds.
// A buffer load out of its range writes zeros: rows past the end, the ragged
// last K tile and tiles past the end need no other handling, and nothing past a
// view's last element is read.  The operands of step k+1 are read while the
// MFMAs of step k run.  One barrier a tile, before its last step: by then every
// wave has read the tile to its end, and the next tile has landed, so the last
// step starts on the next tile and its slots are filled anew.
//
// Measured: 2,343 cycles a 256 x 256 x 64 tile, 2,048 of them the MFMAs'; no bank
// conflicts (counted).  128 x 128 tiles, two workgroups a CU, take 0.6 of the time of a
// 256 x 256 one for a quarter of its work: for products of few tiles.
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

// 16 x 16 x 32: lane l holds row l % 16, k 8 (l / 16) .. + 8 of both operands.
template <typename T>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  const vec8<T> x = __builtin_bit_cast(vec8<T>, a), y = __builtin_bit_cast(vec8<T>, b);
  if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
}

// 32 x 32 x 16: lane l holds row l % 32, k 8 (l / 32) .. + 8.
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
  uint64_t base;       // first byte of the tile to copy next
  uint32_t range;      // bytes from there that the copies may read
  uint32_t step;       // bytes to the next tile
  int kall;            // K left of the item, from `base` on
  uint32_t voff, sstep;
  int k8;              // rows: the lane's first k of a tile
  int rd[TR ? MI : KK];

  // rows: view of `rows` x K, ld elements apart, from row `first`, k0 on.
  // transposed: view of K x `rows`.
  __device__ __forceinline__ void init(const void* p, int64_t ld, int64_t rows, int64_t first, int64_t k0,
                                       int64_t kend, int wave, int part, int lane) {
    const int line = lane / CPR, pos = lane % CPR;
    int64_t bytes;
    if constexpr (TR) {
      rows = (rows + 7) / 8 * 8;         // (a view's rows of k are whole chunks)
      const int chunk = pos ^ (4 * ((LPC * wave + line) & 3));
      base = (uint64_t)p + 2 * (k0 * ld + first);
      bytes = 0x7fffffff;                // (the end of K: see edge)
      step = (uint32_t)(2 * BK * ld);
      voff = (uint32_t)((LPC * wave + line) * (int)(2 * ld) + 16 * chunk);
      if (first + 8 * chunk >= rows) voff = kOut;
      k8 = (int)(2 * (rows - first));    // bytes of a row of k
#pragma unroll
      for (int b = 0; b < MI; ++b) {
        const int i = lane & 15, r = 8 * (lane >> 5) + (i >> 2);
        const int q = 4 * (part * MI + b) + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
        rd[b] = r * (2 * R) + 16 * (q ^ (4 * (r & 3))) + 8 * (i & 1);
      }
    } else {
      const int row = LPC * wave + line;
      const int chunk = pos ^ (row / (128 / BK) % CPR);
      base = (uint64_t)p + 2 * (first * ld + k0);
      // up to the last row's end, seen from the item's first tile: a row past it starts
      // behind that from any tile (the view's rows do not overlap)
      bytes = 2 * ((rows - first - 1) * ld + (kend - k0 + 7) / 8 * 8);   // (whole chunks)
      step = 2 * BK;
      voff = (uint32_t)(row * (int)(2 * ld) + 16 * chunk);
      k8 = 8 * chunk;
      const int r = lane & 31;
#pragma unroll
      for (int k = 0; k < KK; ++k)
        rd[k] = (part * 32 * MI + r) * (2 * BK) + 16 * ((2 * k + (lane >> 5)) ^ (r / (128 / BK) % CPR));
    }
    sstep = (uint32_t)(4 * LPC * (2 * ld));
    range = (uint32_t)(bytes < 0x7fffffff ? bytes : 0x7fffffff);
    kall = (int)(kend - k0);
    if (kall < BK) edge();
  }
  // The item's last tile is not a whole one: chunks (rows of k) past its end are out of
  // range.
  __device__ __forceinline__ void edge() {
    if constexpr (TR) range = (uint32_t)((kall - 1) * (int)(step / BK) + k8);
    else if (k8 >= kall) voff = kOut;
  }

  // Copy j of the wave's for the tile that `base` is at.  (The whole offset is in the
  // lane's register: that is what the range check sees.  kOut plus the copies' rows,
  // under 2^30, stays past every range.)
  __device__ __forceinline__ void copy(int j, uint32_t lds, int wave) const {
    const u32x4 srd = {(uint32_t)base, (uint32_t)(base >> 32), range, 0x00020000u};
    dma(srd, voff + j * sstep, lds + 1024 * (wave + 4 * j));
  }
  // The next tile; true past the item's last.
  __device__ __forceinline__ bool next() {
    base += step;
    kall -= BK;
    if (kall >= BK) return false;
    if (kall <= 0) return true;
    edge();
    return false;
  }
  // No more tiles: the copies write zeros.
  __device__ __forceinline__ void end() {
    range = 0;
    kall = 0x7fffffff;
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
// LDS is a ring of five slots of one operand's tile each, filled in the order A0 B0
// A1 B1 A2 ..: with two tiles of both in use or on their way there is room for a
// third of A, so the copies leave evenly over the four steps of a tile -- the second
// half of B(t+1), A(t+2) in two steps, the first half of B(t+2) -- at the rate at which
// the caches deliver them (42 bytes a cycle and CU, three quarters of what the MFMAs
// leave time for), and each has two steps at least to land.  (Two stages of both,
// copies in one step of four: 8192^3 at 1,184 TFLOP/s, in two 1,234, in three 1,189.)
//
// The K tiles of a workgroup's work items are one stream: while an item is
// multiplied, and while its results go out, the copies run ahead into the next
// (`next_a`, `next_b` set the operands to it), so only the first one waits for memory.
template <typename T, bool ATR, bool BTR, int BM, int BN, int BK>
struct Product {
  typedef Operand<ATR, BM, BK> A;
  typedef Operand<BTR, BN, BK> B;
  static constexpr int MI = A::MI, NI = B::MI, KK = A::KK;
  static constexpr int SLOT = A::BYTES;
  static constexpr int LDS = 5 * SLOT;
  static constexpr int COPIES = A::COPIES, HALF = COPIES / 2;    // of one operand
  static constexpr int READS = MI + NI, NM = NI * MI;
  static_assert(KK == 4 && A::BYTES == B::BYTES && NM % READS == 0 && NM % HALF == 0, "");

  A a;
  B b;
  uint32_t l0;            // LDS address of the ring
  uint32_t fill;          // slot that is being filled, in bytes; in use: A and B of the
  uint32_t at_a, at_b;    // present tile
  const char* lds;
  int wave;
  u32x4 fa[2][MI], fb[2][NI];

  static __device__ __forceinline__ uint32_t after(uint32_t slot, int n) {
    slot += n * SLOT;
    return slot >= LDS ? slot - LDS : slot;
  }
  __device__ __forceinline__ void copy_a(int j) { a.copy(j, l0 + fill, wave); }
  __device__ __forceinline__ void copy_b(int j) { b.copy(j, l0 + fill, wave); }
  template <typename Next>
  __device__ __forceinline__ void done_a(Next& next) {
    fill = after(fill, 1);
    if (a.next()) next();
  }
  template <typename Next>
  __device__ __forceinline__ void done_b(Next& next) {
    fill = after(fill, 1);
    if (b.next()) next();
  }
  __device__ __forceinline__ void read_one(uint32_t from_a, uint32_t from_b, int k, int par, int i) {
    if (i < NI) fb[par][i] = b.read(lds + from_b, i, k);
    else fa[par][i - NI] = a.read(lds + from_a, i - NI, k);
  }
  // The slot that nothing uses between two items.
  __device__ __forceinline__ uint32_t spare() const { return after(fill, 1); }

  // a and b set to the first item: the first tiles on their way, the first one's
  // first operands read.
  template <typename NextA, typename NextB>
  __device__ __forceinline__ void start(char* base, int w, NextA& next_a, NextB& next_b) {
    lds = base;
    l0 = (uint32_t)(uintptr_t)base;
    fill = at_a = 0;
    at_b = SLOT;
    wave = w;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int j = 0; j < COPIES; ++j) copy_a(j);
      done_a(next_a);
#pragma unroll
      for (int j = 0; j < (t ? HALF : COPIES); ++j) copy_b(j);
      if (!t) done_b(next_b);
    }
    wait_barrier<COPIES + HALF>();
#pragma unroll
    for (int i = 0; i < READS; ++i) read_one(at_a, at_b, 0, 0, i);
  }

  // acc += the item's product, nt tiles of K.
  template <typename NextA, typename NextB>
  __device__ __forceinline__ void run(f32x16 (&acc)[NI][MI], int nt, NextA& next_a, NextB& next_b) {
    for (int t = 0; t < nt; ++t) {
#pragma unroll
      for (int k = 0; k < KK; ++k) {
        const bool last = k == KK - 1;
        if (last) {
          // every wave has read this tile to its end, and the next one is here: all
          // copies but those of A(t+2)
          wait_barrier<COPIES>();
          at_a = after(at_a, 2);
          at_b = after(at_b, 2);
        }
        const int kn = last ? 0 : k + 1;
        // the next step's reads between the MFMAs of the first half of this one, the
        // copies between all
        int reads = 0;
        constexpr int PER_COPY = NM / HALF;
#pragma unroll
        for (int i = 0; i < NM; ++i) {
          const int want_r = min(READS, (2 * (i + 1) * READS + NM - 1) / NM);
#pragma unroll
          for (; reads < want_r; ++reads) read_one(at_a, at_b, kn, (k + 1) & 1, reads);
          if (i % PER_COPY == 0) {
            const int c = i / PER_COPY;
            if (k == 0) copy_b(HALF + c);
            else if (last) copy_b(c);
            else copy_a((k - 1) * HALF + c);
          }
          const int n = i / MI, m = i % MI;
          acc[n][m] = mfma<T>(fb[k & 1][n], fa[k & 1][m], acc[n][m]);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (k == 0) done_b(next_b);
        if (k == 2) done_a(next_a);
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
