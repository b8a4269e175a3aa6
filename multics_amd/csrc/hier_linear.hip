// Matrix product with bias, activation, gate and residual in its epilogue, and
// the gradients of it:
//   z = x W^T + b,   y = r + g * act(z)
//   dz = dy * g * act'(z),   dx = dz W,   dW = dz^T x,   db = sum of dz's rows,
//   dg = sum over a gate's rows of dy * act(z)
// (x [M][K], W [N][K], g one row for rows_per_gate rows of y.)  Everything is
// summed in fp32 and y rounded once.  A training step also writes z rounded to
// 16 bits (fp16 with an activation: no lower than -65504; act' and dg are taken at it: an error of half a step of z, as y's own
// rounding is one of y), and dz is rounded to 16 bits as the two products'
// operand; db is summed from dz before that rounding.
//
// The products run on the tiles of hier_gemm.h; few rows of x on kernels that stream
// the weights past them.  Measured, bf16: 18,816 x 8,960 x 1,536 430 us (1,204 TFLOP/s),
// with tanh GELU 477 -- a tile's epilogue takes 9 us beside the 35 of its products, 13
// with the GELU's two transcendentals an element --, of K 7,680 1,304 TFLOP/s: there the
// power limit sets the clock, and nothing but energy is left to save.  6,600 x 1,536 x 8,960 with gate and
// residual 170: 156 tiles, so 100 of 256 CUs idle (a library product of that size 145, 155 with
// gated_residual behind it).  Gradients of 9,408 x 8,960 x 1,536: dz 115, dx 203, dw 206 (1,270 and
// 1,250 TFLOP/s).  1,536 x 1,536 for 660 / 4,620 / 18,816 rows 15 / 28 / 85, library 19 / 27 / 73:
// short K, where a tile's epilogue is a fifth of it.
#include "hier_gemm.h"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace hier {
namespace {

using gemm::f32x16;
using gemm::u32x4;

// ---- epilogue ------------------------------------------------------------------

struct Epilogue {
  const void* bias;
  const void* residual;
  const void* gate;
  void* out;
  void* preact;
  float* partial;          // fp32 [splits][M][ld_part]: sums alone, no epilogue
  int64_t residual_ss, gate_ss, out_ss, preact_ss, ld_part, part_stride;
  Div rows_per_gate;
  int32_t act;
};

__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

// tanh GELU as z sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3): no cancellation
// where z is far below 0.
constexpr float kGeluA = 1.5957691216057308f, kGeluB = 0.044715f;   // 2 sqrt(2/pi)
__device__ __forceinline__ float gelu_gate(float z) {                // sigmoid(2u)
  constexpr float L = -1.4426950408889634f;
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * fmaf(L * kGeluA * kGeluB, z * z, L * kGeluA)));
}

__device__ __forceinline__ void activate8(float* v, int act) {
  if (act == HIER_ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= gelu_gate(v[i]);
  } else if (act == HIER_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= sigmoid(v[i]);
  } else if (act == HIER_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= 0.5f * erfcf(-0.7071067811865476f * v[i]);
  }
}

// act(z) and act'(z).  Past |z| = 30 (SiLU: 100) the slopes are 0 or 1 to fp32: z is kept
// there, so no square of it overflows into inf * 0.  (The clamp takes a NaN to one of its
// bounds: its slope is set right by keep_nans.)
template <int ACT>
__device__ __forceinline__ void activate2(float z, float& a, float& slope) {
  if constexpr (ACT == HIER_ACT_GELU_TANH) {
    const float c = __builtin_amdgcn_fmed3f(z, -30.f, 30.f), s = gelu_gate(c);
    a = z * s;
    slope = fmaf(c * fmaf(3.f * kGeluA * kGeluB, c * c, kGeluA), fmaf(-s, s, s), s);
  } else if constexpr (ACT == HIER_ACT_GELU) {
    const float c = __builtin_amdgcn_fmed3f(z, -30.f, 30.f), half = 0.5f * erfcf(-0.7071067811865476f * z);
    a = z * half;
    slope = half + c * 0.3989422804014327f * __builtin_amdgcn_exp2f(-0.7213475204444817f * c * c);
  } else if constexpr (ACT == HIER_ACT_SILU) {
    const float c = __builtin_amdgcn_fmed3f(z, -100.f, 100.f), s = sigmoid(c);
    a = z * s;
    slope = fmaf(c, fmaf(-s, s, s), s);
  } else {
    a = z;
    slope = 1.f;
  }
}

// dz is NaN where z is.  By the bits: the compiler takes it that there are no NaNs and drops
// comparisons and classes of floats.  One test for eight values, as hardly any row has one
// (a test a value: 118 -> 126 us for 9,408 x 8,960).
__device__ __forceinline__ uint32_t magnitude(float z) { return __float_as_uint(z) << 1; }
__device__ __forceinline__ void keep_nans(const float* z, float* dz) {
  constexpr uint32_t INF = 0xff000000u;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, magnitude(z[i]));
  if (top <= INF) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) dz[i] = magnitude(z[i]) > INF ? z[i] : dz[i];
}

// Eight neighbouring channels of 16 bits, at any even address (the hardware takes
// 16-byte accesses there).
template <typename T>
__device__ __forceinline__ w32x4 raw8(const void* p, int64_t at) {
  w32x4 w;
  __builtin_memcpy(&w, static_cast<const T*>(p) + at, 16);
  return w;
}
template <typename T>
__device__ __forceinline__ void put8(void* p, int64_t at, const float* f) {
  const w32x4 w = narrow<T>(f);
  __builtin_memcpy(static_cast<T*>(p) + at, &w, 16);
}
// The same where fewer than eight are left: zeros behind, which are not written.
template <typename T>
__device__ __forceinline__ void row8(const void* p, int64_t at, int n, int N, float* f) {
  if (n + 8 <= N) {
    widen<T>(raw8<T>(p, at + n), f);
  } else {
    T t[8];                    // (the last one's again past the end: no branch is between the loads)
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = static_cast<const T*>(p)[at + min(n + i, N - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = n + i < N ? (float)t[i] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void put_row8(void* p, int64_t at, int n, int N, const float* f) {
  if (n + 8 <= N) {
    put8<T>(p, at + n, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < N) static_cast<T*>(p)[at + n + i] = (T)f[i];
  }
}

// z as it is kept for the gradient.  Below fp16's range every activation and its slope are
// 0, at -65504 as there, while -inf would make the gate's gradient -inf * 0.  (By the bits,
// as NaNs pass; -inf itself stays, and so does overflow above, as y's own.)
template <typename T>
__device__ __forceinline__ void kept(const float* v, int act, float* z) {
  constexpr uint32_t LOW = 0xc77fe000u, INF = 0xff800000u;      // -65504, -inf
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = v[i];
  if constexpr (__is_same(T, _Float16)) {
    if (act == HIER_ACT_NONE) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = __float_as_uint(v[i]) - LOW < INF - LOW ? -65504.f : v[i];
  }
}

__device__ __forceinline__ uint32_t gate_row(const Epilogue& e, int64_t m) {
  return e.gate ? quotient((uint32_t)m, e.rows_per_gate) : 0u;
}

// The whole epilogue of eight channels of one row: what it reads, and the rest of it.
template <typename T>
struct Finish {
  float bias[8], gate[8], residual[8];
  __device__ __forceinline__ void read(const Epilogue& e, int64_t m, int n, int N) {
    if (e.bias) row8<T>(e.bias, 0, n, N, bias);
    if (e.gate) row8<T>(e.gate, (int64_t)gate_row(e, m) * e.gate_ss, n, N, gate);
    if (e.residual) row8<T>(e.residual, m * e.residual_ss, n, N, residual);
  }
  __device__ __forceinline__ void write(const Epilogue& e, float* v, int64_t m, int n, int N) const {
    if (e.bias) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += bias[i];
    }
    if (e.preact) {
      float z[8];
      kept<T>(v, e.act, z);
      put_row8<T>(e.preact, m * e.preact_ss, n, N, z);
    }
    activate8(v, e.act);
    if (e.gate) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= gate[i];
    }
    if (e.residual) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += residual[i];
    }
    put_row8<T>(e.out, m * e.out_ss, n, N, v);
  }
};
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue& e, float* v, int64_t m, int n, int N) {
  Finish<T> f;
  f.read(e, m, n, N);
  f.write(e, v, m, n, N);
}

// ---- products over LDS tiles -----------------------------------------------------

struct GemmArgs {
  const void* a;
  const void* b;
  int64_t lda, ldb, M, N, K;
  int64_t m_first;             // row of the launch's first tile
  int64_t kchunk;              // K of a split, a multiple of the tile's
  int32_t tm, tn, splits, total;
  Epilogue e;
};

// What a launch's epilogue needs: kPlain has neither gate nor residual, kExtra may
// have them; both take 16-byte rows.  kAny takes any.
enum { kPlain, kExtra, kAny };

// Rows of a tile in one of the epilogue's tensors.  Buffer accesses: one out of
// range is a row or column that is not there, with no branch around it, so the
// compiler knows how many accesses are on their way and a load is not waited for
// with the stores behind it.
struct View {
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ __forceinline__ void init(const void* p, int64_t at) {
    rsrc = __builtin_amdgcn_make_buffer_rsrc((char*)p + at, 0, 0x7fffffff, 0x00020000);
  }
  __device__ __forceinline__ u32x4 load(uint32_t off) const {
    return __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0);
  }
  __device__ __forceinline__ u32x4 load_once(uint32_t off) const {      // not kept in the caches
    return __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 2);
  }
  __device__ __forceinline__ void store(const u32x4& v, uint32_t off) const {
    __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, off, 0, 0);
  }
  // Results: through the L2 as they come (scope of the GPU, non-temporal).  Left in it a
  // round's (4 MB an XCD, all it holds) push the operands out: 18,816 x 8,960 x 1,536
  // 438 -> 429 us, 4,300 x 4,096 x 512 35.4 -> 32.5.  (Parts are read again: left in it.)
  __device__ __forceinline__ void stream(const u32x4& v, uint32_t off) const {
    __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, off, 0, 18);
  }
};

// Pass K's sums (32 rows, COLS x 32 channels) into the wave's part of LDS.
template <int K, int NI, int MI, int COLS>
__device__ __forceinline__ void put_sums_of(const f32x16 (&acc)[NI][MI], char* mine, int lane) {
  constexpr int HALVES = NI / COLS, mi = K / HALVES, ni = K % HALVES * COLS;
  const int r = lane & 31;
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x16& s = acc[ni + c][mi];
      *reinterpret_cast<f32x4*>(mine + r * (COLS * 128) +
                                16 * ((8 * c + 2 * q + (lane >> 5)) ^ (r % (8 * COLS)))) =
          f32x4{s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
    }
  // (unlike in every pass: with their ends merged, the passes would choose their sums by address)
  asm volatile("; pass %0" :: "i"(K) : "memory");
}
// The pass by number: registers cannot be chosen by one, hence a test for each.  (The
// passes are a loop: unrolled they would not fit the instruction cache.)
template <int NI, int MI, int COLS, int... K>
__device__ __forceinline__ void put_sums(const f32x16 (&acc)[NI][MI], char* mine, int lane, int pass,
                                         std::integer_sequence<int, K...>) {
  ((pass == K ? put_sums_of<K, NI, MI, COLS>(acc, mine, lane) : (void)0), ...);
}

// Workgroups in flight: one a CU (WG of them); each takes its XCD's items in
// turn, the XCD's workgroups neighbouring ones.
constexpr int kSlots = 256;

template <typename T, bool ATR, bool BTR, int BM, int BN, int BK, int WG, int KIND>
__global__ __launch_bounds__(256, WG) void gemm_kernel(GemmArgs g) {
  typedef gemm::Product<T, ATR, BTR, BM, BN, BK> P;
  // The sums leave through LDS, 32 rows x 32 COLS channels of a wave at a time, so
  // that a row's channels are neighbours again and the accesses whole lines.
  // 16-byte chunk c of row r sits at c ^ (r % (8 COLS)): neither side meets in a bank.
  constexpr int NI = P::NI, MI = P::MI, COLS = WG == 1 ? 2 : 1, PITCH = COLS * 128;
  constexpr int LPR = COLS * 4, RPI = 64 / LPR, ITS = 32 / RPI;    // lanes a row, rows an access
  constexpr int HALVES = NI / COLS, PASSES = MI * HALVES;
  static_assert(4 * 32 * PITCH == P::SLOT, "the sums leave through the spare slot");
  __shared__ __align__(1024) char lds[P::LDS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int per = (int)gridDim.x / kXcds;           // workgroups of an XCD
  const int chunk = (g.total + kXcds - 1) / kXcds;  // items of an XCD
  const int xcd = blockIdx.x % kXcds;
  const int end = min((xcd + 1) * chunk, g.total);
  const int first = xcd * chunk + blockIdx.x / kXcds;
  if (first >= end) return;

  P p;
  // operand A or B at an item's first tile
  int item_a = first, item_b = first;
  auto set = [&](int item, bool of_a) {
    const int split = item / (g.tm * g.tn);
    int tm, tn;
    gemm::tile_of(item - split * g.tm * g.tn, g.tm, g.tn, tm, tn);
    const int64_t k0 = split * g.kchunk, k1 = min(k0 + g.kchunk, g.K);
    if (of_a) p.a.init(g.a, g.lda, g.M, g.m_first + (int64_t)tm * BM, k0, k1, wave, wm, lane);
    else p.b.init(g.b, g.ldb, g.N, (int64_t)tn * BN, k0, k1, wave, wn, lane);
  };
  auto next_a = [&]() {
    item_a += per;
    if (item_a < end) set(item_a, true);
    else p.a.end();
  };
  auto next_b = [&]() {
    item_b += per;
    if (item_b < end) set(item_b, false);
    else p.b.end();
  };
  set(first, true);
  set(first, false);
  p.start(lds, wave, next_a, next_b);
  const int N = (int)g.N;
  char* mine = nullptr;           // the wave's part of the spare slot
  auto chunk_at = [&](int r, int c) { return mine + r * PITCH + 16 * (c ^ (r % (8 * COLS))); };

  for (int item = first; item < end; item += per) {
    const int split = item / (g.tm * g.tn);
    int tm, tn;
    gemm::tile_of(item - split * g.tm * g.tn, g.tm, g.tn, tm, tn);
    const int64_t k0 = split * g.kchunk;
    const int nt = (int)((min(k0 + g.kchunk, g.K) - k0 + BK - 1) / BK);
    const int64_t m0 = g.m_first + (int64_t)tm * BM + wm * MI * 32;
    const int n0 = tn * BN + wn * NI * 32;
    const int rows = (int)min(g.M - m0, (int64_t)(32 * MI));     // (may be none)
    f32x16 acc[NI][MI];
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][m][i] = 0.f;

    // The lane as the epilogue sees it: opaque, so that what it computes of it is not
    // kept in registers through the product.
    int el = lane;
    if constexpr (KIND == kAny) {
      p.run(acc, nt, next_a, next_b);
      mine = lds + p.spare() + wave * 32 * PITCH;
      asm volatile("" : "+v"(el));
      const int j = el % LPR, row = el / LPR;
#pragma unroll 1
      for (int pass = 0; pass < PASSES; ++pass) {
        put_sums<NI, MI, COLS>(acc, mine, el, pass, std::make_integer_sequence<int, PASSES>{});
        const int n = n0 + 32 * COLS * (pass % HALVES) + 8 * j;
        if (n >= N) continue;
#pragma unroll 1
        for (int it = 0; it < ITS; ++it) {
          const int r = it * RPI + row, mr = pass / HALVES * 32 + r;
          if (mr >= rows) continue;
          const f32x4 lo = *reinterpret_cast<const f32x4*>(chunk_at(r, 2 * j));
          const f32x4 hi = *reinterpret_cast<const f32x4*>(chunk_at(r, 2 * j + 1));
          float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          finish8<T>(g.e, v, m0 + mr, n, N);
        }
      }
    } else {
      // offset of row r (of the wave's part) at channel n in a tensor of row stride ss
      auto off = [&](int r, int n, int64_t ss) {
        return r < rows && n < N ? (uint32_t)(r * (int)(2 * ss) + 2 * n) : gemm::kOut;
      };
      View vb;
      u32x4 bias[HALVES], res[ITS], gate[ITS], held[ITS];
      if (g.e.bias && g.splits == 1) {
        vb.init(g.e.bias, 0);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          const int n = n0 + 32 * COLS * h + 8 * (lane % LPR);
          bias[h] = vb.load(n < N ? 2 * n : gemm::kOut);
        }
      } else {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) bias[h] = u32x4{0u, 0u, 0u, 0u};
      }
      p.run(acc, nt, next_a, next_b);
      mine = lds + p.spare() + wave * 32 * PITCH;
      asm volatile("" : "+v"(el));
      const int j = el % LPR, row = el / LPR;
      View vo, vz, vr, vg;
      vo.init(g.e.out, 2 * m0 * g.e.out_ss);
      vz.init(g.e.preact, 2 * m0 * g.e.preact_ss);
      const uint32_t gate0 = gate_row(g.e, min(m0, g.M - 1));
      if constexpr (KIND == kExtra) {
        vr.init(g.e.residual, 2 * m0 * g.e.residual_ss);
        vg.init(g.e.gate, 2 * (int64_t)gate0 * g.e.gate_ss);
#pragma unroll
        for (int it = 0; it < ITS; ++it) held[it] = u32x4{0u, 0u, 0u, 0u};
      }
      // (here, so that no pass waits for it and with it for the stores of the one before)
#pragma unroll
      for (int h = 0; h < HALVES; ++h) asm volatile("" : "+v"(bias[h]));
      uint32_t to[ITS];
#pragma unroll
      for (int it = 0; it < ITS; ++it) to[it] = gemm::kOut;
#pragma unroll 1
      for (int pass = 0; pass < PASSES; ++pass) {
        const int h = pass % HALVES, n = n0 + 32 * COLS * h + 8 * j, r0 = pass / HALVES * 32 + row;
        if constexpr (KIND == kExtra) {
          // this pass's residual and gate are asked for before the results of the pass
          // before go out: the wait for them is not one for those stores
          if (g.e.gate) {
#pragma unroll
            for (int it = 0; it < ITS; ++it) {
              const int r = r0 + it * RPI;
              const uint32_t gr = gate_row(g.e, min(m0 + r, g.M - 1)) - gate0;
              gate[it] = vg.load(r < rows && n < N ? gr * (uint32_t)(2 * g.e.gate_ss) + 2 * n : gemm::kOut);
            }
          }
          // (without a residual its view takes zeros: out of range)
#pragma unroll
          for (int it = 0; it < ITS; ++it)
            res[it] = vr.load(g.e.residual ? off(r0 + it * RPI, n, g.e.residual_ss) : gemm::kOut);
#pragma unroll
          for (int it = 0; it < ITS; ++it) vo.stream(held[it], to[it]);
        }
        put_sums<NI, MI, COLS>(acc, mine, el, pass, std::make_integer_sequence<int, PASSES>{});
        f32x4 lo[ITS], hi[ITS];
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
          lo[it] = *reinterpret_cast<const f32x4*>(chunk_at(it * RPI + row, 2 * j));
          hi[it] = *reinterpret_cast<const f32x4*>(chunk_at(it * RPI + row, 2 * j + 1));
        }
        if (KIND == kPlain && g.splits > 1) {
          View vp;
          vp.init(g.e.partial, 4 * (split * g.e.part_stride + m0 * g.e.ld_part));
#pragma unroll
          for (int it = 0; it < ITS; ++it) {
            const int r = r0 + it * RPI;
            const bool there = r < rows && n < N;
            const uint32_t at = there ? (uint32_t)(r * (int)(4 * g.e.ld_part) + 4 * n) : gemm::kOut;
            vp.store(__builtin_bit_cast(u32x4, lo[it]), at);
            vp.store(__builtin_bit_cast(u32x4, hi[it]), there ? at + 16 : gemm::kOut);
          }
          continue;
        }
        float b[8];
        u32x4 braw = bias[0];
#pragma unroll
        for (int i = 1; i < HALVES; ++i) braw = h == i ? bias[i] : braw;
        widen<T>(braw, b);
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
          float v[8] = {lo[it][0], lo[it][1], lo[it][2], lo[it][3], hi[it][0], hi[it][1], hi[it][2], hi[it][3]}, t[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += b[i];
          if (g.e.preact) {
            kept<T>(v, g.e.act, t);
            vz.stream(narrow<T>(t), off(r0 + it * RPI, n, g.e.preact_ss));
          }
          activate8(v, g.e.act);
          const uint32_t at = off(r0 + it * RPI, n, g.e.out_ss);
          if constexpr (KIND == kExtra) {
            if (g.e.gate) {
              widen<T>(gate[it], t);
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] *= t[i];
            }
            widen<T>(res[it], t);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += t[i];
            held[it] = narrow<T>(v);
            to[it] = at;
          } else {
            vo.stream(narrow<T>(v), at);
          }
        }
      }
      if constexpr (KIND == kExtra)
#pragma unroll
        for (int it = 0; it < ITS; ++it) vo.stream(held[it], to[it]);
    }
    // every wave is done with the spare slot before it is filled
    barrier_lds();
  }
  // no copy may be on its way when the workgroup ends
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// The splits' sums in their order, and the epilogue.
template <typename T>
__global__ __launch_bounds__(256, 4) void join_kernel(GemmArgs g) {
  const int cpr = (int)((g.N + 7) / 8);
  const int64_t n8 = g.M * cpr;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n8; i += (int64_t)gridDim.x * 256) {
    const int64_t m = n8 >> 32 ? i / cpr : (uint32_t)i / (uint32_t)cpr;
    const int n = 8 * (int)(i - m * cpr);
    const float* p = g.e.partial + m * g.e.ld_part + n;
    float v[8] = {};
    Finish<T> f;
    // (eight splits' loads leave together, the last split's again past the end, and with the
    // first ones those of the epilogue)
    for (int s = 0; s < g.splits; s += 8) {
      f32x4 x[8][2];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i == 4 && s + 4 >= g.splits) break;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          x[i][h] = *reinterpret_cast<const f32x4*>(p + min(s + i, g.splits - 1) * g.e.part_stride + 4 * h);
      }
      if (s == 0) f.read(g.e, m, n, (int)g.N);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (s + i >= g.splits) break;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += x[i][j / 4][j % 4];
      }
    }
    f.write(g.e, v, m, n, (int)g.N);
  }
}

// ---- few rows --------------------------------------------------------------------
//
// Up to 64 rows of x, of weights that are not many (few_rows).  A workgroup of eight
// waves takes 16 output channels, a wave every eighth 128-wide piece of K, with its
// weights straight from memory into the MFMA's registers (16 rows x 32 k: 16 bytes a
// lane); the eight sums meet in LDS.  Bound by a wait for memory a piece and by x,
// read again for every 16 channels: 9 / 64 rows of 1536 x 1536 5.2 / 10.2 us.
// v_mfma_f32_16x16x32: lane l holds row l % 16, k 8 (l / 16) .. + 8 of both operands,
// and of the result row (channel) 4 (l / 16) + i, column (row of x) l % 16.

constexpr int kFewWaves = 8;
constexpr int kFewAhead = 4;       // 32-wide pieces of K in flight

template <typename T, int MT>      // MT groups of 16 rows of x
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(GemmArgs g) {
  __shared__ float sums[kFewWaves][MT][64 * 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, kg = 8 * (lane >> 4);
  const int64_t n0 = 16 * (int64_t)blockIdx.x;
  const T* wp = static_cast<const T*>(g.b) + min(n0 + r, g.N - 1) * g.ldb + kg;
  const T* xp[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
    xp[m] = static_cast<const T*>(g.a) + min((int64_t)(16 * m + r), g.M - 1) * g.lda + kg;
  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  // pieces of kFewAhead x 32 k, in turn over the waves
  constexpr int PIECE = 32 * kFewAhead;
  for (int64_t k0 = (int64_t)wave * PIECE; k0 < g.K; k0 += kFewWaves * PIECE) {
    u32x4 w[kFewAhead], x[MT][kFewAhead];
    const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < kFewAhead; ++j) {
      const int64_t k = k0 + 32 * j;
      const bool in = k + kg < g.K;      // (K is a multiple of 8)
      w[j] = in ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp + k)) : zero;
#pragma unroll
      for (int m = 0; m < MT; ++m) x[m][j] = in ? *reinterpret_cast<const u32x4*>(xp[m] + k) : zero;
    }
#pragma unroll
    for (int j = 0; j < kFewAhead; ++j)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m] = gemm::mfma16<T>(w[j], x[m][j], acc[m]);
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][m][(lane & 15) * 16 + 4 * (lane >> 4) + i] = acc[m][i];
  __syncthreads();
  // thread: row t / 2 of x, eight channels
  const int t = threadIdx.x;
  if (t >= 32 * MT) return;
  const int64_t m = t / 2;
  const int n = (int)n0 + 8 * (t & 1);
  if (m >= g.M || n >= g.N) return;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) s += sums[w][m / 16][(m % 16) * 16 + 8 * (t & 1) + i];
    v[i] = s;
  }
  finish8<T>(g.e, v, m, n, (int)g.N);
}

// ---- fewer rows still ------------------------------------------------------------
//
// At most eight rows of x: one product a weight and row, on the vector units, with
// the weights in the order of memory (a wave's load is 1 KB of one channel, where
// few_rows_kernel's takes 64 bytes of 16).  A workgroup of four waves takes CH
// channels, a wave every fourth 512-wide piece of K of all of them, x's piece read
// once for them; the sums meet in LDS.  Measured for 1 row of K 1536 x N 8960 /
// 8960 x 1536 / 4096 x 16384 (weights of 27.5, 27.5 and 134 MB): 6.2 / 6.4 / 21 us
// (6.3 TB/s), of few_rows_kernel 9.0 / 14.8 / 27; 8 rows 10.5 / 11.6 / 26 for 10.7 /
// 18 / 32.  More channels a workgroup read x less often, fewer make more workgroups:
// two up to two rows, else as many as the rows (1 row with 8: 6.4 / 7.2 / 22; 8 rows
// with 2: 10.7 / 11.6 / 43).

template <typename T>
__device__ __forceinline__ float dot8(const u32x4& a, const u32x4& b, float c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t x = a[e], y = b[e];     // (a bit cast of an element reads the first)
    if constexpr (__is_same(T, __bf16)) {
      typedef __bf16 pair __attribute__((ext_vector_type(2)));
      c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, x), __builtin_bit_cast(pair, y), c, false);
    } else {
      typedef _Float16 pair __attribute__((ext_vector_type(2)));
      c = __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, x), __builtin_bit_cast(pair, y), c, false);
    }
  }
  return c;
}

// Sums of N lanes' values over the wave: lane l returns that of value l % N.  Each step
// hands half of the values to the lanes that keep the other half.
template <int N>
__device__ __forceinline__ float wave_sums(float* v, int lane) {
#pragma unroll
  for (int n = N / 2, d = 1; d < 64; n /= 2, d *= 2) {
    if (n > 0) {
      const bool odd = lane & d;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float keep = odd ? v[2 * i + 1] : v[2 * i], give = odd ? v[2 * i] : v[2 * i + 1];
        v[i] = keep + __shfl_xor(give, d, 64);
      }
    } else {
      v[0] += __shfl_xor(v[0], d, 64);
    }
  }
  return v[0];
}

constexpr int kDotRows = 8;

template <typename T, int M>       // M rows of x at most: 1, 2, 4 or 8
__global__ __launch_bounds__(256) void dot_kernel(GemmArgs g) {
  constexpr int CH = M < 2 ? 2 : M;
  __shared__ float sums[4][M * CH];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)CH * blockIdx.x;
  View wv[CH], xv[M];
#pragma unroll
  for (int c = 0; c < CH; ++c) wv[c].init(g.b, 2 * min(n0 + c, g.N - 1) * g.ldb);
#pragma unroll
  for (int m = 0; m < M; ++m) xv[m].init(g.a, 2 * min((int64_t)m, g.M - 1) * g.lda);
  float acc[M * CH] = {};
  const int K = (int)g.K;
  for (int k0 = 512 * wave; k0 < K; k0 += 2048) {
    const int k = k0 + 8 * lane;
    const uint32_t at = k < K ? 2u * k : gemm::kOut;       // (K is a multiple of 8; out of range gives zeros)
    u32x4 w[CH], x[M];
#pragma unroll
    for (int c = 0; c < CH; ++c) w[c] = wv[c].load_once(at);
#pragma unroll
    for (int m = 0; m < M; ++m) x[m] = xv[m].load(at);
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int c = 0; c < CH; ++c) acc[m * CH + c] = dot8<T>(w[c], x[m], acc[m * CH + c]);
  }
  const float s = wave_sums<M * CH>(acc, lane);
  if (lane < M * CH) sums[wave][lane] = s;
  __syncthreads();
  // thread: a channel of a row
  const int t = threadIdx.x, m = t / CH, n = (int)n0 + t % CH;
  if (t >= M * CH || m >= g.M || n >= g.N) return;
  float v[8] = {sums[0][t] + sums[1][t] + sums[2][t] + sums[3][t]};
  finish8<T>(g.e, v, m, n, n + 1);
}

// ---- rows at any address ---------------------------------------------------------

struct PadArgs {
  HierPadRowsArgs a;
  int64_t first[2];            // chunks of eight elements of the first matrix, of both
  int32_t cpr;
};

__global__ __launch_bounds__(256) void pad_rows_kernel(PadArgs p) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.first[1]; i += (int64_t)gridDim.x * 256) {
    const int which = i >= p.first[0];
    const int64_t j = which ? i - p.first[0] : i;
    const int64_t row = j >> 32 ? j / p.cpr : (uint32_t)j / (uint32_t)p.cpr;
    const int n = 8 * (int)(j - row * p.cpr), C = p.a.C;
    const uint16_t* src = static_cast<const uint16_t*>(which ? p.a.src[1] : p.a.src[0]) +
                          row * (which ? p.a.ss[1] : p.a.ss[0]);
    u32x4 w;
    if (n + 8 <= C) {
      __builtin_memcpy(&w, src + n, 16);
    } else {
      uint16_t t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = src[min(n + e, C - 1)];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = n + 2 * e < C ? t[2 * e] : 0, hi = n + 2 * e + 1 < C ? t[2 * e + 1] : 0;
        w[e] = lo | hi << 16;
      }
    }
    reinterpret_cast<u32x4*>(which ? p.a.dst[1] : p.a.dst[0])[j] = w;
  }
}

// ---- dz, db and dg ---------------------------------------------------------------
//
// One pass over dy and z, eight channels a thread.  A workgroup row takes `rows`
// rows; where a gate's rows are more than that it takes `rows` rows of one gate
// at most (dg's sums then meet in sum_rows), else whole gates.
//
// Bound by memory and, with an activation, by the vector units beside it: 9,408 x 8,960
// (506 MB) with tanh GELU 115 us, 4.4 TB/s.  Tried before a NaN's test, one after the other
// without gaps, where it took 121: a row's loads alone 183, eight rows' 121, twice the
// workgroups 128.

struct DzArgs {
  const void* dy;
  const void* z;
  const void* gate;
  void* dz;
  void* dgate;
  float* db_part;
  float* dg_part;
  int64_t dy_ss, z_ss, gate_ss, dz_ss;
  int64_t M, rpg;              // rows of a gate (M without gates)
  int64_t rows, segs;          // rows of a workgroup; its rows of a gate's, if split
  int32_t N;
  bool split;
};

template <typename T, int ACT, bool VEC>
__global__ __launch_bounds__(256) void dz_kernel(DzArgs d) {
  const int n = 8 * (blockIdx.y * 256 + threadIdx.x);
  if (n >= d.N) return;
  const int64_t seg = blockIdx.x;
  int64_t r0, r1;
  if (d.split) {
    const int64_t gr = seg / d.segs, s = seg - gr * d.segs;
    r0 = gr * d.rpg + s * d.rows;
    r1 = min(r0 + d.rows, min((gr + 1) * d.rpg, d.M));
  } else {
    r0 = seg * d.rows;
    r1 = min(r0 + d.rows, d.M);
  }
  float db[8] = {}, dg[8] = {}, gate[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) gate[i] = 1.f;
  int64_t g = r0 / d.rpg, gend = (g + 1) * d.rpg;
  if (d.gate) row8<T>(d.gate, g * d.gate_ss, n, d.N, gate);
  // AHEAD rows' loads leave together (VEC: no branch is between them)
  constexpr int AHEAD = VEC ? 4 : 1;
  for (int64_t r = r0; r < r1; r += AHEAD) {
    w32x4 yw[AHEAD], zw[AHEAD];
    float y[8], z[8];
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) yw[j] = raw8<T>(d.dy, min(r + j, r1 - 1) * d.dy_ss + n);
      if (d.z)
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) zw[j] = raw8<T>(d.z, min(r + j, r1 - 1) * d.z_ss + n);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (r + j >= r1) break;
      if constexpr (VEC) {
        widen<T>(yw[j], y);
        if (d.z) widen<T>(zw[j], z);
      } else {
        row8<T>(d.dy, r * d.dy_ss, n, d.N, y);
        if (d.z) row8<T>(d.z, r * d.z_ss, n, d.N, z);
      }
      if (!d.z)
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = 0.f;
      if (r + j == gend) {          // the next gate's rows begin (whole gates only)
        if (d.dgate) put_row8<T>(d.dgate, g * (int64_t)d.N, n, d.N, dg);
        ++g;
        gend += d.rpg;
        row8<T>(d.gate, g * d.gate_ss, n, d.N, gate);
#pragma unroll
        for (int i = 0; i < 8; ++i) dg[i] = 0.f;
      }
      float dz[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float a, slope;
        activate2<ACT>(z[i], a, slope);
        dg[i] = fmaf(y[i], a, dg[i]);
        dz[i] = y[i] * gate[i] * slope;
      }
      if constexpr (ACT != HIER_ACT_NONE) keep_nans(z, dz);
#pragma unroll
      for (int i = 0; i < 8; ++i) db[i] += dz[i];
      if (d.dz) put8<T>(d.dz, (r + j) * d.dz_ss + n, dz);
    }
  }
  if (d.db_part) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < d.N) d.db_part[seg * d.N + n + i] = db[i];
  }
  if (d.dgate) {
    if (d.split) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < d.N) d.dg_part[seg * d.N + n + i] = dg[i];
    } else {
      put_row8<T>(d.dgate, g * (int64_t)d.N, n, d.N, dg);
    }
  }
}

// ---- plans -----------------------------------------------------------------------

// How a product is cut: tiles of 256 or 128, and K into `splits` parts.
struct Plan {
  int tile;
  int splits;
  int64_t kchunk;
  int64_t bytes;      // fp32 parts
  int64_t rows;       // by these tiles; the rest by tiles of 128 in a launch of their own
};

constexpr int kBK = 64;

Plan plan_of(int64_t M, int64_t N, int64_t K) {
  Plan best = {};
  double least = 1e30;
  const int64_t kt = (K + kBK - 1) / kBK;
  for (int tile : {256, 128}) {
    const int64_t tiles = ((M + tile - 1) / tile) * ((N + tile - 1) / tile);
    const int64_t slots = tile == 256 ? 256 : 512;
    for (int64_t splits = 1; splits <= 32 && splits <= kt; ++splits) {
      const int64_t per = (kt + splits - 1) / splits;
      if ((kt + per - 1) / per != splits) continue;
      // time in units of a 256-tile's 64 k: rounds of workgroups, each with a
      // start and an end worth four of them; parts written and read again
      const double rounds = (double)((tiles * splits + slots - 1) / slots);
      const double step = tile == 256 ? 1.0 : 0.6;
      double t = rounds * (per * step + 4);
      if (splits > 1) t += 4 + 1e-6 * (double)(splits * M * N) * 2.0;
      if (t < least) {
        least = t;
        best.tile = tile;
        best.splits = (int)splits;
        best.kchunk = per * kBK;
        best.bytes = splits > 1 ? splits * M * ((N + 7) / 8 * 8) * 4 : 0;
      }
    }
  }
  best.rows = M;
  if (best.tile == 256 && best.splits == 1) {
    // a last round of few tiles: the rows past the whole rounds in small tiles, where those
    // and a launch more take less than the round
    const int64_t tn = (N + 255) / 256, rounds = ((M + 255) / 256 * tn + kSlots - 1) / kSlots;
    const int64_t rows = (rounds - 1) * kSlots / tn * 256;
    if (rows > 0 && rows < M) {
      const int64_t small = ((M - rows + 127) / 128) * ((N + 127) / 128);
      if (kt + 8 > 5 + (double)((small + 2 * kSlots - 1) / (2 * kSlots)) * (0.6 * (double)kt + 4)) best.rows = rows;
    }
  }
  return best;
}

template <typename T, bool ATR, bool BTR>
int launch_gemm(GemmArgs g, const Plan& p, float* ws, bool rows16, hipStream_t st) {
  g.splits = p.splits;
  g.kchunk = p.kchunk;
  g.e.partial = ws;
  g.e.ld_part = (g.N + 7) / 8 * 8;
  g.e.part_stride = g.M * g.e.ld_part;
  // rows from g.m_first to `end` in tiles of `tile`
  auto rows = [&](int tile, int64_t end) {
    g.tm = (int)((end - g.m_first + tile - 1) / tile);
    g.tn = (int)((g.N + tile - 1) / tile);
    const int64_t total = (int64_t)g.tm * g.tn * g.splits;
    HIER_REQUIRE(total <= (1ll << 23), HIER_EUNSUPPORTED, "product: too many tiles");
    g.total = (int)total;
    auto run = [&](auto kind) {
      constexpr int KIND = decltype(kind)::value;
      if (tile == 256)
        hipLaunchKernelGGL((gemm_kernel<T, ATR, BTR, 256, 256, kBK, 1, KIND>),
                           dim3((unsigned)xcd_grid(std::min<int64_t>(total, kSlots))), dim3(256), 0, st, g);
      else
        hipLaunchKernelGGL((gemm_kernel<T, ATR, BTR, 128, 128, kBK, 2, KIND>),
                           dim3((unsigned)xcd_grid(std::min<int64_t>(total, 2 * kSlots))), dim3(256), 0, st, g);
    };
    // (the parts' launch writes whole rows of its own)
    if constexpr (ATR || BTR) {
      run(std::integral_constant<int, kPlain>{});
    } else {
      if (p.splits > 1 || (rows16 && !g.e.gate && !g.e.residual)) run(std::integral_constant<int, kPlain>{});
      else if (rows16) run(std::integral_constant<int, kExtra>{});
      else run(std::integral_constant<int, kAny>{});
    }
    return check_launch("gemm_kernel");
  };
  if (int rc = rows(p.tile, p.rows)) return rc;
  if (p.rows < g.M) {
    g.m_first = p.rows;
    g.kchunk = (g.K + kBK - 1) / kBK * kBK;
    if (int rc = rows(128, g.M)) return rc;
  }
  if (p.splits > 1) {
    const int64_t n8 = g.M * ((g.N + 7) / 8);
    hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)std::min<int64_t>((n8 + 255) / 256, 8192)),
                       dim3(256), 0, st, g);
    return check_launch("join_kernel");
  }
  return HIER_OK;
}

template <typename T>
int launch_few(const GemmArgs& g, hipStream_t st) {
  auto dots = [&](auto rows) {
    constexpr int M = decltype(rows)::value, CH = M < 2 ? 2 : M;
    hipLaunchKernelGGL((dot_kernel<T, M>), dim3((unsigned)((g.N + CH - 1) / CH)), dim3(256), 0, st, g);
    return check_launch("dot_kernel");
  };
  if (g.M == 1) return dots(std::integral_constant<int, 1>{});
  if (g.M == 2) return dots(std::integral_constant<int, 2>{});
  if (g.M <= 4) return dots(std::integral_constant<int, 4>{});
  if (g.M <= kDotRows) return dots(std::integral_constant<int, 8>{});
  const dim3 grid((unsigned)((g.N + 15) / 16)), block(64 * kFewWaves);
  if (g.M <= 16) hipLaunchKernelGGL((few_rows_kernel<T, 1>), grid, block, 0, st, g);
  else if (g.M <= 32) hipLaunchKernelGGL((few_rows_kernel<T, 2>), grid, block, 0, st, g);
  else hipLaunchKernelGGL((few_rows_kernel<T, 4>), grid, block, 0, st, g);
  return check_launch("few_rows_kernel");
}

// Whether dot_kernel or few_rows_kernel takes a product.  The second reads x again for
// every 16 channels and waits for memory a thousand of K at a time: past some 200
// million products, or a long K, the tiles win (64 rows of 1536 x 1536 10.1 us for 11.1; 17
// of 1536 x 8960 13.5 for 13.1, 32 of them 17.8 for 14.1; 9 of 8960 x 1536 18.6 for 15.6;
// 16 of 4096 x 16384 38 for 30.7).
bool few_rows(int64_t M, int64_t N, int64_t K) {
  return M <= kDotRows || (M <= 64 && K <= 4096 && M * N * K <= 200000000);
}

// Views that the copies address: 16-byte rows, a tile's rows (256) within 31
// bits of bytes.
int check_view(const char* who, const void* p, int64_t ld, int64_t cols) {
  HIER_REQUIRE(p != nullptr && aligned16(p), HIER_EINVAL, "linear: %s must be a 16-byte aligned pointer", who);
  HIER_REQUIRE(ld % 8 == 0 && (ld >= cols || ld == 0), HIER_EINVAL,
               "linear: %s needs a row stride of a multiple of 8, at least its columns", who);
  HIER_REQUIRE(ld < (1ll << 21), HIER_EUNSUPPORTED, "linear: %s: row stride of 2M elements or more", who);
  return HIER_OK;
}

int check_sizes(int64_t M, int64_t N, int64_t K, int type, int act) {
  HIER_REQUIRE(M >= 0 && N >= 1 && K >= 1, HIER_EINVAL, "linear: invalid M=%lld N=%lld K=%lld", (long long)M,
               (long long)N, (long long)K);
  HIER_REQUIRE(M < (1ll << 31) && N < (1 << 21) && K < (1 << 21), HIER_EUNSUPPORTED, "linear: too large");
  HIER_REQUIRE(type == HIER_BF16 || type == HIER_FP16, HIER_EUNSUPPORTED, "linear: bf16 or fp16");
  HIER_REQUIRE(act >= HIER_ACT_NONE && act <= HIER_ACT_SILU, HIER_EINVAL, "linear: unknown activation %d", act);
  return HIER_OK;
}

int check_gate(const void* gate, int64_t rows_per_gate) {
  HIER_REQUIRE(!gate || (rows_per_gate >= 1 && rows_per_gate < (1ll << 31)), HIER_EINVAL,
               "linear: invalid rows_per_gate=%lld", (long long)rows_per_gate);
  return HIER_OK;
}

// The rows of a workgroup of dz_kernel: 131,072 eight-channel chunks a row of workgroups,
// about nine waves a CU, and at most 128 rows.
struct DzPlan {
  int64_t rows, segs, total;
  bool split;
};
DzPlan dz_plan(int64_t M, int64_t N, int64_t rpg, bool gated) {
  const int64_t lanes = (N + 7) / 8;
  int64_t rows = std::max<int64_t>(4, std::min<int64_t>(128, M * lanes / 131072));
  DzPlan p;
  p.split = gated && rpg > rows;
  if (p.split) {
    p.segs = (rpg + rows - 1) / rows;
    p.rows = (rpg + p.segs - 1) / p.segs;
    p.total = (M / rpg) * p.segs;
  } else {
    if (gated) rows = rows / rpg * rpg;
    p.rows = rows;
    p.segs = 1;
    p.total = (M + rows - 1) / rows;
  }
  return p;
}

int64_t round16(int64_t b) { return (b + 255) / 256 * 256; }

struct BwdPlan {
  Plan dx, dw;
  DzPlan dz;
  int64_t off_dz, off_db, off_dg, off_part, bytes;
};
// dz is dy itself where there is neither an activation nor a gate, and dy has the
// products' rows.
bool dz_is_dy(const HierLinearBwdArgs& a) {
  return a.act == HIER_ACT_NONE && !a.gate && a.N % 8 == 0 && aligned16(a.dy) && a.dy_ss % 8 == 0 && a.dy_ss >= a.N &&
         a.dy_ss < (1 << 21);
}

BwdPlan bwd_plan(const HierLinearBwdArgs& a) {
  BwdPlan p = {};
  const int64_t Np = (a.N + 7) / 8 * 8;
  p.dz = dz_plan(a.M, a.N, a.gate ? a.rows_per_gate : std::max<int64_t>(a.M, 1), a.gate != nullptr);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += round16(bytes);
    return o;
  };
  p.off_dz = dz_is_dy(a) ? 0 : take(a.M * Np * 2);
  p.off_db = a.db ? take(p.dz.total * a.N * 4) : 0;
  p.off_dg = a.dgate && p.dz.split ? take(p.dz.total * a.N * 4) : 0;
  int64_t parts = 0;
  if (a.dx) {
    p.dx = plan_of(a.M, a.K, a.N);
    parts = std::max(parts, p.dx.bytes);
  }
  if (a.dw) {
    p.dw = plan_of(a.N, a.K, a.M);
    parts = std::max(parts, p.dw.bytes);
  }
  p.off_part = take(parts);
  p.bytes = at;
  return p;
}

}  // namespace
}  // namespace hier

using namespace hier;

static int check_linear(const HierLinearArgs& a) {
  if (int rc = check_sizes(a.M, a.N, a.K, a.type, a.act)) return rc;
  HIER_REQUIRE(a.K % 8 == 0, HIER_EINVAL, "linear: K must be a multiple of 8, got %d", a.K);
  return check_gate(a.gate, a.rows_per_gate);
}

extern "C" int64_t hier_linear_workspace(const HierLinearArgs* a) {
  clear_error();
  if (!a || check_linear(*a)) return -1;
  return a->M == 0 || few_rows(a->M, a->N, a->K) ? 0 : plan_of(a->M, a->N, a->K).bytes;
}

extern "C" int hier_linear(const HierLinearArgs* args, void* stream) {
  clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  const HierLinearArgs& a = *args;
  if (int rc = check_linear(a)) return rc;
  if (a.M == 0) return HIER_OK;
  if (int rc = check_view("x", a.x, a.x_ss, a.K)) return rc;
  if (int rc = check_view("weight", a.w, a.w_ss, a.K)) return rc;
  HIER_REQUIRE(a.out != nullptr, HIER_EINVAL, "linear: NULL output");
  HIER_REQUIRE(a.out_ss >= a.N && (!a.preact || a.preact_ss >= a.N) && (!a.residual || a.residual_ss >= 0) &&
                   (!a.gate || a.gate_ss >= 0),
               HIER_EINVAL, "linear: invalid row stride");
  GemmArgs g = {};
  g.a = a.x;
  g.b = a.w;
  g.lda = a.x_ss;
  g.ldb = a.w_ss;
  g.M = a.M;
  g.N = a.N;
  g.K = a.K;
  Epilogue& e = g.e;
  e.bias = a.bias;
  e.residual = a.residual;
  e.gate = a.gate;
  e.out = a.out;
  e.preact = a.preact;
  e.residual_ss = a.residual_ss;
  e.gate_ss = a.gate_ss;
  e.out_ss = a.out_ss;
  e.preact_ss = a.preact_ss;
  e.rows_per_gate = make_div(a.gate ? (uint32_t)a.rows_per_gate : 1u);
  e.act = a.act;
  const hipStream_t st = (hipStream_t)stream;
  if (few_rows(a.M, a.N, a.K)) return a.type == HIER_BF16 ? launch_few<__bf16>(g, st) : launch_few<_Float16>(g, st);
  const Plan p = plan_of(a.M, a.N, a.K);
  HIER_REQUIRE(p.bytes == 0 || (a.workspace && aligned16(a.workspace) && a.workspace_bytes >= p.bytes),
               HIER_EINVAL, "linear: workspace of %lld bytes needed", (long long)p.bytes);
  float* ws = static_cast<float*>(a.workspace);
  auto ok = [](const void* q, int64_t ss) { return !q || (aligned16(q) && ss % 8 == 0 && ss < (1ll << 21)); };
  const bool rows16 = a.N % 8 == 0 && ok(a.bias, 0) && ok(a.residual, a.residual_ss) && ok(a.gate, a.gate_ss) &&
                      ok(a.out, a.out_ss) && ok(a.preact, a.preact_ss);
  return a.type == HIER_BF16 ? launch_gemm<__bf16, false, false>(g, p, ws, rows16, st)
                             : launch_gemm<_Float16, false, false>(g, p, ws, rows16, st);
}

extern "C" int hier_pad_rows(const HierPadRowsArgs* args, void* stream) {
  clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  PadArgs p = {};
  p.a = *args;
  const HierPadRowsArgs& a = p.a;
  HIER_REQUIRE(a.C >= 1 && a.C < (1 << 21) && a.rows[0] >= 0 && a.rows[1] >= 0 && a.rows[0] < (1ll << 31) &&
                   a.rows[1] < (1ll << 31),
               HIER_EINVAL, "pad_rows: invalid sizes");
  for (int i = 0; i < 2; ++i)
    HIER_REQUIRE(a.rows[i] == 0 || (a.src[i] && a.dst[i] && aligned16(a.dst[i]) && (uintptr_t)a.src[i] % 2 == 0 &&
                                    a.ss[i] >= 0),
                 HIER_EINVAL, "pad_rows: needs rows, 16-byte aligned results and strides of at least 0");
  p.cpr = (a.C + 7) / 8;
  p.first[0] = a.rows[0] * p.cpr;
  p.first[1] = p.first[0] + a.rows[1] * p.cpr;
  if (p.first[1] == 0) return HIER_OK;
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)std::min<int64_t>((p.first[1] + 255) / 256, 1 << 16)), dim3(256), 0,
                     (hipStream_t)stream, p);
  return check_launch("pad_rows_kernel");
}

static int check_linear_bwd(const HierLinearBwdArgs& a) {
  if (int rc = check_sizes(a.M, a.N, a.K, a.type, a.act)) return rc;
  HIER_REQUIRE(a.M >= 1, HIER_EINVAL, "linear_bwd: no rows");
  HIER_REQUIRE(a.K % 8 == 0, HIER_EINVAL, "linear_bwd: K must be a multiple of 8, got %d", a.K);
  HIER_REQUIRE(!a.dgate || a.gate, HIER_EINVAL, "linear_bwd: dgate without a gate");
  HIER_REQUIRE(!a.gate || (a.rows_per_gate >= 1 && a.M % a.rows_per_gate == 0), HIER_EINVAL,
               "linear_bwd: %lld rows are not a multiple of rows_per_gate=%lld", (long long)a.M,
               (long long)a.rows_per_gate);
  return HIER_OK;
}

extern "C" int64_t hier_linear_bwd_workspace(const HierLinearBwdArgs* a) {
  clear_error();
  if (!a || check_linear_bwd(*a)) return -1;
  return bwd_plan(*a).bytes;
}

template <typename T>
static int linear_bwd(const HierLinearBwdArgs& a, const BwdPlan& p, hipStream_t st) {
  char* ws = static_cast<char*>(a.workspace);
  const int64_t Np = (a.N + 7) / 8 * 8;
  const bool plain = dz_is_dy(a), products = a.dx || a.dw;
  const void* dz = plain ? a.dy : ws + p.off_dz;
  const int64_t dz_ss = plain ? a.dy_ss : Np;
  if ((!plain && products) || a.db || a.dgate) {
    DzArgs d = {};
    d.dy = a.dy;
    d.z = a.preact;
    d.gate = a.gate;
    d.dz = plain || !products ? nullptr : ws + p.off_dz;
    d.dgate = a.dgate;
    d.db_part = a.db ? reinterpret_cast<float*>(ws + p.off_db) : nullptr;
    d.dg_part = reinterpret_cast<float*>(ws + p.off_dg);
    d.dy_ss = a.dy_ss;
    d.z_ss = a.preact_ss;
    d.gate_ss = a.gate_ss;
    d.dz_ss = Np;
    d.M = a.M;
    d.rpg = a.gate ? a.rows_per_gate : a.M;
    d.rows = p.dz.rows;
    d.segs = p.dz.segs;
    d.N = a.N;
    d.split = p.dz.split;
    const int64_t gy = (Np / 8 + 255) / 256;
    HIER_REQUIRE(gy <= 65535 && p.dz.total < (1ll << 24), HIER_EUNSUPPORTED, "linear_bwd: too many rows");
    const dim3 grid((unsigned)p.dz.total, (unsigned)gy);
    auto run = [&](auto kind) {
      constexpr int ACT = decltype(kind)::value;
      if (a.N % 8 == 0) hipLaunchKernelGGL((dz_kernel<T, ACT, true>), grid, dim3(256), 0, st, d);
      else hipLaunchKernelGGL((dz_kernel<T, ACT, false>), grid, dim3(256), 0, st, d);
    };
    switch (a.act) {
      case HIER_ACT_GELU_TANH: run(std::integral_constant<int, HIER_ACT_GELU_TANH>{}); break;
      case HIER_ACT_GELU: run(std::integral_constant<int, HIER_ACT_GELU>{}); break;
      case HIER_ACT_SILU: run(std::integral_constant<int, HIER_ACT_SILU>{}); break;
      default: run(std::integral_constant<int, HIER_ACT_NONE>{});
    }
    if (int rc = check_launch("dz_kernel")) return rc;
    if (a.db)
      if (int rc = sum_rows(d.db_part, p.dz.total, 1, a.N, a.db, a.type, st)) return rc;
    if (a.dgate && p.dz.split)
      if (int rc = sum_rows(d.dg_part, p.dz.segs, a.M / a.rows_per_gate, a.N, a.dgate, a.type, st)) return rc;
  }
  float* parts = reinterpret_cast<float*>(ws + p.off_part);
  auto product = [&](int64_t M, int64_t N, int64_t K, const void* A, int64_t lda, const void* B, int64_t ldb,
                     void* out, int64_t out_ss) {
    GemmArgs g = {};
    g.a = A;
    g.b = B;
    g.lda = lda;
    g.ldb = ldb;
    g.M = M;
    g.N = N;
    g.K = K;
    g.e.out = out;
    g.e.out_ss = out_ss;
    g.e.rows_per_gate = make_div(1u);
    return g;
  };
  if (a.dx)
    if (int rc = launch_gemm<T, false, true>(
            product(a.M, a.K, a.N, dz, dz_ss, a.w, a.N == 1 ? a.K : a.w_ss, a.dx, a.dx_ss), p.dx, parts, true, st))
      return rc;
  if (a.dw)
    return launch_gemm<T, true, true>(
        product(a.N, a.K, a.M, dz, dz_ss, a.x, a.M == 1 ? a.K : a.x_ss, a.dw, a.dw_ss), p.dw, parts, true, st);
  return HIER_OK;
}

extern "C" int hier_linear_bwd(const HierLinearBwdArgs* args, void* stream) {
  clear_error();
  HIER_REQUIRE(args != nullptr, HIER_EINVAL, "args is NULL");
  const HierLinearBwdArgs& a = *args;
  if (int rc = check_linear_bwd(a)) return rc;
  HIER_REQUIRE(a.dy != nullptr && a.dy_ss >= 0, HIER_EINVAL, "linear_bwd: invalid dy");
  HIER_REQUIRE(a.preact || (a.act == HIER_ACT_NONE && !a.dgate), HIER_EINVAL,
               "linear_bwd: needs the values before the activation");
  HIER_REQUIRE(!a.preact || a.preact_ss >= a.N, HIER_EINVAL, "linear_bwd: invalid row stride");
  if (a.dx)
    if (int rc = check_view("weight", a.w, a.w_ss, a.K)) return rc;
  if (a.dw)
    if (int rc = check_view("x", a.x, a.x_ss, a.K)) return rc;
  // (a row read as several would be read past the last one too, and be inf * 0 there)
  HIER_REQUIRE((!a.dx || a.w_ss > 0 || a.N == 1) && (!a.dw || a.x_ss > 0 || a.M == 1), HIER_EINVAL,
               "linear_bwd: rows of x and weight must not overlap");
  auto ok = [](const void* q, int64_t ss) { return !q || (aligned16(q) && ss % 8 == 0 && ss < (1ll << 21)); };
  HIER_REQUIRE((!a.dx || a.dx_ss >= a.K) && (!a.dw || a.dw_ss >= a.K) && ok(a.dx, a.dx_ss) && ok(a.dw, a.dw_ss),
               HIER_EINVAL, "linear_bwd: dx and dw need 16-byte rows and an output stride of at least K");
  const BwdPlan p = bwd_plan(a);
  HIER_REQUIRE(p.bytes == 0 || (a.workspace && aligned16(a.workspace) && a.workspace_bytes >= p.bytes),
               HIER_EINVAL, "linear_bwd: workspace of %lld bytes needed", (long long)p.bytes);
  return a.type == HIER_BF16 ? linear_bwd<__bf16>(a, p, (hipStream_t)stream)
                             : linear_bwd<_Float16>(a, p, (hipStream_t)stream);
}
