// Matrix products of the dense gated FFN, C[m][n] = sum_k A(m, k) B(n, k), on
// the gfx950 matrix cores, with the FFN's elementwise parts in the epilogue.
//
// One kernel template covers every product of the forward and backward pass.
// An operand is either K-contiguous (rows of m or n, "KC") or K-strided (rows
// of k, "KS"), so that no operand is transposed in memory:
//
//   gate, up    A = x      KC  B = Wg, Wu    KC  -> a = silu(g) u (and g, u)
//   down        A = a      KC  B = Wd        KC  -> y
//   d(act)      A = dy     KC  B = Wd        KS  -> dg, du from g, u
//   dx          A = dg, du KC  B = Wg, Wu    KS  -> dx (K runs over both)
//   dWg, dWu    A = dg, du KS  B = x         KS  (two problems of one launch)
//   dWd         A = dy     KS  B = a         KS
//   int8        A = codes  KC  B = codes     KC  -> y, or a with its row maxima
//
// Tiles.  A K step is 128 bytes of K: 64 16-bit elements, 128 int8, 32 fp32.
// Both operand tiles of a step are copied from memory straight into LDS
// (buffer_load ... lds, 16 bytes a lane), into one of two buffers while the
// other is multiplied.  The copy's buffer descriptor ends at the operand's
// last element, so rows past the end arrive as zeros without a branch; K
// tails and column tails give their lanes an offset behind the descriptor.
//
// A wave owns MT x 4 G tiles of 16 x 16.  B is the MFMA's first operand, so a
// lane's four accumulators are four consecutive n of one m.  For KC B the
// LDS rows of a wave's 64 n are dealt to the MFMA rows so that a lane's 4
// tiles together hold 16 consecutive n (gated: 8 of gate and the same 8 of
// up): stores are whole 16-byte vectors.
//
// LDS positions are swizzled in 16-byte chunks (KC), 32-byte (KS, 16-bit) or
// 64-byte ones (KS, fp32), chosen so that the lanes one LDS pass serves hit
// different banks; the copy applies the swizzle by choosing its source
// address, since its LDS side is linear.  16-bit KS tiles are read with the
// transposing LDS read (4 rows of k x 16 columns per 16 lanes).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "wr_device.h"
#include "wr_ffn_internal.h"

namespace wr {
namespace ffn {

typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kStepBytes = 128;  // bytes of K per step
constexpr unsigned kOutside = 0x80000000u;  // offset behind every descriptor

// ---- 16 x 16 tile products over 64 bytes of K --------------------------------
// The 16-bit and int8 instructions are written as assembly with the sums tied to
// accumulation registers: the compiler's own register allocation moves the sums of
// a 128 x 128 wave tile (all 256 accumulation registers) between registers in the
// loop.  The waits its hazard pass would add are held by construction: fragments
// come from LDS reads alone (no vector instruction writes them), equal sums are at
// least NT products apart, and settle() stands between the sums' first and last
// use and any other instruction on them.
template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
  typedef f32x4 Acc;
  static __device__ __forceinline__ void go(u32x4 a, u32x4 b, Acc& c) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
};
template <>
struct Mma<f16> {
  typedef f32x4 Acc;
  static __device__ __forceinline__ void go(u32x4 a, u32x4 b, Acc& c) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
};
template <>
struct Mma<int8_t> {
  typedef i32x4 Acc;
  static __device__ __forceinline__ void go(u32x4 a, u32x4 b, Acc& c) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
};
// fp32: lane group q holds k = 4 q .. 4 q + 3, one element per MFMA.
template <>
struct Mma<float> {
  typedef f32x4 Acc;
  static __device__ __forceinline__ void go(u32x4 a, u32x4 b, Acc& c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
  }
};

// Orders all accumulators' values between the assembly products and other instructions,
// with the wait states of the longest product (18) in between.
template <typename Acc, int N>
__device__ __forceinline__ void settle(Acc (&acc)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+a"(acc[i]));
  asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+a"(acc[i]));
}

// ---- copying one operand's K step into LDS ---------------------------------
// Swizzle keys: KC tiles are [row][128 bytes], KS tiles [k][ROWS elements].
template <bool NSIDE>
__device__ __forceinline__ int kc_key(int row) {  // xor of the 16-byte chunk index
  // M side: 16 lanes read 16 consecutive rows.  N side: rows 16 q + 4 t + i, q, i < 4.
  return NSIDE ? (((row >> 1) & 1) | (((row >> 4) & 3) << 1)) : ((row >> 1) & 7);
}
template <int ES, int ROWS>
__device__ __forceinline__ int ks_key(int k) {  // xor of the 32- (64-) byte chunk index
  if (ES == 4) return (k >> 2) & 3;
  return ROWS >= 128 ? ((k & 3) | (((k >> 3) & 1) << 2)) : (((k >> 1) & 1) | (((k >> 3) & 1) << 1));
}

// Lane-to-source mapping of a tile of ROWS m or n (times one K step), copied by
// NW waves, PER copies of 1 KB each per wave.
template <typename T, int ROWS, int NW, bool KS, bool NSIDE, bool GATED>
struct TileCopy {
  static constexpr int ES = sizeof(T);
  static constexpr int kCopies = ROWS * kStepBytes / 1024;
  static constexpr int PER = kCopies / NW;
  static_assert(kCopies % NW == 0, "every wave copies whole kilobytes");
  static constexpr int EPC = 16 / ES;  // elements per chunk
  unsigned voff[PER];

  // Chunk of this lane in copy j, as a k offset (KC).
  static __device__ __forceinline__ int k_chunk(int j, int wave, int lane) {
    const int row = (j * NW + wave) * 8 + (lane >> 3);
    return (lane & 7) ^ kc_key<NSIDE>(row);
  }

  // cols: KS only, m (n) elements left from the tile's first one.
  __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int cols) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (KS) {
        constexpr int CPR = ROWS * ES / 16;  // chunks per k row
        const int L = (j * NW + wave) * 64 + lane;
        const int k = L / CPR, p = L % CPR;
        constexpr int G = ES == 4 ? 4 : 2;  // chunks per swizzle unit
        const int c = ((p / G) ^ ks_key<ES, ROWS>(k)) * G + p % G;
        voff[j] = c * EPC < cols ? (unsigned)(k * ld + c * 16) : kOutside;
      } else {
        int row = (j * NW + wave) * 8 + (lane >> 3);
        if (GATED) row = (row >> 4) * 8 + (row & 7);  // rows 8..15 of 16 are the other matrix's
        voff[j] = (unsigned)(row * ld + k_chunk(j, wave, lane) * 16);
      }
    }
  }

  // base: the tile's first byte at this K step; end: the operand's bytes from there
  // on (<= 0: the step does not exist, zeros arrive).
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t source(const char* base, int64_t end) {
    const int records = end > 0x7fffffff ? 0x7fffffff : end < 0 ? 0 : (int)end;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, records, 0x00020000);
  }
  // Copy j; krem: K elements left at this step.
  __device__ __forceinline__ void issue(int j, char* lds, __amdgpu_buffer_rsrc_t r, int krem,
                                        int wave, int lane) const {
    unsigned v = voff[j];
    if (!KS) v = k_chunk(j, wave, lane) * EPC < krem ? v : kOutside;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        r, (__attribute__((address_space(3))) void*)(lds + (j * NW + wave) * 1024), 16, (int)v, 0,
        0, 0);
  }
};

// ---- reading a wave's fragments from LDS -----------------------------------
__device__ __forceinline__ u32x4 lds_b128(const char* p) {
  return *(const __attribute__((address_space(3))) u32x4*)p;
}

// The transposing read: 16 lanes read 4 rows of 16 16-bit elements, 8 bytes each, and lane
// i gets column i.  The restrict marks the access for the alias analysis, without
// which the compiler waits for every copy in flight before each of these reads.
__device__ __forceinline__ u32x2 lds_tr_b64(
    __attribute__((address_space(3))) s16x4* __restrict__ p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
}

// S subtiles of 16 m (n) from subtile sub0 of a tile of ROWS.
template <typename T, int ROWS, int S, bool KS, bool NSIDE>
struct Frag {
  static constexpr int ES = sizeof(T);
  static constexpr int RB = ROWS * ES;  // bytes per k row (KS)
  int addr[KS ? S : 2];

  __device__ __forceinline__ void init(int sub0, int lane) {
    const int r = lane & 15, q = lane >> 4;
    if constexpr (!KS) {
      // M side: row 16 s + r.  N side, per 4 subtiles: subtile t's row r = 4 q' + i is
      // LDS row 16 q' + 4 t + i.
      const int row = sub0 * 16 + (NSIDE ? (r >> 2) * 16 + (r & 3) : r);
      const int key = kc_key<NSIDE>(row);
      addr[0] = row * kStepBytes + (q ^ key) * 16;
      addr[1] = row * kStepBytes + ((4 + q) ^ key) * 16;
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (ES == 2) {
          const int k = 8 * q + (r >> 2);
          addr[s] = k * RB + ((sub0 + s) ^ ks_key<ES, ROWS>(k)) * 32 + (r & 3) * 8;
        } else {
          const int k = 4 * q;
          addr[s] = k * RB + ((sub0 + s) ^ ks_key<ES, ROWS>(k)) * 64 + r * 4;
        }
      }
    }
  }

  // Fragment of subtile s, 64-byte half kk of the K step.
  __device__ __forceinline__ u32x4 get(char* tile, int s, int kk) const {
    if constexpr (!KS) {
      const int row = NSIDE ? (s >> 2) * 64 + (s & 3) * 4 : s * 16;
      return lds_b128(tile + addr[kk] + row * kStepBytes);
    } else if constexpr (ES == 2) {
      typedef __attribute__((address_space(3))) s16x4* P;
      char* a = tile + addr[s] + kk * 32 * RB;
      const u32x2 lo = lds_tr_b64((P)a), hi = lds_tr_b64((P)(a + 4 * RB));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      const char* a = tile + addr[s] + kk * 16 * RB;
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = *(const __attribute__((address_space(3))) uint32_t*)(a + j * RB);
      return v;
    }
  }
};

// ---- epilogues --------------------------------------------------------------
template <typename T>
__device__ __forceinline__ T to_out(float v) {
  return (T)v;
}

__device__ __forceinline__ float sigmoid(float g) { return 1.0f / (1.0f + expf(-g)); }
// g * sigmoid(g)
__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

// N consecutive elements at p[0..N), of which the first `left` exist.  VEC: p is
// aligned to its N elements.
template <typename T, int N>
__device__ __forceinline__ void store_run(T* p, const float* v, int left, bool vec) {
  if (vec && left >= N) {
    typedef T V __attribute__((ext_vector_type(N)));
    V o;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = to_out<T>(v[i]);
    *(V*)p = o;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = to_out<T>(v[i]);
  }
}

// The derivative of a = silu(g) u: du = da silu(g), dg = da u s (1 + g (1 - s)).
__device__ __forceinline__ void gate_grad(float da, float g, float u, float& dg, float& du) {
  const float s = sigmoid(g);
  du = da * silu(g);
  dg = da * u * (s + silu(g) * (1.0f - s));
}

// Rows of the padded intermediate buffers are ldi elements apart; one row's
// valid part is N elements.
template <typename T, int EPI, bool BS>
struct Epilogue {
  typedef typename Mma<T>::Acc Acc;

  // acc[mt][t]: 16 m, and 64 n (gated: 32 of gate, 32 of up) in 4 subtiles.
  template <int MT>
  static __device__ __forceinline__ void run(const GemmArgs& g, Acc (&acc)[MT][4], int prob,
                                             int slice, int m0, int n0, int lane) {
    const int r = lane & 15, q = lane >> 4;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int m = m0 + mt * 16 + r;
      if (EPI == kGatedMax) {
        gated_max(g, acc[mt], m, n0, q);
        continue;
      }
      if (m >= g.M) continue;
      if constexpr (EPI == kGated) {
        gated(g, acc[mt], m, n0 + q * 8);
      } else if constexpr (EPI == kPartGated) {
        const int64_t at = ((int64_t)slice * g.M + m) * 2 * g.ldp;
        const int n = n0 + q * 8;
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (n + (t & 1) * 4 < g.N)
            *(Acc*)(reinterpret_cast<char*>(g.part) +
                    (at + (t >> 1) * g.ldp + n + (t & 1) * 4) * 4) = acc[mt][t];
      } else if constexpr (EPI == kStore && !BS) {
        float v[16];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[t * 4 + i] = acc[mt][t][i];
        const int n = n0 + q * 16;
        T* p = (T*)g.out[prob] + (int64_t)m * g.ldo + n;
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 16; i += V) store_run<T, V>(p + i, v + i, g.N - n - i, g.vec);
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int n = n0 + (BS ? t * 16 + q * 4 : q * 16 + t * 4);
          // dg and du rows are read in whole 16-byte chunks: their zeros past N too.
          if (n < (EPI == kGateGrad ? (g.N + 7) & ~7 : g.N)) tile(g, acc[mt][t], prob, slice, m, n);
        }
      }
    }
  }

  // Four consecutive n of one m.
  static __device__ __forceinline__ void tile(const GemmArgs& g, Acc a, int prob, int slice, int m,
                                              int n) {
    if constexpr (EPI == kPart) {
      const int64_t at = (((int64_t)slice * g.nprob + prob) * g.M + m) * g.ldp + n;
      *(Acc*)(reinterpret_cast<char*>(g.part) + at * 4) = a;  // ldp covers the tail
    } else if constexpr (EPI == kStore) {
      const float v[4] = {a[0], a[1], a[2], a[3]};
      store_run<T, 4>((T*)g.out[prob] + (int64_t)m * g.ldo + n, v, g.N - n, g.vec);
    } else if constexpr (EPI == kGateGrad) {
      const int64_t at = (int64_t)m * g.ldi + n;
      const f32x4 gg = *(const f32x4*)((const float*)g.in[0] + at);
      const f32x4 uu = *(const f32x4*)((const float*)g.in[1] + at);
      float dg[4], du[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) gate_grad(a[i], gg[i], uu[i], dg[i], du[i]);
      store_run<T, 4>((T*)g.out[0] + at, dg, 4, true);
      store_run<T, 4>((T*)g.out[1] + at, du, 4, true);
    } else if constexpr (EPI == kScale) {
      const float sm = g.row_scale[m];
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = n + i < g.N ? (float)a[i] * sm * g.col_scale[0][n + i] : 0.0f;
      const int64_t at = (int64_t)m * g.ldo + n;
      if (g.out_dtype == WR_F32)
        store_run<float, 4>((float*)g.out[0] + at, v, g.N - n, g.vec);
      else if (g.out_dtype == WR_F16)
        store_run<f16, 4>((f16*)g.out[0] + at, v, g.N - n, g.vec);
      else
        store_run<bf16, 4>((bf16*)g.out[0] + at, v, g.N - n, g.vec);
    }
  }

  // 8 gate and 8 up sums of the same n (acc[0..1] and acc[2..3]).  The buffers'
  // rows are padded to ldi (a multiple of 64), so whole vectors are stored.
  static __device__ __forceinline__ void gated(const GemmArgs& g, const Acc (&acc)[4], int m,
                                               int n) {
    if (n >= g.N) return;
    float a[8], gg[8], uu[8];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        gg[t * 4 + i] = acc[t][i];
        uu[t * 4 + i] = acc[t + 2][i];
        a[t * 4 + i] = silu(acc[t][i]) * acc[t + 2][i];
      }
    const int64_t at = (int64_t)m * g.ldi + n;
    constexpr int V = 16 / sizeof(T) < 8 ? 16 / sizeof(T) : 8;
#pragma unroll
    for (int i = 0; i < 8; i += V) store_run<T, V>((T*)g.out[0] + at + i, a + i, V, true);
    if (g.out[1] != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        store_run<float, 4>((float*)g.out[1] + at + i, gg + i, 4, true);
        store_run<float, 4>((float*)g.out[2] + at + i, uu + i, 4, true);
      }
    }
  }

  // int8: a = silu(g) u in fp32 with its row maxima of |a| (as fp32 bits: the
  // maximum of non-negative floats is that of their bits, in any order).
  static __device__ __forceinline__ void gated_max(const GemmArgs& g, const Acc (&acc)[4], int m,
                                                   int n0, int q) {
    const int n = n0 + q * 8;
    unsigned mx = 0;
    if (m < g.M && n < g.N) {
      const float sm = g.row_scale[m];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = n + t * 4 + i;
          v[i] = 0.0f;
          if (c < g.N) {
            const float gg = (float)acc[t][i] * sm * g.col_scale[0][c];
            v[i] = silu(gg) * ((float)acc[t + 2][i] * sm * g.col_scale[1][c]);
          }
          mx = max(mx, __float_as_uint(v[i]) & 0x7fffffffu);
        }
        store_run<float, 4>((float*)g.out[0] + (int64_t)m * g.ldi + n + t * 4, v, 4, true);
      }
    }
    mx = max(mx, (unsigned)__shfl_xor((int)mx, 16));
    mx = max(mx, (unsigned)__shfl_xor((int)mx, 32));
    if (q == 0 && m < g.M) atomicMax(g.row_max + m, mx);
  }
};

// Waits until all but the wave's N newest copies have landed and its LDS reads are
// done, then for the block's other waves.
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Bytes of a row up to the end of its last 16-byte chunk (rows are padded to whole chunks).
__device__ __forceinline__ int64_t chunked(int64_t bytes) { return (bytes + 15) & ~(int64_t)15; }

// ---- the kernel -------------------------------------------------------------
// A block of WM x WN waves, each with MT x 4 G subtiles of 16 x 16.  Both halves' (64
// bytes of K) fragments are held in registers: while one half is multiplied, the
// other's are read.  The K step's only barrier lies between its halves: behind it the
// next step's tiles are in LDS (their copies were issued one step earlier) and
// nobody reads the present ones any more, which the copies of the step after next
// then replace.  Each half is written as MT groups of NT products, with the LDS
// reads and copies dealt to the groups and the groups kept in order, so that
// the matrix cores, the LDS and the copies run side by side in one wave.
//
// 128 x 128 wave tiles (256 x 256, 4 waves) read 128 KB of fragments per K step
// beside 64 KB of copies: at the LDS's 128 bytes a clock three quarters of the
// products' 2048 clocks.  8 waves of 128 x 64 read 192 KB, which takes all of them.
template <typename T, int WM, int WN, int MT, int G, bool AS, bool BS, int EPI>
__global__ __launch_bounds__(WM * WN * 64) void k_dense(GemmArgs g) {
  constexpr bool GATED = EPI == kGated || EPI == kGatedMax || EPI == kPartGated;
  constexpr int NT = 4 * G;
  constexpr int NW = WM * WN, BM = WM * MT * 16, BN = WN * NT * 16;
  constexpr int ABYTES = BM * kStepBytes, BBYTES = BN * kStepBytes, BUF = ABYTES + BBYTES;
  constexpr int ES = sizeof(T), KB = kStepBytes / ES;
  typedef typename Mma<T>::Acc Acc;
  __shared__ __attribute__((aligned(1024))) char smem[2 * BUF];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // Block -> (slice, problem, tile).  Consecutive blocks go to the 8 XCDs in
  // turn, so each XCD takes one run of the tile order; within it 8 m tiles
  // advance together along n, for both operands' reuse in the XCD's L2.
  const TileId id = tile_of(g, (int)blockIdx.x, (int)gridDim.x);
  const int m0 = id.m * BM, n0 = id.n * (GATED ? BN / 2 : BN);
  const int steps = (g.K + KB - 1) / KB, total = steps * g.nseg;
  const int per = (total + g.slices - 1) / g.slices;
  const int s0 = id.slice * per, s1 = min(total, s0 + per);

  typedef TileCopy<T, BM, NW, AS, false, false> CopyA;
  typedef TileCopy<T, BN, NW, BS, true, GATED> CopyB;
  CopyA ca;
  CopyB cb;
  ca.init(wave, lane, g.lda, AS ? g.M - m0 : 0);
  cb.init(wave, lane, g.ldb, BS ? g.N - n0 : 0);
  Frag<T, BM, MT, AS, false> fa;
  Frag<T, BN, NT, BS, true> fb;
  fa.init(wm * MT, lane);
  fb.init(wn * NT, lane);

  const char* const pa0 = g.a[id.prob];
  const char* const pa1 = g.a[1];
  const char* const pb0 = g.b[GATED ? (wave & 1) : 0];
  const char* const pb1 = g.b[1];
  // Where a step's tiles come from.
  struct Source {
    __amdgpu_buffer_rsrc_t a, b;
    int krem;
  };
  auto source = [&](int step) {
    const int seg = step >= steps ? 1 : 0;
    const int k = (step - seg * steps) * KB;
    const bool live = step < s1;
    const char* pa = seg ? pa1 : pa0;
    const int64_t offa = AS ? k * g.lda + (int64_t)m0 * ES : m0 * g.lda + (int64_t)k * ES;
    const int64_t alla = AS ? (g.K - 1) * g.lda + chunked((int64_t)g.M * ES)
                            : (g.M - 1) * g.lda + chunked((int64_t)g.K * ES);
    const char* pb = seg ? pb1 : pb0;
    const int64_t offb = BS ? k * g.ldb + (int64_t)n0 * ES : n0 * g.ldb + (int64_t)k * ES;
    const int64_t allb = BS ? (g.K - 1) * g.ldb + chunked((int64_t)g.N * ES)
                            : (g.N - 1) * g.ldb + chunked((int64_t)g.K * ES);
    return Source{CopyA::source(pa + offa, live ? alla - offa : 0),
                  CopyB::source(pb + offb, live ? allb - offb : 0), g.K - k};
  };
  // Copies lo .. hi - 1 of a step's CopyA::PER + CopyB::PER.
  auto copy = [&](const Source& s, char* lds, int lo, int hi) {
#pragma unroll
    for (int j = 0; j < CopyA::PER + CopyB::PER; ++j) {
      if (j < lo || j >= hi) continue;
      if (j < CopyA::PER)
        ca.issue(j, lds, s.a, s.krem, wave, lane);
      else
        cb.issue(j - CopyA::PER, lds + ABYTES, s.b, s.krem, wave, lane);
    }
  };
  constexpr int COPIES = CopyA::PER + CopyB::PER;

  Acc acc[G * MT * 4];  // [group of 4 n subtiles][m subtile][n subtile]
#pragma unroll
  for (int i = 0; i < G * MT * 4; ++i) acc[i] = Acc{};

  u32x4 a0[MT], b0[NT], a1[MT], b1[NT];
  // Fragments lo .. hi - 1, those of B first: every product needs them.
  auto read = [&](u32x4(&a)[MT], u32x4(&b)[NT], char* tile, int kk, int lo, int hi) {
#pragma unroll
    for (int j = 0; j < MT + NT; ++j) {
      if (j < lo || j >= hi) continue;
      if (j < NT)
        b[j] = fb.get(tile + ABYTES, j, kk);
      else
        a[j - NT] = fa.get(tile, j - NT, kk);
    }
  };
  auto multiply = [&](const u32x4& a, const u32x4(&b)[NT], int i) {
#pragma unroll
    for (int t = 0; t < NT; ++t) Mma<T>::go(b[t], a, acc[((t >> 2) * MT + i) * 4 + (t & 3)]);
  };
  // Reads per group: done two groups before the half's end, for their latency.
  constexpr int RPG = (MT + NT + MT - 3) / (MT - 2);
  constexpr int CPG = (COPIES + MT - 1) / MT;

  {
    const Source first = source(s0), second = source(s0 + 1);
    copy(first, smem, 0, COPIES);
    copy(second, smem + BUF, 0, COPIES);
  }
  wait_copies<COPIES>();
  read(a0, b0, smem, 0, 0, MT + NT);
  settle(acc);
  char* cur = smem;
  char* next = smem + BUF;
  // An empty slice runs one step of zeros (no step of it is live): without a way
  // around the loop the sums stay in their registers.
  int s = s0;
  do {
    const Source after = source(s + 2);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      read(a1, b1, cur, 1, i * RPG, (i + 1) * RPG);
      __builtin_amdgcn_sched_barrier(0);
      multiply(a0[i], b0, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_copies<0>();
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      read(a0, b0, next, 0, i * RPG, (i + 1) * RPG);
      copy(after, cur, i * CPG, (i + 1) * CPG);
      __builtin_amdgcn_sched_barrier(0);
      multiply(a1[i], b1, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    char* t = cur;
    cur = next;
    next = t;
  } while (++s < s1);
  wait_copies<0>();
  settle(acc);
  Acc(&out)[G][MT][4] = reinterpret_cast<Acc(&)[G][MT][4]>(acc);
#pragma unroll
  for (int j = 0; j < G; ++j)
    Epilogue<T, EPI, BS>::run(g, out[j], id.prob, id.slice, m0 + wm * MT * 16,
                              n0 + (wn * G + j) * (GATED ? 32 : 64), lane);
}

// The epilogue of a product split over K: the slices' sums added in order, then as
// in k_dense.  One thread per 4 columns; blockIdx.y counts rows (and problems).
template <typename T, int EPI>
__global__ __launch_bounds__(256) void k_dense_join(GemmArgs g) {
  typedef typename Mma<T>::Acc Acc;
  constexpr bool GATED = EPI == kGated || EPI == kGatedMax;
  const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
  const int limit = EPI == kStore || EPI == kScale ? g.N : (g.N + 7) & ~7;
  for (int64_t row = blockIdx.y; row < (int64_t)g.M * g.nprob; row += gridDim.y) {
    const int prob = (int)(row / g.M), m = (int)(row % g.M);
    const int64_t ld = GATED ? 2 * g.ldp : g.ldp;
    const Acc* p = (const Acc*)g.part + (row * ld + n) / 4;
    const int64_t step = (int64_t)g.nprob * g.M * ld / 4;
    Acc s = Acc{}, u = Acc{};
    if (n < g.N) {
      for (int i = 0; i < g.slices; ++i) {
        s += p[i * step];
        if (GATED) u += p[i * step + g.ldp / 4];
      }
    }
    if constexpr (EPI == kGated) {
      if (n >= limit) continue;
      float a[4], gg[4], uu[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        gg[i] = s[i];
        uu[i] = u[i];
        a[i] = silu(s[i]) * u[i];
      }
      const int64_t at = (int64_t)m * g.ldi + n;
      store_run<T, 4>((T*)g.out[0] + at, a, 4, true);
      if (g.out[1] != nullptr) {
        store_run<float, 4>((float*)g.out[1] + at, gg, 4, true);
        store_run<float, 4>((float*)g.out[2] + at, uu, 4, true);
      }
    } else if constexpr (EPI == kGatedMax) {
      unsigned mx = 0;
      if (n < limit) {
        float v[4];
        const float sm = g.row_scale[m];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = 0.0f;
          if (n + i < g.N) {
            const float gg = (float)s[i] * sm * g.col_scale[0][n + i];
            v[i] = silu(gg) * ((float)u[i] * sm * g.col_scale[1][n + i]);
          }
          mx = max(mx, __float_as_uint(v[i]) & 0x7fffffffu);
        }
        store_run<float, 4>((float*)g.out[0] + (int64_t)m * g.ldi + n, v, 4, true);
      }
#pragma unroll
      for (int d = 1; d < 64; d *= 2) mx = max(mx, (unsigned)__shfl_xor((int)mx, d));
      if ((threadIdx.x & 63) == 0) atomicMax(g.row_max + m, mx);
    } else {
      if (n < limit) Epilogue<T, EPI, true>::tile(g, s, prob, 0, m, n);
    }
  }
}

// ---- launching --------------------------------------------------------------
template <typename T, int WM, int WN, int MT, int G, bool AS, bool BS, int EPI>
hipError_t launch_tile(const GemmArgs& g, hipStream_t s) {
  const int64_t blocks = (int64_t)g.tiles_m * g.tiles_n * g.nprob * g.slices;
  k_dense<T, WM, WN, MT, G, AS, BS, EPI><<<(unsigned)blocks, WM * WN * 64, 0, s>>>(g);
  return hipGetLastError();
}

template <typename T, bool AS, bool BS, int EPI>
hipError_t launch_shape(const GemmArgs& g, int shape, hipStream_t s) {
  switch (shape) {
    case kTile256:  // fp32 is bound by its products, not by the LDS: smaller wave tiles
      if constexpr (sizeof(T) == 4) return launch_tile<T, 2, 4, 8, 1, AS, BS, EPI>(g, s);
      return launch_tile<T, 2, 2, 8, 2, AS, BS, EPI>(g, s);
    case kTile128: return launch_tile<T, 2, 2, 4, 1, AS, BS, EPI>(g, s);
    default: return launch_tile<T, 1, 4, 4, 1, AS, BS, EPI>(g, s);
  }
}

// EPI of the whole product; SPLIT the epilogue of its slices.
template <typename T, bool AS, bool BS, int EPI, int SPLIT>
hipError_t launch_epi(const GemmArgs& g, int shape, hipStream_t s) {
  if (g.slices == 1) return launch_shape<T, AS, BS, EPI>(g, shape, s);
  const hipError_t e = launch_shape<T, AS, BS, SPLIT>(g, shape, s);
  if (e != hipSuccess) return e;
  const int64_t rows = (int64_t)g.M * g.nprob;
  const dim3 grid((g.N + 1023) / 1024, (unsigned)(rows < 65535 ? rows : 65535));
  k_dense_join<T, EPI><<<grid, 256, 0, s>>>(g);
  return hipGetLastError();
}

// The products of a floating-point type.
template <typename T>
hipError_t launch_float(const GemmArgs& g, int shape, int form, hipStream_t s) {
  switch (form) {
    case kFormGated: return launch_epi<T, false, false, kGated, kPartGated>(g, shape, s);
    case kFormKcKc: return launch_epi<T, false, false, kStore, kPart>(g, shape, s);
    case kFormGateGrad: return launch_epi<T, false, true, kGateGrad, kPart>(g, shape, s);
    case kFormKcKs: return launch_epi<T, false, true, kStore, kPart>(g, shape, s);
    default: return launch_epi<T, true, true, kStore, kPart>(g, shape, s);
  }
}

}  // namespace ffn
}  // namespace wr
