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
// (buffer_load ... lds, 16 bytes a lane), into a ring of 2 or 3 buffers of which
// one is multiplied.  The copy's buffer descriptor ends at the operand's
// last element, so rows past the end arrive as zeros without a branch; K
// tails and column tails give their lanes an offset behind the descriptor.
//
// A wave owns MT x 4 tiles of 16 x 16.  B is the MFMA's first operand, so a
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
template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
  typedef f32x4 Acc;
  static __device__ __forceinline__ Acc add(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<f16> {
  typedef f32x4 Acc;
  static __device__ __forceinline__ Acc add(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<int8_t> {
  typedef i32x4 Acc;
  static __device__ __forceinline__ Acc add(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a),
                                                 __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  }
};
// fp32: lane group q holds k = 4 q .. 4 q + 3, one element per MFMA.
template <>
struct Mma<float> {
  typedef f32x4 Acc;
  static __device__ __forceinline__ Acc add(u32x4 a, u32x4 b, Acc c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
};

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

  // left: elements left from the tile's first one, of m (n) (KS) or of K (KC: KB or more
  // except at the last step of a segment).
  __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int left) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      int c;  // chunk of this lane in its row
      unsigned at;
      if (KS) {
        constexpr int CPR = ROWS * ES / 16;  // chunks per k row
        const int L = (j * NW + wave) * 64 + lane;
        const int k = L / CPR, p = L % CPR;
        constexpr int U = ES == 4 ? 4 : 2;  // chunks per swizzle unit
        c = ((p / U) ^ ks_key<ES, ROWS>(k)) * U + p % U;
        at = (unsigned)(k * ld);
      } else {
        int row = (j * NW + wave) * 8 + (lane >> 3);
        c = (lane & 7) ^ kc_key<NSIDE>(row);
        if (GATED) row = (row >> 4) * 8 + (row & 7);  // rows 8..15 of 16 are the other matrix's
        at = (unsigned)(row * ld);
      }
      voff[j] = c * EPC < left ? at + c * 16 : kOutside;
    }
  }

  // Copy j from a descriptor whose base is the tile's first byte at this K step.
  __device__ __forceinline__ void issue(int j, char* lds, __amdgpu_buffer_rsrc_t r, int wave) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        r, (__attribute__((address_space(3))) void*)(lds + (j * NW + wave) * 1024), 16,
        (int)voff[j], 0, 0, 0);
  }
};

// Descriptor of the `end` bytes from base (none: every lane's copy is zero).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(const char* base, int64_t end) {
  const int high = (int)(end >> 31);
  const int records = high == 0 ? (int)end : high < 0 ? 0 : 0x7fffffff;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, records, 0x00020000);
}

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
      // M side: row 16 s + r.  N side: subtile t's row r = 4 q' + i is LDS row 16 q' + 4 t + i.
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
      const int row = s * (NSIDE ? 4 : 16);
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

// N consecutive elements at p[0..N), of which the first `left` exist.  p has its element's
// alignment: a store that is not aligned to its size is still one instruction.
template <typename T, int N>
__device__ __forceinline__ void store_run(T* p, const float* v, int left) {
  if (left >= N) {
    typedef T V __attribute__((ext_vector_type(N)));
    typedef V V_any __attribute__((aligned(sizeof(T))));
    V o;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = to_out<T>(v[i]);
    *(V_any*)p = o;
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

  // What the epilogue of 16 m and 64 n reads, loaded one piece ahead of its use.
  static constexpr int INS = EPI == kGateGrad ? 8 : EPI == kScale || EPI == kGatedMax ? 4 : 1;
  struct In {
    f32x4 v[INS];
    float row;
  };
  // First n of a lane's subtile t.
  static __device__ __forceinline__ int col(int n0, int q, int t) {
    return n0 + (BS ? t * 16 + q * 4 : q * 16 + t * 4);
  }
  // Four column scales from n, zero past N.
  static __device__ __forceinline__ f32x4 cols4(const float* p, int n, int N) {
    typedef f32x4 f32x4_any __attribute__((aligned(4)));
    f32x4 v{};
    if (n + 4 <= N) v = *(const f32x4_any*)(p + n);
    else
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (n + i < N) v[i] = p[n + i];
    return v;
  }
  static __device__ __forceinline__ In load(const GemmArgs& g, int m0, int n0, int lane) {
    const int q = lane >> 4, m = m0 + (lane & 15);
    In in{};
    if constexpr (EPI == kGateGrad) {
      const int n = n0 + (lane & 15) * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = m0 + j * 4 + q;
        if (row >= g.M || n >= ((g.N + 7) & ~7)) continue;
        in.v[j] = *(const f32x4*)((const float*)g.in[0] + (int64_t)row * g.ldi + n);
        in.v[4 + j] = *(const f32x4*)((const float*)g.in[1] + (int64_t)row * g.ldi + n);
      }
      return in;
    }
    if (m >= g.M) return in;
    if constexpr (EPI == kScale) {
      in.row = g.row_scale[m];
#pragma unroll
      for (int t = 0; t < 4; ++t) in.v[t] = cols4(g.col_scale[0], col(n0, q, t), g.N);
    } else if constexpr (EPI == kGatedMax) {
      in.row = g.row_scale[m];
#pragma unroll
      for (int t = 0; t < 4; ++t)
        in.v[t] = cols4(g.col_scale[t >> 1], n0 + q * 8 + (t & 1) * 4, g.N);
    }
    return in;
  }

  // 16 m from m0, and 64 n from n0 (gated: 32 of gate, 32 of up) in 4 subtiles.  lds: 4 KB of the
  // wave's own.
  static __device__ __forceinline__ void run(const GemmArgs& g, const Acc (&acc)[4], const In& in,
                                             int prob, int m0, int n0, int lane, char* lds) {
    const int r = lane & 15, q = lane >> 4, m = m0 + r;
    if constexpr (EPI == kGateGrad) {
      // g, u, dg and du are 12 bytes per element of the tile, so that their lines count: the
      // sums change lanes in LDS, and each access covers whole rows of the piece (256
      // bytes of 4 rows) instead of 64 bytes of 16.
#pragma unroll
      for (int t = 0; t < 4; ++t) *(f32x4*)(lds + r * 256 + ((t * 4 + q) ^ r) * 16) = acc[t];
      __builtin_amdgcn_wave_barrier();
      const int n = n0 + r * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = j * 4 + q;
        const f32x4 da = *(const f32x4*)(lds + row * 256 + (r ^ row) * 16);
        // dg and du rows are read in whole 16-byte chunks: their zeros past N too.
        if (m0 + row >= g.M || n >= ((g.N + 7) & ~7)) continue;
        float dg[4], du[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          gate_grad(da[i], in.v[j][i], in.v[4 + j][i], dg[i], du[i]);
          if (n + i >= g.N) dg[i] = du[i] = 0.0f;
        }
        const int64_t at = (int64_t)(m0 + row) * g.ldi + n;
        store_run<T, 4>((T*)g.out[0] + at, dg, 4);
        store_run<T, 4>((T*)g.out[1] + at, du, 4);
      }
      __builtin_amdgcn_wave_barrier();
    } else if constexpr (EPI == kGatedMax) {
      gated_max(g, acc, in, m, n0 + q * 8);
    } else if (m >= g.M) {
      return;
    } else if constexpr (EPI == kGated) {
      float gg[8], uu[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        gg[i] = acc[i / 4][i % 4];
        uu[i] = acc[i / 4 + 2][i % 4];
      }
      gated<8>(g, gg, uu, m, n0 + q * 8);
    } else if constexpr (!BS) {  // 16 consecutive n a lane
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[i] = (float)acc[i / 4][i % 4];
        if (EPI == kScale) v[i] = v[i] * in.row * in.v[i / 4][i % 4];
      }
      store<16>(g, prob, m, n0 + q * 16, v);
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t) tile(g, acc[t], prob, m, col(n0, q, t));
    }
  }

  // C consecutive n of one m into the output.
  template <typename O, int C>
  static __device__ __forceinline__ void store_as(const GemmArgs& g, int prob, int m, int n,
                                                  const float (&v)[C]) {
    O* const p = (O*)g.out[prob] + (int64_t)m * g.ldo + n;
    constexpr int V = 16 / sizeof(O) < C ? 16 / sizeof(O) : C;
#pragma unroll
    for (int i = 0; i < C; i += V) store_run<O, V>(p + i, v + i, g.N - n - i);
  }
  template <int C>
  static __device__ __forceinline__ void store(const GemmArgs& g, int prob, int m, int n,
                                               const float (&v)[C]) {
    if constexpr (EPI == kStore) store_as<T>(g, prob, m, n, v);
    else if (g.out_dtype == WR_F32) store_as<float>(g, prob, m, n, v);
    else if (g.out_dtype == WR_F16) store_as<f16>(g, prob, m, n, v);
    else store_as<bf16>(g, prob, m, n, v);
  }

  // Four consecutive n of one m.
  static __device__ __forceinline__ void tile(const GemmArgs& g, Acc a, int prob, int m, int n) {
    if (m >= g.M || n >= g.N) return;
    float v[4] = {(float)a[0], (float)a[1], (float)a[2], (float)a[3]};
    if constexpr (EPI == kScale) {
      const float row = g.row_scale[m];
      const f32x4 c = cols4(g.col_scale[0], n, g.N);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = v[i] * row * c[i];
    }
    store<4>(g, prob, m, n, v);
  }

  // C gate and up sums of the same n.  The buffers' rows are padded to ldi (a multiple of
  // 64), so whole vectors are stored; a is read in whole 16-byte chunks, so its values
  // past N are zeros (the sums there are not, where x holds an infinity).
  template <int C>
  static __device__ __forceinline__ void gated(const GemmArgs& g, const float (&gg)[C],
                                               const float (&uu)[C], int m, int n) {
    if (n >= ((g.N + 7) & ~7)) return;
    float a[C];
#pragma unroll
    for (int i = 0; i < C; ++i) a[i] = n + i < g.N ? silu(gg[i]) * uu[i] : 0.0f;
    const int64_t at = (int64_t)m * g.ldi + n;
    constexpr int V = 16 / sizeof(T) < C ? 16 / sizeof(T) : C;
#pragma unroll
    for (int i = 0; i < C; i += V) store_run<T, V>((T*)g.out[0] + at + i, a + i, V);
    if (g.out[1] != nullptr) {
#pragma unroll
      for (int i = 0; i < C; i += 4) {
        store_run<float, 4>((float*)g.out[1] + at + i, gg + i, 4);
        store_run<float, 4>((float*)g.out[2] + at + i, uu + i, 4);
      }
    }
  }

  // int8: a = silu(g) u in fp32 of 8 n from n, with the row maxima of |a| (as fp32 bits: the
  // maximum of non-negative floats is that of their bits, in any order).
  static __device__ __forceinline__ void gated_max(const GemmArgs& g, const Acc (&acc)[4],
                                                   const In& in, int m, int n) {
    unsigned mx = 0;
    if (m < g.M) {
      mx = scaled_gate(g, acc[0], acc[2], m, n, in.row, in.v[0], in.v[2]);
      mx = max(mx, scaled_gate(g, acc[1], acc[3], m, n + 4, in.row, in.v[1], in.v[3]));
    }
    mx = max(mx, (unsigned)__shfl_xor((int)mx, 16));
    mx = max(mx, (unsigned)__shfl_xor((int)mx, 32));
    if ((threadIdx.x & 63) < 16 && m < g.M) atomicMax(g.row_max + m, mx);
  }
  // Four n, with the scales of their row and columns (zero past N); returns their maximum.
  static __device__ __forceinline__ unsigned scaled_gate(const GemmArgs& g, Acc gate, Acc up, int m,
                                                         int n, float row, f32x4 cg, f32x4 cu) {
    unsigned mx = 0;
    if (n >= g.N) return mx;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = silu((float)gate[i] * row * cg[i]) * ((float)up[i] * row * cu[i]);
      if (n + i >= g.N) v[i] = 0.0f;  // a NaN row scale times the zero
      mx = max(mx, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    store_run<float, 4>((float*)g.out[0] + (int64_t)m * g.ldi + n, v, 4);
    return mx;
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
// A block of WM x WN waves, each with MT x 4 subtiles of 16 x 16.  Both halves' (64
// bytes of K) fragments are held in registers: while one half is multiplied, the
// other's are read.  The K step's only barrier lies between its halves: behind it the
// next step's tiles are in LDS (their copies were issued SLOTS - 1 steps earlier)
// and nobody reads the present ones any more, which the copies of step s + SLOTS
// then replace.  Each half is written as MT groups of 4 products, with the LDS
// reads and copies dealt to the groups and the groups kept in order, so that
// the matrix cores, the LDS and the copies run side by side in one wave.
//
// Measured (bf16, 4096 x 14336 by 14336 x 4096): 326 - 343 us, 1400 - 1475 TFLOP/s, the matrix
// cores busy 73% of the clocks at 1.8 GHz; zeros for data take 274 us, and with the
// copies and LDS reads left out the time stays: the chip's power bounds the loop.  4
// waves of 128 x 128 (all 512 registers) take the same time, tiles of 256 x 128 395 us and
// of 128 x 128 404 us: per product they copy 1.5 and 2 times the bytes into LDS, 70
// GB/s per CU.  The launch bound and the LDS given at launch keep 4 waves of 64 x 64 to
// 256 registers: with more the compiler moves sums between register files.
template <typename T, int WM, int WN, int MT, int SLOTS, bool AS, bool BS, int EPI>
__global__ __launch_bounds__(WM * WN * 64, 2) void k_dense(GemmArgs g) {
  constexpr bool GATED = EPI == kGated || EPI == kGatedMax;
  constexpr int NW = WM * WN, BM = WM * MT * 16, BN = WN * 64;
  constexpr int ABYTES = BM * kStepBytes, BBYTES = BN * kStepBytes, BUF = ABYTES + BBYTES;
  constexpr int ES = sizeof(T), KB = kStepBytes / ES;
  typedef typename Mma<T>::Acc Acc;
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // [SLOTS][BUF]

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  const TileId id = tile_of(g, (int)blockIdx.x);
  const int m0 = id.m * BM, n0 = id.n * (GATED ? BN / 2 : BN);
  const int steps = (g.K + KB - 1) / KB, total = steps * g.nseg;
  const int slices = id.tail < 0 ? 1 : g.slices;
  const int per = (total + slices - 1) / slices;
  const int s0 = id.slice * per, s1 = min(total, s0 + per);

  typedef TileCopy<T, BM, NW, AS, false, false> CopyA;
  typedef TileCopy<T, BN, NW, BS, true, GATED> CopyB;
  CopyA ca;
  CopyB cb;
  Frag<T, BM, MT, AS, false> fa;
  Frag<T, BN, 4, BS, true> fb;
  fa.init(wm * MT, lane);
  fb.init(wn * 4, lane);

  // The next step to copy: its first bytes, the operands' bytes from there on, its K
  // elements left.
  const int seg0 = s0 >= steps ? 1 : 0, k0 = (s0 - seg0 * steps) * KB;
  const int64_t stepa = AS ? KB * g.lda : kStepBytes, stepb = BS ? KB * g.ldb : kStepBytes;
  const int64_t offa = AS ? (int64_t)m0 * ES : m0 * g.lda, offb = BS ? (int64_t)n0 * ES : n0 * g.ldb;
  const int64_t alla = AS ? (g.K - 1) * g.lda + chunked((int64_t)g.M * ES)
                          : (g.M - 1) * g.lda + chunked((int64_t)g.K * ES);
  const int64_t allb = BS ? (g.K - 1) * g.ldb + chunked((int64_t)g.N * ES)
                          : (g.N - 1) * g.ldb + chunked((int64_t)g.K * ES);
  const char* const pa1 = g.a[1] + offa;
  const char* const pb1 = g.b[1] + offb;
  const char* pa = (seg0 ? pa1 : g.a[id.prob] + offa) + (s0 - seg0 * steps) * stepa;
  const char* pb = (seg0 ? pb1 : g.b[GATED ? (wave & 1) : 0] + offb) + (s0 - seg0 * steps) * stepb;
  int64_t enda = alla - offa - (s0 - seg0 * steps) * stepa;
  int64_t endb = allb - offb - (s0 - seg0 * steps) * stepb;
  int krem = g.K - k0, todo = s1 - s0;
  auto offsets = [&]() {
    ca.init(wave, lane, g.lda, AS ? g.M - m0 : krem);
    cb.init(wave, lane, g.ldb, BS ? g.N - n0 : krem);
  };
  offsets();
  struct Source {
    __amdgpu_buffer_rsrc_t a, b;
  };
  // The step's descriptors; a step that does not exist (todo <= 0) copies zeros.
  auto source = [&]() {
    const Source r{descriptor(pa, todo > 0 ? enda : 0), descriptor(pb, todo > 0 ? endb : 0)};
    return r;
  };
  // On to the next one.  The lanes' offsets change only around a segment's last step, whose
  // chunks past K they leave out.
  auto advance = [&]() {
    --todo;
    pa += stepa;
    pb += stepb;
    enda -= stepa;
    endb -= stepb;
    krem -= KB;
    if (krem < KB) {
      if (krem <= 0) {
        pa = pa1;
        pb = pb1;
        enda = alla - offa;
        endb = allb - offb;
        krem = g.K;
      }
      offsets();
    }
  };
  // Copies lo .. hi - 1 of a step's CopyA::PER + CopyB::PER.
  auto copy = [&](const Source& s, char* lds, int lo, int hi) {
#pragma unroll
    for (int j = 0; j < CopyA::PER + CopyB::PER; ++j) {
      if (j < lo || j >= hi) continue;
      if (j < CopyA::PER)
        ca.issue(j, lds, s.a, wave);
      else
        cb.issue(j - CopyA::PER, lds + ABYTES, s.b, wave);
    }
  };
  constexpr int COPIES = CopyA::PER + CopyB::PER;

  Acc acc[MT * 4];  // [m subtile][n subtile]
#pragma unroll
  for (int i = 0; i < MT * 4; ++i) acc[i] = Acc{};

  u32x4 a0[MT], b0[4], a1[MT], b1[4];
  // Fragments lo .. hi - 1, those of B first: every product needs them.
  auto read = [&](u32x4(&a)[MT], u32x4(&b)[4], char* tile, int kk, int lo, int hi) {
#pragma unroll
    for (int j = 0; j < MT + 4; ++j) {
      if (j < lo || j >= hi) continue;
      if (j < 4)
        b[j] = fb.get(tile + ABYTES, j, kk);
      else
        a[j - 4] = fa.get(tile, j - 4, kk);
    }
  };
  auto multiply = [&](const u32x4& a, const u32x4(&b)[4], int i) {
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[i * 4 + t] = Mma<T>::add(b[t], a, acc[i * 4 + t]);
  };
  // Reads per group: done two groups before the half's end, for their latency.
  constexpr int RPG = (MT + 4 + MT - 3) / (MT - 2);
  constexpr int CPG = (COPIES + MT - 1) / MT;

#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    copy(source(), smem + i * BUF, 0, COPIES);
    advance();
  }
  wait_copies<(SLOTS - 1) * COPIES>();
  read(a0, b0, smem, 0, 0, MT + 4);
  int at = 0;
  // An empty slice runs one step of zeros (no step of it exists).
  int s = s0;
  do {
    const Source after = source();
    char* const cur = smem + at * BUF;
    at = at + 1 == SLOTS ? 0 : at + 1;
    char* const next = smem + at * BUF;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      read(a1, b1, cur, 1, i * RPG, (i + 1) * RPG);
      __builtin_amdgcn_sched_barrier(0);
      multiply(a0[i], b0, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_copies<(SLOTS - 2) * COPIES>();
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      read(a0, b0, next, 0, i * RPG, (i + 1) * RPG);
      copy(after, cur, i * CPG, (i + 1) * CPG);
      __builtin_amdgcn_sched_barrier(0);
      multiply(a1[i], b1, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    advance();
  } while (++s < s1);
  wait_copies<0>();
  // A slice stores its sums as they lie in the registers.
  Acc* const part = id.tail < 0 ? nullptr
                                : (Acc*)g.part + ((int64_t)(id.tail * g.slices + id.slice) * NW + wave) *
                                                     (MT * 4 * 64) + lane;
  typedef Epilogue<T, EPI, BS> E;
  // Pieces of 16 m x 64 n.
  auto pm = [&](int p) { return m0 + (wm * MT + p) * 16; };
  const int pn = n0 + wn * (GATED ? 32 : 64);
  typename E::In in{};
  if (part == nullptr) in = E::load(g, pm(0), pn, lane);
#pragma unroll
  for (int p = 0; p < MT; ++p) {
    const Acc(&piece)[4] = *reinterpret_cast<Acc(*)[4]>(&acc[p * 4]);
    if (part == nullptr) {
      typename E::In next{};
      if (p + 1 < MT) next = E::load(g, pm(p + 1), pn, lane);
      E::run(g, piece, in, id.prob, pm(p), pn, lane, smem + wave * 4096);
      in = next;
    } else if (pm(p) < g.M) {
#pragma unroll
      for (int t = 0; t < 4; ++t) part[(p * 4 + t) * 64] = piece[t];
    }
    __builtin_amdgcn_sched_barrier(0);  // pieces one after another: registers
  }
}

// The tiles split over K: their slices' sums added in order, then as in k_dense.  One
// wave per 16 m x 64 n (gated: 32 of each matrix) of a tile.
template <typename T, int WM, int WN, int MT, bool BS, int EPI>
__global__ __launch_bounds__(256) void k_dense_join(GemmArgs g) {
  constexpr bool GATED = EPI == kGated || EPI == kGatedMax;
  constexpr int NW = WM * WN, PIECES = NW * MT;
  typedef typename Mma<T>::Acc Acc;
  const int lane = threadIdx.x & 63;
  const int64_t piece = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int tail = (int)(piece / PIECES), rest = (int)(piece % PIECES);
  const int wave = rest / MT, i = rest % MT;
  if (tail >= g.tiles - g.whole) return;
  const TileId id = tile_at(g, g.whole + tail);
  const int m0 = id.m * (WM * MT * 16) + (wave / WN * MT + i) * 16;
  if (m0 >= g.M) return;
  const int n0 = (id.n * WN + wave % WN) * (GATED ? 32 : 64);
  const Acc* p = (const Acc*)g.part + ((int64_t)tail * g.slices * NW + wave) * (MT * 4 * 64) +
                 i * 4 * 64 + lane;
  typedef Epilogue<T, EPI, BS> E;
  const typename E::In in = E::load(g, m0, n0, lane);
  Acc acc[4] = {};
  constexpr int U = 8;  // slices in flight
  for (int s = 0; s < g.slices; s += U) {
    Acc v[U][4];
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        v[j][t] = s + j < g.slices ? p[(int64_t)(s + j) * NW * (MT * 4 * 64) + t * 64] : Acc{};
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (s + j < g.slices) acc[t] += v[j][t];
  }
  __shared__ __attribute__((aligned(16))) char lds[4 * 4096];
  E::run(g, acc, in, id.prob, m0, n0, lane, lds + (threadIdx.x >> 6) * 4096);
}

// ---- few rows of m ---------------------------------------------------------
// M <= 16: bound by the bytes of B, which are read once.  A block owns 16 S rows of B
// (gated: half of them of gate, the same n of up) and splits K over its waves,
// whose sums meet in LDS: one launch, no sums through memory.
//
// k_dense_rows: each wave copies its part of K into a ring of its own in LDS, 128 bytes of
// 8 rows per copy, with kRowSlots - 1 steps in flight and no barrier.
// 16 tokens, gate and up of 4096 x 14336 fp16 (235 MB): 44 us, 5.3 TB/s; loads straight
// into the products' registers (16 rows x 64 bytes per load) take 61 us.  2, 3, 4 and
// 6 slots with 2 to 8 waves: 3 slots and 4 waves are within 3% of the best of them
// for every product measured.
constexpr int kRowSlots = 3;

// Joins the waves' sums (acc[S] of each) in LDS and runs the epilogue.
template <typename T, int S, int EPI>
__device__ __forceinline__ void join_waves(const GemmArgs& g, typename Mma<T>::Acc (&acc)[S],
                                           char* lds, int m0, int n0, int wave, int waves,
                                           int lane) {
  constexpr bool GATED = EPI == kGated || EPI == kGatedMax;
  typedef typename Mma<T>::Acc Acc;
  const int r = lane & 15, q = lane >> 4;
  Acc* const sums = (Acc*)lds;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < S; ++i) sums[(wave * S + i) * 64 + lane] = acc[i];
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int i = 0; i < S; ++i)
    for (int w = 1; w < waves; ++w) acc[i] += sums[(w * S + i) * 64 + lane];
  const int m = m0 + r;
  if constexpr (!GATED) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int n = n0 + i * 16 + q * 4;
      Epilogue<T, EPI, true>::tile(g, acc[i], 0, m, n);
    }
  } else {
    Acc up = acc[S - 1];
    if (S == 1) {  // lane groups 0 and 1 hold gate, 2 and 3 the same n of up
      i32x4 bits = __builtin_bit_cast(i32x4, up);
#pragma unroll
      for (int i = 0; i < 4; ++i) bits[i] = __shfl_xor((int)bits[i], 32);
      up = __builtin_bit_cast(Acc, bits);
    }
    const int n = n0 + q * 4;
    const bool mine = m < g.M && (S == 2 || q < 2);
    if constexpr (EPI == kGated) {
      if (!mine) return;
      float gg[4], uu[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        gg[i] = acc[0][i];
        uu[i] = up[i];
      }
      Epilogue<T, EPI, true>::template gated<4>(g, gg, uu, m, n);
    } else {
      typedef Epilogue<T, EPI, true> E;
      unsigned mx = 0;
      if (mine)
        mx = E::scaled_gate(g, acc[0], up, m, n, g.row_scale[m], E::cols4(g.col_scale[0], n, g.N),
                            E::cols4(g.col_scale[1], n, g.N));
      mx = max(mx, (unsigned)__shfl_xor((int)mx, 16));
      mx = max(mx, (unsigned)__shfl_xor((int)mx, 32));
      if (q == 0 && m < g.M) atomicMax(g.row_max + m, mx);
    }
  }
}

template <typename T, int S, int EPI>
__global__ __launch_bounds__(512) void k_dense_rows(GemmArgs g) {
  constexpr bool GATED = EPI == kGated || EPI == kGatedMax;
  constexpr int ES = sizeof(T), KB = kStepBytes / ES, EPC = 16 / ES;
  constexpr int COPIES = 2 * S + 2, SLOT = COPIES * 1024;  // 16 S rows of B, 16 of A
  typedef typename Mma<T>::Acc Acc;
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // [wave][kRowSlots][SLOT]
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int n0 = blockIdx.x * (GATED ? 8 * S : 16 * S);
  char* const ring = smem + wave * (kRowSlots * SLOT);

  // Copy j: rows 8 j .. 8 j + 7 of B's tile, then of A.
  auto copy = [&](int step, char* slot, bool live) {
    const int k = step * KB;
#pragma unroll
    for (int j = 0; j < COPIES; ++j) {
      const int lr = (j < 2 * S ? j : j - 2 * S) * 8 + (lane >> 3);  // row in the tile
      const int chunk = (lane & 7) ^ ((lr >> 1) & 7);
      const char* base;
      int64_t end;
      unsigned v;
      if (j < 2 * S) {
        const int first = n0 + (GATED ? j % S * 8 : j * 8);  // S copies of gate, then of up
        base = g.b[GATED && j >= S ? 1 : 0] + first * g.ldb + (int64_t)k * ES;
        end = (g.N - 1 - first) * g.ldb + chunked((int64_t)g.K * ES) - (int64_t)k * ES;
        v = (unsigned)((lane >> 3) * g.ldb);
      } else {
        const int first = (j - 2 * S) * 8;
        base = g.a[0] + first * g.lda + (int64_t)k * ES;
        end = (g.M - 1 - first) * g.lda + chunked((int64_t)g.K * ES) - (int64_t)k * ES;
        v = (unsigned)((lane >> 3) * g.lda);
      }
      const int records = !live || end < 0 ? 0 : end > 0x7fffffff ? 0x7fffffff : (int)end;
      const __amdgpu_buffer_rsrc_t src =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, records, 0x00020000);
      v = chunk * EPC < g.K - k ? v + chunk * 16 : kOutside;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          src, (__attribute__((address_space(3))) void*)(slot + j * 1024), 16, (int)v, 0, 0, 0);
    }
  };

  const int steps = (g.K + KB - 1) / KB, per = (steps + waves - 1) / waves;
  const int s0 = wave * per, s1 = min(steps, s0 + per);
  Acc acc[S];
#pragma unroll
  for (int i = 0; i < S; ++i) acc[i] = Acc{};
#pragma unroll
  for (int i = 0; i < kRowSlots - 1; ++i) copy(s0 + i, ring + i * SLOT, s0 + i < s1);
  int at = 0, fill = kRowSlots - 1;
  for (int s = s0; s < s1; ++s) {
    copy(s + kRowSlots - 1, ring + fill * SLOT, s + kRowSlots - 1 < s1);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kRowSlots - 1) * COPIES) : "memory");
    const char* const slot = ring + at * SLOT;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int pos = r * kStepBytes + ((kk * 4 + q) ^ ((r >> 1) & 7)) * 16;
      const u32x4 a = lds_b128(slot + 2 * S * 1024 + pos);
#pragma unroll
      for (int i = 0; i < S; ++i)
        acc[i] = Mma<T>::add(lds_b128(slot + i * 2048 + pos), a, acc[i]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next copy replaces it
    at = at + 1 == kRowSlots ? 0 : at + 1;
    fill = fill + 1 == kRowSlots ? 0 : fill + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  join_waves<T, S, EPI>(g, acc, smem, 0, n0, wave, waves, lane);
}

// k_dense_any: up to 64 rows of m, for rows that are no whole 16-byte chunks (which the tiled
// products need copied first), with loads straight into the products' registers: 16
// bytes of one row a lane, of any alignment.  Rows past
// the matrices' ends read the last one again, their results are dropped.
typedef u32x4 u32x4_any __attribute__((aligned(1)));

// 16 bytes at element k of a row of K elements, zero behind its end.
template <typename T>
__device__ __forceinline__ u32x4 load_tail(const char* row, int k, int K) {
  constexpr int N = 16 / sizeof(T);
  typedef typename std::conditional<sizeof(T) == 1, uint8_t,
                                    typename std::conditional<sizeof(T) == 2, uint16_t,
                                                              uint32_t>::type>::type U;
  typedef U V __attribute__((ext_vector_type(N)));
  V v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = k + i < K ? ((const U*)row)[k + i] : (U)0;
  return __builtin_bit_cast(u32x4, v);
}

template <typename T, int EPI>
__global__ __launch_bounds__(512) void k_dense_any(GemmArgs g) {
  constexpr bool GATED = EPI == kGated || EPI == kGatedMax;
  constexpr int KB = kStepBytes / 2 / sizeof(T), EPC = 16 / sizeof(T);
  constexpr int kUnroll = 8;
  typedef typename Mma<T>::Acc Acc;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  // Blocks 8 apart run on one XCD: its L2 serves B's rows to all their tiles of m.
  const int place = blockIdx.x >> 3;
  const int m0 = place % g.tiles_m * 16;
  const int n0 = (place / g.tiles_m * 8 + (blockIdx.x & 7)) * (GATED ? 8 : 16);
  if (n0 >= g.N) return;
  const int row = min(n0 + (GATED ? r & 7 : r), g.N - 1);
  const char* const pb = g.b[GATED ? r >> 3 : 0] + row * g.ldb;
  const char* const pa = g.a[0] + min(m0 + r, g.M - 1) * g.lda;

  // 64-byte stages of K in whole 128-byte pairs per wave.
  const int stages = (g.K + KB - 1) / KB, per = (stages + 2 * waves - 1) / (2 * waves) * 2;
  const int whole = g.K / KB;  // stages without a tail
  int s = min(stages, wave * per);
  const int end = min(stages, s + per);
  Acc acc[1] = {};
  auto run = [&](auto count) {  // `count` stages without a tail
    constexpr int U = decltype(count)::value;
    u32x4 b[U], a[U];
    const int64_t at = (int64_t)s * 64 + q * 16;
#pragma unroll
    for (int j = 0; j < U; ++j) b[j] = *(const u32x4_any*)(pb + at + j * 64);
#pragma unroll
    for (int j = 0; j < U; ++j) a[j] = *(const u32x4_any*)(pa + at + j * 64);
#pragma unroll
    for (int j = 0; j < U; ++j) acc[0] = Mma<T>::add(b[j], a[j], acc[0]);
    s += U;
  };
  const int fast = min(end, whole);
  while (s + kUnroll <= fast) run(std::integral_constant<int, kUnroll>{});
  if (s + kUnroll / 2 <= fast) run(std::integral_constant<int, kUnroll / 2>{});
  if (s + kUnroll / 4 <= fast) run(std::integral_constant<int, kUnroll / 4>{});
  while (s < fast) run(std::integral_constant<int, 1>{});
  for (; s < end; ++s) {
    const int k = s * KB + q * EPC;
    acc[0] = Mma<T>::add(load_tail<T>(pb, k, g.K), load_tail<T>(pa, k, g.K), acc[0]);
  }
  join_waves<T, 1, EPI>(g, acc, smem, m0, n0, wave, waves, lane);
}

// ---- launching --------------------------------------------------------------
template <typename T, int WM, int WN, int MT, int SLOTS, bool AS, bool BS, int EPI>
hipError_t launch_tile(const GemmArgs& g, hipStream_t s) {
  const int tail = g.tiles - g.whole;
  const int64_t blocks = g.whole + (int64_t)tail * g.slices;
  constexpr size_t kLds = SLOTS * (WM * MT + WN * 4) * 16 * kStepBytes;
  k_dense<T, WM, WN, MT, SLOTS, AS, BS, EPI>
      <<<(unsigned)blocks, WM * WN * 64, kLds, s>>>(g);
  if (tail > 0) {
    const int64_t waves = (int64_t)tail * WM * WN * MT;
    k_dense_join<T, WM, WN, MT, BS, EPI><<<(unsigned)((waves + 3) / 4), 256, 0, s>>>(g);
  }
  return hipGetLastError();
}

template <typename T, int EPI>
hipError_t launch_rows(const GemmArgs& g, int shape, hipStream_t s) {
  const unsigned blocks = (unsigned)g.tiles;
  const int waves = g.slices;
  if (shape == kRowsAny)
    k_dense_any<T, EPI><<<(g.tiles_n + 7) / 8 * 8 * g.tiles_m, waves * 64, waves * 1024, s>>>(g);
  else if (shape == kRows16)
    k_dense_rows<T, 1, EPI><<<blocks, waves * 64, waves * kRowSlots * 4096, s>>>(g);
  else
    k_dense_rows<T, 2, EPI><<<blocks, waves * 64, waves * kRowSlots * 6144, s>>>(g);
  return hipGetLastError();
}

template <typename T, bool AS, bool BS, int EPI>
hipError_t launch_shape(const GemmArgs& g, int shape, hipStream_t s) {
  switch (shape) {
    case kRows16:
    case kRows32:
    case kRowsAny:
      if constexpr (!AS && !BS && EPI != kGateGrad) return launch_rows<T, EPI>(g, shape, s);
      return hipErrorInvalidValue;
    case kTile256: return launch_tile<T, 2, 4, 8, 2, AS, BS, EPI>(g, s);
    case kTile128: return launch_tile<T, 2, 2, 4, 2, AS, BS, EPI>(g, s);
    default: return launch_tile<T, 2, 2, 4, 3, AS, BS, EPI>(g, s);
  }
}

// The products of a floating-point type.
template <typename T>
hipError_t launch_float(const GemmArgs& g, int shape, int form, hipStream_t s) {
  switch (form) {
    case kFormGated: return launch_shape<T, false, false, kGated>(g, shape, s);
    case kFormKcKc: return launch_shape<T, false, false, kStore>(g, shape, s);
    case kFormGateGrad: return launch_shape<T, false, true, kGateGrad>(g, shape, s);
    case kFormKcKs: return launch_shape<T, false, true, kStore>(g, shape, s);
    default: return launch_shape<T, true, true, kStore>(g, shape, s);
  }
}

}  // namespace ffn
}  // namespace wr
