// Host side of the dense gated FFN and the int8 products (include/wr_ffn.h):
// argument checks, workspace, the choice of tiles, and the row kernels around
// the products (padded copies, quantisation).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "wr_device.h"
#include "wr_ffn.h"
#include "wr_ffn_internal.h"
#include "wr_internal.h"

namespace wr {
namespace ffn {
namespace {

constexpr int64_t round_up(int64_t n, int64_t a) { return (n + a - 1) / a * a; }

int elem_bytes(int dtype) { return dtype == WR_F32 ? 4 : 2; }
bool float_dtype(int d) { return d == WR_F32 || d == WR_F16 || d == WR_BF16; }

// ---- row kernels --------------------------------------------------------------
// Rows of a call's operands to rows of whole 16-byte chunks, the tails zero, for the product
// kernels' 16-byte copies: all of a call's in one launch, blockIdx.y the matrix.  Bound
// by the bytes; a thread assembles one chunk from units of U, the element type.
constexpr int kMaxPads = 5;
struct Pads {
  struct {
    const void* src;
    char* dst;
    int64_t rows, ld;  // ld: bytes
    int cols;
  } m[kMaxPads];
  int n;
};
template <typename U>
__global__ __launch_bounds__(256) void k_pad_rows(Pads pads) {
  const auto& job = pads.m[blockIdx.y];
  constexpr int N = 16 / sizeof(U);
  typedef U V __attribute__((ext_vector_type(N)));
  typedef V V_any __attribute__((aligned(sizeof(U))));
  const int per = (int)(job.ld / 16);
  // Four rows a block in turn, a wave each.
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < job.rows;
       row += (int64_t)gridDim.x * 4) {
    const U* const src = (const U*)job.src + row * job.cols;
    for (int i = threadIdx.x & 63; i < per; i += 64) {
      const int c = i * N;
      V v{};
      if (c + N <= job.cols) {
        v = *(const V_any*)(src + c);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (c + j < job.cols) v[j] = src[c + j];
      }
      *(V*)(job.dst + row * job.ld + i * 16) = v;
    }
  }
}

__global__ __launch_bounds__(256) void k_fill_zero(uint32_t* __restrict__ p, int64_t words,
                                                   char* __restrict__ tail, int tail_bytes) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words;
       i += (int64_t)gridDim.x * 256)
    p[i] = 0;
  if (blockIdx.x == 0 && (int)threadIdx.x < tail_bytes) tail[threadIdx.x] = 0;
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(f16 v) { return (float)v; }
__device__ __forceinline__ float as_float(__bf16 v) { return (float)v; }

// 127 x / m rounded to the nearest integer, ties to even, as the exact quotient rounds.
// x times inv = 127 / m in fp32 is off by less than 127 * 2^-22; where that could reach a
// half-integer, or inv leaves the range, the quotient is taken in 64 bits, whose error
// (127 * 2^-53) is below the 2^-34 by which a quotient of two 24-bit numbers misses a
// half-integer that it does not equal.  (A division per element took 20 us where the
// product takes 15, 4096 x 4096 bf16: the vector instructions bound it.)
__device__ __forceinline__ int code_of(float x, float m, float inv) {
  const float t = x * inv, near = rintf(t);
  if (fabsf(t - near) > 0.4999f || m < 1e-30f) return (int)rint((double)x * 127.0 / (double)m);
  return (int)near;
}

// The scale of a row with maximum m (as fp32 bits).
__device__ __forceinline__ float scale_of(unsigned mx) {
  return mx >= 0x7f800000u ? __builtin_nanf("") : mx == 0 ? 1.0f : __uint_as_float(mx) / 127.0f;
}

constexpr int kQuantHeld = 2;  // vectors of a row that a thread keeps from the maximum to the codes

// One block per row: max |row|, then the codes; a row's first kQuantHeld vectors per thread
// stay in registers, what is longer is read again.  codes rows are ldc bytes apart, zero
// from cols on.  zero_max, when set, gets its word of the row cleared.  WHOLE: cols is a
// multiple of a vector.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(1024) void k_quantize(const T* __restrict__ x, int cols,
                                                   int8_t* __restrict__ codes, int64_t ldc,
                                                   float* __restrict__ scales,
                                                   unsigned* __restrict__ zero_max) {
  __shared__ unsigned part[16];
  const int64_t row = blockIdx.x;
  const T* p = x + row * cols;
  constexpr int N = 16 / sizeof(T);
  typedef T V __attribute__((ext_vector_type(N)));
  typedef V V_any __attribute__((aligned(sizeof(T))));
  typedef int8_t Q __attribute__((ext_vector_type(N)));
  typedef Q Q_any __attribute__((aligned(1)));
  const int step = blockDim.x * N;
  auto read = [&](int c) {  // the vector at column c, zero from cols on
    V v{};
    if (WHOLE ? c < cols : c + N <= cols) {
      v = *(const V_any*)(p + c);
    } else if (!WHOLE) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + i < cols) v[i] = p[c + i];
    }
    return v;
  };
  auto top = [](V v) {
    unsigned mx = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) mx = max(mx, __float_as_uint(as_float(v[i])) & 0x7fffffffu);
    return mx;
  };
  V held[kQuantHeld];
  unsigned mx = 0;
#pragma unroll
  for (int j = 0; j < kQuantHeld; ++j) held[j] = read(threadIdx.x * N + j * step);
#pragma unroll
  for (int j = 0; j < kQuantHeld; ++j) mx = max(mx, top(held[j]));
  for (int c = threadIdx.x * N + kQuantHeld * step; c < cols; c += step) mx = max(mx, top(read(c)));
#pragma unroll
  for (int d = 1; d < 64; d *= 2) mx = max(mx, (unsigned)__shfl_xor((int)mx, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
  __syncthreads();
  for (int i = 0; i < (int)blockDim.x / 64; ++i) mx = max(mx, part[i]);
  if (threadIdx.x == 0) {
    scales[row] = scale_of(mx);
    if (zero_max != nullptr) zero_max[row] = 0;
  }
  const bool live = mx < 0x7f800000u && mx != 0;
  const float m = __uint_as_float(mx), inv = 127.0f / m;
  int8_t* const q = codes + row * ldc;
  auto code = [&](int c, V v) {
    if (c >= cols) return;
    Q o{};
    if (live) {
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = (int8_t)code_of(as_float(v[i]), m, inv);
    }
    if (WHOLE || c + N <= cols) {
      *(Q_any*)(q + c) = o;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + i < cols) q[c + i] = o[i];
    }
  };
#pragma unroll
  for (int j = 0; j < kQuantHeld; ++j) code(threadIdx.x * N + j * step, held[j]);
  for (int c = threadIdx.x * N + kQuantHeld * step; c < cols; c += step) code(c, read(c));
  for (int c = cols + threadIdx.x; c < (int)ldc; c += blockDim.x) q[c] = 0;
}

// Codes of fp32 rows whose maxima are known, 4 columns a thread: rows of ldx elements to
// rows of ldx codes, zero from cols on.
__global__ __launch_bounds__(256) void k_quantize_known(const float* __restrict__ x, int64_t ldx,
                                                        int rows, int cols,
                                                        const unsigned* __restrict__ row_max,
                                                        int8_t* __restrict__ codes,
                                                        float* __restrict__ scales) {
  typedef int8_t Q __attribute__((ext_vector_type(4)));
  const int c = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (c >= ldx) return;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const unsigned mx = row_max[row];
    if (c == 0) scales[row] = scale_of(mx);
    Q o{};
    if (mx < 0x7f800000u && mx != 0 && c < cols) {
      const f32x4 v = *(const f32x4*)(x + row * ldx + c);
      const float m = __uint_as_float(mx), inv = 127.0f / m;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < cols) o[i] = (int8_t)code_of(v[i], m, inv);
    }
    *(Q*)(codes + row * ldx + c) = o;
  }
}

template <typename T>
hipError_t launch_quantize_as(const T* x, int rows, int cols, int8_t* codes, int64_t ldc,
                              float* scales, unsigned* zero_max, hipStream_t s) {
  // Two vectors a thread: their latency overlaps, and short rows take few waves.
  constexpr int per = 2 * 16 / sizeof(T);
  const int threads = std::min(1024, std::max(64, (cols + per * 64 - 1) / (per * 64) * 64));
  // A launch holds fewer than 2^32 threads: 2^21 rows of 1024.
  constexpr int most = 1 << 21;
  for (int64_t at = 0; at < rows; at += most) {
    const int n = (int)std::min<int64_t>(most, rows - at);
    unsigned* const zero = zero_max == nullptr ? nullptr : zero_max + at;
    if (cols % (per / 2) == 0)
      k_quantize<T, true>
          <<<n, threads, 0, s>>>(x + at * cols, cols, codes + at * ldc, ldc, scales + at, zero);
    else
      k_quantize<T, false>
          <<<n, threads, 0, s>>>(x + at * cols, cols, codes + at * ldc, ldc, scales + at, zero);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

hipError_t launch_quantize(const void* x, int dtype, int rows, int cols, int8_t* codes, int64_t ldc,
                           float* scales, unsigned* zero_max, hipStream_t s) {
  if (rows == 0) return hipSuccess;
  if (dtype == WR_F32)
    return launch_quantize_as((const float*)x, rows, cols, codes, ldc, scales, zero_max, s);
  if (dtype == WR_F16)
    return launch_quantize_as((const f16*)x, rows, cols, codes, ldc, scales, zero_max, s);
  return launch_quantize_as((const __bf16*)x, rows, cols, codes, ldc, scales, zero_max, s);
}

hipError_t launch_quantize_known(const float* x, int64_t ldx, int rows, int cols,
                                 const unsigned* row_max, int8_t* codes, float* scales,
                                 hipStream_t s) {
  const dim3 grid((unsigned)((ldx + 1023) / 1024), (unsigned)std::min(rows, 65535));
  k_quantize_known<<<grid, 256, 0, s>>>(x, ldx, rows, cols, row_max, codes, scales);
  return hipGetLastError();
}

unsigned row_blocks(int64_t threads) {
  return (unsigned)std::min<int64_t>((threads + 255) / 256, 8192);
}

hipError_t launch_pads(const Pads& p, int es, hipStream_t s) {
  int64_t rows = 0;
  for (int i = 0; i < p.n; ++i) rows = std::max(rows, p.m[i].rows);
  if (rows == 0) return hipSuccess;
  const dim3 grid((unsigned)std::min<int64_t>((rows + 3) / 4, 4096), p.n);
  if (es == 4) k_pad_rows<uint32_t><<<grid, 256, 0, s>>>(p);
  else if (es == 2) k_pad_rows<uint16_t><<<grid, 256, 0, s>>>(p);
  else k_pad_rows<uint8_t><<<grid, 256, 0, s>>>(p);
  return hipGetLastError();
}

hipError_t launch_zero(void* p, int64_t bytes, hipStream_t s) {
  if (bytes == 0) return hipSuccess;
  const int64_t words = bytes / 4;
  k_fill_zero<<<std::max(1u, row_blocks(words)), 256, 0, s>>>(
      (uint32_t*)p, words, (char*)p + words * 4, (int)(bytes - words * 4));
  return hipGetLastError();
}

// ---- the choice of tiles --------------------------------------------------------
// Tiles are dealt to the CUs in rounds.  Those of the last round, which fills the CUs
// only in part, may be split over K into slices that fill it better and are
// shorter; their sums go through memory and a second, short kernel.  The shape and
// number of slices with the least estimated time are taken.
struct ShapeCost {
  int bm, bn, per_cu;  // tile, blocks a CU holds
  float step;          // us per 128 bytes of K, with per_cu blocks on the CU
  float alone;         // the same where a round leaves CUs free, or one block on each
  float fixed;         // us per tile: first copies, epilogue
};
// Measured on one MI355X (bf16; 16 times the clocks for fp32).  Tiles of 128 x 128 with 3
// buffers against 2: 64 x 4096 by 4096 x 14336 (112 tiles) 31 against 41 us, 4096 x
// 2816 by 2816 x 2048 (512 tiles) 55 against 44; against 256 x 256 at 2048 x 4096 by
// 4096 x 14336 207 and 183 us.  64 x 256 tiles were slower than the better 128 x 128 at
// every size measured.
constexpr ShapeCost kCost16[kShapes] = {{256, 256, 1, 1.37f, 1.37f, 5.0f},
                                        {128, 128, 2, 0.92f, 0.58f, 3.0f},
                                        {128, 128, 1, 0.55f, 0.45f, 3.0f}};
constexpr ShapeCost kCost32[kShapes] = {{256, 256, 1, 7.7f, 7.7f, 6.0f},
                                        {128, 128, 2, 4.0f, 2.2f, 4.0f},
                                        {128, 128, 1, 2.2f, 2.2f, 4.0f}};
constexpr int kCUs = 256;
constexpr int kMaxSlices = 32;
constexpr int64_t kMaxPartBytes = (int64_t)512 << 20;

struct Plan {
  int shape, slices, tiles_m, tiles_n, tiles, whole;
  size_t part_bytes;
};

// epi: bytes that the epilogue reads and writes per element of the tile; a CU moves about
// 20 KB a us.
float rounds_us(const ShapeCost& c, int64_t blocks, int steps, float epi) {
  const int64_t cap = (int64_t)kCUs * c.per_cu, rest = blocks % cap;
  const float move = epi * c.bm * c.bn / 20e3f;
  const float full = steps * c.step + c.fixed + move * c.per_cu;
  return blocks / cap * full +
         (rest == 0 ? 0.0f : rest <= kCUs ? steps * c.alone + c.fixed + move : full);
}

// Rows of m up to which a product of two K-contiguous operands goes to k_dense_rows, and,
// where a row is no whole 16-byte chunks, to k_dense_any.
constexpr int kRowsMax = 16, kAnyMax = 64;
// 32 rows of B a block where that leaves 2 blocks a CU, else 16; 8 waves a block
// where there are fewer blocks than CUs, else 4.
Plan plan_rows(int M, int N, int K, int es, bool gated, bool any) {
  const int64_t steps = ((int64_t)K * es + 127) / 128;
  const bool wide = !any && (N + (gated ? 15 : 31)) / (gated ? 16 : 32) >= 2 * kCUs;
  const int rows = (wide ? 32 : 16) / (gated ? 2 : 1), blocks = (N + rows - 1) / rows;
  const int tm = (M + 15) / 16, waves = blocks * tm < kCUs && steps >= 16 ? 8 : 4;
  return {any ? kRowsAny : wide ? kRows32 : kRows16, waves, tm, blocks, blocks * tm, blocks * tm, 0};
}

// M x N x K per problem; gated: N columns of each of two matrices; epi: see rounds_us;
// rows: the few-row kernels, any: for rows of any length.
Plan plan_of(int M, int N, int K, int es, int nseg, int nprob, bool gated, float epi, bool rows,
             bool any) {
  const int kb = 128 / es;
  const int steps = (K + kb - 1) / kb * nseg;
  if (rows) return plan_rows(M, N, K, es, gated, any);
  Plan best{};
  float best_us = 0;
  for (int shape = 0; shape < kShapes; ++shape) {
    const ShapeCost& c = es == 4 ? kCost32[shape] : kCost16[shape];
    const int64_t tm = (M + c.bm - 1) / c.bm, bn = gated ? c.bn / 2 : c.bn;
    const int64_t tn = (N + bn - 1) / bn, tiles = tm * tn * nprob;
    const int64_t cap = (int64_t)kCUs * c.per_cu, rest = tiles % cap;
    for (int S = 1; S <= kMaxSlices && S * 2 <= std::max(2, steps); ++S) {
      const int64_t whole = S == 1 ? tiles : tiles - rest;
      const int64_t part = (tiles - whole) * S * c.bm * c.bn * 4;
      if (S > 1 && (rest == 0 || part > kMaxPartBytes)) break;
      // The slices' sums are written like an epilogue; the join reads them (not those of rows
      // past M) and has the tiles' own epilogue.
      const float moved = (part + (tiles - whole) * c.bm * c.bn * epi) *
                          std::min(1.0f, (float)M / (tm * c.bm));
      const float us = rounds_us(c, whole, steps, epi) +
                       (S == 1 ? 0.0f
                               : rounds_us(c, rest * S, (steps + S - 1) / S, 4.0f) + 4.0f +
                                     moved / 5e6f);
      if (best.tiles == 0 || us < best_us) {
        best = {shape, S, (int)tm, (int)tn, (int)tiles, (int)whole, (size_t)part};
        best_us = us;
      }
    }
  }
  return best;
}

// ---- a call: workspace and launches from the same code --------------------------
// With `ws` null nothing is launched and `used` counts the workspace.
struct Call {
  char* ws;
  hipStream_t stream;
  int dtype;  // of the products' operands, unless int8
  bool int8;
  size_t used = 0, part_at = 0, part_bytes = 0;
  Pads pads{};
  hipError_t err = hipSuccess;

  bool dry() const { return ws == nullptr; }
  int es() const { return int8 ? 1 : elem_bytes(dtype); }
  char* take(int64_t bytes) {
    char* p = dry() ? nullptr : ws + used;
    used += align_up((size_t)bytes, kWsAlign);
    return p;
  }
  void check(hipError_t e) {
    if (err == hipSuccess) err = e;
  }
  bool go() const { return !dry() && err == hipSuccess; }

  // An operand matrix with whole 16-byte rows: itself, or a padded copy, which pad()
  // makes.  any_row: the product takes rows of any length.
  struct Mat {
    const char* p;
    int64_t ld;  // bytes
  };
  Mat rows16(const void* p, int64_t rows, int cols, bool any_row = false) {
    const int64_t bytes = (int64_t)cols * es(), ld = round_up(bytes, 16);
    if (any_row || ld == bytes) return {(const char*)p, bytes};
    char* c = take(rows * ld);
    pads.m[pads.n++] = {p, c, rows, ld, cols};
    return {c, ld};
  }
  void pad() {
    if (go() && pads.n > 0) check(launch_pads(pads, es(), stream));
  }

  // The slices' sums share one region (products of a call run one after another).
  void reserve_part(const Plan& pl) { part_bytes = std::max(part_bytes, pl.part_bytes); }

  void product(GemmArgs g, int form) {
    const bool gated = form == kFormGated || form == kFormGatedMax;
    if (g.M == 0 || g.N == 0) return;
    const bool any = g.lda % 16 != 0 || g.ldb % 16 != 0;
    const bool rows = (any || g.M <= kRowsMax) && form != kFormGateGrad && form != kFormKcKs &&
                      form != kFormKsKs;
    const int out = int8 ? 4 : es();  // int8: whatever the output's type, as the workspace
    const float epi = form == kFormGateGrad    ? 8.0f + 2 * out
                      : form == kFormGatedMax  ? 2.0f
                      : form != kFormGated     ? out
                      : g.out[1] != nullptr    ? out / 2 + 4
                                               : out / 2;
    const Plan pl = plan_of(g.M, g.N, g.K, es(), g.nseg, g.nprob, gated, epi, rows, any);
    reserve_part(pl);
    if (!go()) return;
    g.slices = pl.slices;
    g.tiles_m = pl.tiles_m;
    g.tiles_n = pl.tiles_n;
    g.tiles = pl.tiles;
    g.whole = pl.whole;
    g.part = ws + part_at;
    check(int8 ? launch_i8(g, pl.shape, form, stream)
          : dtype == WR_F32 ? launch_f32(g, pl.shape, form, stream)
          : dtype == WR_F16 ? launch_f16(g, pl.shape, form, stream)
                            : launch_bf16(g, pl.shape, form, stream));
  }
};

GemmArgs gemm(const Call::Mat& a, const Call::Mat& b, int M, int N, int K) {
  GemmArgs g{};
  g.a[0] = g.a[1] = a.p;
  g.b[0] = g.b[1] = b.p;
  g.lda = a.ld;
  g.ldb = b.ld;
  g.M = M;
  g.N = N;
  g.K = K;
  g.nseg = g.nprob = 1;
  return g;
}

void run_forward(Call& c, const wr_ffn_args& a) {
  const int T = a.batch_size, h = a.hidden_dim, I = a.intermediate_dim;
  const int64_t Ip = round_up(I, 64);
  const bool keep = a.saved_act != nullptr;
  const bool few = T <= kAnyMax;
  const Call::Mat x = c.rows16(a.x, T, h, few);
  const Call::Mat wg = c.rows16(a.w_gate, I, h, few), wu = c.rows16(a.w_up, I, h, few);
  const Call::Mat wd = c.rows16(a.w_down, h, I, few);
  c.pad();
  char* own = c.take((int64_t)T * Ip * c.es());  // sized whether saved or not
  const Call::Mat act{keep ? (const char*)a.saved_act : own, Ip * c.es()};

  GemmArgs g = gemm(x, wg, T, I, h);
  g.b[1] = wu.p;
  g.ldi = Ip;
  g.out[0] = const_cast<char*>(act.p);
  g.out[1] = a.saved_gate;
  g.out[2] = a.saved_up;
  c.product(g, kFormGated);

  g = gemm(act, wd, T, h, I);
  g.out[0] = a.out;
  g.ldo = h;
  c.product(g, kFormKcKc);
}

void run_backward(Call& c, const wr_ffn_args& a, bool dx, bool dwg, bool dwu, bool dwd) {
  const int T = a.batch_size, h = a.hidden_dim, I = a.intermediate_dim;
  const int64_t Ip = round_up(I, 64), ldi = Ip * c.es();
  const bool din = dx || dwg || dwu;
  const Call::Mat none{nullptr, 0};
  const Call::Mat dy = c.rows16(a.dout, T, h);
  const Call::Mat wd = din ? c.rows16(a.w_down, h, I) : none;
  const Call::Mat wg = dx ? c.rows16(a.w_gate, I, h) : none;
  const Call::Mat wu = dx ? c.rows16(a.w_up, I, h) : none;
  const Call::Mat x = dwg || dwu ? c.rows16(a.x, T, h) : none;
  c.pad();
  GemmArgs g;
  if (din) {
    char* dgate = c.take(T * ldi);
    char* dup = c.take(T * ldi);
    g = gemm(dy, wd, T, I, h);
    g.ldi = Ip;
    g.in[0] = a.saved_gate;
    g.in[1] = a.saved_up;
    g.out[0] = dgate;
    g.out[1] = dup;
    c.product(g, kFormGateGrad);
    if (dx) {
      g = gemm({dgate, ldi}, wg, T, h, I);
      g.a[1] = dup;
      g.b[1] = wu.p;
      g.nseg = 2;
      g.out[0] = a.dx;
      g.ldo = h;
      c.product(g, kFormKcKs);
    }
    if (dwg || dwu) {
      g = gemm({dwg ? dgate : dup, ldi}, x, I, h, T);
      g.a[1] = dup;
      g.nprob = dwg && dwu ? 2 : 1;
      g.out[0] = dwg ? a.dw_gate : a.dw_up;
      g.out[1] = a.dw_up;
      g.ldo = h;
      c.product(g, kFormKsKs);
    }
  }
  if (dwd) {
    g = gemm(dy, {(const char*)a.saved_act, ldi}, h, I, T);
    g.out[0] = a.dw_down;
    g.ldo = I;
    c.product(g, kFormKsKs);
  }
}

void run_int8(Call& c, const wr_int8_args& a) {
  const bool few = a.rows <= kAnyMax;
  const Call::Mat x = c.rows16(a.x, a.rows, a.in_features, few);
  const Call::Mat w = c.rows16(a.w, a.out_features, a.in_features, few);
  c.pad();
  GemmArgs g = gemm(x, w, a.rows, a.out_features, a.in_features);
  g.out[0] = a.out;
  g.ldo = a.out_features;
  g.out_dtype = a.out_dtype;
  g.row_scale = a.x_scale;
  g.col_scale[0] = a.w_scale;
  c.product(g, kFormScale);
}

void run_ffn_int8(Call& c, const wr_ffn_int8_args& a) {
  const int T = a.batch_size, h = a.hidden_dim, I = a.intermediate_dim;
  const int64_t Ip = round_up(I, 64), hp = round_up(h, 16);
  int8_t* xq = (int8_t*)c.take(T * hp);
  float* sx = (float*)c.take((int64_t)T * 4);
  unsigned* amax = (unsigned*)c.take((int64_t)T * 4);
  float* act = (float*)c.take(T * Ip * 4);
  int8_t* aq = (int8_t*)c.take(T * Ip);
  float* sa = (float*)c.take((int64_t)T * 4);
  const bool few = T <= kAnyMax;
  const Call::Mat wg = c.rows16(a.w_gate, I, h, few), wu = c.rows16(a.w_up, I, h, few);
  const Call::Mat wd = c.rows16(a.w_down, h, I, few);
  c.pad();
  if (c.go())
    c.check(launch_quantize(a.x, a.dtype, T, h, xq, hp, sx, amax, c.stream));
  GemmArgs g = gemm({(const char*)xq, hp}, wg, T, I, h);
  g.b[1] = wu.p;
  g.ldi = Ip;
  g.out[0] = act;
  g.row_scale = sx;
  g.col_scale[0] = a.s_gate;
  g.col_scale[1] = a.s_up;
  g.row_max = amax;
  c.product(g, kFormGatedMax);
  if (c.go())
    c.check(launch_quantize_known(act, Ip, T, I, amax, aq, sa, c.stream));
  g = gemm({(const char*)aq, Ip}, wd, T, h, I);
  g.out[0] = a.out;
  g.ldo = h;
  g.out_dtype = a.dtype;
  g.row_scale = sa;
  g.col_scale[0] = a.s_down;
  c.product(g, kFormScale);
}

// Runs `body` once dry for the workspace's size, then for real.  The slices' sums lie
// behind everything else.
template <typename Body>
size_t workspace_of(int dtype, bool int8, Body body) {
  Call c{nullptr, nullptr, dtype, int8};
  body(c);
  return std::max<size_t>(kWsAlign, c.used + c.part_bytes);
}

template <typename Body>
int run(int dtype, bool int8, void* ws, size_t ws_bytes, void* stream, Body body) {
  Call c{nullptr, nullptr, dtype, int8};
  body(c);
  if (ws == nullptr || ws_bytes < std::max<size_t>(kWsAlign, c.used + c.part_bytes))
    return WR_EINVAL_WORKSPACE;
  Call r{(char*)ws, (hipStream_t)stream, dtype, int8};
  r.part_at = c.used;
  body(r);
  return r.err == hipSuccess ? WR_OK : WR_EHIP;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_ffn(const wr_ffn_args* a) {
  if (a == nullptr) return WR_EINVAL_NULL;
  if (!float_dtype(a->dtype)) return WR_EINVAL_DTYPE;
  if (a->hidden_dim < 1 || a->intermediate_dim < 1 || a->hidden_dim > WR_FFN_MAX_DIM ||
      a->intermediate_dim > WR_FFN_MAX_DIM)
    return WR_EINVAL_SHAPE;
  if (a->batch_size < 0 || a->batch_size > WR_FFN_MAX_ROWS) return WR_EINVAL_BATCH;
  for (const void* p : {a->x, a->w_gate, a->w_up, a->w_down, (const void*)a->workspace,
                        (const void*)a->saved_gate, (const void*)a->saved_up,
                        (const void*)a->saved_act})
    if (!aligned(p)) return WR_EINVAL_ALIGN;
  return WR_OK;
}

}  // namespace
}  // namespace ffn
}  // namespace wr

using namespace wr::ffn;

extern "C" {

int64_t wr_ffn_saved_row(int I) { return I < 1 || I > WR_FFN_MAX_DIM ? 0 : round_up(I, 64); }

size_t wr_ffn_workspace_bytes(int backward, int dtype, int h, int I, int T) {
  wr_ffn_args a{};
  a.dtype = dtype;
  a.hidden_dim = h;
  a.intermediate_dim = I;
  a.batch_size = T;
  if (check_ffn(&a) != WR_OK) return 0;
  // The most that any call of these sizes takes: tiles and slices are chosen for what is
  // kept (forward; the pointers are only compared) and needed (backward: one weight
  // gradient alone has fewer tiles to share, and may be split more).
  size_t most = 0;
  for (const bool alone : {false, true}) {
    if (alone) a.saved_gate = a.saved_up = reinterpret_cast<float*>(a.saved_act = &a);
    most = std::max(most, workspace_of(dtype, false, [&](Call& c) {
                      if (backward)
                        run_backward(c, a, true, true, !alone, true);
                      else
                        run_forward(c, a);
                    }));
  }
  return most;
}

int wr_ffn_forward(const wr_ffn_args* a, void* stream) {
  if (const int st = check_ffn(a)) return st;
  if (a->batch_size == 0) return WR_OK;
  if (!a->x || !a->w_gate || !a->w_up || !a->w_down || !a->out) return WR_EINVAL_NULL;
  const int kept = (a->saved_gate != nullptr) + (a->saved_up != nullptr) + (a->saved_act != nullptr);
  if (kept != 0 && kept != 3) return WR_EINVAL_NULL;
  if (!aligned(a->out)) return WR_EINVAL_ALIGN;
  return run(a->dtype, false, a->workspace, a->workspace_bytes, stream,
             [&](Call& c) { run_forward(c, *a); });
}

int wr_ffn_backward(const wr_ffn_args* a, void* stream) {
  if (const int st = check_ffn(a)) return st;
  for (const void* p : {a->dout, (const void*)a->dx, (const void*)a->dw_gate,
                        (const void*)a->dw_up, (const void*)a->dw_down})
    if (!aligned(p)) return WR_EINVAL_ALIGN;
  const bool dx = a->dx != nullptr, dwg = a->dw_gate != nullptr, dwu = a->dw_up != nullptr,
             dwd = a->dw_down != nullptr;
  if (a->batch_size == 0) {  // no tokens: the weights' gradients are zero
    const int64_t n = (int64_t)a->hidden_dim * a->intermediate_dim *
                      wr::ffn::elem_bytes(a->dtype);
    for (void* p : {a->dw_gate, a->dw_up, a->dw_down})
      if (p != nullptr && launch_zero(p, n, (hipStream_t)stream) != hipSuccess) return WR_EHIP;
    return WR_OK;
  }
  if (!a->dout || ((dwg || dwu) && !a->x) || (dx && (!a->w_gate || !a->w_up)) ||
      ((dx || dwg || dwu) && (!a->w_down || !a->saved_gate || !a->saved_up)) ||
      (dwd && !a->saved_act))
    return WR_EINVAL_NULL;
  return run(a->dtype, false, a->workspace, a->workspace_bytes, stream,
             [&](Call& c) { run_backward(c, *a, dx, dwg, dwu, dwd); });
}

int wr_quantize_int8(const void* x, int dtype, int rows, int cols, int8_t* codes, float* scales,
                     void* stream) {
  if (!float_dtype(dtype)) return WR_EINVAL_DTYPE;
  if (rows < 0 || rows > WR_FFN_MAX_ROWS) return WR_EINVAL_BATCH;
  if (cols < 1 || cols > WR_INT8_MAX_COLS) return WR_EINVAL_SHAPE;
  if (rows == 0) return WR_OK;
  if (!x || !codes || !scales) return WR_EINVAL_NULL;
  if (!aligned(x) || !aligned(codes) || !aligned(scales)) return WR_EINVAL_ALIGN;
  return launch_quantize(x, dtype, rows, cols, codes, cols, scales, nullptr,
                         (hipStream_t)stream) == hipSuccess
             ? WR_OK
             : WR_EHIP;
}

static int check_int8(const wr_int8_args* a) {
  if (a == nullptr) return WR_EINVAL_NULL;
  if (!float_dtype(a->out_dtype)) return WR_EINVAL_DTYPE;
  if (a->out_features < 1 || a->in_features < 1 || a->out_features > WR_FFN_MAX_DIM ||
      a->in_features > WR_INT8_MAX_K)
    return WR_EINVAL_SHAPE;
  if (a->rows < 0 || a->rows > WR_FFN_MAX_ROWS) return WR_EINVAL_BATCH;
  return WR_OK;
}

size_t wr_int8_workspace_bytes(int rows, int out_features, int in_features) {
  wr_int8_args a{};
  a.rows = rows;
  a.out_features = out_features;
  a.in_features = in_features;
  if (check_int8(&a) != WR_OK) return 0;
  return workspace_of(WR_F32, true, [&](Call& c) { run_int8(c, a); });
}

int wr_int8_matmul(const wr_int8_args* a, void* stream) {
  if (const int st = check_int8(a)) return st;
  if (a->rows == 0) return WR_OK;
  if (!a->x || !a->x_scale || !a->w || !a->w_scale || !a->out) return WR_EINVAL_NULL;
  for (const void* p : {(const void*)a->x, (const void*)a->w, (const void*)a->out,
                        (const void*)a->workspace})
    if (!aligned(p)) return WR_EINVAL_ALIGN;
  return run(WR_F32, true, a->workspace, a->workspace_bytes, stream,
             [&](Call& c) { run_int8(c, *a); });
}

static int check_ffn_int8(const wr_ffn_int8_args* a) {
  if (a == nullptr) return WR_EINVAL_NULL;
  if (!float_dtype(a->dtype)) return WR_EINVAL_DTYPE;
  if (a->hidden_dim < 1 || a->intermediate_dim < 1 || a->hidden_dim > WR_INT8_MAX_K ||
      a->intermediate_dim > WR_INT8_MAX_K)
    return WR_EINVAL_SHAPE;
  if (a->batch_size < 0 || a->batch_size > WR_FFN_MAX_ROWS) return WR_EINVAL_BATCH;
  return WR_OK;
}

size_t wr_ffn_int8_workspace_bytes(int h, int I, int T) {
  wr_ffn_int8_args a{};
  a.hidden_dim = h;
  a.intermediate_dim = I;
  a.batch_size = T;
  if (check_ffn_int8(&a) != WR_OK) return 0;
  return workspace_of(WR_F32, true, [&](Call& c) { run_ffn_int8(c, a); });
}

int wr_ffn_int8(const wr_ffn_int8_args* a, void* stream) {
  if (const int st = check_ffn_int8(a)) return st;
  if (a->batch_size == 0) return WR_OK;
  if (!a->x || !a->w_gate || !a->s_gate || !a->w_up || !a->s_up || !a->w_down || !a->s_down ||
      !a->out)
    return WR_EINVAL_NULL;
  for (const void* p : {(const void*)a->x, (const void*)a->w_gate, (const void*)a->w_up,
                        (const void*)a->w_down, (const void*)a->out, (const void*)a->workspace})
    if (!aligned(p)) return WR_EINVAL_ALIGN;
  return run(a->dtype, true, a->workspace, a->workspace_bytes, stream,
             [&](Call& c) { run_ffn_int8(c, *a); });
}

}  // extern "C"
