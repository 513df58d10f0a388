// Interface between the dense FFN's host side (wr_ffn.hip) and its product
// kernels (wr_ffn_gemm.h, one translation unit per element type).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace wr {
namespace ffn {

enum Epi {
  kStore,      // out[prob][m][n]
  kGated,      // out[0] = silu(g) u, and out[1] = g, out[2] = u (fp32) when set; ldi rows
  kGateGrad,   // out[0] = dg, out[1] = du from in[0] = g, in[1] = u (fp32); ldi rows
  kScale,      // int8: out[0] = sum * row_scale[m] * col_scale[0][n], of out_dtype
  kGatedMax,   // int8: out[0] = silu(g) u in fp32, ldi rows; row_max[m] = max |.|
};

// One product (or two of equal shape).  Bytes unless named otherwise.
struct GemmArgs {
  const char* a[2];  // per problem, or per K segment
  const char* b[2];  // per K segment; gated: gate and up matrix
  int64_t lda, ldb;  // bytes between rows of m, n (K-contiguous) or of k (K-strided)
  int M, N, K;       // K of one segment; gated: N of one matrix
  int nseg, nprob;
  int tiles_m, tiles_n, tiles;  // tiles: of all problems
  int whole, slices;  // tiles from `whole` on are split over K into `slices` blocks each
  void* out[3];
  const void* in[2];
  int64_t ldo, ldi;  // elements
  void* part;  // [tile - whole][slice]: the sums as they lie in the registers
  const float* row_scale;
  const float* col_scale[2];
  unsigned* row_max;
  int out_dtype;
};

// Tile shapes (m x n; gated products: n / 2 columns of each matrix): 256 x 256, 128 x 128,
// and 128 x 128 with a deeper ring, one block a CU.
enum Shape { kTile256, kTile128, kTile128Deep, kShapes,
             // few rows: `tiles` blocks of `slices` waves over 16 or 32 rows of B
             kRows16 = kShapes, kRows32, kRowsAny };

// Operand layouts and epilogue of a product.
enum Form { kFormGated, kFormKcKc, kFormGateGrad, kFormKcKs, kFormKsKs, kFormScale, kFormGatedMax };

hipError_t launch_f32(const GemmArgs& g, int shape, int form, hipStream_t s);
hipError_t launch_f16(const GemmArgs& g, int shape, int form, hipStream_t s);
hipError_t launch_bf16(const GemmArgs& g, int shape, int form, hipStream_t s);
hipError_t launch_i8(const GemmArgs& g, int shape, int form, hipStream_t s);

struct TileId {
  int prob, m, n;
  int tail, slice;  // tail < 0: a whole tile
};

// Tile i of the order: within a problem 8 m tiles advance together along n, for both
// operands' reuse in the L2 of the XCD that runs them.
__device__ __forceinline__ TileId tile_at(const GemmArgs& g, int i) {
  const int per = g.tiles_m * g.tiles_n;
  TileId t;
  t.prob = i / per;
  i -= t.prob * per;
  constexpr int kGroup = 8;
  const int first = i / (kGroup * g.tiles_n) * kGroup;
  const int rows = g.tiles_m - first < kGroup ? g.tiles_m - first : kGroup;
  i -= first * g.tiles_n;
  t.m = first + i % rows;
  t.n = i / rows;
  t.tail = -1;
  t.slice = 0;
  return t;
}

// Consecutive blocks go to the 8 XCDs in turn: each XCD takes one run of n places.
__device__ __forceinline__ int xcd_run(int block, int n) {
  const int x = block % 8, rem = n % 8;
  return x * (n / 8) + (x < rem ? x : rem) + block / 8;
}

// The whole tiles first, then the slices of the others, one slice of all of them
// after another.
__device__ __forceinline__ TileId tile_of(const GemmArgs& g, int block) {
  if (block < g.whole) return tile_at(g, xcd_run(block, g.whole));
  const int tail = g.tiles - g.whole;
  const int i = xcd_run(block - g.whole, tail * g.slices);
  TileId t = tile_at(g, g.whole + i % tail);
  t.tail = i % tail;
  t.slice = i / tail;
  return t;
}

}  // namespace ffn
}  // namespace wr
