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
  kPart,       // part[slice][prob][m][n], rows ldp
  kPartGated,  // part[slice][m][2][ldp]: gate sums, then up sums
};

// One product (or two of equal shape).  Bytes unless named otherwise.
struct GemmArgs {
  const char* a[2];  // per problem, or per K segment
  const char* b[2];  // per K segment; gated: gate and up matrix
  int64_t lda, ldb;  // bytes between rows of m, n (K-contiguous) or of k (K-strided)
  int M, N, K;       // K of one segment; gated: N of one matrix
  int nseg, nprob, slices;
  int tiles_m, tiles_n;
  void* out[3];
  const void* in[2];
  int64_t ldo, ldi, ldp;  // elements
  void* part;
  const float* row_scale;
  const float* col_scale[2];
  unsigned* row_max;
  int out_dtype;
  bool vec;  // out rows and pointer are 16-byte aligned
};

// Tile shapes (m x n; gated products: n / 2 columns of each matrix).
enum Shape { kTile256, kTile128, kTile64, kShapes };  // 256 x 256, 128 x 128, 64 x 256

// Operand layouts and epilogue of a product.
enum Form { kFormGated, kFormKcKc, kFormGateGrad, kFormKcKs, kFormKsKs, kFormScale, kFormGatedMax };

hipError_t launch_f32(const GemmArgs& g, int shape, int form, hipStream_t s);
hipError_t launch_f16(const GemmArgs& g, int shape, int form, hipStream_t s);
hipError_t launch_bf16(const GemmArgs& g, int shape, int form, hipStream_t s);
hipError_t launch_i8(const GemmArgs& g, int shape, int form, hipStream_t s);

struct TileId {
  int slice, prob, m, n;
};

// XCD-aware order of the blocks (see k_dense).
__device__ __forceinline__ TileId tile_of(const GemmArgs& g, int block, int blocks) {
  const int x = block % 8, q = blocks / 8, rem = blocks % 8;
  int i = x * q + (x < rem ? x : rem) + block / 8;
  const int tiles = g.tiles_m * g.tiles_n;
  TileId t;
  t.slice = i / (tiles * g.nprob);
  i -= t.slice * tiles * g.nprob;
  t.prob = i / tiles;
  i -= t.prob * tiles;
  constexpr int kGroup = 8;
  const int group = i / (kGroup * g.tiles_n);
  const int first = group * kGroup;
  const int rows = g.tiles_m - first < kGroup ? g.tiles_m - first : kGroup;
  i -= first * g.tiles_n;
  t.m = first + i % rows;
  t.n = i / rows;
  return t;
}

}  // namespace ffn
}  // namespace wr
