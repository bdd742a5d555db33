// w4_ops.h -- the operators of a forward with 8-bit activations: launchers of the row kernels (row_q8.hip) and
// of the products with 4-bit weights (w4_matmul.hip), and the weights' layout, which the host writes
// (w4_weights.cpp) and the kernels read.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qattn {

constexpr int kQ8MaxWidth = 32768;
constexpr int kW4MaxK = 65536;        // |x| <= 128, |w| <= 128: every sum stays below 2^30
constexpr int kW4MaxN = 1 << 22;
constexpr int64_t kW4MaxStride = 1 << 22;  // elements; 256 rows of it stay within 32-bit byte offsets

// The image of an N x K weight: tiles of 16 rows, blocks of 128 columns (both padded with zero weights).
//   codes   [tiles][blocks] of 1 KiB: record (g, n) of 16 bytes at 256 g + 16 n holds the 32 columns of group g of
//           row n, column j < 16 in the low nibble of byte j, column j + 16 in its high nibble
//   groups  [tiles][blocks] of 64 bytes: at 4 n + g, the multiplier in the low nibble, the zero point in the high
//   scales  [tiles][16] f32
// So the 64 records of a block are the 64 lanes of a wavefront in turn: lane (n, g) loads 16 bytes, and its two
// halves are two operands of a 16x16x64 product.
struct W4Layout {
  int64_t tiles, blocks;
  __host__ __device__ W4Layout(int K, int N) : tiles((N + 15) / 16), blocks((K + 127) / 128) {}
  __host__ __device__ int64_t groups_at() const { return tiles * blocks * 1024; }
  __host__ __device__ int64_t scales_at() const { return tiles * blocks * 1088; }
  __host__ __device__ int64_t bytes() const { return scales_at() + tiles * 64; }
};

struct RowQ8 {
  const void* x;
  const void* residual;  // NULL: none
  void* sum;             // x + residual
  const float* weight;   // NULL: no norm
  int8_t* codes;
  float* scales;
  int64_t x_stride, residual_stride, sum_stride, codes_stride;
  int64_t rows;
  int32_t width;
  float eps;
};
hipError_t launch_row_q8(const RowQ8& p, bool bf16, hipStream_t stream);

struct W4Product {
  const int8_t* x;
  const float* x_scale;
  const uint8_t* w;
  void* y;
  int64_t ldx, ldy;
  int32_t M, K, N;  // N: rows of the weight (SwiGLU: gate rows, then up rows)
};
hipError_t launch_w4(const W4Product& p, bool bf16, bool swiglu, hipStream_t stream);

}  // namespace qattn
