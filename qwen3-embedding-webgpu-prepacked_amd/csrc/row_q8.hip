// row_q8.hip -- rows of 16-bit elements into 8-bit codes with one scale each: as they are, or as the RMSNorm of a
// residual sum.
//
//   v = x + r (f32), x' = v rounded to the type, inv = 1 / sqrt(sum(v^2) / width + eps)
//   t = x' * weight, amax = max |t|, code = rint(t * (127 / amax)), scale = amax / 127 * inv
//
// The norm's factor inv is one number for a row, so it cancels in the codes and stands in the scale alone.  The
// sum of squares and the largest value then take one reduction between them, the row is read once and stays in
// registers, and the codes do not depend on the order in which a sum is formed.  Memory bounds it: 8,000 x 1,024 with
// a residual 11.1 us, 5.2 TB/s, 8,000 x 2,048 without the norm 9.0 us, 5.5 TB/s; a few rows take a launch.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "elem.h"
#include "w4_ops.h"

namespace qattn {
namespace {

// Codes of 8 values, four to a dword.  Adding 1.5 * 2^23 rounds a value to a whole number, ties to even, in the
// low byte; the product is rounded to f32 before (contraction would round once).
__device__ inline u32x2 codes8(const float* t, float factor) {
#pragma clang fp contract(off)
  uint32_t c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = __float_as_uint(t[e] * factor + 12582912.f);
  const auto pack = [](uint32_t a, uint32_t b, uint32_t p, uint32_t q) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0400u), hi = __builtin_amdgcn_perm(q, p, 0x04000C0Cu);
    return lo | hi;
  };
  return u32x2{pack(c[0], c[1], c[2], c[3]), pack(c[4], c[5], c[6], c[7])};
}

// A row of bf16 may be so small that its squares leave f32's range: their sum would be 0 and, with an eps of 0, the scale
// infinite.  So below kTinyEps the squares of the values times 2^100 are summed as well, which none leaves downwards.
// That sum counts where the plain one is below kTinySquares, and then stays in range itself; elsewhere what the plain
// one has lost, 2^-150 for a value, is nothing beside kTinySquares or eps.
constexpr float kTinyEps = 0x1p-100f, kTinySquares = 0x1p-80f;

// T threads to a row, C pieces of 8 elements to a thread; memory is the bound.  Up to 512 elements a row takes as many
// lanes as it fills, so that a wavefront holds several narrow ones, and up to 2048 one wavefront, which needs no
// barrier; more take as many threads as leave two pieces to each, for more loads in flight.
template <bool BF16, bool NORM, bool SUM, int T, int C>
__global__ __launch_bounds__(T < 256 ? 256 : T) void row_q8_kernel(RowQ8 p) {
  constexpr int kRows = T < 256 ? 256 / T : 1, kWaves = T / 64;
  static_assert(T <= 64 || T >= 256, "rows that share a workgroup are within a wavefront each");
  const int tid = threadIdx.x % T;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kRows + threadIdx.x / T;
  if (row >= p.rows) return;  // T > 64: one row to a workgroup, so this is uniform; else the T lanes leave together
  const uint16_t* const x = static_cast<const uint16_t*>(p.x) + row * p.x_stride;
  u32x4 a[C], r[C];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int c = 8 * (tid + T * j);
    a[j] = c < p.width ? *reinterpret_cast<const u32x4*>(x + c) : u32x4{};
    if constexpr (SUM)
      r[j] = c < p.width ? *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.residual) + row * p.residual_stride + c)
                         : u32x4{};
  }
  float t[8 * C];
  float squares = 0.f, raised = 0.f;
  const bool tiny_eps = BF16 && NORM && p.eps < kTinyEps;
  uint32_t most = 0;  // the largest magnitude's bits: NaN above infinity above every number
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int c = 8 * (tid + T * j);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = widen<BF16, 0>(a[j][i]);
      v[2 * i + 1] = widen<BF16, 1>(a[j][i]);
      if constexpr (SUM) {
        v[2 * i] += widen<BF16, 0>(r[j][i]);
        v[2 * i + 1] += widen<BF16, 1>(r[j][i]);
      }
    }
    if constexpr (NORM) {
#pragma unroll
      for (int e = 0; e < 8; ++e) squares = fmaf(v[e], v[e], squares);
      if (tiny_eps)
#pragma unroll
        for (int e = 0; e < 8; ++e) raised = fmaf(v[e] * 0x1p100f, v[e] * 0x1p100f, raised);
    }
    if constexpr (SUM) {
      u32x4 s;
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = narrow2<BF16>(v[2 * i], v[2 * i + 1]);
      if (c < p.width) *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.sum) + row * p.sum_stride + c) = s;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = widen<BF16, 0>(s[i]);
        v[2 * i + 1] = widen<BF16, 1>(s[i]);
      }
    }
    if constexpr (NORM) {
      float4 w[2] = {};
      if (c < p.width) {
        w[0] = *reinterpret_cast<const float4*>(p.weight + c);
        w[1] = *reinterpret_cast<const float4*>(p.weight + c + 4);
      }
      const float g[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= g[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t[8 * j + e] = v[e];
      most = max(most, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    }
  }
#pragma unroll
  for (int d = T < 64 ? T / 2 : 32; d; d >>= 1) {
    if constexpr (NORM) squares += __shfl_xor(squares, d, 64);
    if (tiny_eps) raised += __shfl_xor(raised, d, 64);
    most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
  }
  if constexpr (kWaves > 1) {
    __shared__ float part_squares[kWaves], part_raised[kWaves];
    __shared__ uint32_t part_most[kWaves];
    if ((tid & 63) == 0) {
      part_squares[tid >> 6] = squares;
      part_raised[tid >> 6] = raised;
      part_most[tid >> 6] = most;
    }
    __syncthreads();
    squares = part_squares[0];
    raised = part_raised[0];
    most = part_most[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
      squares += part_squares[i];
      raised += part_raised[i];
      most = max(most, part_most[i]);
    }
  }
  // A row with an infinity or a NaN, or whose squares pass f32's range: codes of zero, a scale of NaN.  A row of
  // next to nothing: zeros, with a scale of zero.
  const float amax = __uint_as_float(most);
  const bool lost = most >= 0x7F800000u || (NORM && !(squares < INFINITY)), none = amax < kLeastAmax;
  const float factor = lost || none ? 0.f : 127.f / amax;
  if (tid == 0) {
    float scale = amax / 127.f;
    if (tiny_eps && squares < kTinySquares)
      scale = (float)((double)scale / sqrt((double)raised * 0x1p-200 / p.width + (double)p.eps));
    else if constexpr (NORM)
      scale *= 1.f / sqrtf(squares / (float)p.width + p.eps);
    p.scales[row] = lost ? __builtin_nanf("") : none ? 0.f : scale;
  }
  int8_t* const out = p.codes + row * p.codes_stride;
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int c = 8 * (tid + T * j);
    if (c < p.width) *reinterpret_cast<u32x2*>(out + c) = lost ? u32x2{} : codes8(t + 8 * j, factor);
  }
}

template <bool BF16, bool NORM, bool SUM>
void launch(const RowQ8& p, hipStream_t stream) {
  // A dimension of a grid has to stay below 2^32 threads.
  const auto grid = [&](int rows) {
    const int64_t groups = (p.rows + rows - 1) / rows, x = groups < (1 << 20) ? groups : 1 << 20;
    return dim3((unsigned)x, (unsigned)((groups + x - 1) / x));
  };
#define ROW_Q8(T, C) \
  hipLaunchKernelGGL((row_q8_kernel<BF16, NORM, SUM, T, C>), grid(T < 256 ? 256 / T : 1), dim3(T < 256 ? 256 : T), 0, stream, p)
  // Microseconds on one MI355X over four sets of rows in turn, fp16 with a residual's sum where not said otherwise, the
  // variant taken and others: 20,000 x 64 5.5, a wavefront to a row 9.2; 20,000 x 256 8.5 and 10.7; 20,000 x 512 15.5, half
  // a wavefront 15.0; 8,000 x 1,024 11.1, half a wavefront the same, 256 threads 13.0; 2,048 wide without the norm 9.0
  // for 8,000, 256 threads 10.1, and with the sum, which does not decide, 7.5 and 7.6 for 2,000, 24.8 and 24.0 for 8,000, 52.2
  // either way for 20,000; 1,419 x 2,560 without the sum 5.2, four pieces 5.7, one 5.3; 2,000 x 5,000 15.4, four 18.1, one
  // 16.6; 500 x 16,384 11.4, four 15.2.
  if (p.width <= 64)
    ROW_Q8(8, 1);
  else if (p.width <= 128)
    ROW_Q8(16, 1);
  else if (p.width <= 256)
    ROW_Q8(32, 1);
  else if (p.width <= 512)
    ROW_Q8(64, 1);
  else if (p.width <= 1024)
    ROW_Q8(64, 2);
  else if (p.width <= 2048)
    ROW_Q8(64, 4);
  else if (p.width <= 4096)
    ROW_Q8(256, 2);
  else if (p.width <= 8192)
    ROW_Q8(512, 2);
  else if (p.width <= 16384)
    ROW_Q8(1024, 2);
  else
    ROW_Q8(1024, 4);
#undef ROW_Q8
}

}  // namespace

hipError_t launch_row_q8(const RowQ8& p, bool bf16, hipStream_t stream) {
  if (p.rows <= 0) return hipSuccess;
  const int kind = p.weight ? (p.residual ? 2 : 1) : 0;
  if (bf16)
    kind == 2 ? launch<true, true, true>(p, stream) : kind == 1 ? launch<true, true, false>(p, stream) : launch<true, false, false>(p, stream);
  else
    kind == 2 ? launch<false, true, true>(p, stream) : kind == 1 ? launch<false, true, false>(p, stream) : launch<false, false, false>(p, stream);
  return hipGetLastError();
}

}  // namespace qattn
