// w4_matmul.hip -- products of 8-bit rows with 4-bit weights: y[m][n] = x_scale[m] * w_scale[n] * sum_k x[m][k] *
// (code[n][k] - zero[n][k / 32]) * multiplier[n][k / 32], and SwiGLU of two such products.
//
// A group's scale is a whole number, so it goes into the 8-bit weight and the sum over all of K runs in whole
// numbers on the matrix cores (v_mfma_i32_16x16x64_i8, twice the rate of the 16-bit form); the two f32 scales meet
// it once, at the end.  With an f32 scale for each group every 16 x 16 sum would have to leave the matrix cores at
// each group: 8 vector instructions for 8 clocks of matrix work.  Whole-number sums are exact in any order, so K is
// split and joined as suits a launch and a row's result does not depend on its batch.
//
// Four weights cost three vector instructions and half a shift: nibbles to bytes, byte * multiplier + (128 - zero *
// multiplier) in two 16-bit halves -- neither byte leaves [0, 255], so none carries -- and the top bit flipped.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "elem.h"
#include "w4_ops.h"

namespace qattn {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

#define W4_INLINE __attribute__((always_inline))

// The memory and matrix builtins behind plain (non-template) device functions: hipcc's host pass drops a kernel
// template's host stub when such a builtin sits in a dependent context.
__device__ inline __amdgpu_buffer_rsrc_t rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}
// The range check covers the per-lane offset, not a scalar one: what may lie past a row's end goes into the former.
__device__ inline i32x4 load16(__amdgpu_buffer_rsrc_t rs, uint32_t off) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
}
__device__ inline i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// A group's multiplier in both halves of a dword, and 128 - zero * multiplier in its four bytes.
struct Group {
  uint32_t mult, bias;
};
__device__ inline Group group_of(uint32_t byte) {
  const uint32_t m = byte & 15u, z = byte >> 4 & 15u;
  return {m * 0x00010001u, (128u - m * z) * 0x01010101u};
}
__device__ inline uint32_t weights4(uint32_t nibbles, Group g) {
  const u16x2 v = __builtin_bit_cast(u16x2, nibbles) * __builtin_bit_cast(u16x2, g.mult) + __builtin_bit_cast(u16x2, g.bias);
  return __builtin_bit_cast(uint32_t, v) ^ 0x80808080u;
}
// The 16 weights of a record's low (HIGH = 0) or high nibbles.
template <int HIGH>
__device__ inline i32x4 weights16(i32x4 record, Group g) {
  i32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (int)weights4((uint32_t)record[i] >> (4 * HIGH) & 0x0F0F0F0Fu, g);
  return w;
}

// silu(g) * u.  The hardware's exp2 and reciprocal are within about an f32 ulp, far inside the result's rounding.
__device__ inline float swiglu(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504f)) * u;
}

// ---- few rows: a workgroup to 16 MB rows and 16 NB columns (SwiGLU: 8 NB features), its W wavefronts take the
// blocks of 128 columns of K in turn and add up in LDS.  No operand is staged: a lane's 16 bytes of codes are two
// fragments, and its 32 bytes of x the two that meet them.
template <bool BF16, bool SWIGLU, int MB, int NB, int W>
__global__ __launch_bounds__(64 * W) void w4_small_kernel(W4Product p, int blocks_m) {
  __shared__ i32x4 part[W > 1 ? W - 1 : 1][MB * NB][64];
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m0 = (int64_t)(blockIdx.x % (unsigned)blocks_m) * (16 * MB);
  const int nblk = (int)(blockIdx.x / (unsigned)blocks_m);
  const W4Layout at(p.K, p.N);
  const int blocks = (int)at.blocks;
  // Tiles of 16 weight rows: the gate's, then the up projection's.
  const int tile0 = SWIGLU ? NB / 2 * nblk : NB * nblk;
  const int last = (int)at.tiles - 1;
  const uint8_t *codes[NB], *groups[NB];
  int tile[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    tile[nb] = SWIGLU ? tile0 + nb % (NB / 2) + (nb < NB / 2 ? 0 : p.N >> 5) : tile0 + nb;
    const int t = tile[nb] < last ? tile[nb] : last;  // past the last tile: read it again, store nothing
    codes[nb] = p.w + (int64_t)t * blocks * 1024;
    groups[nb] = p.w + at.groups_at() + (int64_t)t * blocks * 64;
  }
  // Rows past M and what lies behind the last row's K columns read as zeros; columns of K's padding meet zero weights.
  const int rows = (int)(p.M - m0 < 16 * MB ? p.M - m0 : 16 * MB);
  const auto xs = rsrc(p.x + m0 * p.ldx, (uint32_t)(rows - 1) * (uint32_t)p.ldx + (uint32_t)p.K);
  uint32_t x_off[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) x_off[mb] = (uint32_t)(16 * mb + l16) * (uint32_t)p.ldx + 32u * q;

  i32x4 acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB * MB; ++i) acc[i / MB][i % MB] = i32x4{};
  for (int kb = wave; kb < blocks; kb += W) {
    i32x4 x[MB][2];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      x[mb][0] = load16(xs, x_off[mb] + 128u * kb);
      x[mb][1] = load16(xs, x_off[mb] + 128u * kb + 16u);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const i32x4 record = *reinterpret_cast<const i32x4*>(codes[nb] + (int64_t)kb * 1024 + 16 * lane);
      const uint32_t four = *reinterpret_cast<const uint32_t*>(groups[nb] + (int64_t)kb * 64 + 4 * l16);
      const Group g = group_of(four >> (8 * q));
      const i32x4 lo = weights16<0>(record, g), hi = weights16<1>(record, g);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        acc[nb][mb] = mfma(lo, x[mb][0], acc[nb][mb]);
        acc[nb][mb] = mfma(hi, x[mb][1], acc[nb][mb]);
      }
    }
  }
  if constexpr (W > 1) {
    if (wave > 0)
#pragma unroll
      for (int i = 0; i < NB * MB; ++i) part[wave - 1][i][lane] = acc[i / MB][i % MB];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < W - 1; ++w)
#pragma unroll
      for (int i = 0; i < NB * MB; ++i) acc[i / MB][i % MB] += part[w][i][lane];
  }
  // Lane (l16, q) holds row l16 and columns 4 q .. 4 q + 3 of a 16 x 16 block.
  const float* const w_scale = reinterpret_cast<const float*>(p.w + at.scales_at());
  const int n_out = SWIGLU ? p.N >> 1 : p.N;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int64_t m = m0 + 16 * mb + l16;
    if (m >= p.M) continue;
    const float xscale = p.x_scale[m];
    uint16_t* const y = static_cast<uint16_t*>(p.y) + m * p.ldy;
#pragma unroll
    for (int nb = 0; nb < (SWIGLU ? NB / 2 : NB); ++nb) {
      const int n = 16 * (tile0 + nb) + 4 * q;
      if (n >= n_out) continue;
      const float4 s = *reinterpret_cast<const float4*>(w_scale + 16 * tile[nb] + 4 * q);
      const float sn[4] = {s.x, s.y, s.z, s.w};
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (float)acc[nb][mb][e] * sn[e] * xscale;
      if constexpr (SWIGLU) {
        const float4 t = *reinterpret_cast<const float4*>(w_scale + 16 * tile[nb + NB / 2] + 4 * q);
        const float tn[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = swiglu(v[e], (float)acc[nb + NB / 2][mb][e] * tn[e] * xscale);
      }
      const u32x2 d = {narrow2<BF16>(v[0], v[1]), narrow2<BF16>(v[2], v[3])};
      if (n + 4 <= n_out) {
        *reinterpret_cast<u32x2*>(y + n) = d;
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (n + e < n_out) y[n + e] = (uint16_t)(d[e >> 1] >> (16 * (e & 1)));
      }
    }
  }
}

template <bool BF16, bool SWIGLU, int MB, int NB, int W>
void launch_small(const W4Product& p, hipStream_t stream) {
  const int64_t blocks_m = (p.M + 16 * MB - 1) / (16 * MB), tiles = W4Layout(p.K, SWIGLU ? p.N / 2 : p.N).tiles;
  const int64_t per = SWIGLU ? NB / 2 : NB, blocks_n = (tiles + per - 1) / per;
  hipLaunchKernelGGL((w4_small_kernel<BF16, SWIGLU, MB, NB, W>), dim3((unsigned)(blocks_m * blocks_n)), dim3(64 * W), 0,
                     stream, p, (int)blocks_m);
}

template <bool BF16, bool SWIGLU>
hipError_t launch(const W4Product& p, hipStream_t stream) {
  launch_small<BF16, SWIGLU, 2, 2, 4>(p, stream);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_w4(const W4Product& p, bool bf16, bool swiglu, hipStream_t stream) {
  if (p.M <= 0) return hipSuccess;
  if (swiglu) return bf16 ? launch<true, true>(p, stream) : launch<false, true>(p, stream);
  return bf16 ? launch<true, false>(p, stream) : launch<false, false>(p, stream);
}

}  // namespace qattn
