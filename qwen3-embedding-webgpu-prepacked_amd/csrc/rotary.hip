// rotary.hip -- rotary positions of given tokens (qattn_rope): half and interleaved layouts, part of the
// head, scaled frequencies, forward and inverse.
//
// A pair (a, b) turns by angle = position * f: (a cos - b sin, b cos + a sin).  The angle is reduced in
// f64, in turns: position * (f / 2 pi) minus its floor, so positions of 2^31 still have 2^-22 turns; the
// fraction goes to sincospif in f32 (2^-25 turns).  One (cos, sin) serves every head of its token: a
// workgroup takes one token, computes those into LDS, then its threads stream the heads.
// Bound by memory: 4 bytes moved per element for about two operations.  8,000 tokens of 24 heads of 128 take
// 18.9 us, 5.2 TB/s (a copy of as many bytes 19.5); in interleaved pairs 23.2.
#include "shared_ops.h"

#include "elem.h"

namespace qattn {

namespace {

constexpr int kRotaryThreads = 256;
constexpr int kMaxPairs = QATTN_MAX_ROPE_DIM / 2;

// WIDE: 16-byte accesses of eight elements (every address and width a multiple of eight elements); else
// one pair or one element at a time.
template <bool BF16, bool INTERLEAVED, bool WIDE>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  __shared__ float2 table[kMaxPairs];
  const int64_t token = blockIdx.x;
  for (int i = threadIdx.x; i < a.pairs; i += kRotaryThreads) {
    const double turn = (double)a.positions[token] * a.turns[i];
    float s, c;
    sincospif(2.f * (float)(turn - floor(turn)), &s, &c);
    table[i] = float2{c * a.magnitude, s * a.magnitude * a.sign};
  }
  __syncthreads();
  // Units of a head: the pairs (WIDE: eight elements a and their eight b, or four neighbouring pairs), then
  // the elements that pass through.
  const int turned = WIDE ? (INTERLEAVED ? a.pairs / 4 : a.pairs / 8) : a.pairs;
  const int units = turned + (WIDE ? a.tail / 8 : a.tail);
  const int total = a.heads * units;
  for (int i = threadIdx.x; i < total; i += kRotaryThreads) {
    const int head = i / units, unit = i - head * units;
    const bool is_q = head < a.heads_q;
    const RopeBlockArgs& b = is_q ? a.q : a.k;
    const int64_t column = (int64_t)(is_q ? head : head - a.heads_q) * a.head_dim;
    const uint16_t* x = b.x + token * b.x_stride + column;
    uint16_t* out = b.out + token * b.out_stride + column;
    if (unit >= turned) {
      const int c = 2 * a.pairs + (unit - turned) * (WIDE ? 8 : 1);
      if constexpr (WIDE)
        *reinterpret_cast<u32x4*>(out + c) = *reinterpret_cast<const u32x4*>(x + c);
      else
        out[c] = x[c];
    } else if constexpr (!WIDE) {
      const int ia = INTERLEAVED ? 2 * unit : unit, ib = INTERLEAVED ? 2 * unit + 1 : unit + a.pairs;
      const float xa = widen<BF16, 0>(x[ia]), xb = widen<BF16, 0>(x[ib]);
      const float2 r = table[unit];
      const uint32_t y = narrow2<BF16>(xa * r.x - xb * r.y, xb * r.x + xa * r.y);
      out[ia] = (uint16_t)y;
      out[ib] = (uint16_t)(y >> 16);
    } else if constexpr (INTERLEAVED) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(x + 8 * unit);
      u32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float xa = widen<BF16, 0>(v[e]), xb = widen<BF16, 1>(v[e]);
        const float2 r = table[4 * unit + e];
        y[e] = narrow2<BF16>(xa * r.x - xb * r.y, xb * r.x + xa * r.y);
      }
      *reinterpret_cast<u32x4*>(out + 8 * unit) = y;
    } else {
      const u32x4 va = *reinterpret_cast<const u32x4*>(x + 8 * unit);
      const u32x4 vb = *reinterpret_cast<const u32x4*>(x + a.pairs + 8 * unit);
      u32x4 ya, yb;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 r0 = table[8 * unit + 2 * e], r1 = table[8 * unit + 2 * e + 1];
        const float a0 = widen<BF16, 0>(va[e]), a1 = widen<BF16, 1>(va[e]);
        const float b0 = widen<BF16, 0>(vb[e]), b1 = widen<BF16, 1>(vb[e]);
        ya[e] = narrow2<BF16>(a0 * r0.x - b0 * r0.y, a1 * r1.x - b1 * r1.y);
        yb[e] = narrow2<BF16>(b0 * r0.x + a0 * r0.y, b1 * r1.x + a1 * r1.y);
      }
      *reinterpret_cast<u32x4*>(out + 8 * unit) = ya;
      *reinterpret_cast<u32x4*>(out + a.pairs + 8 * unit) = yb;
    }
  }
}

template <bool BF16, bool INTERLEAVED>
void launch(const RotaryArgs& a, bool wide, dim3 grid, hipStream_t stream) {
  if (wide)
    hipLaunchKernelGGL((rotary_kernel<BF16, INTERLEAVED, true>), grid, dim3(kRotaryThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((rotary_kernel<BF16, INTERLEAVED, false>), grid, dim3(kRotaryThreads), 0, stream, a);
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, bool bf16, bool interleaved, bool wide, hipStream_t stream) {
  if (a.tokens <= 0) return hipSuccess;
  const dim3 grid((unsigned)a.tokens);
  if (bf16)
    interleaved ? launch<true, true>(a, wide, grid, stream) : launch<true, false>(a, wide, grid, stream);
  else
    interleaved ? launch<false, true>(a, wide, grid, stream) : launch<false, false>(a, wide, grid, stream);
  return hipGetLastError();
}

}  // namespace qattn
