// kv_cache.hip -- the paged K/V cache: rows quantised as they are written, slots read back into rows.
//
// A vector is one token's head of K or V: head_dim / 16 lanes hold it, 16 elements (32 bytes of the row,
// 16 of the 8-bit codes) each.  The largest magnitude is reduced over those lanes by DPP.
//   e4m3  code = e4m3(x / s), s = 2^(least e with amax <= 448 2^e).  A power of two costs the division no
//         rounding, and a floating code's relative error does not depend on where in its range a value
//         lies, so against amax / 448 nothing is lost but up to one binade of the codes below 2^-6.
//   int8  code = rint(x * (127 / amax)), s = amax / 127, both divisions correctly rounded.
// Both kernels are bound by memory: a write reads 2 bytes an element and writes 1 + 4 / head_dim.
#include "shared_ops.h"

#include "elem.h"

namespace qattn {

namespace {

constexpr int kKvThreads = 256;

// Combined with the lane at xor distance 1, 2 (quad permutations) and, within eight lanes, 4 (the row
// half's mirror: each quad holds one value by then).
template <int CTRL>
__device__ inline float dpp_max(float v) {
  const int i = __float_as_int(v);
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false)));
}
template <int LANES>
__device__ inline float lanes_max(float v) {
  v = dpp_max<0xB1>(v);
  v = dpp_max<0x4E>(v);
  if constexpr (LANES == 8) v = dpp_max<0x141>(v);
  return v;
}

// Where vector `i` lives: vectors run over tokens, then K and V, then heads.
template <int DIM>
struct Place {
  int64_t token;
  int which, head, lane;  // which: 0 K, 1 V; lane: its 16 elements of the vector
  __device__ Place(int64_t thread, int heads) {
    constexpr int kLanes = DIM / 16;
    lane = (int)(thread % kLanes);
    const int64_t vector = thread / kLanes;
    head = (int)(vector % heads);
    which = (int)(vector / heads & 1);
    token = vector / heads >> 1;
  }
};

template <bool BF16, int FORMAT, int DIM>
__global__ __launch_bounds__(kKvThreads) void kv_write_kernel(KvArgs a) {
  constexpr int kLanes = DIM / 16;
  const int heads = a.cache.kv_heads;
  const Place<DIM> at((int64_t)blockIdx.x * kKvThreads + threadIdx.x, heads);
  if (at.token >= a.tokens) return;
  const int64_t slot = a.slots[at.token];
  if (slot < 0 || slot >= (int64_t)a.cache.pages * a.cache.page_size) return;  // alike in a vector's lanes
  const uint16_t* row = at.which ? a.v + at.token * a.v_stride : a.k + at.token * a.k_stride;
  const u32x4* src = reinterpret_cast<const u32x4*>(row + at.head * DIM + 16 * at.lane);
  const u32x4 x[2] = {src[0], src[1]};
  const int64_t page = slot / a.cache.page_size, in_page = slot % a.cache.page_size;
  const int64_t vector = (page * heads + at.head) * a.cache.page_size + in_page;
  char* codes = static_cast<char*>(at.which ? a.cache.v : a.cache.k);
  if constexpr (FORMAT == QATTN_KV_16BIT) {
    u32x4* dst = reinterpret_cast<u32x4*>(codes + vector * (2 * DIM) + 32 * at.lane);
    dst[0] = x[0];
    dst[1] = x[1];
  } else {
    float f[16], amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[2 * e] = widen<BF16, 0>(x[e >> 2][e & 3]);
      f[2 * e + 1] = widen<BF16, 1>(x[e >> 2][e & 3]);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float m = fabsf(f[e]);
      amax = fmaxf(amax, m < __builtin_inff() ? m : 0.f);  // a NaN compares false too
    }
    amax = lanes_max<kLanes>(amax);
    const bool zeros = amax < kLeastAmax;
    float scale = 1.f, inv = 0.f;
    u32x4 out;
    if constexpr (FORMAT == QATTN_KV_E4M3) {
      // amax = 1.m 2^e <= 1.75 2^(8 + s)
      const uint32_t bits = __float_as_uint(amax);
      const int s = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u);
      if (!zeros) {
        scale = __uint_as_float((uint32_t)(127 + s) << 23);
        inv = __uint_as_float((uint32_t)(127 - s) << 23);
      }
      // 256 * 2^8 and 256 * 2^120 are past the largest fp16 and bf16 value: there 240 is the largest code.
      const float most = s >= (BF16 ? 120 : 8) ? 240.f : kE4m3Max;
      float y[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float v = zeros ? (f[e] - f[e] == 0.f ? 0.f : f[e]) : f[e] * inv;  // infinities and NaN stay
        y[e] = v != v ? v : fminf(fmaxf(v, -most), most);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * e], y[4 * e + 1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * e + 2], y[4 * e + 3], w, true);
        out[e] = (uint32_t)w;
      }
    } else {
      if (!zeros) {
        scale = amax / 127.f;
        inv = 127.f / amax;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t w = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const float x1 = f[4 * e + b];
          float v = zeros && x1 - x1 == 0.f ? 0.f : x1 * (zeros ? 1.f : inv);
          v = v != v ? 0.f : fminf(fmaxf(rintf(v), -127.f), 127.f);
          w |= ((uint32_t)(int)v & 255u) << (8 * b);
        }
        out[e] = w;
      }
    }
    *reinterpret_cast<u32x4*>(codes + vector * DIM + 16 * at.lane) = out;
    if (at.lane == 0) (at.which ? a.cache.v_scale : a.cache.k_scale)[vector] = scale;
  }
}

template <bool BF16, int FORMAT, int DIM>
__global__ __launch_bounds__(kKvThreads) void kv_read_kernel(KvArgs a) {
  const int heads = a.cache.kv_heads;
  const Place<DIM> at((int64_t)blockIdx.x * kKvThreads + threadIdx.x, heads);
  if (at.token >= a.tokens) return;
  const int64_t slot = a.slots[at.token];
  u32x4 x[2] = {};
  if (slot >= 0 && slot < (int64_t)a.cache.pages * a.cache.page_size) {
    const int64_t page = slot / a.cache.page_size, in_page = slot % a.cache.page_size;
    const int64_t vector = (page * heads + at.head) * a.cache.page_size + in_page;
    const char* codes = static_cast<const char*>(at.which ? a.cache.v : a.cache.k);
    if constexpr (FORMAT == QATTN_KV_16BIT) {
      const u32x4* src = reinterpret_cast<const u32x4*>(codes + vector * (2 * DIM) + 32 * at.lane);
      x[0] = src[0];
      x[1] = src[1];
    } else {
      const u32x4 c = *reinterpret_cast<const u32x4*>(codes + vector * DIM + 16 * at.lane);
      const float scale = (at.which ? a.cache.v_scale : a.cache.k_scale)[vector];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32x2 y = FORMAT == QATTN_KV_E4M3 ? e4m3_elems<BF16>(c[e], scale) : int8_elems<BF16>(c[e], scale);
        x[e >> 1][2 * (e & 1)] = y[0];
        x[e >> 1][2 * (e & 1) + 1] = y[1];
      }
    }
  }
  uint16_t* row = at.which ? a.v + at.token * a.v_stride : a.k + at.token * a.k_stride;
  u32x4* dst = reinterpret_cast<u32x4*>(row + at.head * DIM + 16 * at.lane);
  dst[0] = x[0];
  dst[1] = x[1];
}

template <bool WRITE, bool BF16, int FORMAT>
void launch(const KvArgs& a, dim3 grid, hipStream_t stream) {
  const dim3 block(kKvThreads);
  if (a.cache.head_dim == 64) {
    if constexpr (WRITE) hipLaunchKernelGGL((kv_write_kernel<BF16, FORMAT, 64>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((kv_read_kernel<BF16, FORMAT, 64>), grid, block, 0, stream, a);
  } else {
    if constexpr (WRITE) hipLaunchKernelGGL((kv_write_kernel<BF16, FORMAT, 128>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((kv_read_kernel<BF16, FORMAT, 128>), grid, block, 0, stream, a);
  }
}

template <bool WRITE>
hipError_t launch_kv(const KvArgs& a, hipStream_t stream) {
  const int64_t threads = a.tokens * 2 * a.cache.kv_heads * (a.cache.head_dim / 16);
  if (threads <= 0) return hipSuccess;
  const dim3 grid((unsigned)((threads + kKvThreads - 1) / kKvThreads));
  const bool bf16 = a.cache.dtype == QATTN_DTYPE_BF16;
  switch (a.cache.format) {
    case QATTN_KV_16BIT: launch<WRITE, false, QATTN_KV_16BIT>(a, grid, stream); break;  // bits are bits
    case QATTN_KV_E4M3:
      bf16 ? launch<WRITE, true, QATTN_KV_E4M3>(a, grid, stream) : launch<WRITE, false, QATTN_KV_E4M3>(a, grid, stream);
      break;
    default:
      bf16 ? launch<WRITE, true, QATTN_KV_INT8>(a, grid, stream) : launch<WRITE, false, QATTN_KV_INT8>(a, grid, stream);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_write(const KvArgs& a, hipStream_t stream) { return launch_kv<true>(a, stream); }
hipError_t launch_kv_read(const KvArgs& a, hipStream_t stream) { return launch_kv<false>(a, stream); }

}  // namespace qattn
