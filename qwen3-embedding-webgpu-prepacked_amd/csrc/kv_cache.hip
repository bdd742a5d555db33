// kv_cache.hip -- the paged K/V cache: rows quantised as they are written, slots read back into rows.
//
// A vector is one token's head of K or V, held by head_dim / 16 lanes when it is written, by head_dim / 8
// when it is read, and a reading thread has two vectors in flight.  At the sizes below, writes of eight
// elements to a lane took 13.9 us, of sixteen 11.5, of sixteen of two vectors 11.9 (and 10.1 since the codes'
// arithmetic got shorter); reads of eight elements 30.8, of sixteen 29.3, of eight of two vectors 27.8.  The
// largest magnitude is reduced over the lanes by DPP.
//   e4m3  code = e4m3(x / s), s = 2^(least e with amax <= 448 2^e).  A power of two costs the division no
//         rounding, and a floating code's relative error does not depend on where in its range a value
//         lies, so against amax / 448 nothing is lost but up to one binade of the codes below 2^-6.
//   int8  code = rint(x * (127 / amax)), s = amax / 127, both divisions correctly rounded.
// Both kernels are bound by memory: a write of codes reads 2 bytes an element and writes 1 + 4 / head_dim, a
// read the reverse.  8,000 tokens of 8 heads of 128 are written as e4m3 in 10.1 us, 4.9 TB/s (int8 10.4, 16 bits
// 12.1); 20,000 are read in 28.3 us, 4.4 TB/s (int8 29.5, 16 bits 34.7), where copies of as many bytes take 7.3, from
// the last-level cache in part, and 24.8.
#include "shared_ops.h"

#include "elem.h"

namespace qattn {

namespace {

constexpr int kKvThreads = 256;
constexpr int kWriteElems = 16, kReadElems = 8, kReadEach = 2;

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

// Where a thread's vectors live: vectors run over tokens, then K and V, then heads.  The workgroup's first
// one takes the 64-bit division, once for all its threads.
struct Place {
  int64_t token;
  int which, head;  // which: 0 K, 1 V
};
template <int LANES, int EACH>
__device__ inline void places(int heads, Place (&at)[EACH]) {
  constexpr int kVectors = kKvThreads / LANES;
  const int64_t first = (int64_t)blockIdx.x * (kVectors * EACH), whole = first / (2 * heads);
  const uint32_t rest = (uint32_t)(first - whole * (2 * heads)) + threadIdx.x / LANES;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const uint32_t vector = rest + i * kVectors, in_token = vector % (uint32_t)(2 * heads);
    const int which = in_token >= (uint32_t)heads;
    at[i] = Place{whole + vector / (uint32_t)(2 * heads), which, (int)in_token - (which ? heads : 0)};
  }
}
// A place's slot, or -1.
__device__ inline int64_t slot_of(const KvArgs& a, const Place& at) {
  const int64_t slot = at.token < a.tokens ? a.slots[at.token] : -1;
  return slot < ((int64_t)a.cache.pages << __builtin_ctz(a.cache.page_size)) ? slot : -1;
}
// The vector of a slot's K or V; page_size is a power of two.
__device__ inline int64_t vector_of(const qattn_kv_cache& c, int64_t slot, int head) {
  const int shift = __builtin_ctz(c.page_size);
  return (((slot >> shift) * c.kv_heads + head) << shift) + (slot & (c.page_size - 1));
}

// A lane's elements of a vector as 8-bit codes, and the vector's scale.  Wavefronts whose vectors have finite
// elements, none of them all but zero, and no code to avoid take the short way: without it the codes'
// arithmetic, not memory, sets the time.
template <bool BF16, int FORMAT, int DIM>
__device__ inline u32x4 encode(const u32x4 (&x)[2], float* scale_out) {
#pragma clang fp contract(off)  // a code is the rounded product rounded
  constexpr int kElems = kWriteElems;
  constexpr uint32_t kExp = Elem<BF16>::kExponent;
  typedef uint16_t Pair __attribute__((ext_vector_type(2)));
  // Magnitudes compare as integers.
  Pair most2 = {0, 0};
#pragma unroll
  for (int e = 0; e < kElems / 2; ++e)
    most2 = __builtin_elementwise_max(most2, __builtin_bit_cast(Pair, x[e >> 2][e & 3] & 0x7FFF7FFFu));
  const uint32_t top = max((uint32_t)most2[0], (uint32_t)most2[1]);
  const bool finite = top < kExp;
  float f[kElems], amax = widen<BF16, 0>(finite ? top : 0);
#pragma unroll
  for (int e = 0; e < kElems / 2; ++e) {
    f[2 * e] = widen<BF16, 0>(x[e >> 2][e & 3]);
    f[2 * e + 1] = widen<BF16, 1>(x[e >> 2][e & 3]);
  }
  if (__any(!finite)) {
    amax = 0.f;
#pragma unroll
    for (int e = 0; e < kElems; ++e) {
      const float m = fabsf(f[e]);
      amax = fmaxf(amax, m < __builtin_inff() ? m : 0.f);  // a NaN compares false too
    }
  }
  amax = lanes_max<DIM / kElems>(amax);
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
    const bool short_codes = s >= (BF16 ? 120 : 8);
    if (__any(!finite || zeros || short_codes)) {
      const float most = short_codes ? 240.f : kE4m3Max;
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        const float v = zeros ? (f[e] - f[e] == 0.f ? 0.f : f[e]) : f[e] * inv;  // infinities and NaN stay
        f[e] = v != v ? v : fminf(fmaxf(v, -most), most);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kElems; ++e) f[e] *= inv;
    }
#pragma unroll
    for (int e = 0; e < kElems / 4; ++e) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * e], f[4 * e + 1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * e + 2], f[4 * e + 3], w, true);
      out[e] = (uint32_t)w;
    }
  } else {
    if (!zeros) {
      scale = amax / 127.f;
      inv = 127.f / amax;
    }
    if (__any(!finite || zeros)) {
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        const float v = zeros && f[e] - f[e] == 0.f ? 0.f : f[e] * (zeros ? 1.f : inv);
        f[e] = v != v ? 0.f : fminf(fmaxf(v, -127.f), 127.f);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kElems; ++e) f[e] *= inv;
    }
    // The low byte of 3 * 2^22 + f is f rounded to an integer.
#pragma unroll
    for (int e = 0; e < kElems / 4; ++e) {
      uint32_t w[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) w[b] = __float_as_uint(f[4 * e + b] + 12582912.f);
      const uint32_t low = __builtin_amdgcn_perm(w[1], w[0], 0x0C0C0400u), high = __builtin_amdgcn_perm(w[3], w[2], 0x04000C0Cu);
      out[e] = low | high;
    }
  }
  *scale_out = scale;
  return out;
}

template <bool BF16, int FORMAT, int DIM>
__global__ __launch_bounds__(kKvThreads) void kv_write_kernel(KvArgs a) {
  constexpr int kLanes = DIM / kWriteElems;
  const int lane = threadIdx.x % kLanes;
  Place places_[1];
  places<kLanes>(a.cache.kv_heads, places_);
  const Place at = places_[0];
  const int64_t slot = slot_of(a, at);
  if (slot < 0) return;  // alike in a vector's lanes
  const uint16_t* row = at.which ? a.v + at.token * a.v_stride : a.k + at.token * a.k_stride;
  const u32x4* src = reinterpret_cast<const u32x4*>(row + at.head * DIM + kWriteElems * lane);
  const u32x4 x[2] = {src[0], src[1]};
  const int64_t vector = vector_of(a.cache, slot, at.head);
  char* codes = static_cast<char*>(at.which ? a.cache.v : a.cache.k);
  if constexpr (FORMAT == QATTN_KV_16BIT) {
    u32x4* dst = reinterpret_cast<u32x4*>(codes + vector * (2 * DIM) + 2 * kWriteElems * lane);
    dst[0] = x[0];
    dst[1] = x[1];
  } else {
    float scale;
    *reinterpret_cast<u32x4*>(codes + vector * DIM + kWriteElems * lane) = encode<BF16, FORMAT, DIM>(x, &scale);
    if (lane == 0) (at.which ? a.cache.v_scale : a.cache.k_scale)[vector] = scale;
  }
}

template <bool BF16, int FORMAT, int DIM>
__global__ __launch_bounds__(kKvThreads) void kv_read_kernel(KvArgs a) {
  constexpr int kLanes = DIM / kReadElems;
  const int lane = threadIdx.x % kLanes;
  Place at[kReadEach];
  places<kLanes>(a.cache.kv_heads, at);
  int64_t slot[kReadEach];
  u32x4 x[kReadEach] = {};
  u32x2 codes[kReadEach] = {};
  float scale[kReadEach] = {};
#pragma unroll
  for (int i = 0; i < kReadEach; ++i) slot[i] = slot_of(a, at[i]);
#pragma unroll
  for (int i = 0; i < kReadEach; ++i) {
    if (slot[i] < 0) continue;
    const int64_t vector = vector_of(a.cache, slot[i], at[i].head);
    const char* pool = static_cast<const char*>(at[i].which ? a.cache.v : a.cache.k);
    if constexpr (FORMAT == QATTN_KV_16BIT) {
      x[i] = *reinterpret_cast<const u32x4*>(pool + vector * (2 * DIM) + 2 * kReadElems * lane);
    } else {
      codes[i] = *reinterpret_cast<const u32x2*>(pool + vector * DIM + kReadElems * lane);
      scale[i] = (at[i].which ? a.cache.v_scale : a.cache.k_scale)[vector];
    }
  }
#pragma unroll
  for (int i = 0; i < kReadEach; ++i) {
    if (at[i].token >= a.tokens) continue;
    if (FORMAT != QATTN_KV_16BIT && slot[i] >= 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u32x2 y = FORMAT == QATTN_KV_E4M3 ? e4m3_elems<BF16>(codes[i][e], scale[i]) : int8_elems<BF16>(codes[i][e], scale[i]);
        x[i][2 * e] = y[0];
        x[i][2 * e + 1] = y[1];
      }
    }
    uint16_t* row = at[i].which ? a.v + at[i].token * a.v_stride : a.k + at[i].token * a.k_stride;
    *reinterpret_cast<u32x4*>(row + at[i].head * DIM + kReadElems * lane) = x[i];
  }
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
  if (a.tokens <= 0) return hipSuccess;
  const int64_t vectors = a.tokens * 2 * a.cache.kv_heads;
  const int64_t block = WRITE ? kKvThreads * kWriteElems / a.cache.head_dim : kKvThreads * kReadElems * kReadEach / a.cache.head_dim;
  const dim3 grid((unsigned)((vectors + block - 1) / block));
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
