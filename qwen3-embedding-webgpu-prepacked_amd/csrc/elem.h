// elem.h -- the two 16-bit storage types of the shared-prefix operators, and the 8-bit cache codes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qattn {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Largest magnitude of an e4m3 code, and the least vector maximum that gets a scale of its own: below it
// 127 / amax and the powers of two would leave f32's normal range.
constexpr float kE4m3Max = 448.f;
constexpr float kLeastAmax = 0x1p-100f;

template <bool BF16>
struct Elem;
template <>
struct Elem<false> {
  typedef _Float16 T;
  typedef _Float16 T2 __attribute__((ext_vector_type(2)));
  typedef _Float16 T8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kExponent = 0x7C00u;
};
template <>
struct Elem<true> {
  typedef __bf16 T;
  typedef __bf16 T2 __attribute__((ext_vector_type(2)));
  typedef __bf16 T8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kExponent = 0x7F80u;
};

// The low (HI = 0) and high element of a dword, widened.  By integer shifts: hipcc has compiled the
// element reads of a packed fp16 vector in an unrolled loop as element 0.
template <bool BF16, int HI>
__device__ inline float widen(uint32_t d) {
  if constexpr (BF16)
    return __uint_as_float(HI ? d & 0xFFFF0000u : d << 16);
  else
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(HI ? d >> 16 : d & 0xFFFFu));
}
// Two values rounded to nearest even, packed.
template <bool BF16>
__device__ inline uint32_t narrow2(float a, float b) {
  typedef typename Elem<BF16>::T T;
  const typename Elem<BF16>::T2 v = {(T)a, (T)b};
  return __builtin_bit_cast(uint32_t, v);
}

// Four e4m3 codes of a dword times a power of two, as four 16-bit elements: one conversion per pair, which
// takes the exponent of `scale`.  Exact, but where the product is below the type's normal range.
template <bool BF16>
__device__ inline u32x2 e4m3_elems(uint32_t codes, float scale) {
  if constexpr (BF16) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))};
  } else {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true))};
  }
}
// Four int8 codes of a dword as fp16, which is exact: 0x6400 | u is 1024 + u, so a byte permute and a packed
// subtraction do it (an integer conversion for each code takes the cache four times the issue slots).
__device__ inline u32x2 int8_halves(uint32_t codes) {
  typedef Elem<false>::T2 H2;
  const uint32_t u = codes ^ 0x80808080u;
  const auto pair = [&](uint32_t select) {
    const H2 raw = __builtin_bit_cast(H2, __builtin_amdgcn_perm(0x64646464u, u, select));
    return __builtin_bit_cast(uint32_t, raw - H2{(_Float16)1152.f, (_Float16)1152.f});
  };
  return u32x2{pair(0x04010400u), pair(0x04030402u)};
}
// The codes times `scale`, each product rounded to f32 and then to 16 bits.
template <bool BF16>
__device__ inline u32x2 int8_elems(uint32_t codes, float scale) {
  const u32x2 h = int8_halves(codes);
  const auto pair = [&](uint32_t x) {
    return narrow2<BF16>(fmaf(widen<false, 0>(x), scale, 0.f), fmaf(widen<false, 1>(x), scale, 0.f));
  };
  return u32x2{pair(h[0]), pair(h[1])};
}

}  // namespace qattn
