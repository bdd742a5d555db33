// w4_weights.cpp -- 4-bit weights with whole-number group scales, laid out on the host for w4_matmul.hip: from a
// caller's own codes, from float rows, or from the Q4_0 tensors of a model file.
//
// A weight is (code - zero) * multiplier * scale: codes of 4 bits, a multiplier and a zero point of 4 bits each for
// a group of 32 columns, one f32 scale for a row.  (code - zero) * multiplier has to fit 8 bits, which bounds the
// pair.  No function here allocates, or needs a device.
#include <cmath>
#include <cstring>

#include "context.h"
#include "w4_ops.h"

using namespace qattn;

namespace {

constexpr int kGroup = 32;
constexpr int kQ4Record = 20;  // the Q4_0 record: f16 scale, 2 pad bytes, 16 quant bytes

bool fits(int mult, int zero) { return zero * mult <= 128 && (15 - zero) * mult <= 127; }

float half_value(uint16_t h) {
  const int exponent = h >> 10 & 31, mantissa = h & 1023;
  const double v = exponent == 31 ? (mantissa ? NAN : INFINITY)
                   : exponent     ? std::ldexp(1024 + mantissa, exponent - 25)
                                  : std::ldexp(mantissa, -24);
  return (float)(h >> 15 ? -v : v);
}

// Where the parts of one group and one row go.
struct Image {
  W4Layout at;
  uint8_t* base;
  Image(void* p, int K, int N) : at(K, N), base(static_cast<uint8_t*>(p)) {}
  // Every byte of the padding: multipliers of zero.
  void clear() { std::memset(base, 0, (size_t)at.bytes()); }
  uint8_t* record(int64_t n, int64_t g) const {
    return base + (((n >> 4) * at.blocks + (g >> 2)) * 4 + (g & 3)) * 256 + (n & 15) * 16;
  }
  uint8_t& group(int64_t n, int64_t g) const {
    return base[at.groups_at() + ((n >> 4) * at.blocks + (g >> 2)) * 64 + (n & 15) * 4 + (g & 3)];
  }
  void scale(int64_t n, float s) const { std::memcpy(base + at.scales_at() + n * 4, &s, 4); }
};

int check(const void* from, const void* image, int64_t image_bytes, int32_t K, int32_t N) {
  if (!from || !image) return fail(nullptr, QATTN_EINVAL, "weights/image is NULL");
  const int64_t need = qattn_w4_bytes(K, N);
  if (need < 0) return fail(nullptr, QATTN_EINVAL, "shape K=%d N=%d: K a multiple of 32 in [32, %d], N in [1, %d]", K, N, kW4MaxK, kW4MaxN);
  if (image_bytes < need)
    return fail(nullptr, QATTN_EINVAL, "image of %lld bytes: %d x %d weights take %lld", (long long)image_bytes, N, K, (long long)need);
  return QATTN_OK;
}

// The image is cleared before its source is read for the last time, so it may not lie over `bytes` of it.
int check_apart(const void* image, int64_t need, const void* from, int64_t bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(image), y = reinterpret_cast<uintptr_t>(from);
  if (x < y ? y - x < (uintptr_t)need : x - y < (uintptr_t)bytes) return fail(nullptr, QATTN_EINVAL, "the image overlaps what it is made from");
  return QATTN_OK;
}

// The rows of `load(n, g, w)`, which gives the 32 weights of a group.
template <typename Load>
int quantize(const Load& load, int32_t K, int32_t N, void* out) {
  const Image image(out, K, N);
  const int groups = K / kGroup;
  float w[kGroup];
  for (int32_t n = 0; n < N; ++n) {  // refused before the image is touched
    for (int g = 0; g < groups; ++g) {
      load(n, g, w);
      for (int j = 0; j < kGroup; ++j)
        if (!std::isfinite(w[j])) return fail(nullptr, QATTN_EINVAL, "row %d, column %d is not finite", n, g * kGroup + j);
    }
  }
  Image(out, K, N).clear();
  for (int32_t n = 0; n < N; ++n) {
    double top = 0;
    for (int g = 0; g < groups; ++g) {
      load(n, g, w);
      for (int j = 0; j < kGroup; ++j) top = std::fmax(top, std::fabs((double)w[j]));
    }
    if (top < 0x1p-100) continue;  // zeros
    const float scale = (float)(top / 120);  // multiplier 15 times 8 steps
    image.scale(n, scale);
    for (int g = 0; g < groups; ++g) {
      load(n, g, w);
      double most = 0;  // the value of the largest magnitude, the first of them
      for (int j = 0; j < kGroup; ++j)
        if (std::fabs((double)w[j]) > std::fabs(most)) most = w[j];
      if (most == 0) continue;
      const int zero = most < 0 ? 8 : 7;
      const int least = (int)std::floor(std::fabs(most) / 8 / (double)scale);
      int best = 0;
      double best_error = INFINITY;
      int8_t best_code[kGroup] = {};
      for (int m = least < 1 ? 1 : least > 15 ? 15 : least; m <= least + 1 && m <= 15; ++m) {
        const double step = (double)scale * m;
        int8_t code[kGroup];
        double error = 0;
        for (int j = 0; j < kGroup; ++j) {
          const double q = std::fmin(std::fmax(std::nearbyint((double)w[j] / step), -zero), 15 - zero);
          code[j] = (int8_t)((int)q + zero);
          const double d = (double)w[j] - q * step;
          error += d * d;
        }
        if (error < best_error) {
          best_error = error;
          best = m;
          std::memcpy(best_code, code, sizeof(code));
        }
      }
      uint8_t* const r = image.record(n, g);
      for (int j = 0; j < 16; ++j) r[j] = (uint8_t)(best_code[j] | best_code[j + 16] << 4);
      image.group(n, g) = (uint8_t)(best | zero << 4);
    }
  }
  return QATTN_OK;
}

}  // namespace

extern "C" {

int64_t qattn_w4_bytes(int32_t K, int32_t N) {
  if (K < kGroup || K % kGroup || K > kW4MaxK || N < 1 || N > kW4MaxN) return -1;
  return W4Layout(K, N).bytes();
}

int qattn_w4_pack(const uint8_t* codes, const uint8_t* groups, const float* scales, int32_t K, int32_t N, void* out,
                  int64_t image_bytes) {
  if (!groups || !scales) return fail(nullptr, QATTN_EINVAL, "groups/scales is NULL");
  int rc = check(codes, out, image_bytes, K, N);
  if (rc) return rc;
  const int64_t per_row = K / kGroup, need = qattn_w4_bytes(K, N);
  if ((rc = check_apart(out, need, codes, N * per_row * 16)) || (rc = check_apart(out, need, groups, N * per_row)) ||
      (rc = check_apart(out, need, scales, 4 * (int64_t)N)))
    return rc;
  for (int32_t n = 0; n < N; ++n) {
    if (!std::isfinite(scales[n])) return fail(nullptr, QATTN_EINVAL, "the scale of row %d is not finite", n);
    for (int64_t g = 0; g < per_row; ++g) {
      const int b = groups[n * per_row + g];
      if (!fits(b & 15, b >> 4))
        return fail(nullptr, QATTN_EINVAL, "row %d, group %lld: multiplier %d and zero point %d leave 8 bits (zero * multiplier <= 128, "
                    "(15 - zero) * multiplier <= 127)", n, (long long)g, b & 15, b >> 4);
    }
  }
  Image image(out, K, N);
  image.clear();
  for (int32_t n = 0; n < N; ++n) {
    image.scale(n, scales[n]);
    for (int64_t g = 0; g < per_row; ++g) {
      const uint8_t* const from = codes + (n * per_row + g) * 16;
      uint8_t* const to = image.record(n, g);
      for (int j = 0; j < 8; ++j) {  // columns 2 j, 2 j + 1 beside 16 + 2 j, 17 + 2 j
        to[2 * j] = (uint8_t)((from[j] & 15) | (from[8 + j] & 15) << 4);
        to[2 * j + 1] = (uint8_t)(from[j] >> 4 | (from[8 + j] & 0xF0));
      }
      image.group(n, g) = groups[n * per_row + g];
    }
  }
  return QATTN_OK;
}

int qattn_w4_quantize(const float* w, int64_t row_stride, int32_t K, int32_t N, void* image, int64_t image_bytes) {
  int rc = check(w, image, image_bytes, K, N);
  if (rc) return rc;
  if (row_stride < K) return fail(nullptr, QATTN_EINVAL, "row_stride %lld: at least K = %d", (long long)row_stride, K);
  if ((rc = check_apart(image, qattn_w4_bytes(K, N), w, 4 * ((N - 1) * row_stride + K)))) return rc;
  return quantize([&](int64_t n, int64_t g, float* out) { std::memcpy(out, w + n * row_stride + g * kGroup, 4 * kGroup); }, K, N, image);
}

int qattn_w4_from_q4(const void* q4, int64_t q4_bytes, int32_t K, int32_t N, void* image, int64_t image_bytes) {
  int rc = check(q4, image, image_bytes, K, N);
  if (rc) return rc;
  const int64_t size = qattn_q4_compact_bytes(K, N);
  if (q4_bytes < size)
    return fail(nullptr, QATTN_EINVAL, "q4_bytes %lld: a %d x %d tile32-compact tensor holds %lld", (long long)q4_bytes, N, K, (long long)size);
  if ((rc = check_apart(image, qattn_w4_bytes(K, N), q4, size))) return rc;
  const uint8_t* const from = static_cast<const uint8_t*>(q4);
  const int64_t blocks = K / kGroup;
  return quantize(
      [&](int64_t n, int64_t g, float* out) {
        const uint8_t* const r = from + (((n >> 5) * blocks + g) * 32 + (n & 31)) * kQ4Record;
        const float scale = half_value((uint16_t)(r[0] | r[1] << 8));
        for (int j = 0; j < 16; ++j) {
          out[j] = scale * (float)((r[4 + j] & 15) - 8);
          out[j + 16] = scale * (float)((r[4 + j] >> 4) - 8);
        }
      },
      K, N, image);
}

}  // extern "C"
