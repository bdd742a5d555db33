// w4_api.hip -- entry points of the operators of a forward with 8-bit activations: rows into 8 bits, and their
// products with 4-bit weights.
#include <hip/hip_runtime.h>

#include "context.h"
#include "w4_ops.h"

using namespace qattn;

namespace {

constexpr int64_t kMaxRows = ((int64_t)1 << 24) - 1;
// Workgroups of a launch, whose grid has to stay below 2^32 threads of at most 1,024 to a workgroup.
constexpr int64_t kMaxGroups = ((int64_t)1 << 22) - 1;

struct Range {
  const char* name;
  const void* p;
  int64_t bytes;
};
// Rows `width` elements wide, `stride` apart.
Range range_of(const char* name, const void* p, int64_t rows, int64_t stride, int64_t width, int64_t size) {
  return {name, p, rows > 0 ? ((rows - 1) * stride + width) * size : 0};
}
bool overlap(const Range& a, const Range& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  return a.p && b.p && a.bytes > 0 && b.bytes > 0 && (x < y ? y - x < (uintptr_t)a.bytes : x - y < (uintptr_t)b.bytes);
}
// What a call writes against everything else it touches.
int check_apart(qattn_ctx* ctx, const Range* written, int count, const Range* read, int reads) {
  for (int i = 0; i < count; ++i) {
    for (int j = i + 1; j < count; ++j)
      if (overlap(written[i], written[j])) return fail(ctx, QATTN_EINVAL, "%s and %s overlap", written[i].name, written[j].name);
    for (int j = 0; j < reads; ++j)
      if (overlap(written[i], read[j])) return fail(ctx, QATTN_EINVAL, "%s overlaps %s", written[i].name, read[j].name);
  }
  return QATTN_OK;
}

bool rows16(const void* p, int64_t stride, int32_t width) { return aligned16(p) && stride >= width && stride % 8 == 0 && stride <= kW4MaxStride; }

int check_row_q8(qattn_ctx* ctx, const RowQ8& p, int32_t dtype) {
  if (!ctx) return fail(ctx, QATTN_EINVAL, "ctx is NULL");
  if (dtype != QATTN_DTYPE_F16 && dtype != QATTN_DTYPE_BF16) return fail(ctx, QATTN_EINVAL, "unknown dtype %d", dtype);
  if (p.rows < 0 || p.rows > kMaxRows) return fail(ctx, QATTN_EINVAL, "rows %lld outside [0, 2^24)", (long long)p.rows);
  if (p.width < 8 || p.width % 8 || p.width > kQ8MaxWidth)
    return fail(ctx, QATTN_EINVAL, "width %d: a multiple of 8 in [8, %d]", p.width, kQ8MaxWidth);
  if (!p.x || !p.codes || !p.scales) return fail(ctx, QATTN_EINVAL, "x/codes/scales is NULL");
  if (!rows16(p.x, p.x_stride, p.width))
    return fail(ctx, QATTN_EINVAL, "x: 16-byte aligned, its stride at least the width, a multiple of 8, at most 2^22");
  if (reinterpret_cast<uintptr_t>(p.codes) % 8 || p.codes_stride < p.width || p.codes_stride % 8 || p.codes_stride > kW4MaxStride)
    return fail(ctx, QATTN_EINVAL, "codes: 8-byte aligned, their stride at least the width, a multiple of 8, at most 2^22");
  if (reinterpret_cast<uintptr_t>(p.scales) % 4) return fail(ctx, QATTN_EINVAL, "scales: 4-byte aligned");
  return QATTN_OK;
}

int check_w4(qattn_ctx* ctx, const W4Product& p, int64_t w_bytes, int32_t out_cols, int32_t dtype) {
  if (!ctx) return fail(ctx, QATTN_EINVAL, "ctx is NULL");
  if (dtype != QATTN_DTYPE_F16 && dtype != QATTN_DTYPE_BF16) return fail(ctx, QATTN_EINVAL, "unknown dtype %d", dtype);
  const int64_t need = qattn_w4_bytes(p.K, p.N);
  if (p.M < 0 || p.M > kMaxRows || need < 0)
    return fail(ctx, QATTN_EINVAL, "shape M=%d K=%d N=%d: M in [0, 2^24), K a multiple of 32 in [32, %d], N in [1, %d]", p.M, p.K, p.N,
                kW4MaxK, kW4MaxN);
  if (!p.x || !p.x_scale || !p.w || !p.y) return fail(ctx, QATTN_EINVAL, "x/x_scale/w/y is NULL");
  if (w_bytes < need) return fail(ctx, QATTN_EINVAL, "w_bytes %lld: %d x %d weights take %lld", (long long)w_bytes, p.N, p.K, (long long)need);
  if (!aligned16(p.x) || p.ldx < p.K || p.ldx % 16 || p.ldx > kW4MaxStride)
    return fail(ctx, QATTN_EINVAL, "x: 16-byte aligned, ldx at least K, a multiple of 16, at most 2^22");
  if (!rows16(p.y, p.ldy, out_cols))
    return fail(ctx, QATTN_EINVAL, "y: 16-byte aligned, ldy at least the %d columns, a multiple of 8, at most 2^22", out_cols);
  if (reinterpret_cast<uintptr_t>(p.x_scale) % 4 || !aligned16(p.w)) return fail(ctx, QATTN_EINVAL, "x_scale not 4-byte or w not 16-byte aligned");
  // Blocks of 32 rows and 16 columns, the smallest that any kernel takes of more than 16 rows (but of few blocks); those of
  // fewer rows have at most 2^17.
  if ((((int64_t)p.M + 31) / 32) * (((int64_t)out_cols + 15) / 16) > kMaxGroups)
    return fail(ctx, QATTN_EINVAL, "M=%d by %d columns: more than 2^22 blocks of a launch", p.M, out_cols);
  const Range written[] = {range_of("y", p.y, p.M, p.ldy, out_cols, 2)};
  const Range read[] = {range_of("x", p.x, p.M, p.ldx, p.K, 1), {"x_scale", p.x_scale, 4 * (int64_t)p.M}, {"w", p.w, need}};
  return check_apart(ctx, written, 1, read, 3);
}

}  // namespace

extern "C" {

int qattn_rmsnorm_q8(qattn_ctx* ctx, const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride,
                     void* sum, int64_t sum_row_stride, const float* weight, int8_t* codes, int64_t codes_row_stride,
                     float* scales, int64_t rows, int32_t width, int32_t dtype, double eps, qattn_stream_t stream) {
  const RowQ8 p{x, residual, sum, weight, codes, scales, x_row_stride, residual_row_stride, sum_row_stride, codes_row_stride,
                rows, width, (float)eps};
  int rc = check_row_q8(ctx, p, dtype);
  if (rc) return rc;
  if (!weight || !aligned16(weight)) return fail(ctx, QATTN_EINVAL, "weight: a 16-byte aligned device pointer");
  if (!(eps >= 0.0) || !(p.eps < INFINITY)) return fail(ctx, QATTN_EINVAL, "eps must be >= 0 and finite");
  if (!residual != !sum) return fail(ctx, QATTN_EINVAL, "residual and sum go together");
  if (residual && (!rows16(residual, residual_row_stride, width) || !rows16(sum, sum_row_stride, width)))
    return fail(ctx, QATTN_EINVAL, "residual/sum: 16-byte aligned, strides at least the width, multiples of 8, at most 2^22");
  // The sum may take the place of x or of the residual, row for row.
  const bool over_x = sum == x && sum_row_stride == x_row_stride, over_r = sum == residual && sum_row_stride == residual_row_stride;
  const Range written[] = {range_of("codes", codes, rows, codes_row_stride, width, 1), {"scales", scales, 4 * rows},
                           range_of("sum", sum, rows, sum_row_stride, width, 2)};
  const Range read[] = {{"weight", weight, 4 * (int64_t)width}, range_of("x", over_x ? nullptr : x, rows, x_row_stride, width, 2),
                        range_of("residual", over_r ? nullptr : residual, rows, residual_row_stride, width, 2)};
  rc = check_apart(ctx, written, 3, read, 3);
  if (rc) return rc;
  DeviceGuard g(ctx->device);
  HIP_TRY(ctx, launch_row_q8(p, dtype == QATTN_DTYPE_BF16, pick_stream(ctx, stream)));
  return QATTN_OK;
}

int qattn_quantize_q8(qattn_ctx* ctx, const void* x, int64_t x_row_stride, int8_t* codes, int64_t codes_row_stride,
                      float* scales, int64_t rows, int32_t width, int32_t dtype, qattn_stream_t stream) {
  const RowQ8 p{x, nullptr, nullptr, nullptr, codes, scales, x_row_stride, 0, 0, codes_row_stride, rows, width, 0.f};
  int rc = check_row_q8(ctx, p, dtype);
  if (rc) return rc;
  const Range written[] = {range_of("codes", codes, rows, codes_row_stride, width, 1), {"scales", scales, 4 * rows}};
  const Range read[] = {range_of("x", x, rows, x_row_stride, width, 2)};
  rc = check_apart(ctx, written, 2, read, 1);
  if (rc) return rc;
  DeviceGuard g(ctx->device);
  HIP_TRY(ctx, launch_row_q8(p, dtype == QATTN_DTYPE_BF16, pick_stream(ctx, stream)));
  return QATTN_OK;
}

int qattn_w4_matmul(qattn_ctx* ctx, const int8_t* x, int64_t ldx, const float* x_scale, int32_t M, int32_t K, const void* w,
                    int64_t w_bytes, int32_t N, void* y, int64_t ldy, int32_t dtype, qattn_stream_t stream) {
  const W4Product p{x, x_scale, static_cast<const uint8_t*>(w), y, ldx, ldy, M, K, N};
  const int rc = check_w4(ctx, p, w_bytes, N, dtype);
  if (rc) return rc;
  DeviceGuard g(ctx->device);
  HIP_TRY(ctx, launch_w4(p, dtype == QATTN_DTYPE_BF16, false, pick_stream(ctx, stream)));
  return QATTN_OK;
}

int qattn_w4_matmul_swiglu(qattn_ctx* ctx, const int8_t* x, int64_t ldx, const float* x_scale, int32_t M, int32_t K,
                           const void* w, int64_t w_bytes, int32_t n_inter, void* y, int64_t ldy, int32_t dtype,
                           qattn_stream_t stream) {
  if (n_inter < 32 || n_inter % 32 || n_inter > kW4MaxN / 2)
    return fail(ctx, QATTN_EINVAL, "n_inter %d: a multiple of 32 in [32, %d]", n_inter, kW4MaxN / 2);
  const W4Product p{x, x_scale, static_cast<const uint8_t*>(w), y, ldx, ldy, M, K, 2 * n_inter};
  const int rc = check_w4(ctx, p, w_bytes, n_inter, dtype);
  if (rc) return rc;
  DeviceGuard g(ctx->device);
  HIP_TRY(ctx, launch_w4(p, dtype == QATTN_DTYPE_BF16, true, pick_stream(ctx, stream)));
  return QATTN_OK;
}

}  // extern "C"
