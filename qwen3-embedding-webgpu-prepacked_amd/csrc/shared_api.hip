// shared_api.hip -- entry points of the operators behind one shared prefix: rotary positions, the paged
// K/V cache.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "context.h"
#include "shared_api.h"
#include "shared_ops.h"

namespace qattn {

int check_kv_cache(qattn_ctx* ctx, const qattn_kv_cache* c, bool needs_pages) {
  if (!c) return fail(ctx, QATTN_EINVAL, "cache is NULL");
  if (c->dtype != QATTN_DTYPE_F16 && c->dtype != QATTN_DTYPE_BF16) return fail(ctx, QATTN_EINVAL, "unknown dtype %d", c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128) return fail(ctx, QATTN_EINVAL, "head_dim %d: 64 or 128", c->head_dim);
  if (c->kv_heads < 1 || c->kv_heads > kMaxKvHeads) return fail(ctx, QATTN_EINVAL, "kv_heads %d outside [1, %d]", c->kv_heads, kMaxKvHeads);
  if (c->format < QATTN_KV_16BIT || c->format > QATTN_KV_INT8) return fail(ctx, QATTN_EINVAL, "unknown cache format %d", c->format);
  if (!needs_pages) return QATTN_OK;
  if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
    return fail(ctx, QATTN_EINVAL, "page_size %d: a power of two in [16, 4096]", c->page_size);
  if (c->pages < 1) return fail(ctx, QATTN_EINVAL, "pages %d: at least 1", c->pages);
  if (!c->k || !c->v || !aligned16(c->k) || !aligned16(c->v))
    return fail(ctx, QATTN_EINVAL, "cache k/v NULL or not 16-byte aligned");
  if (c->format != QATTN_KV_16BIT && (!c->k_scale || !c->v_scale || !aligned16(c->k_scale) || !aligned16(c->v_scale)))
    return fail(ctx, QATTN_EINVAL, "cache k_scale/v_scale NULL or not 16-byte aligned");
  return QATTN_OK;
}

}  // namespace qattn

using namespace qattn;

namespace {

int check_rope_block(qattn_ctx* ctx, const char* name, const qattn_rope_block& b, int32_t head_dim) {
  if (!b.x || !b.out) return fail(ctx, QATTN_EINVAL, "%s: x/out is NULL", name);
  if ((reinterpret_cast<uintptr_t>(b.x) | reinterpret_cast<uintptr_t>(b.out)) & 1)
    return fail(ctx, QATTN_EINVAL, "%s: x/out not 2-byte aligned", name);
  const int64_t width = (int64_t)b.heads * head_dim;
  if (b.x_row_stride < width || b.out_row_stride < width)
    return fail(ctx, QATTN_EINVAL, "%s: row strides (%lld, %lld) below heads*head_dim = %lld", name,
                (long long)b.x_row_stride, (long long)b.out_row_stride, (long long)width);
  if (b.x == b.out && b.x_row_stride != b.out_row_stride)
    return fail(ctx, QATTN_EINVAL, "%s: in place (out = x) with two row strides", name);
  return QATTN_OK;
}

// Turns per position of every pair.
void rope_turns(const qattn_rope_desc& d, double* turns) {
  const double two_pi = 6.283185307179586476925;
  const int pairs = d.rotary_dim / 2;
  double low = 0, high = 0;
  if (d.scaling == QATTN_ROPE_YARN) {
    // The pair that turns n times in the original context: theta^(-2 i / dim) context = 2 pi n.
    const auto pair_of = [&](double n) {
      return d.rotary_dim * std::log(d.original_context / (n * two_pi)) / (2.0 * std::log(d.theta));
    };
    low = std::max(std::floor(pair_of(d.beta_fast)), 0.0);
    high = std::min(std::ceil(pair_of(d.beta_slow)), (double)d.rotary_dim - 1);
  }
  for (int i = 0; i < pairs; ++i) {
    double f = std::pow(d.theta, -2.0 * i / d.rotary_dim);
    if (d.scaling == QATTN_ROPE_LINEAR) f /= d.factor;
    if (d.scaling == QATTN_ROPE_YARN) {
      const double r = std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001)));
      f = f * (1.0 - r) + f / d.factor * r;
    }
    turns[i] = f / two_pi;
  }
}

bool wide_block(const qattn_rope_block& b) {
  return aligned16(b.x) && aligned16(b.out) && !((b.x_row_stride | b.out_row_stride) & 7);
}

int kv_args(qattn_ctx* ctx, const qattn_kv_cache* cache, const void* k, int64_t k_row_stride, const void* v,
            int64_t v_row_stride, const int64_t* slots, int64_t tokens, KvArgs* a) {
  if (!ctx) return fail(ctx, QATTN_EINVAL, "ctx is NULL");
  const int rc = check_kv_cache(ctx, cache, true);
  if (rc) return rc;
  if (tokens < 0 || tokens > kMaxRowTokens) return fail(ctx, QATTN_EINVAL, "tokens %lld outside [0, 2^24)", (long long)tokens);
  if (!tokens) return QATTN_OK;
  if (tokens * cache->kv_heads * cache->head_dim > kMaxRowValues)
    return fail(ctx, QATTN_EINVAL, "tokens*kv_heads*head_dim must be below 2^35");
  if (!k || !v || !slots) return fail(ctx, QATTN_EINVAL, "k/v/slots is NULL");
  if (!aligned16(k) || !aligned16(v) || (reinterpret_cast<uintptr_t>(slots) & 7))
    return fail(ctx, QATTN_EINVAL, "k/v not 16-byte or slots not 8-byte aligned");
  const int64_t width = (int64_t)cache->kv_heads * cache->head_dim;
  if (k_row_stride < width || v_row_stride < width || ((k_row_stride | v_row_stride) & 7))
    return fail(ctx, QATTN_EINVAL, "row strides (k %lld, v %lld): >= kv_heads*head_dim = %lld, multiples of 8",
                (long long)k_row_stride, (long long)v_row_stride, (long long)width);
  *a = KvArgs{*cache, slots, static_cast<uint16_t*>(const_cast<void*>(k)), static_cast<uint16_t*>(const_cast<void*>(v)),
              k_row_stride, v_row_stride, tokens};
  return QATTN_OK;
}

}  // namespace

extern "C" {

int qattn_rope(qattn_ctx* ctx, const qattn_rope_desc* d, qattn_stream_t stream) {
  if (!ctx || !d) return fail(ctx, QATTN_EINVAL, "ctx/desc is NULL");
  if (d->dtype != QATTN_DTYPE_F16 && d->dtype != QATTN_DTYPE_BF16) return fail(ctx, QATTN_EINVAL, "unknown dtype %d", d->dtype);
  if (d->head_dim < 2 || d->head_dim > QATTN_MAX_ROPE_DIM || d->rotary_dim < 2 || d->rotary_dim > d->head_dim || d->rotary_dim % 2)
    return fail(ctx, QATTN_EINVAL, "head_dim %d, rotary_dim %d: rotary_dim even, 2 <= rotary_dim <= head_dim <= %d",
                d->head_dim, d->rotary_dim, QATTN_MAX_ROPE_DIM);
  if (d->layout != QATTN_ROPE_HALF && d->layout != QATTN_ROPE_INTERLEAVED) return fail(ctx, QATTN_EINVAL, "unknown layout %d", d->layout);
  if (d->scaling < QATTN_ROPE_PLAIN || d->scaling > QATTN_ROPE_YARN) return fail(ctx, QATTN_EINVAL, "unknown scaling %d", d->scaling);
  if (!(d->theta > 0.0) || !std::isfinite(d->theta) || !std::isfinite(d->magnitude)) return fail(ctx, QATTN_EINVAL, "bad theta/magnitude");
  if (d->scaling != QATTN_ROPE_PLAIN && (!(d->factor > 0.0) || !std::isfinite(d->factor))) return fail(ctx, QATTN_EINVAL, "factor must be > 0");
  if (d->scaling == QATTN_ROPE_YARN &&
      (!(d->original_context > 0.0) || !std::isfinite(d->original_context) || !(d->beta_slow > 0.0) ||
       !(d->beta_fast > d->beta_slow) || !std::isfinite(d->beta_fast) || !(d->theta > 1.0)))
    return fail(ctx, QATTN_EINVAL, "YaRN: theta > 1, original_context > 0 and beta_fast > beta_slow > 0");
  if (d->q.heads < 1 || d->k.heads < 0 || d->q.heads > kMaxRopeHeads || d->k.heads > kMaxRopeHeads)
    return fail(ctx, QATTN_EINVAL, "heads (q %d, k %d): q in [1, %d], k in [0, %d]", d->q.heads, d->k.heads, kMaxRopeHeads, kMaxRopeHeads);
  if (d->tokens < 0 || d->tokens > kMaxRowTokens) return fail(ctx, QATTN_EINVAL, "tokens %lld outside [0, 2^24)", (long long)d->tokens);
  if (!d->tokens) return QATTN_OK;
  if (!d->positions || (reinterpret_cast<uintptr_t>(d->positions) & 3)) return fail(ctx, QATTN_EINVAL, "positions NULL or not 4-byte aligned");
  int rc = check_rope_block(ctx, "q", d->q, d->head_dim);
  if (!rc && d->k.heads) rc = check_rope_block(ctx, "k", d->k, d->head_dim);
  if (rc) return rc;
  RotaryArgs a{};
  const auto block = [](const qattn_rope_block& b) {
    return RopeBlockArgs{static_cast<const uint16_t*>(b.x), static_cast<uint16_t*>(b.out), b.x_row_stride, b.out_row_stride};
  };
  a.q = block(d->q);
  a.k = d->k.heads ? block(d->k) : a.q;
  a.positions = d->positions;
  a.tokens = d->tokens;
  a.heads_q = d->q.heads;
  a.heads = d->q.heads + d->k.heads;
  a.head_dim = d->head_dim;
  a.pairs = d->rotary_dim / 2;
  const bool in_place = d->q.x == d->q.out && (!d->k.heads || d->k.x == d->k.out);
  a.tail = in_place ? 0 : d->head_dim - d->rotary_dim;
  a.sign = d->inverse ? -1.f : 1.f;
  a.magnitude = (float)(d->magnitude != 0.0 ? d->magnitude
                        : d->scaling == QATTN_ROPE_YARN ? 0.1 * std::log(d->factor) + 1.0 : 1.0);
  rope_turns(*d, a.turns);
  const bool interleaved = d->layout == QATTN_ROPE_INTERLEAVED;
  const bool wide = wide_block(d->q) && (!d->k.heads || wide_block(d->k)) && d->head_dim % 8 == 0 &&
                    d->rotary_dim % (interleaved ? 8 : 16) == 0;
  DeviceGuard g(ctx->device);
  HIP_TRY(ctx, launch_rotary(a, d->dtype == QATTN_DTYPE_BF16, interleaved, wide, pick_stream(ctx, stream)));
  return QATTN_OK;
}

int qattn_kv_write(qattn_ctx* ctx, const qattn_kv_cache* cache, const void* k, int64_t k_row_stride, const void* v,
                   int64_t v_row_stride, const int64_t* slots, int64_t tokens, qattn_stream_t stream) {
  KvArgs a{};
  const int rc = kv_args(ctx, cache, k, k_row_stride, v, v_row_stride, slots, tokens, &a);
  if (rc || !tokens) return rc;
  DeviceGuard g(ctx->device);
  HIP_TRY(ctx, launch_kv_write(a, pick_stream(ctx, stream)));
  return QATTN_OK;
}

int qattn_kv_read(qattn_ctx* ctx, const qattn_kv_cache* cache, const int64_t* slots, int64_t tokens, void* k,
                  int64_t k_row_stride, void* v, int64_t v_row_stride, qattn_stream_t stream) {
  KvArgs a{};
  const int rc = kv_args(ctx, cache, k, k_row_stride, v, v_row_stride, slots, tokens, &a);
  if (rc || !tokens) return rc;
  DeviceGuard g(ctx->device);
  HIP_TRY(ctx, launch_kv_read(a, pick_stream(ctx, stream)));
  return QATTN_OK;
}

}  // extern "C"
