// shared_api.hip -- entry points of the operators behind one shared prefix: rotary positions, the paged
// K/V cache, and the attention over it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

#include "context.h"
#include "shared_attn.h"
#include "shared_ops.h"

using namespace qattn;

namespace {

constexpr int32_t kMaxKvHeads = 256;
constexpr int32_t kMaxRopeHeads = 4096;
// Of a row-wise launch, whose grid has to stay below 2^32 threads.
constexpr int64_t kMaxRowTokens = ((int64_t)1 << 24) - 1;
constexpr int64_t kMaxRowValues = ((int64_t)1 << 34) - 1;  // tokens * kv_heads * head_dim
constexpr int64_t kMaxSharedRows = (int64_t)1 << 22;       // queries * heads of a group
constexpr int64_t kMaxSharedStride = (int64_t)1 << 24;     // elements: 16 rows of it within a 32-bit offset
constexpr int64_t kMaxSharedGroups = ((int64_t)1 << 23) - 1;  // workgroups of a launch: below 2^32 threads

// The geometry of a cache's vectors, and with needs_pages everything else of it.
int check_kv_cache(qattn_ctx* ctx, const qattn_kv_cache* c, bool needs_pages) {
  if (!c) return fail(ctx, QATTN_EINVAL, "cache is NULL");
  if (c->dtype != QATTN_DTYPE_F16 && c->dtype != QATTN_DTYPE_BF16) return fail(ctx, QATTN_EINVAL, "unknown dtype %d", c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128) return fail(ctx, QATTN_EINVAL, "head_dim %d: 64 or 128", c->head_dim);
  if (c->kv_heads < 1 || c->kv_heads > kMaxKvHeads) return fail(ctx, QATTN_EINVAL, "kv_heads %d outside [1, %d]", c->kv_heads, kMaxKvHeads);
  if (!needs_pages) return QATTN_OK;
  if (c->format < QATTN_KV_16BIT || c->format > QATTN_KV_INT8) return fail(ctx, QATTN_EINVAL, "unknown cache format %d", c->format);
  if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
    return fail(ctx, QATTN_EINVAL, "page_size %d: a power of two in [16, 4096]", c->page_size);
  if (c->pages < 1 || (int64_t)c->pages * c->page_size * c->kv_heads >= (int64_t)1 << 35)
    return fail(ctx, QATTN_EINVAL, "pages %d: at least 1, pages*page_size*kv_heads below 2^35", c->pages);
  if (!c->k || !c->v || !aligned16(c->k) || !aligned16(c->v))
    return fail(ctx, QATTN_EINVAL, "cache k/v NULL or not 16-byte aligned");
  if (c->format != QATTN_KV_16BIT && (!c->k_scale || !c->v_scale || !aligned16(c->k_scale) || !aligned16(c->v_scale)))
    return fail(ctx, QATTN_EINVAL, "cache k_scale/v_scale NULL or not 16-byte aligned");
  return QATTN_OK;
}

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
    return fail(ctx, QATTN_EINVAL, "tokens*kv_heads*head_dim must be below 2^34");
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
  for (int32_t i = 0; i < a.pairs; ++i)
    if (!std::isfinite(a.turns[i])) return fail(ctx, QATTN_EINVAL, "theta/factor: pair %d turns past f64's range", i);
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

// ---- attention behind one shared prefix ---------------------------------------------------------------

// Two plan images, as a qattn_run keeps them: the installed plan lives in image `cur`; an update waits for
// the launches that last read the other one (events recorded on their streams when it was retired),
// fills it and switches.
struct qattn_shared_run {
  qattn_ctx* ctx = nullptr;
  qattn_shared_desc desc{};  // without its host arrays
  bool reads_pages = false, reads_rows = false;  // the installed plan
  int32_t format = QATTN_KV_16BIT;               // of its pages
  SharedParams params{};
  void* image[2] = {nullptr, nullptr};
  size_t image_bytes[2] = {0, 0};
  std::vector<hipStream_t> streams[2];
  std::vector<hipEvent_t> fences[2];
  int cur = -1;
  void* partials = nullptr;
  size_t partial_bytes = 0;
  qattn_shared_info info{};
};

namespace {

int check_shared_tensors(qattn_ctx* ctx, const qattn_shared_desc* d, bool needs_pages, bool needs_rows) {
  int rc = check_kv_cache(ctx, &d->cache, needs_pages);
  if (rc) return rc;
  const int64_t group = d->q_heads / d->cache.kv_heads;
  if (d->q_heads < 1 || d->q_heads % d->cache.kv_heads || group > 64)
    return fail(ctx, QATTN_EINVAL, "q_heads %d: a multiple of kv_heads %d, up to 64 times", d->q_heads, d->cache.kv_heads);
  const auto bad_stride = [](int64_t stride, int64_t width) { return stride < width || stride % 8 || stride > kMaxSharedStride; };
  if (!d->q || !d->o || !aligned16(d->q) || !aligned16(d->o)) return fail(ctx, QATTN_EINVAL, "q/o NULL or not 16-byte aligned");
  const int64_t q_width = (int64_t)d->q_heads * d->cache.head_dim, kv_width = (int64_t)d->cache.kv_heads * d->cache.head_dim;
  if (bad_stride(d->q_row_stride, q_width) || bad_stride(d->o_row_stride, q_width))
    return fail(ctx, QATTN_EINVAL, "row strides (q %lld, o %lld): q_heads*head_dim = %lld .. 2^24, multiples of 8",
                (long long)d->q_row_stride, (long long)d->o_row_stride, (long long)q_width);
  if (d->o == d->q || (needs_rows && (d->o == d->k || d->o == d->v))) return fail(ctx, QATTN_EINVAL, "o is q, k or v");
  if (!needs_rows) return QATTN_OK;
  if (!d->k || !d->v || !aligned16(d->k) || !aligned16(d->v)) return fail(ctx, QATTN_EINVAL, "k/v NULL or not 16-byte aligned");
  if (bad_stride(d->k_row_stride, kv_width) || bad_stride(d->v_row_stride, kv_width))
    return fail(ctx, QATTN_EINVAL, "row strides (k %lld, v %lld): kv_heads*head_dim = %lld .. 2^24, multiples of 8",
                (long long)d->k_row_stride, (long long)d->v_row_stride, (long long)kv_width);
  return QATTN_OK;
}

// Of the scores, for exponentials of 2.  (A masked score is -inf: times 0 it would be NaN.)
float scale_log2_of(const qattn_shared_desc& d) {
  return (float)((d.scale > 0.0 ? d.scale : 1.0 / std::sqrt((double)d.cache.head_dim)) * 1.4426950408889634);
}

bool own_keys(const qattn_shared_desc& d) {
  return std::any_of(d.own_len, d.own_len + d.nseq, [](int32_t n) { return n > 0; });
}
bool reads_pages(const qattn_shared_desc& d) { return d.prefix_len > 0 || (d.own_pages && own_keys(d)); }

int check_shared(qattn_ctx* ctx, const qattn_shared_desc* d) {
  if (!d) return fail(ctx, QATTN_EINVAL, "desc is NULL");
  int rc = validate_cu(ctx, d->cu_q, d->nseq);
  if (rc) return rc;
  if (!d->own_len) return fail(ctx, QATTN_EINVAL, "own_len is NULL");
  if (d->prefix_len < 0 || d->prefix_len >= kMaxPosition) return fail(ctx, QATTN_EINVAL, "prefix_len %d outside [0, 2^30)", d->prefix_len);
  int64_t own = 0;
  for (int32_t i = 0; i < d->nseq; ++i) {
    if (d->own_len[i] < 0 || (int64_t)d->prefix_len + d->own_len[i] >= kMaxPosition)
      return fail(ctx, QATTN_EINVAL, "own_len[%d] = %d: >= 0, positions below 2^30", i, d->own_len[i]);
    own += d->own_len[i];
  }
  if (own >= ((int64_t)1 << 31)) return fail(ctx, QATTN_EINVAL, "too many own keys (%lld)", (long long)own);
  rc = check_shared_tensors(ctx, d, reads_pages(*d), !d->own_pages && own);
  if (rc) return rc;
  if (d->mask != QATTN_MASK_CAUSAL && d->mask != QATTN_MASK_PREFIX_LOCAL) return fail(ctx, QATTN_EINVAL, "unknown mask kind %d", d->mask);
  if (d->mask == QATTN_MASK_PREFIX_LOCAL && (d->prefix < 0 || d->window < 0))
    return fail(ctx, QATTN_EINVAL, "prefix (%d) and window (%d) must be >= 0", d->prefix, d->window);
  if (!(d->scale >= 0.0) || !(d->scale < 1e30)) return fail(ctx, QATTN_EINVAL, "scale must be >= 0 and below 1e30");
  if (scale_log2_of(*d) == 0.f) return fail(ctx, QATTN_EINVAL, "scale %g vanishes in f32", d->scale);
  if (d->cu_q[d->nseq] * (int64_t)(d->q_heads / d->cache.kv_heads) > kMaxSharedRows)
    return fail(ctx, QATTN_EINVAL, "%d queries: queries * q_heads / kv_heads up to 2^22", d->cu_q[d->nseq]);
  const int32_t size = d->cache.page_size;
  const auto check_pages = [&](const char* name, const int32_t* pages, int64_t n) -> int {
    if (n && !pages) return fail(ctx, QATTN_EINVAL, "%s is NULL", name);
    for (int64_t i = 0; i < n; ++i)
      if (pages[i] < 0 || pages[i] >= d->cache.pages)
        return fail(ctx, QATTN_EINVAL, "%s[%lld] = %d outside [0, %d)", name, (long long)i, pages[i], d->cache.pages);
    return QATTN_OK;
  };
  if (d->prefix_len) rc = check_pages("prefix_pages", d->prefix_pages, (d->prefix_len + (int64_t)size - 1) / size);
  if (rc || !d->own_pages || !own) return rc;
  int64_t n = 0;
  for (int32_t i = 0; i < d->nseq; ++i) n += (d->own_len[i] + (int64_t)size - 1) / size;
  return check_pages("own_pages", d->own_pages, n);
}

// A checked description as it is planned and launched: where no page is read, the fields of the cache that
// nothing has looked at may hold anything.
qattn_shared_desc as_planned(qattn_shared_desc d) {
  if (!reads_pages(d)) {
    d.cache.pages = 0;
    d.cache.page_size = 16;
    d.cache.format = QATTN_KV_16BIT;
    d.cache.k = d.cache.v = nullptr;
    d.cache.k_scale = d.cache.v_scale = nullptr;
  }
  return d;
}

// Plans a checked description (as_planned); refuses what no launch could hold.
int make_shared_plan(qattn_ctx* ctx, const qattn_shared_desc& d, int compute_units, SharedPlan* plan) {
  plan_shared(d, compute_units, plan);
  const int64_t heads = d.cache.kv_heads;
  if ((int64_t)plan->items.size() * heads > kMaxSharedGroups || (int64_t)plan->merges.size() * heads > kMaxSharedGroups ||
      plan->partial_rows >= ((int64_t)1 << 31))
    return fail(ctx, QATTN_EINVAL, "too many rows for one launch (%zu items, %zu merged rows, %lld KV heads)", plan->items.size(),
                plan->merges.size(), (long long)heads);
  return QATTN_OK;
}

void bind_shared(SharedParams* p, const qattn_shared_desc& d) {
  p->q = static_cast<const uint16_t*>(d.q);
  p->o = static_cast<uint16_t*>(d.o);
  p->cache[0] = static_cast<const char*>(d.cache.k);
  p->cache[1] = static_cast<const char*>(d.cache.v);
  p->cache_scale[0] = d.cache.k_scale;
  p->cache_scale[1] = d.cache.v_scale;
  p->rows[0] = static_cast<const uint16_t*>(d.k);
  p->rows[1] = static_cast<const uint16_t*>(d.v);
}

int retire_shared(qattn_shared_run* run, int i) {
  for (hipStream_t s : run->streams[i]) {
    hipEvent_t ev = nullptr;
    HIP_TRY(run->ctx, hipEventCreateWithFlags(&ev, hipEventDisableTiming));
    const hipError_t e = hipEventRecord(ev, s);
    if (e != hipSuccess) {
      (void)hipEventDestroy(ev);
      return fail(run->ctx, QATTN_EHIP, "hipEventRecord: %s", hipGetErrorString(e));
    }
    try {
      run->fences[i].push_back(ev);
    } catch (const std::bad_alloc&) {
      (void)hipEventDestroy(ev);
      return fail(run->ctx, QATTN_ENOMEM, "out of host memory");
    }
  }
  run->streams[i].clear();
  return QATTN_OK;
}

int wait_shared(qattn_shared_run* run, int i) {
  auto& f = run->fences[i];
  while (!f.empty()) {
    HIP_TRY(run->ctx, hipEventSynchronize(f.back()));
    (void)hipEventDestroy(f.back());
    f.pop_back();
  }
  return QATTN_OK;
}

// Plans `d` into the run's other image and switches to it; on failure the installed plan stays.
int install_shared_plan(qattn_shared_run* run, const qattn_shared_desc& desc) {
  qattn_ctx* ctx = run->ctx;
  const qattn_shared_desc d = as_planned(desc);
  SharedPlan plan;
  int rc = make_shared_plan(ctx, d, std::max(1, ctx->cu_count), &plan);
  if (rc) return rc;
  std::vector<char> host;
  const auto put = [&](const void* data, size_t bytes) {
    const size_t at = (host.size() + 63) / 64 * 64;
    host.resize(at + bytes);
    if (bytes) std::memcpy(host.data() + at, data, bytes);
    return at;
  };
  const size_t items = put(plan.items.data(), plan.items.size() * sizeof(SharedItem));
  const size_t segs = put(plan.segs.data(), plan.segs.size() * sizeof(SharedSeg));
  const size_t starts = put(plan.starts.data(), plan.starts.size() * sizeof(SharedStart));
  const size_t merges = put(plan.merges.data(), plan.merges.size() * sizeof(SharedMerge));
  const size_t positions = put(plan.positions.data(), plan.positions.size() * sizeof(int32_t));
  const size_t groups = put(plan.groups.data(), plan.groups.size() * sizeof(int32_t));
  DeviceGuard g(ctx->device);
  const int next = run->cur < 0 ? 0 : run->cur ^ 1;
  if (run->cur >= 0 && (rc = retire_shared(run, run->cur))) return rc;
  if ((rc = wait_shared(run, next))) return rc;
  if (host.size() > run->image_bytes[next]) {
    void* grown = nullptr;
    const size_t bytes = host.size() + host.size() / 4;  // room for a few steps
    const hipError_t e = plan_malloc(&grown, bytes);
    if (e != hipSuccess) return fail(ctx, QATTN_ENOMEM, "hipMalloc(plan, %zu): %s", bytes, hipGetErrorString(e));
    if (run->image[next]) (void)hipFree(run->image[next]);
    run->image[next] = grown;
    run->image_bytes[next] = bytes;
  }
  const size_t values = (size_t)plan.partial_rows * d.cache.kv_heads;
  const size_t part_bytes = values * (d.cache.head_dim * sizeof(float) + sizeof(float2));
  if (part_bytes > run->partial_bytes) {
    // Launches of the installed plan may still use the workspace.
    if (run->cur >= 0 && (rc = wait_shared(run, run->cur))) return rc;
    void* grown = nullptr;
    const size_t bytes = part_bytes + part_bytes / 4;
    const hipError_t e = plan_malloc(&grown, bytes);
    if (e != hipSuccess) return fail(ctx, QATTN_ENOMEM, "hipMalloc(workspace, %zu): %s", bytes, hipGetErrorString(e));
    if (run->partials) (void)hipFree(run->partials);
    run->partials = grown;
    run->partial_bytes = bytes;
    // The installed plan keeps working, should the upload below fail: its rows fit the larger workspace.
    run->params.part_o = static_cast<float*>(grown);
    run->params.part_ml = reinterpret_cast<float2*>(run->params.part_o + (size_t)run->info.partial_rows * d.cache.kv_heads * d.cache.head_dim);
  }
  if (!host.empty()) HIP_TRY(ctx, hipMemcpy(run->image[next], host.data(), host.size(), hipMemcpyHostToDevice));
  SharedParams p{};
  bind_shared(&p, d);
  p.q_stride = d.q_row_stride;
  p.o_stride = d.o_row_stride;
  p.row_stride[0] = d.k_row_stride;
  p.row_stride[1] = d.v_row_stride;
  const char* image = static_cast<const char*>(run->image[next]);
  p.items = reinterpret_cast<const SharedItem*>(image + items);
  p.segs = reinterpret_cast<const SharedSeg*>(image + segs);
  p.starts = reinterpret_cast<const SharedStart*>(image + starts);
  p.merges = reinterpret_cast<const SharedMerge*>(image + merges);
  p.positions = reinterpret_cast<const int32_t*>(image + positions);
  p.groups = reinterpret_cast<const int32_t*>(image + groups);
  p.part_o = static_cast<float*>(run->partials);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + values * d.cache.head_dim);
  p.n_blocks = (int32_t)plan.items.size() - plan.flat_items;
  p.n_flat = plan.flat_items;
  p.flat_first = plan.flat_first;
  p.n_merges = (int32_t)plan.merges.size();
  p.most_parts = plan.most_parts;
  p.kv_heads = d.cache.kv_heads;
  p.group = d.q_heads / d.cache.kv_heads;
  p.page_shift = __builtin_ctz(d.cache.page_size);  // a power of two
  p.mask = d.mask;
  p.prefix = d.prefix;
  p.window = std::min(d.window, kMaxPosition);
  p.scale_log2 = scale_log2_of(d);
  run->params = p;
  run->info = plan.info;
  run->reads_pages = reads_pages(d);
  run->reads_rows = !d.own_pages && own_keys(d);
  run->format = d.cache.format;
  run->desc = desc;
  run->desc.prefix_pages = run->desc.cu_q = run->desc.own_len = nullptr;
  if (d.own_pages) run->desc.own_pages = reinterpret_cast<const int32_t*>(run);  // only whether there are any
  run->cur = next;
  return QATTN_OK;
}

int install_shared(qattn_shared_run* run, const qattn_shared_desc& d) {
  try {
    return install_shared_plan(run, d);
  } catch (const std::bad_alloc&) {
    return fail(run->ctx, QATTN_ENOMEM, "out of host memory for the plan");
  }
}

}  // namespace

extern "C" {

int qattn_shared_run_create(qattn_ctx* ctx, const qattn_shared_desc* desc, qattn_shared_run** out) {
  if (!ctx || !out) return fail(ctx, QATTN_EINVAL, "ctx/out is NULL");
  *out = nullptr;
  int rc = check_shared(ctx, desc);
  if (rc) return rc;
  auto* run = new (std::nothrow) qattn_shared_run();
  if (!run) return fail(ctx, QATTN_ENOMEM, "out of host memory");
  run->ctx = ctx;
  rc = install_shared(run, *desc);
  if (rc) {
    qattn_shared_run_destroy(run);
    return rc;
  }
  *out = run;
  return QATTN_OK;
}

int qattn_shared_run_encode(qattn_shared_run* run, qattn_stream_t stream) {
  if (!run) return fail(nullptr, QATTN_EINVAL, "run is NULL");
  DeviceGuard g(run->ctx->device);
  const hipStream_t s = pick_stream(run->ctx, stream);
  auto& used = run->streams[run->cur];
  try {
    if (std::find(used.begin(), used.end(), s) == used.end()) used.push_back(s);
  } catch (const std::bad_alloc&) {
    return fail(run->ctx, QATTN_ENOMEM, "out of host memory");
  }
  HIP_TRY(run->ctx, launch_shared_attn(run->params, run->desc.cache.dtype, run->format, run->desc.cache.head_dim, s));
  return QATTN_OK;
}

int qattn_shared_run_update(qattn_shared_run* run, const int32_t* prefix_pages, int32_t prefix_len, const int32_t* cu_q,
                            int32_t nseq, const int32_t* own_len, const int32_t* own_pages) {
  if (!run) return fail(nullptr, QATTN_EINVAL, "run is NULL");
  if ((own_pages != nullptr) != (run->desc.own_pages != nullptr))
    return fail(run->ctx, QATTN_EINVAL, "own_pages must be given as when the run was created");
  qattn_shared_desc d = run->desc;
  d.prefix_pages = prefix_pages;
  d.prefix_len = prefix_len;
  d.cu_q = cu_q;
  d.nseq = nseq;
  d.own_len = own_len;
  d.own_pages = own_pages;
  const int rc = check_shared(run->ctx, &d);
  return rc ? rc : install_shared(run, d);
}

int qattn_shared_run_rebind(qattn_shared_run* run, const void* q, void* o, const qattn_kv_cache* cache, const void* k,
                            const void* v) {
  if (!run) return fail(nullptr, QATTN_EINVAL, "run is NULL");
  if (!cache) return fail(run->ctx, QATTN_EINVAL, "cache is NULL");
  qattn_shared_desc d = run->desc;
  const qattn_kv_cache& c = d.cache;
  if (cache->pages != c.pages || cache->page_size != c.page_size || cache->kv_heads != c.kv_heads || cache->head_dim != c.head_dim ||
      cache->dtype != c.dtype || cache->format != c.format)
    return fail(run->ctx, QATTN_EINVAL, "the cache has another geometry than the run's");
  d.q = q;
  d.o = o;
  d.cache = *cache;
  d.k = k;
  d.v = v;
  const int rc = check_shared_tensors(run->ctx, &d, run->reads_pages, run->reads_rows);
  if (rc) return rc;
  bind_shared(&run->params, d);
  run->desc = d;
  return QATTN_OK;
}

void qattn_shared_run_destroy(qattn_shared_run* run) {
  if (!run) return;
  DeviceGuard g(run->ctx->device);
  for (int i = 0; i < 2; ++i) {
    if (retire_shared(run, i) != QATTN_OK)
      for (hipStream_t s : run->streams[i]) (void)hipStreamSynchronize(s);
    (void)wait_shared(run, i);
  }
  for (void* image : run->image)
    if (image) (void)hipFree(image);
  if (run->partials) (void)hipFree(run->partials);
  delete run;
}

int qattn_shared_run_get_info(const qattn_shared_run* run, qattn_shared_info* info) {
  if (!run || !info) return fail(nullptr, QATTN_EINVAL, "NULL argument");
  *info = run->info;
  return QATTN_OK;
}

int qattn_shared_plan_describe(const qattn_shared_desc* desc, int32_t* words, int64_t capacity, int64_t* count,
                               qattn_shared_info* info) {
  if (!count) return fail(nullptr, QATTN_EINVAL, "count is NULL");
  int rc = check_shared(nullptr, desc);
  if (rc) return rc;
  SharedPlan plan;
  try {
    rc = make_shared_plan(nullptr, as_planned(*desc), 256, &plan);
  } catch (const std::bad_alloc&) {
    rc = fail(nullptr, QATTN_ENOMEM, "out of host memory for the plan");
  }
  if (rc) return rc;
  const int32_t head[8] = {(int32_t)plan.items.size(), (int32_t)plan.segs.size(), (int32_t)plan.merges.size(),
                           (int32_t)plan.positions.size(), (int32_t)plan.groups.size(), (int32_t)plan.starts.size(), 0, 0};
  *count = 8 + (int64_t)(plan.items.size() * 32 + plan.segs.size() * 12 + plan.merges.size() * 8 + plan.positions.size() +
                         plan.groups.size() + plan.starts.size() * 16);
  if (info) *info = plan.info;
  if (!words) return QATTN_OK;
  if (capacity < *count) return fail(nullptr, QATTN_EINVAL, "capacity %lld < %lld words", (long long)capacity, (long long)*count);
  const auto put = [&](const void* data, size_t bytes) {
    if (bytes) std::memcpy(words, data, bytes);
    words += bytes / sizeof(int32_t);
  };
  put(head, sizeof(head));
  put(plan.items.data(), plan.items.size() * sizeof(SharedItem));
  put(plan.segs.data(), plan.segs.size() * sizeof(SharedSeg));
  put(plan.merges.data(), plan.merges.size() * sizeof(SharedMerge));
  put(plan.positions.data(), plan.positions.size() * sizeof(int32_t));
  put(plan.groups.data(), plan.groups.size() * sizeof(int32_t));
  put(plan.starts.data(), plan.starts.size() * sizeof(SharedStart));
  return QATTN_OK;
}

}  // extern "C"
