// shared_api.h -- limits and checks that the entry points behind one shared prefix share.
#pragma once
#include <stdint.h>

#include "../../include/qattn.h"

namespace qattn {

constexpr int32_t kMaxKvHeads = 256;
constexpr int32_t kMaxRopeHeads = 4096;
// Of a row-wise launch, whose grid has to stay below 2^32 threads.
constexpr int64_t kMaxRowTokens = ((int64_t)1 << 24) - 1;
constexpr int64_t kMaxRowValues = ((int64_t)1 << 35) - 1;  // tokens * kv_heads * head_dim: eight to a thread

// Geometry, and with needs_pages the tensors, of a cache.
int check_kv_cache(qattn_ctx* ctx, const qattn_kv_cache* c, bool needs_pages);

}  // namespace qattn
