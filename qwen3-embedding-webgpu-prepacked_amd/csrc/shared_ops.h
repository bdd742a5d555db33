// shared_ops.h -- launch arguments of the row-wise operators behind a shared prefix (rotary.hip,
// kv_cache.hip), shared with the host entry points that fill them (shared_api.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/qattn.h"

namespace qattn {

struct RopeBlockArgs {
  const uint16_t* x;
  uint16_t* out;
  int64_t x_stride, out_stride;
};
struct RotaryArgs {
  RopeBlockArgs q, k;
  const int32_t* positions;
  int64_t tokens;
  int32_t heads_q, heads;  // heads of q, of q and k together
  int32_t head_dim, pairs;
  int32_t tail;            // elements from tail_begin on that are copied (0 in place)
  float sign, magnitude;
  double turns[QATTN_MAX_ROPE_DIM / 2];  // turns per position of each pair
};
hipError_t launch_rotary(const RotaryArgs& a, bool bf16, bool interleaved, bool wide, hipStream_t stream);

struct KvArgs {
  qattn_kv_cache cache;
  const int64_t* slots;
  uint16_t* k;  // rows: read by a write, written by a read
  uint16_t* v;
  int64_t k_stride, v_stride, tokens;
};
hipError_t launch_kv_write(const KvArgs& a, hipStream_t stream);
hipError_t launch_kv_read(const KvArgs& a, hipStream_t stream);

}  // namespace qattn
