// shared_attn.h -- work items and launch arguments of the attention behind one shared prefix
// (shared_attn.hip), filled by its host planner (shared_plan.cpp).
//
// Row r of the launch is head r % group of query r / group, the same for every KV head.  A plan is made
// for one KV head; workgroup b runs item b / kv_heads for KV head b % kv_heads.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <vector>

#include "../../include/qattn.h"

namespace qattn {

constexpr int kSharedThreads = 512;
// Tall: eight wavefronts x 32 rows share a tile of 128 keys.  Split: four x 32 rows, twice: one four takes the
// tile's first 64 keys, the other its last.  Flat: eight wavefronts x the same 16 rows, a tile of 32 keys each.
constexpr int kTallRows = 256, kSplitRows = 128, kTallKeys = 128;
constexpr int kFlatRows = 16, kFlatKeys = 32, kFlatWaves = 8;
constexpr int32_t kMaxPosition = 1 << 30;

enum SharedSource { kPrefixPages = 0, kOwnPages = 1, kOwnRows = 2 };
enum SharedKind { kTall = 0, kSplit = 1, kFlat = 2 };

// Tiles tile_begin .. tile_end - 1 (of the item kind's size) of `keys` keys, seen by rows row_begin ..
// row_end - 1 only.  base: where the source's groups begin in the plan's list, or its first row.  A group is 16
// keys of a page: its number times 16 is the pool row (of KV head 0) of the first; a source's list is
// filled up to whole 128-key tiles with its last group.  whole: every row of the item sees every key of
// these tiles.
struct SharedSeg {
  int32_t source, whole, base, keys, position, tile_begin, tile_end, row_begin, row_end;
  int32_t pad[3];
};
// Rows row0 .. row0 + rows - 1 over the tiles of segments seg_begin .. seg_end - 1.  Results go to the output
// (part < 0) or, unnormalised, to partial rows part, part + 1, ...  The first segment and the groups of a
// block's first tile come with the item, so that a workgroup asks for its first keys after one dependent load.
struct SharedItem {
  int32_t row0, rows, seg_begin, seg_end, part, tiles, kind;
  int32_t least, greatest;  // query positions among the rows
  int32_t pad[3];
  SharedSeg seg;
  int32_t group[8];
};
// The tiles that one wavefront of a flat item takes, one after another: `tiles` of them, from tile_begin of
// its copy of segment `seg` on; `group`: the first one's.
struct SharedStart {
  int32_t source, whole, base, keys, position, tile_begin, tile_end, row_begin, row_end;
  int32_t seg, tiles;
  int32_t group[2];
  int32_t pad[3];
};
// A row whose results are merged: `count` partial rows from `first` on, `step` apart, in two groups.
struct SharedMerge {
  int32_t row;
  struct Group {
    int32_t first, count, step;
  } group[2];
  int32_t pad;
};
static_assert(sizeof(SharedItem) == 128 && sizeof(SharedSeg) == 48 && sizeof(SharedStart) == 64 && sizeof(SharedMerge) == 32,
              "plan words");

struct SharedPlan {
  std::vector<SharedItem> items;
  std::vector<SharedSeg> segs;
  std::vector<SharedStart> starts;  // kFlatWaves to a flat item, in their order
  std::vector<SharedMerge> merges;
  std::vector<int32_t> positions;  // of each query
  std::vector<int32_t> groups;
  int64_t partial_rows = 0;
  int32_t flat_items = 0;  // the last of them
  bool flat_first = false;
  int32_t most_parts = 0;  // partial rows of a merged row, at most
  qattn_shared_info info{};
};
// `d`: validated.  compute_units: of the device.
void plan_shared(const qattn_shared_desc& d, int compute_units, SharedPlan* plan);

struct SharedParams {
  const uint16_t* q;
  uint16_t* o;
  const char* cache[2];         // codes of K, V
  const float* cache_scale[2];
  const uint16_t* rows[2];      // own K, V rows
  int64_t q_stride, o_stride, row_stride[2];
  const SharedItem* items;
  const SharedSeg* segs;
  const SharedStart* starts;
  const SharedMerge* merges;
  const int32_t* positions;
  const int32_t* groups;
  float* part_o;                // [partial row][kv_heads][head_dim]
  float2* part_ml;              // [partial row][kv_heads]: the row's reference (log2) and sum
  int32_t n_blocks, n_flat;     // items that are not flat, and flat ones, which follow them in the list
  int32_t flat_first;           // the flat items' workgroups come first
  int32_t n_merges, most_parts, kv_heads, group, page_shift;
  int32_t mask, prefix, window;
  float scale_log2;
};
hipError_t launch_shared_attn(const SharedParams& p, int dtype, int format, int head_dim, hipStream_t stream);

}  // namespace qattn
