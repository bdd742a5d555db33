// shared_plan.cpp -- host planner of the attention behind one shared prefix.
//
// Row blocks.  The rows of all sequences are stacked and cut into blocks of 256 or 128, so that short
// sequences fill a block together and a tile of prefix keys is read once for all its rows.  A block also
// visits the own keys of its sequences, one segment each, in which only their rows see anything.
// Sequences of up to 16 rows (single tokens) would waste most of a block on their own keys: those go to
// flat items of 16 rows, several sequences to an item or each by itself, and so may the prefix of a batch of
// up to kMostFlatRows rows (beyond, an item for every 16 rows reads it too often: with 512 rows, 2,048 keys
// take as long as by blocks, 24.5 us, and 8,192 keys 60 against 45).
//
// Cuts.  Items are cut along their keys where that shortens the launch: into equal chunks of a range of sizes, or
// one after another wherever a slot's share of the work ends.  The planner compares, for each of these ways,
// the time at which the last of the GPU's slots ends, by a cost model.
#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstring>
#include <queue>

#include "shared_attn.h"

namespace qattn {

namespace {

// Costs in microseconds, from measured launches (one workgroup to a CU): a block, and each of its 128-key tiles
// with 256 and with 128 rows; a flat item, and the bytes that it reads; partial results; the second launch;
// bytes that all items read from memory.
constexpr double kBlockItem = 5.9, kTallTile = 4.0, kSplitTile = 2.4, kFlatItem = 3.2, kItemBytesPerUs = 45e3;
constexpr double kFlatRound = 0.3, kFlatInt8 = 1.1, kFlatMasked = 0.4, kDim64 = 0.8;
constexpr double kPartial = 0.5, kMergeLaunch = 2.8, kBytesPerUs = 5e6;
constexpr int kMostSimulated = 16384, kMostInTurn = 1024, kMostFlatRows = 512;

struct Sequence {
  int32_t first, queries, keys;  // first query; own keys
  int32_t base, source;
};

struct Draft {
  SharedItem item;
  std::vector<SharedSeg> segs;
  int masked = 0;       // tiles that not every row sees whole
  bool merged = false;  // its rows have partial results elsewhere too
  std::vector<int> cuts;  // its chunks: 0, .., units()
  int first_part = 0;
  int chunks() const { return (int)cuts.size() - 1; }
  int units() const { return item.kind == kFlat ? (item.tiles + kFlatWaves - 1) / kFlatWaves : item.tiles; }
};

class Planner {
 public:
  Planner(const qattn_shared_desc& d, int compute_units, SharedPlan* plan)
      : d_(d), plan_(plan), group_(d.q_heads / d.cache.kv_heads),
        slots_(std::max(1, compute_units / d.cache.kv_heads)),
        key_bytes_(d.cache.head_dim * (d.cache.format == QATTN_KV_16BIT ? 4 : 2)) {}

  void run() {
    read();
    draft();
    emit();
  }

 private:
  static int tile_of(int kind) { return kind == kFlat ? kFlatKeys : kTallKeys; }
  bool local() const { return d_.mask == QATTN_MASK_PREFIX_LOCAL; }
  int64_t window() const { return std::min<int64_t>(d_.window, kMaxPosition); }

  void read() {
    int32_t first_row = 0;
    const int32_t page_size = std::max(1, d_.cache.page_size);
    const int32_t page_groups = d_.cache.kv_heads * (page_size / 16);
    // Appends the groups of `keys` keys, and takes `pages` past their pages.
    const auto add_groups = [&](const int32_t*& pages, int32_t keys) {
      const int32_t groups = (int32_t)(((int64_t)keys + 15) / 16);
      for (int32_t i = 0; i < groups; ++i)
        plan_->groups.push_back(pages[i / (page_size / 16)] * page_groups + i % (page_size / 16));
      while (groups && plan_->groups.size() % (kTallKeys / 16)) plan_->groups.push_back(plan_->groups.back());
      pages += ((int64_t)keys + page_size - 1) / page_size;
    };
    const int32_t* pages = d_.prefix_pages;
    if (d_.prefix_len) add_groups(pages, d_.prefix_len);
    pages = d_.own_pages;
    plan_->positions.resize(d_.cu_q[d_.nseq]);
    qattn_shared_info& info = plan_->info;
    info.tokens = d_.cu_q[d_.nseq];
    info.keys = d_.prefix_len;
    for (int32_t i = 0; i < d_.nseq; ++i) {
      Sequence s{d_.cu_q[i], d_.cu_q[i + 1] - d_.cu_q[i], d_.own_len[i], 0, kOwnRows};
      if (d_.own_pages) {
        s.source = kOwnPages;
        s.base = (int32_t)plan_->groups.size();
        add_groups(pages, s.keys);
      } else {
        s.base = first_row;
        first_row += s.keys;
      }
      info.keys += s.keys;
      for (int32_t j = 0; j < s.queries; ++j) {
        const int64_t at = (int64_t)d_.prefix_len + s.keys - s.queries + j;
        plan_->positions[s.first + j] = (int32_t)std::max<int64_t>(at, -1);
        if (at < 0) continue;
        int64_t seen = at + 1;
        if (local()) {
          const int64_t always = std::min<int64_t>(seen, d_.prefix);
          seen = always + std::max<int64_t>(0, at - std::max(at - window() + 1, always) + 1);
        }
        info.pairs += seen;
      }
      if (s.queries) sequences_.push_back(s);
    }
    info.flops = 4ll * d_.cache.head_dim * d_.q_heads * info.pairs;
  }

  // The tiles of `keys` keys from `position` on that queries at least .. greatest can see, as segments.
  void add_segs(std::vector<SharedSeg>* out, SharedSeg s, int tile, int32_t least, int32_t greatest) const {
    const int64_t end = std::min<int64_t>(s.keys, (int64_t)greatest - s.position + 1);
    if (end <= 0) return;
    const auto tiles = [&](int64_t n) { return (int32_t)((n + tile - 1) / tile); };
    const auto add = [&](int32_t a, int32_t b) {
      if (a >= b) return;
      s.tile_begin = a;
      s.tile_end = b;
      out->push_back(s);
    };
    if (!local()) return add(0, tiles(end));
    const int64_t always = std::clamp<int64_t>((int64_t)d_.prefix - s.position, 0, end);
    const int64_t start = std::clamp<int64_t>((int64_t)least - window() + 1 - s.position, 0, end);
    if (start / tile <= tiles(always)) return add(0, start < end ? tiles(end) : tiles(always));
    add(0, tiles(always));
    add((int32_t)(start / tile), start < end ? tiles(end) : (int32_t)(start / tile));
  }

  // Sequences by the rows that they have: whose own keys an item visits.
  enum Own { kLong = 1, kShort = 2, kAll = 3 };
  bool chosen(const Sequence& s, Own own) const {
    return own & ((int64_t)s.queries * group_ <= kFlatRows ? kShort : kLong);
  }

  // A block's segments: the prefix if asked for, and the own keys of its sequences that `own` names.
  Draft block(int64_t row0, int64_t rows, size_t first_sequence, int kind, bool prefix, Own own) const {
    const int tile = tile_of(kind);
    Draft b;
    b.item = SharedItem{(int32_t)row0, (int32_t)rows, 0, 0, -1, 0, kind};
    const int32_t t0 = (int32_t)(row0 / group_), t1 = (int32_t)((row0 + rows - 1) / group_);
    b.item.least = *std::min_element(&plan_->positions[t0], &plan_->positions[t1] + 1);
    b.item.greatest = *std::max_element(&plan_->positions[t0], &plan_->positions[t1] + 1);
    if (prefix && d_.prefix_len)
      add_segs(&b.segs, SharedSeg{kPrefixPages, 0, 0, d_.prefix_len, 0, 0, 0, (int32_t)row0, (int32_t)(row0 + rows)}, tile,
               b.item.least, b.item.greatest);
    for (size_t i = first_sequence; i < sequences_.size() && sequences_[i].first <= t1; ++i) {
      const Sequence& s = sequences_[i];
      if (!chosen(s, own)) continue;
      const int64_t begin = std::max<int64_t>(row0, (int64_t)s.first * group_);
      const int64_t end = std::min<int64_t>(row0 + rows, ((int64_t)s.first + s.queries) * group_);
      if (begin >= end || !s.keys) continue;
      add_segs(&b.segs, SharedSeg{s.source, 0, s.base, s.keys, d_.prefix_len, 0, 0, (int32_t)begin, (int32_t)end}, tile,
               plan_->positions[begin / group_], plan_->positions[(end - 1) / group_]);
    }
    finish(&b);
    return b;
  }

  // Counts a draft's tiles and takes apart the ones that all its rows see wholly, which the kernel neither
  // masks nor looks through.
  void finish(Draft* b) const {
    const int tile = tile_of(b->item.kind);
    std::vector<SharedSeg> segs;
    segs.swap(b->segs);
    for (const SharedSeg& s : segs) {
      b->item.tiles += s.tile_end - s.tile_begin;
      const bool all_rows = s.row_begin == b->item.row0 && s.row_end == b->item.row0 + b->item.rows;
      const auto whole = [&](int t) {
        const int64_t from = (int64_t)s.position + (int64_t)t * tile, to = from + tile - 1;
        return all_rows && (int64_t)(t + 1) * tile <= s.keys && to <= b->item.least &&
               (!local() || to < d_.prefix || from > b->item.greatest - window());
      };
      for (int t = s.tile_begin; t < s.tile_end;) {
        SharedSeg part = s;
        part.whole = whole(t);
        part.tile_begin = t;
        while (t < s.tile_end && whole(t) == (part.whole != 0)) ++t;
        part.tile_end = t;
        if (!part.whole) b->masked += part.tile_end - part.tile_begin;
        b->segs.push_back(part);
      }
    }
  }

  // Blocks of stacked rows of the sequences that have something to visit: `aligned` starts a block at every
  // sequence of a block's rows or more.
  std::vector<Draft> blocks(int kind, bool aligned, bool prefix, Own own) const {
    const int64_t most = kind == kTall ? kTallRows : kind == kSplit ? kSplitRows : kFlatRows;
    std::vector<Draft> out;
    int64_t begin = -1, end = 0;  // pending rows
    size_t first = 0;             // a sequence at or before them
    const auto flush = [&](int64_t upto) {
      while (begin >= 0 && begin < upto) {
        while (first < sequences_.size() && ((int64_t)sequences_[first].first + sequences_[first].queries) * group_ <= begin) ++first;
        const int64_t rows = std::min<int64_t>(most, upto - begin);
        out.push_back(block(begin, rows, first, kind, prefix, own));
        begin += rows;
      }
      begin = -1;
    };
    for (const Sequence& s : sequences_) {
      if (!(prefix && d_.prefix_len) && !chosen(s, own)) {
        flush(end);
        continue;
      }
      const int64_t row = (int64_t)s.first * group_, rows = (int64_t)s.queries * group_;
      if (begin < 0 || row != end || (aligned && rows >= most)) {
        flush(end);
        begin = row;
      }
      end = row + rows;
    }
    flush(end);
    return out;
  }

  // The fewest tiles: aligned blocks straddle fewer sequences, the others waste fewer rows.
  std::vector<Draft> best_blocks(int kind, bool prefix, Own own) const {
    const auto tiles = [](const std::vector<Draft>& v) {
      int64_t n = 0;
      for (const Draft& b : v) n += b.item.tiles + 2;
      return n;
    };
    std::vector<Draft> a = blocks(kind, true, prefix, own), b = blocks(kind, false, prefix, own);
    return tiles(a) <= tiles(b) ? a : b;
  }

  // The drafts that suit the batch best, cut.
  void draft() {
    const int64_t rows = (int64_t)plan_->positions.size() * group_;
    double best = 0;
    const auto consider = [&](std::vector<Draft> drafts, const std::vector<Draft>& more) {
      drafts.insert(drafts.end(), more.begin(), more.end());
      mark_merged(&drafts, rows);
      const double s = cut(&drafts);
      if (!drafts_.empty() && s >= best) return;
      best = s;
      drafts_ = std::move(drafts);
    };
    // The own keys of short sequences, which waste most of a larger block: in flat items, several
    // sequences to an item or each by itself.
    const std::vector<Draft> packed = blocks(kFlat, false, false, kShort);
    std::vector<Draft> single;
    for (size_t i = 0; i < sequences_.size(); ++i) {
      const Sequence& s = sequences_[i];
      if (s.keys && chosen(s, kShort))
        single.push_back(block((int64_t)s.first * group_, (int64_t)s.queries * group_, i, kFlat, false, kShort));
    }
    if (rows <= kMostFlatRows) {
      consider(blocks(kFlat, false, true, kAll), {});
      consider(blocks(kFlat, false, true, kLong), single);
    }
    if (rows <= kFlatRows) return;
    for (int kind : {kTall, kSplit}) {
      const std::vector<Draft> large = best_blocks(kind, true, kLong);
      consider(large, single);
      if (packed.size() < single.size()) consider(large, packed);
    }
  }

  // Drops drafts that see nothing; rows of two items are merged, and with them all rows of those items.
  static void mark_merged(std::vector<Draft>* drafts, int64_t rows) {
    drafts->erase(std::remove_if(drafts->begin(), drafts->end(), [](const Draft& b) { return b.item.tiles == 0; }), drafts->end());
    std::vector<uint8_t> cover(rows, 0);
    for (const Draft& b : *drafts)
      for (int32_t r = 0; r < b.item.rows; ++r) ++cover[b.item.row0 + r];
    for (Draft& b : *drafts)
      for (int32_t r = 0; r < b.item.rows; ++r) b.merged |= cover[b.item.row0 + r] > 1;
  }

  // The time that an item takes: fixed, and for each unit of work (cuts leave it whole: a tile; a round
  // of the eight wavefronts).
  static double fixed(const Draft& b) { return b.item.kind == kFlat ? kFlatItem : kBlockItem; }
  double unit(const Draft& b) const {
    if (b.item.kind != kFlat) return (b.item.kind == kTall ? kTallTile : kSplitTile) * (d_.cache.head_dim == 64 ? kDim64 : 1);
    return kFlatRound + kFlatWaves * kFlatKeys * key_bytes_ / kItemBytesPerUs + (d_.cache.format == QATTN_KV_INT8 ? kFlatInt8 : 0) +
           kFlatMasked * b.masked / std::max(1, b.item.tiles);
  }
  double cost(const Draft& b, int units) const { return fixed(b) + unit(b) * units; }
  // The units that `time` is enough for.  (The quotient of cost(b, n) may fall just below n.)
  int fit(const Draft& b, double time) const { return (int)std::floor((time - fixed(b)) / unit(b) * (1 + 1e-9)); }

  // Every draft in equal chunks that take `target` at most, if they can; false if they are more than `most`.
  bool cut_equally(std::vector<Draft>* drafts, double target, int64_t most) const {
    int64_t all = 0;
    for (Draft& b : *drafts) {
      const int64_t n = b.units(), each = std::max(1, fit(b, target)), chunks = (n + each - 1) / each;
      if ((all += chunks) > most) return false;
      b.cuts.resize(chunks + 1);
      for (int64_t i = 0; i <= chunks; ++i) b.cuts[i] = (int)(n * i / chunks);
    }
    return true;
  }
  // The drafts one after another, cut wherever a slot has had `target`; returns the slots it takes.
  int cut_in_turn(std::vector<Draft>* drafts, double target) const {
    int used = 1;
    double room = target;
    for (Draft& b : *drafts) {
      const int n = b.units();
      b.cuts.assign(1, 0);
      while (b.cuts.back() < n) {
        const int most = fit(b, room);
        if (most < std::min(2, n - b.cuts.back()) && room < target) {
          ++used;
          room = target;
          continue;
        }
        const int take = std::min(std::max(1, most), n - b.cuts.back());
        b.cuts.push_back(b.cuts.back() + take);
        room -= cost(b, take) + kPartial;
      }
    }
    return used;
  }

  // The time at which the last slot ends, longest item first, or the flat items' bytes have been read.
  double span(const std::vector<Draft>& drafts) const {
    std::vector<double> costs;
    double partial_rows = 0, flat_keys = 0;
    bool split = false;
    for (const Draft& b : drafts) {
      const bool part = b.chunks() > 1 || b.merged;
      if (part) partial_rows += (double)b.chunks() * b.item.rows;
      split |= part;
      if (b.item.kind == kFlat) flat_keys += (double)b.item.tiles * kFlatKeys;
      for (int i = 0; i < b.chunks(); ++i) costs.push_back((part ? kPartial : 0) + cost(b, b.cuts[i + 1] - b.cuts[i]));
    }
    std::sort(costs.begin(), costs.end(), std::greater<double>());
    std::priority_queue<double, std::vector<double>, std::greater<double>> ends;
    double last = 0;
    for (double c : costs) {
      double start = 0;
      if ((int)ends.size() == slots_) {
        start = ends.top();
        ends.pop();
      }
      ends.push(start + c);
      last = std::max(last, start + c);
    }
    last = std::max(last, kFlatItem + flat_keys * key_bytes_ * d_.cache.kv_heads / kBytesPerUs);
    return last + (split ? kMergeLaunch + partial_rows * d_.cache.kv_heads * d_.cache.head_dim * 8 / kBytesPerUs : 0);
  }

  // Chooses every draft's chunks; returns the launch's time.
  double cut(std::vector<Draft>* drafts) const {
    double longest = 0, total = 0;
    for (const Draft& b : *drafts) {
      longest = std::max(longest, cost(b, b.units()));
      total += cost(b, b.units());
    }
    for (Draft& b : *drafts) b.cuts = {0, b.units()};
    if (drafts->size() > kMostSimulated) return total / slots_;  // the slots are full
    double best = span(*drafts);
    std::vector<std::vector<int>> best_cuts(drafts->size());
    const auto keep = [&]() {
      for (size_t i = 0; i < best_cuts.size(); ++i) best_cuts[i] = (*drafts)[i].cuts;
    };
    const auto keep_better = [&]() {
      const double s = span(*drafts);
      if (s >= best * 0.98) return;
      best = s;
      keep();
    };
    keep();
    // More chunks than a few to a slot only add to the merge.
    const int64_t most = std::min<int64_t>(kMostSimulated, std::max<int64_t>(2 * drafts->size(), 4 * slots_));
    const double step = drafts->size() <= 256 ? 0.93 : 0.85;
    for (double target = longest * step; target > kFlatItem; target *= target > longest / 2 ? step : 0.8) {
      if (!cut_equally(drafts, target, most)) break;
      keep_better();
    }
    if (drafts->size() <= kMostInTurn) {
      double target = std::max(total / slots_, kFlatItem + 1);
      while (target < longest && cut_in_turn(drafts, target) > slots_) target *= 1.02;
      if (target < longest) keep_better();
    }
    for (size_t i = 0; i < best_cuts.size(); ++i) (*drafts)[i].cuts.swap(best_cuts[i]);
    return best;
  }

  void emit() {
    std::vector<std::pair<double, SharedItem>> items;
    for (Draft& b : drafts_) {
      const int rows = b.item.rows;
      const bool part = b.chunks() > 1 || b.merged;
      if (part) {
        b.first_part = (int32_t)plan_->partial_rows;
        plan_->partial_rows += (int64_t)b.chunks() * rows;
      }
      const int round = b.item.kind == kFlat ? kFlatWaves : 1;
      for (int c = 0; c < b.chunks(); ++c) {
        int begin = std::min(b.item.tiles, b.cuts[c] * round);
        int end = std::min(b.item.tiles, b.cuts[c + 1] * round);
        SharedItem it = b.item;
        it.seg_begin = (int32_t)plan_->segs.size();
        it.tiles = end - begin;
        it.part = part ? b.first_part + c * rows : -1;
        for (SharedSeg s : b.segs) {
          const int n = s.tile_end - s.tile_begin;
          if (begin < n && end > 0) {
            s.tile_end = s.tile_begin + std::min(n, end);
            s.tile_begin += std::max(0, begin);
            plan_->segs.push_back(s);
          }
          begin -= n;
          end -= n;
        }
        it.seg_end = (int32_t)plan_->segs.size();
        if (it.kind != kFlat) first_groups(&it);
        it.seg = plan_->segs[it.seg_begin];
        items.emplace_back(cost(b, (it.tiles + round - 1) / round), it);
      }
    }
    // Longest first, the flat items behind the others (their workgroups may come first all the same).
    std::stable_sort(items.begin(), items.end(), [](const auto& a, const auto& b) { return a.first > b.first; });
    std::stable_partition(items.begin(), items.end(), [](const auto& i) { return i.second.kind != kFlat; });
    for (const auto& i : items) {
      plan_->items.push_back(i.second);
      if (i.second.kind != kFlat) continue;
      ++plan_->flat_items;
      add_starts(i.second);
    }
    const size_t blocks = plan_->items.size() - plan_->flat_items;
    plan_->flat_first = blocks && plan_->flat_items && items[blocks].first > items[0].first;
    merge_rows();
    plan_->info.items = (int32_t)plan_->items.size();
    plan_->info.merged_rows = (int32_t)plan_->merges.size();
    plan_->info.partial_rows = plan_->partial_rows;
  }

  int32_t group_at(const SharedSeg& s, int32_t key) const { return s.source == kOwnRows ? 0 : plan_->groups[s.base + key / 16]; }

  // A block's copy of the groups of its first tile.
  void first_groups(SharedItem* it) const {
    const SharedSeg& s = plan_->segs[it->seg_begin];
    for (int i = 0; i < kTallKeys / 16; ++i) it->group[i] = group_at(s, s.tile_begin * kTallKeys + 16 * i);
  }

  // A flat item's tiles, in runs for its wavefronts.
  void add_starts(const SharedItem& it) const {
    int32_t seg = it.seg_begin, tile = it.seg.tile_begin;
    for (int w = 0; w < kFlatWaves; ++w) {
      SharedStart start{};
      start.tiles = (int32_t)((int64_t)it.tiles * (w + 1) / kFlatWaves - (int64_t)it.tiles * w / kFlatWaves);
      if (start.tiles) {
        const SharedSeg& s = plan_->segs[seg];
        std::memcpy(&start, &s, offsetof(SharedStart, seg));
        start.tile_begin = tile;
        start.seg = seg;
        for (int b = 0; b < 2; ++b) start.group[b] = group_at(s, tile * kFlatKeys + 16 * b);
      }
      plan_->starts.push_back(start);
      for (int n = start.tiles; n;) {
        const int step = std::min(n, plan_->segs[seg].tile_end - tile);
        n -= step;
        tile += step;
        if (tile == plan_->segs[seg].tile_end && ++seg < it.seg_end) tile = plan_->segs[seg].tile_begin;
      }
    }
  }

  // Rows with partial results, and rows that no item computes (merged from nothing: zeros).
  void merge_rows() {
    const int64_t rows = (int64_t)plan_->positions.size() * group_;
    std::vector<SharedMerge> all(rows, SharedMerge{});
    std::vector<uint8_t> direct(rows, 0);
    for (const Draft& b : drafts_)
      for (int32_t r = 0; r < b.item.rows; ++r) {
        const int64_t row = (int64_t)b.item.row0 + r;
        if (b.chunks() == 1 && !b.merged) {
          direct[row] = 1;
          continue;
        }
        SharedMerge& m = all[row];
        m.group[m.group[0].count ? 1 : 0] = {b.first_part + r, b.chunks(), b.item.rows};
      }
    for (int64_t row = 0; row < rows; ++row)
      if (!direct[row]) {
        all[row].row = (int32_t)row;
        plan_->most_parts = std::max(plan_->most_parts, all[row].group[0].count + all[row].group[1].count);
        plan_->merges.push_back(all[row]);
      }
  }

  const qattn_shared_desc& d_;
  SharedPlan* plan_;
  const int group_;
  const int slots_;
  const double key_bytes_;  // of a key's K and V for one KV head
  std::vector<Sequence> sequences_;
  std::vector<Draft> drafts_;
};

}  // namespace

void plan_shared(const qattn_shared_desc& d, int compute_units, SharedPlan* plan) { Planner(d, compute_units, plan).run(); }

}  // namespace qattn
