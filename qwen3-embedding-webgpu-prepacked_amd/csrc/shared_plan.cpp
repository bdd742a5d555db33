// shared_plan.cpp -- host planner of the attention behind one shared prefix.
//
// Row blocks.  The rows of all sequences are stacked and cut into blocks of 256 or 128, so that short
// sequences fill a block together and a tile of prefix keys is read once for all its rows.  A block also
// visits the own keys of its sequences, one segment each, in which only their rows see anything.
// Sequences of up to 16 rows (single tokens) would waste most of a block on their own keys: those go to
// items of 16 rows whose four wavefronts take a tile of keys each, and so do the prefix's if the launch has
// no more rows than that.
//
// Cuts.  Items are cut along their keys where that shortens the launch.  The planner compares, for both block
// sizes and a range of chunk sizes, the time at which the last of the GPU's slots ends, by a cost model.
#include <algorithm>
#include <cmath>
#include <queue>

#include "shared_attn.h"

namespace qattn {

namespace {

// Costs in microseconds, from measured launches (one workgroup to a CU): an item's start and end, a 128-key
// tile of a 256- and of a 128-row block, a round of four 32-key tiles of a pair of flat items, an item's
// partial results, the second launch, and the partial rows' bytes (written and read).
constexpr double kBlockItem = 4.0, kTallTile = 3.6, kSplitTile = 2.0, kFlatItem = 3.0, kFlatRound = 1.4;
constexpr double kPartial = 1.0, kMergeLaunch = 4.0, kBytesPerUs = 5e6;
constexpr int kMostSimulated = 16384;

struct Sequence {
  int32_t first, queries, keys;  // first query; own keys
  int32_t base, source;
};

struct Draft {
  SharedItem item;
  std::vector<SharedSeg> segs;
  bool merged = false;  // its rows have partial results elsewhere too
  int chunks = 1, first_part = 0;
  // Units of work that cuts leave whole (tiles; rounds of the four wavefronts), and their cost.
  int units() const { return item.kind == kFlat ? (item.tiles + 3) / 4 : item.tiles; }
  double fixed() const { return item.kind == kFlat ? kFlatItem : kBlockItem; }
  double unit() const { return item.kind == kFlat ? kFlatRound : item.kind == kTall ? kTallTile : kSplitTile; }
  double cost(int n) const { return fixed() + unit() * n; }
};

class Planner {
 public:
  Planner(const qattn_shared_desc& d, int compute_units, SharedPlan* plan)
      : d_(d), plan_(plan), group_(d.q_heads / d.cache.kv_heads),
        slots_(std::max(1, compute_units / d.cache.kv_heads)) {}

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

  // A block's segments: the prefix, and the own keys of its sequences that are not left to flat items.
  Draft block(int64_t row0, int64_t rows, size_t first_sequence, int kind, bool with_own) const {
    const int tile = tile_of(kind);
    Draft b;
    b.item = SharedItem{(int32_t)row0, (int32_t)rows, 0, 0, -1, 0, kind};
    const int32_t t0 = (int32_t)(row0 / group_), t1 = (int32_t)((row0 + rows - 1) / group_);
    b.item.least = *std::min_element(&plan_->positions[t0], &plan_->positions[t1] + 1);
    b.item.greatest = *std::max_element(&plan_->positions[t0], &plan_->positions[t1] + 1);
    if (d_.prefix_len)
      add_segs(&b.segs, SharedSeg{kPrefixPages, 0, 0, d_.prefix_len, 0, 0, 0, (int32_t)row0, (int32_t)(row0 + rows)}, tile,
               b.item.least, b.item.greatest);
    for (size_t i = first_sequence; with_own && i < sequences_.size() && sequences_[i].first <= t1; ++i) {
      const Sequence& s = sequences_[i];
      if (flat_own(s)) continue;
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
        b->segs.push_back(part);
      }
    }
  }

  bool flat_own(const Sequence& s) const { return !flat_all_ && (int64_t)s.queries * group_ <= kFlatRows; }

  // Blocks of stacked rows: `aligned` starts a block at every sequence of a block's rows or more.
  std::vector<Draft> blocks(int kind, bool aligned) const {
    const int64_t most = kind == kTall ? kTallRows : kSplitRows;
    std::vector<Draft> out;
    int64_t begin = -1, end = 0;  // pending rows
    size_t first = 0;             // a sequence at or before them
    const auto flush = [&](int64_t upto) {
      while (begin >= 0 && begin < upto) {
        while (first < sequences_.size() && ((int64_t)sequences_[first].first + sequences_[first].queries) * group_ <= begin) ++first;
        const int64_t rows = std::min<int64_t>(most, upto - begin);
        out.push_back(block(begin, rows, first, kind, true));
        begin += rows;
      }
      begin = -1;
    };
    for (const Sequence& s : sequences_) {
      if (!d_.prefix_len && flat_own(s)) {
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

  // The drafts that suit the batch best, cut.
  void draft() {
    if (sequences_.empty()) return;
    const int64_t rows = (int64_t)plan_->positions.size() * group_;
    std::vector<Draft> flat;
    if (rows <= kFlatRows && sequences_.size() == 1) {
      // One short sequence: prefix and own keys in one item.
      flat_all_ = true;
      flat.push_back(block((int64_t)sequences_[0].first * group_, rows, 0, kFlat, true));
    } else {
      if (rows <= kFlatRows && d_.prefix_len) flat.push_back(block(0, rows, 0, kFlat, false));
      for (const Sequence& s : sequences_)
        if (flat_own(s) && s.keys) {
          Draft f;
          const int64_t row0 = (int64_t)s.first * group_, n = (int64_t)s.queries * group_;
          f.item = SharedItem{(int32_t)row0, (int32_t)n, 0, 0, -1, 0, kFlat, plan_->positions[s.first],
                              plan_->positions[s.first + s.queries - 1]};
          add_segs(&f.segs, SharedSeg{s.source, 0, s.base, s.keys, d_.prefix_len, 0, 0, (int32_t)row0, (int32_t)(row0 + n)},
                   kFlatKeys, f.item.least, f.item.greatest);
          finish(&f);
          flat.push_back(std::move(f));
        }
    }
    double best = 0;
    const auto consider = [&](std::vector<Draft> blocks) {
      blocks.insert(blocks.end(), flat.begin(), flat.end());
      mark_merged(&blocks, rows);
      const double s = cut(&blocks);
      if (!drafts_.empty() && s >= best) return;
      best = s;
      drafts_ = std::move(blocks);
    };
    if (rows <= kFlatRows) return consider({});
    for (int kind : {kTall, kSplit}) {
      // Aligned blocks straddle fewer sequences, the others waste fewer rows: fewer tiles decide.
      const auto tiles = [](const std::vector<Draft>& v) {
        int64_t n = 0;
        for (const Draft& b : v) n += b.item.tiles + 2;
        return n;
      };
      std::vector<Draft> a = blocks(kind, true), b = blocks(kind, false);
      consider(tiles(a) <= tiles(b) ? std::move(a) : std::move(b));
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

  static int chunks_for(const Draft& b, double target) {
    const int n = b.units(), fit = std::max(1, (int)std::floor((target - b.fixed()) / b.unit()));
    return (n + fit - 1) / fit;
  }

  // The time at which the last slot ends, longest unit first, two flat items to a unit.
  double span(const std::vector<Draft>& drafts, double target) const {
    std::vector<double> costs, flat;
    double partial_rows = 0;
    bool split = false;
    for (const Draft& b : drafts) {
      const int c = chunks_for(b, target), units = b.units();
      const bool part = c > 1 || b.merged;
      if (part) partial_rows += (double)c * b.item.rows;
      split |= part;
      auto& to = b.item.kind == kFlat ? flat : costs;
      for (int i = 0; i < c; ++i) to.push_back((part ? kPartial : 0) + b.cost(units * (i + 1) / c - units * i / c));
      if (costs.size() + flat.size() > kMostSimulated) return 1e30;
    }
    std::sort(flat.begin(), flat.end(), std::greater<double>());
    for (size_t i = 0; i < flat.size(); i += 2) costs.push_back(flat[i]);
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
    return last + (split ? kMergeLaunch + partial_rows * d_.cache.kv_heads * d_.cache.head_dim * 8 / kBytesPerUs : 0);
  }

  // Chooses every draft's chunks; returns the launch's time.
  double cut(std::vector<Draft>* drafts) const {
    double longest = 0;
    for (const Draft& b : *drafts) longest = std::max(longest, b.cost(b.units()));
    double best_span = span(*drafts, longest), best = longest;
    for (double target = longest * 0.85; target > kBlockItem + kSplitTile; target *= target > longest / 2 ? 0.85 : 0.7) {
      const double s = span(*drafts, target);
      if (s < best_span * 0.97) {
        best_span = s;
        best = target;
      }
    }
    double total = 0;
    for (Draft& b : *drafts) {
      b.chunks = best > 0 ? chunks_for(b, best) : 1;
      total += b.cost(b.units());
    }
    return best_span < 1e30 ? best_span : total / slots_;  // too many to simulate: the slots are full
  }

  void emit() {
    std::vector<std::pair<double, SharedItem>> items;
    for (Draft& b : drafts_) {
      const int rows = b.item.rows;
      const bool part = b.chunks > 1 || b.merged;
      if (part) {
        b.first_part = (int32_t)plan_->partial_rows;
        plan_->partial_rows += (int64_t)b.chunks * rows;
      }
      const int round = b.item.kind == kFlat ? 4 : 1, units = b.units();
      for (int c = 0; c < b.chunks; ++c) {
        int begin = std::min(b.item.tiles, (int)((int64_t)units * c / b.chunks) * round);
        int end = std::min(b.item.tiles, (int)((int64_t)units * (c + 1) / b.chunks) * round);
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
        first_groups(&it);
        items.emplace_back(b.cost((it.tiles + round - 1) / round), it);
      }
    }
    // Longest first, the flat items behind the others (their workgroups may come first all the same).
    std::stable_sort(items.begin(), items.end(), [](const auto& a, const auto& b) { return a.first > b.first; });
    std::stable_partition(items.begin(), items.end(), [](const auto& i) { return i.second.kind != kFlat; });
    for (const auto& i : items) {
      plan_->items.push_back(i.second);
      plan_->flat_items += i.second.kind == kFlat;
    }
    const size_t blocks = plan_->items.size() - plan_->flat_items;
    plan_->flat_first = blocks && plan_->flat_items && items[blocks].first > items[0].first;
    merge_rows();
    plan_->info.items = (int32_t)plan_->items.size();
    plan_->info.merged_rows = (int32_t)plan_->merges.size();
    plan_->info.partial_rows = plan_->partial_rows;
  }

  // The item's own copy of its first segment and of the groups of its first tiles.
  void first_groups(SharedItem* it) const {
    it->seg = plan_->segs[it->seg_begin];
    const int tile = tile_of(it->kind);
    int32_t seg = it->seg_begin, at = it->seg.tile_begin;
    for (int i = 0; i < 8; ++i) {
      const SharedSeg& s = plan_->segs[seg];
      const int32_t first = at * tile + 16 * i % tile;
      it->group[i] = s.source == kOwnRows ? 0 : plan_->groups[s.base + first / 16];
      if ((16 * (i + 1)) % tile) continue;
      if (++at < s.tile_end) continue;
      if (++seg == it->seg_end) break;  // no further tile
      at = plan_->segs[seg].tile_begin;
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
        if (b.chunks == 1 && !b.merged) {
          direct[row] = 1;
          continue;
        }
        SharedMerge& m = all[row];
        m.group[m.group[0].count ? 1 : 0] = {b.first_part + r, b.chunks, b.item.rows};
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
  bool flat_all_ = false;
  std::vector<Sequence> sequences_;
  std::vector<Draft> drafts_;
};

}  // namespace

void plan_shared(const qattn_shared_desc& d, int compute_units, SharedPlan* plan) { Planner(d, compute_units, plan).run(); }

}  // namespace qattn
