// shared_attn.hip -- attention of a batch of sequences behind one shared prefix (qattn_shared_run_*).
//
// o[r] = sum_j p_rj v_j / sum_j p_rj, p_rj = 2^(c q_r . k_j - m_r), over the keys that row r sees: the
// prefix's, read from a paged cache that may hold 8-bit codes, and its sequence's own.  Rows of all
// sequences are stacked (row = query * group + head of the group), so one tile of prefix keys serves 128
// rows, whatever sequences they belong to.  Two kinds of item share a launch:
//   tall  128 rows, 32 to a wavefront, over 64-key tiles that the four wavefronts share in LDS;
//         S^T = K Q^T and O^T = V^T P^T on 32x32x16 MFMAs, a query row to a lane.  Codes become 16-bit
//         elements once, on their way into LDS.  Bound by the matrix cores, the softmax's exponentials
//         and LDS reads.
//   flat  16 rows over 32-key tiles, every fourth tile to a wavefront, which keeps its own sum; K goes from
//         memory straight into the MFMA operand, V through the wavefront's own 8 KiB of LDS for the
//         transposed read; the four sums are joined at the end.  Bound by the cache's bytes.
// An item whose rows have keys elsewhere too (other chunks, other items) leaves its unnormalised f32
// sums, the row's reference m and its sum of p; shared_merge_kernel joins them.
//
// A row's reference moves only when a tile's maximum exceeds it by kLazy (in log2): p then stays below
// 2^kLazy, far inside fp16, and most tiles rescale nothing.  p is rounded to the storage type for the PV
// product, which moves each weight by at most half a step of that type; l sums the unrounded p in f32.
#include "shared_attn.h"

#include "elem.h"

namespace qattn {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16x __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;
typedef __attribute__((address_space(4))) const int32_t const_i32;

constexpr float kLazy = 8.f;
constexpr float kNone = -INFINITY;

template <bool BF16>
__device__ inline f16x mfma32(u32x4 a, u32x4 b, f16x c) {
  typedef typename Elem<BF16>::T8 T8;
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
}
template <bool BF16>
__device__ inline f4 mfma16(u32x4 a, u32x4 b, f4 c) {
  typedef typename Elem<BF16>::T8 T8;
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
}

// Combined with the other half-wavefront (lane ^ 32), and with the other 16-lane rows (lane ^ 16, ^ 32).
__device__ inline float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ inline float rows_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ inline float rows_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}
__device__ inline SharedSeg seg_at(const const_i32* w) {
  return SharedSeg{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8], {0, 0, 0}};
}
// All of an item but its groups.
__device__ inline SharedItem item_at(const SharedParams& p, int i) {
  const const_i32* w = (const const_i32*)(p.items + i);
  return SharedItem{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8], {0, 0, 0}, seg_at(w + 12), {}};
}
__device__ inline int item_group(const SharedParams& p, int i, int which) {
  return ((const const_i32*)(p.items + i))[24 + which];
}

// The tiles of an item one after another, through its segments.
struct Cursor {
  const const_i32* words;
  int tile;
  SharedSeg seg;
  __device__ Cursor(const SharedParams& p, const SharedItem& it)
      : words((const const_i32*)(p.segs + it.seg_begin)), tile(it.seg.tile_begin), seg(it.seg) {}
  // `n` tiles on; the item has that many.
  __device__ void advance(int n) {
    tile += n;
    while (tile >= seg.tile_end) {
      const int over = tile - seg.tile_end;
      words += sizeof(SharedSeg) / 4;
      seg = seg_at(words);
      tile = seg.tile_begin + over;
    }
  }
};

// This KV head's keys: uniform pointers, K's and V's.
template <int FORMAT, int DIM>
struct Keys {
  static constexpr bool kCodes = FORMAT != QATTN_KV_16BIT;
  static constexpr int kBytes = kCodes ? DIM : 2 * DIM;  // of a pool row
  const char* cache[2];
  const char* scale[2];
  const char* rows[2];
  uint32_t stride[2];  // bytes between rows
  __device__ Keys(const SharedParams& p, int kvh) {
    const int64_t head = (int64_t)kvh << p.page_shift;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      cache[i] = p.cache[i] + head * kBytes;
      scale[i] = reinterpret_cast<const char*>(p.cache_scale[i] + head);
      rows[i] = reinterpret_cast<const char*>(p.rows[i] + kvh * DIM);
      stride[i] = (uint32_t)p.row_stride[i] * 2;
    }
  }
  // Byte `offset` of a group (its 16 rows lie together; offset below their bytes), and of its scales.
  __device__ const char* in_group(int i, uint32_t group, uint32_t offset) const {
    return cache[i] + ((uint64_t)group * (16 * kBytes) | offset);
  }
  __device__ float scale_of(int i, uint32_t group, uint32_t row) const {
    return *reinterpret_cast<const float*>(scale[i] + ((uint64_t)group * 64 | 4 * row));
  }
  __device__ const char* row(int i, uint32_t row, uint32_t offset) const {
    return rows[i] + ((uint64_t)row * stride[i] + offset);
  }
};
// The group of key `first` of a segment, loaded as a vector: it is waited for with the tile's other loads.
__device__ inline uint32_t group_of(const SharedParams& p, const SharedSeg& s, int first, int zero) {
  return s.source == kOwnRows ? 0 : (uint32_t)p.groups[zero + s.base + (first >> 4)];
}

// 16 codes as two 16-byte chunks of 16-bit elements.
template <bool BF16, int FORMAT>
__device__ inline void expand(u32x4 codes, float scale, u32x4 (&out)[2]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const u32x2 y = FORMAT == QATTN_KV_E4M3 ? e4m3_elems<BF16>(codes[e], scale) : int8_elems<BF16>(codes[e], scale);
    out[e >> 1][2 * (e & 1)] = y[0];
    out[e >> 1][2 * (e & 1) + 1] = y[1];
  }
}

// ---- values that a row must not see ----------------------------------------------------------------
// A masked key's p is 0, but 0 times an infinity or NaN is NaN.  In tiles that some row of the item sees
// only part of, such elements of V are replaced by 0 on their way into LDS, and if there were any, the
// rows that do see the key get them added at the end (p times an infinity is that infinity, whatever the
// reference).
template <bool BF16>
__device__ inline bool drop_nonfinite(u32x4& chunk) {
  constexpr uint32_t kExp = Elem<BF16>::kExponent;
  bool any = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool low = (chunk[e] & kExp) == kExp, high = ((chunk[e] >> 16) & kExp) == kExp;
    any |= low | high;
    chunk[e] &= (low ? 0xFFFF0000u : 0xFFFFFFFFu) & (high ? 0x0000FFFFu : 0xFFFFFFFFu);
  }
  return any;
}
// Elements d .. d + 3 of key `key`'s V.
template <bool BF16, int FORMAT, int DIM>
__device__ inline f4 value_at(const SharedParams& p, const Keys<FORMAT, DIM>& keys, const SharedSeg& s, int key, int d) {
  u32x2 x;
  if (s.source == kOwnRows) {
    x = *reinterpret_cast<const u32x2*>(keys.row(1, s.base + key, 2 * d));
  } else {
    const uint32_t group = group_of(p, s, key, 0), row = key & 15;
    const char* at = keys.in_group(1, group, row * keys.kBytes + (keys.kCodes ? d : 2 * d));
    if constexpr (FORMAT == QATTN_KV_16BIT) {
      x = *reinterpret_cast<const u32x2*>(at);
    } else {
      const uint32_t codes = *reinterpret_cast<const uint32_t*>(at);
      const float scale = keys.scale_of(1, group, row);
      x = FORMAT == QATTN_KV_E4M3 ? e4m3_elems<BF16>(codes, scale) : int8_elems<BF16>(codes, scale);
    }
  }
  return f4{widen<BF16, 0>(x[0]), widen<BF16, 1>(x[0]), widen<BF16, 0>(x[1]), widen<BF16, 1>(x[1])};
}
__device__ inline float nonfinite(float v, bool seen) { return seen && !(fabsf(v) < INFINITY) ? v : 0.f; }
// Calls add(value, seen) for every key of the item's tiles first, first + step, ... (of `size` keys) that not
// all rows see: value(d) is elements d .. d + 3 of its V, seen whether row `row` at position `at` sees it.
template <bool BF16, int FORMAT, int DIM, class Add>
__device__ inline void each_nonfinite(const SharedParams& p, const Keys<FORMAT, DIM>& keys, const SharedItem& it, int row, int at,
                                      int size, int first, int step, Add add) {
  Cursor c(p, it);
  c.advance(first);
  for (int t = first;;) {
    const SharedSeg s = c.seg;
    if (!s.whole) {
      const int mine = row >= s.row_begin && row < s.row_end ? at : -1;
      for (int key = c.tile * size; key < min(s.keys, (c.tile + 1) * size); ++key) {
        const int pos = s.position + key;
        add([&](int d) { return value_at<BF16, FORMAT, DIM>(p, keys, s, key, d); },
            pos <= mine && (p.mask == QATTN_MASK_CAUSAL || pos < p.prefix || pos > mine - p.window));
      }
    }
    if ((t += step) >= it.tiles) return;
    c.advance(step);
  }
}

// ---- tall items -----------------------------------------------------------------------------------

template <bool BF16, int FORMAT, int DIM>
struct Tall {
  static constexpr int kRow = 2 * DIM;                  // bytes of a row in LDS
  static constexpr int kTile = kTallKeys * kRow;        // of K or V
  static constexpr int kLds = 4 * kTile;                // K and V, double buffered
  // 16-byte chunks of a row in memory, rows of a wavefront's load, loads per tile: of 16-bit rows, codes.
  static constexpr int kChunks16 = kRow / 16, kRows16 = 64 / kChunks16, kLoads16 = 16 / kRows16;
  static constexpr int kChunks8 = DIM / 16, kRows8 = 64 / kChunks8, kLoads8 = 16 / kRows8;
  static constexpr bool kCodes = FORMAT != QATTN_KV_16BIT;

  // 16-byte chunk c of row r, swizzled so that 16 rows' reads of one chunk (K) and the transposed reads
  // of four rows by four chunks (V) cover all 64 banks.
  __device__ static uint32_t k_at(int r, int c) { return r * kRow + ((c ^ (DIM == 128 ? r & 15 : (r >> 1) & 7)) << 4); }
  __device__ static uint32_t v_at(int r, int c) { return r * kRow + ((c ^ (DIM == 128 ? (r & 3) << 2 : (r & 2) << 1)) << 4); }

  // Where the 16 rows of a tile that this wavefront loads lie.  Rows of keys past the last are read as they
  // are, if a page holds them (their tile is not whole: their scores are masked, and infinities and NaN of
  // their V taken out), or as the last key's.
  struct Spot {
    uint32_t group;  // of pages
    int row, left;   // of p.rows: the first, and how many further there are
    bool rows;
  };

  u32x4 raw[2][kLoads16];
  float scale[2][kCodes ? kLoads8 : 1];

  // K (I = 0) or V (1) of a tile into registers.
  template <int I>
  __device__ void load(const Keys<FORMAT, DIM>& keys, const Spot& at, int lane) {
    if (at.rows) {
#pragma unroll
      for (int j = 0; j < kLoads16; ++j)
        raw[I][j] = *reinterpret_cast<const u32x4*>(
            keys.row(I, at.row + min(j * kRows16 + lane / kChunks16, at.left), lane % kChunks16 * 16));
    } else {
      const char* src = keys.in_group(I, at.group, lane * 16);
#pragma unroll
      for (int j = 0; j < (kCodes ? kLoads8 : kLoads16); ++j) raw[I][j] = *reinterpret_cast<const u32x4*>(src + j * 1024);
      if constexpr (kCodes) {
#pragma unroll
        for (int j = 0; j < kLoads8; ++j) scale[I][j] = keys.scale_of(I, at.group, lane / kChunks8 + j * kRows8);
      }
    }
  }

  // Half h of the loaded K (I = 0) or V (1) into LDS as 16-bit elements.  partly: infinities and NaN are
  // taken out (of V, in tiles that some row sees only part of); returns whether this lane had any.
  template <int I>
  __device__ bool store(char* lds, bool rows, int wave, int lane, int h, bool partly) {
    bool any = false;
    const auto put = [&](int r, int c, u32x4 x) {
      if (I && partly) any |= drop_nonfinite<BF16>(x);
      *reinterpret_cast<u32x4*>(lds + (I ? v_at(r, c) : k_at(r, c))) = x;
    };
    if (!kCodes || rows) {
#pragma unroll
      for (int j = h * kLoads16 / 2; j < (h + 1) * kLoads16 / 2; ++j)
        put(16 * wave + j * kRows16 + lane / kChunks16, lane % kChunks16, raw[I][j]);
    } else {
      constexpr int kEach = (kLoads8 + 1) / 2;
#pragma unroll
      for (int j = h * kEach; j < (h + 1) * kEach && j < kLoads8; ++j) {
        const int r = 16 * wave + j * kRows8 + lane / kChunks8, c = 2 * (lane % kChunks8);
        u32x4 x[2];
        expand<BF16, FORMAT>(raw[I][j], scale[I][kCodes ? j : 0], x);
        put(r, c, x[0]);
        put(r, c + 1, x[1]);
      }
    }
    return any;
  }
};

// Offset of accumulator element r (0 .. 31 over the two 32-key blocks) from the tile's first key + 4 hl.
__device__ constexpr int key_off(int r) { return 32 * (r >> 4) + 8 * ((r & 15) >> 2) + (r & 3); }

// Iteration t computes the scores of tile t, then its weights while the matrix cores add P(t - 1) V(t - 1);
// K(t + 1) and V(t), in registers since the iteration before, go to LDS, and K(t + 2) and V(t + 1) are asked
// for.
template <bool BF16, int FORMAT, int DIM>
__device__ inline void tall_item(const SharedParams& p, const SharedItem& it, int index, int kvh, char* lds, uint32_t* dropped) {
  typedef Tall<BF16, FORMAT, DIM> T;
  constexpr int kBlocks = DIM / 32, kSteps = DIM / 16;
  const int lane = threadIdx.x & 63, lq = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int end_row = it.row0 + it.rows, wave_row = it.row0 + 32 * wave;
  const int row = wave_row + lq;
  const bool exists = row < end_row;
  const int token = exists ? row / p.group : 0;
  const int head = kvh * p.group + row - token * p.group;
  const int at = exists ? p.positions[token] : -1;
  const bool local = p.mask != QATTN_MASK_CAUSAL;
  const auto k_buf = [&](int t) { return lds + (t & 1) * T::kTile; };
  const auto v_buf = [&](int t) { return lds + (2 + (t & 1)) * T::kTile; };

  // What the scores of a tile need to know of it.
  struct Info {
    int whole, from, last, row_begin, row_end;  // from: position of its first key; last: of its segment's last
  };
  const Keys<FORMAT, DIM> keys(p, kvh);
  Cursor ahead(p, it);  // the next K tile to ask for, its group on the way
  T tile;
  int zero = 0;
  asm volatile("" : "+v"(zero));
  uint32_t group = item_group(p, index, wave);
  typename T::Spot spot{}, spot_v{};
  int asked = 0;
  bool whole_v = true;  // the V tile in registers
  bool found = false;   // infinities or NaN were dropped from V
  if (threadIdx.x == 0) *dropped = 0;
  Info now{}, next{};   // of the scores to come, of the K tile in registers
  // K of the next tile, if there is one, and V of the tile before it.
  const auto ask_k = [&]() {
    if (asked == it.tiles) return;
    const SharedSeg& s = ahead.seg;
    const int first = ahead.tile * kTallKeys + 16 * wave;
    spot.rows = s.source == kOwnRows;
    spot.group = group;
    spot.row = s.base + min(first, s.keys - 1);
    spot.left = max(s.keys - 1 - first, 0);
    tile.template load<0>(keys, spot, lane);
    next = Info{s.whole, s.position + ahead.tile * kTallKeys, s.position + s.keys - 1, s.row_begin, s.row_end};
    if (++asked < it.tiles) {
      ahead.advance(1);
      group = group_of(p, ahead.seg, ahead.tile * kTallKeys + 16 * wave, zero);
    }
  };
  const auto ask_v = [&]() { tile.template load<1>(keys, spot_v, lane); };

  ask_k();  // K(0)
  // Q (B operand of S^T = K Q^T): this lane's row, dims 16 st + 8 hl .. + 7 at step st.
  u32x4 q[kSteps];
  {
    const uint16_t* src = p.q + (int64_t)token * p.q_stride + head * DIM + 8 * hl;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) q[st] = exists ? *reinterpret_cast<const u32x4*>(src + 16 * st) : u32x4{};
    // Here, once: a use inside the loop would wait for its tile's loads too.
#pragma unroll
    for (int st = 0; st < kSteps; ++st) asm volatile("" : "+v"(q[st]));
  }
  f16x o[kBlocks];
#pragma unroll
  for (int db = 0; db < kBlocks; ++db) o[db] = f16x{};
  float m = kNone, l = 0.f;

  // LDS read addresses.  K: rows lq, lq + 32.  V^T through the transposing read: in each 16-lane group G
  // lane a reads 4 elements of key 4 (G >> 1) + (a >> 2) (+ 16 t, + 8) at dims 32 db + 16 (G & 1) + 4 (a & 3)
  // and receives those keys' elements of dim 32 db + 16 (G & 1) + a.
  uint32_t v_read[kBlocks];
  {
    const int a = lane & 15, G = lane >> 4, r = 4 * (G >> 1) + (a >> 2);
#pragma unroll
    for (int db = 0; db < kBlocks; ++db) v_read[db] = T::v_at(r, 4 * db + 2 * (G & 1) + ((a & 3) >> 1)) + ((a & 1) << 3);
  }
  // O^T += V^T P^T for the tile in `v`.  Step st covers keys 16 st .. 16 st + 15; slot j of half hl is key
  // 16 st + 8 (j >> 2) + 4 hl + (j & 3), whose p is element j of pf[st].
  const auto v_frag = [&](const char* v, int i) {
    const char* src = v + v_read[i % kBlocks] + i / kBlocks * 16 * T::kRow;
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)src));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(src + 8 * T::kRow)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  // beside(i): other work, issued after product i.  Operands are read kDeep products ahead; the scheduling
  // barriers keep the compiler from reading them all at once, for which there are no registers.
  constexpr int kDeep = 2;
  const auto add_pv = [&](const char* v, const u32x4 (&pf)[4], auto beside) {
    u32x4 a[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) a[i] = v_frag(v, i);
#pragma unroll
    for (int i = 0; i < 4 * kBlocks; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      o[i % kBlocks] = mfma32<BF16>(a[i % kDeep], pf[i / kBlocks], o[i % kBlocks]);
      if (i + kDeep < 4 * kBlocks) a[i % kDeep] = v_frag(v, i + kDeep);
      beside(i);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto nothing = [](int) {};
  // p of elements r, r + 1.
  const auto weights = [&](const f16x (&sc)[2], int r, float ref, u32x4 (&pf)[4], float& sum) {
    const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[r >> 4][r & 15], p.scale_log2, -ref));
    const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[r >> 4][(r & 15) + 1], p.scale_log2, -ref));
    sum += p0 + p1;
    pf[r >> 3][(r & 7) >> 1] = narrow2<BF16>(p0, p1);
  };

#pragma unroll
  for (int h = 0; h < 2; ++h) tile.template store<0>(k_buf(0), spot.rows, wave, lane, h, false);
  now = next;
  spot_v = spot;
  whole_v = now.whole;
  ask_v();
  ask_k();
  // Scores of tile t, masked.
  // (beside(i): other work, issued after product i.)
  const auto scores = [&](const Info& cur, const char* k, f16x (&sc)[2], auto beside) {
    // Rows lq and lq + 32, chunk 2 st + hl: its swizzled place is 2 st xor'ed onto chunk hl's.  (Formed here:
    // hoisted, the addresses of all steps would take a register each.)
    uint32_t place = T::k_at(lq, hl) - lq * T::kRow;
    asm volatile("" : "+v"(place));
    const auto k_frag = [&](int i) {
      return *reinterpret_cast<const u32x4*>(k + lq * T::kRow + ((uint32_t)(i >> 1 << 5) ^ place) + 32 * (i & 1) * T::kRow);
    };
    constexpr int kAhead = 4;
    u32x4 a[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) a[i] = k_frag(i);
    __builtin_amdgcn_s_setprio(1);  // before the other wavefront's vector work
#pragma unroll
    for (int i = 0; i < 2 * kSteps; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      sc[i & 1] = mfma32<BF16>(a[i % kAhead], q[i >> 1], i < 2 ? f16x{} : sc[i & 1]);
      if (i + kAhead < 2 * kSteps) a[i % kAhead] = k_frag(i + kAhead);
      beside(i);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    if (!cur.whole) {
      // Offsets from this lane's first key: the last one seen, and where the prefix and the window leave a gap.
      const int mine = row >= cur.row_begin && row < cur.row_end ? at : -1;
      const int base = cur.from + 4 * hl, last = min(mine, cur.last) - base;
#pragma unroll
      for (int r = 0; r < 32; ++r) sc[r >> 4][r & 15] = key_off(r) > last ? kNone : sc[r >> 4][r & 15];
      if (local && cur.from + kTallKeys > p.prefix && cur.from <= it.greatest - p.window) {
        const int gap = p.prefix - base, window = mine - p.window - base;
#pragma unroll
        for (int r = 0; r < 32; ++r) {
          const int off = key_off(r);
          sc[r >> 4][r & 15] = (int)(off >= gap) & (int)(off <= window) ? kNone : sc[r >> 4][r & 15];
        }
      }
    }
  };
  // Moves the row's reference if the tile calls for it; returns what the sums so far are to be scaled by.
  const auto refer = [&](const f16x (&sc)[2]) {
    float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), sc[0][2]);
#pragma unroll
    for (int r = 3; r < 31; r += 2) top = fmaxf(fmaxf(top, sc[r >> 4][r & 15]), sc[(r + 1) >> 4][(r + 1) & 15]);
    top = half_max(fmaxf(top, sc[1][15])) * p.scale_log2;
    const float moved = top > m + kLazy ? top : m;  // from -inf too: any score exceeds it
    const float shrink = m == moved ? 1.f : __builtin_amdgcn_exp2f(m - moved);
    m = moved;
    return shrink;
  };
  // Beside the products of S(t): V(t) and K(t + 1) go to LDS, V(t + 1) and K(t + 2) are asked for.
  const auto move_on = [&](int t, int i) {
    constexpr int kEvery = kSteps / 4;
    if (i % kEvery) return;
    const bool more = t + 1 < it.tiles;
    switch (i / kEvery) {
      case 1: found |= tile.template store<1>(v_buf(t), spot_v.rows, wave, lane, 0, !whole_v); break;
      case 2: found |= tile.template store<1>(v_buf(t), spot_v.rows, wave, lane, 1, !whole_v); break;
      case 3:
        if (more) tile.template store<0>(k_buf(t + 1), spot.rows, wave, lane, 0, false);
        break;
      case 4:
        if (more) tile.template store<0>(k_buf(t + 1), spot.rows, wave, lane, 1, false);
        break;
      case 5:
        if (more) {
          now = next;
          spot_v = spot;
          whole_v = now.whole;
          ask_v();
        }
        break;
      case 6:
        if (more) ask_k();
        break;
    }
  };

  u32x4 pf[4];
  {
    __syncthreads();
    const Info cur = now;
    f16x sc[2];
    scores(cur, k_buf(0), sc, [&](int i) { move_on(0, i); });
    refer(sc);
    const float ref = m == kNone ? 0.f : m;
#pragma unroll
    for (int r = 0; r < 32; r += 2) weights(sc, r, ref, pf, l);
  }
  for (int t = 1; t < it.tiles; ++t) {
    // K(t) and V(t - 1) are in LDS, and every wavefront is done with the other buffers.
    __syncthreads();
    const Info cur = now;
    f16x sc[2];
    scores(cur, k_buf(t), sc, [&](int i) { move_on(t, i); });
    const float shrink = refer(sc);
    const float ref = m == kNone ? 0.f : m;
    // The weights beside the matrix cores' work on the tile before.
    u32x4 next_pf[4];
    float sum = 0.f;
    constexpr int kEach = 32 / (4 * kBlocks);
    add_pv(v_buf(t - 1), pf, [&](int i) {
#pragma unroll
      for (int r = kEach * i; r < kEach * (i + 1); r += 2) {
        weights(sc, r, ref, next_pf, sum);
      }
    });
    if (__any(shrink != 1.f)) {
#pragma unroll
      for (int db = 0; db < kBlocks; ++db) o[db] *= shrink;
    }
    l = l * shrink + sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) pf[i] = next_pf[i];
  }
  __syncthreads();
  add_pv(v_buf(it.tiles - 1), pf, nothing);
  if (found) *dropped = 1;
  __syncthreads();
  if (*dropped)
    each_nonfinite<BF16, FORMAT, DIM>(p, keys, it, row, at, kTallKeys, 0, 1, [&](auto value, bool seen) {
#pragma unroll
      for (int db = 0; db < kBlocks; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f4 x = value(32 * db + 8 * g + 4 * hl);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[db][4 * g + e] += nonfinite(x[e], seen);
        }
    });

  // O^T: this lane holds dims 32 db + 8 g + 4 hl .. + 3 of its row.
  l = half_sum(l);
  if (it.part < 0) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN stays one
    uint16_t* dst = p.o + (int64_t)token * p.o_stride + head * DIM + 8 * hl;
#pragma unroll
    for (int db = 0; db < kBlocks; ++db)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        const f16x& x = o[db];
        const int a = 4 * g, b = 4 * g + 4;
        const auto r0 = __builtin_amdgcn_permlane32_swap(narrow2<BF16>(x[a] * inv, x[a + 1] * inv),
                                                         narrow2<BF16>(x[b] * inv, x[b + 1] * inv), false, false);
        const auto r1 = __builtin_amdgcn_permlane32_swap(narrow2<BF16>(x[a + 2] * inv, x[a + 3] * inv),
                                                         narrow2<BF16>(x[b + 2] * inv, x[b + 3] * inv), false, false);
        if (exists) *reinterpret_cast<u32x4*>(dst + 32 * db + 8 * g) = u32x4{r0[0], r1[0], r0[1], r1[1]};
      }
  } else if (exists) {
    const int64_t part = ((int64_t)it.part + row - it.row0) * p.kv_heads + kvh;
    float* dst = p.part_o + part * DIM + 4 * hl;
#pragma unroll
    for (int db = 0; db < kBlocks; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f4*>(dst + 32 * db + 8 * g) = f4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
    if (hl == 0) p.part_ml[part] = float2{m, l};
  }
}

// ---- flat items -----------------------------------------------------------------------------------

template <bool BF16, int FORMAT, int DIM>
struct Flat {
  static constexpr int kRow = 2 * DIM;
  static constexpr int kLds = 4 * kFlatKeys * kRow;  // each wavefront's V tile, later its 16 rows of O in f32
  static constexpr int kSteps = DIM / 32;            // K: two 16-byte loads of codes, four of 16-bit elements per 128 dims
  static constexpr int kChunks16 = kRow / 16, kRows16 = 64 / kChunks16, kLoads16 = 16 / kRows16;
  static constexpr int kChunks8 = DIM / 16, kRows8 = 64 / kChunks8, kLoads8 = 16 / kRows8;
  static constexpr bool kCodes = FORMAT != QATTN_KV_16BIT;
  static_assert(kLds >= 4 * kFlatRows * DIM * 4, "O of four wavefronts");

  // Eight rows by two chunks cover all 64 banks.
  __device__ static uint32_t v_at(int r, int c) { return r * kRow + ((c ^ (DIM == 128 ? (r & 7) << 1 : (r & 6))) << 4); }

  // Per 16-key group: K's operand chunks (key lane & 15, dims 64 h + 16 (lane >> 4) + 8 half at step 2 h +
  // half) and V's rows as they lie.
  u32x4 k[2][kSteps], v[2][kLoads16];
  float ks[2], vs[2][kCodes ? kLoads8 : 1];

  // Tile `tile` of segment s, whose two groups are `group`.  (Rows past the last key: as in Tall.)
  __device__ void load(const Keys<FORMAT, DIM>& keys, const SharedSeg& s, int tile, const uint32_t (&group)[2], int lane) {
    const int key = lane & 15, c = lane >> 4;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (s.source == kOwnRows) {
        const int first = tile * kFlatKeys + 16 * b, last = s.keys - 1;
        const char* src = keys.row(0, s.base + min(first + key, last), 32 * c);
#pragma unroll
        for (int st = 0; st < kSteps; ++st) k[b][st] = *reinterpret_cast<const u32x4*>(src + 128 * (st >> 1) + 16 * (st & 1));
#pragma unroll
        for (int j = 0; j < kLoads16; ++j)
          v[b][j] = *reinterpret_cast<const u32x4*>(
              keys.row(1, s.base + min(first + j * kRows16 + lane / kChunks16, last), lane % kChunks16 * 16));
      } else {
        const char* src = keys.in_group(0, group[b], key * keys.kBytes + (kCodes ? 16 : 32) * c);
        const char* rows = keys.in_group(1, group[b], lane * 16);
        if constexpr (kCodes) {
#pragma unroll
          for (int h = 0; h < DIM / 64; ++h) k[b][h] = *reinterpret_cast<const u32x4*>(src + 64 * h);
          ks[b] = keys.scale_of(0, group[b], key);
        } else {
#pragma unroll
          for (int st = 0; st < kSteps; ++st) k[b][st] = *reinterpret_cast<const u32x4*>(src + 128 * (st >> 1) + 16 * (st & 1));
        }
#pragma unroll
        for (int j = 0; j < (kCodes ? kLoads8 : kLoads16); ++j) {
          v[b][j] = *reinterpret_cast<const u32x4*>(rows + j * 1024);
          if constexpr (kCodes) vs[b][j] = keys.scale_of(1, group[b], j * kRows8 + lane / kChunks8);
        }
      }
    }
  }
  // The K operands of group b at every step.
  __device__ void operands(int b, const SharedSeg& s, u32x4 (&out)[kSteps]) const {
    if (!kCodes || s.source == kOwnRows) {
#pragma unroll
      for (int st = 0; st < kSteps; ++st) out[st] = k[b][st];
    } else {
#pragma unroll
      for (int h = 0; h < DIM / 64; ++h) {
        u32x4 x[2];
        expand<BF16, FORMAT>(k[b][h], ks[b], x);
        out[2 * h] = x[0];
        out[2 * h + 1] = x[1];
      }
    }
  }
  __device__ bool store(char* lds, const SharedSeg& s, int lane, bool partly) const {
    bool any = false;
    const auto put = [&](int r, int c, u32x4 x) {
      if (partly) any |= drop_nonfinite<BF16>(x);
      *reinterpret_cast<u32x4*>(lds + v_at(r, c)) = x;
    };
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (!kCodes || s.source == kOwnRows) {
#pragma unroll
        for (int j = 0; j < kLoads16; ++j) put(16 * b + j * kRows16 + lane / kChunks16, lane % kChunks16, v[b][j]);
      } else {
#pragma unroll
        for (int j = 0; j < kLoads8; ++j) {
          const int r = 16 * b + j * kRows8 + lane / kChunks8, c = 2 * (lane % kChunks8);
          u32x4 x[2];
          expand<BF16, FORMAT>(v[b][j], vs[b][kCodes ? j : 0], x);
          put(r, c, x[0]);
          put(r, c + 1, x[1]);
        }
      }
    }
    return partly && __any(any);
  }
};

template <bool BF16, int FORMAT, int DIM>
__device__ inline void flat_item(const SharedParams& p, const SharedItem& it, int index, int kvh, char* lds_all, float2* stats) {
  typedef Flat<BF16, FORMAT, DIM> T;
  constexpr int kBlocks = DIM / 16;
  const int lane = threadIdx.x & 63, n = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* lds = lds_all + wave * (T::kLds / 4);
  const int end_row = it.row0 + it.rows, row = it.row0 + n;
  const bool exists = row < end_row;
  const int token = exists ? row / p.group : 0;
  const int at = exists ? p.positions[token] : -1;
  const bool local = p.mask != QATTN_MASK_CAUSAL;

  // Q (B operand): this lane's row, the dims of K's chunks.
  u32x4 q[T::kSteps];
  {
    const int head = kvh * p.group + row - token * p.group;
    const uint16_t* src = p.q + (int64_t)token * p.q_stride + head * DIM + 16 * c;
#pragma unroll
    for (int st = 0; st < T::kSteps; ++st)
      q[st] = exists ? *reinterpret_cast<const u32x4*>(src + 64 * (st >> 1) + 8 * (st & 1)) : u32x4{};
  }
  f4 o[kBlocks];
#pragma unroll
  for (int db = 0; db < kBlocks; ++db) o[db] = f4{};
  float m = kNone, l = 0.f;
  // V^T: the 16 lanes of group c read keys 4 c .. 4 c + 3 (and 16 more) by the 16 dims of a block.
  const int vr = 4 * c + (n >> 2);

  const Keys<FORMAT, DIM> keys(p, kvh);
  if (wave < it.tiles) {
    bool found = false;  // infinities or NaN were dropped from V
    Cursor now(p, it);
    now.advance(wave);
    T tile;
    uint32_t group[2] = {(uint32_t)item_group(p, index, 2 * wave), (uint32_t)item_group(p, index, 2 * wave + 1)};
    tile.load(keys, now.seg, now.tile, group, lane);
    // The next tile's groups are on the way while this one is worked on.
    int zero = 0;
    asm volatile("" : "+v"(zero));
    Cursor ahead = now;
    const auto ask_groups = [&]() {
      ahead.advance(4);
#pragma unroll
      for (int b = 0; b < 2; ++b) group[b] = group_of(p, ahead.seg, ahead.tile * kFlatKeys + 16 * b, zero);
    };
    if (wave + 4 < it.tiles) ask_groups();
    for (int t = wave; t < it.tiles; t += 4) {
      const SharedSeg s = now.seg;
      const int first = now.tile * kFlatKeys, from = s.position + first;
      f4 sc[2] = {};
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        u32x4 a[T::kSteps];
        tile.operands(b, s, a);
#pragma unroll
        for (int st = 0; st < T::kSteps; ++st) sc[b] = mfma16<BF16>(a[st], q[st], sc[b]);
      }
      const bool part = !s.whole;
      found |= tile.store(lds, s, lane, part);
      if (t + 4 < it.tiles) {
        now = ahead;
        tile.load(keys, now.seg, now.tile, group, lane);
        if (t + 8 < it.tiles) ask_groups();
      }
      const bool mine = row >= s.row_begin && row < s.row_end;
      const int limit = min(mine ? at : -1, s.position + s.keys - 1);
      const int window_from = (mine ? at : -1) - p.window;
      if (part) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int pos = from + 16 * (r >> 2) + 4 * c + (r & 3);
          const bool hidden = (int)(pos > limit) | ((int)local & (int)(pos >= p.prefix) & (int)(pos <= window_from));
          sc[r >> 2][r & 3] = hidden ? kNone : sc[r >> 2][r & 3];
        }
      }
      float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                        fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
      top = rows_max(top) * p.scale_log2;
      if (__any(top > m + kLazy || (m == kNone && top > kNone))) {
        const float next = top > m + kLazy || m == kNone ? fmaxf(top, m) : m;
        const float keep = m == next ? 1.f : __builtin_amdgcn_exp2f(m - next);
#pragma unroll
        for (int db = 0; db < kBlocks; ++db) o[db] *= keep;
        l *= keep;
        m = next;
      }
      const float ref = m == kNone ? 0.f : m;
      u32x4 pf;
#pragma unroll
      for (int r = 0; r < 8; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[r >> 2][r & 3], p.scale_log2, -ref));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[r >> 2][(r & 3) + 1], p.scale_log2, -ref));
        l += p0 + p1;
        pf[r >> 1] = narrow2<BF16>(p0, p1);
      }
#pragma unroll
      for (int db = 0; db < kBlocks; ++db) {
        const char* src = lds + T::v_at(vr, 2 * db + ((n & 3) >> 1)) + ((n & 1) << 3);
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)src));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(src + 16 * T::kRow)));
        o[db] = mfma16<BF16>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pf, o[db]);
      }
    }
    if (found)
      each_nonfinite<BF16, FORMAT, DIM>(p, keys, it, row, at, kFlatKeys, wave, 4, [&](auto value, bool seen) {
#pragma unroll
        for (int db = 0; db < kBlocks; ++db) {
          const f4 x = value(16 * db + 4 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[db][e] += nonfinite(x[e], seen);
        }
      });
  }

  // The four wavefronts' sums: lane (n, c) holds dims 16 db + 4 c .. + 3 of row n.
  l = rows_sum(l);
  float* own = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int db = 0; db < kBlocks; ++db) *reinterpret_cast<f4*>(own + n * DIM + 16 * db + 4 * c) = o[db];
  if (c == 0) stats[16 * wave + n] = float2{m, l};
  __syncthreads();
  const int r = threadIdx.x >> 4, d = (threadIdx.x & 15) * (DIM / 16);
  if (it.row0 + r >= end_row) return;
  float2 st[4];
  float top = kNone, sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    st[w] = stats[16 * w + r];
    top = fmaxf(top, st[w].x);
  }
  float x[DIM / 16] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = __builtin_amdgcn_exp2f(st[w].x - (top == kNone ? 0.f : top));
    sum += f * st[w].y;
    const float* src = reinterpret_cast<const float*>(lds_all + w * (T::kLds / 4)) + r * DIM + d;
#pragma unroll
    for (int e = 0; e < DIM / 16; ++e) x[e] += f * src[e];
  }
  const int out_row = it.row0 + r, out_token = out_row / p.group;
  if (it.part < 0) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.o + (int64_t)out_token * p.o_stride +
                                                (kvh * p.group + out_row - out_token * p.group) * DIM + d);
#pragma unroll
    for (int e = 0; e < DIM / 16; e += 2) dst[e / 2] = narrow2<BF16>(x[e] * inv, x[e + 1] * inv);
  } else {
    const int64_t part = ((int64_t)it.part + r) * p.kv_heads + kvh;
#pragma unroll
    for (int e = 0; e < DIM / 16; ++e) p.part_o[part * DIM + d + e] = x[e];
    if (d == 0) p.part_ml[part] = float2{top, sum};
  }
}

template <bool BF16, int FORMAT, int DIM>
__global__ __launch_bounds__(kSharedThreads, 2) void shared_attn_kernel(SharedParams p) {
  __shared__ __attribute__((aligned(1024))) char lds[Tall<BF16, FORMAT, DIM>::kLds];
  __shared__ __attribute__((aligned(16))) float2 stats[4 * kFlatRows];
  const int kvh = (int)(blockIdx.x % (uint32_t)p.kv_heads);
  const int index = (int)(blockIdx.x / (uint32_t)p.kv_heads);
  const SharedItem it = item_at(p, index);
  if (it.kind == kTall)
    tall_item<BF16, FORMAT, DIM>(p, it, index, kvh, lds, reinterpret_cast<uint32_t*>(stats));
  else
    flat_item<BF16, FORMAT, DIM>(p, it, index, kvh, lds, stats);
}

// Merged rows: sum over a row's partial rows of 2^(m_i - max m) times its sums; a partial row that saw no
// key has m = -inf and weighs 0.  Without partial rows: zeros.  DIM / 4 lanes hold a row, a float4 each, and a
// lane's loads go out eight partial rows at a time.  WIDE: a whole workgroup takes one row, its groups of
// lanes every kGroups'th partial row (rows cut into many chunks: a chain of loads would set the time);
// else each group takes a row of its own.  Bound by latency: three dependent accesses.
template <bool BF16, int DIM, bool WIDE>
__global__ __launch_bounds__(kSharedThreads) void shared_merge_kernel(SharedParams p) {
  constexpr int kLanes = DIM / 4, kGroups = kSharedThreads / kLanes;
  __shared__ f4 sums[WIDE ? kSharedThreads : 1];
  __shared__ float2 stats[WIDE ? kGroups : 1];
  const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int64_t index = WIDE ? blockIdx.x : (int64_t)blockIdx.x * kGroups + group;
  const bool exists = index < (int64_t)p.n_merges * p.kv_heads;
  const int kvh = (int)(index % p.kv_heads);
  SharedMerge e{};
  if (exists) e = p.merges[index / p.kv_heads];
  const int count = e.group[0].count + e.group[1].count;
  constexpr int kFirst = WIDE ? 1 : 0, kStep = WIDE ? kGroups : 1, kBatch = 8;
  float top = kNone, sum = 0.f;
  f4 x = {};
  for (int i0 = kFirst * group; i0 < count; i0 += kBatch * kStep) {
    float2 ml[kBatch];
    f4 y[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * kStep;
      ml[j] = float2{kNone, 0.f};
      y[j] = f4{};
      if (i < count) {
        const bool second = i >= e.group[0].count;
        const int64_t row = second ? e.group[1].first + (int64_t)(i - e.group[0].count) * e.group[1].step
                                   : e.group[0].first + (int64_t)i * e.group[0].step;
        const int64_t part = row * p.kv_heads + kvh;
        ml[j] = p.part_ml[part];
        y[j] = *reinterpret_cast<const f4*>(p.part_o + part * DIM + 4 * lane);
      }
    }
    float most = top;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) most = fmaxf(most, ml[j].x);
    const float ref = most == kNone ? 0.f : most, keep = __builtin_amdgcn_exp2f(top - ref);
    sum *= keep;
    x *= keep;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float f = __builtin_amdgcn_exp2f(ml[j].x - ref);
      sum += f * ml[j].y;
      x += f * y[j];
    }
    top = most;
  }
  if constexpr (WIDE) {
    sums[threadIdx.x] = x;
    if (lane == 0) stats[group] = float2{top, sum};
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) top = fmaxf(top, stats[g].x);
    const float ref = top == kNone ? 0.f : top;
    sum = 0.f;
    x = f4{};
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const float f = __builtin_amdgcn_exp2f(stats[g].x - ref);
      sum += f * stats[g].y;
      x += f * sums[g * kLanes + lane];
    }
  }
  if (!exists) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int token = e.row / p.group;
  uint16_t* dst = p.o + (int64_t)token * p.o_stride + (kvh * p.group + e.row - token * p.group) * DIM + 4 * lane;
  *reinterpret_cast<u32x2*>(dst) = u32x2{narrow2<BF16>(x[0] * inv, x[1] * inv), narrow2<BF16>(x[2] * inv, x[3] * inv)};
}

template <bool BF16, int FORMAT, int DIM>
void launch_attn(const SharedParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((shared_attn_kernel<BF16, FORMAT, DIM>), dim3((unsigned)p.n_items * p.kv_heads), dim3(kSharedThreads),
                     0, stream, p);
}
template <bool BF16, int DIM>
hipError_t launch(const SharedParams& p, int format, hipStream_t stream) {
  if (p.n_items > 0) {
    switch (format) {
      case QATTN_KV_16BIT: launch_attn<BF16, QATTN_KV_16BIT, DIM>(p, stream); break;
      case QATTN_KV_E4M3: launch_attn<BF16, QATTN_KV_E4M3, DIM>(p, stream); break;
      default: launch_attn<BF16, QATTN_KV_INT8, DIM>(p, stream);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.n_merges > 0) {
    const int64_t rows = (int64_t)p.n_merges * p.kv_heads;
    constexpr int kGroups = kSharedThreads / (DIM / 4);
    if (p.most_parts > 8)
      hipLaunchKernelGGL((shared_merge_kernel<BF16, DIM, true>), dim3((unsigned)rows), dim3(kSharedThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((shared_merge_kernel<BF16, DIM, false>), dim3((unsigned)((rows + kGroups - 1) / kGroups)),
                         dim3(kSharedThreads), 0, stream, p);
    return hipGetLastError();
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_shared_attn(const SharedParams& p, int dtype, int format, int head_dim, hipStream_t stream) {
  if (dtype == QATTN_DTYPE_BF16)
    return head_dim == 64 ? launch<true, 64>(p, format, stream) : launch<true, 128>(p, format, stream);
  return head_dim == 64 ? launch<false, 64>(p, format, stream) : launch<false, 128>(p, format, stream);
}

}  // namespace qattn
