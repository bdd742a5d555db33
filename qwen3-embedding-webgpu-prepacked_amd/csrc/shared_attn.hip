// shared_attn.hip -- attention of a batch of sequences behind one shared prefix (qattn_shared_run_*).
//
// o[r] = sum_j p_rj v_j / sum_j p_rj, p_rj = 2^(c q_r . k_j - m_r), over the keys that row r sees: the
// prefix's, read from a paged cache that may hold 8-bit codes, and its sequence's own.  Rows of all
// sequences are stacked (row = query * group + head of the group), so one tile of prefix keys serves many
// rows, whatever sequences they belong to.  Three kinds of items share a launch, one workgroup to an item
// and KV head; the plan picks them by the costs that it lists:
//   tall   256 rows, 32 to each of eight wavefronts, over 128-key tiles that they share in LDS.
//   split  128 rows: four wavefronts take the tile's first 64 keys, four its last, and their sums are joined
//          at the end.  2.4 us a tile against tall's 4.0 (head_dim 128): dearer for a row, sooner done (16
//          queries of 10 to 150 tokens: 25 us, by tall items 33; 16 x 500 tokens: 457 us, by tall 366).
//   flat   16 rows (up to 16 single tokens of several sequences) over 32-key tiles, a run of them to each of
//          eight wavefronts, which keeps its own sum; K goes from memory straight into the MFMA operand, V
//          through the wavefront's own 8 KiB of LDS for the transposed read; the sums are joined at the end.
// Blocks (tall and split): S^T = K Q^T and O^T = V^T P^T on 32x32x16 MFMAs, a query row to a lane.  Codes
// become 16-bit elements once, on their way into LDS.  16 x 500 tokens behind 5,000 e4m3 keys (16 heads over
// 8, head_dim 128) take 366 us, 939 TFLOP/s where the library's 8,192-cubed product reaches 1,222.  Bound by
// the matrix cores and, in turn with them, the softmax's vector work: without its exponentials a launch is 8 %
// shorter, without its LDS reads 3 %; the wavefronts of a SIMD hardly overlap the two, staggered by half a step
// neither (that was 13 % slower), and one workgroup fills a CU's LDS and half its registers.  (At head_dim 128
// codes take all 256 of a lane's, int8 ones spill five; scalar registers are spilled by every kernel of blocks, 9
// to 78 of them.)
// Flat items are bound by latency (a step of 16 tokens takes 9.4 us with its merge, a call 3.8 at least), or
// by the cache's bytes: 256 tokens with 1,024 e4m3 keys each take 98 us, 5.6 TB/s of reads (a copy, which writes
// half of its bytes, moves 5.2).
// An item whose rows have keys elsewhere too (other chunks, other items) leaves its unnormalised f32
// sums, the row's reference m and its sum of p; shared_merge_kernel joins them.
//
// A row's reference moves only when a tile's maximum exceeds it by kLazy (in log2): p then stays below
// 2^kLazy, far inside fp16, and most tiles rescale nothing.  p is rounded to the storage type for the PV
// product, which moves each weight by at most half a step of that type; l sums the unrounded p in f32.
#include "shared_attn.h"

#include <utility>

#include "elem.h"

namespace qattn {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16x __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;
typedef __attribute__((address_space(4))) const int32_t const_i32;

constexpr int kMergeThreads = 256;
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
// Lane I of each 16-lane row, in all its lanes: an operand modifier.
template <int I>
__device__ inline float row_lane(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + I, 0xf, 0xf, true));
}
template <class F, int... I>
__device__ inline void each_index(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>{}), ...);
}
__device__ inline int wave_max(int x) {
  for (int d = 32; d; d >>= 1) x = max(x, __shfl_xor(x, d));
  return __builtin_amdgcn_readfirstlane(x);
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

// Tiles one after another, through segments: of a block, or of one wavefront of a flat item.
struct Cursor {
  const const_i32* words;
  int tile;
  SharedSeg seg;
  __device__ Cursor(const SharedParams& p, const SharedItem& it)
      : words((const const_i32*)(p.segs + it.seg_begin)), tile(it.seg.tile_begin), seg(it.seg) {}
  __device__ Cursor(const SharedParams& p, const const_i32* start)
      : words((const const_i32*)(p.segs + start[9])), tile(start[5]), seg(seg_at(start)) {}
  __device__ void advance() {
    if (++tile < seg.tile_end) return;
    words += sizeof(SharedSeg) / 4;
    seg = seg_at(words);
    tile = seg.tile_begin;
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
  __device__ f4 scales_of(int i, uint32_t group, uint32_t row) const {
    return *reinterpret_cast<const f4*>(scale[i] + ((uint64_t)group * 64 | 4 * row));
  }
  __device__ const char* row(int i, uint32_t row, uint32_t offset) const {
    return rows[i] + ((uint64_t)row * stride[i] + offset);
  }
};
// The rows behind a source's last key, in the last group of its last page, may hold anything.  Their scores are
// masked, but an infinity or NaN among their V must not start the repair that such values of keys need: it takes
// many times a launch (64 tokens behind 8,190 int8 keys 2,006 us in place of 29; 16-bit ones 317 in place of 26).
// So V is read from no row behind last_row, the last key's in the groups that end a source (its list is filled up
// with its last group), but of int8 caches: there any code is finite, and such rows' scales are passed over.
__device__ inline uint32_t last_row(int keys, int first) { return first + 16 <= keys ? 15 : (keys - 1) & 15; }
// The group of key `first` of a segment, loaded as a vector: it is waited for with the tile's other loads.
__device__ inline uint32_t group_of(const SharedParams& p, const SharedSeg& s, int first, int zero) {
  return s.source == kOwnRows ? 0 : (uint32_t)p.groups[zero + s.base + (first >> 4)];
}

// ---- int8 caches -----------------------------------------------------------------------------------
// A code times its scale would have to be rounded to a 16-bit element, K's and V's, which doubles the result's
// error.  Instead the products take the codes, which are exact: K's scale goes to the key's scores in f32, and
// V's to its weights.  A weight is rounded to 16 bits after that, so V's elements are the codes times a power
// of two 2^e near the scale (exact too, and finite for any code), and the weight's factor is scale / 2^e: for the
// scales that kv_write gives 1 to 2.02 (bf16, whose greatest scale is 2^121: 4.03), less for fp16 ones under 2^-24.
template <bool BF16>
__device__ inline float near_power(float scale) {
  const int e = min(max((int)(__float_as_uint(scale) >> 23 & 255u) - 127, BF16 ? -110 : -24), BF16 ? 119 : 8);
  return copysignf(ldexpf(1.f, e), scale);
}
// Not below 2^-8: a scale of 0 gives values that vanish in rounding.
template <bool BF16>
__device__ inline float value_factor(float scale) {
  const float f = scale / near_power<BF16>(scale);
  return f < 0x1p-8f ? 0x1p-8f : f;
}

// 16 codes of K (I = 0) or V (1) as two 16-byte chunks of 16-bit elements: an e4m3 code times its power of
// two, exactly but below the type's normal range; of an int8 code, exactly, the factor of its key is left out.
template <bool BF16, int FORMAT, int I>
__device__ inline void expand(u32x4 codes, float scale, u32x4 (&out)[2]) {
  typedef Elem<false>::T2 H2;
  if constexpr (FORMAT == QATTN_KV_E4M3) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const u32x2 y = e4m3_elems<BF16>(codes[e], scale);
      out[e >> 1][2 * (e & 1)] = y[0];
      out[e >> 1][2 * (e & 1) + 1] = y[1];
    }
  } else {
    const float two = I ? near_power<BF16>(scale) : 1.f;
    const H2 two2 = {(_Float16)two, (_Float16)two};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t h = int8_halves(codes[e >> 1])[e & 1];
      if constexpr (BF16)
        h = narrow2<true>(fmaf(widen<false, 0>(h), two, 0.f), fmaf(widen<false, 1>(h), two, 0.f));
      else if constexpr (I == 1)
        h = __builtin_bit_cast(uint32_t, __builtin_bit_cast(H2, h) * two2);
      out[e >> 2][e & 3] = h;
    }
  }
}

// ---- values that a row must not see ----------------------------------------------------------------
// A masked key's p is 0, but 0 times an infinity or NaN is NaN.  In tiles that some row of the item sees
// only part of, such elements of V are replaced by 0 on their way into LDS, and if there were any, the
// rows that do see the key get them added at the end: p times an infinity is that infinity.  (An int8 code's
// infinity or NaN is its key's factor's.)  Elsewhere it meets p as it was rounded, and sums that are scaled down:
// an infinity whose weight underflows there becomes NaN.
template <bool BF16>
__device__ inline void drop_nonfinite(u32x4& chunk) {
  constexpr uint32_t kExp = Elem<BF16>::kExponent;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool low = (chunk[e] & kExp) == kExp, high = ((chunk[e] >> 16) & kExp) == kExp;
    chunk[e] &= (low ? 0xFFFF0000u : 0xFFFFFFFFu) & (high ? 0x0000FFFFu : 0xFFFFFFFFu);
  }
}
// Bits 15 and 31 of the result are set if `seen`'s were or an element is infinite or NaN: adding the
// exponent's lowest bit carries out of an exponent of ones, and of no other.
template <bool BF16>
__device__ inline uint32_t see_nonfinite(uint32_t seen, u32x4 chunk) {
  constexpr uint32_t kExp = Elem<BF16>::kExponent, kLow = kExp & (0u - kExp);
#pragma unroll
  for (int e = 0; e < 4; ++e) seen |= (chunk[e] & (kExp << 16 | kExp)) + (kLow << 16 | kLow);
  return seen;
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
      if constexpr (FORMAT == QATTN_KV_INT8) {
        const u32x2 h = int8_halves(codes);
        return f4{widen<false, 0>(h[0]), widen<false, 1>(h[0]), widen<false, 0>(h[1]), widen<false, 1>(h[1])} * scale;
      }
      x = e4m3_elems<BF16>(codes, scale);
    }
  }
  return f4{widen<BF16, 0>(x[0]), widen<BF16, 1>(x[0]), widen<BF16, 0>(x[1]), widen<BF16, 1>(x[1])};
}
__device__ inline float nonfinite(float v, bool seen) { return seen && !(fabsf(v) < INFINITY) ? v : 0.f; }
// Calls add(value, seen) for every key of `tiles` tiles (of `size` keys) from c on that not all rows see (int8: for
// every key): value(d) is elements d .. d + 3 of its V, seen whether row `row` at position `at` sees it.
template <bool BF16, int FORMAT, int DIM, class Add>
__device__ inline void each_nonfinite(const SharedParams& p, const Keys<FORMAT, DIM>& keys, Cursor c, int tiles, int row,
                                      int at, int size, Add add) {
  for (int t = 0;;) {
    const SharedSeg s = c.seg;
    if (!s.whole || FORMAT == QATTN_KV_INT8) {
      const int mine = row >= s.row_begin && row < s.row_end ? at : -1;
      for (int key = c.tile * size; key < min(s.keys, (c.tile + 1) * size); ++key) {
        const int pos = s.position + key;
        add([&](int d) { return value_at<BF16, FORMAT, DIM>(p, keys, s, key, d); },
            pos <= mine && (p.mask == QATTN_MASK_CAUSAL || pos < p.prefix || pos > mine - p.window));
      }
    }
    if (++t >= tiles) return;
    c.advance();
  }
}

// ---- tall items -----------------------------------------------------------------------------------

template <bool BF16, int FORMAT, int DIM>
struct Tall {
  static constexpr int kRow = 2 * DIM;                  // bytes of a row in LDS
  static constexpr int kTile = kTallKeys * kRow;        // of K or V
  static constexpr int kLds = 4 * kTile;                // K and V, double buffered; O of four wavefronts in f32
  // 16-byte chunks of a row in memory, rows of a wavefront's load, loads per tile: of 16-bit rows, codes.
  static constexpr int kChunks16 = kRow / 16, kRows16 = 64 / kChunks16, kLoads16 = 16 / kRows16;
  static constexpr int kChunks8 = DIM / 16, kRows8 = 64 / kChunks8, kLoads8 = 16 / kRows8;
  static constexpr bool kCodes = FORMAT != QATTN_KV_16BIT;

  // 16-byte chunk c of row r, swizzled so that 16 rows' reads of one chunk (K) and the transposed reads
  // of four rows by four chunks (V) cover all 64 banks.
  __device__ static uint32_t k_at(int r, int c) { return r * kRow + ((c ^ (DIM == 128 ? r & 15 : (r >> 1) & 7)) << 4); }
  __device__ static uint32_t v_at(int r, int c) { return r * kRow + ((c ^ (DIM == 128 ? (r & 3) << 2 : (r & 2) << 1)) << 4); }

  // Where the 16 rows of a tile that this wavefront loads lie.  Rows of keys past the last are read as they
  // are (K and int8 codes of pages: their scores are masked) or as the last key's.
  struct Spot {
    uint32_t group;  // of pages
    uint32_t last;   // last_row
    int row, left;   // of p.rows: the first, and how many further there are
    int held;        // how many hold keys: 16 or more, all; 0 or less, none
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
      if constexpr (I && FORMAT != QATTN_KV_INT8) {
        constexpr int kRows = kCodes ? kRows8 : kRows16, kChunks = kCodes ? kChunks8 : kChunks16;
#pragma unroll
        for (int j = 0; j < (kCodes ? kLoads8 : kLoads16); ++j) {
          const uint32_t r = min((uint32_t)(j * kRows + lane / kChunks), at.last);
          raw[I][j] = *reinterpret_cast<const u32x4*>(keys.in_group(I, at.group, r * keys.kBytes + lane % kChunks * 16));
          if constexpr (kCodes) scale[I][j] = keys.scale_of(I, at.group, r);
        }
        return;
      }
      const char* src = keys.in_group(I, at.group, lane * 16);
#pragma unroll
      for (int j = 0; j < (kCodes ? kLoads8 : kLoads16); ++j) raw[I][j] = *reinterpret_cast<const u32x4*>(src + j * 1024);
      if constexpr (kCodes) {
#pragma unroll
        for (int j = 0; j < kLoads8; ++j) scale[I][j] = keys.scale_of(I, at.group, lane / kChunks8 + j * kRows8);
      }
    }
  }

  // The loaded K (I = 0) or V (1) into LDS as 16-bit elements, and in runs with an int8 cache its keys' factors: of
  // scores (K; scale_log2 included) and of weights (V).  partly: infinities and NaN are taken
  // out (of V, in tiles that some row sees only part of); returns whether there were any.
  template <int I>
  __device__ bool store(char* lds, float* factors, float scale_log2, const Spot& spot, int wave, int lane, bool partly) {
    const bool rows = spot.rows, fold = FORMAT == QATTN_KV_INT8 && !rows;
    const auto each = [&](auto put) {
      if (!kCodes || rows) {
#pragma unroll
        for (int j = 0; j < kLoads16; ++j)
          put(16 * wave + j * kRows16 + lane / kChunks16, lane % kChunks16, raw[I][j]);
      } else {
#pragma unroll
        for (int j = 0; j < kLoads8; ++j) {
          const int r = 16 * wave + j * kRows8 + lane / kChunks8, c = 2 * (lane % kChunks8);
          u32x4 x[2];
          expand<BF16, FORMAT, I>(raw[I][j], scale[I][kCodes ? j : 0], x);
          put(r, c, x[0]);
          put(r, c + 1, x[1]);
        }
      }
    };
    uint32_t seen = 0;
    each([&](int r, int c, u32x4 x) {
      if (I && partly && !fold) seen = see_nonfinite<BF16>(seen, x);
      *reinterpret_cast<u32x4*>(lds + (I ? v_at(r, c) : k_at(r, c))) = x;
    });
    if constexpr (FORMAT == QATTN_KV_INT8) {
      bool any = false;
#pragma unroll
      for (int j = 0; j < kLoads8; ++j) {
        float f = !fold ? 1.f : I ? value_factor<BF16>(scale[I][j]) : scale[I][j];
        if (I && !(f < INFINITY)) {
          any |= j * kRows8 + lane / kChunks8 < spot.held;
          f = 1.f;
        }
        float* at = factors + 16 * wave + j * kRows8 + lane / kChunks8;
        if (lane % kChunks8 == 0) at[I * kTallKeys] = I ? f : f * scale_log2;
      }
      if (fold) return I && __any(any);
    }
    if (!I || !partly || !__any(seen & 0x80008000u)) return false;
    each([&](int r, int c, u32x4 x) {
      drop_nonfinite<BF16>(x);
      *reinterpret_cast<u32x4*>(lds + v_at(r, c)) = x;
    });
    return true;
  }
};

// Offset of accumulator element r (0 .. 31 over the two 32-key blocks) from the tile's first key + 4 hl.
__device__ constexpr int key_off(int r) { return 32 * (r >> 4) + 8 * ((r & 15) >> 2) + (r & 3); }

// Tile t is in LDS while tile t + 1 is in registers or on its way there: at the end of an iteration those go
// into the other buffers and tile t + 2 is asked for.
template <bool BF16, int FORMAT, int DIM>
__device__ inline void tall_item(const SharedParams& p, const SharedItem& it, int index, int kvh, char* lds, float* factors,
                                 float2* stats, uint32_t* dropped) {
  typedef Tall<BF16, FORMAT, DIM> T;
  constexpr int kBlocks = DIM / 32, kSteps = DIM / 16;
  const int lane = threadIdx.x & 63, lq = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The wavefront's rows, and its 64-key parts of a tile: both, or one of them.
  const bool split = it.kind == kSplit;
  const int part_begin = split ? wave >> 2 : 0, part_end = split ? part_begin + 1 : 2;
  const int end_row = it.row0 + it.rows, wave_row = it.row0 + 32 * (split ? wave & 3 : wave);
  const int row = wave_row + lq;
  const bool exists = row < end_row;
  const int token = exists ? row / p.group : 0;
  const int head = kvh * p.group + row - token * p.group;
  const int at = exists ? p.positions[token] : -1;
  const bool local = p.mask != QATTN_MASK_CAUSAL;

  // What the scores of a tile need to know of it.
  struct Info {
    int whole, from, last, row_begin, row_end;  // from: position of its first key; last: of its segment's last
  };
  const Keys<FORMAT, DIM> keys(p, kvh);
  Cursor ahead(p, it);  // the next tile to ask for, its group on the way
  T tile;
  int zero = 0;
  asm volatile("" : "+v"(zero));
  uint32_t group = item_group(p, index, wave);
  typename T::Spot spot{};
  int asked = 0;
  bool found = false;  // infinities or NaN were dropped from V
  if (threadIdx.x == 0) *dropped = 0;
  Info next{};  // of the tile in registers
  const auto ask = [&]() {
    const SharedSeg& s = ahead.seg;
    const int first = ahead.tile * kTallKeys + 16 * wave;
    spot.rows = s.source == kOwnRows;
    spot.group = group;
    spot.row = s.base + min(first, s.keys - 1);
    spot.left = max(s.keys - 1 - first, 0);
    spot.held = s.keys - first;
    spot.last = last_row(s.keys, first);
    tile.template load<0>(keys, spot, lane);
    tile.template load<1>(keys, spot, lane);
    next = Info{s.whole, s.position + ahead.tile * kTallKeys, s.position + s.keys - 1, s.row_begin, s.row_end};
    if (++asked < it.tiles) {
      ahead.advance();
      group = group_of(p, ahead.seg, ahead.tile * kTallKeys + 16 * wave, zero);
    }
  };
  const auto keep = [&](int t) {
    char* buf = lds + (t & 1) * 2 * T::kTile;
    float* f = factors + (t & 1) * 2 * kTallKeys;
    tile.template store<0>(buf, f, p.scale_log2, spot, wave, lane, false);
    found |= tile.template store<1>(buf + T::kTile, f, p.scale_log2, spot, wave, lane, !next.whole);
  };

  ask();
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
  const int greatest = wave_max(at);

  f16x o[kBlocks];
#pragma unroll
  for (int db = 0; db < kBlocks; ++db) o[db] = f16x{};
  float m = kNone, l = 0.f;

  // LDS read addresses.  K: rows lq, lq + 32.  V^T through the transposing read: in each 16-lane group G
  // lane a reads 4 elements of key 4 (G >> 1) + (a >> 2) (+ 16 st, + 8) at dims 32 db + 16 (G & 1) + 4 (a & 3)
  // and receives those keys' elements of dim 32 db + 16 (G & 1) + a.
  uint32_t v_read[kBlocks];
  {
    const int a = lane & 15, G = lane >> 4, r = 4 * (G >> 1) + (a >> 2);
#pragma unroll
    for (int db = 0; db < kBlocks; ++db) v_read[db] = T::v_at(r, 4 * db + 2 * (G & 1) + ((a & 3) >> 1)) + ((a & 1) << 3);
  }
  // Scores, weights and sums of the 64 keys at k, v, of which the first stands at position `from`.  Operands
  // are read ahead; the scheduling barriers keep the compiler from reading them all at once, for which there
  // are no registers.
  const auto add_part = [&](const Info& cur, int from, const char* k, const char* v, const float* f) {
    f16x sc[2];
    {
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
      __builtin_amdgcn_s_setprio(1);  // before the other wavefront's vector work: 2 %
#pragma unroll
      for (int i = 0; i < 2 * kSteps; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        sc[i & 1] = mfma32<BF16>(a[i % kAhead], q[i >> 1], i < 2 ? f16x{} : sc[i & 1]);
        if (i + kAhead < 2 * kSteps) a[i % kAhead] = k_frag(i + kAhead);
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(0);
    }
    // int8: this lane's row of 16 holds the factors of its half's keys, elements 0 .. 15 and 16 .. 31; the scores get
    // theirs, with scale_log2, here, else that comes in with the exponential.  (A read of LDS for each lane's
    // operands would take twice the bandwidth that K and V do at head_dim 64.)
    constexpr bool kFold = FORMAT == QATTN_KV_INT8;
    const float unit = kFold ? 1.f : p.scale_log2;
    float kf[2] = {}, vf[2] = {};
    if constexpr (kFold) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float* mine = f + 32 * b + 8 * ((lane & 15) >> 2) + 4 * hl + (lane & 3);
        kf[b] = mine[0];
        vf[b] = mine[kTallKeys];
      }
      each_index(std::make_integer_sequence<int, 32>{}, [&](auto r) {
        constexpr int R = decltype(r)::value;
        sc[R >> 4][R & 15] *= row_lane<R & 15>(kf[R >> 4]);
      });
    }
    if (!cur.whole) {
      // Offsets from this lane's first key: the last one seen, and where the prefix and the window leave a gap.
      const int mine = row >= cur.row_begin && row < cur.row_end ? at : -1;
      const int base = from + 4 * hl, last = min(mine, cur.last) - base;
#pragma unroll
      for (int r = 0; r < 32; ++r) sc[r >> 4][r & 15] = key_off(r) > last ? kNone : sc[r >> 4][r & 15];
      if (local && from + 64 > p.prefix && from <= it.greatest - p.window) {
        const int gap = p.prefix - base, window = mine - p.window - base;
#pragma unroll
        for (int r = 0; r < 32; ++r) {
          const int off = key_off(r);
          sc[r >> 4][r & 15] = (int)(off >= gap) & (int)(off <= window) ? kNone : sc[r >> 4][r & 15];
        }
      }
    }
    float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), sc[0][2]);
#pragma unroll
    for (int r = 3; r < 31; r += 2) top = fmaxf(fmaxf(top, sc[r >> 4][r & 15]), sc[(r + 1) >> 4][(r + 1) & 15]);
    top = half_max(fmaxf(top, sc[1][15])) * unit;
    if (__any(top > m + kLazy)) {  // from -inf too: any score exceeds it
      const float moved = top > m + kLazy ? top : m;
      const float shrink = m == moved ? 1.f : __builtin_amdgcn_exp2f(m - moved);
      m = moved;
      l *= shrink;
#pragma unroll
      for (int db = 0; db < kBlocks; ++db) o[db] *= shrink;
    }
    const float ref = m == kNone ? 0.f : m;
    // Slot j of half hl at step st is key 16 st + 8 (j >> 2) + 4 hl + (j & 3): element 8 st + j of the scores.
    u32x4 pf[4];
    float sum[2] = {};
    each_index(std::make_integer_sequence<int, 16>{}, [&](auto i) {
      constexpr int R = 2 * decltype(i)::value, B = R >> 4, E = R & 15;
      float p0 = __builtin_amdgcn_exp2f(kFold ? sc[B][E] - ref : fmaf(sc[B][E], unit, -ref));
      float p1 = __builtin_amdgcn_exp2f(kFold ? sc[B][E + 1] - ref : fmaf(sc[B][E + 1], unit, -ref));
      sum[0] += p0;
      sum[1] += p1;
      if constexpr (kFold) {
        p0 *= row_lane<E>(vf[B]);
        p1 *= row_lane<E + 1>(vf[B]);
      }
      pf[R >> 3][(R & 7) >> 1] = narrow2<BF16>(p0, p1);
    });
    l += sum[0] + sum[1];
    const auto v_frag = [&](int i) {
      const char* src = v + v_read[i % kBlocks] + i / kBlocks * 16 * T::kRow;
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)src));
      const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(src + 8 * T::kRow)));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    constexpr int kDeep = 4;
    u32x4 a[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) a[i] = v_frag(i);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < 4 * kBlocks; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      o[i % kBlocks] = mfma32<BF16>(a[i % kDeep], pf[i / kBlocks], o[i % kBlocks]);
      if (i + kDeep < 4 * kBlocks) a[i % kDeep] = v_frag(i + kDeep);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
  };

  keep(0);
  Info now = next;
  if (it.tiles > 1) ask();
  for (int t = 0; t < it.tiles; ++t) {
    __syncthreads();
    const char* buf = lds + (t & 1) * 2 * T::kTile;
    // Parts of which some row of this wavefront sees a key.
    if (wave_row < end_row && (now.whole || (now.row_begin < wave_row + 32 && now.row_end > wave_row))) {
      for (int part = part_begin; part < part_end; ++part) {
        const int from = now.from + 64 * part;
        if (now.whole || from <= min(greatest, now.last))
          add_part(now, from, buf + part * 64 * T::kRow, buf + T::kTile + part * 64 * T::kRow,
                   factors + (t & 1) * 2 * kTallKeys + 64 * part);
      }
    }
    if (t + 1 < it.tiles) {
      keep(t + 1);
      now = next;
      if (t + 2 < it.tiles) ask();
    }
  }
  if (found) *dropped = 1;
  __syncthreads();

  l = half_sum(l);
  if (split) {
    // The sums of wavefront w + 4 join those of w, over the tiles' LDS.
    f4* sums = reinterpret_cast<f4*>(lds) + (wave & 3) * (DIM / 8) * 64 + lane;
    if (wave >= 4) {
#pragma unroll
      for (int i = 0; i < DIM / 8; ++i)
        sums[64 * i] = f4{o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1], o[i >> 2][4 * (i & 3) + 2], o[i >> 2][4 * (i & 3) + 3]};
      if (hl == 0) stats[32 * (wave & 3) + lq] = float2{m, l};
    }
    __syncthreads();
    if (wave >= 4) return;
    const float2 other = stats[32 * wave + lq];
    const float top = fmaxf(m, other.x), ref = top == kNone ? 0.f : top;
    const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(other.x - ref);
    l = f0 * l + f1 * other.y;
    m = top;
#pragma unroll
    for (int i = 0; i < DIM / 8; ++i) {
      const f4 x = sums[64 * i];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i >> 2][4 * (i & 3) + e] = f0 * o[i >> 2][4 * (i & 3) + e] + f1 * x[e];
    }
  }
  // After the join, where a half that sees no key weighs 0, and 0 times an infinity is NaN.
  if (*dropped)
    each_nonfinite<BF16, FORMAT, DIM>(p, keys, Cursor(p, it), it.tiles, row, at, kTallKeys, [&](auto value, bool seen) {
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
  static constexpr int kLds = kFlatWaves * kFlatKeys * kRow;  // each wavefront's V tile, later its 16 rows of O in f32
  static constexpr int kSteps = DIM / 32;            // K: two 16-byte loads of codes, four of 16-bit elements per 128 dims
  static constexpr int kChunks16 = kRow / 16, kRows16 = 64 / kChunks16, kLoads16 = 16 / kRows16;
  static constexpr int kChunks8 = DIM / 16, kRows8 = 64 / kChunks8, kLoads8 = 16 / kRows8;
  static constexpr bool kCodes = FORMAT != QATTN_KV_16BIT;
  static_assert(kLds >= kFlatWaves * kFlatRows * DIM * 4, "O of the wavefronts");

  // Eight rows by two chunks cover all 64 banks.
  __device__ static uint32_t v_at(int r, int c) { return r * kRow + ((c ^ (DIM == 128 ? (r & 7) << 1 : (r & 6))) << 4); }

  // Per 16-key group: K's operand chunks (key lane & 15, dims 64 h + 16 (lane >> 4) + 8 half at step 2 h +
  // half) and V's rows as they lie.
  u32x4 k[2][kSteps], v[2][kLoads16];
  float ks[2], vs[2][kCodes ? kLoads8 : 1];
  f4 kf[2], vf[2];  // int8: the scales of keys 4 (lane >> 4) + 0 .. 3 of each group

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
        // V's row at load j.
        const uint32_t last = FORMAT == QATTN_KV_INT8 ? 15 : last_row(s.keys, tile * kFlatKeys + 16 * b);
        constexpr int kRows = kCodes ? kRows8 : kRows16, kChunks = kCodes ? kChunks8 : kChunks16;
        const auto row_of = [&](int j) { return min((uint32_t)(j * kRows + lane / kChunks), last); };
        if constexpr (kCodes) {
#pragma unroll
          for (int h = 0; h < DIM / 64; ++h) k[b][h] = *reinterpret_cast<const u32x4*>(src + 64 * h);
          if constexpr (FORMAT == QATTN_KV_INT8) {
            kf[b] = keys.scales_of(0, group[b], 4 * c);
            vf[b] = keys.scales_of(1, group[b], 4 * c);
          } else {
            ks[b] = keys.scale_of(0, group[b], key);
          }
        } else {
#pragma unroll
          for (int st = 0; st < kSteps; ++st) k[b][st] = *reinterpret_cast<const u32x4*>(src + 128 * (st >> 1) + 16 * (st & 1));
        }
#pragma unroll
        for (int j = 0; j < (kCodes ? kLoads8 : kLoads16); ++j) {
          v[b][j] = *reinterpret_cast<const u32x4*>(keys.in_group(1, group[b], row_of(j) * keys.kBytes + lane % kChunks * 16));
          if constexpr (kCodes) vs[b][j] = keys.scale_of(1, group[b], row_of(j));
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
        expand<BF16, FORMAT, 0>(k[b][h], ks[b], x);
        out[2 * h] = x[0];
        out[2 * h + 1] = x[1];
      }
    }
  }
  __device__ bool store(char* lds, const SharedSeg& s, int lane, bool partly) const {
    const auto each = [&](auto put) {
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
            expand<BF16, FORMAT, 1>(v[b][j], vs[b][kCodes ? j : 0], x);
            put(r, c, x[0]);
            put(r, c + 1, x[1]);
          }
        }
      }
    };
    const bool fold = FORMAT == QATTN_KV_INT8 && s.source != kOwnRows;
    uint32_t seen = 0;
    each([&](int r, int c, u32x4 x) {
      if (partly && !fold) seen = see_nonfinite<BF16>(seen, x);
      *reinterpret_cast<u32x4*>(lds + v_at(r, c)) = x;
    });
    if (!partly || fold || !__any(seen & 0x80008000u)) return false;
    each([&](int r, int c, u32x4 x) {
      drop_nonfinite<BF16>(x);
      *reinterpret_cast<u32x4*>(lds + v_at(r, c)) = x;
    });
    return true;
  }
};

template <bool BF16, int FORMAT, int DIM>
__device__ inline void flat_item(const SharedParams& p, const SharedItem& it, int index, int kvh, char* lds_all, float2* stats) {
  typedef Flat<BF16, FORMAT, DIM> T;
  constexpr int kBlocks = DIM / 16;
  const int lane = threadIdx.x & 63, n = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* lds = lds_all + wave * (T::kLds / kFlatWaves);
  // Lanes past the item's rows repeat the last one; their results go nowhere.
  const int end_row = it.row0 + it.rows, row = min(it.row0 + n, end_row - 1);
  const int token = row / p.group;
  const int at = p.positions[token];
  const bool local = p.mask != QATTN_MASK_CAUSAL;

  // Q (B operand): this lane's row, the dims of K's chunks.
  u32x4 q[T::kSteps];
  {
    const int head = kvh * p.group + row - token * p.group;
    const uint16_t* src = p.q + (int64_t)token * p.q_stride + head * DIM + 16 * c;
#pragma unroll
    for (int st = 0; st < T::kSteps; ++st) q[st] = *reinterpret_cast<const u32x4*>(src + 64 * (st >> 1) + 8 * (st & 1));
  }
  f4 o[kBlocks];
#pragma unroll
  for (int db = 0; db < kBlocks; ++db) o[db] = f4{};
  float m = kNone, l = 0.f;
  // V^T: the 16 lanes of group c read keys 4 c .. 4 c + 3 (and 16 more) by the 16 dims of a block.
  const int vr = 4 * c + (n >> 2);

  const Keys<FORMAT, DIM> keys(p, kvh);
  const const_i32* start = (const const_i32*)(p.starts + index * kFlatWaves + wave);
  const int tiles = start[10];
  if (tiles) {
    bool found = false;  // infinities or NaN were dropped from V
    Cursor now(p, start);
    T tile;
    uint32_t group[2] = {(uint32_t)start[11], (uint32_t)start[12]};
    tile.load(keys, now.seg, now.tile, group, lane);
    // The next tile's groups are on the way while this one is worked on.
    int zero = 0;
    asm volatile("" : "+v"(zero));
    Cursor ahead = now;
    const auto ask_groups = [&]() {
      ahead.advance();
#pragma unroll
      for (int b = 0; b < 2; ++b) group[b] = group_of(p, ahead.seg, ahead.tile * kFlatKeys + 16 * b, zero);
    };
    if (tiles > 1) ask_groups();
    for (int t = 0; t < tiles; ++t) {
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
      f4 factor[2] = {{1.f, 1.f, 1.f, 1.f}, {1.f, 1.f, 1.f, 1.f}};
      if constexpr (FORMAT == QATTN_KV_INT8)
        if (s.source != kOwnRows) {
          bool any = false;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            sc[r >> 2][r & 3] *= tile.kf[r >> 2][r & 3];
            float f = value_factor<BF16>(tile.vf[r >> 2][r & 3]);
            if (!(f < INFINITY)) {
              any |= 16 * (r >> 2) + 4 * c + (r & 3) < s.keys - first;
              f = 1.f;
            }
            factor[r >> 2][r & 3] = f;
          }
          found |= __any(any);
        }
      found |= tile.store(lds, s, lane, part);
      if (t + 1 < tiles) {
        now = ahead;
        tile.load(keys, now.seg, now.tile, group, lane);
        if (t + 2 < tiles) ask_groups();
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
        pf[r >> 1] = FORMAT == QATTN_KV_INT8 ? narrow2<BF16>(p0 * factor[r >> 2][r & 3], p1 * factor[r >> 2][(r & 3) + 1])
                                             : narrow2<BF16>(p0, p1);
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
      each_nonfinite<BF16, FORMAT, DIM>(p, keys, Cursor(p, start), tiles, row, at, kFlatKeys, [&](auto value, bool seen) {
#pragma unroll
        for (int db = 0; db < kBlocks; ++db) {
          const f4 x = value(16 * db + 4 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[db][e] += nonfinite(x[e], seen);
        }
      });
  }

  // The wavefronts' sums: lane (n, c) holds dims 16 db + 4 c .. + 3 of row n.  Rows start at the same bank: their
  // 16-byte chunks are swizzled.
  const auto chunk_at = [](int r, int chunk) { return r * DIM + ((chunk ^ (r & 3) << 2) << 2); };
  l = rows_sum(l);
  float* own = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int db = 0; db < kBlocks; ++db) *reinterpret_cast<f4*>(own + chunk_at(n, 4 * db + c)) = o[db];
  if (c == 0) stats[kFlatRows * wave + n] = float2{m, l};
  __syncthreads();
  constexpr int kLanes = kSharedThreads / kFlatRows, kEach = DIM / kLanes;
  typedef float Part __attribute__((ext_vector_type(kEach)));
  const int r = threadIdx.x / kLanes, d = threadIdx.x % kLanes * kEach;
  if (it.row0 + r >= end_row) return;
  float2 st[kFlatWaves];
  float top = kNone, sum = 0.f;
#pragma unroll
  for (int w = 0; w < kFlatWaves; ++w) {
    st[w] = stats[kFlatRows * w + r];
    top = fmaxf(top, st[w].x);
  }
  Part x = {};
#pragma unroll
  for (int w = 0; w < kFlatWaves; ++w) {
    const float f = __builtin_amdgcn_exp2f(st[w].x - (top == kNone ? 0.f : top));
    sum += f * st[w].y;
    x += f * *reinterpret_cast<const Part*>(reinterpret_cast<const float*>(lds_all + w * (T::kLds / kFlatWaves)) + chunk_at(r, d / 4) + d % 4);
  }
  const int out_row = it.row0 + r, out_token = out_row / p.group;
  if (it.part < 0) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.o + (int64_t)out_token * p.o_stride +
                                                (kvh * p.group + out_row - out_token * p.group) * DIM + d);
#pragma unroll
    for (int e = 0; e < kEach; e += 2) dst[e / 2] = narrow2<BF16>(x[e] * inv, x[e + 1] * inv);
  } else {
    const int64_t part = ((int64_t)it.part + r) * p.kv_heads + kvh;
    *reinterpret_cast<Part*>(p.part_o + part * DIM + d) = x;
    if (d == 0) p.part_ml[part] = float2{top, sum};
  }
}

template <bool BF16, int FORMAT, int DIM>
__global__ __launch_bounds__(kSharedThreads, 2) void shared_attn_kernel(SharedParams p) {
  constexpr int kTallLds = Tall<BF16, FORMAT, DIM>::kLds, kFlatLds = Flat<BF16, FORMAT, DIM>::kLds;
  static_assert(kTallLds >= kFlatLds && kTallLds >= 4 * 32 * DIM * 4, "O of four wavefronts");
  __shared__ __attribute__((aligned(1024))) char lds[kTallLds];
  __shared__ __attribute__((aligned(16))) float2 stats[128];
  __shared__ __attribute__((aligned(16))) float factors[FORMAT == QATTN_KV_INT8 ? 4 * kTallKeys : 1];  // of two tiles' keys
  __shared__ uint32_t dropped;
  const int kvh = (int)(blockIdx.x % (uint32_t)p.kv_heads);
  const int unit = (int)(blockIdx.x / (uint32_t)p.kv_heads);
  const int index = !p.flat_first ? unit : unit < p.n_flat ? p.n_blocks + unit : unit - p.n_flat;
  const SharedItem it = item_at(p, index);
  if (index < p.n_blocks)
    tall_item<BF16, FORMAT, DIM>(p, it, index, kvh, lds, factors, stats, &dropped);
  else
    flat_item<BF16, FORMAT, DIM>(p, it, index - p.n_blocks, kvh, lds, stats);
}

// Launches of flat items alone: with half the LDS, a workgroup starts sooner (single tokens with 32 keys: 4.5 us,
// by the kernel of all kinds 5.7).
template <bool BF16, int FORMAT, int DIM>
__global__ __launch_bounds__(kSharedThreads, 2) void shared_flat_kernel(SharedParams p) {
  __shared__ __attribute__((aligned(1024))) char lds[Flat<BF16, FORMAT, DIM>::kLds];
  __shared__ __attribute__((aligned(16))) float2 stats[kFlatWaves * kFlatRows];
  const int kvh = (int)(blockIdx.x % (uint32_t)p.kv_heads), index = (int)(blockIdx.x / (uint32_t)p.kv_heads);
  flat_item<BF16, FORMAT, DIM>(p, item_at(p, index), index, kvh, lds, stats);
}

// Merged rows: sum over a row's partial rows of 2^(m_i - max m) times its sums; a partial row that saw no
// key has m = -inf and weighs 0.  Without partial rows: zeros.  DIM / 4 lanes hold a row, a float4 each, and a
// lane's loads go out eight partial rows at a time.  WIDE, for rows of more than eight partial rows: a whole
// workgroup takes one row, its groups of lanes every kGroups'th partial row, for a chain of loads would set
// the time (8 tokens, 38 partial rows: 12.9 us for both launches against 16.3); else each group takes a row
// of its own (3,000 rows of up to three: 53 us against 74).  Bound by latency, three dependent accesses (3 us
// for a step of eight), then by the partial rows' bytes.
template <bool BF16, int DIM, bool WIDE>
__global__ __launch_bounds__(kMergeThreads) void shared_merge_kernel(SharedParams p) {
  constexpr int kLanes = DIM / 4, kGroups = kMergeThreads / kLanes;
  __shared__ f4 sums[WIDE ? kMergeThreads : 1];
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
  const dim3 grid((unsigned)(p.n_blocks + p.n_flat) * p.kv_heads);
  if (p.n_blocks == 0)
    hipLaunchKernelGGL((shared_flat_kernel<BF16, FORMAT, DIM>), grid, dim3(kSharedThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((shared_attn_kernel<BF16, FORMAT, DIM>), grid, dim3(kSharedThreads), 0, stream, p);
}
template <bool BF16, int DIM>
hipError_t launch(const SharedParams& p, int format, hipStream_t stream) {
  if (p.n_blocks + p.n_flat > 0) {
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
    constexpr int kGroups = kMergeThreads / (DIM / 4);
    if (p.most_parts > 8)
      hipLaunchKernelGGL((shared_merge_kernel<BF16, DIM, true>), dim3((unsigned)rows), dim3(kMergeThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((shared_merge_kernel<BF16, DIM, false>), dim3((unsigned)((rows + kGroups - 1) / kGroups)),
                         dim3(kMergeThreads), 0, stream, p);
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
