// w4_matmul.hip -- products of 8-bit rows with 4-bit weights: y[m][n] = x_scale[m] * w_scale[n] * sum_k x[m][k] *
// (code[n][k] - zero[n][k / 32]) * multiplier[n][k / 32], and SwiGLU of two such products.
//
// A group's scale is a whole number, so it goes into the 8-bit weight and the sum over all of K runs in whole
// numbers on the matrix cores (v_mfma_i32_16x16x64_i8, twice the rate of the 16-bit form); the two f32 scales meet
// it once, at the end.  With an f32 scale for each group every 16 x 16 sum would have to leave the matrix cores at
// each group: 8 vector instructions for 8 clocks of matrix work.  Whole-number sums are exact in any order, so K is
// split and joined as suits a launch and a row's result does not depend on its batch.
//
// Four weights cost three vector instructions and half a shift: nibbles to bytes, byte * multiplier + (128 - zero *
// multiplier) in two 16-bit halves -- neither byte leaves [0, 255], so none carries -- and the top bit flipped.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "elem.h"
#include "w4_ops.h"

namespace qattn {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

#define W4_INLINE __attribute__((always_inline))

// The memory and matrix builtins behind plain (non-template) device functions: hipcc's host pass drops a kernel
// template's host stub when such a builtin sits in a dependent context.
__device__ inline __amdgpu_buffer_rsrc_t rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}
// The range check covers the per-lane offset, not a scalar one: what may lie past a row's end goes into the former.
__device__ inline i32x4 load16(__amdgpu_buffer_rsrc_t rs, uint32_t off) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
}
__device__ inline uint32_t load1(__amdgpu_buffer_rsrc_t rs, uint32_t off) { return __builtin_amdgcn_raw_buffer_load_b8(rs, off, 0, 0); }
__device__ inline i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

typedef __attribute__((address_space(3))) void lds_void_t;
__device__ inline void dma16(__amdgpu_buffer_rsrc_t rs, char* dst, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)dst, 16, off, 0, 0, 0);
}
// Waits for all but the newest V vector-memory operations, or for all LDS reads, of this wavefront.
template <int V>
__device__ inline void wait_but() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(V) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}
__device__ inline void wait_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A group's multiplier in both halves of a dword, and 128 - zero * multiplier in its four bytes.
struct Group {
  uint32_t mult, bias;
};
__device__ inline Group group_of(uint32_t byte) {
  const uint32_t m = byte & 15u, z = byte >> 4 & 15u;
  return {__builtin_amdgcn_perm(0, m, 0x0C000C00u), __builtin_amdgcn_perm(0, 128u - m * z, 0u)};
}
__device__ inline uint32_t weights4(uint32_t nibbles, Group g) {
  const u16x2 v = __builtin_bit_cast(u16x2, nibbles) * __builtin_bit_cast(u16x2, g.mult) + __builtin_bit_cast(u16x2, g.bias);
  return __builtin_bit_cast(uint32_t, v) ^ 0x80808080u;
}
// The 16 weights of a record's low (HIGH = 0) or high nibbles.
template <int HIGH>
__device__ inline i32x4 weights16(i32x4 record, Group g) {
  i32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (int)weights4((uint32_t)record[i] >> (4 * HIGH) & 0x0F0F0F0Fu, g);
  return w;
}

// Results rounded to f32 before they are to 16 bits: otherwise some are by one instruction that multiplies and rounds
// once, and a row's result would depend on the kernel that its batch takes.
template <bool BF16>
__device__ inline u32x2 narrow4(const float (&f)[4]) {
  float a = f[0], b = f[1], c = f[2], d = f[3];
  asm("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
  return u32x2{narrow2<BF16>(a, b), narrow2<BF16>(c, d)};
}

// silu(g) * u.  The hardware's exp2 and reciprocal are within about an f32 ulp, far inside the result's rounding.
__device__ inline float swiglu(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504f)) * u;
}

// ---- few rows: a workgroup to 16 MB rows and 16 NB columns (SwiGLU: 8 NB features), whose W wavefronts take the
// blocks of 128 columns of K in turn, U of them in flight, and add up in LDS.  A lane's 16 bytes of codes are two
// fragments as they come.  X goes through LDS, a region to each wavefront: the 16 rows of a fragment are as many cache
// lines to a load of its own, which the address unit takes one by one (64 clocks; 16 by rows, as here).
// One row is bound by the weights (1 x 4,096 -> 8,192: 5.1 us, 3.5 TB/s with the launch), 16 to 64 by launch and latency (16 x
// 1,024 -> 4,096: 3.1 us), more by the blocks that a wavefront takes one after the other (333 x 2,592 -> 1,001: 6.3 us).
template <bool BF16, bool SWIGLU, int MB, int NB, int W, int U>
__global__ __launch_bounds__(64 * W) void w4_small_kernel(W4Product p, int blocks_m) {
  static_assert(!SWIGLU || NB % 2 == 0, "as many gate tiles as up tiles");
  static_assert(U >= 1 && U <= 2 && NB * MB * 1024 <= U * 2048 * MB, "two buffers, which take a wavefront's sums in the end");
  constexpr int kRegion = 2048 * MB;
  __shared__ __attribute__((aligned(1024))) char sX0[W * kRegion];
  __shared__ __attribute__((aligned(1024))) char sX1[U > 1 ? W * kRegion : 16];
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m0 = (int64_t)(blockIdx.x % (unsigned)blocks_m) * (16 * MB);
  const int nblk = (int)(blockIdx.x / (unsigned)blocks_m);
  const W4Layout at(p.K, p.N);
  const int blocks = (int)at.blocks;
  // Tiles of 16 weight rows (SwiGLU: the gate's, then the up projection's); those past the last read as zeros, and so
  // do blocks past K: a group byte of zero makes weights of zero.
  const int tile0 = SWIGLU ? NB / 2 * nblk : NB * nblk;
  __amdgpu_buffer_rsrc_t codes[NB], groups[NB];
  int tile[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    tile[nb] = SWIGLU ? tile0 + nb % (NB / 2) + (nb < NB / 2 ? 0 : p.N >> 5) : tile0 + nb;
    const bool here = tile[nb] < at.tiles;
    codes[nb] = rsrc(p.w + (int64_t)tile[nb] * blocks * 1024, here ? (uint32_t)blocks * 1024u : 0u);
    groups[nb] = rsrc(p.w + at.groups_at() + (int64_t)tile[nb] * blocks * 64, here ? (uint32_t)blocks * 64u : 0u);
  }
  // Rows past M and what lies behind the last row's K columns read as zeros; columns of K's padding meet zero weights.
  // Rows of 128 bytes in LDS, piece c of row r at c ^ ((r >> 1) & 7).
  const int rows = (int)(p.M - m0 < 16 * MB ? p.M - m0 : 16 * MB);
  const uint32_t x_bytes = (uint32_t)(rows - 1) * (uint32_t)p.ldx + (uint32_t)p.K;
  uint32_t x_src[2 * MB];
#pragma unroll
  for (int j = 0; j < 2 * MB; ++j) {
    const int row = 8 * j + (lane >> 3);
    x_src[j] = (uint32_t)row * (uint32_t)p.ldx + 16u * ((lane & 7) ^ ((row >> 1) & 7));
  }
  const uint32_t x_rd = l16 * 128 + (((2 * q) ^ ((l16 >> 1) & 7)) << 4);
  auto region = [&](int i) W4_INLINE { return (i ? sX1 : sX0) + wave * kRegion; };

  struct Weights {
    i32x4 record[NB];
    uint32_t group[NB];
  };
  auto load_x = [&](char* dst, int kb) W4_INLINE {
    const auto xs = rsrc(p.x + m0 * p.ldx, kb < blocks ? x_bytes : 0u);  // nothing past the last block
#pragma unroll
    for (int j = 0; j < 2 * MB; ++j) dma16(xs, dst + 1024 * j, x_src[j] + 128u * (uint32_t)kb);
  };
  auto load_w = [&](Weights& w, int kb) W4_INLINE {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      w.record[nb] = load16(codes[nb], 1024u * (uint32_t)kb + 16u * lane);
      w.group[nb] = load1(groups[nb], 64u * (uint32_t)kb + 4u * l16 + q);
    }
  };
  i32x4 acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB * MB; ++i) acc[i / MB][i % MB] = i32x4{};
  // Of the 16 x 16 sums (SwiGLU: pairs of them) each of the first wavefronts finishes as many; their scales.
  constexpr int kUnits = SWIGLU ? MB * NB / 2 : MB * NB, kEach = kUnits > W ? kUnits / W : 1;
  static_assert(kUnits <= W || kUnits % W == 0, "as many for each wavefront");
  float x_scale[kEach];
  float4 w_scale[kEach], up_scale[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int unit = wave + W * j, nb = unit / MB, row = 16 * (unit % MB) + l16;
    x_scale[j] = 0.f;
    w_scale[j] = up_scale[j] = float4{};
    if (unit >= kUnits) continue;
    const float4* const scales = reinterpret_cast<const float4*>(p.w + at.scales_at());
    if (row < rows) x_scale[j] = p.x_scale[m0 + row];
    if (tile0 + nb < at.tiles) w_scale[j] = scales[4 * (tile0 + nb) + q];
    if (SWIGLU && tile0 + nb + (p.N >> 5) < at.tiles) up_scale[j] = scales[4 * (tile0 + nb + (p.N >> 5)) + q];
  }
  __builtin_amdgcn_sched_barrier(0);
  Weights ring[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    load_x(region(i), wave + W * i);
    load_w(ring[i], wave + W * i);
    __builtin_amdgcn_sched_barrier(0);
  }
  // Blocks past the end are loads of zeros: as many loads are in flight at each wait.
  for (int kb = wave; kb < blocks; kb += W * U) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      // X of this block has landed: newer are the U - 1 blocks behind it.
      wait_but<(U - 1) * (2 * MB + 2 * NB)>();
      i32x4 x[MB][2];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        x[mb][0] = *reinterpret_cast<const i32x4*>(region(i) + x_rd + 2048 * mb);
        x[mb][1] = *reinterpret_cast<const i32x4*>(region(i) + (x_rd ^ 16) + 2048 * mb);
      }
      wait_lds();
      load_x(region(i), kb + W * (U + i));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const Group g = group_of(ring[i].group[nb]);
        const i32x4 lo = weights16<0>(ring[i].record[nb], g), hi = weights16<1>(ring[i].record[nb], g);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[nb][mb] = mfma(lo, x[mb][0], acc[nb][mb]);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[nb][mb] = mfma(hi, x[mb][1], acc[nb][mb]);
      }
      load_w(ring[i], kb + W * (U + i));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // A wavefront's sums take the place of its X, once the last of that has landed.
  wait_but<0>();
  auto part = [&](int w, int i) W4_INLINE {
    return reinterpret_cast<i32x4*>((i < 2 * MB ? sX0 : sX1) + w * kRegion + 1024 * (i % (2 * MB)) + 16 * lane);
  };
#pragma unroll
  for (int i = 0; i < NB * MB; ++i) *part(wave, i) = acc[i / MB][i % MB];
  __syncthreads();
  const int n_out = SWIGLU ? p.N >> 1 : p.N;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int unit = wave + W * j;
    if (unit >= kUnits) return;
    // Lane (l16, q) holds row l16, columns 4 q .. 4 q + 3 of its 16 x 16.
    auto sum = [&](int i, float4 scale, float (&f)[4]) W4_INLINE {
      i32x4 t = *part(0, i);
#pragma unroll
      for (int w = 1; w < W; ++w) t += *part(w, i);
      const float s[4] = {scale.x, scale.y, scale.z, scale.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = (float)t[e] * s[e] * x_scale[j];
    };
    float v[4];
    sum(unit, w_scale[j], v);
    if constexpr (SWIGLU) {
      float t[4];
      sum(unit + kUnits, up_scale[j], t);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = swiglu(v[e], t[e]);
    }
    const int n = 16 * (tile0 + unit / MB) + 4 * q, row = 16 * (unit % MB) + l16;
    if (row >= rows || n >= n_out) continue;
    uint16_t* const y = static_cast<uint16_t*>(p.y) + (m0 + row) * p.ldy + n;
    const u32x2 d = narrow4<BF16>(v);
    if (n + 4 <= n_out) {
      *reinterpret_cast<u32x2*>(y) = d;
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (n + e < n_out) y[e] = (uint16_t)(d[e >> 1] >> (16 * (e & 1)));
    }
  }
}

template <bool BF16, bool SWIGLU, int MB, int NB, int W, int U>
void launch_small(const W4Product& p, hipStream_t stream) {
  const int64_t blocks_m = ((int64_t)p.M + 16 * MB - 1) / (16 * MB), tiles = W4Layout(p.K, SWIGLU ? p.N / 2 : p.N).tiles;
  const int64_t per = SWIGLU ? NB / 2 : NB, blocks_n = (tiles + per - 1) / per;
  hipLaunchKernelGGL((w4_small_kernel<BF16, SWIGLU, MB, NB, W, U>), dim3((unsigned)(blocks_m * blocks_n)), dim3(64 * W), 0,
                     stream, p, (int)blocks_m);
}

constexpr uint32_t kNowhere = 0x80000000u;  // past every range of a tile: 256 rows of at most 2^22 elements

__device__ inline i32x4 load16s(__amdgpu_buffer_rsrc_t rs, uint32_t off, uint32_t soff) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, soff, 0));
}
__device__ inline uint32_t load1s(__amdgpu_buffer_rsrc_t rs, uint32_t off, uint32_t soff) {
  return __builtin_amdgcn_raw_buffer_load_b8(rs, off, soff, 0);
}
__device__ inline void store16(u32x4 v, __amdgpu_buffer_rsrc_t rs, uint32_t off) {
  __builtin_amdgcn_raw_buffer_store_b128(v, rs, off, 0, 0);
}
// Past the L2s, for tiles of many rows whose result takes up to kFarBytes: a kernel's end writes back what its L2s hold, and
// of a small result that is all.  Of a larger one the call that reads it loses more than the product gains, so the two
// together decide: the product and qattn_quantize_q8 of its result, microseconds on one MI355X, past the L2s and plainly:
// 1,500 x 1,024 -> 4,096 (12 MB) 17.4 and 18.2, 2,400 rows (20 MB) 24.2 and 24.7, 3,200 (26 MB) 27.7 and 27.1, 8,000 (66 MB)
// 62.3 and 59.9, 12,000 (98 MB) 88.1 and 85.8, 20,000 (164 MB) 141.5 either way.  SwiGLU's results, half as large for their
// products, go past them at any size: 1,024 -> 2 x 2,816 of 3,200 rows 35.9 and 36.4, 8,000 71.3 and 74.2, 12,000 103.0 and
// 100.9, 20,000 166 and 167.
constexpr int64_t kFarBytes = 24 << 20;
__device__ inline void store16_far(u32x4 v, __amdgpu_buffer_rsrc_t rs, uint32_t off) {
  __builtin_amdgcn_raw_buffer_store_b128(v, rs, off, 0, 2);
}
__device__ inline void store2(uint16_t v, __amdgpu_buffer_rsrc_t rs, uint32_t off) {
  __builtin_amdgcn_raw_buffer_store_b16(v, rs, off, 0, 0);
}
// Waits for all but the newest V vector-memory operations and for all LDS operations of this wavefront, then meets
// the workgroup.  One block of its own: the compiler's barrier would wait for every LDS-DMA load in flight.
template <int V>
__device__ inline void barrier_but() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(V) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// ---- in between: workgroup tiles of 16 MF rows and 128 columns, groups of four wavefronts of 16 MF x 32, K in blocks
// of 128.  X comes by LDS-DMA, three blocks ahead; each wavefront takes its own weights apart, straight into
// fragments: no store to LDS and one barrier a block, for which the taking apart, done once for each tile of rows, is
// most of the vector work and, with the chain of loads, the bound (1,419 x 2,048 -> 1,024: 8.9 us, vector units 36 % of
// the cycles, waiting 38 %).  G groups share K and add up in LDS.
//
// LDS rows of X have 128 bytes; the eight 16-byte pieces of row r lie at c ^ ((r >> 1) & 7), so that 16 rows reading
// one piece cover all banks.
template <bool BF16, bool SWIGLU, int MF, int G>
__global__ __launch_bounds__(256 * G, 2) void w4_mid_kernel(W4Product p, int tiles_n, int tiles_total, int per_xcd) {
  constexpr int kTileM = 16 * MF, kStage = kTileM * 128, XJ = MF / 2;  // X loads per wavefront and block
  __shared__ __attribute__((aligned(1024))) char sX0[G * kStage];
  __shared__ __attribute__((aligned(1024))) char sX1[G * kStage];
  __shared__ __attribute__((aligned(1024))) char sX2[G * kStage];
  __shared__ __attribute__((aligned(1024))) char sX3[G * kStage];

  const int u = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (u >= tiles_total) return;
  const int64_t m0 = (int64_t)(u / tiles_n) * kTileM;
  const int n0 = (u % tiles_n) * 128;
  const int gwave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = gwave >> 2, wave = gwave & 3;
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
  const W4Layout at(p.K, p.N);
  const int blocks = (int)at.blocks, share = (blocks + G - 1) / G;
  const int block0 = grp * share;
  const int mine = G == 1 ? blocks : __builtin_amdgcn_readfirstlane(max(0, min(share, blocks - block0)));

  // A block's range starts at its first column and ends with the last row's K columns.
  const int rows = (int)(p.M - m0 < kTileM ? p.M - m0 : kTileM);
  const int8_t* const x0 = p.x + m0 * p.ldx;
  const int x_bytes = (rows - 1) * (int)p.ldx + p.K;
  uint32_t x_src[XJ];
#pragma unroll
  for (int j = 0; j < XJ; ++j) {
    const int row = 8 * (XJ * wave + j) + (lane >> 3);
    x_src[j] = (uint32_t)row * (uint32_t)p.ldx + 16u * ((lane & 7) ^ ((row >> 1) & 7));
  }
  const uint32_t x_dst = grp * kStage + 1024 * XJ * wave;
  auto load_x = [&](char* dst, int kb) W4_INLINE {
    const int first = 128 * (block0 + kb);
    const int left = __builtin_amdgcn_readfirstlane(kb < mine ? max(x_bytes - first, 0) : 0);
    const auto rs = rsrc(x0 + first, (uint32_t)left);
#pragma unroll
    for (int j = 0; j < XJ; ++j) dma16(rs, dst + x_dst + 1024 * j, x_src[j]);
  };
  // The wavefront's two tiles of 16 weight rows (SwiGLU: of the gate and the up projection).
  const int tile0 = SWIGLU ? (n0 >> 5) + wave : (n0 >> 4) + 2 * wave, tile1 = SWIGLU ? tile0 + (p.N >> 5) : tile0 + 1;
  const uint8_t *const codes0 = p.w + (int64_t)tile0 * blocks * 1024, *const codes1 = p.w + (int64_t)tile1 * blocks * 1024;
  const uint8_t *const groups0 = p.w + at.groups_at() + (int64_t)tile0 * blocks * 64, *const groups1 = p.w + at.groups_at() + (int64_t)tile1 * blocks * 64;
  const uint32_t here0 = tile0 < at.tiles, here1 = tile1 < at.tiles;
  struct WRegs {
    i32x4 r0, r1;
    uint32_t g0, g1;
  };
  auto load_w = [&](WRegs& r, int kb) W4_INLINE {
    const uint32_t k = (uint32_t)(block0 + kb), some = kb < mine ? (uint32_t)blocks : 0u;
    r.g0 = load1s(rsrc(groups0, here0 * some * 64u), 4u * l16 + q, k * 64u);
    r.r0 = load16s(rsrc(codes0, here0 * some * 1024u), 16u * lane, k * 1024u);
    r.g1 = load1s(rsrc(groups1, here1 * some * 64u), 4u * l16 + q, k * 64u);
    r.r1 = load16s(rsrc(codes1, here1 * some * 1024u), 16u * lane, k * 1024u);
  };
  i32x4 acc[MF][2];
#pragma unroll
  for (int mb = 0; mb < MF; ++mb) acc[mb][0] = acc[mb][1] = i32x4{};
  const uint32_t x_rd = grp * kStage + l16 * 128 + (((2 * q) ^ ((l16 >> 1) & 7)) << 4);
  WRegs wreg[4];
  load_x(sX0, 0);
  __builtin_amdgcn_sched_barrier(0);
  load_w(wreg[0], 0);
  __builtin_amdgcn_sched_barrier(0);
  load_x(sX1, 1);
  __builtin_amdgcn_sched_barrier(0);
  load_w(wreg[1], 1);
  __builtin_amdgcn_sched_barrier(0);
  load_x(sX2, 2);
  __builtin_amdgcn_sched_barrier(0);
  load_w(wreg[2], 2);
  // The scales: a row's to a thread of the first group, a column's to one.
  const int tid = threadIdx.x;
  float my_xs = 0.f, my_ws = 0.f;
  if (tid < rows) my_xs = p.x_scale[m0 + tid];
  if (tid < 128) {  // SwiGLU: 16 gate columns, then 16 of the up projection, for each wavefront
    const int64_t n = SWIGLU ? (tid >> 4 & 1 ? p.N >> 1 : 0) + (n0 >> 1) + 16 * (tid >> 5) + (tid & 15) : n0 + tid;
    if (n < 16 * at.tiles) my_ws = reinterpret_cast<const float*>(p.w + at.scales_at())[n];
  }
  // Block kb: its X has landed by the barrier, which also frees the buffer of kb - 1 for kb + 3.  Newer at the barrier
  // than its X loads are those of two blocks, X and weights: 2 (XJ + 4).
  auto step = [&](const char* cur, char* next, const WRegs& w, WRegs& w_next, int kb) W4_INLINE {
    barrier_but<2 * (XJ + 4)>();
    load_x(next, kb + 3);
    __builtin_amdgcn_sched_barrier(0);
    load_w(w_next, kb + 3);
    i32x4 x[MF][2];
#pragma unroll
    for (int mb = 0; mb < MF; ++mb) {
      x[mb][0] = *reinterpret_cast<const i32x4*>(cur + x_rd + 2048 * mb);
      x[mb][1] = *reinterpret_cast<const i32x4*>(cur + (x_rd ^ 16) + 2048 * mb);
    }
    const Group g0 = group_of(w.g0), g1 = group_of(w.g1);
    i32x4 b0 = weights16<0>(w.r0, g0), b1 = weights16<0>(w.r1, g1);
#pragma unroll
    for (int mb = 0; mb < MF; ++mb) {
      acc[mb][0] = mfma(b0, x[mb][0], acc[mb][0]);
      acc[mb][1] = mfma(b1, x[mb][0], acc[mb][1]);
    }
    b0 = weights16<1>(w.r0, g0), b1 = weights16<1>(w.r1, g1);
#pragma unroll
    for (int mb = 0; mb < MF; ++mb) {
      acc[mb][0] = mfma(b0, x[mb][1], acc[mb][0]);
      acc[mb][1] = mfma(b1, x[mb][1], acc[mb][1]);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll 1
  for (int kb = 0; kb < share; kb += 4) {  // blocks past the end add zero products
    step(sX0, sX3, wreg[0], wreg[3], kb);
    step(sX1, sX0, wreg[1], wreg[0], kb + 1);
    step(sX2, sX1, wreg[2], wreg[1], kb + 2);
    step(sX3, sX2, wreg[3], wreg[2], kb + 3);
  }
  barrier_but<0>();

  // G > 1: group g finishes row fragments g MF / G and on of every wavefront's tile; the others' sums of them lie at
  // [wavefront][g][sender] in the X buffers.
  constexpr int kMine = MF / G;
  if constexpr (G > 1) {
    constexpr int kPart = 2 * kMine * 1024, kWave = G * (G - 1) * kPart;
    static_assert(kWave <= G * kStage, "a wavefront's parts fit an X buffer");
    char* const ex = (wave == 0 ? sX0 : wave == 1 ? sX1 : wave == 2 ? sX2 : sX3) + 16 * lane;
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (g != grp)
#pragma unroll
        for (int i = 0; i < 2 * kMine; ++i)
          *reinterpret_cast<i32x4*>(ex + (g * (G - 1) + (grp < g ? grp : grp - 1)) * kPart + 1024 * i) = acc[g * kMine + i / 2][i % 2];
    __syncthreads();
#pragma unroll
    for (int g = 0; g < G; ++g)  // (a constant index for the registers)
      if (g == grp)
#pragma unroll
        for (int i = 0; i < 2 * kMine; ++i) {
          i32x4 t = acc[g * kMine + i / 2][i % 2];
#pragma unroll
          for (int from = 0; from < G - 1; ++from) t += *reinterpret_cast<const i32x4*>(ex + (g * (G - 1) + from) * kPart + 1024 * i);
          acc[i / 2][i % 2] = t;
        }
    __syncthreads();
  }
  // Output through LDS, stored as whole rows of the tile.  Lane (l16, q) holds row 16 mb + l16, columns 4 q .. + 3 of
  // the wavefront's two 16.
  constexpr int kPieces = SWIGLU ? 8 : 16;  // 16-byte pieces of a row
  static_assert(kTileM * 256 <= G * kStage * 2, "the tile's rows fit two X buffers");
  float *const sXs = reinterpret_cast<float*>(sX2), *const sWs = reinterpret_cast<float*>(sX3);
  if (tid < kTileM) sXs[tid] = my_xs;
  if (tid < 128) sWs[tid] = my_ws;
  __syncthreads();
  auto place = [&](int row, int c) W4_INLINE {
    return (row < kTileM / 2 ? sX0 : sX1) + row % (kTileM / 2) * (16 * kPieces) + ((SWIGLU ? c ^ ((row >> 1) & 7) : c ^ (row & 15)) << 4);
  };
  const float4 w0 = *reinterpret_cast<const float4*>(sWs + 32 * wave + 4 * q), w1 = *reinterpret_cast<const float4*>(sWs + 32 * wave + 16 + 4 * q);
  const float s0[4] = {w0.x, w0.y, w0.z, w0.w}, s1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int row = 16 * (kMine * grp + i) + l16;
    const float xs = sXs[row];
    float f[4], t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = (float)acc[i][0][e] * s0[e] * xs;
      t[e] = (float)acc[i][1][e] * s1[e] * xs;
    }
    if constexpr (SWIGLU) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = swiglu(f[e], t[e]);
      *reinterpret_cast<u32x2*>(place(row, 2 * wave + (q >> 1)) + 8 * (q & 1)) = narrow4<BF16>(f);
    } else {
      *reinterpret_cast<u32x2*>(place(row, 4 * wave + (q >> 1)) + 8 * (q & 1)) = narrow4<BF16>(f);
      *reinterpret_cast<u32x2*>(place(row, 4 * wave + 2 + (q >> 1)) + 8 * (q & 1)) = narrow4<BF16>(t);
    }
  }
  __syncthreads();
  const int n_out = SWIGLU ? p.N >> 1 : p.N, col0 = SWIGLU ? n0 >> 1 : n0;
  const auto yrs = rsrc(static_cast<uint16_t*>(p.y) + m0 * p.ldy, ((uint32_t)(rows - 1) * (uint32_t)p.ldy + (uint32_t)n_out) * 2u);
  constexpr int kRowsPer = 256 * G / kPieces;  // rows per store of the workgroup
#pragma unroll
  for (int i = 0; i < (kTileM + kRowsPer - 1) / kRowsPer; ++i) {
    const int row = kRowsPer * i + tid / kPieces, c = tid % kPieces, n = col0 + 8 * c;
    if (kTileM % kRowsPer && row >= kTileM) break;
    store16(*reinterpret_cast<const u32x4*>(place(row, c)), yrs,
            row < rows && n + 8 <= n_out ? ((uint32_t)row * (uint32_t)p.ldy + (uint32_t)n) * 2u : kNowhere);
  }
  // A last piece of fewer than 8 columns goes element by element.
  const int part = (n_out - col0) >> 3;
  if ((n_out & 7) && part < kPieces) {
#pragma unroll 1
    for (int i = tid; i < kTileM * 8; i += 256 * G) {
      const int row = i >> 3, n = col0 + 8 * part + (i & 7);
      const uint16_t v = *reinterpret_cast<const uint16_t*>(place(row, part) + 2 * (i & 7));
      store2(v, yrs, row < rows && n < n_out ? ((uint32_t)row * (uint32_t)p.ldy + (uint32_t)n) * 2u : kNowhere);
    }
  }
}

template <bool BF16, bool SWIGLU, int MF, int G>
void launch_mid(const W4Product& p, hipStream_t stream) {
  const int64_t tiles_m = ((int64_t)p.M + 16 * MF - 1) / (16 * MF), tiles_n = ((int64_t)p.N + 127) / 128;
  const int64_t tiles = tiles_m * tiles_n, per_xcd = (tiles + 7) / 8;
  hipLaunchKernelGGL((w4_mid_kernel<BF16, SWIGLU, MF, G>), dim3((unsigned)(8 * per_xcd)), dim3(256 * G), 0, stream, p, (int)tiles_n,
                     (int)tiles, (int)per_xcd);
}

// ---- many rows: workgroup tiles of 32 MF rows and 64 NWN columns, 2 x NWN wavefronts of 16 MF x 64, K in steps of 64.
// X comes by LDS-DMA, three steps ahead; every weight is taken apart once for the workgroup, into an LDS tile of
// 8-bit weights.
//
// LDS tiles have rows of 64 bytes; the four 16-byte pieces of row r lie at c ^ ((r >> 2) & 3), so that 16 rows
// reading one piece cover all banks.
//
// Step kb (X tile and weight tile kb in LDS, the first half's fragments in registers): half 1 reads the other row
// fragments, takes weights kb + 1 apart into the free weight tile and runs the first half's products; the barrier
// publishes that tile and X tile kb + 1; half 2 reads the next step's fragments under the other half's products.
// X tile kb + 3 goes into the buffer that tile kb - 1 left at the previous barrier.
//
// 8,000 x 4,096 -> 4,096: 117 us over four sets of buffers in turn, 2,290 TOP/s, 111 where one is used again (a loop of
// nothing but these instructions reaches 3,495).  LDS is busy half of the time, the matrix cores a little less, vector
// units 40 %, and the clock follows their power: with zeros for X 102 us.
__device__ inline uint32_t lds_off(int row, int piece) { return row * 64 + ((piece ^ ((row >> 2) & 3)) << 4); }

template <bool BF16, bool SWIGLU, int MF, int NWN>
__global__ __launch_bounds__(128 * NWN, 2) void w4_tile_kernel(W4Product p, int tiles_n, int tiles_total, int per_xcd, int far) {
  constexpr int kWaves = 2 * NWN;
  constexpr int kTileM = 32 * MF, kTileN = 64 * NWN;
  constexpr int kBytesA = kTileM * 64, kBytesB = kTileN * 64;
  constexpr int AJ = MF / NWN;                  // X loads per wavefront and step
  constexpr int A1 = AJ / 2, A2 = AJ - A1;      // ... in the first / second half step
  constexpr int H = MF / 2;                     // row fragments per half step
  __shared__ __attribute__((aligned(1024))) char sA0[kBytesA];
  __shared__ __attribute__((aligned(1024))) char sA1[kBytesA];
  __shared__ __attribute__((aligned(1024))) char sA2[kBytesA];
  __shared__ __attribute__((aligned(1024))) char sA3[kBytesA];
  __shared__ __attribute__((aligned(1024))) char sB0[kBytesB];
  __shared__ __attribute__((aligned(1024))) char sB1[kBytesB];

  // Consecutive workgroups of an XCD (workgroup b runs on XCD b % 8) walk the column tiles of one row tile: its X
  // rows stay in that XCD's L2.
  const int u = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (u >= tiles_total) return;
  const int64_t m0 = (int64_t)(u / tiles_n) * kTileM;
  const int n0 = (u % tiles_n) * kTileN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l16 = lane & 15, kq = lane >> 4;
  const int wr = 16 * MF * (wave & 1), wc = 64 * (wave >> 1);
  const W4Layout at(p.K, p.N);
  const int blocks = (int)at.blocks;
  const int steps = 2 * blocks;  // K is padded to whole blocks of two steps

  // X rows of the tile.  A range starts at its step's first column and ends with the last row's K columns, so that
  // a load past either reads zeros; what it reads past a row's end inside the tensor meets zero weights.
  const int rows = (int)(p.M - m0 < kTileM ? p.M - m0 : kTileM);
  const int8_t* const x0 = p.x + m0 * p.ldx;
  const int x_bytes = (rows - 1) * (int)p.ldx + p.K;  // below 2^30
  uint32_t a_src[AJ];
#pragma unroll
  for (int j = 0; j < AJ; ++j) {
    const int row = 16 * (AJ * wave + j) + (lane >> 2);
    a_src[j] = (uint32_t)row * (uint32_t)p.ldx + 16u * ((lane & 3) ^ ((row >> 2) & 3));
  }
  const uint32_t a_dst = 1024 * AJ * wave;
  auto load_a = [&](char* dst, int kb, int j0, int n) W4_INLINE {
    const int first = 64 * kb;
    // In a scalar register (the compiler's saturating difference is a vector one, and would be looped over).
    const int left = __builtin_amdgcn_readfirstlane(kb < steps ? max(x_bytes - first, 0) : 0);
    const auto rs = rsrc(x0 + first, (uint32_t)left);
#pragma unroll
    for (int j = j0; j < j0 + n; ++j) dma16(rs, dst + a_dst + 1024 * j, a_src[j]);
  };
  // Thread (row = tid / 2, half = tid & 1) takes the record of group 2 kb + half of its weight row apart: columns 0-15
  // (piece 2 half) and 16-31 (piece 2 half + 1) of 32 half.  A wavefront's 32 rows are two tiles of the image.
  // SWIGLU: of each 64 rows 32 are the gate's of 32 features, then the up projection's.
  const int first_tile = (SWIGLU ? (wave & 1 ? p.N >> 5 : 0) + ((n0 + 32 * (wave & ~1)) >> 5) : (n0 + 32 * wave) >> 4);
  const int my_tiles = __builtin_amdgcn_readfirstlane(max(0, min(2, (int)at.tiles - first_tile)));
  const uint8_t* const codes = p.w + (int64_t)first_tile * blocks * 1024;
  const uint8_t* const groups = p.w + at.groups_at() + (int64_t)first_tile * blocks * 64;
  const int brow = 32 * wave + (lane >> 1), half = lane & 1;
  const uint32_t w_rec = (uint32_t)(lane >> 5) * (uint32_t)blocks * 1024u + 256u * half + 16u * ((lane >> 1) & 15);
  const uint32_t w_grp = (uint32_t)(lane >> 5) * (uint32_t)blocks * 64u + 4u * ((lane >> 1) & 15) + half;
  const uint32_t b_lo = lds_off(brow, 2 * half), b_hi = lds_off(brow, 2 * half + 1);
  struct WRegs {
    i32x4 record;
    uint32_t group;
  };
  auto load_wg = [&](WRegs& r, int kb) W4_INLINE {
    const uint32_t k = (uint32_t)kb;
    r.group = load1s(rsrc(groups, kb < steps ? (uint32_t)my_tiles * (uint32_t)blocks * 64u : 0u), w_grp, (k >> 1) * 64u + 2u * (k & 1u));
  };
  auto load_wr = [&](WRegs& r, int kb) W4_INLINE {
    r.record = load16s(rsrc(codes, kb < steps ? (uint32_t)my_tiles * (uint32_t)blocks * 1024u : 0u), w_rec, (uint32_t)kb * 512u);
  };
  auto store_b = [&](char* dst, const WRegs& r) W4_INLINE {
    const Group g = group_of(r.group);
    *reinterpret_cast<i32x4*>(dst + b_lo) = weights16<0>(r.record, g);
    *reinterpret_cast<i32x4*>(dst + b_hi) = weights16<1>(r.record, g);
  };
  i32x4 acc[MF][4];
#pragma unroll
  for (int mb = 0; mb < MF; ++mb)
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) acc[mb][nb] = i32x4{};
  const uint32_t a_rd = lds_off(wr + l16, kq), b_rd = lds_off(wc + l16, kq);

  WRegs wreg[4];
  i32x4 a_lo[H], a_hi[H], b0[4], b1[4];
  auto read_a = [&](i32x4 (&f)[H], const char* q) W4_INLINE {
#pragma unroll
    for (int i = 0; i < H; ++i) f[i] = *reinterpret_cast<const i32x4*>(q + 1024 * i);
  };
  auto read_b = [&](i32x4 (&f)[4], const char* q) W4_INLINE {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const i32x4*>(q + 1024 * i);
  };
  auto mma = [&](const i32x4 (&b)[4], const i32x4 (&a)[H], int m8) W4_INLINE {
#pragma unroll
    for (int mb = 0; mb < H; ++mb)
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) acc[m8 + mb][nb] = mfma(b[nb], a[mb], acc[m8 + mb][nb]);
  };
  // The tile's scales, the oldest loads of all: a row's and a column's to a thread, shared out at the end.
  const int tid = threadIdx.x;
  float my_xs = 0.f, my_ws = 0.f;
  if (tid < rows) my_xs = p.x_scale[m0 + tid];
  if (tid < kTileN) {
    const int64_t n = SWIGLU ? (tid >> 5 & 1 ? p.N >> 1 : 0) + (n0 >> 1) + 32 * (tid >> 6) + (tid & 31) : n0 + tid;
    if (n < 16 * at.tiles) my_ws = reinterpret_cast<const float*>(p.w + at.scales_at())[n];
  }
  __builtin_amdgcn_sched_barrier(0);
  load_wg(wreg[0], 0);
  load_wr(wreg[0], 0);
  load_a(sA0, 0, 0, AJ);
  __builtin_amdgcn_sched_barrier(0);
  load_wg(wreg[1], 1);
  load_a(sA1, 1, 0, AJ);
  __builtin_amdgcn_sched_barrier(0);
  load_wr(wreg[1], 1);
  load_wg(wreg[2], 2);
  load_a(sA2, 2, 0, AJ);
  __builtin_amdgcn_sched_barrier(0);
  load_wr(wreg[2], 2);
  store_b(sB0, wreg[0]);
  barrier_but<4 + 2 * AJ>();  // X tile 0: newer are the weights and X of 1 and 2
  read_b(b0, sB0 + b_rd);
  read_a(a_lo, sA0 + a_rd);
  auto step = [&](const char* a_cur, const char* a_nxt, char* a_new, char* b_nxt, i32x4 (&b_cur)[4], i32x4 (&b_new)[4],
                  const WRegs& w_use, WRegs& w_new, int kb) W4_INLINE {
    read_a(a_hi, a_cur + a_rd + 1024 * H);
    load_wg(w_new, kb + 3);
    load_a(a_new, kb + 3, 0, A1);
    store_b(b_nxt, w_use);
    mma(b_cur, a_lo, 0);
    // X tile kb + 1: newer are at least step kb - 1's AJ + 2 loads and this half's 1 + A1.
    barrier_but<3 + AJ + A1>();
    read_b(b_new, b_nxt + b_rd);
    read_a(a_lo, a_nxt + a_rd);
    load_a(a_new, kb + 3, A1, A2);
    load_wr(w_new, kb + 3);
    mma(b_cur, a_hi, H);
    // The next step's fragments between this half's first products: left alone they are read after the last ones, and
    // the next half starts with a wait (8,000 x 4,096 -> 4,096 117 us against 123).
#pragma unroll
    for (int i = 0; i < H + 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix instructions
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // reads of LDS
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 3 * H - 4, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll 1
  for (int kb = 0; kb < steps; kb += 4) {  // steps past the end add zero products
    step(sA0, sA1, sA3, sB1, b0, b1, wreg[1], wreg[3], kb);
    step(sA1, sA2, sA0, sB0, b1, b0, wreg[2], wreg[0], kb + 1);
    step(sA2, sA3, sA1, sB1, b0, b1, wreg[3], wreg[1], kb + 2);
    step(sA3, sA0, sA2, sB0, b1, b0, wreg[0], wreg[2], kb + 3);
  }
  barrier_but<0>();

  // Output through LDS, kRows rows of a wavefront at a time: stores of 16 bytes in whole 128-byte lines.  Lane (l16,
  // kq) holds row 16 mb + l16, columns 16 nb + 4 kq .. + 3.
  constexpr int kHold = 4 * kBytesA / 128 / kWaves;
  constexpr int kMost = kHold < 64 ? kHold : 64;
  constexpr int kRows = 16 * MF < kMost ? 16 * MF : kMost;
  constexpr int kPer = kBytesA / (128 * kRows);  // wavefronts per X buffer
  static_assert(4 * kPer >= kWaves && 16 * MF % kRows == 0 && kRows % 16 == 0, "a stage per wavefront, whole fragments");
  const int slot = wave / kPer;
  char* const stage = (slot == 0 ? sA0 : slot == 1 ? sA1 : slot == 2 ? sA2 : sA3) + 128 * kRows * (wave % kPer);
  const int n_out = SWIGLU ? p.N >> 1 : p.N;
  const int row0 = wr, col0 = SWIGLU ? (n0 + wc) >> 1 : n0 + wc;
  const auto yrs = rsrc(static_cast<uint16_t*>(p.y) + m0 * p.ldy, ((uint32_t)(rows - 1) * (uint32_t)p.ldy + (uint32_t)n_out) * 2u);
  constexpr int kPieces = SWIGLU ? 4 : 8;     // 16-byte pieces of a row
  auto place = [&](int row, int c) W4_INLINE {
    return stage + row * (16 * kPieces) + ((SWIGLU ? c ^ ((row >> 2) & 3) : c ^ ((row >> 1) & 7)) << 4);
  };
  // The weight tiles are free: the scales' place.
  float *const sXs = reinterpret_cast<float*>(sB0), *const sWs = reinterpret_cast<float*>(sB1);
  static_assert(128 * NWN >= kTileM && 128 * NWN >= kTileN && kBytesB >= 4 * kTileM, "a thread and a place for every scale");
  if (tid < kTileM) sXs[tid] = my_xs;
  if (tid < kTileN) sWs[tid] = my_ws;
  __syncthreads();
  float4 ws[4];
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) ws[nb] = *reinterpret_cast<const float4*>(sWs + wc + 16 * nb + 4 * kq);
#pragma unroll
  for (int pass = 0; pass < 16 * MF / kRows; ++pass) {
#pragma unroll
    for (int mb = 0; mb < kRows / 16; ++mb) {
      const i32x4(&v)[4] = acc[pass * (kRows / 16) + mb];
      const int row = 16 * mb + l16;
      const float xs = sXs[row0 + kRows * pass + row];
      auto scaled = [&](int nb, float (&f)[4]) W4_INLINE {
        const float s[4] = {ws[nb].x, ws[nb].y, ws[nb].z, ws[nb].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = (float)v[nb][e] * s[e] * xs;
      };
#pragma unroll
      for (int nb = 0; nb < (SWIGLU ? 2 : 4); ++nb) {
        float f[4];
        scaled(nb, f);
        if constexpr (SWIGLU) {  // columns 0-31: gate, 32-63: up, of the same 32 features
          float t[4];
          scaled(nb + 2, t);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = swiglu(f[e], t[e]);
        }
        *reinterpret_cast<u32x2*>(place(row, 2 * nb + (kq >> 1)) + 8 * (kq & 1)) = narrow4<BF16>(f);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    constexpr int kRowsPer = 64 / kPieces;  // rows per store instruction
#pragma unroll
    for (int i = 0; i < kRows / kRowsPer; ++i) {
      const int row = kRowsPer * i + lane / kPieces, c = lane % kPieces;
      const u32x4 v = *reinterpret_cast<const u32x4*>(place(row, c));
      const int m = row0 + kRows * pass + row, n = col0 + 8 * c;
      const uint32_t at_y = m < rows && n + 8 <= n_out ? ((uint32_t)m * (uint32_t)p.ldy + (uint32_t)n) * 2u : kNowhere;
      if (SWIGLU || far)
        store16_far(v, yrs, at_y);
      else
        store16(v, yrs, at_y);
    }
    // A last piece of fewer than 8 columns goes element by element.
    const int part = (n_out - col0) >> 3;
    if ((n_out & 7) && n_out > col0 && part < kPieces) {
#pragma unroll 1
      for (int i = 0; i < kRows / 8; ++i) {
        const int row = 8 * i + (lane >> 3), m = row0 + kRows * pass + row, n = col0 + 8 * part + (lane & 7);
        const uint16_t v = *reinterpret_cast<const uint16_t*>(place(row, part) + 2 * (lane & 7));
        store2(v, yrs, m < rows && n < n_out ? ((uint32_t)m * (uint32_t)p.ldy + (uint32_t)n) * 2u : kNowhere);
      }
    }
  }
}

template <bool BF16, bool SWIGLU, int MF, int NWN>
void launch_tile(const W4Product& p, hipStream_t stream) {
  const int64_t tiles_m = ((int64_t)p.M + 32 * MF - 1) / (32 * MF), tiles_n = ((int64_t)p.N + 64 * NWN - 1) / (64 * NWN);
  const int64_t tiles = tiles_m * tiles_n, per_xcd = (tiles + 7) / 8;
  hipLaunchKernelGGL((w4_tile_kernel<BF16, SWIGLU, MF, NWN>), dim3((unsigned)(8 * per_xcd)), dim3(128 * NWN), 0, stream, p,
                     (int)tiles_n, (int)tiles, (int)per_xcd, SWIGLU || (int64_t)p.M * p.N * 2 <= kFarBytes);
}

template <bool BF16, bool SWIGLU>
hipError_t launch(const W4Product& p, hipStream_t stream) {
  const auto tiles = [&](int tm, int tn) { return (((int64_t)p.M + tm - 1) / tm) * (((int64_t)p.N + tn - 1) / tn); };
  // Workgroups that fit the card at once less those of a launch's last round; whether so much of a launch's tiles is
  // rows and columns that there are.
  const auto idle = [](int64_t groups, int at_once) { return (at_once - groups % at_once) % at_once; };
  const auto full = [&](int tm, int tn, int percent) { return 100 * (int64_t)p.M * p.N >= percent * tiles(tm, tn) * tm * tn; };
  const int64_t small = tiles(32, 32), whole = tiles(256, 256);
  // Figures: microseconds on one MI355X, M x K -> N, the variant taken and the next best one.
  //
  // Few rows, or few tiles: wavefronts that share K fill the card (700 x 256 -> 1,024 3.9 and, in tiles of 64 x 128, 4.9;
  // 700 x 2,048 -> 1,024 7.3 and 8.8; but 300 x 1,024 -> 4,096, 1,280 tiles, 7.7 and 6.6).  Sums of one or two blocks let
  // more tiles through (20,000 x 128 -> 40 4.4 and 6.1).  Of these kernels
  // - 16 rows where there are no more or tiles are few (50 x 4,096 -> 96 3.8, of 32 rows 4.4), long sums two blocks
  //   ahead (1 x 65,536 -> 4,096 36 and 41; 1 x 4,096 -> 8,192 5.2 either way);
  // - 32 rows two blocks ahead for long sums of few tiles (64 x 4,096 -> 4,096 5.6 and 7.1), 64 rows for long sums of
  //   more (333 x 8,192 -> 1,000 10.6 and 13.1), else 32 rows one block ahead (100 x 1,024 -> 4,096 4.3, two ahead 4.7;
  //   50 x 1,024 -> 2 x 2,816 4.1, of 64 rows 4.2);
  // - beyond, 64 rows and four wavefronts as long as they fit at once (1,000 x 2,048 -> 1,024 7.7 and, in tiles of 64 x
  //   128, 8.8; 200 x 1,024 -> 4,096 5.9 and 6.4; but 300 x 1,024 -> 4,096 7.7 and 6.6).
  if (p.M <= 16 || small <= 96) {
    if (p.K > 8192)
      launch_small<BF16, SWIGLU, 1, 2, 8, 2>(p, stream);
    else
      launch_small<BF16, SWIGLU, 1, 2, 8, 1>(p, stream);
  } else if (p.M <= 32 || small <= (p.K <= 256 ? 1280 : 704)) {
    if (p.K >= 2048 && small <= 256)
      launch_small<BF16, SWIGLU, 2, 2, 4, 2>(p, stream);
    else if (p.K >= 2048 && tiles(64, 32) <= 256)
      launch_small<BF16, SWIGLU, 4, 2, 8, 1>(p, stream);
    else
      launch_small<BF16, SWIGLU, 2, 2, 4, 1>(p, stream);
  } else if (tiles(64, 32) <= 512) {
    launch_small<BF16, SWIGLU, 4, 2, 4, 1>(p, stream);
    // The largest tiles for long sums where their last round leaves few places (8,000 x 4,096 -> 4,096 120, in halves of
    // them 132; 2,400 x 1,024 -> 4,096 16.5 and 18.4; gate/up of 20,000 x 1,024 -> 2 x 2,816 121 and 125; but 5,000 x
    // 1,024 -> 4,096, a second round of 64 tiles, 34 and 30, and of shorter sums, with what reads the result, 20,000 x 512
    // -> 1,024 38.1 and 34.8, 8,000 x 512 -> 4,096 45.4 and 44.7, over four sets of buffers 46.5 and 49.3).
  } else if (p.K >= 1024 && full(256, 256, 80) && (idle(whole, 256) <= 96 || idle(whole, 256) <= whole / 8)) {
    launch_tile<BF16, SWIGLU, 8, 4>(p, stream);
    // Half of them where they are enough (1,500 x 1,024 -> 4,096 12.1, of 128 x 128 13.3; 6,000 x 1,024 -> 4,096 32.6 and
    // 35.7; 8,000 x 256 -> 4,096 24 and 32; but 20,000 x 1,024 -> 300, a fifth of whose tiles is empty, 14.1 and 13.2).
  } else if (tiles(256, 128) >= 160 && full(256, 128, 80)) {
    launch_tile<BF16, SWIGLU, 8, 2>(p, stream);
    // In between two workgroups to a compute unit, of 128 rows unless a round would be mostly empty (2,000 x 2,048 -> 2,048
    // 14.8 and, of 64 rows, 15.2; 100 x 1,024 -> 40,000 12.5 and 13.2; but 3,000 x 1,024 -> 1,024 9.2 and 9.1, and 64 x
    // 1,024 -> 70,016 18.7 and 13.3), and two groups that share a long sum where there is one workgroup to a unit
    // (1,419 x 2,048 -> 1,024 8.9 and 9.7; 500 x 1,024 -> 4,096 7.4 and 7.0).
  } else if (idle(tiles(128, 128), 512) <= 300 && full(128, 128, 70)) {
    launch_mid<BF16, SWIGLU, 8, 1>(p, stream);
  } else if (tiles(64, 128) <= 256 && p.K >= 2048) {
    launch_mid<BF16, SWIGLU, 4, 2>(p, stream);
  } else {
    launch_mid<BF16, SWIGLU, 4, 1>(p, stream);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_w4(const W4Product& p, bool bf16, bool swiglu, hipStream_t stream) {
  if (p.M <= 0) return hipSuccess;
  if (swiglu) return bf16 ? launch<true, true>(p, stream) : launch<false, true>(p, stream);
  return bf16 ? launch<true, false>(p, stream) : launch<false, false>(p, stream);
}

}  // namespace qattn
