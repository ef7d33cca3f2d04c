#pragma once

// A bounded KV cache: attention that accumulates the weight every cached key receives, the choice
// of the rows to keep by that weight, and their move into another cache. No reference counterpart
// (the reference's cache only grows). Shapes and cache layouts are attention_decode.hpp's and
// attention_decode_fp8.hpp's; an accumulator is weights [2][max_ctx] f32, the sum over every query
// seen so far of the softmax weights its KV head's 8 query heads gave each row.

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "attention_decode.hpp"
#include "attention_decode_fp8.hpp"
#include "cdna4_wave.hpp"

namespace miso::kernels {

// ------------------------------------------------------------------------------------------------
// Decode with weights
//
// weights[g][j] += sum over the heads h of KV head g of 2^(s[h][j] - M[h]) / L[h], s in log2 units.
// M and L are known only once every split is done, so the split stores its scores (64 bytes per
// key, both KV heads, beside the 2048 it reads) and the launch that merges the partials also turns
// them into weights. The result of the attention is attn_decode's, bit for bit.
// ------------------------------------------------------------------------------------------------

// The scores' row length for len keys: the padding lets a span store whole groups of 4.
__host__ __device__ constexpr std::size_t attn_scores_stride(unsigned len) {
  return (std::size_t{len} + 31) / 32 * 32;
}

// Floats of the workspace: m2 [2][n_splits][8], then the scores [16][attn_scores_stride(len)].
__host__ __device__ constexpr std::size_t attn_decode_weights_floats(unsigned len,
                                                                     unsigned n_splits) {
  return attn::kQHeads * (std::size_t{n_splits} + attn_scores_stride(len));
}

namespace decode_detail {
__device__ __attribute__((always_inline)) inline SplitScores scores_of(float* ws, unsigned len,
                                                                      unsigned n_splits,
                                                                      unsigned kvh) {
  const std::size_t stride = attn_scores_stride(len);
  return {ws + attn::kQHeads * std::size_t{n_splits} + kvh * kGroup * stride, stride, ws};
}
}  // namespace decode_detail

// attn_split_kernel, the scores stored. Grid dim3(n_splits, 2) x 256.
template <int kBlock>
__global__ void __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(1, 1)))
attn_split_scores_kernel(AttnSplitParams p, float* ws) {
  static_assert(kBlock == 256, "four waves per split workgroup");
  using namespace decode_detail;
  __shared__ TileShared sh;
  const unsigned kvh = blockIdx.y, split = blockIdx.x;
  const std::size_t head = std::size_t{kvh} * p.max_ctx * attn::kDim;
  const AttnSpan span = attn_split_span(p.len, p.n_splits, split);
  const LinearTiles tl{p.k_cache + head, p.v_cache + head};
  const std::size_t base = std::size_t{kvh} * p.n_splits + split;
  const SplitScores sc = scores_of(ws, p.len, p.n_splits, kvh);
  if (span.end - span.begin > kSplitWavesMinKeys)  // as attn_split_op
    split_partial_waves(p.q, tl, span, kvh, p.part_m, p.part_l, p.part_o, base, sh, false, sc);
  else
    split_partial_tiles<LinearTiles, false>(p.q, tl, span, kvh, p.part_m, p.part_l, p.part_o,
                                            base, sh, false, 0u, sc);
}

// attn_split_fp8_kernel, the scores stored. Grid dim3(n_splits, 2) x 256.
template <int kBlock>
__global__ void __launch_bounds__(kBlock) attn_split_fp8_scores_kernel(AttnSplitFp8Params p,
                                                                       float* ws) {
  static_assert(kBlock == 256, "four waves per split workgroup");
  using namespace decode_detail;
  __shared__ Fp8WaveShared sh;
  const unsigned kvh = blockIdx.y, split = blockIdx.x;
  const std::size_t rows = std::size_t{kvh} * p.max_ctx;
  split_partial_fp8_waves(p.q, p.k8 + rows * attn::kDim, p.v8 + rows * attn::kDim,
                          p.k_scale + rows, p.v_scale + rows,
                          attn_split_span(p.len, p.n_splits, split), kvh, p.part_m, p.part_l,
                          p.part_o, std::size_t{kvh} * p.n_splits + split, sh, false,
                          scores_of(ws, p.len, p.n_splits, kvh));
}

struct AttnWeightsParams {
  AttnCombineParams c;
  const float* ws;   // the split's workspace (attn_decode_weights_floats)
  float* weights;    // [2][max_ctx]
  unsigned len, max_ctx;
};

constexpr unsigned kCombineItems = attn::kQHeads * (attn::kDim / 64);  // 64-thread workgroups
constexpr unsigned kWeightKeys = 256;  // keys per workgroup of the weights' part

// Workgroups [0, 64): attn_combine_kernel's; the others one 256-key block of one KV head each:
// every lane forms the head statistics from the splits' and adds 4 keys' weights, 64 apart. Grid
// 64 + 2 ceil(len / 256), x 64.
template <int = 0>
__global__ void __launch_bounds__(64) attn_combine_weights_kernel(AttnWeightsParams p) {
  using decode_detail::kGroup;
  if (blockIdx.x < kCombineItems) {
    attn_combine_op<64, true, 4>(p.c, 0, kCombineItems);
    return;
  }
  const unsigned item = blockIdx.x - kCombineItems, lane = threadIdx.x;
  const unsigned blocks = (p.len + kWeightKeys - 1) / kWeightKeys;
  const unsigned kvh = item / blocks, k0 = (item % blocks) * kWeightKeys + lane;
  const unsigned n = p.c.n_splits;
  const std::size_t stride = attn_scores_stride(p.len);
  const float* s = p.ws + attn::kQHeads * std::size_t{n} + kvh * kGroup * stride;
  constexpr unsigned kPer = kWeightKeys / 64;
  float x[kGroup][kPer], old[kPer];
  float* w = p.weights + std::size_t{kvh} * p.max_ctx;
#pragma unroll
  for (unsigned j = 0; j < kPer; ++j) {
    const unsigned key = k0 + 64 * j;
    const bool in = key < p.len;
#pragma unroll
    for (unsigned h = 0; h < kGroup; ++h)
      x[h][j] = in ? s[h * stride + key] : -__builtin_inff();
    old[j] = in ? w[key] : 0.0f;
  }
  // Lane (split slot lane / 8, head lane % 8): the head's largest maximum and its sum, over the
  // splits in fixed order. Head 0's lane 0 .. head 7's lane 7 then serve every lane.
  const std::size_t i0 = std::size_t{kvh} * n * kGroup;
  float M = -__builtin_inff(), L = 0.0f;
  for (unsigned c0 = lane >> 3; c0 < n; c0 += 128) {
    float m[16], l[16], top = M;
#pragma unroll
    for (unsigned i = 0; i < 16; ++i) {
      const unsigned c = c0 + 8 * i;
      const std::size_t at = i0 + (c < n ? c : c0) * kGroup + (lane & 7u);
      m[i] = c < n ? p.ws[at] : -__builtin_inff();
      l[i] = p.c.part_l[at];
      top = fmaxf(top, m[i]);
    }
    if (top != -__builtin_inff()) {
      L *= __builtin_amdgcn_exp2f(M - top);
#pragma unroll
      for (unsigned i = 0; i < 16; ++i)
        L = __builtin_fmaf(__builtin_amdgcn_exp2f(m[i] - top), l[i], L);
      M = top;
    }
  }
  const float top = cdna4::max_xor32(
      cdna4::max_xor16(fmaxf(M, cdna4::dpp_mov<cdna4::kRowRor8>(M))));
  L = M == -__builtin_inff() ? 0.0f : L * __builtin_amdgcn_exp2f(M - top);
  L += cdna4::dpp_mov<cdna4::kRowRor8>(L);
  L = cdna4::sum_xor32(cdna4::sum_xor16(L));
  const float inv = 1.0f / L;
  float sum[kPer] = {};
#pragma unroll
  for (unsigned h = 0; h < kGroup; ++h) {
    const float mh = cdna4::as_float(__builtin_amdgcn_readlane(cdna4::as_uint(top), h));
    const float ih = cdna4::as_float(__builtin_amdgcn_readlane(cdna4::as_uint(inv), h));
#pragma unroll
    for (unsigned j = 0; j < kPer; ++j)
      sum[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(x[h][j] - mh), ih, sum[j]);
  }
#pragma unroll
  for (unsigned j = 0; j < kPer; ++j)
    if (k0 + 64 * j < p.len)
      w[k0 + 64 * j] = old[j] + sum[j];
}

// ------------------------------------------------------------------------------------------------
// The weights of a prompt chunk
//
// Queries q[t][h], t < n, at rows pos0 + t: weights[g][j] += sum over t and the heads h of g of
// p[t][h][j], p the causal softmax over j <= pos0 + t. A weight needs its row's maximum and sum
// before it can join its column's sum, so the products q k are formed twice: the row pass gives
// each query's lse = M + log2 L, the column pass sums 2^(s - lse) over the queries. (Keeping the
// scores instead would move 64 bytes per token and key through memory twice, against 1024 flop.)
// A query is 32 bits wide and the matrix cores take 16: each row is scaled by the power of two that
// puts its largest element in [2^13, 2^14), and cut into f16 halves x = hi + lo, exact to 2^-22 of
// x, or 2^-38 of the row's largest element where lo is subnormal. hi k + lo k are exact products
// summed in f32, the row's scale comes off in the exponent's fma. So a score costs 1024 flop of
// f16 matrix work per pass, and the passes are bound by it once there are some hundred queries.
//
// A KV head's queries are columns c = 8 t + h % 8, in blocks of 32 (4 tokens): the B operand of
// v_mfma_f32_32x32x16_f16, whose A operand is 32 K rows. The row pass writes the halves as the
// column pass reads them: per KV head and block [hi, lo][k-step][lane][8], one lane's 16 bytes
// after the other's.
// ------------------------------------------------------------------------------------------------

struct AttnKeyWeightsParams {
  const float* q;                // [n][16][256]
  const attn::half_t* k_cache;   // [2][k_ctx][256]
  float* weights;                // [2][max_ctx]
  attn::half_t* halves;          // [2][blocks][2][16][64][8]
  float* meta;                   // [2][blocks][32 scales, 32 lse]: a scale is log2(e) / 16 over the
                                 // row's power of two, an lse in log2 units, +inf in padding columns
  float2* stats;                 // [row parts][2][32 blocks]: (maximum, sum)
  float* sums;                   // [column parts][2][pos0 + n]
  unsigned pos0, n, max_ctx, k_ctx;
  unsigned blocks;               // column blocks: ceil(n / 4)
  unsigned row_blocks;           // column blocks of a row pass workgroup, <= 8
  unsigned row_tiles;            // key tiles of a row part
  unsigned col_blocks;           // column blocks of a column part
};

namespace weights_detail {

constexpr unsigned kCols = 32, kKeys = 32, kSteps = 16;  // of a tile; k-steps of 16 dimensions
constexpr unsigned kTokens = kCols / decode_detail::kGroup;
constexpr std::size_t kBlockHalves = 2 * kSteps * 64 * 8;  // one column block's halves

__device__ __attribute__((always_inline)) inline cdna4::float16_t mfma32(
    const cdna4::half8_t& a, const cdna4::half8_t& b, const cdna4::float16_t& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Row of a tile that a lane's result i belongs to.
__device__ __attribute__((always_inline)) inline unsigned tile_row(unsigned lane, unsigned i) {
  return 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
}

// This lane's halves of column lane % 32 of a block: dimensions 16 s + 8 (lane / 32) .. + 7.
struct Halves {
  cdna4::half8_t hi[kSteps], lo[kSteps];
};

// Reads and cuts the lane's column (zeros in the padding columns); returns the column's scale.
__device__ __attribute__((always_inline)) inline float cut_column(Halves& b,
                                                                 const AttnKeyWeightsParams& p,
                                                                 unsigned kvh, unsigned block,
                                                                 unsigned lane) {
  const unsigned col = kCols * block + (lane & 31u);
  const unsigned t = col / decode_detail::kGroup, h = col % decode_detail::kGroup;
  const bool in = t < p.n;
  const float* row = p.q + (std::size_t{in ? t : 0} * attn::kQHeads + kvh * decode_detail::kGroup +
                            h) * attn::kDim + 8 * (lane >> 5);
  float4 x[kSteps][2];
#pragma unroll
  for (unsigned s = 0; s < kSteps; ++s) {
    x[s][0] = *reinterpret_cast<const float4*>(row + 16 * s);
    x[s][1] = *reinterpret_cast<const float4*>(row + 16 * s + 4);
  }
  float top = 0.0f;
#pragma unroll
  for (unsigned s = 0; s < kSteps; ++s)
#pragma unroll
    for (unsigned j = 0; j < 2; ++j) {
      if (!in)
        x[s][j] = float4{0.0f, 0.0f, 0.0f, 0.0f};
      top = fmaxf(top, fmaxf(fmaxf(__builtin_fabsf(x[s][j].x), __builtin_fabsf(x[s][j].y)),
                             fmaxf(__builtin_fabsf(x[s][j].z), __builtin_fabsf(x[s][j].w))));
    }
  top = cdna4::max_xor32(top);
  // 2^(13 - e), e the exponent of top; rows of zeros or beyond 2^-87 keep a finite factor, and one
  // that holds an infinity stays as it is (its scores are infinite or NaN either way).
  int e = 13 - (static_cast<int>(cdna4::as_uint(top) >> 23) - 127);
  e = top == 0.0f || top == __builtin_inff() ? 0 : (e < 100 ? e : 100);
  const float up = __builtin_ldexpf(1.0f, e);
#pragma unroll
  for (unsigned s = 0; s < kSteps; ++s) {
    const float v[8] = {x[s][0].x, x[s][0].y, x[s][0].z, x[s][0].w,
                        x[s][1].x, x[s][1].y, x[s][1].z, x[s][1].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = v[j] * up;  // a power of two: exact
      const _Float16 hi = static_cast<_Float16>(y);
      b.hi[s][j] = hi;
      b.lo[s][j] = static_cast<_Float16>(y - static_cast<float>(hi));
    }
  }
  return __builtin_ldexpf(decode_detail::kLog2e / 16.0f, -e);
}

// K rows k0 + lane % 32 (clamped to `last`), as the A operand.
__device__ __attribute__((always_inline)) inline void load_keys(cdna4::half8_t (&a)[kSteps],
                                                               const attn::half_t* K, unsigned k0,
                                                               unsigned last, unsigned lane) {
  const unsigned row = k0 + (lane & 31u) < last ? k0 + (lane & 31u) : last;
  const attn::half_t* at = K + std::size_t{row} * attn::kDim + 8 * (lane >> 5);
#pragma unroll
  for (unsigned s = 0; s < kSteps; ++s)
    a[s] = *reinterpret_cast<const cdna4::half8_t*>(at + 16 * s);
}

// Row pass: a ring of K tiles, chunk c of row r at position c ^ (r % 16) of the row (the A operand
// read of 16 lanes takes one chunk of 16 rows: 16 positions).
constexpr unsigned kRowWaves = 8, kRowStages = 4, kRowTileBytes = kKeys * attn::kDim * 2;
struct alignas(1024) RowShared {
  unsigned char k[kRowStages][kRowTileBytes];
};

// Column pass: a ring of column blocks' halves, as they lie in memory, and each wave's copy of the
// block's scales and lse.
constexpr unsigned kColWaves = 4, kColStages = 4;
constexpr unsigned kColKeys = 2 * kKeys * kColWaves;  // keys of a workgroup, 64 a wave
struct alignas(1024) ColShared {
  unsigned char b[kColStages][kBlockHalves * 2];
  float meta[kColStages][kColWaves][2 * kCols];
};

// 256 bytes, 4 per lane, to LDS.
__device__ __attribute__((always_inline)) inline void lds_load4(const void* gaddr, unsigned lds) {
  unsigned saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %1, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(gaddr), "s"(lds)
      : "memory");
}

constexpr float kNoScore = -3e38f;  // below every score, and finite: differences stay numbers

// The running maximum m and sum l (relative to it) of a lane's column over its 16 keys of a tile;
// hidden keys are -inf.
__device__ __attribute__((always_inline)) inline void add_tile(float& m, float& l,
                                                              const cdna4::float16_t& x,
                                                              float scale) {
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < 15; i += 2)
    mx = decode_detail::tile_max3(mx, x[i], x[i + 1]);
  mx = decode_detail::tile_max(mx, x[15]);
  const float top = decode_detail::tile_max(m, mx * scale);
  float part[4] = {l * __builtin_amdgcn_exp2f(m - top), 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    part[i % 4] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], scale, -top));
  l = (part[0] + part[1]) + (part[2] + part[3]);
  m = top;
}

}  // namespace weights_detail

// Row pass. A workgroup takes `row_blocks` column blocks of one KV head (one a wave, its halves in
// registers; further waves only copy) and one part of the keys they see, 32 at a time through LDS.
// Items (part, group of blocks, KV head), the head fastest: an XCD's workgroups read one head's
// keys, and about the same ones at a time. Iteration t forms the scores of tile t while the vector
// units take tile t - 1 into the running sums.
template <int = 0>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
attn_key_weights_rows_kernel(AttnKeyWeightsParams p) {
  using namespace weights_detail;
  __shared__ RowShared sh;
  const unsigned lane = threadIdx.x & 63u;
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned groups = (p.blocks + p.row_blocks - 1) / p.row_blocks;
  const unsigned kvh = blockIdx.x % 2, group = blockIdx.x / 2 % groups;
  const unsigned part = blockIdx.x / 2 / groups;
  const unsigned block = group * p.row_blocks + wave;
  // Keys the group's last token sees, and the part's tiles of them.
  unsigned t_end = kTokens * (group + 1) * p.row_blocks;
  t_end = t_end < p.n ? t_end : p.n;
  const unsigned keys = p.pos0 + t_end, tiles = (keys + kKeys - 1) / kKeys;
  const unsigned first = part * p.row_tiles;
  if (first >= tiles)
    return;
  const unsigned past = first + p.row_tiles < tiles ? first + p.row_tiles : tiles;
  const attn::half_t* K = p.k_cache + std::size_t{kvh} * p.k_ctx * attn::kDim;
  const unsigned ring = cdna4::lds_offset(sh.k[0]);

  // Tile ti into its stage: this wave copies rows 4 wave .. + 3, two an instruction.
  auto issue = [&](unsigned ti) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned i = 0; i < 2; ++i) {
      const unsigned r = 4 * wave + 2 * i + (lane >> 5);
      const unsigned row = ti * kKeys + r < keys ? ti * kKeys + r : keys - 1;
      cdna4::lds_load16(K + std::size_t{row} * attn::kDim + 8 * ((lane & 31u) ^ (r & 15u)),
                        ring + ti % kRowStages * kRowTileBytes + 512 * (4 * wave + 2 * i));
    }
  };
#pragma unroll
  for (unsigned i = 0; i < kRowStages - 1; ++i)
    if (first + i < past)
      issue(first + i);

  const bool active = wave < p.row_blocks && block < p.blocks;  // wave-uniform
  Halves b;
  float scale = 0.0f;
  const std::size_t at = std::size_t{kvh} * p.blocks + block;
  if (active) {
    scale = cut_column(b, p, kvh, block, lane);
    if (part == 0) {
      attn::half_t* out = p.halves + at * kBlockHalves + 8 * lane;
#pragma unroll
      for (unsigned s = 0; s < kSteps; ++s) {
        *reinterpret_cast<cdna4::half8_t*>(out + 512 * s) = b.hi[s];
        *reinterpret_cast<cdna4::half8_t*>(out + 512 * (kSteps + s)) = b.lo[s];
      }
      if (lane < kCols)
        p.meta[at * 2 * kCols + lane] = scale;
    }
  }
  // Operand address of k-step s: row lane % 32, chunk 2 s + lane / 32, i.e. kl ^ 32 s.
  const unsigned kl = 512 * (lane & 31u) + 16 * ((lane >> 5) ^ (lane & 15u));
  const unsigned t = kTokens * block + (lane & 31u) / decode_detail::kGroup;
  const unsigned seen = p.pos0 + t;                // the lane's token sees keys up to its own
  const unsigned open = p.pos0 + kTokens * block;  // and every token of the block these
  auto mask = [&](cdna4::float16_t& x, unsigned k0) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned i = 0; i < 16; ++i)
      x[i] = k0 + tile_row(lane, i) <= seen ? x[i] : -__builtin_inff();
  };

  float m = kNoScore, l = 0.0f;
  cdna4::float16_t prev;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    prev[i] = -__builtin_inff();
  for (unsigned ti = first; ti < past; ++ti) {
    // Tile ti has landed: this wave's copies by the count, every wave's by the barrier, which also
    // says that every wave has read tile ti - 1, whose stage the next copy takes.
    const unsigned after = past - 1 - ti;
    if (after >= 2)
      cdna4::wait_vmcnt<4>();
    else if (after == 1)
      cdna4::wait_vmcnt<2>();
    else
      cdna4::wait_vmcnt<0>();
    decode_detail::tile_barrier();
    if (ti + kRowStages - 1 < past)
      issue(ti + kRowStages - 1);
    if (!active)
      continue;
    if (ti > first && ti * kKeys - 1 > open)  // the tile before reaches past what all see
      mask(prev, (ti - 1) * kKeys);
    const unsigned slot = ring + ti % kRowStages * kRowTileBytes + kl;
    cdna4::float16_t acc = {};
#pragma unroll
    for (unsigned s = 0; s < kSteps; ++s) {
      const cdna4::half8_t a = decode_detail::lds_b128(slot ^ (32u * s));
      acc = mfma32(a, b.hi[s], acc);
      acc = mfma32(a, b.lo[s], acc);
    }
    add_tile(m, l, prev, scale);
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (unsigned s = 0; s < kSteps; ++s) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
    }
    prev = acc;
  }
  if (!active)
    return;
  if (past * kKeys - 1 > open)
    mask(prev, (past - 1) * kKeys);
  add_tile(m, l, prev, scale);
  // The two halves of the wave hold the other keys of the same columns.
  const float top = cdna4::max_xor32(m);
  const float sum = cdna4::sum_xor32(l * __builtin_amdgcn_exp2f(m - top));
  if (lane < kCols)
    p.stats[(std::size_t{part} * 2 * p.blocks + at) * kCols + lane] = float2{top, sum};
}

// lse of every column from the row parts, in part order. One thread per column.
template <int = 0>
__global__ void __launch_bounds__(256) attn_key_weights_lse_kernel(AttnKeyWeightsParams p) {
  using namespace weights_detail;
  const std::size_t cols = std::size_t{2} * p.blocks * kCols;
  const std::size_t col = std::size_t{blockIdx.x} * 256 + threadIdx.x;
  if (col >= cols)
    return;
  const unsigned block = static_cast<unsigned>(col / kCols % p.blocks);
  const unsigned t = kTokens * block + static_cast<unsigned>(col % kCols) / decode_detail::kGroup;
  unsigned t_end = kTokens * (block / p.row_blocks + 1) * p.row_blocks;  // as the row pass
  t_end = t_end < p.n ? t_end : p.n;
  const unsigned parts = (p.pos0 + t_end + kKeys * p.row_tiles - 1) / (kKeys * p.row_tiles);
  float m = kNoScore, l = 0.0f;
  for (unsigned part = 0; part < parts; ++part)
    m = fmaxf(m, p.stats[part * cols + col].x);
  for (unsigned part = 0; part < parts; ++part) {
    const float2 s = p.stats[part * cols + col];
    l = __builtin_fmaf(s.y, __builtin_amdgcn_exp2f(s.x - m), l);
  }
  p.meta[col / kCols * 2 * kCols + kCols + col % kCols] =
      t < p.n ? m + __builtin_amdgcn_logf(l) : __builtin_inff();
}

// Column pass. A workgroup takes 256 keys of one KV head, 64 a wave, in registers, and one part of
// the column blocks, whose halves come through LDS in the order of the operands. Iteration t forms
// the scores of block t while the vector units turn block t - 1 into weights and sum them.
template <int = 0>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))
attn_key_weights_cols_kernel(AttnKeyWeightsParams p) {
  using namespace weights_detail;
  __shared__ ColShared sh;
  const unsigned lane = threadIdx.x & 63u;
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned rows = p.pos0 + p.n, key_blocks = (rows + kColKeys - 1) / kColKeys;
  const unsigned kvh = blockIdx.x % 2, kb = blockIdx.x / 2 % key_blocks;
  const unsigned part = blockIdx.x / 2 / key_blocks;
  // Tokens before kb's first key see none of its keys.
  const unsigned k_wg = kb * kColKeys;
  const unsigned b_min = k_wg > p.pos0 ? (k_wg - p.pos0) / kTokens : 0;
  const unsigned b1 = (part + 1) * p.col_blocks < p.blocks ? (part + 1) * p.col_blocks : p.blocks;
  const unsigned b0 = part * p.col_blocks > b_min ? part * p.col_blocks : b_min;
  if (b0 >= b1)
    return;
  const attn::half_t* halves = p.halves + std::size_t{kvh} * p.blocks * kBlockHalves;
  const float* meta = p.meta + std::size_t{kvh} * p.blocks * 2 * kCols;
  auto issue = [&](unsigned block) __attribute__((always_inline)) {
    const unsigned stage = block % kColStages;
    const attn::half_t* in = halves + block * kBlockHalves + 4096 * wave + 8 * lane;
    const unsigned lds = cdna4::lds_offset(sh.b[stage]) + 8192 * wave;
#pragma unroll
    for (unsigned i = 0; i < 8; ++i)
      cdna4::lds_load16(in + 512 * i, lds + 1024 * i);
    lds_load4(meta + std::size_t{block} * 2 * kCols + lane,
              cdna4::lds_offset(sh.meta[stage][wave]));
  };
#pragma unroll
  for (unsigned i = 0; i < kColStages - 1; ++i)
    if (b0 + i < b1)
      issue(b0 + i);

  const unsigned k0 = k_wg + 2 * kKeys * wave;  // the wave's first key
  const attn::half_t* K = p.k_cache + std::size_t{kvh} * p.k_ctx * attn::kDim;
  cdna4::half8_t a[2][kSteps];
  load_keys(a[0], K, k0, rows - 1, lane);
  load_keys(a[1], K, k0 + kKeys, rows - 1, lane);

  float sum[2][16] = {};
  cdna4::float16_t prev[2];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    prev[0][i] = prev[1][i] = -__builtin_inff();
  float scale = 1.0f, lse = 0.0f;  // of the block before
  auto mask = [&](unsigned block) __attribute__((always_inline)) {
    const unsigned seen = p.pos0 + kTokens * block + (lane & 31u) / decode_detail::kGroup;
#pragma unroll
    for (unsigned j = 0; j < 2; ++j)
#pragma unroll
      for (unsigned i = 0; i < 16; ++i)
        prev[j][i] = k0 + kKeys * j + tile_row(lane, i) <= seen ? prev[j][i] : -__builtin_inff();
  };
  auto add = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (unsigned j = 0; j < 2; ++j)
#pragma unroll
      for (unsigned i = 0; i < 16; ++i)
        sum[j][i] += __builtin_amdgcn_exp2f(__builtin_fmaf(prev[j][i], scale, -lse));
  };
  // Block b reaches keys that some of its tokens do not see.
  auto cut = [&](unsigned b) { return k0 + 2 * kKeys - 1 > p.pos0 + kTokens * b; };
  for (unsigned block = b0; block < b1; ++block) {
    const unsigned after = b1 - 1 - block;  // as the row pass: 9 copies a block
    if (after >= 2)
      cdna4::wait_vmcnt<18>();
    else if (after == 1)
      cdna4::wait_vmcnt<9>();
    else
      cdna4::wait_vmcnt<0>();
    decode_detail::tile_barrier();
    if (block + kColStages - 1 < b1)
      issue(block + kColStages - 1);
    if (block > b0 && cut(block - 1))
      mask(block - 1);
    const unsigned stage = block % kColStages;
    const unsigned slot = cdna4::lds_offset(sh.b[stage]) + 16 * lane;
    cdna4::float16_t acc[2] = {};
#pragma unroll
    for (unsigned s = 0; s < kSteps; ++s) {
      const cdna4::half8_t hi = decode_detail::lds_b128(slot + 1024 * s);
      const cdna4::half8_t lo = decode_detail::lds_b128(slot + 1024 * (kSteps + s));
      acc[0] = mfma32(a[0][s], hi, acc[0]);
      acc[1] = mfma32(a[1][s], hi, acc[1]);
      acc[0] = mfma32(a[0][s], lo, acc[0]);
      acc[1] = mfma32(a[1][s], lo, acc[1]);
    }
    add();
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
    for (unsigned s = 0; s < 2 * kSteps; ++s) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
    }
    prev[0] = acc[0];
    prev[1] = acc[1];
    scale = sh.meta[stage][wave][lane & 31u];
    lse = sh.meta[stage][wave][kCols + (lane & 31u)];
  }
  if (cut(b1 - 1))
    mask(b1 - 1);
  add();
  // A key's sum over the 32 columns of its lanes.
#pragma unroll
  for (unsigned j = 0; j < 2; ++j)
#pragma unroll
    for (unsigned i = 0; i < 16; ++i) {
      float v = sum[j][i];
      v += cdna4::dpp_mov<cdna4::kQuadXor1>(v);
      v += cdna4::dpp_mov<cdna4::kQuadXor2>(v);
      v += cdna4::dpp_mov<cdna4::kRowHalfMirror>(v);
      v += cdna4::dpp_mov<cdna4::kRowMirror>(v);
      v = cdna4::sum_xor16(v);
      const unsigned key = k0 + kKeys * j + tile_row(lane, i);
      if ((lane & 31u) == 0 && key < rows) {
        if (p.col_blocks >= p.blocks)  // one part
          p.weights[std::size_t{kvh} * p.max_ctx + key] += v;
        else
          p.sums[(std::size_t{part} * 2 + kvh) * rows + key] = v;
      }
    }
}

// weights += the column parts' sums, in part order (the parts before a key's block was seen wrote
// none). One thread per key.
template <int = 0>
__global__ void __launch_bounds__(256) attn_key_weights_join_kernel(AttnKeyWeightsParams p) {
  using namespace weights_detail;
  const std::size_t rows = p.pos0 + p.n, i = std::size_t{blockIdx.x} * 256 + threadIdx.x;
  if (i >= 2 * rows)
    return;
  const unsigned k_wg = static_cast<unsigned>(i % rows) / kColKeys * kColKeys;
  const unsigned b_min = k_wg > p.pos0 ? (k_wg - p.pos0) / kTokens : 0;
  const unsigned parts = (p.blocks + p.col_blocks - 1) / p.col_blocks;
  float v = 0.0f;
  for (unsigned part = b_min / p.col_blocks; part < parts; ++part)
    v += p.sums[part * 2 * rows + i];
  p.weights[(i / rows) * p.max_ctx + i % rows] += v;
}

// K codes [2][max_ctx][256] widened to f16 [2][n][256] (attn_kv_fp8_widen_kernel's values, K alone).
// One wave per row, 4 per workgroup, grid-stride.
template <int = 0>
__global__ void __launch_bounds__(256) attn_k_fp8_widen_kernel(const uint8_t* k8,
                                                               const float* k_scale,
                                                               attn::half_t* out, unsigned n,
                                                               unsigned max_ctx) {
  const unsigned lane = threadIdx.x & 63u;
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (std::size_t r = 4 * std::size_t{blockIdx.x} + wave; r < 2 * std::size_t{n};
       r += 4 * std::size_t{gridDim.x}) {
    const std::size_t src = r < n ? r : r - n + max_ctx;
    const unsigned w = *reinterpret_cast<const unsigned*>(k8 + src * attn::kDim + 4 * lane);
    const float sc = k_scale[src];
    const cdna4::half2_t a = cdna4::as_half2(fp8kv::pair_lo(w));
    const cdna4::half2_t b = cdna4::as_half2(fp8kv::pair_hi(w));
    const float e[4] = {static_cast<float>(a[0]), static_cast<float>(a[1]),
                        static_cast<float>(b[0]), static_cast<float>(b[1])};
    _Float16 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = static_cast<_Float16>(fminf(fmaxf(e[i] * sc, -65504.0f), 65504.0f));
    *reinterpret_cast<uint2*>(out + r * attn::kDim + 4 * lane) = __builtin_bit_cast(uint2, h);
  }
}

// How a launch is cut. A row workgroup takes up to 8 column blocks, evenly, and row_tiles key tiles
// of 32; a column workgroup 256 keys and col_blocks column blocks. Both units of work, one tile for
// 8 column blocks and one block for 256 keys, take 2048 matrix cycles of a CU.
struct AttnKeyWeightsCut {
  unsigned blocks, row_blocks, row_tiles, row_parts, col_blocks, col_parts;
};
__host__ __device__ constexpr unsigned attn_key_weights_span(std::size_t units, unsigned most) {
  const std::size_t span = (units + 1023) / 1024;  // about 4 workgroups per CU
  return span < 4 ? 4u : span < most ? static_cast<unsigned>(span) : most;
}
__host__ __device__ constexpr AttnKeyWeightsCut attn_key_weights_cut(unsigned pos0, unsigned n) {
  using namespace weights_detail;
  const unsigned rows = pos0 + n, tiles = (rows + kKeys - 1) / kKeys;
  AttnKeyWeightsCut c{};
  c.blocks = (n + kTokens - 1) / kTokens;
  const unsigned groups = (c.blocks + kRowWaves - 1) / kRowWaves;
  c.row_blocks = (c.blocks + groups - 1) / groups;
  // Of the n x n square of new keys half is seen.
  const std::size_t row_units = std::size_t{groups} * (2 * std::size_t{pos0} + n) / kKeys;
  const std::size_t col_units = std::size_t{c.blocks} * (2 * std::size_t{pos0} + n) / kColKeys;
  c.row_tiles = attn_key_weights_span(row_units, 128);
  c.col_blocks = attn_key_weights_span(col_units, 64);
  c.row_tiles = c.row_tiles < tiles ? c.row_tiles : tiles;
  c.col_blocks = c.col_blocks < c.blocks ? c.col_blocks : c.blocks;
  c.row_parts = (tiles + c.row_tiles - 1) / c.row_tiles;
  c.col_parts = (c.blocks + c.col_blocks - 1) / c.col_blocks;
  return c;
}

// The workspace's parts, in bytes from its start, each 256-byte aligned.
struct AttnKeyWeightsLayout {
  std::size_t halves, meta, stats, sums, k_wide, bytes;
};
__host__ __device__ constexpr AttnKeyWeightsLayout attn_key_weights_layout(
    unsigned rows, const AttnKeyWeightsCut& cut, bool fp8) {
  const std::size_t cols = std::size_t{2} * cut.blocks * weights_detail::kCols;
  AttnKeyWeightsLayout l{};
  std::size_t at = 0;
  auto take = [&](std::size_t bytes) {
    const std::size_t was = at;
    at += (bytes + 255) / 256 * 256;
    return was;
  };
  l.halves = take(2 * cut.blocks * weights_detail::kBlockHalves * sizeof(attn::half_t));
  l.meta = take(cols * 8);
  l.stats = take(cols * 8 * cut.row_parts);
  l.sums = take(cut.col_parts > 1 ? std::size_t{2} * rows * 4 * cut.col_parts : 0);
  l.k_wide = take(fp8 ? std::size_t{2} * rows * attn::kDim * sizeof(attn::half_t) : 0);
  l.bytes = at;
  return l;
}

// Bytes that serve every launch of up to max_n tokens over up to max_rows rows, each part at its
// largest. Blocks times row parts: where row_tiles is 128, at most blocks (tiles / 128 + 1); below,
// row_tiles >= units / 1024 and units >= groups tiles less roundings, or row_tiles = 4 with at most
// 4096 units, either way at most 16400 and 3 a block. Rows times column parts likewise: rows (blocks
// / 64 + 1), or 256 keys a unit, 300000 and 2 a row.
__host__ __device__ constexpr std::size_t attn_key_weights_bytes(unsigned max_n, unsigned max_rows,
                                                                 bool fp8) {
  using namespace weights_detail;
  const std::size_t rows = max_rows, blocks = (std::size_t{max_n} + kTokens - 1) / kTokens;
  const std::size_t row_items = blocks * (rows / (kKeys * 128) + 4) + 16400;
  const std::size_t col_items = rows * (blocks / 64 + 3) + 300000;
  return 2 * blocks * kBlockHalves * sizeof(attn::half_t) + 2 * blocks * kCols * 8 +
         2 * row_items * kCols * 8 + 2 * col_items * 4 +
         (fp8 ? 2 * rows * attn::kDim * sizeof(attn::half_t) : 0) + 5 * 256;
}

// The launches of a chunk whose arguments are good (workspace of at least the layout's bytes). k8 /
// k_scale: the codes of an e4m3 cache of max_ctx rows (k_cache then unused), widened first.
inline void attn_key_weights_launch(const float* q, const attn::half_t* k_cache,
                                    const uint8_t* k8, const float* k_scale, float* weights,
                                    unsigned pos0, unsigned n, unsigned max_ctx, void* workspace,
                                    hipStream_t stream) {
  const AttnKeyWeightsCut cut = attn_key_weights_cut(pos0, n);
  const AttnKeyWeightsLayout l = attn_key_weights_layout(pos0 + n, cut, k8 != nullptr);
  char* const ws = static_cast<char*>(workspace);
  AttnKeyWeightsParams p{q,
                         k_cache,
                         weights,
                         reinterpret_cast<attn::half_t*>(ws + l.halves),
                         reinterpret_cast<float*>(ws + l.meta),
                         reinterpret_cast<float2*>(ws + l.stats),
                         reinterpret_cast<float*>(ws + l.sums),
                         pos0,
                         n,
                         max_ctx,
                         max_ctx,
                         cut.blocks,
                         cut.row_blocks,
                         cut.row_tiles,
                         cut.col_blocks};
  const unsigned rows = pos0 + n;
  if (k8 != nullptr) {
    attn::half_t* const wide = reinterpret_cast<attn::half_t*>(ws + l.k_wide);
    const unsigned grid = (2 * rows + 3) / 4;
    attn_k_fp8_widen_kernel<><<<grid < 4096 ? grid : 4096, 256, 0, stream>>>(k8, k_scale, wide,
                                                                             rows, max_ctx);
    p.k_cache = wide;
    p.k_ctx = rows;
  }
  const unsigned groups = (cut.blocks + cut.row_blocks - 1) / cut.row_blocks;
  const unsigned key_blocks = (rows + weights_detail::kColKeys - 1) / weights_detail::kColKeys;
  attn_key_weights_rows_kernel<><<<2 * groups * cut.row_parts, 512, 0, stream>>>(p);
  attn_key_weights_lse_kernel<><<<(64 * cut.blocks + 255) / 256, 256, 0, stream>>>(p);
  attn_key_weights_cols_kernel<><<<2 * key_blocks * cut.col_parts, 256, 0, stream>>>(p);
  if (cut.col_parts > 1)
    attn_key_weights_join_kernel<><<<(2 * rows + 255) / 256, 256, 0, stream>>>(p);
}

// ------------------------------------------------------------------------------------------------
// The rows to keep
//
// Per KV head: rows [0, sinks), rows [len - recent, len) and, of the rows between, the
// keep - sinks - recent of the largest weight; of equal weights the lower row. A NaN ranks below
// every number, -0 equals +0. index [2][keep], ascending.
// ------------------------------------------------------------------------------------------------

struct AttnEvictSelectParams {
  const float* weights;  // [2][max_ctx]
  int* index;            // [2][keep]
  unsigned len, max_ctx, keep, sinks, recent;
};

namespace evict_detail {

// An unsigned that orders as the weight does: NaN lowest, then the numbers.
__device__ __attribute__((always_inline)) inline unsigned rank_of(float x) {
  if (x != x)
    return 0;
  const unsigned u = cdna4::as_uint(x == 0.0f ? 0.0f : x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

}  // namespace evict_detail

// One workgroup of 1024 per KV head. Four passes over the rows narrow the rank of the last kept
// row 8 bits at a time (histograms in LDS); a last one writes the kept rows in order.
template <int = 0>
__global__ void __launch_bounds__(1024) attn_evict_select_kernel(AttnEvictSelectParams p) {
  __shared__ unsigned hist[256], found[2], waves[16], equals[16];
  const unsigned kvh = blockIdx.x, t = threadIdx.x, lane = t & 63u, wave = t >> 6;
  const float* w = p.weights + std::size_t{kvh} * p.max_ctx;
  const unsigned lo = p.sinks, hi = p.len - p.recent;
  unsigned want = p.keep - p.sinks - p.recent;  // rows of the middle still to be found
  unsigned prefix = 0;
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (t < 256)
        hist[t] = 0;
      __syncthreads();
      for (unsigned i = lo + t; i < hi; i += 1024) {
        const unsigned r = evict_detail::rank_of(w[i]);
        if (shift == 24 || r >> (shift + 8) == prefix >> (shift + 8))
          atomicAdd(&hist[r >> shift & 255u], 1u);
      }
      __syncthreads();
      if (t == 0) {
        unsigned above = 0;
        int d = 255;
        while (d > 0 && above + hist[d] < want)
          above += hist[d--];
        found[0] = static_cast<unsigned>(d);
        found[1] = above;
      }
      __syncthreads();
      prefix |= found[0] << shift;
      want -= found[1];
      __syncthreads();
    }
  }
  // Kept: the ends, ranks above the prefix, and the first `want` of those equal to it.
  unsigned at = 0, same = 0;
  for (unsigned i0 = 0; i0 < p.len; i0 += 1024) {
    const unsigned i = i0 + t;
    bool end = false, above = false, equal = false;
    if (i < p.len) {
      end = i < lo || i >= hi;
      if (!end && p.keep > p.sinks + p.recent) {
        const unsigned r = evict_detail::rank_of(w[i]);
        above = r > prefix;
        equal = r == prefix;
      }
    }
    const unsigned long long eq = __ballot(equal);
    const unsigned long long below = lane == 0 ? 0ull : ~0ull >> (64 - lane);
    if (lane == 0)
      equals[wave] = __popcll(eq);
    __syncthreads();
    unsigned eq0 = same, eq_all = 0;
    for (unsigned k = 0; k < 16; ++k) {
      eq0 += k < wave ? equals[k] : 0;
      eq_all += equals[k];
    }
    const bool kept = end || above || (equal && eq0 + __popcll(eq & below) < want);
    const unsigned long long kb = __ballot(kept);
    if (lane == 0)
      waves[wave] = __popcll(kb);
    __syncthreads();
    unsigned k0 = at, k_all = 0;
    for (unsigned k = 0; k < 16; ++k) {
      k0 += k < wave ? waves[k] : 0;
      k_all += waves[k];
    }
    if (kept)
      p.index[std::size_t{kvh} * p.keep + k0 + __popcll(kb & below)] = static_cast<int>(i);
    at += k_all;
    same += eq_all;
  }
}

// ------------------------------------------------------------------------------------------------
// The move of the kept rows
//
// Row j < keep of the destination: row index[g][j] of the source; a row whose index is outside
// [0, max_ctx) becomes zero, with weight 0. Rows from keep on keep what they hold, but their
// weights become 0 (the tokens appended next start without any).
// ------------------------------------------------------------------------------------------------

struct AttnEvictGatherParams {
  const void* k;         // [2][max_ctx][256] f16, or e4m3 codes
  const void* v;
  const float* weights;  // [2][max_ctx]
  const int* index;      // [2][keep]
  void* k_out;           // [2][out_ctx][256]
  void* v_out;
  float* weights_out;    // [2][out_ctx]
  unsigned max_ctx, keep, out_ctx;
  const float* k_scale;  // e4m3: [2][max_ctx]
  const float* v_scale;
  float* k_scale_out;    // e4m3: [2][out_ctx]
  float* v_scale_out;
};

// One row per 32 lanes (f16: 16 bytes of K and of V each; e4m3: 8). Rows [0, 2 keep) are moved, the
// 2 (out_ctx - keep) weights behind them cleared. Grid-stride, x 256.
template <bool kFp8>
__global__ void __launch_bounds__(256) attn_evict_gather_kernel(AttnEvictGatherParams p) {
  using Chunk = std::conditional_t<kFp8, uint2, uint4>;
  const unsigned lane = threadIdx.x & 31u;
  const std::size_t moved = 2 * std::size_t{p.keep};
  for (std::size_t r = 8 * std::size_t{blockIdx.x} + threadIdx.x / 32; r < moved;
       r += 8 * std::size_t{gridDim.x}) {
    const unsigned kvh = r >= p.keep, j = static_cast<unsigned>(r - (kvh ? p.keep : 0));
    const int from = p.index[r];
    const bool in = static_cast<unsigned>(from) < p.max_ctx;
    const std::size_t src = std::size_t{kvh} * p.max_ctx + (in ? from : 0);
    const std::size_t dst = std::size_t{kvh} * p.out_ctx + j;
    Chunk a = static_cast<const Chunk*>(p.k)[src * 32 + lane];
    Chunk b = static_cast<const Chunk*>(p.v)[src * 32 + lane];
    if (!in)
      a = b = Chunk{};
    static_cast<Chunk*>(p.k_out)[dst * 32 + lane] = a;
    static_cast<Chunk*>(p.v_out)[dst * 32 + lane] = b;
    if (lane == 0)
      p.weights_out[dst] = in ? p.weights[src] : 0.0f;
    if (kFp8 && lane == 1)
      p.k_scale_out[dst] = in ? p.k_scale[src] : 0.0f;
    if (kFp8 && lane == 2)
      p.v_scale_out[dst] = in ? p.v_scale[src] : 0.0f;
  }
  const std::size_t rest = p.out_ctx - p.keep;
  for (std::size_t i = std::size_t{blockIdx.x} * 256 + threadIdx.x; i < 2 * rest;
       i += 256 * std::size_t{gridDim.x})
    p.weights_out[(i / rest) * p.out_ctx + p.keep + i % rest] = 0.0f;
}

}  // namespace miso::kernels
