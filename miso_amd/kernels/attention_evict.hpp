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
//
// Bound by the K and V stream, as attn_decode: 32768 keys take 18.8 us against 18.4 without
// weights, 262144 104 against 88.4 (5.2 TB/s of what must move), of which 5 are the merge's and the
// others the score stores among the loads; 301 keys 11 to 12 against 9.4, two launches (8.7 on the
// card) and the host's call. 100003 e4m3 keys 30.2 against 25.8: half the bytes of K and V, the same
// scores (the split 26.6 against 22.5).
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

// attn_prep_split_kernel (a layer step's split, the token prepared in it), the scores stored. The
// token's row is s.len - 1, its rotation p.rope's. Grid dim3(n_splits, 2) x 256.
template <int kBlock>
__global__ void __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(1, 1)))
attn_prep_split_scores_kernel(AttnPrepSplitParams p, float* ws) {
  static_assert(kBlock == 256, "four waves per split workgroup");
  using namespace decode_detail;
  __shared__ TileShared sh;
  __shared__ __attribute__((aligned(16))) PrepShared ps;
  const unsigned split = blockIdx.x, kvh = blockIdx.y;
  const std::size_t head = std::size_t{kvh} * p.s.max_ctx * attn::kDim;
  const std::size_t row = head + std::size_t{p.s.len - 1} * attn::kDim;
  const AttnSpan span = attn_split_span(p.s.len, p.s.n_splits, split);
  const LinearTiles tl{p.s.k_cache + head, p.s.v_cache + head};
  const std::size_t base = std::size_t{kvh} * p.s.n_splits + split;
  const PrepQuery q{p.proj, p.q_norm, p.k_norm, p.rope,
                    split == 0 ? p.q + std::size_t{kvh} * kGroup * attn::kDim : nullptr,
                    p.k_cache + row, p.v_cache + row, &ps, p.eps, p.s.len - 1};
  const SplitScores sc = scores_of(ws, p.s.len, p.s.n_splits, kvh);
  if (span.end - span.begin > kSplitWavesMinKeys)  // as attn_prep_split_kernel
    split_partial_waves(q, tl, span, kvh, p.s.part_m, p.s.part_l, p.s.part_o, base, sh, false, sc);
  else
    split_partial_tiles<LinearTiles, false>(q, tl, span, kvh, p.s.part_m, p.s.part_l, p.s.part_o,
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
  float* h;            // a layer step's residual row [2048]: h += delta; nullptr: none
  const float* delta;
};

constexpr unsigned kCombineItems = attn::kQHeads * (attn::kDim / 64);  // 64-thread workgroups
constexpr unsigned kWeightKeys = 256;  // keys per workgroup of the weights' part

// Workgroups [0, 64): attn_combine_kernel's; with h, 8 more for the residual row; the others one
// 256-key block of one KV head each: every lane forms the head statistics from the splits' and adds
// 4 keys' weights, 64 apart (blocks of 64 threads, so that few keys still fill many CUs and the
// scores are asked for before the statistics are joined). 3.7 us at 301 keys, 4.2 at 32768, 9.9 at
// 262144: the stream of the scores. Grid attn_combine_weights_grid, x 64.
__host__ __device__ constexpr unsigned attn_combine_weights_grid(unsigned len, bool add) {
  return kCombineItems + (add ? 8 : 0) + 2 * (len / kWeightKeys + (len % kWeightKeys != 0));
}
template <int = 0>
__global__ void __launch_bounds__(64) attn_combine_weights_kernel(AttnWeightsParams p) {
  using decode_detail::kGroup;
  if (blockIdx.x < kCombineItems) {
    attn_combine_op<64, true, 4>(p.c, 0, kCombineItems);
    return;
  }
  const unsigned lane = threadIdx.x, adds = p.h != nullptr ? 8 : 0;
  if (blockIdx.x < kCombineItems + adds) {
    const unsigned e = 256 * (blockIdx.x - kCombineItems) + 4 * lane;
    const float4 a = *reinterpret_cast<const float4*>(p.h + e);
    const float4 d = *reinterpret_cast<const float4*>(p.delta + e);
    *reinterpret_cast<float4*>(p.h + e) = float4{a.x + d.x, a.y + d.y, a.z + d.z, a.w + d.w};
    return;
  }
  const unsigned item = blockIdx.x - kCombineItems - adds;
  const unsigned blocks = p.len / kWeightKeys + (p.len % kWeightKeys != 0);
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
// before it can join its column's sum, so the products q k are formed twice: the first pass gives
// each query's maximum and sum, the second sums 2^(s - lse) over the queries. (Keeping the scores
// instead would move the 16 heads' 64 bytes per token and key through memory twice, 27 ps at a large
// copy's rate, against 16 x 1024 flop, 14 ps at a large product's.)
//
// A query is 32 bits wide and the matrix cores take 16: each block of 32 columns is scaled by the
// power of two that puts its largest element in [2^13, 2^14), multiplied by log2(e), and cut into
// f16 halves x = hi + lo, in all exact to 2^-22 of x, or 2^-38 of the block's largest element where lo
// is subnormal (what counts is a score's absolute error: beside a query element of 1000, that is 4e-9
// per unit of K). hi k + lo k are exact products summed in f32. What comes off in the exponent's fma is
// a power of two, so that a maximum taken of scaled scores is the very number that the fma subtracts
// from, however large the scores (a scale with log2(e) in it left its rounding, 2^-25 of a score, in
// the exponent: infinite weights from scores of 2^32 on). A scale per column would take 16 registers
// more in the second pass, which has 4 left of its 256. So a score costs 1024 flop of f16 matrix work
// per pass, and the passes are bound by it once there are some hundred queries.
//
// A KV head's queries are columns c = 8 t + h % 8 in blocks of 32 (4 tokens). A wave holds one
// block's halves in registers (128 VGPRs) and a workgroup of W waves, W blocks (a group), streams K
// tiles of 32 rows through an LDS ring: one read of a K operand serves the hi and the lo product,
// and the ring takes 64 of the 128 bytes a clock that LDS gives. Both passes have this form; in the
// first a tile's result has the keys in registers and the columns in lanes (the running maximum and
// sum stay in a lane), in the second the columns in registers and the keys in lanes (a key's sum
// over the block is 16 adds).
//
// The work of a pass is the tiles of (KV head, group), laid end to end and cut into equal spans,
// one per workgroup: causal groups differ in length, and a span takes up where the one before it
// ends.
//
// Measured: 8192 tokens after 8192 in 2.55-2.60 ms, 1270-1300 TFLOP/s of f16 products (1.3 ms a
// pass, the matrix units busy in 73 and 77% of the cycles; zeros for data take as many cycles in 0.95
// to 0.99 ms, so the card's power, which sets the clock, bounds it); 2048 tokens 95.3 us (passes of
// 42, with zeros 37; the matrix units busy in 54 and 52% of the cycles: a span has 17 tiles behind a
// start of 6 us); 1001 after 5003 e4m3 rows 156-160; 33 after 12001 37.5 us (four launches; passes of
// 15.5 and 19, 5 of them in tiles).
// ------------------------------------------------------------------------------------------------

struct AttnKeyWeightsParams {
  const float* q;               // [n][16][256]
  const attn::half_t* k_cache;  // [2][k_ctx][256]
  float* weights;               // [2][max_ctx]
  attn::half_t* halves;         // [2][blocks][hi, lo][16][64][8], in the order of the operands
  float* scale;                 // [2][blocks]: 1 / 16 over the block's power of two
  float2* stats;                // [span + group][32 W]: a span's (maximum, sum) of a group's columns
  float* sums;                  // [2][groups][row_tiles][32]: a group's sums of its keys
  unsigned pos0, n, max_ctx, k_ctx;
  unsigned blocks;              // column blocks: ceil(n / 4)
  unsigned groups;              // ceil(blocks / W)
  unsigned row_tiles;           // tiles of 32 rows: ceil((pos0 + n) / 32)
  unsigned spans;               // workgroups of a pass
  unsigned long long span;      // tiles of one
};

namespace weights_detail {

constexpr unsigned kCols = 32, kKeys = 32, kSteps = 16;  // of a tile; k-steps of 16 dimensions
constexpr unsigned kTokens = kCols / decode_detail::kGroup;
constexpr std::size_t kBlockHalves = 2 * kSteps * 64 * 8;  // one column block's halves

__host__ __device__ constexpr unsigned div_up(unsigned a, unsigned b) {
  return a / b + (a % b != 0);
}

// Tiles of group g, for W = 8 (32 tokens) and W = 4 (16): those up to the last row that a token of
// its 32-token run sees. It may name one tile past the rows for the last groups, whose keys nobody
// sees.
__host__ __device__ constexpr unsigned group_tiles(unsigned W, unsigned pos0, unsigned g) {
  return div_up(pos0, kKeys) + 1 + (W == 8 ? g : g / 2);
}
// Their sum over the groups before g.
__host__ __device__ constexpr unsigned long long tiles_before(unsigned W, unsigned pos0,
                                                              unsigned g) {
  const unsigned long long x = g, h = g / 2;
  return x * (div_up(pos0, kKeys) + 1) +
         (W == 8 ? x * (x - (x != 0)) / 2 : h * (h - (h != 0)) + (g % 2 ? h : 0));
}

__device__ __attribute__((always_inline)) inline cdna4::float16_t mfma32(
    const cdna4::half8_t& a, const cdna4::half8_t& b, const cdna4::float16_t& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Row of a tile's result that a lane's value i belongs to.
__device__ __attribute__((always_inline)) inline unsigned tile_row(unsigned lane, unsigned i) {
  return 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
}

constexpr int kVmcnt0 = 0x0F70;  // s_waitcnt vmcnt(0), the other counters as they are

constexpr float kNoScore = -3e38f;  // below every score, and finite: differences stay numbers

// A ring of K tiles, chunk c of row r at position c ^ (r % 16) of the row (the operand read of 16
// lanes takes one chunk of 16 rows: 16 positions); in the second pass, the waves' sums of W tiles,
// twice, and the columns' lse.
constexpr unsigned kStages = 4, kTileBytes = kKeys * attn::kDim * 2;
template <unsigned W>
struct alignas(1024) PassShared {
  unsigned char k[kStages][kTileBytes];
  float red[2][W][W][64];  // [run of W tiles][tile][wave][lane]
  float lse[W][kCols];
};

// The statistics of N spans a wave half, v0 .. w1 at most, of a lane's column of group lin, joined
// into (m, l): all loads in flight together.
template <unsigned W, unsigned N>
__device__ __attribute__((always_inline)) inline void add_stats(float& m, float& l,
                                                               const float2* stats, unsigned lin,
                                                               unsigned v0, unsigned w1,
                                                               unsigned wave, unsigned lane) {
  float2 one[N];
#pragma unroll
  for (unsigned i = 0; i < N; ++i) {
    const unsigned v = v0 + 2 * i + (lane >> 5);  // 32-bit offsets: at most 512 + 2 groups slots
    const unsigned at = ((v < w1 ? v : w1) + lin) * (W * kCols) + wave * kCols + (lane & 31u);
    one[i] = stats[at];
    one[i] = v <= w1 ? one[i] : float2{kNoScore, 0.0f};
  }
  float top = m;
#pragma unroll
  for (unsigned i = 0; i < N; ++i)
    top = fmaxf(top, one[i].x);
  l *= __builtin_amdgcn_exp2f(m - top);
#pragma unroll
  for (unsigned i = 0; i < N; ++i)
    l = __builtin_fmaf(one[i].y, __builtin_amdgcn_exp2f(one[i].x - top), l);
  m = top;
}

// This lane's halves of its block: column lane % 32, dimensions 16 s + 8 (lane / 32) .. + 7.
struct Halves {
  cdna4::half8_t hi[kSteps], lo[kSteps];
};

}  // namespace weights_detail

struct AttnKWidenParams {
  const uint8_t* k8;     // [2][max_ctx][256]
  const float* k_scale;  // [2][max_ctx]
  attn::half_t* out;     // [2][n][256]
  unsigned n, max_ctx;
};

namespace weights_detail {
// K codes widened to f16 (attn_kv_fp8_widen_kernel's values, K alone: the matrix cores take f16, a
// code's 4 bits fit it exactly, and only row scales below 2^-15 make subnormals, off by 2^-25 at
// most, which is below what f32 sums of ordinary scores lose): workgroup `first` of
// `groups` of 4 waves, 8 codes a lane, 8 rows of a wave in flight.
constexpr unsigned kWidenRows = 32;  // a workgroup's at a time
__device__ __attribute__((always_inline)) inline void widen_rows(const AttnKWidenParams& p,
                                                                unsigned first, unsigned groups) {
  const unsigned lane = threadIdx.x & 31u, half = threadIdx.x >> 5;
  const std::size_t rows = 2 * std::size_t{p.n};
  for (std::size_t r0 = std::size_t{kWidenRows} * first + half; r0 < rows;
       r0 += std::size_t{kWidenRows} * groups) {
    uint2 w[4];
    float sc[4];
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
      const std::size_t r = r0 + 8 * i < rows ? r0 + 8 * i : r0;
      const std::size_t src = r < p.n ? r : r - p.n + p.max_ctx;
      w[i] = *reinterpret_cast<const uint2*>(p.k8 + src * attn::kDim + 8 * lane);
      sc[i] = p.k_scale[src];
    }
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
      const cdna4::half2_t e[4] = {
          cdna4::as_half2(fp8kv::pair_lo(w[i].x)), cdna4::as_half2(fp8kv::pair_hi(w[i].x)),
          cdna4::as_half2(fp8kv::pair_lo(w[i].y)), cdna4::as_half2(fp8kv::pair_hi(w[i].y))};
      cdna4::half8_t h;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        h[k] = static_cast<_Float16>(
            fminf(fmaxf(static_cast<float>(e[k / 2][k % 2]) * sc[i], -65504.0f), 65504.0f));
      if (r0 + 8 * i < rows)
        *reinterpret_cast<cdna4::half8_t*>(p.out + (r0 + 8 * i) * attn::kDim + 8 * lane) = h;
    }
  }
}
}  // namespace weights_detail

// The queries' halves and scales. One workgroup of 4 waves per (KV head, column block): wave w
// reads columns 8 w .. 8 w + 7, one row of 1 KiB an instruction, and the halves go out through LDS
// in the order of the operands, 16 bytes a lane. In LDS the 512 bytes of a k-step's half (s,
// dimension / 8 % 2) are 528 apart, so that the 32 of them that one row touches lie in different
// banks. Padding columns are zero. Bound by memory, 8 bytes per query element: 42 us for 8192
// tokens (268 MB), 11 for 2048.
//
// kFp8: the workgroups from 2 p.blocks on widen the rows of an e4m3 cache, which the cut does not
// need (33 tokens after 12001 rows: 41.8 us, with a launch of its own 44.6).
template <bool kFp8>
__global__ void __launch_bounds__(256) attn_key_weights_cut_kernel(AttnKeyWeightsParams p,
                                                                  AttnKWidenParams widen) {
  using namespace weights_detail;
  if constexpr (kFp8)
    if (blockIdx.x >= 2 * p.blocks) {
      widen_rows(widen, blockIdx.x - 2 * p.blocks, gridDim.x - 2 * p.blocks);
      return;
    }
  constexpr unsigned kPer = kCols / 4, kStep = 528, kHalf = 2 * kSteps * kStep;
  __shared__ __attribute__((aligned(16))) unsigned char sh[2 * kHalf];
  __shared__ float most[4];
  const unsigned t = threadIdx.x, lane = t & 63u, wave = t >> 6;
  const unsigned kvh = blockIdx.x / p.blocks, block = blockIdx.x % p.blocks;
  float4 x[kPer];
  float top = 0.0f;
#pragma unroll
  for (unsigned i = 0; i < kPer; ++i) {
    const unsigned c = kPer * wave + i, tok = kTokens * block + c / decode_detail::kGroup;
    x[i] = float4{0.0f, 0.0f, 0.0f, 0.0f};
    if (tok < p.n)  // wave-uniform
      x[i] = *reinterpret_cast<const float4*>(
          p.q + (std::size_t{tok} * attn::kQHeads + kvh * decode_detail::kGroup +
                 c % decode_detail::kGroup) * attn::kDim + 4 * lane);
  }
#pragma unroll
  for (unsigned i = 0; i < kPer; ++i)
    top = fmaxf(top, fmaxf(fmaxf(__builtin_fabsf(x[i].x), __builtin_fabsf(x[i].y)),
                           fmaxf(__builtin_fabsf(x[i].z), __builtin_fabsf(x[i].w))));
  top = cdna4::wave_allmax(top);
  if (lane == 0)
    most[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
  // 2^(13 - e), e the exponent of top; blocks of zeros or below 2^-87 keep a finite factor, and one
  // that holds an infinity stays as it is (its scores are infinite or NaN either way).
  int e = 13 - (static_cast<int>(cdna4::as_uint(top) >> 23) - 127);
  e = top == 0.0f || top == __builtin_inff() ? 0 : (e < 100 ? e : 100);
  const float up = __builtin_ldexpf(1.0f, e);
#pragma unroll
  for (unsigned i = 0; i < kPer; ++i) {
    const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    cdna4::half4_t hi, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float y = v[j] * up * decode_detail::kLog2e;  // up: a power of two, exact
      // One value for both halves: the product must not be rounded to f16 within one instruction here
      // and to f32 there, which near the middle of two f16 are a step of f16 apart.
      asm("" : "+v"(y));
      hi[j] = static_cast<_Float16>(y);
      lo[j] = static_cast<_Float16>(y - static_cast<float>(hi[j]));
    }
    unsigned char* at = sh + lane / 2 * kStep + 16 * (kPer * wave + i) + 8 * (lane % 2);
    *reinterpret_cast<cdna4::half4_t*>(at) = hi;
    *reinterpret_cast<cdna4::half4_t*>(at + kHalf) = lo;
  }
  __syncthreads();
  uint4* out = reinterpret_cast<uint4*>(p.halves + std::size_t{blockIdx.x} * kBlockHalves);
#pragma unroll
  for (unsigned i = 0; i < 8; ++i) {
    const unsigned at = 256 * i + t;  // 32 lanes of 16 bytes per half of a k-step
    out[at] = *reinterpret_cast<const uint4*>(sh + at / 1024 * kHalf + at % 1024 / 32 * kStep +
                                              at % 32 * 16);
  }
  if (t == 0)
    p.scale[blockIdx.x] = __builtin_ldexpf(1.0f / 16.0f, -e);
}

// One span of a pass (kSum: the second), x 64 W, one workgroup of 8 waves or two of 4 per CU.
// Iteration t of a segment (the span's tiles of one group) forms the scores of tile t while the
// vector units work on those of tile t - 1.
template <unsigned W, bool kSum>
__global__ void __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2, 2)))
attn_key_weights_pass_kernel(AttnKeyWeightsParams p) {
  using namespace weights_detail;
  using cdna4::float16_t;
  __shared__ PassShared<W> sh;
  const unsigned lane = threadIdx.x & 63u;
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Neighbouring spans on one XCD (blocks go round robin), so that its L2 serves one KV head.
  const unsigned w = blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
  if (w >= p.spans)
    return;
  const unsigned long long per_head = tiles_before(W, p.pos0, p.groups);
  unsigned long long x = w * p.span;
  const unsigned long long x_end = x + p.span < 2 * per_head ? x + p.span : 2 * per_head;
  unsigned kvh = x >= per_head;
  unsigned group = 0, tile;
  {  // the group that holds tile x - kvh per_head
    const unsigned long long at = x - kvh * per_head;
    unsigned past = p.groups;
    while (past - group > 1) {
      const unsigned mid = (group + past) / 2;
      if (tiles_before(W, p.pos0, mid) <= at)
        group = mid;
      else
        past = mid;
    }
    tile = static_cast<unsigned>(at - tiles_before(W, p.pos0, group));
  }
  const unsigned ring = cdna4::lds_offset(sh.k[0]);
  const unsigned rows = p.pos0 + p.n;
  const unsigned kl = 512 * (lane & 31u) + 16 * ((lane >> 5) ^ (lane & 15u));

  for (bool again = false; x < x_end; again = true) {
    const unsigned tiles = group_tiles(W, p.pos0, group);
    const unsigned first = tile;
    const unsigned past =
        tiles - first < x_end - x ? tiles : first + static_cast<unsigned>(x_end - x);
    const attn::half_t* K = p.k_cache + std::size_t{kvh} * p.k_ctx * attn::kDim;
    // Tile ti into its stage: this wave copies rows 32 / W wave .. , two an instruction.
    constexpr unsigned kCopies = kKeys / W / 2;
    auto issue = [&](unsigned ti) __attribute__((always_inline)) {
#pragma unroll
      for (unsigned i = 0; i < kCopies; ++i) {
        const unsigned r0 = kKeys / W * wave + 2 * i, r = r0 + (lane >> 5);
        const unsigned row = ti * kKeys + r < rows ? ti * kKeys + r : rows - 1;
        cdna4::lds_load16(K + std::size_t{row} * attn::kDim + 8 * ((lane & 31u) ^ (r & 15u)),
                          ring + ti % kStages * kTileBytes + 512 * r0);
      }
    };
    // Says to the compiler that no load is under way: it does not know of the waits below, and
    // would wait for the copies before it loads into registers that the segment before loaded.
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    if (again)
      decode_detail::tile_barrier();  // every wave is done with the segment before
#pragma unroll
    for (unsigned i = 0; i < kStages - 1; ++i)
      if (first + i < past)
        issue(first + i);

    const unsigned block = group * W + wave;
    const bool active = block < p.blocks;  // wave-uniform
    const unsigned lin = kvh * p.groups + group;
    Halves b;
    float scale, lse[kSum ? 16 : 1];
    if (active) {
      const std::size_t at = std::size_t{kvh} * p.blocks + block;
      const attn::half_t* in = p.halves + at * kBlockHalves + 8 * lane;
#pragma unroll
      for (unsigned s = 0; s < kSteps; ++s) {
        b.hi[s] = *reinterpret_cast<const cdna4::half8_t*>(in + 512 * s);
        b.lo[s] = *reinterpret_cast<const cdna4::half8_t*>(in + 512 * (kSteps + s));
      }
      scale = p.scale[at];
      if constexpr (kSum) {
        // The column's lse from the spans that hold tiles of the group: each half of the wave takes
        // every other one, in its order; a long chunk has a few of them, a short one over a long
        // cache a hundred.
        const unsigned long long g0 = kvh * per_head + tiles_before(W, p.pos0, group);
        const unsigned w0 = static_cast<unsigned>(g0 / p.span);
        const unsigned w1 = static_cast<unsigned>((g0 + tiles - 1) / p.span);
        float m = kNoScore, l = 0.0f;
        if (w1 - w0 < 4)
          add_stats<W, 2>(m, l, p.stats, lin, w0, w1, wave, lane);
        else
          for (unsigned v = w0; v <= w1; v += 32)
            add_stats<W, 16>(m, l, p.stats, lin, v, w1, wave, lane);
        const float top = cdna4::max_xor32(m);
        const float all = cdna4::sum_xor32(l * __builtin_amdgcn_exp2f(m - top));
        const unsigned t = kTokens * block + (lane & 31u) / decode_detail::kGroup;
        // Both halves of the wave write the same values.
        sh.lse[wave][lane & 31u] = t < p.n ? top + __builtin_amdgcn_logf(all) : __builtin_inff();
#pragma unroll
        for (unsigned i = 0; i < 16; ++i)
          lse[i] = sh.lse[wave][tile_row(lane, i)];
      }
    }
    const unsigned open = p.pos0 + kTokens * block;  // every token of the block sees keys up to it
    // First pass: the column's sum l relative to the reference m, which follows the largest score
    // only when a tile's weights sum to more than kLead (sums stay far inside f32's range, the
    // exponentials need not wait for a tile's maximum, and most tiles need none).
    constexpr float kLead = 0x1p40f;
    float m = kNoScore, l = 0.0f;
    float part[4];
    float16_t acc[2];
    cdna4::half8_t a[4];  // the operands of the next four k-steps

    // The scores of tile ti with the keys that a column does not see as -inf.
    auto mask = [&](float16_t& y, unsigned ti) __attribute__((always_inline)) {
      if (ti * kKeys + kKeys - 1 <= open)  // wave-uniform
        return;
#pragma unroll
      for (unsigned i = 0; i < 16; ++i) {
        const unsigned key = ti * kKeys + (kSum ? lane & 31u : tile_row(lane, i));
        const unsigned seen = open + (kSum ? i / 4 : (lane & 31u) / decode_detail::kGroup);
        y[i] = key <= seen ? y[i] : -__builtin_inff();
      }
    };
    auto exponent = [&](const float16_t& y, unsigned i) __attribute__((always_inline)) {
      return __builtin_fmaf(y[i], scale, kSum ? -lse[kSum ? i : 0] : -m);
    };
    auto weight = [&](const float16_t& y, unsigned i) __attribute__((always_inline)) {
      return __builtin_amdgcn_exp2f(exponent(y, i));
    };
    auto largest = [&](const float16_t& y) __attribute__((always_inline)) {
      float mx = y[0];
#pragma unroll
      for (int i = 1; i < 15; i += 2)
        mx = decode_detail::tile_max3(mx, y[i], y[i + 1]);
      return decode_detail::tile_max(mx, y[15]) * scale;
    };
    // After a tile's weights: its sums to LDS (second pass), or into l.
    auto finish = [&](const float16_t& y, unsigned ti) __attribute__((always_inline)) {
      if constexpr (kSum) {
        sh.red[ti / W % 2][ti % W][wave][lane] = (part[0] + part[1]) + (part[2] + part[3]);
      } else {
        float sum = (part[0] + part[1]) + (part[2] + part[3]);
        if (__builtin_amdgcn_ballot_w64(sum > kLead)) {  // rare, and every column's first tile
          const float top = fmaxf(m, largest(y));
          l *= __builtin_amdgcn_exp2f(m - top);
          m = top;
          part[0] = part[1] = part[2] = part[3] = 0.0f;
#pragma unroll
          for (unsigned i = 0; i < 16; ++i)
            part[i % 4] += weight(y, i);
          sum = (part[0] + part[1]) + (part[2] + part[3]);
        }
        l += sum;
      }
    };
    // The waves' sums of a run of W tiles, one tile a wave, added in wave order.
    auto take = [&](unsigned run) __attribute__((always_inline)) {
      const unsigned ti = run * W + wave;
      if (ti < first || ti >= past || ti >= p.row_tiles)
        return;
      float v[W];
#pragma unroll
      for (unsigned k = 0; k < W; ++k)
        v[k] = sh.red[run % 2][wave][k][lane];
#pragma unroll
      for (unsigned k = 1; k < W; ++k)
        v[0] += v[k];
      const float all = cdna4::sum_xor32(v[0]);
      if (p.groups == 1) {  // nothing to join
        const unsigned key = ti * kKeys + lane;
        if (lane < kKeys && key < rows)
          p.weights[std::size_t{kvh} * p.max_ctx + key] += all;
      } else if (lane < kKeys) {
        p.sums[(std::size_t{lin} * p.row_tiles + ti) * kKeys + lane] = all;
      }
    };
    // K-step s of tile ti, at kl ^ 32 s of its stage (the ring is 1 KiB aligned, so the bits that
    // change are kl's own; kl has no bit of 256).
    auto read = [&](unsigned ti, unsigned s) __attribute__((always_inline)) {
      return decode_detail::lds_b128(((ring + ti % kStages * kTileBytes + kl) ^ (32u * (s % 8))) +
                                     32u * (s & 8u));
    };
    // The scores of tile ti into cur and the weights of tile ti - 1, whose scores prev holds.
    // Between two matrix instructions stand one fma, one exponential and one sum, of three
    // neighbouring weights, so that none waits for another; the next copies and the sums of a run
    // of tiles go behind the first matrix instructions.
    auto step = [&](float16_t& cur, float16_t& prev, unsigned ti) __attribute__((always_inline)) {
      mask(prev, ti - 1);
      part[0] = part[1] = part[2] = part[3] = 0.0f;
      float x1 = 0.0f, e1 = 0.0f;
#pragma unroll
      for (unsigned s = 0; s < kSteps; ++s) {
        __builtin_amdgcn_sched_barrier(0);
        const cdna4::half8_t next = s + 4 < kSteps ? read(ti, s + 4) : read(ti + 1, s + 4 - kSteps);
        const float16_t from = s == 0 ? float16_t{} : cur;
        cur = kSum ? mfma32(b.hi[s], a[s % 4], from) : mfma32(a[s % 4], b.hi[s], from);
        const float x = exponent(prev, s);
        if (s > 1)
          part[(s - 2) % 4] += e1;
        const float e = __builtin_amdgcn_exp2f(x1);
        cur = kSum ? mfma32(b.lo[s], a[s % 4], cur) : mfma32(a[s % 4], b.lo[s], cur);
        a[s % 4] = next;
        e1 = e;
        x1 = x;
        if (s == 1 && ti + kStages - 1 < past)
          issue(ti + kStages - 1);
        if constexpr (kSum)
          if (s == 3 && (ti - 2) % W == W - 1 && ti > first + 1)
            take((ti - 2) / W);
      }
      __builtin_amdgcn_sched_barrier(0);
      part[2] += e1;
      part[3] += __builtin_amdgcn_exp2f(x1);
    };
    // Tile ti + 1 has landed: this wave's copies by the count, every wave's by the barrier, which
    // also says that every wave has read tile ti - 1, whose stage the next copy takes. So a wave
    // reads the first operands of tile ti + 1 at the end of its tile ti.
    auto turn = [&](unsigned ti) __attribute__((always_inline)) {
      if (ti + 2 < past)
        cdna4::wait_vmcnt<kCopies>();
      else
        cdna4::wait_vmcnt<0>();
      decode_detail::tile_barrier();
    };

    if (!active) {  // copies, and sums nothing
      if constexpr (kSum) {
#pragma unroll
        for (unsigned i = 0; i < 2 * W; ++i)
          sh.red[i / W][i % W][wave][lane] = 0.0f;
      }
      for (unsigned ti = first; ti < past; ++ti) {
        turn(ti);
        if (ti + kStages - 1 < past)
          issue(ti + kStages - 1);
        if constexpr (kSum)
          if ((ti - 2) % W == W - 1 && ti > first + 1)
            take((ti - 2) / W);
      }
    } else {
      turn(first);
#pragma unroll
      for (unsigned s = 0; s < 4; ++s)
        a[s] = read(first, s);
#pragma unroll
      for (unsigned s = 0; s < kSteps; ++s) {
        const cdna4::half8_t next =
            s + 4 < kSteps ? read(first, s + 4) : read(first + 1, s + 4 - kSteps);
        const float16_t from = s == 0 ? float16_t{} : acc[0];
        acc[0] = kSum ? mfma32(b.hi[s], a[s % 4], from) : mfma32(a[s % 4], b.hi[s], from);
        acc[0] = kSum ? mfma32(b.lo[s], a[s % 4], acc[0]) : mfma32(a[s % 4], b.lo[s], acc[0]);
        a[s % 4] = next;
      }
      if (first + kStages - 1 < past)
        issue(first + kStages - 1);
      unsigned ti = first + 1;
      for (; ti + 1 < past; ti += 2) {
        turn(ti);
        step(acc[1], acc[0], ti);
        finish(acc[0], ti - 1);
        turn(ti + 1);
        step(acc[0], acc[1], ti + 1);
        finish(acc[1], ti);
      }
      if (ti < past) {
        turn(ti);
        step(acc[1], acc[0], ti);
        finish(acc[0], ti - 1);
        acc[0] = acc[1];
      }
      mask(acc[0], past - 1);
      part[0] = part[1] = part[2] = part[3] = 0.0f;
#pragma unroll
      for (unsigned i = 0; i < 16; ++i)
        part[i % 4] += weight(acc[0], i);
      finish(acc[0], past - 1);
      if constexpr (!kSum) {  // the two halves of the wave hold the other keys of the same columns
        const float top = cdna4::max_xor32(m);
        const float sum = cdna4::sum_xor32(l * __builtin_amdgcn_exp2f(m - top));
        if (lane < kCols)
          p.stats[(std::size_t{w} + lin) * (W * kCols) + wave * kCols + lane] = float2{top, sum};
      }
    }
    if constexpr (kSum) {
      decode_detail::tile_barrier();
      // The last run, and the one before it where that ended with tile past - 2 (its turn to be
      // taken would have come with a tile `past`).
      if (past % W == 1 && past - first > 1)
        take((past - 2) / W);
      take((past - 1) / W);
    }
    x += past - first;
    tile = past;
    if (tile == tiles) {
      tile = 0;
      if (++group == p.groups) {
        group = 0;
        ++kvh;
      }
    }
  }
}

// weights += the groups' sums, in a fixed order: one workgroup per (KV head, tile of rows), 8
// slices of the groups that hold the tile, joined in slice order. Bound by memory: 256 groups over
// 16384 rows (8192 tokens after 8192, 25 MB of sums) 6.6 us.
template <unsigned W>
__global__ void __launch_bounds__(256) attn_key_weights_join_kernel(AttnKeyWeightsParams p) {
  using namespace weights_detail;
  __shared__ float part[8][kKeys];
  const unsigned kvh = blockIdx.x / p.row_tiles, tile = blockIdx.x % p.row_tiles;
  const unsigned lane = threadIdx.x % kKeys, slice = threadIdx.x / kKeys;
  const unsigned base = div_up(p.pos0, kKeys);  // group_tiles(g) > tile from here on
  const unsigned g0 = tile > base ? (tile - base) * (W == 8 ? 1 : 2) : 0;
  const float* s = p.sums + (std::size_t{kvh} * p.groups * p.row_tiles + tile) * kKeys + lane;
  float v = 0.0f;
#pragma unroll 4
  for (unsigned g = g0 + slice; g < p.groups; g += 8)
    v += s[std::size_t{g} * p.row_tiles * kKeys];
  part[slice][lane] = v;
  __syncthreads();
  const unsigned key = tile * kKeys + lane;
  if (slice != 0 || key >= p.pos0 + p.n)
    return;
#pragma unroll
  for (unsigned i = 1; i < 8; ++i)
    v += part[i][lane];
  p.weights[std::size_t{kvh} * p.max_ctx + key] += v;
}

// How a chunk is cut: column blocks, the waves W of a workgroup, the groups, and the spans of a
// pass. W = 8 is one workgroup per CU, W = 4 two, which hide each other's starts and barriers but
// stream K twice. Two while K stays in an XCD's L2 (us, W = 4 against 8: 300 tokens 18.1 against
// 20.9, 2048 96 against 109, 4000 after 100 280 against 289; level with many rows before the chunk,
// 1000 after 1000 68.6 against 68.8, and behind at the rule's edge, 2000 after 2000 188 against 180).
// One beyond (2048 after 12001 731 against 690; 17 after 40000, 5 blocks, 56.6 against 50), except
// for few blocks that fill groups of 4 better (33 after 40000, 9 blocks, 72 against 79.5; over fewer
// rows it can be the other way, 33 after 12001 38.2 against 36.2, and 64 after 5000, 16 blocks, which
// fill either, 30.2 against 33.1).
struct AttnKeyWeightsCut {
  unsigned blocks, waves, groups, row_tiles, spans;
  unsigned long long span;
};
// Groups of 4 also keep within the bound of the sums: 9 to 11 of them up to 762000 rows or more.
constexpr unsigned kWeightsCus = 256, kWeightsNearRows = 4096;
// The (group, row) sums of a KV head, for a piece over `rows` rows: 8 groups' at least, so that a
// streamed K serves them together (2.1 million rows, 256 tokens: 13.7 ms, in pieces of 4 groups 15.2).
__host__ __device__ constexpr std::size_t attn_key_weights_most_sums(std::size_t rows) {
  return 8 * rows > std::size_t{1} << 23 ? 8 * rows : std::size_t{1} << 23;
}
__host__ __device__ constexpr AttnKeyWeightsCut attn_key_weights_cut(unsigned pos0, unsigned n) {
  using namespace weights_detail;
  AttnKeyWeightsCut c{};
  c.blocks = div_up(n, kTokens);
  const unsigned rows = pos0 + n;
  const bool fills = c.blocks < 64 && 27 * div_up(c.blocks, 4) < 50 * div_up(c.blocks, 8) &&
                     std::size_t{div_up(c.blocks, 4)} * rows <= attn_key_weights_most_sums(rows);
  c.waves = rows <= kWeightsNearRows || fills ? 4 : 8;
  c.groups = div_up(c.blocks, c.waves);
  c.row_tiles = div_up(rows, kKeys);
  const unsigned long long tiles = 2 * tiles_before(c.waves, pos0, c.groups);
  const unsigned most = kWeightsCus * (8 / c.waves);
  c.span = (tiles + most - 1) / most;
  c.spans = static_cast<unsigned>((tiles + c.span - 1) / c.span);
  return c;
}

// A chunk runs in pieces of at most this many tokens, so that the groups' sums (8 bytes per group
// and row) stay within 64 MiB, or 64 bytes a row beyond 2^20 rows (where the cache has 2048).
__host__ __device__ constexpr unsigned attn_key_weights_tokens(unsigned rows) {
  const std::size_t few = rows < 64 ? 64 : rows;
  return 32 * static_cast<unsigned>(attn_key_weights_most_sums(few) / few);
}

// The groups that a piece of up to `blocks` column blocks over up to `rows` rows has at most, where
// its groups of 4 are not among the near rows' (those are counted by themselves).
__host__ __device__ constexpr std::size_t attn_key_weights_groups(std::size_t blocks) {
  return (blocks < 64 ? blocks / 4 : blocks < 120 ? 15 : blocks / 8) + 1;
}
// Floats of the groups' sums of pieces of up to `blocks` column blocks over up to `rows` rows (whole
// tiles): never less for more blocks or rows. A piece's groups, 513 at most, times its rows are
// within attn_key_weights_most_sums, so times its whole tiles' rows at most 2^14 above it.
__host__ __device__ constexpr std::size_t attn_key_weights_sums(std::size_t blocks,
                                                                std::size_t rows) {
  const std::size_t far = attn_key_weights_groups(blocks) * rows;
  const std::size_t near_blocks = blocks < kWeightsNearRows / 4 ? blocks : kWeightsNearRows / 4;
  const std::size_t near =
      (near_blocks / 4 + 1) * (rows < kWeightsNearRows ? rows : std::size_t{kWeightsNearRows});
  const std::size_t most = attn_key_weights_most_sums(rows) + (1u << 14);
  const std::size_t sums = far > near ? far : near;
  return 2 * (sums < most ? sums : most);
}

// The workspace's parts, in bytes from its start, each 256-byte aligned.
struct AttnKeyWeightsLayout {
  std::size_t halves, scale, stats, sums, k_wide, bytes;
};
__host__ __device__ constexpr AttnKeyWeightsLayout attn_key_weights_parts(
    std::size_t blocks, std::size_t sums_floats, std::size_t wide_rows) {
  using namespace weights_detail;
  AttnKeyWeightsLayout l{};
  std::size_t at = 0;
  auto take = [&](std::size_t bytes) {
    const std::size_t was = at;
    at += (bytes + 255) / 256 * 256;
    return was;
  };
  l.halves = take(2 * blocks * kBlockHalves * sizeof(attn::half_t));
  l.scale = take(2 * blocks * 4);
  // (spans + 2 groups) x 32 W columns, spans x W <= 8 x 256, groups x W <= 8 (blocks / 8 + 1)
  l.stats = take((kWeightsCus + 2 * (blocks / 8 + 1)) * 8 * kCols * sizeof(float2));
  l.sums = take(sums_floats * 4);
  l.k_wide = take(2 * wide_rows * attn::kDim * sizeof(attn::half_t));
  l.bytes = at;
  return l;
}

// Of one chunk.
__host__ __device__ constexpr AttnKeyWeightsLayout attn_key_weights_layout(unsigned pos0, unsigned n,
                                                                           bool fp8) {
  using namespace weights_detail;
  const unsigned rows = pos0 + n, most = attn_key_weights_tokens(rows);
  const unsigned blocks = div_up(n < most ? n : most, kTokens);
  return attn_key_weights_parts(
      blocks,
      attn_key_weights_sums(blocks, std::size_t{div_up(rows, kKeys)} * kKeys),
      fp8 ? rows : 0);
}

// Bytes that serve every chunk of up to max_n tokens over up to max_rows rows. A piece has at most
// 16384 tokens (its tokens times its rows, at least as many, are at most 2^28, or it has 256).
__host__ __device__ constexpr std::size_t attn_key_weights_bytes(unsigned max_n, unsigned max_rows,
                                                                 bool fp8) {
  using namespace weights_detail;
  const std::size_t blocks = div_up(max_n < 16384 ? max_n : 16384, kTokens);
  const std::size_t rows = std::size_t{div_up(max_rows, kKeys)} * kKeys;
  return attn_key_weights_parts(blocks, attn_key_weights_sums(blocks, rows), fp8 ? max_rows : 0)
      .bytes;
}

template <unsigned W>
void attn_key_weights_passes(const AttnKeyWeightsParams& p, hipStream_t stream) {
  const unsigned grid = (p.spans + 7) / 8 * 8;
  attn_key_weights_pass_kernel<W, false><<<grid, 64 * W, 0, stream>>>(p);
  attn_key_weights_pass_kernel<W, true><<<grid, 64 * W, 0, stream>>>(p);
  if (p.groups > 1)
    attn_key_weights_join_kernel<W><<<2 * p.row_tiles, 256, 0, stream>>>(p);
}

// The launches of a chunk whose arguments are good, with a workspace of the bytes of its own layout
// at least. k8 / k_scale: the codes of an e4m3 cache of max_ctx rows (k_cache then unused), widened
// beside the first piece's cut.
inline void attn_key_weights_launch(const float* q, const attn::half_t* k_cache,
                                    const uint8_t* k8, const float* k_scale, float* weights,
                                    unsigned pos0, unsigned n, unsigned max_ctx, void* workspace,
                                    hipStream_t stream) {
  const unsigned rows = pos0 + n;
  const AttnKeyWeightsLayout l = attn_key_weights_layout(pos0, n, k8 != nullptr);
  char* const ws = static_cast<char*>(workspace);
  unsigned k_ctx = max_ctx;
  AttnKWidenParams widen{};
  if (k8 != nullptr) {
    attn::half_t* const wide = reinterpret_cast<attn::half_t*>(ws + l.k_wide);
    widen = {k8, k_scale, wide, rows, max_ctx};
    k_cache = wide;
    k_ctx = rows;
  }
  const unsigned most = attn_key_weights_tokens(rows);
  for (unsigned t = 0; t < n; t += most) {
    const unsigned m = n - t < most ? n - t : most;
    const AttnKeyWeightsCut cut = attn_key_weights_cut(pos0 + t, m);
    const AttnKeyWeightsParams p{q + std::size_t{t} * attn::kQHeads * attn::kDim,
                                 k_cache,
                                 weights,
                                 reinterpret_cast<attn::half_t*>(ws + l.halves),
                                 reinterpret_cast<float*>(ws + l.scale),
                                 reinterpret_cast<float2*>(ws + l.stats),
                                 reinterpret_cast<float*>(ws + l.sums),
                                 pos0 + t,
                                 m,
                                 max_ctx,
                                 k_ctx,
                                 cut.blocks,
                                 cut.groups,
                                 cut.row_tiles,
                                 cut.spans,
                                 cut.span};
    if (k8 != nullptr && t == 0) {
      const unsigned grid = 2 * rows / weights_detail::kWidenRows + 1;
      attn_key_weights_cut_kernel<true>
          <<<2 * cut.blocks + (grid < 4096 ? grid : 4096), 256, 0, stream>>>(p, widen);
    } else {
      attn_key_weights_cut_kernel<false><<<2 * cut.blocks, 256, 0, stream>>>(p, widen);
    }
    if (cut.waves == 8)
      attn_key_weights_passes<8>(p, stream);
    else
      attn_key_weights_passes<4>(p, stream);
  }
}

// ------------------------------------------------------------------------------------------------
// The rows to keep
//
// Per KV head: rows [0, sinks), rows [len - recent, len) and, of the rows between, the
// keep - sinks - recent of the largest weight; of equal weights the lower row. A NaN ranks below
// every number, -0 equals +0. index [2][keep], ascending.
//
// A row's rank is an unsigned that orders as its weight does, all ones for the rows that are kept
// in any case and 0 for what lies behind the last row. The last kept row's rank is found digit by
// digit, 11, 11 and 10 bits: a histogram of the rows that agree so far, and the bin in which the
// count from the top reaches what is still to be kept. Then the rows above that rank are kept, and
// of those equal to it the first ones. Counts are whole numbers, so their order does not matter.
//
// Bound by latencies, not bytes: 6.3 us for 2048 rows (4.4 on the card, the host's call), 22.6 for
// 262144 (2 MB, four launches). Joining all groups' histograms in every launch instead of adding
// them up in memory took 35.6: 512 KiB to read per workgroup.
// ------------------------------------------------------------------------------------------------

struct AttnEvictSelectParams {
  const float* weights;  // [2][max_ctx]
  int* index;            // [2][keep]
  unsigned len, max_ctx, keep, sinks, recent;
  // Caches of several workgroups a head: their number, a workgroup's rows, and the workspace
  // [2][evict_detail::part_words(groups)].
  unsigned groups, rows;
  unsigned* ws;
};

namespace evict_detail {

constexpr unsigned kSelectWaves = 16;

// The rank of row `row`, whose weight is x: NaN 1, then the numbers, -0 as +0.
__device__ __attribute__((always_inline)) inline unsigned rank_of(const AttnEvictSelectParams& p,
                                                                 unsigned row, float x) {
  const unsigned u = cdna4::as_uint(x + 0.0f);  // -0 becomes +0
  unsigned rank = u & 0x80000000u ? ~u : u | 0x80000000u;
  rank = x != x ? 1u : rank;
  rank = row < p.sinks || row >= p.len - p.recent ? ~0u : rank;
  return row < p.len ? rank : 0u;
}

// Bits [kLow, kHigh) of a rank, and whether the rank agrees with the prefix found above them.
template <unsigned kLow, unsigned kHigh>
__device__ __attribute__((always_inline)) inline unsigned digit_of(unsigned rank) {
  return rank >> kLow & ((1u << (kHigh - kLow)) - 1);
}
template <unsigned kHigh>
__device__ __attribute__((always_inline)) inline bool agrees(unsigned rank, unsigned prefix) {
  return kHigh == 32 || rank >> (kHigh % 32) == prefix >> (kHigh % 32);
}

// The inclusive sum over the lanes up to this one: within rows of 16 lanes by row shifts, then the
// last lane of a row into the next one and of the lower half into the upper (DPP moves; the same
// sum by shuffles through LDS took a quarter of a microsecond).
template <int kCtrl, int kRows>
__device__ __attribute__((always_inline)) inline unsigned add_lanes(unsigned x) {
  return x + __builtin_amdgcn_update_dpp(0u, x, kCtrl, kRows, 0xF, false);
}
__device__ __attribute__((always_inline)) inline unsigned wave_scan(unsigned x) {
  x = add_lanes<0x111, 0xF>(x);  // row_shr:1, 2, 4, 8
  x = add_lanes<0x112, 0xF>(x);
  x = add_lanes<0x114, 0xF>(x);
  x = add_lanes<0x118, 0xF>(x);
  x = add_lanes<0x142, 0xA>(x);   // row_bcast:15 into rows 1 and 3
  return add_lanes<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
}

// Lanes below this one that are set in a wave's mask.
__device__ __attribute__((always_inline)) inline unsigned lanes_below(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(mask), 0));
}

template <unsigned kBins>
struct SelectShared {
  unsigned hist[kBins];
  unsigned waves[2][kSelectWaves];
  unsigned digit, above, count;
};

// One row a lane into the histogram of bits [kLow, kHigh), each bin kCopies times (lanes of one bin
// follow one another). Where all of the wave's rows that agree with the prefix have one digit
// (untouched rows, the newest ones), they are added in one go.
template <unsigned kLow, unsigned kHigh, unsigned kCopies>
__device__ __attribute__((always_inline)) inline void count_digit(unsigned* hist, unsigned rank,
                                                                 unsigned prefix, unsigned lane) {
  const bool counts = agrees<kHigh>(rank, prefix);
  const unsigned long long which = __builtin_amdgcn_ballot_w64(counts);
  if (which == 0)  // wave-uniform
    return;
  const unsigned bin = digit_of<kLow, kHigh>(rank) * kCopies;
  const unsigned one = __builtin_amdgcn_readlane(bin, __builtin_ctzll(which));
  if (__builtin_amdgcn_ballot_w64(counts && bin != one) == 0) {  // wave-uniform
    if (lane == 0)
      atomicAdd(&hist[one], static_cast<unsigned>(__popcll(which)));
  } else if (counts) {
    atomicAdd(&hist[bin + lane % kCopies], 1u);
  }
}

template <unsigned kBins>
__device__ __attribute__((always_inline)) inline void clear_digits(SelectShared<kBins>& sh) {
#pragma unroll
  for (unsigned i = 0; i < kBins; i += 1024)
    sh.hist[i + threadIdx.x] = 0;
  __syncthreads();
}

// The bin in which the count from the top reaches `want` (sh.digit), its count (sh.count) and that
// of the bins above it (sh.above); thread t holds c[i] of bin top - kPer t - i. 1 <= want <= the
// histogram's total. Ends with a barrier.
template <unsigned kPer, unsigned kBins>
__device__ __attribute__((always_inline)) inline void find_digit(SelectShared<kBins>& sh,
                                                                const unsigned (&c)[kPer],
                                                                unsigned top, unsigned want) {
  const unsigned t = threadIdx.x, lane = t & 63u, wave = t >> 6;
  unsigned mine = 0;
#pragma unroll
  for (unsigned i = 0; i < kPer; ++i)
    mine += c[i];
  const unsigned incl = wave_scan(mine);
  if (lane == 63)
    sh.waves[0][wave] = incl;
  __syncthreads();
  unsigned above = incl - mine;
#pragma unroll
  for (unsigned k = 0; k < kSelectWaves; ++k)
    above += k < wave ? sh.waves[0][k] : 0;
  if (above < want && want <= above + mine) {  // one thread
    unsigned i = 0, count = c[0];
#pragma unroll
    for (unsigned k = 0; k + 1 < kPer; ++k)
      if (i == k && want > above + count) {
        above += count;
        count = c[k + 1];
        ++i;
      }
    sh.digit = top - kPer * t - i;
    sh.above = above;
    sh.count = count;
  }
  __syncthreads();
}

// Where this wave's kept rows go. `sure` and `equals`: its rows above the found rank and equal to
// it (wave-uniform); `before` and `same`: kept rows and equal rows before the workgroup; `want`:
// how many equal rows are kept. Returns the place of the wave's first kept row and moves `same` on
// to the equal rows before the wave.
template <unsigned kBins>
__device__ __attribute__((always_inline)) inline unsigned place_wave(SelectShared<kBins>& sh,
                                                                    unsigned sure, unsigned equals,
                                                                    unsigned before,
                                                                    unsigned& same, unsigned want) {
  const unsigned wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63u) == 0) {
    sh.waves[0][wave] = sure;
    sh.waves[1][wave] = equals;
  }
  __syncthreads();
  const unsigned kept = same < want ? same : want;  // equal rows kept before the workgroup
#pragma unroll
  for (unsigned k = 0; k < kSelectWaves; ++k) {
    before += k < wave ? sh.waves[0][k] : 0;
    same += k < wave ? sh.waves[1][k] : 0;
  }
  return before + (same < want ? same : want) - kept;
}

// Writes the kept rows of 64, row `row` of rank `rank` this lane's, from out[at] on; never past
// `keep` of them, which only weights that change under the selection could ask for.
__device__ __attribute__((always_inline)) inline void write_kept(int* out, unsigned keep,
                                                                unsigned& at, unsigned& same,
                                                                unsigned want, unsigned rank,
                                                                unsigned last, unsigned row) {
  const unsigned long long equal = __builtin_amdgcn_ballot_w64(rank == last);
  const bool mine = rank > last || (rank == last && same + lanes_below(equal) < want);
  const unsigned long long kept = __builtin_amdgcn_ballot_w64(mine);
  if (mine && at + lanes_below(kept) < keep)
    out[at + lanes_below(kept)] = static_cast<int>(row);
  at += __popcll(kept);
  same += __popcll(equal);
}

}  // namespace evict_detail

// One workgroup of 1024 per KV head for up to 1024 R rows, their ranks in registers: wave w's
// register i holds row 64 (R w + i) + lane, so that the registers in turn are the rows' order.
template <unsigned R>
__global__ void __launch_bounds__(1024) attn_evict_select_kernel(AttnEvictSelectParams p) {
  using namespace evict_detail;
  constexpr unsigned kBins = 2048;
  __shared__ SelectShared<3 * kBins> sh;
  const unsigned kvh = blockIdx.x, t = threadIdx.x, lane = t & 63u;
  const unsigned wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const float* w = p.weights + std::size_t{kvh} * p.max_ctx;
  const unsigned row0 = 64 * R * wave + lane;
  float x[R];
  unsigned rank[R];
#pragma unroll
  for (unsigned i = 0; i < R; ++i)
    x[i] = row0 + 64 * i < p.len ? w[row0 + 64 * i] : 0.0f;
#pragma unroll
  for (unsigned i = 0; i < R; ++i)
    rank[i] = rank_of(p, row0 + 64 * i, x[i]);
  unsigned want = p.keep, last = 0;
  clear_digits(sh);
  auto digit = [&](auto which, auto low, auto high) __attribute__((always_inline)) {
    unsigned* const hist = sh.hist + decltype(which)::value * kBins;
#pragma unroll
    for (unsigned i = 0; i < R; ++i)
      count_digit<decltype(low)::value, decltype(high)::value, 1>(hist, rank[i], last, lane);
    __syncthreads();
    const unsigned c[2] = {hist[kBins - 1 - 2 * t], hist[kBins - 2 - 2 * t]};
    find_digit(sh, c, kBins - 1, want);
    last |= sh.digit << decltype(low)::value;
    want -= sh.above;
  };
  using std::integral_constant;
  using Zero = integral_constant<unsigned, 0>;
  digit(Zero{}, integral_constant<unsigned, 21>{}, integral_constant<unsigned, 32>{});
  digit(integral_constant<unsigned, 1>{}, integral_constant<unsigned, 10>{},
        integral_constant<unsigned, 21>{});
  // Two digits are enough where every row that agrees with them is kept (most often a single one):
  // the rows above the rank before theirs, and none equal to it. 8192 rows: 6.9 us against 7.6;
  // with 16 rows a lane that is rarer and the branch itself costs more (16384 rows: 13.8 against
  // 11.8).
  if (R <= 8 && sh.count == want && last != 0) {
    --last;
    want = 0;
  } else {
    digit(integral_constant<unsigned, 2>{}, Zero{}, integral_constant<unsigned, 10>{});
  }
  unsigned sure = 0, equals = 0, same = 0;
#pragma unroll
  for (unsigned i = 0; i < R; ++i) {
    sure += __popcll(__builtin_amdgcn_ballot_w64(rank[i] > last));
    equals += __popcll(__builtin_amdgcn_ballot_w64(rank[i] == last));
  }
  unsigned at = place_wave(sh, sure, equals, 0, same, want);
  int* out = p.index + std::size_t{kvh} * p.keep;
#pragma unroll
  for (unsigned i = 0; i < R; ++i)
    write_kept(out, p.keep, at, same, want, rank[i], last, row0 + 64 * i);
}

// Longer caches: `groups` workgroups per head (64 at most), p.rows rows each, in four launches, a
// digit of 8, 12 and 12 bits each and the writing. A head's part of the workspace:
//   first [groups][256]: the groups' histograms of the first digit, which every workgroup of the
//     second launch joins for itself;
//   hist [2][4096]: those of the other two over all groups, cleared by the first launch, added to by
//     every workgroup (counts: the order of the additions does not matter) and read by the next;
//   upto [groups][4100]: after the third launch, a group's rows that agree with the first two digits
//     and whose third is at least b, and its rows above them, at [b], b <= 4096: from it the last
//     launch has the kept rows before a workgroup's with two loads a group;
//   state [4]: (prefix, rows still to be kept) after the first and the second digit.
// Grid dim3(groups, 2) x 1024.
namespace evict_detail {
constexpr unsigned kFirstBins = 256, kPartBins = 4096, kUpto = kPartBins + 4;
__host__ __device__ constexpr std::size_t part_words(std::size_t groups) {
  return groups * (kFirstBins + kUpto) + 2 * kPartBins + 4;
}
}  // namespace evict_detail
template <unsigned kLaunch>
__global__ void __launch_bounds__(1024) attn_evict_select_part_kernel(AttnEvictSelectParams p) {
  using namespace evict_detail;
  __shared__ SelectShared<kPartBins> sh;
  const unsigned kvh = blockIdx.y, g = blockIdx.x, t = threadIdx.x, lane = t & 63u;
  const unsigned wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const float* w = p.weights + std::size_t{kvh} * p.max_ctx;
  const unsigned r0 = g * p.rows;
  const unsigned r1 = p.len - r0 < p.rows ? p.len : r0 + p.rows;
  unsigned* const hist = p.ws + kvh * part_words(p.groups);
  unsigned* const first = hist + 2 * kPartBins;
  unsigned* const upto = first + p.groups * kFirstBins;
  unsigned* const state = upto + std::size_t{p.groups} * kUpto;
  // Each wave takes a stretch of the rows, 64 at a time; the first 512 are loaded before all else.
  const unsigned per = p.rows / kSelectWaves;
  const unsigned s0 = r0 + wave * per < r1 ? r0 + wave * per : r1;
  const unsigned s1 = s0 + per < r1 ? s0 + per : r1;
  constexpr unsigned kChunk = 512;
  float x[kChunk / 64];
  auto load = [&](unsigned from) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned i = 0; i < kChunk / 64; ++i) {
      const unsigned row = from + 64 * i + lane;
      x[i] = row < s1 ? w[row] : 0.0f;
    }
  };
  auto rank_at = [&](unsigned from, unsigned i) __attribute__((always_inline)) {
    const unsigned row = from + 64 * i + lane;
    return row < s1 ? rank_of(p, row, x[i]) : 0u;
  };
  load(s0);
  unsigned want = p.keep, last = 0;
  if constexpr (kLaunch == 0) {
    for (unsigned i = g * 1024 + t; i < 2 * kPartBins; i += p.groups * 1024)
      hist[i] = 0;
  } else if constexpr (kLaunch == 1) {
    // A quarter of the threads per quarter of the groups, 16 at most: all loads in flight.
    const unsigned bin = kFirstBins - 1 - t % kFirstBins;
    unsigned one[16], c[1] = {0};
#pragma unroll
    for (unsigned i = 0; i < 16; ++i) {
      const unsigned k = t / kFirstBins + 4 * i;
      one[i] = first[(k < p.groups ? k : 0) * kFirstBins + bin];
      c[0] += k < p.groups ? one[i] : 0;
    }
    sh.hist[t] = c[0];
    __syncthreads();
    c[0] = 0;
    if (t < kFirstBins)
      c[0] = sh.hist[t] + sh.hist[t + 256] + sh.hist[t + 512] + sh.hist[t + 768];
    find_digit(sh, c, kFirstBins - 1, want);
    last = sh.digit << 24;
  } else {
    last = state[2 * (kLaunch - 2)];
    want = state[2 * (kLaunch - 2) + 1];
    const uint4 four = *reinterpret_cast<const uint4*>(hist + (kLaunch - 2) * kPartBins +
                                                       kPartBins - 4 - 4 * t);
    const unsigned c[4] = {four.w, four.z, four.y, four.x};
    find_digit(sh, c, kPartBins - 1, want);
    last |= sh.digit << (kLaunch == 2 ? 12 : 0);
  }
  if constexpr (kLaunch > 0)
    want -= sh.above;
  if constexpr (kLaunch == 1 || kLaunch == 2) {
    if (g == 0 && t == 0) {
      state[2 * (kLaunch - 1)] = last;
      state[2 * (kLaunch - 1) + 1] = want;
    }
  }
  if constexpr (kLaunch < 3) {
    constexpr unsigned kLow = kLaunch == 0 ? 24 : kLaunch == 1 ? 12 : 0;
    constexpr unsigned kHigh = kLaunch == 0 ? 32 : kLow + 12, kCopies = kLaunch == 0 ? 16 : 1;
    unsigned sure = 0;  // rows above the prefix
    clear_digits(sh);
    for (unsigned from = s0; from < s1; from += kChunk) {  // wave-uniform
      if (from != s0)
        load(from);
#pragma unroll
      for (unsigned i = 0; i < kChunk / 64; ++i) {
        const unsigned rank = rank_at(from, i);
        count_digit<kLow, kHigh, kCopies>(sh.hist, rank, last, lane);
        if (kLaunch == 2)
          sure += __popcll(__builtin_amdgcn_ballot_w64(rank >> 12 > last >> 12));
      }
    }
    if (kLaunch == 2 && lane == 0)
      sh.waves[1][wave] = sure;
    __syncthreads();
    if constexpr (kLaunch == 0) {
      if (t < kFirstBins) {
        unsigned all = 0;
#pragma unroll
        for (unsigned i = 0; i < kCopies; ++i)
          all += sh.hist[kCopies * t + (i + t) % kCopies];
        first[g * kFirstBins + t] = all;
      }
    } else {
      unsigned* const out = hist + (kLaunch - 1) * kPartBins;
#pragma unroll
      for (unsigned i = 0; i < kPartBins; i += 1024)  // neighbouring bins to neighbouring lanes
        if (const unsigned n = sh.hist[i + t])
          atomicAdd(&out[i + t], n);
      if constexpr (kLaunch == 2) {
        const unsigned bin = kPartBins - 4 - 4 * t;
        const uint4 c = *reinterpret_cast<const uint4*>(&sh.hist[bin]);
        const unsigned mine = c.x + c.y + c.z + c.w;
        const unsigned incl = wave_scan(mine);
        if (lane == 63)
          sh.waves[0][wave] = incl;
        __syncthreads();
        unsigned before = 0, at = incl - mine;
#pragma unroll
        for (unsigned k = 0; k < kSelectWaves; ++k) {
          before += sh.waves[1][k];
          at += k < wave ? sh.waves[0][k] : 0;
        }
        at += before;
        uint4 up;
        up.w = at + c.w;
        up.z = up.w + c.z;
        up.y = up.z + c.y;
        up.x = up.y + c.x;
        unsigned* const u = upto + std::size_t{g} * kUpto;
        *reinterpret_cast<uint4*>(u + bin) = up;
        if (t == 0)
          u[kPartBins] = before;
      }
    }
  } else {
    // Rows above the found rank, and rows equal to it, in the workgroups before this one: a group
    // a lane, every wave for itself.
    const unsigned* u = upto + std::size_t{lane < g ? lane : 0} * kUpto + (last & 4095u);
    const unsigned from_last = u[0], past_last = u[1];
    unsigned before = wave_scan(lane < g ? past_last : 0);
    unsigned same = wave_scan(lane < g ? from_last - past_last : 0);
    before = __builtin_amdgcn_readlane(before, 63);
    same = __builtin_amdgcn_readlane(same, 63);
    before += same < want ? same : want;
    // Each wave counts its stretch, and writes behind the waves before it.
    unsigned sure = 0, equals = 0;
    for (unsigned from = s0; from < s1; from += kChunk) {
      if (from != s0)
        load(from);
#pragma unroll
      for (unsigned i = 0; i < kChunk / 64; ++i) {
        const unsigned rank = rank_at(from, i);
        sure += __popcll(__builtin_amdgcn_ballot_w64(rank > last));
        equals += __popcll(__builtin_amdgcn_ballot_w64(rank == last));
      }
    }
    unsigned at = place_wave(sh, sure, equals, before, same, want);
    int* out = p.index + std::size_t{kvh} * p.keep;
    for (unsigned from = s0; from < s1; from += kChunk) {
      if (per > kChunk)
        load(from);
#pragma unroll
      for (unsigned i = 0; i < kChunk / 64; ++i)
        write_kept(out, p.keep, at, same, want, rank_at(from, i), last, from + 64 * i + lane);
    }
  }
}

// Up to this many rows one workgroup a head holds them all (11.8 us at 16384 rows; the four
// launches take 19, and one workgroup for 20000 rows 21.8). Beyond, workgroups of whole runs of
// 1024 rows, at most 64 (262144 rows: half a microsecond faster than 32).
constexpr unsigned kSelectOneGroup = 16384, kSelectMostGroups = 64;
__host__ __device__ constexpr unsigned attn_evict_group_rows(unsigned len) {
  return ((len - 1) / kSelectMostGroups / 1024 + 1) * 1024;
}

// Bytes of the selection's workspace for len rows (more rows never need less).
__host__ __device__ constexpr std::size_t attn_evict_bytes(unsigned len) {
  if (len <= kSelectOneGroup)
    return 256;
  const std::size_t runs = len / 1024 + (len % 1024 != 0);
  return 2 * evict_detail::part_words(runs < kSelectMostGroups ? runs : kSelectMostGroups) *
         sizeof(unsigned);
}

// The launches of a selection whose arguments are good; ws of attn_evict_bytes(p.len).
inline void attn_evict_select_launch(AttnEvictSelectParams p, void* ws, hipStream_t stream) {
  p.ws = static_cast<unsigned*>(ws);
  if (p.len <= 2048) {
    attn_evict_select_kernel<2><<<2, 1024, 0, stream>>>(p);
  } else if (p.len <= 8192) {
    attn_evict_select_kernel<8><<<2, 1024, 0, stream>>>(p);
  } else if (p.len <= kSelectOneGroup) {
    attn_evict_select_kernel<16><<<2, 1024, 0, stream>>>(p);
  } else {
    p.rows = attn_evict_group_rows(p.len);
    p.groups = (p.len - 1) / p.rows + 1;
    const dim3 grid(p.groups, 2);
    attn_evict_select_part_kernel<0><<<grid, 1024, 0, stream>>>(p);
    attn_evict_select_part_kernel<1><<<grid, 1024, 0, stream>>>(p);
    attn_evict_select_part_kernel<2><<<grid, 1024, 0, stream>>>(p);
    attn_evict_select_part_kernel<3><<<grid, 1024, 0, stream>>>(p);
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

// A row of K or V is 32 (f16) or 16 (e4m3) lanes of 16 bytes; a thread moves its chunk of both, of
// two rows over e4m3 rows (65535 rows: 30.3 us against 33.6; over f16 rows one is faster, 51.5
// against 53.8). Rows [0, 2 keep) are moved, the 2 (out_ctx - keep) weights behind them cleared.
// Grid-stride, x 256. Bound by memory: 8192 f16 rows of 32768 in 8.1 us (33.8 MB, 4.2 TB/s), 65535
// e4m3 rows of 131072 in 30.2 (138 MB, 4.6 TB/s).
template <bool kFp8>
__global__ void __launch_bounds__(256) attn_evict_gather_kernel(AttnEvictGatherParams p) {
  constexpr unsigned kLanes = kFp8 ? 16 : 32, kRows = 256 / kLanes, kTwo = kFp8 ? 2 : 1;
  const unsigned lane = threadIdx.x % kLanes;
  const std::size_t moved = 2 * std::size_t{p.keep};
  for (std::size_t r0 = std::size_t{blockIdx.x} * kRows * kTwo; r0 < moved;
       r0 += std::size_t{gridDim.x} * kRows * kTwo) {
    uint4 a[kTwo], b[kTwo];
    std::size_t src[kTwo], dst[kTwo];
    bool here[kTwo], in[kTwo];
#pragma unroll
    for (unsigned i = 0; i < kTwo; ++i) {
      const std::size_t r = r0 + kRows * i + threadIdx.x / kLanes;
      here[i] = r < moved;
      const unsigned kvh = r >= p.keep, j = static_cast<unsigned>(r - (kvh ? p.keep : 0));
      const unsigned from = here[i] ? static_cast<unsigned>(p.index[r]) : ~0u;
      in[i] = from < p.max_ctx;
      src[i] = std::size_t{kvh} * p.max_ctx + from;
      dst[i] = std::size_t{kvh} * p.out_ctx + j;
    }
#pragma unroll
    for (unsigned i = 0; i < kTwo; ++i) {
      a[i] = b[i] = uint4{};
      if (in[i]) {
        a[i] = static_cast<const uint4*>(p.k)[src[i] * kLanes + lane];
        b[i] = static_cast<const uint4*>(p.v)[src[i] * kLanes + lane];
      }
    }
#pragma unroll
    for (unsigned i = 0; i < kTwo; ++i)
      if (here[i]) {
        static_cast<uint4*>(p.k_out)[dst[i] * kLanes + lane] = a[i];
        static_cast<uint4*>(p.v_out)[dst[i] * kLanes + lane] = b[i];
        if (lane == 0)
          p.weights_out[dst[i]] = in[i] ? p.weights[src[i]] : 0.0f;
        if (kFp8 && lane == 1)
          p.k_scale_out[dst[i]] = in[i] ? p.k_scale[src[i]] : 0.0f;
        if (kFp8 && lane == 2)
          p.v_scale_out[dst[i]] = in[i] ? p.v_scale[src[i]] : 0.0f;
      }
  }
  const std::size_t rest = p.out_ctx - p.keep;
#pragma unroll
  for (unsigned kvh = 0; kvh < 2; ++kvh) {
    float* w = p.weights_out + std::size_t{kvh} * p.out_ctx + p.keep;
    for (std::size_t i = std::size_t{blockIdx.x} * 256 + threadIdx.x; i < rest;
         i += 256 * std::size_t{gridDim.x})
      w[i] = 0.0f;
  }
}

// Workgroups of a move: the rows' steps, and at most 4 steps of the clearing (16 rows into a cache
// of 262144: 7.4 us, e4m3 9.4, most of it the host's call; sized by the rows alone 60 and 230).
template <bool kFp8>
constexpr unsigned attn_evict_gather_grid(unsigned keep, unsigned out_ctx) {
  const std::size_t rows = kFp8 ? 32 : 8;  // of a workgroup's step
  const std::size_t moves = (2 * std::size_t{keep} + rows - 1) / rows;
  const std::size_t clears = (std::size_t{out_ctx} - keep + 1023) / 1024;
  const std::size_t groups = moves > clears ? moves : clears;
  return groups < (1u << 20) ? static_cast<unsigned>(groups) : 1u << 20;
}

}  // namespace miso::kernels
