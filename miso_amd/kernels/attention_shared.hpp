#pragma once

// Batched decode behind a prefix that all sequences share, for MI355X (gfx950 / CDNA4); no reference
// counterpart (the reference is batch-1). The ragged and paged decodes (attention_decode.hpp) read the
// prefix once per sequence: 64 sequences behind 32768 keys stream 4.3 GB. Here the queries of all
// sequences meet the prefix's keys together, so that K and V are read once per 16 sequences (8
// behind short prefixes):
//   attn_shared_split_kernel: partials of 8 query rows per sequence and KV head over spans of the prefix,
//                             and the streaming split over each sequence's own keys behind it
//   attn_shared_merge_kernel: both partials joined, the gate applied
// Precision is the decodes': every f32 operand (queries, numerators) enters the matrix units as a pair
// of f16, sums are f32.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "attention_decode.hpp"
#include "attention_evict.hpp"
#include "attention_prefill.hpp"
#include "cdna4_wave.hpp"

namespace miso::kernels {

// The prefix's rows: contiguous, K and V [2][ctx][256], or pages of a pool.
struct AttnSharedPrefix {
  const attn::half_t* k;
  const attn::half_t* v;
  const int32_t* table;  // nullptr: contiguous
  std::size_t ctx;       // rows of a KV head where contiguous
  unsigned log2_page;
  unsigned len;  // keys
};

struct AttnSharedParams {
  const float* q;     // [batch][16][256] (unscaled)
  const float* gate;  // [batch][16][256]
  float* core;        // [batch][16][256]
  const uint32_t* lens;  // [batch]: own keys, or (whole) all keys, the prefix's among them
  AttnSharedPrefix prefix;
  float4* part_o;    // [span][KV head][row block][dimension block of 32][4][64 lanes]
  float2* part_ml;   // [span][KV head][row of 8 batch, padded]: reference (log2 units), sum
  unsigned batch;
  unsigned spans, span_tiles;  // of the prefix; 0: no prefix
  unsigned blocks;             // row blocks (of 32 rows: 4 sequences x 8 heads)
  bool whole;
  // The own keys' partials, [batch][2][s_max][8] and 256 times that, as the ragged decode's, but the maxima
  // in log2 units: to natural ones and back a maximum of 1000 moves by 6e-5, the weights with it.
  float* own_m;
  float* own_l;
  float* own_o;
  unsigned s_max, chunk, own_cap;  // s_max 0: nobody has own keys
  unsigned* balanced;
  // Of a split launch: workgroups of the prefix, the first of the own keys, sequences.
  unsigned prefix_grid, own_first, own_batch;
  unsigned* chosen;    // word for the spans where the kernel chooses them (AttnSharedCut), or nullptr
  unsigned own_least;  // and the workgroups that the own keys take at least
  bool own_waves;      // sequences of few own keys may be a wave's each
};

// Own keys of one sequence in tiles, as attn_shared_cost counts them, both heads': four waves at a time, or
// a wave each (wave_items).
__host__ __device__ constexpr float attn_shared_own_tiles(unsigned keys, bool waves) {
  const unsigned n = waves ? 32 : 128, rounds = keys / n + (keys % n != 0);
  return waves ? 1.5f * static_cast<float>(rounds) : 8.0f * static_cast<float>(rounds);
}

// Partials of a sequence of `mine` own keys. Without any, `chunk` may be a word that nobody wrote: the cut
// that the kernel chooses for a batch of no own keys can take every workgroup for the prefix, and then none
// is left to choose the own keys' span.
__host__ __device__ inline unsigned attn_shared_own_splits(unsigned mine, unsigned s_max,
                                                           unsigned chunk) {
  return mine != 0 ? attn_ragged_seq_splits(mine, s_max, chunk) : 0;
}

// Where a split launch cuts the prefix.
struct AttnSharedCut {
  unsigned spans, span_tiles, grid;  // grid: the prefix's workgroups, a multiple of 8
  bool both;                         // the own keys are every workgroup's, behind its span
};

// What the tiles of a launch cost on `cus` CUs, a workgroup each, in us without the fixed part: the
// slower side, or the span and its share of the `own` tiles of own keys (both heads') one after the
// other. A tile of a span behind 64 sequences takes 1.5 us (32768 keys of 40 tiles a span: 70 us), behind
// 8 1.0 (9 tiles: 23 us, 12: 26), behind 3 0.9; of the own keys 1.5 (48 workgroups: 72 us, 32: 97), four
// at a time, a wave each: a sequence of 5 keys counts as four tiles (106 of them on 32 CUs: 45 us); the own
// keys' start behind a span 14 (256 behind 8192 keys, 256 each: 92 us of 32 tiles and 12, 80 of 43 beside 48).
template <unsigned kRowBlocks>
constexpr float kAttnSharedTile = kRowBlocks == 4 ? 1.5f : kRowBlocks == 2 ? 1.0f : 0.9f;
constexpr float kAttnSharedOwnTile = 1.5f, kAttnSharedOwnStart = 14.0f;
template <unsigned kRowBlocks>
__host__ __device__ constexpr float attn_shared_cost(const AttnSharedCut& c, float own, unsigned cus) {
  const float prefix = kAttnSharedTile<kRowBlocks> * static_cast<float>(c.span_tiles);
  const float keys = kAttnSharedOwnTile * own / static_cast<float>(c.both ? cus : cus - c.grid);
  return c.both ? prefix + kAttnSharedOwnStart + keys : prefix < keys ? keys : prefix;
}

// Row blocks of a workgroup of the prefix. More share a tile's way from memory, fewer make its time shorter
// and the workgroups more. 4 sequences: 11.4 us of one behind 4096 keys, 12.2 of two, 12.8 of four; 20.3, 19.8,
// 21.8 behind 32768. 8: 28.9, 22.9, 23.8 behind 32768. Above, two where the shortest spans fill half of the CUs
// at most: 64 behind 512 13.1 against 15.0 of four, 16 behind 4096 14.6 and 15.1; beyond that four: 32 behind 4096
// 16.9 against 18.8 of two, 12 behind 32768 27.4 and 33.3.
constexpr unsigned kAttnSharedFewTiles = 4;  // of a span, at least
__host__ __device__ constexpr unsigned attn_shared_row_blocks(unsigned batch, unsigned prefix,
                                                              unsigned cus) {
  constexpr std::size_t kSpan = 32 * kAttnSharedFewTiles;
  const std::size_t spans = (std::size_t{prefix} + kSpan - 1) / kSpan, pairs = 2 * ((std::size_t{batch} + 7) / 8);
  return batch <= 4 ? 1 : batch <= 8 || 2 * pairs * spans <= cus ? 2 : 4;
}

// The cut of `tiles` tiles for `pairs` (group of row blocks, KV head) pairs that costs least: beside the
// own keys on CUs of their own, `least` or more, or on all CUs. 8 sequences behind 32768 keys, 300 own
// keys each: 23.7 us of 9 tiles a span with 28 CUs for the own keys, 34.4 of 8 with all CUs and the
// own keys behind them; 256 behind 8192, 256 each: 79 of 43 with 64 CUs, 94 of 32.
// Spans shorter than 4 tiles only add partials: 8 behind 8192 22.0 us of 4, 24.1 of 3 (the merge's
// time among them).
template <unsigned kRowBlocks>
__host__ __device__ constexpr AttnSharedCut attn_shared_cut(unsigned tiles, unsigned pairs, float own,
                                                            unsigned cus, unsigned least) {
  if (tiles == 0)
    return AttnSharedCut{0, 0, 0, false};
  const auto cut = [=](unsigned spans, bool both) {
    const unsigned each = (tiles + spans - 1) / spans;
    spans = (tiles + each - 1) / each;
    return AttnSharedCut{spans, each, 8 * ((pairs * spans + 7) / 8), both};
  };
  unsigned most = cus / pairs;
  most = most < tiles / kAttnSharedFewTiles ? most : tiles / kAttnSharedFewTiles;
  most = most < 1 ? 1 : most;
  if (own == 0.0f || cut(most, false).grid > cus)
    return cut(most, false);
  AttnSharedCut best = cut(most, true);
  float cost = attn_shared_cost<kRowBlocks>(best, own, cus);
  // The spans with which both sides end together, and one more; no more than leave `least` CUs.
  const float prefix = kAttnSharedTile<kRowBlocks> * static_cast<float>(tiles);
  const float keys = kAttnSharedOwnTile * own;
  const unsigned even = static_cast<unsigned>(prefix * static_cast<float>(cus) /
                                              (keys + prefix * static_cast<float>(pairs)));
  const unsigned room = cus > least + 7 ? (cus - least) / 8 * 8 / pairs : 0;
  const unsigned top = room < most ? room : most;
  if (top == 0)
    return best;
  for (unsigned i = 0; i < 2; ++i) {
    const unsigned spans = even + i < top ? even + i : top;
    const AttnSharedCut c = cut(spans < 1 ? 1 : spans, false);
    if (c.grid + least > cus)
      continue;
    const float cost_c = attn_shared_cost<kRowBlocks>(c, own, cus);
    if (cost_c < cost) {
      cost = cost_c;
      best = c;
    }
  }
  return best;
}

// Sequences of up to kAttnSharedWaveKeys own keys, kAttnSharedWaveBatch or more of them, may be a wave's each
// (wave_items): longer ones would leave one wave to work when the others are done, fewer leave waves idle. Of up
// to 250 own keys behind 4096: 48 sequences 19.9 us with four waves an item, 20.3 with one; 64 26.3 and 22.3;
// 200 51.8 and 48.8. Of more keys, the call with four waves an item and with one: behind 4096 keys 130 of up to
// 500 48.6 and 50.4, 200 of up to 260 58.6 and 60.4, of up to 500 58.3 and 53.8, 400 of up to 400 124.8 and
// 88.1: beyond the limit one wave costs a little for some batches and saves much for the largest. One sequence
// above it sends the whole batch to four waves.
constexpr unsigned kAttnSharedWaveKeys = 256, kAttnSharedWaveBatch = 64;

namespace shared_detail {

using cdna4::float16_t;
using cdna4::half8_t;
using decode_detail::kGroup;
using weights_detail::mfma32;

constexpr unsigned kKeys = 32, kSteps = 16, kStages = 5;
constexpr unsigned kTileBytes = kKeys * attn::kDim * 2;    // K or V of a tile
constexpr unsigned kStageBytes = 2 * kTileBytes;           // K, then V
constexpr unsigned kBlockRows = 32;                        // of the matrix instruction's columns
constexpr unsigned kSeqs = kBlockRows / kGroup;            // sequences of a row block
constexpr float kNoScore = -3e38f;  // below every score, and finite: differences stay numbers
// Numerators are 2^(s - m) with m kLead below the first tile's maximum, and m follows when a lane's
// numerators of a tile sum to more than kMost: below f16's 65504, and the f16 pair of a numerator of 1
// relative to the row's largest keeps 2^-25 / 2^6 of it.
constexpr float kLead = 6.0f, kMost = 32768.0f;

struct alignas(1024) PrefixShared {
  unsigned char ring[kStages * kStageBytes];
};
static_assert(sizeof(PrefixShared) == 160 * 1024, "the CU's LDS");

// S += A B for the lo halves of the queries, which lie in AGPRs beside O (64 and 128 registers; the hi
// halves and the scores in VGPRs). These MFMAs and prefill_detail's are assembly, so that the compiler
// keeps each block where it is (with the builtins it spilled 66 registers around 1670 moves). Back-to-back
// accumulation into one register block chains in hardware. The compiler does not know their other wait
// states, also where it copies a block by itself: they stand at the start and the end of each step.
__device__ __attribute__((always_inline)) inline void score_lo(float16_t& s, const half8_t& a,
                                                               const half8_t& b) {
  asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(s) : "v"(a), "a"(b));
}

// o *= c element by element in the AGPRs, inside the caller's rare branch (attention_prefill.hpp's
// scale_acc for fewer blocks). The no-ops cover the last MFMA's result.
template <unsigned N>
__device__ __attribute__((always_inline)) inline void scale_values(float16_t (&o)[N], float c) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
  for (unsigned b = 0; b < N; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float x = o[b][r], tmp;
      asm volatile(
          "v_accvgpr_read_b32 %1, %0\n\t"
          "v_mul_f32 %1, %1, %2\n\t"
          "v_accvgpr_write_b32 %0, %1"
          : "+a"(x), "=&v"(tmp)
          : "v"(c));
      o[b][r] = x;
    }
}

// Rows 2 i and 2 i + 1 of the 8 at `row` to LDS (attention_decode.hpp's copy_tile, one instruction of it),
// the lane offset `off` less 1024 i: the instruction's offset counts on both sides. `lanes`: all, or none
// (a branch would part what the compiler places between the MFMAs).
template <unsigned kI>
__device__ __attribute__((always_inline)) inline void copy_rows_at(const attn::half_t* row,
                                                                   unsigned off, unsigned to,
                                                                   unsigned long long lanes) {
  unsigned m0;
  unsigned long long exec;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %4\n\t"
      "s_and_saveexec_b64 %1, %5\n\t"
      "global_load_lds_dwordx4 %2, %3 offset:%6\n\t"
      "s_mov_b64 exec, %1\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(m0), "=&s"(exec)
      : "v"(off), "s"(row), "s"(to), "s"(lanes), "n"(1024 * kI)
      : "memory", "scc");
}
__device__ __attribute__((always_inline)) inline void copy_rows(const attn::half_t* row, unsigned off,
                                                                unsigned to, unsigned i,
                                                                unsigned long long lanes) {
  if (i == 0)
    copy_rows_at<0>(row, off, to, lanes);
  else if (i == 1)
    copy_rows_at<1>(row, off, to, lanes);
  else if (i == 2)
    copy_rows_at<2>(row, off, to, lanes);
  else
    copy_rows_at<3>(row, off, to, lanes);
}

// Wait states behind the last MFMA of O, tied to its registers: what the compiler copies of them, it
// copies after these.
template <unsigned N>
__device__ __attribute__((always_inline)) inline void drain_values(float16_t (&o)[N]) {
  if constexpr (N == 2)
    asm volatile("s_nop 7\n\ts_nop 7" : "+a"(o[0]), "+a"(o[1]));
  else if constexpr (N == 4)
    asm volatile("s_nop 7\n\ts_nop 7" : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]));
  else
    asm volatile("s_nop 7\n\ts_nop 7"
                 : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]),
                   "+a"(o[6]), "+a"(o[7]));
}

// Wait states between the queries' way into their registers and the first MFMA that reads them.
__device__ __attribute__((always_inline)) inline void settle_operands(half8_t (&h)[kSteps],
                                                                      half8_t (&l)[kSteps]) {
  static_assert(kSteps == 16);
#pragma unroll
  for (unsigned i = 0; i < kSteps; i += 8) {
    asm volatile("s_nop 4"
                 : "+v"(h[i]), "+v"(h[i + 1]), "+v"(h[i + 2]), "+v"(h[i + 3]), "+v"(h[i + 4]),
                   "+v"(h[i + 5]), "+v"(h[i + 6]), "+v"(h[i + 7]));
    asm volatile("s_nop 4"
                 : "+a"(l[i]), "+a"(l[i + 1]), "+a"(l[i + 2]), "+a"(l[i + 3]), "+a"(l[i + 4]),
                   "+a"(l[i + 5]), "+a"(l[i + 6]), "+a"(l[i + 7]));
  }
}

// Two values as halves: hi rounded towards zero, lo what is left (2^-21 of the value, or 2^-25).
// Volatile: the compiler would move a tile's numerators below the MFMAs that they stand between. The
// no-op: they come from exponentials, whose results need a wait state.
__device__ __attribute__((always_inline)) inline void half_pair(float a, float b, unsigned& h,
                                                                unsigned& l) {
  float rest;
  asm volatile(
      "s_nop 0\n\t"
      "v_cvt_pkrtz_f16_f32 %0, %3, %4\n\t"
      "v_fma_mix_f32 %1, %0, -1.0, %3 op_sel_hi:[1,0,0]\n\t"
      "v_fma_mix_f32 %2, %0, -1.0, %4 op_sel:[1,0,0] op_sel_hi:[1,0,0]\n\t"
      "v_cvt_pk_f16_f32 %1, %1, %2"
      : "=&v"(h), "=&v"(l), "=&v"(rest)
      : "v"(a), "v"(b));
}

// Keys of the prefix that a sequence sees.
__device__ __attribute__((always_inline)) inline unsigned prefix_keys(const AttnSharedParams& p,
                                                                      unsigned seq) {
  if (seq >= p.batch)
    return 0;
  return p.whole ? min(p.lens[seq], p.prefix.len) : p.prefix.len;
}

// And its own, seq < batch.
__device__ __attribute__((always_inline)) inline unsigned own_keys(const AttnSharedParams& p,
                                                                   unsigned seq) {
  const unsigned len = p.lens[seq], skip = p.whole ? p.prefix.len : 0;
  return min(len > skip ? len - skip : 0u, p.own_cap);
}

}  // namespace shared_detail

// One workgroup per (span, KV head, group of kRowBlocks row blocks). kRowBlocks waves side by side
// hold 32 rows each: their queries as f16 pairs in 128 registers, a tile's scores S^T = K Q^T by 32
// MFMAs, each K operand read serving both halves; and each of the 4 / kRowBlocks waves of a row block
// adds P V for its share of the 256 dimensions (all 8 blocks of 32 dimensions: 32 MFMAs). So a wave's
// tile is 64, 48 or 40 MFMAs of 32 cycles for 4, 2 and 1 row blocks: with few rows the memory sets the
// pace (32 KiB a tile and CU), with many the matrix units. More rows a workgroup would read the tiles less
// often, but 32 rows a wave take 420 of its 512 registers (O 128, queries 128, scores and numerators 48).
//
// Softmax in one pass: per row a reference m (log2 units), the sum of numerators 2^(s - m), and O relative
// to 2^m; m starts kLead below the first tile's maximum and moves only when numerators grow too large.
// Tiles come through a ring of five stages, three under way; a step adds the scores of a tile while the
// numerators of the one before are formed between its MFMAs, then that one's P V.
//
// 64 sequences behind 131072 keys: 1.77 us a tile and CU, 1210 TFLOP/s of f16 products (an 8192^3 library
// product: 1076), 2860 cycles for 2048 of MFMAs at 1.62 GHz. There the power sets the pace: 2980 cycles, with
// the copies elsewhere, ran at 1.68 GHz. Behind 32768, beside own keys on 56 CUs, it holds 1.97 GHz: 1.48 us a
// tile. 8 behind 32768 keys: 23.3 us, 3.1 TB/s, 11 of them in the loop at 5.2
// TB/s, 5 before it (queries from memory and cut, three tiles on their way).
namespace shared_detail {
template <unsigned kRowBlocks, bool kPaged>
__device__ __attribute__((always_inline)) inline void prefix_span(const AttnSharedParams& p,
                                                                 PrefixShared& sh) {
  constexpr unsigned kParts = 4 / kRowBlocks;       // waves of a row block
  constexpr unsigned kDimBlocks = 8 / kParts;       // of 32 dimensions, per wave
  constexpr unsigned kStageRows = 32 / kParts;      // query rows that a wave lays out
  const unsigned lane = threadIdx.x & 63u, col = lane & 31u, hi = lane >> 5;
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups go to the XCDs round robin: neighbours of the list (span, KV head, row group), whose
  // row groups read the same tiles, on one XCD, so that its L2 serves them.
  const unsigned groups = (p.blocks + kRowBlocks - 1) / kRowBlocks;
  const unsigned place = blockIdx.x % 8 * (p.prefix_grid / 8) + blockIdx.x / 8;
  const unsigned combo = place / groups, group = place % groups;
  if (combo >= 2 * p.spans)
    return;
  const unsigned kvh = combo % 2, span = combo / 2;
  const unsigned t0 = span * p.span_tiles, last = p.prefix.len - 1;
  const unsigned t1 = min(t0 + p.span_tiles, last / kKeys + 1);
  const unsigned lds = cdna4::lds_offset(sh.ring);
  const unsigned local = wave / kParts, part = wave % kParts;
  const unsigned block = group * kRowBlocks + local;  // this wave's row block
  const bool active = block < p.blocks;               // wave-uniform

  // ---- Tiles: this wave copies rows 8 wave .. + 7 of K and V (instruction i rows 2 i + lane / 32 of
  // them, chunks swizzled as attention_prefill.hpp's tiles). Rows past the prefix's last one repeat it
  // (they are masked at use): the last tile's, so that its offsets can take the place of the others'. The
  // lane offsets are unsigned, and a repeated row lies up to 3 KiB below its instruction's: offsets
  // are that much larger, their base that much lower.
  constexpr unsigned kBelow = 3 * 1024;
  unsigned koff[4], voff[4];
#pragma unroll
  for (unsigned i = 0; i < 4; ++i) {
    const unsigned r = 2 * i + (lane >> 5);
    koff[i] = kBelow + 512 * r + 16 * prefill_detail::swz_k(8 * wave + r, lane & 31u) - 1024 * i;
    voff[i] = kBelow + 512 * r + 16 * prefill_detail::swz_v(8 * wave + r, lane & 31u) - 1024 * i;
  }
  int pages = 0;  // lane i: the page of this wave's rows of tile page0 + i
  unsigned page0 = t0 - 64;
  struct Place {
    const attn::half_t* k;
    const attn::half_t* v;
  };
  auto place_of = [&](unsigned ti) __attribute__((always_inline)) {
    const unsigned want = ti * kKeys + 8 * wave, row = want < last ? want : last;
    if (last - row < 7) {  // uniform
#pragma unroll
      for (unsigned i = 0; i < 4; ++i) {
        const unsigned r = 2 * i + (lane >> 5), past = r > last - row ? r - (last - row) : 0u;
        koff[i] -= 512 * past;
        voff[i] -= 512 * past;
      }
    }
    std::size_t at;  // of the row, in halves
    if constexpr (kPaged) {
      if (ti - page0 >= 64u) {  // uniform
        page0 = ti;
        const unsigned r = (ti + lane) * kKeys + 8 * wave;
        pages = p.prefix.table[(r < last ? r : last) >> p.prefix.log2_page];
        // Here and not where the paths meet: there it would wait for the copies under way in every step.
        __builtin_amdgcn_s_waitcnt(weights_detail::kVmcnt0);
      }
      const unsigned page = decode_detail::lane_value(static_cast<unsigned>(pages), ti - page0);
      at = (((std::size_t{page} * attn::kKvHeads + kvh) << p.prefix.log2_page) +
            (row & ((1u << p.prefix.log2_page) - 1u))) * attn::kDim;
    } else {
      at = (std::size_t{kvh} * p.prefix.ctx + row) * attn::kDim;
    }
    const std::size_t base = 2 * at - kBelow;  // in bytes
    return Place{decode_detail::uniform(reinterpret_cast<const attn::half_t*>(
                     reinterpret_cast<std::uintptr_t>(p.prefix.k) + base)),
                 decode_detail::uniform(reinterpret_cast<const attn::half_t*>(
                     reinterpret_cast<std::uintptr_t>(p.prefix.v) + base))};
  };
  // Copy j < 8 of a tile to its stage: two rows of K, then of V.
  auto copy = [&](const Place& from, unsigned to, unsigned j, unsigned long long lanes = ~0ull)
      __attribute__((always_inline)) {
    if (j < 4)
      copy_rows(from.k, koff[j], to + 4096 * wave, j, lanes);
    else
      copy_rows(from.v, voff[j - 4], to + 4096 * wave + kTileBytes, j - 4, lanes);
  };
  // Stages are named by their offset in the ring; tile t0 takes the last one.
  auto issue = [&](unsigned ti, unsigned to) __attribute__((always_inline)) {
    const Place from = place_of(ti);
#pragma unroll
    for (unsigned j = 0; j < 8; ++j)
      copy(from, lds + to, j);
  };
  // ---- Queries: row r of a block is sequence 4 block + r / 8, head 8 kvh + r % 8. The waves of a block
  // copy its rows to LDS (1 KiB each, 16-byte chunk c of row r at c ^ (r % 16)) and every lane reads the
  // 128 dimensions of its row that its B operands hold. Times log2(e) and a power of two of the row's own
  // (its largest element near 2^13) they are cut into f16 halves hi + lo (2^-21 of an element, 2^-38 of
  // the row's largest).
  // They pass through the stages that the first tiles leave: with four row blocks all but the first's.
  const unsigned area = lds + 32768 * (4 - kRowBlocks + local);
  constexpr unsigned kEarly = kRowBlocks == 4 ? 1 : 3;  // tiles under way meanwhile
#pragma unroll
  for (unsigned i = 0; i < kStageRows; ++i) {
    const unsigned r = kStageRows * part + i, seq = min(kSeqs * block + r / kGroup, p.batch - 1);
    cdna4::lds_load16(p.q + (std::size_t{seq} * attn::kQHeads + kvh * kGroup + r % kGroup) *
                                attn::kDim + 4 * (lane ^ (r & 15u)),
                      area + 1024 * r);
  }
  // Tile t0 takes the last stage, the next ones those from the first on.
  issue(t0, (kStages - 1) * kStageBytes);
  if (kEarly > 1 && t0 + 1 < t1)
    issue(t0 + 1, 0);
  if (kEarly > 2 && t0 + 2 < t1)
    issue(t0 + 2, kStageBytes);
  if (kEarly > 2 && t0 + 2 < t1)
    cdna4::wait_vmcnt<24>();
  else if (kEarly > 1 && t0 + 1 < t1)
    cdna4::wait_vmcnt<16>();
  else
    cdna4::wait_vmcnt<8>();
  decode_detail::tile_barrier();
  half8_t qh[kSteps], ql[kSteps];
  float scale;  // of the scores of this lane's row
  {
    const unsigned at = area + 1024 * col + 16 * ((2 * hi) ^ (col & 15u));
    cdna4::float4_t v[2 * kSteps];
#pragma unroll
    for (unsigned c = 0; c < 2 * kSteps; ++c)
      v[c] = *reinterpret_cast<const __attribute__((address_space(3))) cdna4::float4_t*>(
          at ^ (64u * (c / 2) + 16u * (c % 2)));
    float top = 0.0f;
#pragma unroll
    for (unsigned c = 0; c < 2 * kSteps; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        top = fmaxf(top, __builtin_fabsf(v[c][j]));
    top = cdna4::max_xor32(top);
    int e = 13 - (static_cast<int>(cdna4::as_uint(top) >> 23) - 127);
    e = top == 0.0f || !(top < __builtin_inff()) ? 0 : (e < 100 ? e : 100);
    const float up = __builtin_ldexpf(decode_detail::kLog2e, e);
    scale = __builtin_ldexpf(1.0f / 16.0f, -e);
#pragma unroll
    for (unsigned k = 0; k < kSteps; ++k) {
      struct alignas(16) Halves {
        unsigned w[4];
      } h, l;
#pragma unroll
      for (unsigned j = 0; j < 4; ++j)
        half_pair(v[2 * k + j / 2][2 * (j % 2)] * up, v[2 * k + j / 2][2 * (j % 2) + 1] * up, h.w[j],
                  l.w[j]);
      qh[k] = __builtin_bit_cast(half8_t, h);
      ql[k] = __builtin_bit_cast(half8_t, l);
    }
  }
  if constexpr (kEarly == 1) {
    decode_detail::tile_barrier();  // every wave has its operands: the ring takes the space
#pragma unroll
    for (unsigned i = 1; i < 3; ++i)
      if (t0 + i < t1)
        issue(t0 + i, (i - 1) * kStageBytes);
  }

  // ---- Keys this lane's row sees, and whether every row of the wave sees the whole span.
  const unsigned seq = kSeqs * block + col / kGroup;
  const unsigned sees = prefix_keys(p, seq);
  const bool full = __builtin_amdgcn_ballot_w64(seq < p.batch && sees < t1 * kKeys) == 0;

  // And those that some row of the workgroup sees, with the first tile of the span that has others (~0: none
  // has; only in the paged form an entry may see less than the prefix).
  unsigned seen = 0, unseen_from = ~0u;
  if constexpr (kPaged) {
    const unsigned mine = prefix_keys(p, kSeqs * kRowBlocks * group + lane % (kSeqs * kRowBlocks));
    if (__builtin_amdgcn_ballot_w64(mine >= min(t1 * kKeys, p.prefix.len)) == 0) {  // rare
#pragma unroll
      for (unsigned i = 0; i < kSeqs * kRowBlocks; ++i)
        seen = max(seen, decode_detail::lane_value(mine, i));
      unseen_from = seen / kKeys;
    }
  }

  // ---- Operand addresses of a stage (attention_prefill.hpp: the same tiles and swizzles).
  const unsigned kb = col * 512 + 16 * (hi ^ (col & 15u));
  unsigned vb[4];
  {
    const unsigned g = lane >> 4, j = lane & 15u;
    const unsigned vrow = 4 * (g >> 1) + j / 4, vchunk = 2 * (g & 1u) + (j % 4) / 2;
    const unsigned base = vrow * 512 + 8 * (j & 1u) + 16 * prefill_detail::swz_v(vrow, vchunk);
#pragma unroll
    for (unsigned c = 0; c < 4; ++c)
      vb[c] = base ^ (64u * c);
  }

  float16_t o[kDimBlocks];
#pragma unroll
  for (unsigned b = 0; b < kDimBlocks; ++b)
    o[b] = float16_t{};
  float m = kNoScore, l = 0.0f;
  float16_t cur;  // the scores of a tile under way
  float x[16];    // those of the tile before
  float w[16];    // its numerators
  half8_t a[4];   // the K operands of the next four k-steps
  half8_t va[4];  // the V operands of the next four products
  unsigned ka[8];  // where the current tile's K operands k and k + 8 (256 bytes on) lie
  // Stages: of the tile before the current one, the current, the next; of the copy under way.
  unsigned before = 0, here = lds + (kStages - 1) * kStageBytes, after = lds,
           spare = lds + 2 * kStageBytes;
  auto rotate = [&]() __attribute__((always_inline)) {
    before = here;
    here = after;
    after = after == lds + (kStages - 1) * kStageBytes ? lds : after + kStageBytes;
    spare = spare == lds + (kStages - 1) * kStageBytes ? lds : spare + kStageBytes;
  };
  // Tile ti has landed in stage `base`: this wave's copies by the count (two tiles more are under way), every
  // wave's by the barrier, which also says that every wave has read tile ti - 2, whose stage the next copy
  // takes. Rows of V that none of the workgroup's rows sees are cleared before: their numerators are 0, but
  // they may hold NaN or infinity.
  auto turn = [&](unsigned ti, unsigned base) __attribute__((always_inline)) {
    const unsigned behind = t1 - 1 - ti;
    if (behind >= 2)
      cdna4::wait_vmcnt<16>();
    else if (behind == 1)
      cdna4::wait_vmcnt<8>();
    else
      cdna4::wait_vmcnt<0>();
    if (kPaged && __builtin_expect(ti >= unseen_from, 0)) {
#pragma unroll 1
      for (unsigned r = 8 * wave + (lane >> 5); r < 8 * wave + 8; r += 2)
        if (ti * kKeys + r >= seen)
          *reinterpret_cast<__attribute__((address_space(3))) cdna4::float4_t*>(
              base + kTileBytes + 512 * r + 16 * (lane & 31u)) = cdna4::float4_t{};
    }
    decode_detail::tile_barrier();
  };
  auto first_operands = [&](unsigned base) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned k = 0; k < 8; ++k)
      ka[k] = (base + kb) ^ (32u * k);
#pragma unroll
    for (unsigned k = 0; k < 4; ++k)
      a[k] = decode_detail::lds_b128(ka[k]);
  };
  // Two score MFMAs of k-step k, and the operand four steps on.
  auto score_hi = [&](unsigned k) __attribute__((always_inline)) {
    if (k == 0)
      prefill_detail::s_mfma_first(cur, a[0], qh[0]);
    else
      prefill_detail::s_mfma(cur, a[k % 4], qh[k]);
  };
  auto operand = [&](unsigned k) __attribute__((always_inline)) {
    return k + 4 < kSteps ? decode_detail::lds_b128(ka[(k + 4) % 8] + 256u * ((k + 4) / 8))
                          : a[k % 4];
  };
  auto mask = [&](unsigned ti) __attribute__((always_inline)) {
    if (full)  // uniform
      return;
#pragma unroll
    for (unsigned i = 0; i < 16; ++i)
      x[i] = ti * kKeys + weights_detail::tile_row(lane, i) < sees ? x[i] : -__builtin_inff();
  };
  unsigned ph[8], pl[8];  // pairs of numerators, hi and lo halves
  auto pair = [&](unsigned i) __attribute__((always_inline)) {
    half_pair(w[i], w[i + 1], ph[i / 2], pl[i / 2]);
  };
  // The reference for scores x.
  auto reference = [&]() __attribute__((always_inline)) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i)
      top = fmaxf(top, x[i]);
    return fmaxf(m, cdna4::max_xor32(top) * scale - kLead);
  };
  // After a tile's numerators w (their sum given): the reference follows where they are too large.
  auto settle = [&](float sum) __attribute__((always_inline)) {
    if (__builtin_amdgcn_ballot_w64(sum > kMost) != 0) {  // rare
      const float top = reference();
      const float corr = __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= corr;
      scale_values(o, corr);
      sum = 0.0f;
#pragma unroll
      for (unsigned i = 0; i < 16; ++i) {
        w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], scale, -m));
        sum += w[i];
      }
#pragma unroll
      for (unsigned i = 0; i < 8; i += 2)
        pair(i);
    }
    l += sum;
  };
  // V operand i of the tile in stage `base`: key step i / kDimBlocks, dimension block part kDimBlocks + d
  // of 8: 64 bytes (block % 4) by the XOR, 256 (block / 4) further.
  auto values = [&](unsigned base, unsigned i) __attribute__((always_inline)) {
    const unsigned step = i / kDimBlocks, d = i % kDimBlocks;
    const unsigned upper = kParts == 4 ? part >> 1 : kParts == 2 ? part : d / 4;
    const unsigned v = kParts == 4 ? vb[0] ^ (64u * (d + 2 * (part & 1u))) : vb[d % 4];
    const unsigned at = base + kTileBytes + v + 256u * upper + 8192u * step;
    const cdna4::half4_t lo = prefill_detail::read_tr(at);
    const cdna4::half4_t up = prefill_detail::read_tr(upper ? at + 4096u - 256u
                                                            : at + 4096u + 256u);
    return half8_t{lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
  };
  constexpr unsigned kValues = 2 * kDimBlocks;
  static_assert(kValues >= 4);
  auto halves = [&](const unsigned (&h)[8], unsigned step) __attribute__((always_inline)) {
    return __builtin_bit_cast(half8_t, cdna4::u32x4_t{h[4 * step], h[4 * step + 1],
                                                      h[4 * step + 2], h[4 * step + 3]});
  };
  // O += P V of the tile in stage `base`, two MFMAs an operand, numerators 0 .. 7 in pairs already and
  // the others made beside the first half; `beside(i)` goes between the two MFMAs of operand i.
  auto add_values = [&](unsigned base, auto beside) __attribute__((always_inline)) {
    half8_t bh, bl;
#pragma unroll
    for (unsigned i = 0; i < kValues; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      const unsigned step = i / kDimBlocks, d = i % kDimBlocks;
      if (i % kDimBlocks == 0) {
        bh = halves(ph, step);
        bl = halves(pl, step);
        asm volatile("s_nop 4" : "+v"(bh), "+v"(bl));  // VALU to MFMA
      }
      half8_t next = va[i % 4];
      if (i + 4 < kValues)
        next = values(base, i + 4);
      prefill_detail::pv_mfma(o[d], va[i % 4], bh);
      __builtin_amdgcn_sched_barrier(0);
      if (step == 0)
#pragma unroll
        for (unsigned j = 8 + 8 * d / kDimBlocks / 2 * 2; j < 8 + 8 * (d + 1) / kDimBlocks / 2 * 2;
             j += 2)
          pair(j);
      beside(i);
      prefill_detail::pv_mfma(o[d], va[i % 4], bl);
      va[i % 4] = next;
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  turn(t0, here);
  if (t0 + 3 < t1)
    issue(t0 + 3, 2 * kStageBytes);
  if (!active) {
    for (unsigned ti = t0 + 1; ti < t1; ++ti) {
      rotate();
      turn(ti, here);
      if (ti + 3 < t1)
        issue(ti + 3, spare - lds);
    }
    return;
  }
  first_operands(here);
  settle_operands(qh, ql);
#pragma unroll
  for (unsigned k = 0; k < kSteps; ++k) {
    const half8_t next = operand(k);
    score_hi(k);
    score_lo(cur, a[k % 4], ql[k]);
    a[k % 4] = next;
  }
  prefill_detail::drain_scores(cur);
#pragma unroll
  for (unsigned i = 0; i < 16; ++i)
    x[i] = cur[i];
  mask(t0);
  m = reference();

  // Step ti: the scores of tile ti into cur, beside them the numerators of tile ti - 1 (x), then its
  // P V; tile ti + 3 is copied meanwhile. Between two score MFMAs stand an fma, an exponential and a sum
  // of different numerators, so that none waits for another, and the last ones are done before the last
  // MFMAs; between those of P V the other half's pairs, the moves of cur to x, and behind the last V
  // operand the barrier and the next tile's first operands.
  if (t0 + 1 < t1) {
    turn(t0 + 1, after);
    first_operands(after);
    for (unsigned ti = t0 + 1;;) {
      rotate();
      mask(ti - 1);
      Place from{};
      const bool more = ti + 3 < t1, next_tile = ti + 1 < t1;  // uniform
      unsigned long long lanes;  // more ? ~0 : 0 (as C++ the compiler takes it through VGPRs)
      asm("s_cmp_lt_u32 %1, %2\n\ts_cselect_b64 %0, -1, 0" : "=s"(lanes) : "s"(ti + 3), "s"(t1) : "scc");
      float sum[2] = {0.0f, 0.0f}, e[16];
      // Numerators of k-step k: 16 in 13 steps.
      constexpr auto at = [](unsigned k) { return k >= 13 ? 16u : (16 * k + 12) / 13; };
#pragma unroll
      for (unsigned k = 0; k < kSteps; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        const half8_t next = operand(k);
        score_hi(k);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (unsigned i = at(k); i < at(k + 1); ++i)
          e[i] = __builtin_fmaf(x[i], scale, -m);
        if (k > 0)
#pragma unroll
          for (unsigned i = at(k - 1); i < at(k); ++i)
            w[i] = __builtin_amdgcn_exp2f(e[i]);
        if (k % 2 == 1)
          copy(from, spare, k / 2, lanes);
        score_lo(cur, a[k % 4], ql[k]);
        if (k > 1)
#pragma unroll
          for (unsigned i = at(k - 2); i < at(k - 1); ++i)
            sum[i % 2] += w[i];
        if (k >= 9 && k < 13)
          pair(2 * (k - 9));
        a[k % 4] = next;
        if (k == 0 && more)
          from = place_of(ti + 3);
        if (k >= kSteps - 4)
          va[k + 4 - kSteps] = values(before, k + 4 - kSteps);
      }
      __builtin_amdgcn_sched_barrier(0);
      settle(sum[0] + sum[1]);
      add_values(before, [&](unsigned i) __attribute__((always_inline)) {
        // The next tile's scores, done since the first MFMA of P V.
        if (i != 0)
#pragma unroll
          for (unsigned j = (i - 1) * 16 / (kValues - 1); j < i * 16 / (kValues - 1); ++j) {
            x[j] = cur[j];
            asm volatile("" : "+v"(x[j]));
          }
        if (i == kValues - 3 && next_tile) {  // the V operands are here
          turn(ti + 1, after);
          first_operands(after);
        }
      });
      if (++ti >= t1) {
        drain_values(o);
        break;
      }
    }
  }
  {  // the last tile
    mask(t1 - 1);
    float sum = 0.0f;
#pragma unroll
    for (unsigned i = 0; i < 16; ++i) {
      w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], scale, -m));
      sum += w[i];
    }
#pragma unroll
    for (unsigned i = 0; i < 8; i += 2)
      pair(i);
    settle(sum);
#pragma unroll
    for (unsigned i = 0; i < 4; ++i)
      va[i] = values(here, i);
    add_values(here, [](unsigned) {});
    drain_values(o);
  }
  // ---- The partial, relative to 2^m, in the accumulators' order (whole 1 KiB a store).
  const std::size_t at = (std::size_t{span} * attn::kKvHeads + kvh) * p.blocks + block;
  float4* out = p.part_o + (at * 8 + part * kDimBlocks) * 256 + lane;
#pragma unroll
  for (unsigned b = 0; b < kDimBlocks; ++b)
#pragma unroll
    for (unsigned i = 0; i < 4; ++i)
      out[256 * b + 64 * i] = float4{o[b][4 * i], o[b][4 * i + 1], o[b][4 * i + 2], o[b][4 * i + 3]};
  const float all = cdna4::sum_xor32(l);
  if (part == 0 && hi == 0)
    p.part_ml[at * kBlockRows + col] = float2{m, all};
}
}  // namespace shared_detail

// ------------------------------------------------------------------------------------------------
// Own keys: the streaming split of the ragged and paged decode over what lies behind the prefix.
// ------------------------------------------------------------------------------------------------

namespace decode_detail {

// Pages behind the prefix: sequence s's own keys are in table row rows[s] (row s without rows), their
// number is lens[s] less the prefix's.
struct SharedPagedSource {
  static constexpr float kUnit = 1.0f;  // maxima stay in log2 units, as the prefix's references
  PagedStreamSource base;
  const int32_t* rows;
  unsigned prefix_len, table_row = 0;  // lane j: item j's row
  __device__ __attribute__((always_inline)) void describe(unsigned seq, unsigned, unsigned) {
    table_row = rows != nullptr ? static_cast<unsigned>(rows[seq]) : seq;
  }
  __device__ __attribute__((always_inline)) void prepare(unsigned, unsigned kvh, unsigned k0,
                                                         unsigned last_row, unsigned j) {
    base.prepare(lane_value(table_row, j), kvh, k0, last_row, j);
  }
  template <bool kV>
  __device__ __attribute__((always_inline)) void issue(unsigned j, unsigned k0, unsigned last_row,
                                                       unsigned lds, const WaveCopy& cp,
                                                       unsigned lane) const {
    base.template issue<kV>(j, k0, last_row, lds, cp, lane);
  }
};
// Contiguous own keys: the ragged decode's. (A type of its own: its launch's workgroups start elsewhere.)
struct SharedRaggedSource : RaggedStreamSource {
  static constexpr float kUnit = 1.0f;
};
__device__ __attribute__((always_inline)) inline unsigned stream_length(
    const SharedPagedSource& src, const StreamBatch& p, unsigned s) {
  const unsigned len = p.lens[s], mine = len > src.prefix_len ? len - src.prefix_len : 0;
  return mine < p.len_cap ? mine : p.len_cap;
}

// The streaming split where every sequence has few keys: an item (sequence, KV head) is one wave's, its
// tiles one after the other, since four waves on it would each take a tile or none and wait for one another:
// 6 us a round of four tiles, here 3.6 a tile of each wave. 490 sequences of at most 5 keys behind 2560 (the
// whole split): 68 us with four waves an item, 54 here; 300 of at most 60 behind 2048: 43 and 34; 203 of 1 ..
// 203 behind 12000: 90 either way. Each wave for itself: item j of wave w is w + j times the launch's waves; a
// K and a V tile and the queries of an item in LDS, the next tile's copies issued as soon as the operands of the
// one before are in registers. Partials as the streaming split's, of one span.
template <class Src>
__device__ __attribute__((always_inline)) inline void wave_items(const StreamBatch& p, Src& src,
                                                                StreamShared& sh, unsigned first) {
  using cdna4::half8_t;
  const unsigned t = threadIdx.x, lane = t & 63u;
  const unsigned wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const unsigned stride = 4 * (gridDim.x - first), w = 4 * (blockIdx.x - first) + wave;
  if (p.balanced != nullptr && w == 0 && lane == 0)
    *p.balanced = p.chunk;
  const unsigned all = attn::kKvHeads * p.batch, n_items = w < all ? (all - w + stride - 1) / stride : 0;
  unsigned it_len = 0, it_seq = 0, it_kvh = 0;  // lane j: item j
  if (lane < n_items) {
    const unsigned k = w + lane * stride;
    it_seq = k / attn::kKvHeads;
    it_kvh = k % attn::kKvHeads;
    it_len = stream_length(src, p, it_seq);
    src.describe(it_seq, it_kvh, it_len);
  }
  auto next_item = [&](unsigned j) __attribute__((always_inline)) {  // first with keys >= j
    while (j < n_items && lane_value(it_len, j) == 0)
      ++j;
    return j;
  };
  // The waits count as in stream_items.
  unsigned issued = 0;
  const unsigned k_lds = cdna4::lds_offset(sh.k[wave]), v_lds = cdna4::lds_offset(sh.v[wave]);
  // The queries' 8 KiB a wave take the place of sh.q and, behind it, sh.merge.
  static_assert(offsetof(StreamShared, merge) == offsetof(StreamShared, q) + sizeof(sh.q) &&
                sizeof(sh.q) + sizeof(sh.merge) == 4 * sizeof(sh.q[0]));
  float(*const q)[attn::kDim] = reinterpret_cast<float(*)[attn::kDim]>(
      reinterpret_cast<unsigned char*>(&sh) + offsetof(StreamShared, q) + sizeof(sh.q[0]) * wave);
  const unsigned q_lds = cdna4::lds_offset(q);
  const WaveCopy cp = wave_copy_offsets(lane);
  auto prepare = [&](unsigned j, unsigned ti) __attribute__((always_inline)) {
    src.prepare(lane_value(it_seq, j), lane_value(it_kvh, j), ti * kTileKeys,
                lane_value(it_len, j) - 1, j);
  };
  auto issue_k = [&](unsigned j, unsigned ti) __attribute__((always_inline)) {
    src.template issue<false>(j, ti * kTileKeys, lane_value(it_len, j) - 1, k_lds, cp, lane);
    issued += 16;
  };
  auto issue_v = [&](unsigned j, unsigned ti) __attribute__((always_inline)) {
    src.template issue<true>(j, ti * kTileKeys, lane_value(it_len, j) - 1, v_lds, cp, lane);
    issued += 16;
  };
  auto issue_q = [&](unsigned j) __attribute__((always_inline)) {
    const float* from = p.q + (std::size_t{lane_value(it_seq, j)} * attn::kQHeads +
                               lane_value(it_kvh, j) * kGroup) * attn::kDim;
#pragma unroll
    for (unsigned h = 0; h < kGroup; ++h)
      cdna4::lds_load16(from + h * attn::kDim + 4 * lane, q_lds + h * attn::kDim * 4);
    issued += kGroup;
  };
  unsigned jc = next_item(0);
  if (jc >= n_items)  // uniform
    return;
  issue_q(jc);
  unsigned mark_q = issued;
  prepare(jc, 0);
  issue_k(jc, 0);
  unsigned mark_k = issued;
  issue_v(jc, 0);
  unsigned mark_v = issued;
  const TileLane tln = tile_lane(lane);
  const WaveOperands op = wave_operands(lane);
  WaveTileState st;
  for (;;) {
    wait_vm_at_most(issued - mark_q);
    wave_start(st, q, lane, tln);
    const unsigned jn = next_item(jc + 1), end = lane_value(it_len, jc);
    if (jn < n_items) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the queries are in registers
      issue_q(jn);
      mark_q = issued;
    }
    for (unsigned k0 = 0; k0 < end; k0 += kTileKeys) {
      const unsigned mk = mark_k, mv = mark_v;
      const bool last = k0 + kTileKeys >= end, next = !last || jn < n_items;
      const unsigned nj = last ? jn : jc, nt = last ? 0 : k0 / kTileKeys + 1;
      if (next)
        prepare(nj, nt);
      wait_vm_at_most(issued - mk);
      half8_t ka[2][8];
      read_k(ka, k_lds + op.kl);
      __builtin_amdgcn_sched_barrier(0);
      f32x4 s[2];
      wave_scores(s, ka, st);
      if (next) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the K operands are in registers
        issue_k(nj, nt);
        mark_k = issued;
      }
      wait_vm_at_most(issued - mv);
      half8_t va[16];
      read_v_all(va, v_lds, op.vl);
      __builtin_amdgcn_sched_barrier(0);
      TileSoftmax sm;
      wave_softmax(sm, st, s, k0, end, k0 == 0, lane, tln);
      if (next) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the V operands are in registers
        issue_v(nj, nt);
        mark_v = issued;
      }
      wave_pv(st, sm, va);
    }
    WaveResult r;
    wave_result(r, st, true);
    const unsigned g = lane >> 4, c = lane & 15u;
    if (c < kGroup) {  // lane (g, c): head c, dimensions 4 (4 b + g) ..
      const std::size_t row =
          (std::size_t{lane_value(it_seq, jc)} * attn::kKvHeads + lane_value(it_kvh, jc)) * p.s_max *
              kGroup + c;
#pragma unroll
      for (unsigned b = 0; b < 16; ++b)
        *reinterpret_cast<float4*>(p.part_o + row * attn::kDim + 4 * (4 * b + g)) =
            float4{r.o[b][0], r.o[b][1], r.o[b][2], r.o[b][3]};
      if (g == 0) {
        p.part_m[row] = r.mt * kStreamUnit<Src>;
        p.part_l[row] = r.l;
      }
    }
    issued += 8;  // stores, at least
    jc = jn;
    if (jc >= n_items)
      break;
  }
}

}  // namespace decode_detail

// Where the own keys lie: pages, or contiguous as the ragged decode's (page_table nullptr).
struct AttnSharedOwn {
  const attn::half_t* k;
  const attn::half_t* v;
  const int32_t* page_table;  // [..][max_pages], from the first entry behind the prefix
  const int32_t* rows;        // [batch] table rows, or nullptr: 0 .. batch - 1
  unsigned max_pages, log2_page;
  const uint64_t* kv_offsets;
};

// The cut for `own` tiles of own keys (AttnSharedCut), in the launch's own workgroups.
template <unsigned kRowBlocks>
__device__ __attribute__((always_inline)) inline void choose_cut(AttnSharedParams& p, float own) {
  const AttnSharedCut cut = attn_shared_cut<kRowBlocks>(
      (p.prefix.len - 1) / 32 + 1, 2 * ((p.blocks + kRowBlocks - 1) / kRowBlocks), own, gridDim.x,
      p.own_least);
  p.spans = __builtin_amdgcn_readfirstlane(cut.spans);
  p.span_tiles = __builtin_amdgcn_readfirstlane(cut.span_tiles);
  p.prefix_grid = __builtin_amdgcn_readfirstlane(cut.grid);
  p.own_first = __builtin_amdgcn_readfirstlane(cut.both ? 0u : cut.grid);
  if (blockIdx.x == 0 && threadIdx.x == 0)
    *p.chosen = p.spans;
}

// The first p.prefix_grid workgroups take the prefix's spans, those from p.own_first on the sequences' own
// keys: one launch, side by side (3 sequences behind 512 keys 10.5 us, in two launches 17). Where the
// lengths decide on how many CUs either does best, which only the device knows, each wave makes the choice
// before anything else, 1.1 us.
template <unsigned kRowBlocks, bool kPaged>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))
attn_shared_split_kernel(AttnSharedParams p, AttnSharedOwn own) {
  __shared__ decode_detail::StreamShared sh;
  static_assert(sizeof(sh) >= sizeof(shared_detail::PrefixShared));
  bool waves = false;  // uniform
  if (p.chosen != nullptr || p.own_waves) {
    float fours = 0.0f, ones = 0.0f;
    unsigned most = 0;
    for (unsigned s = threadIdx.x & 63u; s < p.batch; s += 64) {
      const unsigned n = shared_detail::own_keys(p, s);
      fours += attn_shared_own_tiles(n, false);
      ones += attn_shared_own_tiles(n, true);
      most = max(most, n);
    }
    waves = p.own_waves && __builtin_amdgcn_ballot_w64(most > kAttnSharedWaveKeys) == 0;
    ones = cdna4::wave_allsum(waves ? ones : fours);
    if (p.chosen != nullptr)
      choose_cut<kRowBlocks>(p, ones);
  }
  if (blockIdx.x < p.prefix_grid) {  // uniform
    shared_detail::prefix_span<kRowBlocks, kPaged>(
        p, reinterpret_cast<shared_detail::PrefixShared&>(sh));
    if (blockIdx.x < p.own_first || p.s_max == 0)
      return;
    __syncthreads();  // the ring's space is the stream's
  }
  waves = waves && p.own_batch >= gridDim.x - p.own_first;  // two items a workgroup
  const decode_detail::StreamBatch batch{p.q,     p.own_m, p.own_l,   p.own_o, p.lens,
                                         p.own_batch, p.s_max, p.own_cap, p.chunk, p.balanced};
  if constexpr (kPaged) {
    decode_detail::SharedPagedSource src{
        {own.k, own.v, own.page_table, own.max_pages, own.log2_page}, own.rows, p.prefix.len};
    if (waves)
      decode_detail::wave_items(batch, src, sh, p.own_first);
    else
      decode_detail::stream_items(batch, src, sh, p.own_first);
  } else {
    decode_detail::SharedRaggedSource src{{own.k, own.v, own.kv_offsets}};
    if (waves)
      decode_detail::wave_items(batch, src, sh, p.own_first);
    else
      decode_detail::stream_items(batch, src, sh, p.own_first);
  }
}

// ------------------------------------------------------------------------------------------------
// Merge: a workgroup per (KV head, row block, 8 kQuads dimensions). Its waves take the prefix's spans in
// turn, each lane the row of its column as the partials lie (M the largest reference, O and L summed
// relative to 2^M in span order), and meet in LDS; then a thread per (row, 4 dimensions) adds the
// waves' sums and the own keys' splits in order, divides and applies the gate. The order is fixed.
// Bound by the partials it reads, 1 KiB a row and span; a CU takes in only so much of them, so with
// few row blocks their dimensions are spread over four times the workgroups (8 sequences, 114 spans: 6.6 us;
// 12 with 32 dimensions a workgroup), and where that leaves CUs, over twice the waves (6.0; with 33
// sequences and 20 spans 7.7 against 5.9). 3 sequences, 4 spans: 3.9 us, 64 and 26: 8.4, 256 and 6: 9.0.
// ------------------------------------------------------------------------------------------------

template <unsigned kQuads, unsigned kWaves>
__global__ void __launch_bounds__(64 * kWaves) attn_shared_merge_kernel(AttnSharedParams p) {
  using namespace shared_detail;
  static_assert(kQuads == 1 || kQuads == 4);
  constexpr unsigned kBatch = 16 / kQuads, kDims = 8 * kQuads;  // spans, dimensions at a time
  constexpr unsigned kRow = kDims + 1;  // floats of a staged row
  constexpr unsigned kPieces = attn::kDim / kDims;
  __shared__ float rows[kWaves][kBlockRows * kRow];
  __shared__ float2 ml[kWaves][kBlockRows];
  const unsigned t = threadIdx.x, lane = t & 63u, wave = t >> 6, col = lane & 31u, hi = lane >> 5;
  const unsigned d = blockIdx.x % kPieces, kvh = blockIdx.x / kPieces % 2;
  const unsigned block = blockIdx.x / (2 * kPieces);
  // This wave's spans of the prefix.
  const unsigned spans = p.chosen != nullptr ? *p.chosen : p.spans;
  float m = kNoScore, l = 0.0f;
  float4 o[kQuads] = {};
  for (unsigned s0 = wave; s0 < spans; s0 += kWaves * kBatch) {
    float2 x[kBatch];
    float4 y[kBatch][kQuads];
#pragma unroll
    for (unsigned i = 0; i < kBatch; ++i) {
      const unsigned s = min(s0 + kWaves * i, spans - 1);
      const std::size_t at = (std::size_t{s} * attn::kKvHeads + kvh) * p.blocks + block;
      x[i] = p.part_ml[at * kBlockRows + col];
      x[i] = s0 + kWaves * i < spans ? x[i] : float2{kNoScore, 0.0f};
#pragma unroll
      for (unsigned j = 0; j < kQuads; ++j)
        y[i][j] = p.part_o[at * 8 * 256 + 64 * (kQuads * d + j) + lane];
    }
    float top = m;
#pragma unroll
    for (unsigned i = 0; i < kBatch; ++i)
      top = fmaxf(top, x[i].x);
    const float old = __builtin_amdgcn_exp2f(m - top);
    m = top;
    l *= old;
#pragma unroll
    for (unsigned j = 0; j < kQuads; ++j)
      o[j] = float4{o[j].x * old, o[j].y * old, o[j].z * old, o[j].w * old};
#pragma unroll
    for (unsigned i = 0; i < kBatch; ++i) {
      if (s0 + kWaves * i >= spans)  // uniform: a repeated span is left out (0 x infinity is NaN)
        break;
      const float e = __builtin_amdgcn_exp2f(x[i].x - top);
      l = __builtin_fmaf(x[i].y, e, l);
#pragma unroll
      for (unsigned j = 0; j < kQuads; ++j) {
        o[j].x = __builtin_fmaf(y[i][j].x, e, o[j].x);
        o[j].y = __builtin_fmaf(y[i][j].y, e, o[j].y);
        o[j].z = __builtin_fmaf(y[i][j].z, e, o[j].z);
        o[j].w = __builtin_fmaf(y[i][j].w, e, o[j].w);
      }
    }
  }
#pragma unroll
  for (unsigned j = 0; j < kQuads; ++j) {  // dimensions 8 j + 4 hi .. + 3 of the piece
    float* at = &rows[wave][col * kRow + 8 * j + 4 * hi];
    at[0] = o[j].x, at[1] = o[j].y, at[2] = o[j].z, at[3] = o[j].w;
  }
  if (hi == 0)
    ml[wave][col] = float2{m, l};
  __syncthreads();

  const unsigned row = t / (2 * kQuads), dim = 4 * (t % (2 * kQuads));
  const unsigned seq = kSeqs * block + row / kGroup;
  if (row >= kBlockRows || seq >= p.batch)
    return;
  const std::size_t out =
      (std::size_t{seq} * attn::kQHeads + kvh * kGroup + row % kGroup) * attn::kDim + kDims * d + dim;
  const float4 g = *reinterpret_cast<const float4*>(p.gate + out);
  float top = kNoScore;
#pragma unroll
  for (unsigned w = 0; w < kWaves; ++w)
    top = fmaxf(top, ml[w][row].x);
  float all = 0.0f, v[4] = {};
#pragma unroll
  for (unsigned w = 0; w < kWaves; ++w) {
    const float e = __builtin_amdgcn_exp2f(ml[w][row].x - top);
    all = __builtin_fmaf(ml[w][row].y, e, all);
#pragma unroll
    for (unsigned j = 0; j < 4; ++j)
      v[j] = __builtin_fmaf(rows[w][row * kRow + dim + j], e, v[j]);
  }
  if (p.s_max != 0) {
    const unsigned mine = own_keys(p, seq);
    const unsigned chunk = p.balanced != nullptr ? *p.balanced : p.chunk;
    const unsigned n = attn_shared_own_splits(mine, p.s_max, chunk);
    const std::size_t at0 =
        ((std::size_t{seq} * attn::kKvHeads + kvh) * p.s_max) * kGroup + row % kGroup;
    constexpr unsigned kSplits = 4;
    for (unsigned s0 = 0; s0 < n; s0 += kSplits) {
      float sm[kSplits], sl[kSplits];
      float4 so[kSplits];
#pragma unroll
      for (unsigned i = 0; i < kSplits; ++i) {
        const std::size_t at = at0 + static_cast<std::size_t>(min(s0 + i, n - 1)) * kGroup;
        sm[i] = p.own_m[at];
        sl[i] = p.own_l[at];
        so[i] = *reinterpret_cast<const float4*>(p.own_o + at * attn::kDim + kDims * d + dim);
      }
#pragma unroll
      for (unsigned i = 0; i < kSplits; ++i) {
        if (s0 + i >= n)
          break;
        if (!(sl[i] != 0.0f))  // an empty span
          continue;
        const float next = fmaxf(top, sm[i]);
        const float a = __builtin_amdgcn_exp2f(top - next), b = __builtin_amdgcn_exp2f(sm[i] - next);
        top = next;
        all = __builtin_fmaf(sl[i], b, all * a);
        v[0] = __builtin_fmaf(so[i].x, b, v[0] * a);
        v[1] = __builtin_fmaf(so[i].y, b, v[1] * a);
        v[2] = __builtin_fmaf(so[i].z, b, v[2] * a);
        v[3] = __builtin_fmaf(so[i].w, b, v[3] * a);
      }
    }
  }
  // Without keys 0, also where the gate is NaN.
  const float inv = all != 0.0f ? 1.0f / all : 0.0f;
  const float gv[4] = {g.x, g.y, g.z, g.w};
  float r[4];
#pragma unroll
  for (unsigned j = 0; j < 4; ++j)
    r[j] = all != 0.0f ? v[j] * inv / (1.0f + __expf(-gv[j])) : 0.0f;
  *reinterpret_cast<float4*>(p.core + out) = float4{r[0], r[1], r[2], r[3]};
}

// ------------------------------------------------------------------------------------------------
// Launch
// ------------------------------------------------------------------------------------------------

constexpr unsigned kAttnSharedCus = 256;
constexpr unsigned kAttnSharedOwnLeast = 16;  // workgroups of the own keys beside the prefix's

// Row blocks x spans of a KV head's partials: no less than any smaller batch or shorter prefix takes.
__host__ __device__ constexpr std::size_t attn_shared_part_blocks(unsigned batch, unsigned prefix) {
  const std::size_t blocks = (std::size_t{batch} + 3) / 4, tiles = (std::size_t{prefix} + 31) / 32;
  const std::size_t most = blocks <= 1 ? 128 : blocks <= 2 ? 256 : blocks < 512 ? 512 : blocks;
  return most < blocks * tiles ? most : blocks * tiles;
}

// The workspace: the prefix's partials, then the own keys' (as the ragged decode's balanced scratch).
struct AttnSharedLayout {
  std::size_t part_ml, own_m, own_l, own_o, bytes;  // part_o first
};
__host__ __device__ constexpr AttnSharedLayout attn_shared_layout(unsigned batch, unsigned max_own,
                                                                  unsigned prefix) {
  const std::size_t blocks = attn::kKvHeads * attn_shared_part_blocks(batch, prefix);
  const std::size_t own = attn_ragged_balanced_rows(batch, max_own) * attn::kQHeads + 4;
  AttnSharedLayout a{};
  a.part_ml = blocks * 32 * attn::kDim * sizeof(float);
  a.own_o = a.part_ml + blocks * 32 * sizeof(float2);
  a.own_m = a.own_o + own * attn::kDim * sizeof(float);
  a.own_l = a.own_m + own * sizeof(float);
  a.bytes = a.own_l + own * sizeof(float);
  return a;
}

// What a call launches.
struct AttnSharedRule {
  AttnSharedCut cut;               // of the prefix, unless the kernel chooses it (chosen)
  unsigned grid;                   // workgroups of the first split launch; 0: none
  unsigned own_first, own_grid;    // of the own keys: the first workgroup, their number
  unsigned own_least;              // AttnSharedParams'
  unsigned s_max, chunk;           // AttnSharedParams'
  unsigned step;                   // sequences of a split launch
  bool chosen, balanced, own_waves;
};
template <unsigned kRowBlocks>
inline AttnSharedRule attn_shared_rule(unsigned batch, unsigned prefix, unsigned max_own, unsigned cus) {
  AttnSharedRule r{};
  const unsigned blocks = (batch + 3) / 4;
  const unsigned tiles = prefix / 32 + (prefix % 32 != 0);
  const unsigned pairs = 2 * ((blocks + kRowBlocks - 1) / kRowBlocks);
  const unsigned shared_cus = std::min(cus, kAttnSharedCus);
  r.cut = attn_shared_cut<kRowBlocks>(tiles, pairs, 0.0f, shared_cus, 0);
  r.step = batch;
  r.grid = r.cut.grid;
  if (max_own == 0)
    return r;
  // The CUs that the prefix leaves, all of them where it leaves less than half; at most one streaming
  // launch's sequences and items at a time.
  r.own_grid = 2 * r.cut.grid <= cus ? cus - r.cut.grid : cus;
  r.s_max = std::min(attn_ragged_balanced_splits(batch, max_own),
                     kRaggedStreamMaxItems * r.own_grid / attn::kKvHeads);
  r.chunk = attn_ragged_chunk(batch, max_own, cus);
  const std::size_t items = std::size_t{batch} * attn::kKvHeads * r.s_max;
  const std::size_t least = (items + kRaggedStreamMaxItems - 1) / kRaggedStreamMaxItems;
  r.own_grid = static_cast<unsigned>(std::min<std::size_t>(r.own_grid, items));
  if (tiles != 0 && r.cut.grid <= shared_cus && batch <= kRaggedStreamMaxBatch &&
      least <= shared_cus) {
    // One round of workgroups, cut for no own keys or for max_own of every sequence; where either could
    // cost much beside the other, the kernel chooses (1.1 us: 16 sequences behind 4096 keys, 1024 each,
    // 17.3 us of the first cut, 18.6 of a chosen one).
    constexpr float kMuch = 3.0f;
    r.own_least = static_cast<unsigned>(
        std::min(items, std::max<std::size_t>(least, kAttnSharedOwnLeast)));
    r.own_waves = batch >= kAttnSharedWaveBatch;
    const float most = static_cast<float>(batch) *
                       attn_shared_own_tiles(max_own, r.own_waves && max_own <= kAttnSharedWaveKeys);
    const auto as = [&](float own_tiles) {
      return attn_shared_cut<kRowBlocks>(tiles, pairs, own_tiles, shared_cus, r.own_least);
    };
    const auto cost = [&](const AttnSharedCut& c, float own_tiles) {
      return attn_shared_cost<kRowBlocks>(c, own_tiles, shared_cus);
    };
    const AttnSharedCut few = as(1.0f), many = as(most);
    r.cut = cost(few, most) <= cost(many, most) + kMuch ? few : many;
    r.chosen = cost(r.cut, 1.0f) > cost(few, 1.0f) + kMuch;
    r.own_grid = r.cut.both
                     ? shared_cus
                     : static_cast<unsigned>(std::min<std::size_t>(shared_cus - r.cut.grid, items));
    r.grid = r.cut.both || r.chosen ? shared_cus : r.cut.grid + r.own_grid;
    r.own_first = r.cut.both ? 0 : r.cut.grid;
  } else {  // the own keys' workgroups follow the prefix's
    r.own_first = r.cut.grid;
    r.grid = r.cut.grid + r.own_grid;
    if (batch > kRaggedStreamMaxBatch || least > r.own_grid)
      r.step = std::min(kRaggedStreamMaxBatch,
                        std::max(1u, kRaggedStreamMaxItems * r.own_grid / (attn::kKvHeads * r.s_max)));
  }
  r.balanced = r.step >= batch &&
               attn_ragged_balanced(batch, max_own, cus, r.chosen ? r.own_least : r.own_grid);
  return r;
}

// p: q, gate, core, lens, prefix, batch, whole and own_cap given; the workspace holds
// attn_shared_layout(batch, max_own, p.prefix.len).
template <unsigned kRowBlocks, bool kPaged>
inline void attn_shared_launch_as(AttnSharedParams p, const AttnSharedOwn& own, unsigned max_own,
                                  char* ws, unsigned cus, hipStream_t stream) {
  const AttnSharedLayout at = attn_shared_layout(p.batch, max_own, p.prefix.len);
  p.part_o = reinterpret_cast<float4*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + at.part_ml);
  p.own_m = reinterpret_cast<float*>(ws + at.own_m);
  p.own_l = reinterpret_cast<float*>(ws + at.own_l);
  p.own_o = reinterpret_cast<float*>(ws + at.own_o);
  unsigned* const words = reinterpret_cast<unsigned*>(p.own_l) - 4;
  p.blocks = (p.batch + 3) / 4;
  const AttnSharedRule r = attn_shared_rule<kRowBlocks>(p.batch, p.prefix.len, max_own, cus);
  p.s_max = r.s_max;
  p.chunk = r.chunk;
  p.own_first = r.own_first;
  p.own_least = r.own_least;
  p.own_waves = r.own_waves;
  p.balanced = r.balanced ? words : nullptr;
  p.chosen = r.chosen ? words + 1 : nullptr;
  p.spans = r.cut.spans;
  p.span_tiles = r.cut.span_tiles;
  p.prefix_grid = r.cut.grid;
  for (unsigned s = 0; r.grid != 0 && s < p.batch; s += r.step) {
    const std::size_t row = std::size_t{s} * attn::kKvHeads * p.s_max * decode_detail::kGroup;
    AttnSharedParams a = p;
    AttnSharedOwn o = own;
    a.own_batch = std::min(r.step, p.batch - s);
    if (s != 0) {  // the own keys of more sequences
      a.prefix_grid = a.own_first = 0;
      a.q += std::size_t{s} * attn::kQHeads * attn::kDim;
      a.lens += s;
      a.own_m += row;
      a.own_l += row;
      a.own_o += row * attn::kDim;
      if (own.page_table == nullptr)
        o.kv_offsets += s;
      else if (own.rows != nullptr)
        o.rows += s;
      else
        o.page_table += std::size_t{s} * own.max_pages;
    }
    attn_shared_split_kernel<kRowBlocks, kPaged>
        <<<s == 0 ? r.grid : r.own_grid, 256, 0, stream>>>(a, o);
  }
  if (64 * p.blocks <= cus)
    attn_shared_merge_kernel<1, 8><<<64 * p.blocks, 512, 0, stream>>>(p);
  else if (16 * p.blocks < cus)
    attn_shared_merge_kernel<1, 4><<<64 * p.blocks, 256, 0, stream>>>(p);
  else
    attn_shared_merge_kernel<4, 4><<<16 * p.blocks, 256, 0, stream>>>(p);
}

inline void attn_shared_launch(const AttnSharedParams& p, const AttnSharedOwn& own, unsigned max_own,
                               char* ws, unsigned cus, hipStream_t stream) {
  const auto as = [&](auto paged) {
    constexpr bool kPaged = decltype(paged)::value;
    const unsigned rb = attn_shared_row_blocks(p.batch, p.prefix.len, cus);
    (rb == 1   ? attn_shared_launch_as<1, kPaged>
     : rb == 2 ? attn_shared_launch_as<2, kPaged>
               : attn_shared_launch_as<4, kPaged>)(p, own, max_own, ws, cus, stream);
  };
  if (own.page_table != nullptr)
    as(std::true_type{});
  else
    as(std::false_type{});
}

}  // namespace miso::kernels
