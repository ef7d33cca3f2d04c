#pragma once

// A batch of requests over a KV page pool, for MI355X (gfx950 / CDNA4); no reference counterpart (the
// reference serves one sequence over one contiguous cache).
//   attn_page_plan:  the step's page tables, slots and positions from request lengths, on the GPU.
//   attn_prep_paged: RMSNorm and rotation of the step's tokens, K / V appended to their slots.
// Page g of a pool holds [2 KV heads][page][256] f16 of K (and of V in a second pool), as the paged
// decode reads it (attention_decode.hpp); slot page x page_size + row names a row of both heads.

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "attention_decode.hpp"
#include "cdna4_wave.hpp"

namespace miso::kernels {

// ------------------------------------------------------------------------------------------------
// Page plan. Per request s: lens[s] keys so far, n_new[s] tokens in this step.
//   1. ended[s]: its pages from entry prefix_pages on go back on the stack of free pages, in the order
//      of request and entry, and its length becomes 0.
//   2. A request of length 0 that gets tokens starts behind the shared prefix: its first prefix_pages
//      entries are prefix_table's, its length theirs.
//   3. With cum[s] the pages that requests 0 .. s need, a request that needs pages gets them while
//      cum[s] <= free pages; the k-th page handed out is the k-th from the top. One that does not fit
//      (pages, its table row, the step's tokens) keeps its length; status says why.
//   4. Token t of the step (request by request): its request, position, slot and the keys it sees.
// Nothing here is more than a few words per request and token: the launches and the dependent steps
// (loads, three scans, a search per page and token) are its time. One workgroup does it, since the
// steps depend on sums over all requests; with more than kAttnPlanOneLaunch tokens a second launch spreads
// the pages and tokens over the CUs. 64 requests of a token each: 4.9 us. 512 with prompts, 66 thousand
// tokens, some ending: 9.8 + 7.3 us (13.4 + 7.0 with the pages handed out by the first launch and one
// search at a time).
// ------------------------------------------------------------------------------------------------

struct AttnPagePlanParams {
  const uint32_t* lens;
  const uint32_t* n_new;
  const uint32_t* ended;  // or nullptr: none
  int32_t* page_table;    // [batch][max_pages]
  const int32_t* prefix_table;
  int32_t* free_pages;  // [pool_pages]
  const uint32_t* n_free;
  uint32_t* lens_out;    // may be lens
  uint32_t* n_free_out;  // may be n_free
  int32_t* status;       // [batch]
  uint32_t* starts;      // [batch + 1]
  int32_t* slots;        // [max_tokens], as the following
  uint32_t* positions;
  int32_t* rows;
  uint32_t* visible;
  unsigned batch, max_pages, log2_page, prefix_pages, pool_pages, max_tokens;
};

constexpr unsigned kAttnPlanMaxBatch = 8192;

namespace pages_detail {

constexpr unsigned kThreads = 1024, kWaves = kThreads / cdna4::kLanes;
constexpr unsigned kNotHere = ~0u;  // base of a request that gets no tokens

enum : int32_t { kFits = 0, kNoPages = 1, kNoTable = 2, kNoTokens = 3 };

struct PlanShared {
  unsigned tokens[kAttnPlanMaxBatch];  // running sums, each with its request's own
  unsigned back[kAttnPlanMaxBatch];    // pages that go back
  unsigned need[kAttnPlanMaxBatch];
  unsigned base[kAttnPlanMaxBatch];  // length before the tokens
  unsigned wave[2][kWaves];
};

__device__ __attribute__((always_inline)) inline unsigned pages_of(unsigned long long keys,
                                                                   unsigned log2_page) {
  return static_cast<unsigned>((keys + (1ull << log2_page) - 1) >> log2_page);
}

// For each k the first request whose running sum exceeds it (n if none): kMany searches side by side, since
// one waits for LDS at each of its steps.
template <unsigned kMany>
__device__ __attribute__((always_inline)) inline void owners_of(const unsigned* sums, unsigned n,
                                                                const unsigned (&k)[kMany],
                                                                unsigned (&owner)[kMany]) {
#pragma unroll
  for (unsigned i = 0; i < kMany; ++i)
    owner[i] = 0;
  for (unsigned step = 1u << (31 - __builtin_clz(n)); step != 0; step /= 2) {
    unsigned sum[kMany];
#pragma unroll
    for (unsigned i = 0; i < kMany; ++i)
      sum[i] = sums[min(owner[i] + step, n) - 1];
#pragma unroll
    for (unsigned i = 0; i < kMany; ++i)
      owner[i] += owner[i] + step <= n && sum[i] <= k[i] ? step : 0u;
  }
}

// visit(k, s, place of k among request s's) for k = first, first + stride, .. below n; kMany at a time.
template <unsigned kMany, typename Visit>
__device__ __attribute__((always_inline)) inline void each_of_many(const unsigned* sums, unsigned batch,
                                                                   unsigned first, unsigned stride,
                                                                   unsigned n, Visit visit) {
  for (unsigned k0 = first; k0 < n; k0 += kMany * stride) {
    unsigned k[kMany], s[kMany];
#pragma unroll
    for (unsigned i = 0; i < kMany; ++i)
      k[i] = min(k0 + i * stride, n - 1);
    owners_of(sums, batch, k, s);
#pragma unroll
    for (unsigned i = 0; i < kMany; ++i)
      if (k0 + i * stride < n)
        visit(k[i], s[i], k[i] - (s[i] != 0 ? sums[s[i] - 1] : 0u));
  }
}
template <typename Visit>
__device__ __attribute__((always_inline)) inline void each_of(const unsigned* sums, unsigned batch,
                                                              unsigned first, unsigned stride,
                                                              unsigned n, Visit visit) {
  if (n <= stride)  // uniform
    each_of_many<1>(sums, batch, first, stride, n, visit);
  else
    each_of_many<4>(sums, batch, first, stride, n, visit);
}

// The sum of x over the threads before this one, and over all (in `all`); `words`: one per wave, not
// in use by a scan that some wave may still be reading.
__device__ __attribute__((always_inline)) inline unsigned scan_threads(unsigned x, unsigned* words,
                                                                       unsigned& all) {
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const unsigned incl = decode_detail::wave_prefix_sum(x);
  if (lane == 63)
    words[wave] = incl;
  __syncthreads();
  unsigned before = 0;
  all = 0;
#pragma unroll
  for (unsigned w = 0; w < kWaves; ++w) {
    const unsigned v = words[w];
    before += w < wave ? v : 0u;
    all += v;
  }
  return before + incl - x;
}

// The step's tokens first, first + stride, .. of kMany x stride (a part of max_tokens): ends, need: running
// sums of tokens and of pages handed out; base: lengths before; the pages handed out lie below `top`.
template <unsigned kMany>
__device__ __attribute__((always_inline)) inline void put_tokens(
    const AttnPagePlanParams& p, unsigned t0, unsigned stride, const unsigned* ends,
    const unsigned* need, const unsigned* base, unsigned top) {
  unsigned t[kMany], s[kMany], at[kMany], seen[kMany];
  int32_t page[kMany];
#pragma unroll
  for (unsigned i = 0; i < kMany; ++i)
    t[i] = t0 + i * stride;
  owners_of(ends, p.batch, t, s);
#pragma unroll
  for (unsigned i = 0; i < kMany; ++i) {
    const bool any = s[i] < p.batch;
    const unsigned row = any ? s[i] : 0u, before = row != 0 ? row - 1 : 0u;
    const unsigned from = base[row], pos = from + (t[i] - (row != 0 ? ends[before] : 0u));
    const unsigned entry = pos >> p.log2_page, held = pages_of(from, p.log2_page);
    const unsigned taken = (row != 0 ? need[before] : 0u) + (entry - held);
    // (A sum of n_new beyond 32 bits breaks the order: entries and stack are checked.)
    const bool good = any && from != kNotHere && t[i] < p.max_tokens && entry < p.max_pages &&
                      (entry < held || taken < top);
    page[i] = -1;
    if (good)
      page[i] = entry < held ? p.page_table[std::size_t{row} * p.max_pages + entry]
                             : p.free_pages[top - 1 - taken];
    s[i] = row;
    at[i] = good ? pos : 0u;
    seen[i] = good ? pos + 1 : 0u;
  }
#pragma unroll
  for (unsigned i = 0; i < kMany; ++i) {
    if (t[i] >= p.max_tokens)
      break;
    const bool good = static_cast<unsigned>(page[i]) < p.pool_pages;
    p.slots[t[i]] = good ? (page[i] << p.log2_page) +
                               static_cast<int32_t>(at[i] & ((1u << p.log2_page) - 1u))
                         : -1;
    p.positions[t[i]] = at[i];
    p.rows[t[i]] = static_cast<int32_t>(s[i]);
    p.visible[t[i]] = seen[i];
  }
}

// Entries of the pages handed out, by `stride` threads.
__device__ __attribute__((always_inline)) inline void put_pages(const AttnPagePlanParams& p,
                                                                unsigned thread, unsigned stride,
                                                                const unsigned* need,
                                                                const unsigned* base, unsigned top,
                                                                unsigned taken) {
  each_of(need, p.batch, thread, stride, taken, [&](unsigned k, unsigned s, unsigned at) {
    p.page_table[std::size_t{s} * p.max_pages + pages_of(base[s], p.log2_page) + at] =
        p.free_pages[top - 1 - k];
  });
}

}  // namespace pages_detail

// The lengths, the stack and the prefix's entries, one workgroup, a thread holding kPer requests in order;
// kTokens: the pages handed out and the step's tokens too, which attn_page_tokens_kernel does otherwise.
template <unsigned kPer, bool kTokens>
__global__ void __launch_bounds__(pages_detail::kThreads) attn_page_plan_kernel(
    AttnPagePlanParams p) {
  using namespace pages_detail;
  __shared__ PlanShared sh;
  const unsigned t = threadIdx.x, lane = t & 63u;
  const unsigned long long cap = static_cast<unsigned long long>(p.max_pages) << p.log2_page;
  unsigned len[kPer], grow[kPer], back[kPer], n_back = 0, n_tokens = 0;
#pragma unroll
  for (unsigned i = 0; i < kPer; ++i) {
    const unsigned s = t * kPer + i;
    len[i] = grow[i] = back[i] = 0;
    if (s < p.batch) {
      len[i] = p.lens[s];
      grow[i] = p.n_new[s];
      if (p.ended != nullptr && p.ended[s] != 0) {
        const unsigned held = min(pages_of(len[i], p.log2_page), p.max_pages);
        back[i] = held > p.prefix_pages ? held - p.prefix_pages : 0;
        len[i] = 0;
      }
    }
    n_back += back[i];
    n_tokens += grow[i];
  }
  const unsigned free0 = min(*p.n_free, p.pool_pages);
  unsigned all_back, all_tokens;
  unsigned at_back = scan_threads(n_back, sh.wave[0], all_back);
  unsigned at_token = scan_threads(n_tokens, sh.wave[1], all_tokens);
  const unsigned top = min(free0 + all_back, p.pool_pages);

  // What each request needs, its place in the step known.
  unsigned need[kPer], base[kPer], first[kPer], n_need = 0;
  int32_t why[kPer];
#pragma unroll
  for (unsigned i = 0; i < kPer; ++i) {
    const unsigned s = t * kPer + i;
    first[i] = at_token;
    at_token += grow[i];
    at_back += back[i];
    need[i] = 0;
    why[i] = kFits;
    base[i] = len[i] == 0 && grow[i] != 0 ? p.prefix_pages << p.log2_page : len[i];
    if (grow[i] != 0) {
      const unsigned long long end = static_cast<unsigned long long>(base[i]) + grow[i];
      why[i] = end > cap ? kNoTable : at_token > p.max_tokens || at_token < first[i] ? kNoTokens
                                                                                     : kFits;
      if (why[i] == kFits)
        need[i] = pages_of(end, p.log2_page) - pages_of(base[i], p.log2_page);
    }
    n_need += need[i];
    if (s < p.batch) {
      sh.back[s] = at_back;
      sh.tokens[s] = at_token;
    }
  }
  __syncthreads();  // sh.back whole, and the scans' words free again
  each_of(sh.back, p.batch, t, kThreads, all_back, [&](unsigned k, unsigned s, unsigned at) {
    if (free0 + k < p.pool_pages)
      p.free_pages[free0 + k] = p.page_table[std::size_t{s} * p.max_pages + p.prefix_pages + at];
  });
  unsigned all_need;
  unsigned at_need = scan_threads(n_need, sh.wave[0], all_need);  // its barrier: the stack is whole

  unsigned taken = 0;  // pages handed out, up to this thread's last request that got some
  unsigned long long starting[kPer];  // of the wave's lanes: those whose request starts
#pragma unroll
  for (unsigned i = 0; i < kPer; ++i) {
    const unsigned s = t * kPer + i;
    at_need += need[i];
    if (need[i] != 0) {
      if (at_need > top)
        why[i] = kNoPages;
      else
        taken = at_need;
    }
    const bool grows = grow[i] != 0 && why[i] == kFits;
    if (s < p.batch) {
      sh.need[s] = at_need;
      sh.base[s] = grows ? base[i] : kNotHere;
    }
    starting[i] = __builtin_amdgcn_ballot_w64(s < p.batch && grows && len[i] == 0);
    if (s < p.batch) {
      p.lens_out[s] = grows ? base[i] + grow[i] : len[i];
      p.status[s] = why[i];
      p.starts[s + 1] = first[i] + grow[i];
    }
  }
  // The prefix's entries of the requests that start, a wave at a time.
  for (unsigned j = lane; j - lane < p.prefix_pages; j += 64) {
    const int32_t page = p.prefix_table[min(j, p.prefix_pages - 1)];
#pragma unroll
    for (unsigned i = 0; i < kPer; ++i)
      for (unsigned long long left = starting[i]; left != 0; left &= left - 1) {
        const unsigned s = (t - lane + static_cast<unsigned>(__builtin_ctzll(left))) * kPer + i;
        if (j < p.prefix_pages)
          p.page_table[std::size_t{s} * p.max_pages + j] = page;
      }
  }
#pragma unroll
  for (unsigned o = 1; o < 64; o *= 2)
    taken = max(taken, static_cast<unsigned>(__shfl_xor(static_cast<int>(taken), o)));
  if (lane == 0)
    sh.wave[1][t >> 6] = taken;
  __syncthreads();
  taken = sh.wave[1][lane % kWaves];
#pragma unroll
  for (unsigned o = 1; o < kWaves; o *= 2)
    taken = max(taken, static_cast<unsigned>(__shfl_xor(static_cast<int>(taken), o)));
  if (t == 0) {
    p.starts[0] = 0;
    *p.n_free_out = top - taken;
  }
  if constexpr (kTokens) {
    put_pages(p, t, kThreads, sh.need, sh.base, top, taken);
    if (p.max_tokens <= kThreads) {
      if (t < p.max_tokens)
        put_tokens<1>(p, t, kThreads, sh.tokens, sh.need, sh.base, top);
    } else {
      for (unsigned t0 = t; t0 < p.max_tokens; t0 += 4 * kThreads)
        put_tokens<4>(p, t0, kThreads, sh.tokens, sh.need, sh.base, top);
    }
  }
}

// The pages handed out and the step's tokens where those are many, 1024 tokens a workgroup, behind the
// launch above: what that one knew of the requests follows from what it left.
template <int = 0>
__global__ void __launch_bounds__(256) attn_page_tokens_kernel(AttnPagePlanParams p) {
  using namespace pages_detail;
  __shared__ unsigned ends[kAttnPlanMaxBatch], need[kAttnPlanMaxBatch], base[kAttnPlanMaxBatch];
  __shared__ unsigned words[4];
  const unsigned t = threadIdx.x, lane = t & 63u;
  for (unsigned s = t; s < p.batch; s += 256) {
    const unsigned end = p.starts[s + 1], grow = end - p.starts[s];
    const unsigned len = p.lens_out[s], from = len - grow;
    const bool here = grow != 0 && p.status[s] == kFits;
    ends[s] = end;
    base[s] = here ? from : kNotHere;
    need[s] = here ? pages_of(len, p.log2_page) - pages_of(from, p.log2_page) : 0u;
  }
  __syncthreads();
  // need's running sums, each thread's share of the requests in order.
  const unsigned per = (p.batch + 255) / 256, s0 = min(t * per, p.batch), s1 = min(s0 + per, p.batch);
  unsigned mine = 0;
  for (unsigned s = s0; s < s1; ++s)
    mine += need[s];
  const unsigned incl = decode_detail::wave_prefix_sum(mine);
  if (lane == 63)
    words[t >> 6] = incl;
  __syncthreads();
  unsigned sum = incl - mine;
  for (unsigned w = 0; w < t >> 6; ++w)
    sum += words[w];
  for (unsigned s = s0; s < s1; ++s)
    need[s] = sum += need[s];
  __syncthreads();
  const unsigned taken = need[p.batch - 1], top = *p.n_free_out + taken;
  put_tokens<4>(p, 1024 * blockIdx.x + t, 256, ends, need, base, top);
  put_pages(p, 256 * blockIdx.x + t, 256 * gridDim.x, need, base, top, taken);
}

// Up to this many tokens are placed by the first launch: 64 requests with 3523 tokens 6.8 us there, 3.7 +
// 4.7 in two; 512 with 2434 12.7 and 9.2 + 5.8, with 4450 15.0 and 9.2 + 6.5.
constexpr unsigned kAttnPlanOneLaunch = 4096;

inline void attn_page_plan_launch(const AttnPagePlanParams& p, hipStream_t stream) {
  using pages_detail::kThreads;
  const bool one = p.max_tokens <= kAttnPlanOneLaunch;
  if (p.batch <= kThreads) {
    if (one)
      attn_page_plan_kernel<1, true><<<1, kThreads, 0, stream>>>(p);
    else
      attn_page_plan_kernel<1, false><<<1, kThreads, 0, stream>>>(p);
  } else {
    constexpr unsigned kPer = kAttnPlanMaxBatch / kThreads;
    if (one)
      attn_page_plan_kernel<kPer, true><<<1, kThreads, 0, stream>>>(p);
    else
      attn_page_plan_kernel<kPer, false><<<1, kThreads, 0, stream>>>(p);
  }
  if (!one)
    attn_page_tokens_kernel<<<(p.max_tokens + 1023) / 1024, 256, 0, stream>>>(p);
}

// ------------------------------------------------------------------------------------------------
// Paged prep. Token t: x <- x / sqrt(mean x^2 + eps) * w for its 16 query and 2 key heads, the first
// rope_dims values of each turned by pos_t x inv_freq[i], in pairs (i, i + rope_dims / 2), or
// (2 i, 2 i + 1) where interleaved, cos and sin times rot_scale; K and V to f16 (nearest even) in row
// slots[t] of the pool, queries and gates to dense rows. A token without a slot (outside [0, rows of
// the pool)) is left out: nothing of it is read or written.
//
// The angle is formed and reduced to (-pi, pi] in 64 bits: pos x inv_freq in f32 is off by up to 0.008
// rad at position 262143, and the rotation by as much. K and V are rounded to f16, half a step, as the caches
// hold them; all else is f32.
//
// A workgroup per token, a head a wave at a time (64 lanes x 4 dimensions), three heads a wave with all
// loads in flight before the first use: the rotation's partners lie in the same wave, its sines are
// computed once for the token. Bound by memory: 70 KiB a token. 4096 tokens 55.9 us, 5.2 TB/s of those
// bytes (the caches keep some of them); 1001 11.7; 64 3.9; 1 2.7, a launch.
// ------------------------------------------------------------------------------------------------

struct AttnPrepPagedParams {
  const float* qg;  // token t at t * proj_stride, as attn_prep_batch
  const float* k;
  const float* v;
  const float* q_norm;
  const float* k_norm;
  const float* inv_freq;  // [rope_dims / 2]
  attn::half_t* k_pages;
  attn::half_t* v_pages;
  const int32_t* slots;       // [n]
  const uint32_t* positions;  // [n]
  float* q;                   // [n][16][256]
  float* gate;                // [n][16][256], or nullptr
  unsigned n, proj_stride, log2_page, pool_rows, rope_dims;
  float rot_scale, eps;
};

// One workgroup of 6 waves per token: a wave has three of the 18 rows to normalise and three of the
// 18 to copy (16 gates, 2 V), all in flight while the token's angles are computed.
template <bool kInterleaved>
__global__ void __launch_bounds__(384) attn_prep_paged_kernel(AttnPrepPagedParams p) {
  using namespace attn;
  constexpr unsigned kRows = 3;
  __shared__ __attribute__((aligned(16))) float turn[2][kDim / 2];  // cos, sin
  const unsigned t = blockIdx.x, lane = threadIdx.x & 63u;
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned slot = static_cast<unsigned>(p.slots[t]);
  if (slot >= p.pool_rows)  // uniform
    return;
  const std::size_t src = std::size_t{t} * p.proj_stride + 4 * lane;
  float4 x[kRows], y[kRows];
#pragma unroll
  for (unsigned i = 0; i < kRows; ++i) {
    const unsigned head = kRows * wave + i;
    x[i] = *reinterpret_cast<const float4*>(
        (head < kQHeads ? p.qg + head * 2 * kDim : p.k + (head - kQHeads) * kDim) + src);
    if (head >= kQHeads || p.gate != nullptr)  // uniform
      y[i] = *reinterpret_cast<const float4*>(
          (head < kQHeads ? p.qg + head * 2 * kDim + kDim : p.v + (head - kQHeads) * kDim) + src);
  }
  const float4 wq = *reinterpret_cast<const float4*>(p.q_norm + 4 * lane);
  const float4 wk = *reinterpret_cast<const float4*>(p.k_norm + 4 * lane);
  if (threadIdx.x < p.rope_dims / 2) {
    const double turns = static_cast<double>(p.positions[t]) *
                         static_cast<double>(p.inv_freq[threadIdx.x]) * 0.15915494309189533577;
    float s, c;
    sincosf(static_cast<float>((turns - __builtin_rint(turns)) * 6.28318530717958647693), &s, &c);
    turn[0][threadIdx.x] = c * p.rot_scale;
    turn[1][threadIdx.x] = s * p.rot_scale;
  }
  __syncthreads();
  const unsigned eighth = p.rope_dims / 8;  // lanes of half the rotated part
#pragma unroll
  for (unsigned i = 0; i < kRows; ++i) {
    const unsigned head = kRows * wave + i;
    const bool is_q = head < kQHeads;
    const float4 w = is_q ? wq : wk;
    const float ss = cdna4::wave_allsum(__builtin_fmaf(
        x[i].w, x[i].w,
        __builtin_fmaf(x[i].z, x[i].z, __builtin_fmaf(x[i].y, x[i].y, x[i].x * x[i].x))));
    const float r = rsqrtf(ss / kDim + p.eps);
    float v[4] = {x[i].x * r * w.x, x[i].y * r * w.y, x[i].z * r * w.z, x[i].w * r * w.w};
    if constexpr (kInterleaved) {
      if (lane < 2 * eighth) {
        const float2 c = *reinterpret_cast<const float2*>(&turn[0][2 * lane]);
        const float2 s = *reinterpret_cast<const float2*>(&turn[1][2 * lane]);
        const float a0 = v[0], a1 = v[2];
        v[0] = a0 * c.x - v[1] * s.x;
        v[1] = a0 * s.x + v[1] * c.x;
        v[2] = a1 * c.y - v[3] * s.y;
        v[3] = a1 * s.y + v[3] * c.y;
      }
    } else {
      const bool low = lane < eighth;
      const unsigned other = low ? lane + eighth : lane - eighth;
      float partner[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        partner[j] = __shfl(v[j], static_cast<int>(other));
      if (lane < 2 * eighth) {
        const float4 c = *reinterpret_cast<const float4*>(&turn[0][4 * (low ? lane : other)]);
        const float4 s = *reinterpret_cast<const float4*>(&turn[1][4 * (low ? lane : other)]);
        const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = v[j] * cs[j] + (low ? -partner[j] : partner[j]) * sn[j];
      }
    }
    if (is_q) {
      const std::size_t at = (std::size_t{t} * kQHeads + head) * kDim + 4 * lane;
      *reinterpret_cast<float4*>(p.q + at) = float4{v[0], v[1], v[2], v[3]};
      if (p.gate != nullptr)
        *reinterpret_cast<float4*>(p.gate + at) = y[i];
    } else {
      const std::size_t page = slot >> p.log2_page, row = slot & ((1u << p.log2_page) - 1u);
      const std::size_t at =
          (((page * kKvHeads + (head - kQHeads)) << p.log2_page) + row) * kDim + 4 * lane;
      *reinterpret_cast<cdna4::half4_t*>(p.k_pages + at) =
          cdna4::half4_t{static_cast<_Float16>(v[0]), static_cast<_Float16>(v[1]),
                         static_cast<_Float16>(v[2]), static_cast<_Float16>(v[3])};
      *reinterpret_cast<cdna4::half4_t*>(p.v_pages + at) =
          cdna4::half4_t{static_cast<_Float16>(y[i].x), static_cast<_Float16>(y[i].y),
                         static_cast<_Float16>(y[i].z), static_cast<_Float16>(y[i].w)};
    }
  }
}

}  // namespace miso::kernels
