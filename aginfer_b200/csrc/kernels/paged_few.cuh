// Attention over a paged cache for few rows a sequence and key head (a decoding step: one token, a few drafted ones):
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),  one pass over the keys with a running maximum m and sum.
//
// Bound by memory: a key and a value are 4 head_dim bytes and meet at most 32 rows.  So the unit of work is a tile of 64 keys of
// one sequence and key head, all units of the batch in one line, and every CTA takes an equal run of it, however unequal the
// sequences are.  Runs are even shares in a batch that fills the card, and longer, on fewer CTAs, where parts to be added would cost
// more (see run_length).  Sequences and heads that a run cuts leave unnormalised sums, their maximum and weight in scratch, and the
// last CTA of such an item to arrive adds them in order (nobody waits for another CTA; sums do not depend on who arrives when).
//
// A CTA: one loading warp that brings tiles in by bulk copies, a copy per page (or the part of it in the tile) and 64-column
// block, into a ring; four warps that share a tile's keys, 16 each, with maximum, sum and outputs of their own until the item ends.
// The rows of the query heads that share a key head are columns of one, two or four mma.sync tiles (m16n8k16) with the keys as rows:
// S^T = K Q^T, O^T += V^T P^T.  With the rows as rows, seven or eight of them would pay for sixteen, and these products (30 clocks of
// a scheduler's tensor pipe each) took longer than the bytes.  Keys and values lie in shared memory as they lie in the pool,
// swizzled, so ldmatrix reads them without bank conflicts.
//
// Weights are rounded to bf16 to meet the values in the tensor core, sums are of the unrounded ones, in 32 bits: the outputs are then
// 2.0 - 2.3e-3 (2-norm, relative) off the definition where weights in 32 bits and the outputs' own rounding leave 1.6 - 1.7e-3.  Weights
// in two bf16 pieces would take that back for twice the products of P V.
//
// A value behind the sequence's end is whatever the page held before, NaN perhaps, and weight zero does not make it zero: such
// values are masked as they are read.
#pragma once

#include "attention.cuh"
#include "gemm_tc.cuh"
#include "paged.cuh"

namespace few {

using namespace paged;

constexpr unsigned kKeys = 64, kConsumers = 128, kThreads = 160;
// The last CTA of an item adds its parts, four loads at a time, so a run is longer than an even share where that would make many parts:
// one tile a part costs 0.7 us of a CTA on its own, four more parts 1.4 us of the last one, which n tiles balance at runs of sqrt(n / 2).
// One token, 16 query heads on 2, us (these runs | even shares | at most 12 parts whatever the length):
//   1500 keys 12.3 | 14.3 | 12.3, 8192 18.4 | 39.7 | 22.5, 32000 31 - 33 | 43.6 | 47, 131072 56 | 71 | 150.
// Twelve parts are few enough below 72 tiles (700 keys 12.3, runs of sqrt(n / 2) 14.3).  Where the batch is large enough to keep memory
// busy, a third more than an even share is better than more parts (four sequences of 32000 keys on 4 heads 59.6, without it 62.4).
constexpr unsigned kFewParts = 12;
__device__ __forceinline__ unsigned run_length(unsigned total, unsigned longest, unsigned ctas) {
  const unsigned even = (total + ctas - 1) / ctas, balanced = unsigned(ceilf(sqrtf(float(longest) * 0.5f)));
  return max(even, min((longest + kFewParts - 1) / kFewParts, max(balanced, even + even / 3)));
}
constexpr float kSlack = 8.f;               // log2 of how far scores may exceed the maximum that weights are relative to

// How many units one sequence is: its key heads x row blocks x key tiles.
struct Items {
  Span span;
  Visible seen;
  unsigned blocks, units;             // row blocks of a key head; units of the sequence
};
template <unsigned kRows>
__device__ __forceinline__ Items items_of(const Batch& batch, const Claim& claim, unsigned group, unsigned kv_heads, unsigned window, unsigned sinks) {
  Items it;
  it.span = span_of(batch, claim);
  it.seen = visible_of<kKeys>(it.span.first, int(it.span.length) - 1, it.span.length, window, sinks);
  it.blocks = (it.span.fresh * group + kRows - 1) / kRows;
  it.units = it.blocks * kv_heads * it.seen.count;
  return it;
}

// Partial results of an item that more than one CTA works on: slot 0 of a CTA where the item began before its run, slot 1 where
// the item goes on behind it.  [cta][slot][row][head_dim] and [cta][slot][row][2] (maximum in units of log2, weight).
template <unsigned kRows, unsigned kDim>
struct Scratch {
  float* sums;
  float* ends;
  __device__ __forceinline__ float* sum(unsigned cta, unsigned slot, unsigned row) const { return sums + (size_t(cta * 2 + slot) * kRows + row) * kDim; }
  __device__ __forceinline__ float* end(unsigned cta, unsigned slot, unsigned row) const { return ends + (size_t(cta * 2 + slot) * kRows + row) * 2; }
};

// The run of a CTA in the line of units, found by every warp for itself, a lane per sequence: no barrier, one trip to memory for up to
// 32 sequences.
struct Run {
  unsigned per, from, to;             // units of a run; this one's
  unsigned seq, first;                // the sequence that holds unit `from`, and its first unit
  Claim claim;                        // what the batch says of it
};
template <unsigned kRows>
__device__ __forceinline__ Run run_of(const Batch& batch, unsigned group, unsigned kv_heads, unsigned window, unsigned sinks) {
  const unsigned lane = threadIdx.x & 31;
  bool ordered = true;
  unsigned units = 0, total = 0, longest = 0;
  Claim claim{0, 0, 0};
#pragma unroll 2
  for (unsigned i = lane; i < batch.sequences; i += 32) {
    claim = claim_of(batch, i);
    ordered = in_order(batch, claim) && ordered;
    const Items it = items_of<kRows>(batch, claim, group, kv_heads, window, sinks);
    units = it.units;
    total += units;
    if (units) longest = max(longest, it.seen.count);
  }
  total = __reduce_add_sync(0xffffffffu, total);
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (!__all_sync(0xffffffffu, ordered)) total = 0;
  Run run;
  run.per = run_length(total, longest, gridDim.x);
  run.from = min(run.per * blockIdx.x, total);
  run.to = min(run.from + run.per, total);
  run.seq = run.first = 0;
  run.claim = claim;
  if (run.from >= run.to) return run;
  unsigned below = 0;
#pragma unroll 1
  for (unsigned base = 0;; base += 32) {
    if (batch.sequences > 32) {
      units = 0;
      if (base + lane < batch.sequences) {
        claim = claim_of(batch, base + lane);
        units = items_of<kRows>(batch, claim, group, kv_heads, window, sinks).units;
      }
    }
    unsigned up_to = units;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned other = __shfl_up_sync(0xffffffffu, up_to, d);
      if (lane >= unsigned(d)) up_to += other;
    }
    const unsigned holds = __ballot_sync(0xffffffffu, run.from < below + up_to);
    if (holds) {
      const unsigned at = __ffs(holds) - 1;
      run.seq = base + at;
      run.first = below + __shfl_sync(0xffffffffu, up_to - units, at);
      run.claim = Claim{__shfl_sync(0xffffffffu, claim.from, at), __shfl_sync(0xffffffffu, claim.to, at), __shfl_sync(0xffffffffu, claim.length, at)};
      return run;
    }
    below += __shfl_sync(0xffffffffu, up_to, 31);
  }
}

template <int HD16, int kN>
__device__ __forceinline__ void attention_body(const bf16* q, bf16* o, const bf16* k_pool, const bf16* v_pool, const Batch& batch, float* own_sums,
                                               float* own_ends, float* scratch, unsigned* counters, unsigned q_heads, unsigned kv_heads,
                                               unsigned q_stride, unsigned o_stride, unsigned window, unsigned sinks, float scale_log2, unsigned stages,
                                               unsigned own_only) {
  constexpr unsigned kDim = HD16 * 16, kBlocks = kDim / 64, kRows = 8 * kN;
  constexpr unsigned kTileBytes = kKeys * kDim * 2, kStageBytes = 2 * kTileBytes, kBlockBytes = kKeys * 128;
  constexpr unsigned kMaxStages = 6;
  extern __shared__ unsigned char dynamic_smem[];
  __shared__ __align__(8) unsigned long long full_bar[kMaxStages], empty_bar[kMaxStages];
  __shared__ unsigned gave_up, last_flag;
  __shared__ float warp_max_of[4][kRows], warp_sum_of[4][kRows];
  const unsigned tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned ring = (tc::smem_u32(dynamic_smem) + 127u) & ~127u;
  float* const exchange = reinterpret_cast<float*>(dynamic_smem + (ring - tc::smem_u32(dynamic_smem)) + stages * kStageBytes);   // [4][8][head_dim]
  auto cell = [&](unsigned w, unsigned r8, unsigned d) { return exchange + (w * 8 + r8) * kDim + (d ^ ((r8 >> 1) * 8)); };      // no bank conflicts
  const unsigned group = q_heads / kv_heads;

  if (tid == 0) {
    for (unsigned s = 0; s < stages; ++s) {
      tc::mbar_init(&full_bar[s], 1);
      tc::mbar_init(&empty_bar[s], 4);
    }
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  // In front of a prefix's launch, which begins without waiting for this one, what this one waits for has to be complete.
  if (own_only) grid_dependency_wait_then_release();
  else grid_dependency_wait();
  if (!(aligned16(q) && aligned16(o) && aligned16(k_pool) && aligned16(v_pool))) {
    if (tid == 0) report(batch.status, kMisaligned);
    return;
  }
  const Run run = run_of<kRows>(batch, group, kv_heads, window, sinks);
  if (run.from >= run.to) return;

  // Walks the run item by item: f(sequence, key head, row block, its items, first tile, last tile + 1, first unit of the item).
  auto walk = [&](auto&& f) {
    unsigned seq = run.seq, first = run.first, unit = run.from;
    Claim claim = run.claim;
#pragma unroll 1
    while (unit < run.to) {
      const Items it = items_of<kRows>(batch, claim, group, kv_heads, window, sinks);
#pragma unroll 1
      while (unit < run.to && unit < first + it.units) {
        const unsigned at = (unit - first) / it.seen.count;                // which item of the sequence
        const unsigned item_first = first + at * it.seen.count, begin = unit - item_first, end = min(it.seen.count, begin + (run.to - unit));
        const unsigned head = at / it.blocks;
        f(seq, head, at - head * it.blocks, it, begin, end, item_first);
        unit += end - begin;
      }
      first += it.units;
      if (unit < run.to && ++seq < batch.sequences) claim = claim_of(batch, seq);
    }
  };
  auto await = [&](unsigned long long* bar, unsigned parity, unsigned code) {
    if (!*(volatile unsigned*)&gave_up && !tc::mbar_wait(bar, parity, batch.status, code)) *(volatile unsigned*)&gave_up = 1;
  };

  if (warp == 4) {
    // ---- loading warp: a lane per piece (keys or values, 64-column block, page or part of one) of a tile ----
    const unsigned shift = 31 - __clz(batch.page), run_tokens = min(batch.page, kKeys), pieces = kKeys / run_tokens;
    const bool values = lane >= pieces * kBlocks;
    const unsigned block = (lane / pieces) % kBlocks, piece = lane % pieces;
    const bool live = lane < 2 * kBlocks * pieces;
    const unsigned to_slot = (values ? kTileBytes : 0u) + block * kBlockBytes + piece * run_tokens * 128;
    const unsigned page_bytes = kv_heads * kBlocks * batch.page * 128;
    unsigned s = 0, phase = 1;
    walk([&](unsigned seq, unsigned head, unsigned, const Items& it, unsigned begin, unsigned end, unsigned) {
      const int* const pages_of = batch.table + size_t(seq) * batch.width;
      const unsigned char* const pool = reinterpret_cast<const unsigned char*>(values ? v_pool : k_pool) + size_t((head * kBlocks + block) * batch.page) * 128;
      auto token_of = [&](unsigned t) { return it.seen.tile(t) * kKeys + piece * run_tokens; };
      auto tokens_of = [&](unsigned t) {      // that this lane brings in
        const unsigned token = token_of(t);
        const bool wanted = live && token < it.seen.end && (token < it.seen.sink_end || token + run_tokens > it.seen.start);
        return wanted ? min(run_tokens, it.seen.end - token) : 0u;
      };
      unsigned count = tokens_of(begin), page_id = count ? unsigned(pages_of[token_of(begin) >> shift]) : 0u;
#pragma unroll 1
      for (unsigned t = begin; t < end; ++t) {
        if (page_id >= batch.pages) {
          report(batch.status, kBadPage);
          count = 0;
        }
        const unsigned char* const from_page = pool + size_t(page_id) * page_bytes + (token_of(t) & (batch.page - 1)) * 128;
        const unsigned bytes = count * 128, all = __reduce_add_sync(0xffffffffu, bytes);
        unsigned next_count = 0, next_page = 0;      // the page of the tile behind it, while this one's slot is awaited
        if (t + 1 < end) {
          next_count = tokens_of(t + 1);
          if (next_count) next_page = unsigned(pages_of[token_of(t + 1) >> shift]);
        }
        if (lane == 0) {
          await(&empty_bar[s], phase, tc::kTimeoutEmpty | s);
          tc::expect_bytes(&full_bar[s], all);
        }
        __syncwarp();
        if (bytes) tc::bulk_copy(ring + s * kStageBytes + to_slot, from_page, bytes, &full_bar[s]);
        count = next_count;
        page_id = next_page;
        if (++s == stages) { s = 0; phase ^= 1; }
      }
    });
    return;
  }

  // ---- four warps: 16 keys each of every tile ----
  const Scratch<kRows, kDim> parts{scratch, scratch + size_t(gridDim.x) * 2 * kRows * kDim};
  const unsigned g = lane >> 2, t4 = lane & 3;
  auto consumers_sync = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
  unsigned s = 0, phase = 0;
  walk([&](unsigned seq, unsigned head, unsigned block, const Items& it, unsigned begin, unsigned end, unsigned item_first) {
    const Span& span = it.span;
    const unsigned row0 = block * kRows, rows = min(kRows, span.fresh * group - row0);
    const Rows pairs(row0, group);
    // Q as the B operand: row r of the item (token, query head) is column r
    unsigned qb[kN][HD16][2];
    int index[kN][2];                // of rows 2 t and 2 t + 1, whose scores this thread holds
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      unsigned token, sub;
      pairs.at(j * 8 + g, token, sub);
      const bool live = j * 8 + g < rows;
      const unsigned* from_row = reinterpret_cast<const unsigned*>(q + (live ? size_t(span.row + token) * q_stride + (head * group + sub) * kDim : 0)) + t4;
#pragma unroll
      for (int ks = 0; ks < HD16; ++ks) {
        qb[j][ks][0] = live ? __ldcg(from_row + ks * 8) : 0u;
        qb[j][ks][1] = live ? __ldcg(from_row + ks * 8 + 4) : 0u;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        pairs.at(j * 8 + 2 * t4 + e, token, sub);
        index[j][e] = j * 8 + 2 * t4 + e < rows ? span.first + int(token) : -1;
      }
    }
    float top[kN][2], sum[kN][2], out[kN][HD16][4];
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      top[j][0] = top[j][1] = -INFINITY;
      sum[j][0] = sum[j][1] = 0.f;
#pragma unroll
      for (int m = 0; m < HD16; ++m) out[j][m][0] = out[j][m][1] = out[j][m][2] = out[j][m][3] = 0.f;
    }
    const int low = span.first + int(pairs.token);                 // the item's first row
#pragma unroll 1
    for (unsigned t = begin; t < end; ++t) {
      await(&full_bar[s], phase, tc::kTimeoutFull | s);
      __syncwarp();
      const unsigned key0 = it.seen.tile(t) * kKeys + warp * 16, slot = ring + s * kStageBytes;
      if (key0 < it.seen.end) {
        // scores, keys as rows: S^T = K Q^T.  Lanes 0-7 | 8-15 | 16-23 | 24-31 address the 8 x 8 blocks (keys 0-7, chunk c) | (8-15, c) |
        // (0-7, c + 1) | (8-15, c + 1).  Two accumulators a column group: half the chain of dependent products.
        float score[kN][2][4];
#pragma unroll
        for (int j = 0; j < kN; ++j)
#pragma unroll
          for (int n = 0; n < 2; ++n) score[j][n][0] = score[j][n][1] = score[j][n][2] = score[j][n][3] = 0.f;
        const unsigned k_row = slot + (warp * 16 + (lane & 15)) * 128;
#pragma unroll
        for (int ks = 0; ks < HD16; ++ks) {
          unsigned a0, a1, a2, a3;
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                       : "=r"(a0), "=r"(a1), "=r"(a2), "=r"(a3)
                       : "r"(k_row + (ks / 4) * kBlockBytes + ((((ks % 4) * 2 + (lane >> 4)) ^ (lane & 7)) << 4)));
#pragma unroll
          for (int j = 0; j < kN; ++j) skinny_mma_bf16(score[j][ks & 1], a0, a1, a2, a3, qb[j][ks][0], qb[j][ks][1]);
        }
        // does every row see all of these keys?  (columns behind the item's rows may hold anything)
        const bool whole = int(key0) + 15 <= low && key0 + 16 <= it.seen.end && (window == 0 || int(key0) > int(span.length) - 1 - int(window));
        unsigned pb[kN][2];
        bool grows = false;
        float x[kN][4], now[kN][2];
#pragma unroll
        for (int j = 0; j < kN; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {       // key g (+ 8), row 2 t (+ 1)
            x[j][i] = (score[j][0][i] + score[j][1][i]) * scale_log2;
            const unsigned key = key0 + g + (i >> 1) * 8;
            if (!whole && !(key < it.seen.end && sees(index[j][i & 1], key, window, sinks))) x[j][i] = -INFINITY;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float peak = fmaxf(x[j][e], x[j][e + 2]);
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 4));
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 8));
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 16));
            now[j][e] = peak;
            grows = grows || peak > top[j][e] + kSlack;
          }
        }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int j = 0; j < kN; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float next = fmaxf(top[j][e], now[j][e]), old = next == -INFINITY ? 1.f : exp2_of(top[j][e] - next);
              top[j][e] = next;
              sum[j][e] *= old;
#pragma unroll
              for (int m = 0; m < HD16; ++m) {
                out[j][m][e] *= old;
                out[j][m][e + 2] *= old;
              }
            }
        }
#pragma unroll
        for (int j = 0; j < kN; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[j][i] = exp2_of(x[j][i] - (top[j][i & 1] == -INFINITY ? 0.f : top[j][i & 1]));
          sum[j][0] += x[j][0] + x[j][2];
          sum[j][1] += x[j][1] + x[j][3];
          const bf162 first = __floats2bfloat162_rn(x[j][0], x[j][1]), second = __floats2bfloat162_rn(x[j][2], x[j][3]);
          // keys as rows -> keys as columns: P^T as the B operand of O^T += V^T P^T
          asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb[j][0]) : "r"(*reinterpret_cast<const unsigned*>(&first)));
          asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb[j][1]) : "r"(*reinterpret_cast<const unsigned*>(&second)));
        }
        // values: keys 2 t, 2 t + 1 (and + 8) of a column; those that no row of the sequence sees are taken as zero
        unsigned keep[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned key = key0 + i * 8 + 2 * t4;
          auto held = [&](unsigned j) { return j < it.seen.end && (j >= it.seen.start || j < it.seen.sink_end); };
          keep[i] = (held(key) ? 0xffffu : 0u) | (held(key + 1) ? 0xffff0000u : 0u);
        }
        const unsigned v_row = slot + kTileBytes + (warp * 16 + (lane >> 4) * 8 + (lane & 7)) * 128;
#pragma unroll
        for (int m = 0; m < HD16; ++m) {
          unsigned a0, a1, a2, a3;
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                       : "=r"(a0), "=r"(a1), "=r"(a2), "=r"(a3)
                       : "r"(v_row + (m / 4) * kBlockBytes + ((((m % 4) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4)));
          a0 &= keep[0];
          a1 &= keep[0];
          a2 &= keep[1];
          a3 &= keep[1];
#pragma unroll
          for (int j = 0; j < kN; ++j) skinny_mma_bf16(out[j][m], a0, a1, a2, a3, pb[j][0], pb[j][1]);
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&empty_bar[s]);
      if (++s == stages) { s = 0; phase ^= 1; }
    }

    // ---- the four warps' shares meet, eight rows at a time ----
    const bool whole_item = begin == 0 && end == it.seen.count;
    const unsigned slot = begin > 0 ? 0u : 1u;
    // four columns of a row, divided, or as they are with the row's maximum and weight
    auto leave = [&](unsigned r, unsigned c, float4 v, float peak, float weight) {
      unsigned token, sub;
      pairs.at(r, token, sub);
      const unsigned row = span.row + token, q_head = head * group + sub;
      if (own_only) {
        const Own own{own_sums, own_ends, batch.rows * group, kDim};
        *own.sum(head, c / 4, row * group + sub) = v;
        if (c == 0) *own.end(head, row * group + sub) = make_float2(peak, weight);
        return;
      }
      const float inv = weight > 0.f ? 1.f / weight : 0.f;
      const bf162 pair[2] = {__floats2bfloat162_rn(v.x * inv, v.y * inv), __floats2bfloat162_rn(v.z * inv, v.w * inv)};
      *reinterpret_cast<uint2*>(o + size_t(row) * o_stride + q_head * kDim + c) = *reinterpret_cast<const uint2*>(pair);
    };
#pragma unroll
    for (int j = 0; j < kN; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float all = sum[j][e];
        all += __shfl_xor_sync(0xffffffffu, all, 4);
        all += __shfl_xor_sync(0xffffffffu, all, 8);
        all += __shfl_xor_sync(0xffffffffu, all, 16);
        if (g == 0) {
          warp_max_of[warp][j * 8 + 2 * t4 + e] = top[j][e];
          warp_sum_of[warp][j * 8 + 2 * t4 + e] = all;
        }
      }
#pragma unroll
      for (int m = 0; m < HD16; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) *cell(warp, 2 * t4 + (i & 1), m * 16 + g + (i >> 1) * 8) = out[j][m][i];
      consumers_sync();
#pragma unroll 1
      for (unsigned i = tid; i < 8 * (kDim / 4); i += kConsumers) {
        // columns side by side for a row of outputs, rows side by side for sums that are kept
        const unsigned r8 = own_only ? i % 8 : i / (kDim / 4), c = (own_only ? i / 8 : i % (kDim / 4)) * 4, r = j * 8 + r8;
        const float peak = fmaxf(fmaxf(warp_max_of[0][r], warp_max_of[1][r]), fmaxf(warp_max_of[2][r], warp_max_of[3][r]));
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float weight = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float by = peak == -INFINITY ? 0.f : exp2_of(warp_max_of[w][r] - peak);
          const float4 part = *reinterpret_cast<const float4*>(cell(w, r8, c));
          v.x += part.x * by; v.y += part.y * by; v.z += part.z * by; v.w += part.w * by;
          weight += warp_sum_of[w][r] * by;
        }
        if (r < rows) {
          if (whole_item) {
            leave(r, c, v, peak, weight);
          } else {
            *reinterpret_cast<float4*>(parts.sum(blockIdx.x, slot, r) + c) = v;
            if (c == 0) *reinterpret_cast<float2*>(parts.end(blockIdx.x, slot, r)) = make_float2(peak, weight);
          }
        }
      }
      consumers_sync();
    }
    if (whole_item) return;

    // ---- an item of several CTAs: the last of them to arrive adds the parts, in order ----
    const unsigned first_cta = item_first / run.per, last_cta = (item_first + it.seen.count - 1) / run.per;
    if (tid == 0) {
      __threadfence();
      last_flag = atomicAdd(&counters[first_cta], 1u) == last_cta - first_cta;
      __threadfence();
    }
    consumers_sync();
    if (!last_flag) return;
#pragma unroll 1
    for (unsigned i = tid; i < rows * (kDim / 4); i += 2 * kConsumers) {      // two places a thread, the loads of four parts side by side
      constexpr unsigned kBatch = 4;
      float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
      float peak[2] = {-INFINITY, -INFINITY}, weight[2] = {0.f, 0.f};
      unsigned r[2], c[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const unsigned place = min(i + e * kConsumers, rows * (kDim / 4) - 1);
        r[e] = place / (kDim / 4);
        c[e] = (place % (kDim / 4)) * 4;
      }
#pragma unroll 1
      for (unsigned a0 = first_cta; a0 <= last_cta; a0 += kBatch) {
        float2 ends[2][kBatch];
        float4 sums[2][kBatch];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (unsigned b = 0; b < kBatch; ++b) {
            const unsigned a = min(a0 + b, last_cta);
            ends[e][b] = __ldcg(reinterpret_cast<const float2*>(parts.end(a, a == first_cta, r[e])));
            sums[e][b] = __ldcg(reinterpret_cast<const float4*>(parts.sum(a, a == first_cta, r[e]) + c[e]));
          }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (unsigned b = 0; b < kBatch; ++b) {
            if (a0 + b > last_cta) continue;
            const float next = fmaxf(peak[e], ends[e][b].x);
            const float before = next == -INFINITY ? 0.f : exp2_of(peak[e] - next), by = next == -INFINITY ? 0.f : exp2_of(ends[e][b].x - next);
            v[e].x = v[e].x * before + sums[e][b].x * by;
            v[e].y = v[e].y * before + sums[e][b].y * by;
            v[e].z = v[e].z * before + sums[e][b].z * by;
            v[e].w = v[e].w * before + sums[e][b].w * by;
            weight[e] = weight[e] * before + ends[e][b].y * by;
            peak[e] = next;
          }
      }
      leave(r[0], c[0], v[0], peak[0], weight[0]);
      if (i + kConsumers < rows * (kDim / 4)) leave(r[1], c[1], v[1], peak[1], weight[1]);
    }
    if (tid == 0) counters[first_cta] = 0;               // as the next launch expects it
  });
}

}  // namespace few

// grid: any number of CTAs that `scratch` has room for, block = 160, dynamic shared memory = stages * 256 * head_dim + 128 * head_dim + 128.
// counters: one word per CTA, zero between launches.  own_only: sums, maxima and
// weights to own_sums and own_ends instead of o (prefix attention adds the prefix to them).
#define AGI_PAGED_FEW(NAME, HD16, N, PER_SM)                                                                                          \
  extern "C" __global__ void __launch_bounds__(few::kThreads, PER_SM)                                                                 \
  NAME(const bf16* q, bf16* o, const bf16* k_pool, const bf16* v_pool, const int* starts, const int* lengths, const int* table,       \
       float* own_sums, float* own_ends, float* scratch, unsigned* counters, unsigned* status, unsigned rows, unsigned sequences,     \
       unsigned pages, unsigned page, unsigned width, unsigned q_heads, unsigned kv_heads, unsigned q_stride, unsigned o_stride,      \
       unsigned window, unsigned sinks, float scale_log2, unsigned stages, unsigned own_only) {                       \
    const paged::Batch batch{starts, lengths, table, status, rows, sequences, pages, page, width};                                    \
    few::attention_body<HD16, N>(q, o, k_pool, v_pool, batch, own_sums, own_ends, scratch, counters, q_heads, kv_heads, q_stride,     \
                                 o_stride, window, sinks, scale_log2, stages, own_only);                                       \
  }
AGI_PAGED_FEW(agi_paged_few_bf16_d64_r8, 4, 1, 2)
AGI_PAGED_FEW(agi_paged_few_bf16_d64_r16, 4, 2, 2)
AGI_PAGED_FEW(agi_paged_few_bf16_d64_r32, 4, 4, 2)
AGI_PAGED_FEW(agi_paged_few_bf16_d128_r8, 8, 1, 2)
AGI_PAGED_FEW(agi_paged_few_bf16_d128_r16, 8, 2, 2)
AGI_PAGED_FEW(agi_paged_few_bf16_d128_r32, 8, 4, 1)
#undef AGI_PAGED_FEW
