// Attention over a paged cache for few rows a sequence and key head (a decoding step: one token, a few drafted ones):
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),  one pass over the keys with a running maximum m and sum.
//
// Bound by memory: a key and a value are 4 head_dim bytes and meet at most 32 rows.  So the unit of work is a tile of 64 keys of
// one sequence and key head, all units of the batch in one line, and every CTA takes an equal run of it, however unequal the
// sequences are: sequences and heads that a run cuts leave unnormalised sums, their maximum and weight in scratch, and the last
// CTA of such an item to arrive adds them in order (nobody waits for another CTA; sums do not depend on who arrives when).
//
// A CTA: one loading warp that brings tiles in by bulk copies, a copy per page (or the part of it in the tile) and 64-column
// block, into a ring; four warps that share a tile's keys, 16 each, with maximum, sum and outputs of their own until the item ends.
// The rows of the query heads that share a key head are the rows of one mma.sync tile (m16n8k16; twice that with kM = 2).  Keys
// and values lie in shared memory as they lie in the pool, swizzled, so ldmatrix reads them without bank conflicts.
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
constexpr unsigned kMergeColumns = 32;      // columns of the outputs that the four warps exchange at a time

// How many units one sequence is: its key heads x row blocks x key tiles.
struct Items {
  Span span;
  Visible seen;
  unsigned blocks, units;             // row blocks of a key head; units of the sequence
};
template <unsigned kRows>
__device__ __forceinline__ Items items_of(const Batch& batch, unsigned seq, unsigned group, unsigned kv_heads, unsigned window, unsigned sinks) {
  Items it;
  it.span = span_of(batch, seq);
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

template <int HD16, int kM>
__device__ __forceinline__ void attention_body(const bf16* q, bf16* o, const bf16* k_pool, const bf16* v_pool, const Batch& batch, float* own_sums,
                                               float* own_ends, float* scratch, unsigned* counters, unsigned q_heads, unsigned kv_heads, unsigned q_stride, unsigned o_stride,
                                               unsigned window, unsigned sinks, float scale_log2, unsigned stages, unsigned least,
                                               unsigned own_only) {
  constexpr unsigned kDim = HD16 * 16, kBlocks = kDim / 64, kRows = 16 * kM;
  constexpr unsigned kTileBytes = kKeys * kDim * 2, kStageBytes = 2 * kTileBytes, kBlockBytes = kKeys * 128;
  constexpr unsigned kMaxStages = 8;
  extern __shared__ unsigned char dynamic_smem[];
  __shared__ __align__(8) unsigned long long full_bar[kMaxStages], empty_bar[kMaxStages];
  __shared__ unsigned run_base[kThreads / 32], run_seq, run_first, gave_up, last_flag;
  __shared__ float warp_max_of[4][kRows], warp_sum_of[4][kRows];
  const unsigned tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned ring = (tc::smem_u32(dynamic_smem) + 1023u) & ~1023u;
  float* const exchange = reinterpret_cast<float*>(dynamic_smem + (ring - tc::smem_u32(dynamic_smem)) + stages * kStageBytes);   // [4][16][32]
  const unsigned group = q_heads / kv_heads;

  if (tid == 0) {
    for (unsigned s = 0; s < stages; ++s) {
      tc::mbar_init(&full_bar[s], 1);
      tc::mbar_init(&empty_bar[s], 4);
    }
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  grid_dependency_wait();
  if (!(aligned16(q) && aligned16(o) && aligned16(k_pool) && aligned16(v_pool))) {
    if (tid == 0) report(batch.status, kMisaligned);
    return;
  }

  // ---- this CTA's run: units [from, to) of all, and the sequence that holds the first of them ----
  unsigned mine = 0, total;
  bool ordered = true;
  const unsigned share = (batch.sequences + kThreads - 1) / kThreads, seq0 = min(tid * share, batch.sequences), seq1 = min(seq0 + share, batch.sequences);
#pragma unroll 1
  for (unsigned i = seq0; i < seq1; ++i) {
    ordered = in_order(batch, i) && ordered;
    mine += items_of<kRows>(batch, i, group, kv_heads, window, sinks).units;
  }
  unsigned below = sum_before<kThreads>(mine, run_base, &total);
  const unsigned per = max((total + gridDim.x - 1) / gridDim.x, least), from = min(per * blockIdx.x, total), to = min(from + per, total);
  if (from < to && from >= below && from < below + mine) {
#pragma unroll 1
    for (unsigned i = seq0; i < seq1; ++i) {
      const unsigned units = items_of<kRows>(batch, i, group, kv_heads, window, sinks).units;
      if (from < below + units) {
        run_seq = i;
        run_first = below;
        break;
      }
      below += units;
    }
  }
  if (__syncthreads_or(!ordered) || from >= to) return;

  // Walks the run item by item: f(sequence, key head, row block, its items, first tile, last tile + 1, first unit of the item).
  auto walk = [&](auto&& f) {
    unsigned seq = run_seq, first = run_first, unit = from;
#pragma unroll 1
    while (unit < to && seq < batch.sequences) {
      const Items it = items_of<kRows>(batch, seq, group, kv_heads, window, sinks);
#pragma unroll 1
      while (unit < to && unit < first + it.units) {
        const unsigned at = (unit - first) / it.seen.count;                // which item of the sequence
        const unsigned item_first = first + at * it.seen.count, begin = unit - item_first, end = min(it.seen.count, begin + (to - unit));
        const unsigned head = at / it.blocks;
        f(seq, head, at - head * it.blocks, it, begin, end, item_first);
        unit += end - begin;
      }
      first += it.units;
      ++seq;
    }
  };

  if (warp == 4) {
    // ---- loading warp: a lane per piece (keys or values, 64-column block, page or part of one) of a tile ----
    const unsigned run = min(batch.page, kKeys), pieces = kKeys / run;
    const bool values = lane >= pieces * kBlocks;
    const unsigned block = (lane / pieces) % kBlocks, piece = lane % pieces;
    const bool live = lane < 2 * kBlocks * pieces;
    const unsigned to_slot = (values ? kTileBytes : 0u) + block * kBlockBytes + piece * run * 128;
    const bf16* const pool = values ? v_pool : k_pool;
    unsigned s = 0, phase = 1;
    walk([&](unsigned seq, unsigned head, unsigned, const Items& it, unsigned begin, unsigned end, unsigned) {
      const int* const pages_of = batch.table + size_t(seq) * batch.width;
      // tokens of a tile that this lane brings in, and the page that holds them
      auto tokens_of = [&](unsigned t) {
        const unsigned token = it.seen.tile(t) * kKeys + piece * run;
        const bool wanted = live && token < it.seen.end && (token < it.seen.sink_end || token + run > it.seen.start);
        return wanted ? min(run, it.seen.end - token) : 0u;
      };
      auto page_of = [&](unsigned t) { return unsigned(pages_of[(it.seen.tile(t) * kKeys + piece * run) / batch.page]); };
      unsigned count = tokens_of(begin), page_id = count ? page_of(begin) : 0u;
      for (unsigned t = begin; t < end; ++t) {
        if (page_id >= batch.pages) {
          report(batch.status, kBadPage);
          count = 0;
        }
        const unsigned token = it.seen.tile(t) * kKeys + piece * run;
        const bf16* const from_page = pool + (block_offset(page_id, kv_heads, head, kBlocks, block, batch.page) + token % batch.page) * 64;
        const unsigned bytes = count * 128, all = __reduce_add_sync(0xffffffffu, bytes);
        unsigned next_count = 0, next_page = 0;      // the page numbers of the tile behind it, while this one's slot is awaited
        if (t + 1 < end) {
          next_count = tokens_of(t + 1);
          if (next_count) next_page = page_of(t + 1);
        }
        if (lane == 0) {
          if (!*(volatile unsigned*)&gave_up && !tc::mbar_wait(&empty_bar[s], phase, batch.status, tc::kTimeoutEmpty | s)) *(volatile unsigned*)&gave_up = 1;
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
    // Q fragments: row r of the item is token r / group, query head head * group + r % group
    unsigned qa[kM][HD16][4];
    int index[kM][2];
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned r = m * 16 + g + h * 8;
        unsigned token, sub;
        pairs.at(r, token, sub);
        const bool live = r < rows;
        index[m][h] = live ? span.first + int(token) : -1;
        const bf16* from_row = q + size_t(span.row + token) * q_stride + (head * group + sub) * kDim + 2 * t4;
#pragma unroll
        for (int ks = 0; ks < HD16; ++ks) {
          qa[m][ks][h] = live ? __ldcg(reinterpret_cast<const unsigned*>(from_row + ks * 16)) : 0u;
          qa[m][ks][h + 2] = live ? __ldcg(reinterpret_cast<const unsigned*>(from_row + ks * 16 + 8)) : 0u;
        }
      }
    float top[kM][2], sum[kM][2], out[kM][2 * HD16][4];
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      top[m][0] = top[m][1] = -INFINITY;
      sum[m][0] = sum[m][1] = 0.f;
#pragma unroll
      for (int c = 0; c < 2 * HD16; ++c) out[m][c][0] = out[m][c][1] = out[m][c][2] = out[m][c][3] = 0.f;
    }
    const int low = span.first + int(pairs.token);                 // the item's first row
    for (unsigned t = begin; t < end; ++t) {
      if (!*(volatile unsigned*)&gave_up && !tc::mbar_wait(&full_bar[s], phase, batch.status, tc::kTimeoutFull | s)) *(volatile unsigned*)&gave_up = 1;
      __syncwarp();
      const unsigned key0 = it.seen.tile(t) * kKeys + warp * 16, slot = ring + s * kStageBytes;
      if (key0 < it.seen.end) {
        // scores of 16 keys: lanes 0-7 | 8-15 | 16-23 | 24-31 address the 8 x 8 blocks (keys 0-7, chunk c) | (0-7, c + 1) | (8-15, c) | (8-15, c + 1)
        float score[kM][2][4];
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n) score[m][n][0] = score[m][n][1] = score[m][n][2] = score[m][n][3] = 0.f;
        const unsigned k_row = slot + (warp * 16 + (lane >> 4) * 8 + (lane & 7)) * 128;
#pragma unroll
        for (int ks = 0; ks < HD16; ++ks) {
          unsigned b0, b1, b2, b3;
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                       : "=r"(b0), "=r"(b1), "=r"(b2), "=r"(b3)
                       : "r"(k_row + (ks / 4) * kBlockBytes + ((((ks % 4) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4)));
#pragma unroll
          for (int m = 0; m < kM; ++m) {
            skinny_mma_bf16(score[m][0], qa[m][ks][0], qa[m][ks][1], qa[m][ks][2], qa[m][ks][3], b0, b1);
            skinny_mma_bf16(score[m][1], qa[m][ks][0], qa[m][ks][1], qa[m][ks][2], qa[m][ks][3], b2, b3);
          }
        }
        // does every row see all of these keys?
        const bool whole = int(key0) + 15 <= low && key0 + 16 <= it.seen.end && rows == kRows &&
                           (window == 0 || int(key0) > int(it.span.length) - 1 - int(window));
        unsigned pa[kM][4];
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const unsigned key = key0 + (i >> 1) * 8 + 2 * t4 + (i & 1);
              const float v = score[m][i >> 1][2 * h + (i & 1)] * scale_log2;
              x[i] = whole || (key < it.seen.end && sees(index[m][h], key, window, sinks)) ? v : -INFINITY;
            }
            float peak = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
            peak = fmaxf(peak, top[m][h]);
            const float base = peak == -INFINITY ? 0.f : peak, old = exp2_of(top[m][h] - base);
            top[m][h] = peak;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = exp2_of(x[i] - base);
            sum[m][h] = sum[m][h] * old + ((x[0] + x[1]) + (x[2] + x[3]));
#pragma unroll
            for (int c = 0; c < 2 * HD16; ++c) {
              out[m][c][2 * h] *= old;
              out[m][c][2 * h + 1] *= old;
            }
            // the scores' layout is that of P as the next product's A operand: a0 | a1 rows g | g + 8 of keys 0-7, a2 | a3 of keys 8-15
            const bf162 first = __floats2bfloat162_rn(x[0], x[1]), second = __floats2bfloat162_rn(x[2], x[3]);
            pa[m][h] = *reinterpret_cast<const unsigned*>(&first);
            pa[m][h + 2] = *reinterpret_cast<const unsigned*>(&second);
          }
        // values: keys 2 t, 2 t + 1 (and + 8) of a column; those that no row of the sequence sees are taken as zero
        unsigned keep[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned key = key0 + i * 8 + 2 * t4;
          auto held = [&](unsigned j) { return j < it.seen.end && (j >= it.seen.start || j < it.seen.sink_end); };
          keep[i] = (held(key) ? 0xffffu : 0u) | (held(key + 1) ? 0xffff0000u : 0u);
        }
        const unsigned v_row = slot + kTileBytes + (warp * 16 + (lane & 15)) * 128;
#pragma unroll
        for (int c = 0; c < HD16; ++c) {
          unsigned b0, b1, b2, b3;
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                       : "=r"(b0), "=r"(b1), "=r"(b2), "=r"(b3)
                       : "r"(v_row + (c / 4) * kBlockBytes + ((((c % 4) * 2 + (lane >> 4)) ^ (lane & 7)) << 4)));
          b0 &= keep[0];
          b1 &= keep[1];
          b2 &= keep[0];
          b3 &= keep[1];
#pragma unroll
          for (int m = 0; m < kM; ++m) {
            skinny_mma_bf16(out[m][2 * c], pa[m][0], pa[m][1], pa[m][2], pa[m][3], b0, b1);
            skinny_mma_bf16(out[m][2 * c + 1], pa[m][0], pa[m][1], pa[m][2], pa[m][3], b2, b3);
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&empty_bar[s]);
      if (++s == stages) { s = 0; phase ^= 1; }
    }

    // ---- the four warps' shares meet: maxima and weights first, then the outputs, 32 columns at a time ----
    const bool whole_item = begin == 0 && end == it.seen.count;
    const unsigned slot = begin > 0 ? 0u : 1u;
    // four columns of a row, divided, or as they are with the row's maximum and weight
    auto leave = [&](unsigned r, unsigned c, float4 v, float peak, float weight) {
      unsigned token, sub;
      pairs.at(r, token, sub);
      const unsigned row = span.row + token, q_head = head * group + sub;
      if (own_only) {
        const size_t flat = size_t(row) * q_heads + q_head;
        *reinterpret_cast<float4*>(own_sums + flat * kDim + c) = v;
        if (c == 0) *reinterpret_cast<float2*>(own_ends + flat * 2) = make_float2(peak, weight);
        return;
      }
      const float inv = weight > 0.f ? 1.f / weight : 0.f;
      const bf162 pair[2] = {__floats2bfloat162_rn(v.x * inv, v.y * inv), __floats2bfloat162_rn(v.z * inv, v.w * inv)};
      *reinterpret_cast<uint2*>(o + size_t(row) * o_stride + q_head * kDim + c) = *reinterpret_cast<const uint2*>(pair);
    };
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sum[m][h] += __shfl_xor_sync(0xffffffffu, sum[m][h], 1);
        sum[m][h] += __shfl_xor_sync(0xffffffffu, sum[m][h], 2);
        if (t4 == 0) {
          warp_max_of[warp][m * 16 + g + h * 8] = top[m][h];
          warp_sum_of[warp][m * 16 + g + h * 8] = sum[m][h];
        }
      }
    consumers_sync();
    const unsigned r16 = tid / 8, c4 = (tid % 8) * 4;      // a thread per row and four of 32 columns
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      const unsigned r = m * 16 + r16;
      const float peak = fmaxf(fmaxf(warp_max_of[0][r], warp_max_of[1][r]), fmaxf(warp_max_of[2][r], warp_max_of[3][r]));
      float by[4], weight = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        by[w] = peak == -INFINITY ? 0.f : exp2_of(warp_max_of[w][r] - peak);
        weight += warp_sum_of[w][r] * by[w];
      }
#pragma unroll
      for (unsigned c0 = 0; c0 < kDim; c0 += kMergeColumns) {
#pragma unroll
        for (unsigned n = 0; n < kMergeColumns / 8; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2*>(exchange + (warp * 16 + g + h * 8) * kMergeColumns + n * 8 + 2 * t4) =
                make_float2(out[m][c0 / 8 + n][2 * h], out[m][c0 / 8 + n][2 * h + 1]);
        consumers_sync();
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 part = *reinterpret_cast<const float4*>(exchange + (w * 16 + r16) * kMergeColumns + c4);
          v.x += part.x * by[w]; v.y += part.y * by[w]; v.z += part.z * by[w]; v.w += part.w * by[w];
        }
        if (r < rows) {
          if (whole_item) {
            leave(r, c0 + c4, v, peak, weight);
          } else {
            *reinterpret_cast<float4*>(parts.sum(blockIdx.x, slot, r) + c0 + c4) = v;
            if (c0 == 0 && c4 == 0) *reinterpret_cast<float2*>(parts.end(blockIdx.x, slot, r)) = make_float2(peak, weight);
          }
        }
        consumers_sync();
      }
    }
    if (whole_item) return;

    // ---- an item of several CTAs: the last of them to arrive adds the parts, in order ----
    const unsigned first_cta = item_first / per, last_cta = (item_first + it.seen.count - 1) / per;
    __threadfence();
    consumers_sync();
    if (tid == 0) last_flag = atomicAdd(&counters[first_cta], 1u) == last_cta - first_cta;
    consumers_sync();
    if (!last_flag) return;
    __threadfence();
    for (unsigned i = tid; i < rows * (kDim / 4); i += kConsumers) {
      const unsigned r = i / (kDim / 4), c = (i % (kDim / 4)) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float peak = -INFINITY, weight = 0.f;
      for (unsigned a = first_cta; a <= last_cta; ++a) peak = fmaxf(peak, __ldcg(parts.end(a, a == first_cta, r)));
#pragma unroll 4
      for (unsigned a = first_cta; a <= last_cta; ++a) {
        const float2 end_of = __ldcg(reinterpret_cast<const float2*>(parts.end(a, a == first_cta, r)));
        const float4 part = __ldcg(reinterpret_cast<const float4*>(parts.sum(a, a == first_cta, r) + c));
        const float f = end_of.x == -INFINITY ? 0.f : exp2_of(end_of.x - peak);
        v.x += part.x * f; v.y += part.y * f; v.z += part.z * f; v.w += part.w * f;
        weight += end_of.y * f;
      }
      leave(r, c, v, peak, weight);
    }
    if (tid == 0) counters[first_cta] = 0;               // as the next launch expects it
  });
}

}  // namespace few

// grid: any number of CTAs that `scratch` has room for, block = 160, dynamic shared memory = stages * 256 * head_dim + 8192 + 1024.
// least: units that a CTA takes at the least; counters: one word per CTA, zero between launches.  own_only: sums, maxima and
// weights to own_sums [rows][q_heads][head_dim] and own_ends [rows][q_heads][2] instead of o (prefix attention adds the prefix to them).
#define AGI_PAGED_FEW(NAME, HD16, M, PER_SM)                                                                                          \
  extern "C" __global__ void __launch_bounds__(few::kThreads, PER_SM)                                                                 \
  NAME(const bf16* q, bf16* o, const bf16* k_pool, const bf16* v_pool, const int* starts, const int* lengths, const int* table,       \
       float* own_sums, float* own_ends, float* scratch, unsigned* counters, unsigned* status, unsigned rows, unsigned sequences,     \
       unsigned pages, unsigned page, unsigned width, unsigned q_heads, unsigned kv_heads, unsigned q_stride, unsigned o_stride,      \
       unsigned window, unsigned sinks, float scale_log2, unsigned stages, unsigned least, unsigned own_only) {                       \
    const paged::Batch batch{starts, lengths, table, status, rows, sequences, pages, page, width};                                    \
    few::attention_body<HD16, M>(q, o, k_pool, v_pool, batch, own_sums, own_ends, scratch, counters, q_heads, kv_heads, q_stride,     \
                                 o_stride, window, sinks, scale_log2, stages, least, own_only);                                       \
  }
AGI_PAGED_FEW(agi_paged_few_bf16_d64_m1, 4, 1, 2)
AGI_PAGED_FEW(agi_paged_few_bf16_d64_m2, 4, 2, 1)
AGI_PAGED_FEW(agi_paged_few_bf16_d128_m1, 8, 1, 2)
AGI_PAGED_FEW(agi_paged_few_bf16_d128_m2, 8, 2, 1)
#undef AGI_PAGED_FEW
