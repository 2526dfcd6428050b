// Pages of a cache in 8 bits brought back as pages of bf16: x = code * scale, exact (see paged.cuh).
//
// Bound by memory: head_dim + 2 bytes are read and 2 head_dim written for a token, key head and pool.  Only pages are read that hold a
// token which some row of the batch sees; page i of sequence b goes to page b * width + i of the pools behind, and `table_out` says so to
// the launches that read them (a page outside the pool is left out and named so that they leave it out too).  With kByPage a page keeps its
// number in the pools behind, and the batch's own table says where it is: for tables with far more places than the pool has pages (sequences
// that share the page then write the same bytes to the same place).  Pages of the batch
// form one line, found by every block as in the attention kernels, of which a warp takes 16 tokens of a page and head at a time: its
// keys and values are up to sixteen 8-byte loads a lane, asked for before the first of them is used.  Eight codes are one 16-byte store,
// so that a warp's store fills whole lines (with 16 codes and two stores of every other 16 bytes 527 MB took 290 us).
//
// Measured: a pass of `read_long` of perf/more_operators.py (527 MB) 121 us, 4.4 TB/s of the measured 6.55; `read_window` 10, most of it the call.
// Counters of 64 sequences of 8000 tokens on 4 heads (1.58 GB): 294 us, DRAM 5.2 TB/s, issue slots 44 %, load and store 53 %, stalls on loads.
#pragma once

#include "paged.cuh"

namespace reading {

using namespace paged;

constexpr unsigned kThreads = 256, kTokens = 16, kMaxSequences = 4096;
enum Flag : unsigned {
  kFreshOnly = 1,      // sequences without new tokens are left out
  kNoStarts = 2,       // `starts` is not there: no sequence has new tokens
  kByPage = 4,         // pages keep their numbers, `table_out` is not written
};

// The pages of a sequence that hold a visible token: [0, sink) and [window, end).
struct Seen {
  unsigned sink, window, count, length;
};

// Eight codes times a scale.
__device__ __forceinline__ Bf16x8 widen(const uint2& codes, float scale) {
  Bf16x8 to;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 pair(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((i < 2 ? codes.x : codes.y) >> (16 * (i & 1))), __NV_E4M3));
    const float2 f = __half22float2(pair);
    to.v[i] = __floats2bfloat162_rn(f.x * scale, f.y * scale);
  }
  return to;
}

}  // namespace reading

// grid: any number of blocks, block = 256.  At most 4096 sequences; head_dim 64 or 128; page a power of two from 16 to 128.
extern "C" __global__ void __launch_bounds__(reading::kThreads)
agi_kv_read_e4m3(const unsigned char* k_pool, const unsigned char* v_pool, const bf16* k_scale, const bf16* v_scale, const int* starts,
                 const int* lengths, const int* table, bf16* k_out, bf16* v_out, int* table_out, unsigned* status, unsigned rows,
                 unsigned sequences, unsigned pages, unsigned page, unsigned width, unsigned kv_heads, unsigned head_dim, unsigned window,
                 unsigned sinks, unsigned flags) {
  using namespace reading;
  __shared__ unsigned begins[kMaxSequences + 1], of_warp[kThreads / 32];
  const unsigned tid = threadIdx.x, lane = tid & 31, page_shift = 31 - __clz(page);
  const Batch batch{starts, lengths, table, status, rows, sequences, pages, page, width};
  grid_dependency_wait();
  if (!(aligned16(k_pool) && aligned16(v_pool) && aligned16(k_scale) && aligned16(v_scale) && aligned16(k_out) && aligned16(v_out))) {
    if (tid == 0) report(status, kMisaligned);
    return;
  }
  auto claimed = [&](unsigned seq) { return flags & kNoStarts ? Claim{0, 0, lengths[seq]} : claim_of(batch, seq); };
  auto seen_of = [&](const Claim& claim) {
    const Span span = span_of(batch, claim);
    Seen s{0, 0, 0, span.length};
    if (span.length == 0 || ((flags & kFreshOnly) && span.fresh == 0)) return s;
    const unsigned start = window == 0 ? 0u : unsigned(max(span.first - int(window) + 1, 0)), end = (span.length + page - 1) >> page_shift;
    s.sink = (min(sinks, start) + page - 1) >> page_shift;
    s.sink = min(s.sink, end);
    s.window = start < span.length ? max(start >> page_shift, s.sink) : end;      // the next row may see no token that is there
    s.count = s.sink + (end > s.window ? end - s.window : 0u);
    return s;
  };
  unsigned below = 0;
  int ordered = 1;
#pragma unroll 1
  for (unsigned i0 = 0; i0 < sequences; i0 += kThreads) {
    const unsigned i = i0 + tid;
    unsigned mine = 0, all;
    if (i < sequences) {
      const Claim claim = claimed(i);
      if (in_order(batch, claim)) mine = seen_of(claim).count;
      else ordered = 0;
    }
    const unsigned first = below + sum_before<kThreads>(mine, of_warp, &all);
    if (i < sequences) begins[i] = first;
    below += all;
    ordered = __syncthreads_and(ordered);
  }
  if (!ordered) return;

  const unsigned pieces = page / kTokens, lane_shift = head_dim == 128 ? 4 : 3, blocks = head_dim / 64;       // lanes of a token: eight codes each
  const unsigned step = 32 >> lane_shift, loads = kTokens / step;        // tokens that the lanes cover at a time
  const unsigned items = below * kv_heads * pieces, stride = gridDim.x * (kThreads / 32);
  const unsigned eight = lane & ((1u << lane_shift) - 1), lane_token = lane >> lane_shift;
#pragma unroll 1
  for (unsigned item = blockIdx.x * (kThreads / 32) + (tid >> 5); item < items; item += stride) {
    const unsigned piece = item & (pieces - 1), rest = item / pieces, line = rest / kv_heads, head = rest - line * kv_heads;
    unsigned seq = 0;      // the last sequence that begins at or before the page
    for (unsigned above = sequences; above - seq > 1;) {
      const unsigned middle = (seq + above) / 2;
      if (begins[middle] <= line) seq = middle; else above = middle;
    }
    const Seen seen = seen_of(claimed(seq));
    const unsigned at = line - begins[seq], slot = at < seen.sink ? at : seen.window + (at - seen.sink), to = seq * width + slot;
    const unsigned page_id = unsigned(table[to]);
    if (piece == 0 && head == 0 && lane == 0) {
      if (!(flags & kByPage)) table_out[to] = page_id < pages ? int(to) : -1;
      if (page_id >= pages) report(status, kBadPage);
    }
    if (page_id >= pages) continue;
    const unsigned held = min(seen.length - slot * page, page);       // tokens of the page
    const size_t from = block_offset(page_id, kv_heads, head, 1, 0, page), to_row = block_offset(flags & kByPage ? page_id : to, kv_heads, head, blocks, 0, page);
    uint2 codes[2][8];
    float scale[2][8];
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
      const unsigned token = piece * kTokens + lane_token + i * step;
      if (i < loads && token < held) {
        codes[0][i] = reinterpret_cast<const uint2*>(k_pool + (from + token) * head_dim)[eight];
        codes[1][i] = reinterpret_cast<const uint2*>(v_pool + (from + token) * head_dim)[eight];
        scale[0][i] = __bfloat162float(k_scale[from + token]);
        scale[1][i] = __bfloat162float(v_scale[from + token]);
      }
    }
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
      const unsigned token = piece * kTokens + lane_token + i * step;
      if (i >= loads || token >= held) continue;
      const unsigned chunk = code_chunk(eight >> 1, token, head_dim);       // exchanging chunks is its own inverse
      const size_t to_eight = (to_row + size_t(chunk / 4) * page + token) * 64 + (((chunk & 3) * 2 + (eight & 1)) ^ (token & 7)) * 8;
      *reinterpret_cast<Bf16x8*>(k_out + to_eight) = widen(codes[0][i], scale[0][i]);
      *reinterpret_cast<Bf16x8*>(v_out + to_eight) = widen(codes[1][i], scale[1][i]);
    }
  }
}
