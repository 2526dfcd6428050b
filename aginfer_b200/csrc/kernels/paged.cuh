// Paged K/V cache: what its kernels share, and the kernel that appends a step's keys and values to it.
//
// A cache is two pools [pages][kv_heads][head_dim / 64][page][64] of bf16, one of keys and one of values; the 16-byte chunk c of
// a token's 64-column block lies at position c ^ (token & 7).  A run of consecutive tokens of one page, head and block is
// therefore one contiguous run of memory and the byte image of a 128B-swizzled shared-memory tile: one bulk copy brings it in,
// and both ldmatrix and tcgen05.mma read it without bank conflicts.
//
// A batch is `sequences` of them: rows starts[b] .. starts[b + 1) are the new tokens of sequence b, lengths[b] the tokens that it
// holds once they are in, table[b * width + i] the page of its tokens [i * page, (i + 1) * page).  Row r of sequence b stands at
// index lengths[b] - (starts[b + 1] - r) of its sequence; a row at a negative index is not appended and sees no key.
//
// starts, lengths and table are read on the device, so that one launch serves every step of a replayed graph.  What they must not
// say is checked here: a page outside the pool or an index outside the table leaves a code in the status word and nothing is
// read or written there.
#pragma once

#include "common.cuh"

namespace paged {

enum Status : unsigned {
  kBadPage = 0x400,      // a table names a page outside the pool
  kBadLength = 0x500,    // a sequence is longer than its row of the table
  kMisaligned = 0x600,   // a tensor that is moved in 16-byte pieces does not start at a multiple of 16 bytes
};

__device__ __forceinline__ void report(unsigned* status, unsigned code) { atomicCAS(status, 0u, code); }

// The sequence that holds a row: the number of sequences that end at or before it (`sequences` where none holds it).
// Called by whole warps.
__device__ __forceinline__ unsigned sequence_of(const int* starts, unsigned sequences, unsigned row) {
  unsigned before = 0;
  for (unsigned i = threadIdx.x & 31; i < sequences; i += 32) before += *(starts + i + 1) <= int(row) ? 1u : 0u;
  return __reduce_add_sync(0xffffffffu, before);
}

// The index of a row of sequence `seq` in it; whatever the tensors hold, the difference wraps and does not trap.
__device__ __forceinline__ int index_of(const int* starts, const int* lengths, unsigned seq, unsigned row) {
  return int(unsigned(*(lengths + seq)) - (unsigned(*(starts + seq + 1)) - row));
}

// 2^x, zero for minus infinity; relative error 2^-22.
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<size_t>(p) & 15) == 0; }

// Offset, in 64-column rows, of token t of a page's block.
__device__ __forceinline__ size_t block_offset(unsigned page_id, unsigned kv_heads, unsigned head, unsigned blocks, unsigned block,
                                               unsigned page) {
  return ((size_t(page_id) * kv_heads + head) * blocks + block) * page;
}

// The batch as the attention kernels take it.
struct Batch {
  const int *starts, *lengths, *table;
  unsigned* status;
  unsigned rows, sequences, pages, page, width;
};

// A sequence of it: its first row, its new tokens, the index of the first of them (negative: in front of the sequence) and the
// tokens that it holds; a length beyond the table is cut to it.
struct Span {
  unsigned row, fresh;
  int first;
  unsigned length;
};
__device__ __forceinline__ Span span_of(const Batch& b, unsigned seq) {
  const int from = b.starts[seq], to = b.starts[seq + 1], length = b.lengths[seq];
  Span s;
  s.row = unsigned(from);
  s.fresh = unsigned(to - from);
  s.length = min(unsigned(max(length, 0)), b.width * b.page);
  s.first = int(s.length) - int(s.fresh);
  return s;
}
// What a launch checks of every sequence before it uses any: rows in order and a length that the table has room for.  Rows out of
// order leave the whole launch without work, so that rows add up to no more than there are.
__device__ __forceinline__ bool in_order(const Batch& b, unsigned seq) {
  const int from = b.starts[seq], to = b.starts[seq + 1];
  const bool ordered = from >= 0 && to >= from && unsigned(to) <= b.rows;
  if (!ordered || b.lengths[seq] > int(b.width * b.page)) report(b.status, kBadLength);
  return ordered;
}

// Sum over the threads in front of this one, and over all.  `of_warp`: a word per warp, used once a kernel.
template <unsigned kThreads>
__device__ __forceinline__ unsigned sum_before(unsigned mine, unsigned* of_warp, unsigned* all) {
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned below = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned other = __shfl_up_sync(0xffffffffu, below, d);
    if (lane >= unsigned(d)) below += other;
  }
  if (lane == 31) of_warp[warp] = below;
  __syncthreads();
  below -= mine;
  unsigned total = 0;
#pragma unroll
  for (unsigned w = 0; w < kThreads / 32; ++w) {
    if (w < warp) below += of_warp[w];
    total += of_warp[w];
  }
  *all = total;
  return below;
}

// Rows of a block are (token, query head of the key head) pairs, heads fastest: row i of one that begins at row `first` of its sequence.
// The quotient by a reciprocal is exact: i + group stays far below 2^20.
struct Rows {
  unsigned token, head, group;
  float reciprocal;
  __device__ __forceinline__ Rows(unsigned first, unsigned group_) : token(first / group_), head(first % group_), group(group_), reciprocal(1.f / float(group_)) {}
  __device__ __forceinline__ void at(unsigned i, unsigned& token_of, unsigned& head_of) const {
    const unsigned t = __float2uint_rz((float(head + i) + 0.5f) * reciprocal);
    token_of = token + t;
    head_of = head + i - t * group;
  }
};

// The key tiles that rows at indices [low, high] see: those of the first `sinks` tokens that lie before the window of the first
// row, then those from that window to the last row.  At least one, which may hold no visible key: it makes a row that sees
// nothing zero.
struct Visible {
  unsigned end, start, sink_end;            // keys [0, sink_end) and [start, end)
  unsigned sink_tiles, window_tile, count;
  __device__ __forceinline__ unsigned tile(unsigned i) const { return i < sink_tiles ? i : window_tile + (i - sink_tiles); }
};
template <unsigned kTile>
__device__ __forceinline__ Visible visible_of(int low, int high, unsigned length, unsigned window, unsigned sinks) {
  Visible v;
  v.end = min(unsigned(max(high + 1, 0)), length);
  v.start = window == 0 ? 0u : unsigned(max(low - int(window) + 1, 0));
  v.sink_end = min(sinks, v.start);
  v.sink_tiles = (v.sink_end + kTile - 1) / kTile;
  v.window_tile = max(v.start / kTile, v.sink_tiles);
  const unsigned tiles = (v.end + kTile - 1) / kTile;
  v.count = max(v.sink_tiles + (tiles > v.window_tile ? tiles - v.window_tile : 0u), 1u);
  return v;
}
__device__ __forceinline__ bool sees(int index, unsigned key, unsigned window, unsigned sinks) {
  const int back = index - int(key);
  return back >= 0 && (window == 0 || unsigned(back) < window || key < sinks);
}

}  // namespace paged

// Queries and keys of a step's new tokens turned by their positions (half-split pairs, see rope.cuh), queries written to `q_out`,
// keys and values to their pages.  Bound by memory: every row is read and written once.  Angles are formed in 64 bits: at
// position 100000 a product in 32 bits would already be off by more than a bf16 rounding of the result; the sixty-four frequencies
// are computed once a block and kept for its rows.
// A block takes rows blockIdx.x, + gridDim.x, ...; a thread turns eight pairs of a head at a time (two 16-byte vectors), and
// requests them before it computes the angles.
// s0 says where a position comes from (below).  log2_theta + log2_theta_rest: log2 of theta in two pieces.
// block = 128.  head_dim 64 or 128, strides multiples of 8.
constexpr unsigned kPositionsFromCache = 0xffffffffu;   // s0: the index in the sequence, plus *offset where has_offset
constexpr unsigned kPositionsOneAxis = 0xfffffffeu;     // s0: pos[row]; otherwise pos[3][rows] with sections s0, s1, rest
extern "C" __global__ void __launch_bounds__(128)
agi_kv_append_bf16(const bf16* q, const bf16* k, const bf16* v, unsigned k_column, unsigned v_column, bf16* q_out, bf16* k_pool,
                   bf16* v_pool, const int* starts, const int* lengths, const int* table, const int* pos, const int* offset,
                   unsigned* status, unsigned rows, unsigned sequences, unsigned pages, unsigned page, unsigned width,
                   unsigned q_heads, unsigned kv_heads, unsigned head_dim, unsigned q_stride, unsigned kv_stride,
                   unsigned out_stride, float log2_theta, float log2_theta_rest, unsigned s0, unsigned s1, unsigned ladder,
                   unsigned has_offset) {
  __shared__ __align__(16) float cosine[64], sine[64];
  grid_dependency_wait();
  const unsigned half = head_dim / 2, vecs = half / 8, turned = (q_heads + kv_heads) * vecs;
  const unsigned blocks = head_dim / 64, copied = kv_heads * head_dim / 8;
  k += k_column;
  v += v_column;
  if (!(paged::aligned16(q) && paged::aligned16(k) && paged::aligned16(v) && paged::aligned16(q_out) && paged::aligned16(k_pool) &&
        paged::aligned16(v_pool))) {
    if (threadIdx.x == 0) paged::report(status, paged::kMisaligned);
    return;
  }
  const unsigned pair = threadIdx.x;
  // turns per position of this thread's pair
  double frequency = 0.;
  if (pair < half)
    frequency = exp2(-(double(log2_theta) + double(log2_theta_rest)) * (double(pair % ladder) / double(ladder))) * 0.15915494309189534;
  for (unsigned row = blockIdx.x; row < rows; row += gridDim.x) {
    const unsigned seq = paged::sequence_of(starts, sequences, row);
    if (seq >= sequences) continue;      // the same for the whole block
    const int index = paged::index_of(starts, lengths, seq, row);
    unsigned page_id = 0;
    bool stored = index >= 0;
    if (stored) {
      if (unsigned(index) / page >= width) {
        stored = false;
        if (threadIdx.x == 0) paged::report(status, paged::kBadLength);
      } else {
        page_id = unsigned(*(table + size_t(seq) * width + unsigned(index) / page));
        if (page_id >= pages) {
          stored = false;
          if (threadIdx.x == 0) paged::report(status, paged::kBadPage);
        }
      }
    }
    const unsigned token = unsigned(index) % page;
    const bf16* const q_row = q + size_t(row) * q_stride;
    const bf16* const k_row = k + size_t(row) * kv_stride;
    __syncthreads();      // the angles of the row before are no longer needed
    if (pair < half) {
      int at;
      if (s0 == kPositionsFromCache) at = int(unsigned(index) + (has_offset ? unsigned(*offset) : 0u));
      else if (s0 == kPositionsOneAxis) at = *(pos + row);
      else at = *(pos + size_t(pair < s0 ? 0u : pair < s0 + s1 ? 1u : 2u) * rows + row);
      const double turns = double(at) * frequency;
      sincospif(2.f * float(turns - rint(turns)), &sine[pair], &cosine[pair]);
    }
    __syncthreads();
    for (unsigned item = threadIdx.x; item < turned; item += 128) {
      const unsigned head = item / vecs, c = item - head * vecs;
      const bf16* from = (head < q_heads ? q_row + head * head_dim : k_row + (head - q_heads) * head_dim) + c * 8;
      float a[8], b[8], x[8], y[8];
      unpack8(*reinterpret_cast<const Bf16x8*>(from), a);
      unpack8(*reinterpret_cast<const Bf16x8*>(from + half), b);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float co = cosine[c * 8 + j], si = sine[c * 8 + j];
        x[j] = a[j] * co - b[j] * si;
        y[j] = b[j] * co + a[j] * si;
      }
      if (head < q_heads) {
        bf16* to = q_out + size_t(row) * out_stride + head * head_dim + c * 8;
        *reinterpret_cast<Bf16x8*>(to) = pack8(x);
        *reinterpret_cast<Bf16x8*>(to + half) = pack8(y);
      } else if (stored) {
        // chunk c of the head's first half, chunk c + vecs of the whole row: columns of one block (64 wide) or of two
        const unsigned lo = c, hi = c + vecs;
        bf16* first = k_pool + (paged::block_offset(page_id, kv_heads, head - q_heads, blocks, lo / 8, page) + token) * 64;
        bf16* second = k_pool + (paged::block_offset(page_id, kv_heads, head - q_heads, blocks, hi / 8, page) + token) * 64;
        *reinterpret_cast<Bf16x8*>(first + (((lo & 7) ^ (token & 7)) * 8)) = pack8(x);
        *reinterpret_cast<Bf16x8*>(second + (((hi & 7) ^ (token & 7)) * 8)) = pack8(y);
      }
    }
    if (stored)
      for (unsigned item = threadIdx.x; item < copied; item += 128) {
        const unsigned head = item / (blocks * 8), c = item % (blocks * 8);
        bf16* to = v_pool + (paged::block_offset(page_id, kv_heads, head, blocks, c / 8, page) + token) * 64;
        *reinterpret_cast<uint4*>(to + (((c & 7) ^ (token & 7)) * 8)) =
            *reinterpret_cast<const uint4*>(v + size_t(row) * kv_stride + head * head_dim + c * 8);
      }
  }
}
