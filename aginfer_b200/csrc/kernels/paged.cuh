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
// What the batch says of a sequence, as it stands in memory.
struct Claim {
  int from, to, length;
};
__device__ __forceinline__ Claim claim_of(const Batch& b, unsigned seq) { return Claim{b.starts[seq], b.starts[seq + 1], b.lengths[seq]}; }
__device__ __forceinline__ Span span_of(const Batch& b, const Claim& c) {
  Span s;
  s.row = unsigned(c.from);
  s.fresh = unsigned(c.to - c.from);
  s.length = min(unsigned(max(c.length, 0)), b.width * b.page);
  s.first = int(s.length) - int(s.fresh);
  return s;
}
// What a launch checks of every sequence before it uses any: rows in order and, where it reads keys, a length that the table has
// room for.  Rows out of order leave the whole launch without work, so that rows add up to no more than there are.
__device__ __forceinline__ bool rows_in_order(int from, int to, unsigned rows) { return from >= 0 && to >= from && unsigned(to) <= rows; }
__device__ __forceinline__ bool in_order(const Batch& b, const Claim& c) {
  const bool ordered = rows_in_order(c.from, c.to, b.rows);
  if (!ordered || c.length > int(b.width * b.page)) report(b.status, kBadLength);
  return ordered;
}

// Sum over the threads in front of this one, and over all.  `of_warp`: a word per warp; a barrier goes in front of its
// next use.
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

// The part of prefix attention that a row's own sequence makes, unnormalised: [kv_heads][head_dim / 4][rows x group][4] sums and
// [kv_heads][rows x group][2] (maximum in units of log2, weight).  Rows lie side by side, as the threads that own one read them.
struct Own {
  float *sums, *ends;
  unsigned rows, dim;
  __device__ __forceinline__ float4* sum(unsigned head, unsigned c4, unsigned row) const {
    return reinterpret_cast<float4*>(sums) + (size_t(head) * (dim / 4) + c4) * rows + row;
  }
  __device__ __forceinline__ float2* end(unsigned head, unsigned row) const { return reinterpret_cast<float2*>(ends) + size_t(head) * rows + row; }
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
// keys and values to their pages.  Bound by memory: every row is read and written once.  A block owns a row; its threads request
// the row's first vectors, then find the row's sequence (a lane per sequence), page and angles while those are on their way, and
// turn eight pairs of a head at a time.  Angles are formed in 64 bits: at position 100000 a product in 32 bits would already be
// off by more than a bf16 rounding of the result.
// s0 says where a position comes from (below).  log2_theta + log2_theta_rest: log2 of theta in two pieces.
// grid = rows, block = 128.  head_dim 64 or 128, strides multiples of 8.
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
  const unsigned half = head_dim / 2, vec_shift = head_dim == 128 ? 3 : 2, turned = (q_heads + kv_heads) << vec_shift;
  const unsigned blocks = head_dim / 64, copied = kv_heads * blocks * 8, row = blockIdx.x, lane = threadIdx.x & 31;
  k += k_column;
  v += v_column;
  if (!(paged::aligned16(q) && paged::aligned16(k) && paged::aligned16(v) && paged::aligned16(q_out) && paged::aligned16(k_pool) &&
        paged::aligned16(v_pool))) {
    if (threadIdx.x == 0) paged::report(status, paged::kMisaligned);
    return;
  }
  const bf16* const q_row = q + size_t(row) * q_stride;
  const bf16* const k_row = k + size_t(row) * kv_stride;
  const bf16* const v_row = v + size_t(row) * kv_stride;
  auto from_of = [&](unsigned item) {
    const unsigned head = item >> vec_shift, c = item & ((1u << vec_shift) - 1);
    return (head < q_heads ? q_row + head * head_dim : k_row + (head - q_heads) * head_dim) + c * 8;
  };
  constexpr unsigned kAhead = 2;      // vectors of a thread that do not wait for where the row goes
  Bf16x8 lo[kAhead], hi[kAhead];
  uint4 value = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (unsigned u = 0; u < kAhead; ++u)
    if (threadIdx.x + u * 128 < turned) {
      lo[u] = *reinterpret_cast<const Bf16x8*>(from_of(threadIdx.x + u * 128));
      hi[u] = *reinterpret_cast<const Bf16x8*>(from_of(threadIdx.x + u * 128) + half);
    }
  if (threadIdx.x < copied) value = *reinterpret_cast<const uint4*>(v_row + threadIdx.x * 8);

  // A position that does not follow from the cache is asked for here too, and turns per position, 1 / (2 pi theta^(pair mod ladder /
  // ladder)), are computed while all of this is on its way.
  const unsigned pair = threadIdx.x, first = min(lane, sequences - 1);
  int from = starts[first], to = starts[first + 1], length = lengths[first], at_position = 0;
  if (s0 < kPositionsOneAxis && pair < half) at_position = pos[size_t(pair < s0 ? 0u : pair < s0 + s1 ? 1u : 2u) * rows + row];
  if (s0 == kPositionsOneAxis) at_position = pos[row];
  double frequency = 0.;
  if (pair < half)
    frequency = exp2(-(double(log2_theta) + double(log2_theta_rest)) * (double(pair % ladder) / double(ladder))) * 0.15915494309189534;

  // Rows out of order leave the whole launch without work.  The first 32 sequences are at hand; more of them cost a trip per 128.
  bool ordered = paged::rows_in_order(from, to, rows);
  for (unsigned i = 32 + threadIdx.x; i < sequences; i += 128) ordered = paged::rows_in_order(starts[i], starts[i + 1], rows) && ordered;

  // the row's sequence: the first that ends behind it
  int index = 0;
  unsigned seq = sequences;
  for (unsigned base = 0; base < sequences; base += 32) {
    if (base > 0) {
      const unsigned i = min(base + lane, sequences - 1);
      from = starts[i];
      to = starts[i + 1];
      length = lengths[i];
    }
    const unsigned behind = __ballot_sync(0xffffffffu, base + lane < sequences && to > int(row));
    if (behind == 0) continue;
    const int at = __ffs(behind) - 1;
    if (__shfl_sync(0xffffffffu, from, at) <= int(row)) seq = base + at;
    index = int(unsigned(__shfl_sync(0xffffffffu, length, at)) - (unsigned(__shfl_sync(0xffffffffu, to, at)) - row));
    break;
  }
  const bool nobodys = seq >= sequences;      // as all that follows from the row alone, the same for the whole block
  unsigned page_id = 0;
  bool stored = index >= 0 && !nobodys;
  if (stored && unsigned(index) / page >= width) {
    stored = false;
    if (threadIdx.x == 0) paged::report(status, paged::kBadLength);
  }
  if (stored) page_id = unsigned(table[size_t(seq) * width + unsigned(index) / page]);
  if (pair < half) {
    if (s0 == kPositionsFromCache) at_position = int(unsigned(index) + (has_offset ? unsigned(*offset) : 0u));
    const double turns = double(at_position) * frequency;
    sincospif(2.f * float(turns - rint(turns)), &sine[pair], &cosine[pair]);
  }
  if (stored && page_id >= pages) {
    stored = false;
    if (threadIdx.x == 0) paged::report(status, paged::kBadPage);
  }
  const unsigned token = unsigned(index) % page;
  if (!__syncthreads_and(ordered)) {
    if (threadIdx.x == 0) paged::report(status, paged::kBadLength);
    return;
  }
  if (nobodys) return;
  const unsigned c = threadIdx.x & ((1u << vec_shift) - 1);      // the same pairs in every head that this thread turns
  float co[8], si[8];
#pragma unroll
  for (int j = 0; j < 8; j += 4) {
    *reinterpret_cast<float4*>(co + j) = *reinterpret_cast<const float4*>(cosine + c * 8 + j);
    *reinterpret_cast<float4*>(si + j) = *reinterpret_cast<const float4*>(sine + c * 8 + j);
  }
  auto turn = [&](unsigned item, const Bf16x8& l, const Bf16x8& h) {
    const unsigned head = item >> vec_shift;
    float a[8], b[8], x[8], y[8];
    unpack8(l, a);
    unpack8(h, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = a[j] * co[j] - b[j] * si[j];
      y[j] = b[j] * co[j] + a[j] * si[j];
    }
    if (head < q_heads) {
      bf16* to = q_out + size_t(row) * out_stride + head * head_dim + c * 8;
      *reinterpret_cast<Bf16x8*>(to) = pack8(x);
      *reinterpret_cast<Bf16x8*>(to + half) = pack8(y);
    } else if (stored) {
      // chunk c of the head's first half and the same chunk of its second half: of one 64-column block, or of two
      const unsigned behind = c + (1u << vec_shift);
      bf16* first = k_pool + (paged::block_offset(page_id, kv_heads, head - q_heads, blocks, c / 8, page) + token) * 64;
      bf16* second = k_pool + (paged::block_offset(page_id, kv_heads, head - q_heads, blocks, behind / 8, page) + token) * 64;
      *reinterpret_cast<Bf16x8*>(first + (((c & 7) ^ (token & 7)) * 8)) = pack8(x);
      *reinterpret_cast<Bf16x8*>(second + (((behind & 7) ^ (token & 7)) * 8)) = pack8(y);
    }
  };
  auto keep = [&](unsigned item, const uint4& from) {
    const unsigned head = item / (blocks * 8), c = item % (blocks * 8);
    bf16* to = v_pool + (paged::block_offset(page_id, kv_heads, head, blocks, c / 8, page) + token) * 64;
    *reinterpret_cast<uint4*>(to + (((c & 7) ^ (token & 7)) * 8)) = from;
  };
#pragma unroll
  for (unsigned u = 0; u < kAhead; ++u)
    if (threadIdx.x + u * 128 < turned) turn(threadIdx.x + u * 128, lo[u], hi[u]);
  if (stored && threadIdx.x < copied) keep(threadIdx.x, value);
#pragma unroll 1
  for (unsigned item = threadIdx.x + kAhead * 128; item < turned; item += 128)
    turn(item, *reinterpret_cast<const Bf16x8*>(from_of(item)), *reinterpret_cast<const Bf16x8*>(from_of(item) + half));
  if (stored) {
#pragma unroll 1
    for (unsigned item = threadIdx.x + 128; item < copied; item += 128) keep(item, *reinterpret_cast<const uint4*>(v_row + item * 8));
  }
}
