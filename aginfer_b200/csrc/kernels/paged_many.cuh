// Attention over a paged cache for many rows a sequence and key head (prompts, chunks of prompts, a batch over a shared prefix), on
// the fifth-generation tensor core: S = Q K^T and O += P V with tcgen05.mma, accumulators and P in tensor memory.
//
// An item is up to 256 rows of one sequence and key head, its query heads side by side as rows (row r of the sequence: token
// r / group, query head r % group), so that a key head's keys are read once for all of them.  Key tiles hold 128 keys.  All key
// tiles of all items form one line, of which every CTA (one an SM) takes an equal run, whatever the lengths and masks; an item that
// a cut divides leaves unnormalised parts in scratch, which agi_paged_join_bf16 adds in order.
//
// Two streams share the tensor core: while one stream's scores are exponentiated by its four warps, the other's products run.
// An item of more than 128 rows gives each stream 128 rows and every key tile; a smaller one gives both streams the same rows
// and every other tile, and the first stream adds the second one's outputs where they lie in tensor memory.  A thread owns a row: it
// reads the row's 128 scores from tensor memory, needs no shuffles for maximum and sum, and writes P back over them as bf16.  Sums are of
// the unrounded weights, in 32 bits; the outputs are 1.9 - 2.3e-3 (2-norm, relative) off the definition, 1.6 - 1.7e-3 of it their own
// rounding.  Weights in two bf16 pieces would cost half as many products again, where the tensor core works two thirds of a tile's
// time already.  Outputs are rescaled only when a row's maximum has grown by more than 2^8 since they were last scaled; all of it
// cancels in the quotient.
//
// Keys and values come in by one bulk copy per page (or its part in a tile) and 64-column block: the pool holds the image that
// the tensor core reads, rows of keys K-major for S, the same image MN-major for P V.  Tokens behind a sequence's end and pages that
// no row of the item sees are not copied; their values are set to zero in shared memory, since weight zero does not make a NaN
// zero.  Other tokens of a tile are multiplied by weight zero where a row does not see them.
//
// Warps: 0-3 and 4-7 a stream each, 8 issues the products, 9 and 10 bring keys and values in, 11 the queries of the next item.
// Tensor memory (512 columns): scores and P of the streams at 0 and 128, outputs at 256 and 384.
//
// What bounds it, head_dim 128: a tile of 256 rows by 128 keys takes 3200 clocks, of which the tensor core works 2100 and the
// special-function unit 2050; the rest is the chain of a stream (scores 150 clocks to registers, maximum 450, weights 1400, products
// 1200 until the next scores are there) that two streams do not cover.  8192 tokens, 28 query heads on 4, window 2048: 253 us in
// short runs, 279 in long ones: 830 and 760 TFLOP/s, about half the rate measured for a library product.  An item costs 8500 clocks
// besides, a launch 9000 before its first scores.
#pragma once

#include "gemm_tc.cuh"
#include "paged.cuh"

namespace many {

using namespace paged;

constexpr unsigned kKeys = 128, kStreamRows = 128, kRows = 256, kThreads = 384;
// Registers after the warp groups have traded: a row's 128 scores stay in registers (168 a thread, the launch's share, would spill 480
// bytes), the group of the loading and the issuing warp gives its own for that (2 x 208 + 88 = 3 x 168).
constexpr unsigned kSoftmaxRegs = 208, kHelperRegs = 88;
constexpr unsigned kStagePitch = 80;        // bytes of a row's 32 columns in a warp's staging memory, and 16 against bank conflicts
constexpr unsigned kItemCost = 3;           // what an item costs besides its tiles (queries in, outputs out), in tiles
constexpr unsigned kOutColumn = 256;
constexpr float kSlack = 8.f;               // log2 of how far scores may exceed the maximum that weights are relative to

// 32 columns of this thread's lane; the values may be used after tmem_loaded().
__device__ __forceinline__ void tmem_load32(unsigned addr, float* v) {
  unsigned* r = reinterpret_cast<unsigned*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(addr));
}
// Waits for loads; the empty statements tie the values to the wait, so that nothing that uses them moves in front of it.
template <unsigned kCount>
__device__ __forceinline__ void tmem_loaded(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (unsigned i = 0; i < kCount; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void tmem_store32(unsigned addr, const unsigned* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_store16(unsigned addr, const unsigned* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
               "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ bool is_done(unsigned long long* bar, unsigned parity) {
  unsigned done;
  asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(done) : "r"(tc::smem_u32(bar)), "r"(parity) : "memory");
  return done != 0;
}

// D[128 x N] (+)= A . B with A (bf16 pairs) in tensor memory.
__device__ __forceinline__ void mma_from_tmem(unsigned d, unsigned a, unsigned long long b, unsigned idesc, unsigned accumulate) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b),
               "r"(idesc), "r"(accumulate)
               : "memory");
}
// fp32 accumulators, bf16 operands, M = 128, N columns; B K-major or MN-major.
__device__ __forceinline__ constexpr unsigned instruction(unsigned n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// 128-byte-swizzled MN-major operand: 64 columns (one 128-byte row of each key) to the next 64 `leading` bytes on, 8 keys to the
// next 8 keys 1024 bytes on.
__device__ __forceinline__ unsigned long long mn_descriptor(unsigned addr, unsigned leading) {
  return (unsigned long long)((addr & 0x3FFFFu) >> 4) | ((unsigned long long)(leading >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// Rows of an item and what they see.  kPrefix: all rows of the launch over the one shared prefix.
struct Item {
  unsigned row;              // first row of the sequence (or launch)
  int first;                 // index of the first of them
  unsigned row0, rows;       // rows of the item among the sequence's fresh * group
  unsigned head;
  Visible seen;
};

// Parts of items that runs cut, as in the kernel for few rows: slot 0 of a CTA where the item began before its run, slot 1 where it
// goes on behind it.  A slot is [head_dim / 4][256 rows][4] sums and [256][2] (maximum in units of log2, weight).
// note[cta]: the item that begins in slot 1 of a CTA (pieces = 0: none).
struct Note {
  unsigned pieces, row, row0, rows, head, unused[3];
};
template <unsigned kDim>
struct Parts {
  float* base;
  Note* notes;
  static constexpr size_t kSlot = size_t(kRows) * kDim + 2 * kRows;
  __device__ __forceinline__ float4* sum(unsigned cta, unsigned slot, unsigned row, unsigned c4) const {
    return reinterpret_cast<float4*>(base + (size_t(cta) * 2 + slot) * kSlot) + c4 * kRows + row;
  }
  __device__ __forceinline__ float2* end(unsigned cta, unsigned slot, unsigned row) const {
    return reinterpret_cast<float2*>(base + (size_t(cta) * 2 + slot) * kSlot + size_t(kRows) * kDim) + row;
  }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two values at a time.
__device__ __forceinline__ unsigned long long pair_bits(float2 v) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 pair_of(unsigned long long bits) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(bits));
  return v;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
  return pair_of(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return pair_of(d);
}

// Which of the 32 keys from `key` on a row at `index` of a sequence of `end` tokens sees, a bit each.
__device__ __forceinline__ unsigned visible_bits(unsigned key, int index, unsigned end, unsigned window, unsigned sinks) {
  auto first = [](int count) { return count <= 0 ? 0u : count >= 32 ? 0xffffffffu : (1u << count) - 1; };      // the bits of so many keys
  const unsigned up_to = first(min(index + 1, int(end)) - int(key));
  return window == 0 ? up_to : up_to & (~first(index + 1 - int(window) - int(key)) | first(int(sinks) - int(key)));
}

// Another part of a row's sums (its maximum and weight in `other`) is added to this one's: what both are multiplied by.
__device__ __forceinline__ void join(float& top, float& sum, float2 other, float& mine_by, float& other_by) {
  const float next = fmaxf(top, other.x);
  mine_by = next == -INFINITY ? 0.f : exp2_of(top - next);
  other_by = next == -INFINITY ? 0.f : exp2_of(other.x - next);
  sum = sum * mine_by + other.y * other_by;
  top = next;
}

template <int HD16, bool kPrefix>
__device__ __forceinline__ void attention_body(const bf16* q, bf16* o, const bf16* k_pool, const bf16* v_pool, const Batch& batch,
                                               const int* prefix_table, const int* prefix_length, unsigned prefix_pages, float* own_sums,
                                               float* own_ends, float* scratch, Note* notes, unsigned q_heads, unsigned kv_heads, unsigned q_stride,
                                               unsigned o_stride, unsigned window, unsigned sinks, float scale_log2, unsigned stages,
                                               unsigned least, unsigned own_only) {
  constexpr unsigned kDim = HD16 * 16, kBlocks = kDim / 64, kBlockBytes = kKeys * 128, kSlotBytes = kBlocks * kBlockBytes;
  // Tiles that are not cut off an item (ragged chunks 0 57.5 us, 1 55.5, 2 56.2; a prefix's few, long items 31, 33, 35).
  constexpr unsigned kSnap = kPrefix ? 0 : 1;
  constexpr unsigned kQBytes = kStreamRows * kDim * 2, kMaxStages = 6;
  extern __shared__ unsigned char dynamic_smem[];
  __shared__ __align__(8) unsigned long long k_full[kMaxStages], k_empty[kMaxStages], v_full[kMaxStages], v_empty[kMaxStages];
  __shared__ __align__(8) unsigned long long q_full[2], q_empty[2], s_full[2], p_half[2], p_full[2], o_full[2], o_empty[2];
  __shared__ float2 shared_end[kStreamRows];
  __shared__ unsigned block_base[kThreads / 32], tile_base[kThreads / 32], run_seq, run_block, run_first, gave_up, tmem_slot;
  __shared__ Span run_span;
  const unsigned tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned base = (tc::smem_u32(dynamic_smem) + 1023u) & ~1023u;
  unsigned char* const base_ptr = dynamic_smem + (base - tc::smem_u32(dynamic_smem));
  const unsigned ring = base + 2 * kQBytes;
  const unsigned group = q_heads / kv_heads;
  const Parts<kDim> parts{scratch, notes};
  const Own own{own_sums, own_ends, batch.rows * group, kDim};

  if (tid == 0) {
    for (unsigned s = 0; s < stages; ++s) {
      tc::mbar_init(&k_full[s], 1);
      tc::mbar_init(&k_empty[s], 1);
      tc::mbar_init(&v_full[s], 1);
      tc::mbar_init(&v_empty[s], 1);
    }
    for (unsigned s = 0; s < 2; ++s) {
      tc::mbar_init(&q_full[s], 1);
      tc::mbar_init(&q_empty[s], 1);
      tc::mbar_init(&s_full[s], 1);
      tc::mbar_init(&p_half[s], kStreamRows);
      tc::mbar_init(&p_full[s], kStreamRows);
      tc::mbar_init(&o_full[s], 1);
      tc::mbar_init(&o_empty[s], kStreamRows);
    }
    gave_up = 0;
    run_seq = run_block = 0;
    run_first = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) tc::tmem_alloc(&tmem_slot, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const unsigned tmem = tmem_slot;
  // The prefix does not wait for its rows' own sequences, which the launch before is still working on, until it adds them; that launch
  // has let this one begin only when everything in front of it was complete.
  if (kPrefix) grid_dependency_release();
  else grid_dependency_wait();

  const bool aligned = aligned16(q) && aligned16(o) && aligned16(k_pool) && aligned16(v_pool);
  if (!aligned && tid == 0) report(batch.status, kMisaligned);

  // ---- the run of this CTA: key tiles [from, to) of all ----
  const unsigned sequences = kPrefix ? 1u : batch.sequences;
  auto span_at = [&](unsigned seq) {
    if (!kPrefix) return span_of(batch, claim_of(batch, seq));
    return Span{0u, batch.rows, 0, min(unsigned(max(*prefix_length, 0)), prefix_pages * batch.page)};
  };
  auto seen_at = [&](const Span& s, unsigned block) {
    if (kPrefix) return visible_of<kKeys>(0, int(s.length) - 1, s.length, 0, 0);
    const unsigned last = min((block + 1) * kRows, s.fresh * group) - 1;
    return visible_of<kKeys>(s.first + int(block * kRows / group), s.first + int(last / group), s.length, window, sinks);
  };
  auto blocks_of = [&](const Span& s) { return (s.fresh * group + kRows - 1) / kRows; };
  unsigned from = 0, to = 0, per = 1;
  if (kPrefix) {      // blocks are alike: every thread finds the run by itself
    // The launch before does nothing for rows out of order; no part of it would be there to be added.
    bool ordered = true;
    for (unsigned i = tid; i < batch.sequences; i += kThreads) ordered = rows_in_order(batch.starts[i], batch.starts[i + 1], batch.rows) && ordered;
    const Span span = span_at(0);
    const unsigned tiles = (seen_at(span, 0).count + kItemCost) * kv_heads, total = __syncthreads_and(ordered && aligned) ? blocks_of(span) * tiles : 0u;
    if (tid == 0 && *prefix_length > int(prefix_pages * batch.page)) report(batch.status, kBadLength);
    per = max((total + gridDim.x - 1) / gridDim.x, least);
    from = min(per * blockIdx.x, total);
    to = min(from + per, total);
    if (tid == 0) {
      run_seq = 0;
      run_block = from / tiles;
      run_first = from / tiles * tiles;
      run_span = span;
    }
  } else {
    // what the batch says of every sequence and where its blocks of rows begin (in Q's memory, before Q is there) ...
    int4* const places = reinterpret_cast<int4*>(base_ptr);
    unsigned below_blocks = 0, ordered = aligned;
#pragma unroll 1
    for (unsigned i0 = 0; i0 < sequences; i0 += kThreads) {
      const unsigned i = i0 + tid;
      Claim claim{0, 0, 0};
      if (i < sequences) {
        claim = claim_of(batch, i);
        if (!in_order(batch, claim)) {
          ordered = 0;
          claim = Claim{0, 0, 0};
        }
      }
      unsigned all;
      const unsigned begins = below_blocks + sum_before<kThreads>(blocks_of(span_of(batch, claim)), block_base, &all);
      if (i < sequences) places[i] = make_int4(claim.from, claim.to, claim.length, int(begins));
      below_blocks += all;
      ordered = __syncthreads_and(ordered);
    }
    const unsigned all_blocks = ordered ? below_blocks : 0u;
    // ... then their key tiles: a run of blocks a thread
    const unsigned share = (all_blocks + kThreads - 1) / kThreads, b0 = min(tid * share, all_blocks), b1 = min(b0 + share, all_blocks);
    unsigned holder = 0;      // the sequence with block b0: the last one that begins at or before it
    for (unsigned above = sequences; above - holder > 1;) {
      const unsigned middle = (holder + above) / 2;
      if (unsigned(places[middle].w) <= b0) holder = middle; else above = middle;
    }
    auto tiles_of = [&](unsigned& seq, unsigned b) {
      while (seq + 1 < sequences && unsigned(places[seq + 1].w) <= b) ++seq;
      const int4 place = places[seq];
      return (seen_at(span_of(batch, Claim{place.x, place.y, place.z}), b - unsigned(place.w)).count + kItemCost) * kv_heads;
    };
    unsigned mine = 0, total, seq = holder;
#pragma unroll 1
    for (unsigned b = b0; b < b1; ++b) mine += tiles_of(seq, b);
    unsigned below = sum_before<kThreads>(mine, tile_base, &total);
    per = max((total + gridDim.x - 1) / gridDim.x, least);
    from = min(per * blockIdx.x, total);
    to = min(from + per, total);
    if (from < to && from >= below && from < below + mine) {      // this thread's blocks hold the run's first tile
      seq = holder;
      for (unsigned b = b0;; ++b) {
        const unsigned tiles = tiles_of(seq, b);
        if (from < below + tiles) {
          const int4 place = places[seq];
          run_seq = seq;
          run_block = b - unsigned(place.w);
          run_first = below;
          run_span = span_of(batch, Claim{place.x, place.y, place.z});
          break;
        }
        below += tiles;
      }
    }
  }
  if (tid == 0) parts.notes[blockIdx.x].pieces = 0;
  // `places` of a batch of many sequences reaches into the keys' ring, which bulk copies write next
  if (!kPrefix) tc::fence_async_shared();
  __syncthreads();

  auto give_up = [&] { *(volatile unsigned*)&gave_up = 1; };
  auto await = [&](unsigned long long* bar, unsigned parity, unsigned code) {
    if (is_done(bar, parity)) return;
    if (!*(volatile unsigned*)&gave_up && !tc::mbar_wait(bar, parity, batch.status, code)) give_up();
  };
  // f(item, first key tile, last key tile + 1, number of the item's first unit, sequence)
  auto walk = [&](auto&& f) {
    unsigned seq = run_seq, block = run_block, first = run_first, unit = from;
    Span span = run_span;
#pragma unroll 1
    while (unit < to) {
      if (block >= blocks_of(span)) {
        block = 0;
        if (++seq >= sequences) break;
        span = span_at(seq);
        continue;
      }
      Item it;
      it.row = span.row;
      it.first = span.first;
      it.row0 = block * kRows;
      it.rows = min(kRows, span.fresh * group - it.row0);
      it.seen = seen_at(span, block);
      const unsigned length = it.seen.count + kItemCost;
#pragma unroll 1
      while (unit < to && unit < first + length * kv_heads) {
        it.head = (unit - first) / length;
        // The item's tiles stand behind the units that it costs besides.  A cut among those, or so few tiles behind the first or in front of
        // the end that its part would cost more than it evens out, is moved there; the CTAs on both sides see it alike.
        const unsigned tiles_at = first + it.head * length + kItemCost, next = tiles_at + it.seen.count;
        auto cut = [&](unsigned at) {
          if (at >= next) return next;
          return at <= tiles_at + kSnap ? tiles_at : at + kSnap >= next ? next : at;
        };
        const unsigned begin = cut(from) - tiles_at, end = cut(to) - tiles_at;
        if (begin < end) f(it, begin, end, tiles_at, seq);
        unit = next;
      }
      first += length * kv_heads;
      ++block;
    }
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kHelperRegs));
    if (warp == 9 || warp == 10) {
      // ---- a warp each for keys and values: a lane per piece (64-column block, page or part of one) of a tile ----
      const bool values = warp == 10;
      const unsigned shift = 31 - __clz(batch.page), run = min(batch.page, kKeys), pieces = kKeys / run;
      const unsigned block = (lane / pieces) % kBlocks, piece = lane % pieces;
      const bool live = lane < kBlocks * pieces;
      const unsigned page_bytes = kv_heads * kBlocks * batch.page * 128, slots = ring + (values ? stages * kSlotBytes : 0u);
      unsigned long long* const full = values ? v_full : k_full;
      unsigned long long* const empty = values ? v_empty : k_empty;
      unsigned s = 0, phase = 1;
      walk([&](const Item& it, unsigned begin, unsigned end, unsigned, unsigned seq) {
        const int* const pages_of = kPrefix ? prefix_table : batch.table + size_t(seq) * batch.width;
        const unsigned char* const pool = reinterpret_cast<const unsigned char*>(values ? v_pool : k_pool) + size_t((it.head * kBlocks + block) * batch.page) * 128;
        auto token_of = [&](unsigned t) { return it.seen.tile(t) * kKeys + piece * run; };
        auto tokens_of = [&](unsigned t) {      // that this lane brings in
          const unsigned token = token_of(t);
          return live && token < it.seen.end && (token < it.seen.sink_end || token + run > it.seen.start) ? min(run, it.seen.end - token) : 0u;
        };
        unsigned count = tokens_of(begin), page_id = count ? unsigned(pages_of[token_of(begin) >> shift]) : 0u;
#pragma unroll 1
        for (unsigned t = begin; t < end; ++t) {
          if (page_id >= batch.pages) {
            report(batch.status, kBadPage);
            count = 0;
          }
          const unsigned char* const from_page = pool + size_t(page_id) * page_bytes + (token_of(t) & (batch.page - 1)) * 128;
          const unsigned slot = slots + s * kSlotBytes, all = __reduce_add_sync(0xffffffffu, count * 128);
          unsigned next_count = 0, next_page = 0;      // the page of the tile behind it, while this one's slot is awaited
          if (t + 1 < end) {
            next_count = tokens_of(t + 1);
            if (next_count) next_page = unsigned(pages_of[token_of(t + 1) >> shift]);
          }
          if (lane == 0) await(&empty[s], phase, tc::kTimeoutEmpty | s);
          __syncwarp();
          if (values && all < kSlotBytes) {      // zero what is not copied
            for (unsigned p = 0; p < pieces; ++p) {
              const unsigned held = __shfl_sync(0xffffffffu, count, p);       // the same for every block of the piece
              for (unsigned i = lane; i < (run - held) * 8 * kBlocks; i += 32) {
                const unsigned b = i / ((run - held) * 8), rest = i % ((run - held) * 8);
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(slot + b * kBlockBytes + (p * run + held) * 128 + rest * 16), "r"(0u)
                             : "memory");
              }
            }
            tc::fence_async_shared();
            __syncwarp();
          }
          if (lane == 0) tc::expect_bytes(&full[s], all);
          __syncwarp();
          if (count) tc::bulk_copy(slot + block * kBlockBytes + piece * run * 128, from_page, count * 128, &full[s]);
          count = next_count;
          page_id = next_page;
          if (++s == stages) { s = 0; phase ^= 1; }
        }
      });
    } else if (warp == 8) {
      // ---- one thread issues the products ----
      if (elect_one()) {
        constexpr unsigned kScores = instruction(kKeys, false), kOutputs = instruction(kDim, true);
        unsigned ks = 0, k_phase = 0, vs = 0, v_phase = 0, q_phases = 0, p_phases = 0, o_phases = 3;       // the last three: a bit per stream
        auto flips = [&](unsigned long long* bars, unsigned& phases, unsigned stream, unsigned code) {
          await(&bars[stream], (phases >> stream) & 1, tc::kTimeoutAccum | code | stream);
          phases ^= 1u << stream;
          tc::tc_fence_after();
        };
        auto scores = [&](unsigned stream, unsigned q_stream, unsigned slot) {
          const unsigned long long a = tc::smem_descriptor(base + q_stream * kQBytes), b = tc::smem_descriptor(ring + slot * kSlotBytes);
#pragma unroll
          for (unsigned k = 0; k < HD16; ++k)
            tc::mma<false>(tmem + stream * kKeys, a + (k / 4) * (kStreamRows * 128 >> 4) + (k % 4) * 2, b + (k / 4) * (kBlockBytes >> 4) + (k % 4) * 2,
                           kScores, k != 0);
          tc::tc_commit(&s_full[stream]);
        };
        auto arrived = [&](unsigned long long* bars, unsigned& s, unsigned& phase) {      // the next tile has landed: its slot
          await(&bars[s], phase, tc::kTimeoutFull | s);
          const unsigned slot = s;
          if (++s == stages) { s = 0; phase ^= 1; }
          return slot;
        };
        // P V of a stream's tile: the first half of the keys while the weights of the second half are still being formed
        auto outputs = [&](unsigned stream, unsigned slot, bool first) {
          const unsigned long long b = mn_descriptor(ring + (stages + slot) * kSlotBytes, kBlockBytes);
          const unsigned d = tmem + kOutColumn + stream * 128, a = tmem + stream * kKeys;
          if (first) flips(o_empty, o_phases, stream, 0x80);
          await(&p_half[stream], (p_phases >> stream) & 1, tc::kTimeoutAccum | 0x30 | stream);
          tc::tc_fence_after();
#pragma unroll
          for (unsigned k = 0; k < kKeys / 32; ++k) mma_from_tmem(d, a + k * 8, b + k * (16 * 128 >> 4), kOutputs, !first || k != 0);
          flips(p_full, p_phases, stream, 0x20);
#pragma unroll
          for (unsigned k = kKeys / 32; k < kKeys / 16; ++k) mma_from_tmem(d, a + k * 8, b + k * (16 * 128 >> 4), kOutputs, 1);
        };
        walk([&](const Item& it, unsigned begin, unsigned end, unsigned, unsigned) {
          const unsigned n = end - begin;
          const bool shared_rows = it.rows <= kStreamRows;
          // step i: scores of tile i (i < n), behind the outputs of the tile that used the same columns before
          const unsigned lead = shared_rows ? min(n, 2u) : 1u;
          unsigned values = 0, keys = 0;
#pragma unroll 1
          for (unsigned i = 0; i < n + lead; ++i) {
#pragma unroll 1
            for (unsigned half = 0; half < (shared_rows ? 1u : 2u); ++half) {
              const unsigned stream = shared_rows ? (i >= lead ? (i - lead) & 1 : i) : half, area = shared_rows ? 0u : stream;
              const bool last_use = shared_rows || half == 1;
              if (i >= lead && half == 0) values = arrived(v_full, vs, v_phase);
              if (i < n && half == 0) keys = arrived(k_full, ks, k_phase);
              if (i >= lead) {
                const unsigned j = i - lead;
                outputs(stream, values, j < lead);
                if (last_use) tc::tc_commit(&v_empty[values]);
                if (j + lead >= n) tc::tc_commit(&o_full[stream]);
              }
              if (i < n) {
                if (i == 0) flips(q_full, q_phases, area, 0x10);
                tc::tc_fence_after();
                scores(stream, area, keys);
                if (last_use) tc::tc_commit(&k_empty[keys]);
                if (i == n - 1) tc::tc_commit(&q_empty[area]);
              }
            }
          }
        });
      }
      __syncwarp();
    } else {
      // ---- a warp brings the queries in (zero past the item's rows), as soon as the item before has formed its last scores ----
      constexpr unsigned kChunks = kDim / 8, kStep = 32 / kChunks;      // 16-byte chunks of a row, rows that the warp copies at a time
      const unsigned c = lane % kChunks, lane_row = lane / kChunks, token_step = kStep / group, sub_step = kStep % group;
      const size_t ahead = (size_t(token_step) * q_stride + sub_step * kDim) * 2, wraps = (size_t(q_stride) - group * kDim) * 2;
      unsigned phases = 3;
      bool first_item = true;            // its queries the softmax warps bring in, which have nothing else to do yet
      walk([&](const Item& it, unsigned, unsigned, unsigned, unsigned) {
        if (first_item) {
          first_item = false;
          phases ^= it.rows <= kStreamRows ? 1u : 3u;
          return;
        }
#pragma unroll 1
        for (unsigned stream = 0; stream < (it.rows <= kStreamRows ? 1u : 2u); ++stream) {
          const unsigned rows_before = stream * kStreamRows, live = min(it.rows - rows_before, kStreamRows);
          const unsigned q_area = base + stream * kQBytes + (c / 8) * (kStreamRows * 128) + lane_row * 128;
          const unsigned first = it.row0 + rows_before + lane_row, token = first / group;
          unsigned sub = first - token * group;
          const unsigned char* from_row = reinterpret_cast<const unsigned char*>(q + size_t(it.row + token) * q_stride + (it.head * group + sub) * kDim + c * 8);
          await(&q_empty[stream], (phases >> stream) & 1, tc::kTimeoutAccum | 0x50 | stream);
          phases ^= 1u << stream;
          __syncwarp();
#pragma unroll 1
          for (unsigned row = 0; row < kStreamRows; row += 8) {
#pragma unroll
            for (unsigned i = 0; i < 8; i += kStep) {      // a row in front of the item's end is read, one behind it is zero
              const bool held = row + i + lane_row < live;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(q_area + (row + i) * 128 + (((c & 7) ^ (i + lane_row)) << 4)),
                           "l"(held ? from_row : reinterpret_cast<const unsigned char*>(q)), "r"(held ? 16u : 0u) : "memory");
              from_row += ahead;
              sub += sub_step;
              if (sub >= group) {
                sub -= group;
                from_row += wraps;
              }
            }
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          tc::fence_async_shared();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&q_full[stream]);
        }
      });
    }
  } else {
    // ---- softmax and outputs: four warps a stream, a thread a row ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const unsigned stream = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;       // row of the stream
    const unsigned lanes = (quarter * 32u) << 16;
    const unsigned score_at = tmem + stream * kKeys + lanes, out_at = tmem + kOutColumn + stream * 128 + lanes;
    unsigned char* const staged = base_ptr + 2 * kQBytes + 2 * stages * kSlotBytes + warp * (32 * kStagePitch);
    unsigned s_phase = 0, o_phases = 0, shared_items = 0;
    bool first_item = true;
    auto outputs_done = [&](unsigned of_stream) {
      await(&o_full[of_stream], (o_phases >> of_stream) & 1, tc::kTimeoutAccum | 0x40 | of_stream);
      __syncwarp();
      tc::tc_fence_after();
    };
    walk([&](const Item& it, unsigned begin, unsigned end, unsigned tiles_at, unsigned) {
      const unsigned n = end - begin;
      const bool shared_rows = it.rows <= kStreamRows;
      const unsigned rows_before = shared_rows ? 0u : stream * kStreamRows;                 // of the item's, in front of this stream's
      const bool is_live = rows_before + r < it.rows;
      const Rows pairs(it.row0 + rows_before, group);
      if (first_item && (!shared_rows || stream == 0)) {
        constexpr unsigned kBatch = kDim / 8;
        const unsigned live = min(it.rows - rows_before, kStreamRows);
#pragma unroll 1
        for (unsigned i0 = r; i0 < kStreamRows * (kDim / 8); i0 += 128 * kBatch) {
          uint4 v[kBatch];
#pragma unroll
          for (unsigned b = 0; b < kBatch; ++b) {
            const unsigned row = (i0 + b * 128) / (kDim / 8), c = (i0 + b * 128) % (kDim / 8);
            unsigned token, sub;
            pairs.at(row, token, sub);
            const bf16* from_row = q + size_t(it.row + token) * q_stride + (it.head * group + sub) * kDim + c * 8;
            v[b] = row < live ? __ldcg(reinterpret_cast<const uint4*>(from_row)) : make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll
          for (unsigned b = 0; b < kBatch; ++b) {
            const unsigned row = (i0 + b * 128) / (kDim / 8), c = (i0 + b * 128) % (kDim / 8);
            *reinterpret_cast<uint4*>(base_ptr + stream * kQBytes + (c / 8) * (kStreamRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v[b];
          }
        }
        tc::fence_async_shared();
        __syncwarp();
        if (stream == 0) asm volatile("bar.sync 3, 128;" ::: "memory");
        else asm volatile("bar.sync 4, 128;" ::: "memory");
        if (r == 0) tc::mbar_arrive(&q_full[stream]);
      }
      first_item = false;
      unsigned token, sub;
      pairs.at(r, token, sub);
      const int index = kPrefix ? 0x3fffffff : is_live ? it.first + int(token) : -1;
      // the rows of this warp: does a tile need a mask?
      const int low = it.first + int(__shfl_sync(0xffffffffu, token, 0)), high = it.first + int(__shfl_sync(0xffffffffu, token, 31));
      float top = -INFINITY, sum = 0.f;       // what weights are relative to (in units of log2), their sum
      bool done = false;
#pragma unroll 1
      for (unsigned j = shared_rows ? stream : 0u; j < n; j += shared_rows ? 2u : 1u) {
        await(&s_full[stream], s_phase, tc::kTimeoutAccum | stream);
        s_phase ^= 1;
        __syncwarp();
        tc::tc_fence_after();
        float x[kKeys];
#pragma unroll
        for (unsigned c = 0; c < kKeys; c += 32) tmem_load32(score_at + c, x + c);
        const unsigned key0 = it.seen.tile(begin + j) * kKeys;
        const bool whole = key0 + kKeys <= it.seen.end && (kPrefix || (int(key0 + kKeys) - 1 <= low && (window == 0 || int(key0) > high - int(window))));
        tmem_loaded<kKeys>(x);
        if (!whole) {
#pragma unroll
          for (unsigned c = 0; c < kKeys; c += 32) {
            const unsigned bits = visible_bits(key0 + c, index, it.seen.end, kPrefix ? 0u : window, sinks);
#pragma unroll
            for (unsigned i = 0; i < 32; ++i) x[c + i] = (bits >> i) & 1 ? x[c + i] : -INFINITY;
          }
        }
        float peak[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (unsigned i = 4; i < kKeys; i += 2) peak[(i / 2) & 3] = max3(peak[(i / 2) & 3], x[i], x[i + 1]);
        const float now = max3(fmaxf(peak[0], peak[1]), peak[2], peak[3]) * scale_log2;
        if (__any_sync(0xffffffffu, now > top + kSlack)) {
          const float next = fmaxf(top, now), factor = next == -INFINITY ? 1.f : exp2_of(top - next);
          top = next;
          sum *= factor;
          if (done) {
#pragma unroll 1
            for (unsigned c = 0; c < kDim; c += 16) {
              float v[16];
              tc::tmem_load16(out_at + c, v);
              tmem_loaded<16>(v);
#pragma unroll
              for (unsigned i = 0; i < 16; ++i) v[i] *= factor;
              tmem_store16(out_at + c, reinterpret_cast<const unsigned*>(v));
            }
            tmem_stored();
          }
        }
        const float2 by = make_float2(scale_log2, scale_log2), back = top == -INFINITY ? make_float2(0.f, 0.f) : make_float2(-top, -top);
        float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (unsigned half = 0; half < 2; ++half) {
          unsigned packed[32];
#pragma unroll
          for (unsigned i = 0; i < 32; ++i) {
            float2 p = fma2(make_float2(x[half * 64 + 2 * i], x[half * 64 + 2 * i + 1]), by, back);
            p.x = exp2_of(p.x);
            p.y = exp2_of(p.y);
            part[i & 1] = add2(part[i & 1], p);
            const bf162 pair = __floats2bfloat162_rn(p.x, p.y);
            packed[i] = *reinterpret_cast<const unsigned*>(&pair);
          }
          tmem_store32(score_at + half * 32, packed);
          tmem_stored();
          tc::tc_fence_before();
          tc::mbar_arrive(half == 0 ? &p_half[stream] : &p_full[stream]);
        }
        sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
        done = true;
      }
      const bool cut = begin != 0 || end != it.seen.count, both = shared_rows && n >= 2;
      const unsigned slot = begin > 0 ? 0u : 1u;
      float2 other = make_float2(-INFINITY, 0.f);
      if (shared_rows) {      // the first stream adds the second one's share, which it reads where that left it
        if (stream == 1) {
          if (shared_items++) asm volatile("bar.sync 2, 256;" ::: "memory");      // that of the item before has been read
          shared_end[r] = make_float2(top, sum);
          asm volatile("bar.arrive 1, 256;" ::: "memory");
          o_phases ^= both ? 3u : 1u;
          return;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        other = shared_end[r];
        asm volatile("bar.arrive 2, 256;" ::: "memory");
      }
      outputs_done(stream);
      if (both) outputs_done(1);
      o_phases ^= shared_rows && !both ? 1u : 3u;
      float mine_by = 1.f, other_by = 0.f;
      if (both) join(top, sum, other, mine_by, other_by);
      // rows of no sequence are left alone
      const unsigned row = it.row + token;
      const bool stays = is_live && (!kPrefix || (int(row) >= batch.starts[0] && int(row) < batch.starts[batch.sequences]));
      const unsigned flat = row * group + sub;
      const bool merges = kPrefix && !cut && stays, divides = !cut && !own_only;
      float own_by = 0.f;
      if (merges) {
        float all_by;
        grid_dependency_only_wait();
        join(top, sum, __ldcg(own.end(it.head, flat)), all_by, own_by);
        mine_by *= all_by;
        other_by *= all_by;
      }
      if (divides) {
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        mine_by *= inv;
        other_by *= inv;
        own_by *= inv;
      }
      bf16* const to_row = o + size_t(row) * o_stride + (it.head * group + sub) * kDim;
#pragma unroll 1
      for (unsigned c0 = 0; c0 < kDim; c0 += 32) {
        float v[32];
        __syncwarp();       // rows that merge, stay or are live took branches of their own; tensor memory is read by the whole warp
        tmem_load32(out_at + c0, v);
        tmem_loaded<32>(v);
#pragma unroll
        for (unsigned i = 0; i < 32; ++i) v[i] *= mine_by;
        if (both) {
          float w[32];
          tmem_load32(out_at + 128 + c0, w);
          tmem_loaded<32>(w);
#pragma unroll
          for (unsigned i = 0; i < 32; ++i) v[i] = fmaf(w[i], other_by, v[i]);
        }
        if (merges) {
#pragma unroll
          for (unsigned i = 0; i < 32; i += 4) {
            const float4 w = __ldcg(own.sum(it.head, (c0 + i) / 4, flat));
            v[i] = fmaf(w.x, own_by, v[i]);
            v[i + 1] = fmaf(w.y, own_by, v[i + 1]);
            v[i + 2] = fmaf(w.z, own_by, v[i + 2]);
            v[i + 3] = fmaf(w.w, own_by, v[i + 3]);
          }
        }
        if (divides) {      // through shared memory, so that rows leave in whole sectors: eight rows of 64 bytes a store
          __syncwarp();
#pragma unroll
          for (unsigned i = 0; i < 32; i += 8) *reinterpret_cast<Bf16x8*>(staged + lane * kStagePitch + i * 2) = pack8(v + i);
          __syncwarp();
#pragma unroll
          for (unsigned i = 0; i < 32; i += 8) {
            const unsigned other_row = i + lane / 4;
            const unsigned long long at = __shfl_sync(0xffffffffu, stays ? reinterpret_cast<unsigned long long>(to_row) : 0ull, other_row);
            if (at) *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(at) + c0 + (lane & 3) * 8) =
                *reinterpret_cast<const uint4*>(staged + other_row * kStagePitch + (lane & 3) * 16);
          }
        } else if (is_live) {
#pragma unroll
          for (unsigned i = 0; i < 32; i += 4)
            *(cut ? parts.sum(blockIdx.x, slot, rows_before + r, (c0 + i) / 4) : own.sum(it.head, (c0 + i) / 4, flat)) =
                make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
      tc::tc_fence_before();
      tc::mbar_arrive(&o_empty[stream]);
      if (both) tc::mbar_arrive(&o_empty[1]);
      if (!divides && is_live) *(cut ? parts.end(blockIdx.x, slot, rows_before + r) : own.end(it.head, flat)) = make_float2(top, sum);
      if (cut && begin == 0 && tid == 0) {
        Note& note = parts.notes[blockIdx.x];
        note.row = it.row;
        note.row0 = it.row0;
        note.rows = it.rows;
        note.head = it.head;
        // the cuts inside the item, and one
        note.pieces = (tiles_at + it.seen.count - kSnap - 1) / per - (tiles_at + kSnap) / per + 1;
      }
    });
  }
  if (kPrefix) grid_dependency_only_wait();       // whoever waits for this launch may rely on the one before too
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc::tc_fence_after();
    tc::tmem_free(tmem, 512);
  }
}

// The parts of items that runs cut, added in order.  Every block reads the notes of all CTAs and counts the groups of eight rows that
// cut items have; it takes groups blockIdx.x, + gridDim.x, ...  A thread takes four columns of a row: eight rows of a column group
// are one line of a slot.
constexpr unsigned kJoinRows = 8, kMaxCtas = 160;
template <int HD16, bool kPrefix>
__device__ __forceinline__ void join_body(bf16* o, const int* starts, unsigned sequences, float* own_sums, float* own_ends, float* scratch, Note* notes,
                                          unsigned ctas, unsigned rows_of_launch, unsigned q_heads, unsigned kv_heads, unsigned o_stride,
                                          unsigned own_only) {
  constexpr unsigned kDim = HD16 * 16, kJoinThreads = kJoinRows * kDim / 4, kBatch = kPrefix ? 6 : 4;
  __shared__ unsigned begins[kMaxCtas + 1];
  const unsigned tid = threadIdx.x, lane = tid & 31, group = q_heads / kv_heads;
  if (own_only) grid_dependency_wait_then_release();       // a prefix's launch is next
  else grid_dependency_wait();
  const Parts<kDim> parts{scratch, notes};
  const Own own{own_sums, own_ends, rows_of_launch * group, kDim};
  for (unsigned i = tid; i < kMaxCtas; i += kJoinThreads) {
    uint4 a = make_uint4(0u, 0u, 0u, 0u);
    if (i < ctas) a = __ldcg(reinterpret_cast<const uint4*>(notes + i));
    begins[i + 1] = a.x ? (a.w + kJoinRows - 1) / kJoinRows : 0u;
  }
  __syncthreads();
  if (tid < 32) {
    constexpr unsigned kEach = kMaxCtas / 32;
    unsigned sum = 0, of[kEach];
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) sum += of[i] = begins[lane * kEach + i + 1];
    unsigned up_to = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned other = __shfl_up_sync(0xffffffffu, up_to, d);
      if (lane >= unsigned(d)) up_to += other;
    }
    up_to -= sum;
    if (lane == 0) begins[0] = 0;
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) begins[lane * kEach + i + 1] = up_to += of[i];
  }
  __syncthreads();
#pragma unroll 1
  for (unsigned work = blockIdx.x; work < begins[kMaxCtas]; work += gridDim.x) {
    unsigned first = 0;       // the CTA whose item has this group of rows: the last one that begins at or before it (none without groups)
    for (unsigned above = kMaxCtas; above - first > 1;) {
      const unsigned middle = (first + above) / 2;
      if (begins[middle] <= work) first = middle; else above = middle;
    }
    const uint4 a = __ldcg(reinterpret_cast<const uint4*>(notes + first));
    const unsigned pieces = a.x, rows = a.w, head = __ldcg(&notes[first].head);
    const unsigned r = (work - begins[first]) * kJoinRows + tid % kJoinRows, c4 = tid / kJoinRows;
    if (r >= rows) continue;
    const unsigned row = a.y + (a.z + r) / group, q_head = head * group + (a.z + r) % group;
    if (kPrefix && !(int(row) >= starts[0] && int(row) < starts[sequences])) continue;
    const unsigned flat = row * group + (a.z + r) % group;
    float top = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float2 end, const float4 part) {
      float mine_by, other_by;
      join(top, sum, end, mine_by, other_by);
      v.x = v.x * mine_by + part.x * other_by;
      v.y = v.y * mine_by + part.y * other_by;
      v.z = v.z * mine_by + part.z * other_by;
      v.w = v.w * mine_by + part.w * other_by;
    };
#pragma unroll 1
    for (unsigned p0 = 0; p0 < pieces; p0 += kBatch) {
      float2 ends[kBatch];
      float4 sums[kBatch];
#pragma unroll
      for (unsigned b = 0; b < kBatch; ++b) {
        const unsigned p = kPrefix ? min(p0 + b, pieces - 1) : p0 + b;
        if (p >= pieces) continue;
        ends[b] = __ldcg(parts.end(first + p, p == 0, r));
        sums[b] = __ldcg(parts.sum(first + p, p == 0, r, c4));
      }
#pragma unroll
      for (unsigned b = 0; b < kBatch; ++b)
        if (p0 + b < pieces) add(ends[b], sums[b]);
    }
    if (own_only) {
      *own.sum(head, c4, flat) = v;
      if (c4 == 0) *own.end(head, flat) = make_float2(top, sum);
      continue;
    }
    if (kPrefix) add(__ldcg(own.end(head, flat)), __ldcg(own.sum(head, c4, flat)));
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    const bf162 pair[2] = {__floats2bfloat162_rn(v.x * inv, v.y * inv), __floats2bfloat162_rn(v.z * inv, v.w * inv)};
    *reinterpret_cast<uint2*>(o + size_t(row) * o_stride + q_head * kDim + c4 * 4) = *reinterpret_cast<const uint2*>(pair);
  }
}

}  // namespace many

// grid: one CTA an SM (or fewer), block = 384, dynamic shared memory = 512 * head_dim (Q) + stages * 512 * head_dim (keys, values) + 20480 (staging) + 1024.
// own_only: the rows' own sequences' part of prefix attention, left in own_sums and own_ends instead of o.
#define AGI_PAGED_MANY(NAME, HD16, PREFIX)                                                                                              \
  extern "C" __global__ void __launch_bounds__(many::kThreads, 1)                                                                       \
  NAME(const bf16* q, bf16* o, const bf16* k_pool, const bf16* v_pool, const int* starts, const int* lengths, const int* table,         \
       const int* prefix_table, const int* prefix_length, float* own_sums, float* own_ends, float* scratch, many::Note* notes,          \
       unsigned* status, unsigned rows, unsigned sequences, unsigned pages, unsigned page, unsigned width, unsigned prefix_pages,       \
       unsigned q_heads, unsigned kv_heads, unsigned q_stride, unsigned o_stride, unsigned window, unsigned sinks, float scale_log2,    \
       unsigned stages, unsigned least, unsigned own_only) {                                                                            \
    const paged::Batch batch{starts, lengths, table, status, rows, sequences, pages, page, width};                                      \
    many::attention_body<HD16, PREFIX>(q, o, k_pool, v_pool, batch, prefix_table, prefix_length, prefix_pages, own_sums, own_ends,      \
                                       scratch, notes, q_heads, kv_heads, q_stride, o_stride, window, sinks, scale_log2, stages, least, \
                                       own_only);                                                                                       \
  }
AGI_PAGED_MANY(agi_paged_many_bf16_d64, 4, false)
AGI_PAGED_MANY(agi_paged_many_bf16_d128, 8, false)
AGI_PAGED_MANY(agi_paged_prefix_bf16_d64, 4, true)
AGI_PAGED_MANY(agi_paged_prefix_bf16_d128, 8, true)
#undef AGI_PAGED_MANY

// grid: any number of blocks, block = 2 * head_dim; ctas: the CTAs of the launch before, 160 at most.
#define AGI_PAGED_JOIN(NAME, HD16, PREFIX)                                                                                             \
  extern "C" __global__ void __launch_bounds__(many::kJoinRows * HD16 * 4)                                                             \
  NAME(bf16* o, const int* starts, unsigned sequences, float* own_sums, float* own_ends, float* scratch, many::Note* notes,            \
       unsigned ctas, unsigned rows, unsigned q_heads, unsigned kv_heads, unsigned o_stride, unsigned own_only) {                      \
    many::join_body<HD16, PREFIX>(o, starts, sequences, own_sums, own_ends, scratch, notes, ctas, rows, q_heads, kv_heads, o_stride,   \
                                  own_only);                                                                                           \
  }
AGI_PAGED_JOIN(agi_paged_join_bf16_d64, 4, false)
AGI_PAGED_JOIN(agi_paged_join_bf16_d128, 8, false)
AGI_PAGED_JOIN(agi_paged_join_prefix_bf16_d64, 4, true)
AGI_PAGED_JOIN(agi_paged_join_prefix_bf16_d128, 8, true)
#undef AGI_PAGED_JOIN
