// Products with 4-bit weights for few tokens: Y[M, N] = epilogue(X[M, K] . W[N, K]^T), W[n, k] = (code[n, k] - 8) * scale[n, k / group].
//
// Bound by memory: half a byte a weight, and 2 / group bytes of scales.  Codes lie in the order in which the lanes of a warp take them
// (layout.pack_w4): a tile of 16 rows by 64 columns is 512 bytes, 16 a lane.
//
// What an SM can issue stands between them and the products: a tile has to go through in 22 clocks, and integer instructions run at half
// rate (f16 weights take 20 of them and 16 fused multiply-adds a tile: 22.7 us for 37888 x 3584, of which 13 are the bytes' own).  So products
// are of integers (m16n8k32, unsigned weights as rows, signed tokens as columns).  A byte of codes holds row g in its low half and row g + 8
// of the same column in its high half: the low halves alone, one mask a word, are the operand of row g; the bytes as they are, no
// instruction at all, are that of row g + 8, whose sum is then 16 times its own and once row g's, which is taken off again, exactly.
//
// Tokens are 15-bit integers relative to the power of two next to the largest value of their block of 64 columns, which becomes 2^13 .. 2^14: they
// are off by half a unit, 2^-14 of that value at most, and exact where they are 2^-6 of it or more; outputs in bf16 are off by up to 2^-8 of
// theirs.  They go in as two columns, the upper eight bits and the lower seven.  The 8 that is too much of every code is taken off the sums:
// they begin at -8 (or -136) times the sum of the columns.  A block's sums are exact; they are multiplied by the scales and added up in fp32.
//
// That is too little for neighbours of a value thousands of times theirs, whose own weight may be zero.  So a block is one of integers only if each
// eight of its values (what a lane holds of even or of odd columns) has one of 2^-4 of the power of two or more, 2^9 units, in all of the CTA's
// tokens: normal values have, and so have products of two of them but for one block in ten.  Other blocks, and those below 2^-113, where
// the unit would leave fp32, are zero as integers and go through bf16 products besides, exact but for sums in 32 bits: rows of x from L2,
// codes - 8 as bf16 from the ring.  us with such a value in no | one | every block: 37888 x 3584, 1 token 17.9 | 18.6 | 37.9, 8 tokens 30.0 | 30.5 |
// 73.6; 2048 x 11008, 1 token 8.8 | 8.9 | 12.9.
//
// A CTA is one an SM: it lays its part of the tokens (of gridDim.z parts of K) into shared memory once, as the products take them, then two
// teams of eight warps stream row tiles past them.  `ways` warps share the columns of a tile, so that there are tiles for all warps
// or, where rows are few, warps for all columns; a warp that goes on with a tile for long has less to do besides.  Every warp fills a ring
// of its own by bulk copies of `chunk` blocks of 64 columns and their scales.  A ninth warp of the team adds the eight warps' sums and
// finishes their tiles while they are at the next ones.  Parts of K meet in scratch, where the last team to arrive at a tile adds them in
// order, so sums do not depend on who that is.  Weights are no earlier launch's work (`early`): the rings fill before the launch before
// has ended.
//
// Measured in a chain of launches (codes from memory, groups of 64): 37888 x 3584 with 1 token 17.9 us (4.0 TB/s; 17.2 before blocks were looked at
// for uneven values), where the same copies without the products took 12.9 to 13.6; with 4 tokens 18.7, 8 tokens (two groups) 30.0, 16 tokens
// 48.2.  Three teams a CTA were slower (1 token 18.7 to 20.3 where two took 17.4).  Two blocks unrolled, not four: 18.1 to 17.4 at four ways.
#pragma once

#include "attention.cuh"
#include "gemm_tc.cuh"
#include "gemm_simt.cuh"
#include "paged.cuh"

namespace w4 {

constexpr unsigned kWarps = 8, kTeams = 2, kTeamThreads = 288, kThreads = kTeams * kTeamThreads, kTileRows = 16, kBlock = 64, kBlockBytes = 512;
constexpr unsigned kMaxBlocks = 512;       // of a part of K: shared memory holds fewer
constexpr unsigned kMaxStages = 8, kBlockTokens = 512, kBlockOffs = 64;      // bytes of eight columns of tokens, of what their sums begin at
constexpr unsigned kPitch = 20;            // floats from one column of a warp's sums to the next: 16 rows, no bank conflicts
constexpr unsigned kTimeout = 0x700;       // a copy that does not arrive

// Pair i of a word's codes as bf16 weights without their scale: a code in the low bits of 0x4300 is the bf16 128 + code.
__device__ __forceinline__ unsigned weights_of(unsigned word, int i) {
  const unsigned raised = ((word >> (4 * i)) & 0x000f000fu) | 0x43004300u;
  const bf162 pair = __hsub2(*reinterpret_cast<const bf162*>(&raised), __floats2bfloat162_rn(136.f, 136.f));
  return *reinterpret_cast<const unsigned*>(&pair);
}
// D = A B + C: unsigned bytes, signed bytes, exact.
__device__ __forceinline__ void product(int* d, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1, int c0, int c1, int c2, int c3) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}
// The larger of two pairs of bf16 without their signs, NaN above all, as bits.
__device__ __forceinline__ unsigned larger_pair(unsigned a, unsigned b) { return __vmaxu2(a, b); }
// Four values of a token (low: 0 and 1, high: 2 and 3) times `by` as integers, of which the bits from `shift` on under `mask`, in the order 0, 2, 1, 3.
// Added to 1.5 * 2^23 a value is an integer in the low bits of the sum.
__device__ __forceinline__ unsigned piece_of(unsigned low, unsigned high, float by, unsigned shift, unsigned mask) {
  constexpr float kRound = 12582912.f;
  const unsigned v0 = __float_as_uint(fmaf(__uint_as_float(low << 16), by, kRound)), v1 = __float_as_uint(fmaf(__uint_as_float(low & 0xffff0000u), by, kRound));
  const unsigned v2 = __float_as_uint(fmaf(__uint_as_float(high << 16), by, kRound)), v3 = __float_as_uint(fmaf(__uint_as_float(high & 0xffff0000u), by, kRound));
  return __byte_perm(__byte_perm(v0, v2, 0x5410) >> shift, __byte_perm(v1, v3, 0x5410) >> shift, 0x6420) & mask;
}
// Codes, read once: not kept in L1.  A launch before may write codes and scales while this one already lives, so they are no constants of it: read
// with ld.global.nc, behind the wait for that launch, products of 410 tokens were of an earlier run's codes.
__device__ __forceinline__ uint4 stream_load(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// kEights: eights of columns: both pieces of four tokens, or one piece of eight tokens each.  kGroup: columns that share a scale, 32, 64 or 128.
template <int kEights, unsigned kGroup>
__device__ __forceinline__ void body(const bf16* x, const uint4* codes, const bf16* scales, bf16* y, const bf16* bias, const bf16* residual,
                                     float* partial, unsigned* counters, unsigned* status, unsigned M, unsigned N, unsigned K, unsigned ldx,
                                     unsigned ldy, unsigned flags, unsigned ways, unsigned chunk, unsigned stages, unsigned early) {
  constexpr unsigned kTokens = kEights * 4, kColumns = kEights == 1 ? 8 : kTokens, kOutputs = kTileRows * kTokens;      // columns of sums that a warp leaves
  constexpr unsigned kHalves = kGroup == 32 ? 2 : 1;
  extern __shared__ __align__(128) unsigned char w4_smem[];       // rings [warp][stage] | tokens [block][eight][lane][16] | offs [block][half][eight][t][4] | units [block][eight][8]
  __shared__ __align__(16) float sums[kTeams][2][kWarps][kColumns * kPitch];
  __shared__ __align__(8) unsigned long long full[kTeams * kWarps][kMaxStages];
  __shared__ unsigned char apart[kMaxBlocks];       // 1: this block of the part is no block of integers; 2: its values are near the largest there are, too
  const unsigned tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t4 = lane & 3, warp = tid >> 5, team = warp / (kWarps + 1), mate = warp % (kWarps + 1);
  const unsigned tiles = (N + kTileRows - 1) / kTileRows, blocks = K / kBlock, groups = K / kGroup;
  const unsigned per = (blocks + gridDim.z - 1) / gridDim.z, part0 = min(blockIdx.z * per, blocks), part = min(per, blocks - part0);
  // tiles of the team: one for each set of `ways` warps, `step` further on in each round
  const unsigned sets = kWarps / ways, first_tile = (team * gridDim.x + blockIdx.x) * sets, step = kTeams * gridDim.x * sets, slot_bytes = chunk * (kBlockBytes + 64), token0 = blockIdx.y * kTokens, live_tokens = min(M - token0, kTokens);
  uint4* const tokens = reinterpret_cast<uint4*>(w4_smem + kTeams * kWarps * stages * slot_bytes);
  int4* const offs = reinterpret_cast<int4*>(tokens + per * kEights * (kBlockTokens / 16));
  float* const units = reinterpret_cast<float*>(offs + per * kHalves * kEights * (kBlockOffs / 16));
  if (!(paged::aligned16(x) && paged::aligned16(codes) && paged::aligned16(scales))) {
    grid_dependency_wait();
    if (tid == 0) paged::report(status, paged::kMisaligned);
    return;
  }

  // ---- the rings: columns [begin, begin + count) of every tile of the warp's set, `chunk` blocks a copy ----
  const unsigned set = mate / ways, way = mate % ways;
  const unsigned count = mate < kWarps ? part / ways + (way < part % ways ? 1 : 0) : 0, begin = part0 + way * (part / ways) + min(way, part % ways);
  const unsigned ring_of = team * kWarps + min(mate, kWarps - 1), chunks = (count + chunk - 1) / chunk;
  unsigned char* const ring = w4_smem + ring_of * stages * slot_bytes;
  unsigned long long* const bars = full[ring_of];
  unsigned ask_tile = first_tile + set, ask_at = 0;
  auto ask = [&](unsigned s) {      // the next copy in order, into slot s: one lane
    if (count == 0 || ask_tile >= tiles) return;
    const unsigned at = begin + ask_at, held = min(chunk, count - ask_at), from = at * kBlock / kGroup;
    const unsigned scale_bytes = (((at + held) * kBlock + kGroup - 1) / kGroup - from) * 32, slot = tc::smem_u32(ring + s * slot_bytes);
    tc::expect_bytes(&bars[s], held * kBlockBytes + scale_bytes);
    tc::bulk_copy(slot, codes + (size_t(ask_tile) * blocks + at) * 32, held * kBlockBytes, &bars[s]);
    tc::bulk_copy(slot + chunk * kBlockBytes, scales + (size_t(ask_tile) * groups + from) * 16, scale_bytes, &bars[s]);
    ask_at += chunk;
    if (ask_at >= count) {
      ask_at = 0;
      ask_tile += step;
    }
  };
  if (mate < kWarps) {
    if (lane == 0) {
      for (unsigned s = 0; s < stages; ++s) tc::mbar_init(&bars[s], 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
  }
  if (!early) grid_dependency_wait();
  if (mate < kWarps && lane == 0)
    for (unsigned s = 0; s < stages; ++s) ask(s);
  if (early) grid_dependency_wait();
  __syncthreads();

  // ---- the tokens, a block of columns and eight columns of products a warp at a time ----
#pragma unroll 2
  for (unsigned i = warp; i < part * kEights; i += kTeams * (kWarps + 1)) {
    const unsigned block = i / kEights, eight = i % kEights, column = eight * 8 + g;
    const bool lower = column >= kTokens;
    // columns behind the last token repeat it
    const uint4* const from = reinterpret_cast<const uint4*>(x + size_t(min(token0 + column % kTokens, M - 1)) * ldx + (part0 + block) * kBlock + t4 * 8);
    const uint4 v[2] = {from[0], from[4]};
    unsigned pair = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      pair = larger_pair(larger_pair(larger_pair(v[h].x & 0x7fff7fffu, v[h].y & 0x7fff7fffu), larger_pair(v[h].z & 0x7fff7fffu, v[h].w & 0x7fff7fffu)), pair);
    const unsigned least = min(pair & 0xffffu, pair >> 16);      // of the lane's eights the one with the least largest value
    pair = larger_pair(pair, __shfl_xor_sync(0xffffffffu, pair, 1));
    pair = larger_pair(pair, __shfl_xor_sync(0xffffffffu, pair, 2));
    const unsigned peak = max(pair & 0xffffu, pair >> 16), exponent = peak >> 7;
    // 2^13 / 2^exponent: values below 2^14.  A block that is not finite is zero, times NaN
    const unsigned unit = exponent == 255 ? 0u : min(267u - exponent, 253u) << 23;
    const bool uneven = unit && peak && (exponent < 14 || least < (exponent - 4) << 7), any_uneven = __any_sync(0xffffffffu, uneven);
    const bool any_huge = __any_sync(0xffffffffu, unit && exponent >= 240);
    if (lane == 0) apart[block] = any_uneven ? 1 + any_huge : 0;       // the same for both eights, which hold the same tokens
    const float by = __uint_as_float(any_uneven ? 0u : unit);
    const unsigned shift = lower ? 0 : 7, mask = lower ? 0x7f7f7f7fu : 0xffffffffu;
    uint4 piece = make_uint4(0u, 0u, 0u, 0u);
    if (unit) piece = make_uint4(piece_of(v[0].x, v[0].y, by, shift, mask), piece_of(v[0].z, v[0].w, by, shift, mask), piece_of(v[1].x, v[1].y, by, shift, mask),
                                 piece_of(v[1].z, v[1].w, by, shift, mask));
    __syncwarp();
    tokens[i * 32 + lane] = piece;
    constexpr unsigned kOnes = 0x01010101u;
    int c[2][4];
    product(c[0], kOnes, kOnes, kOnes, kOnes, piece.x, piece.y, 0, 0, 0, 0);
    if (kGroup == 32) product(c[1], kOnes, kOnes, kOnes, kOnes, piece.z, piece.w, 0, 0, 0, 0);
    else product(c[0], kOnes, kOnes, kOnes, kOnes, piece.z, piece.w, c[0][0], c[0][1], c[0][2], c[0][3]);
    if (g == 0) {
#pragma unroll
      for (unsigned h = 0; h < kHalves; ++h)
        offs[((block * kHalves + h) * kEights + eight) * 4 + t4] = make_int4(-8 * c[h][0], -8 * c[h][1], -136 * c[h][0], -136 * c[h][1]);
    }
    if (t4 == 0) units[i * 8 + g] = unit ? __uint_as_float((254u << 23) - unit) * (lower ? 1.f : 128.f) : __uint_as_float(0x7fc00000u);
  }
  __syncthreads();
  // instructions of a whole warp, behind branches of single lanes
  auto meet = [&](unsigned bar) {
    __syncwarp();
    asm volatile("bar.sync %0, 288;" ::"r"(1 + team * 4 + bar) : "memory");
  };
  auto pass = [&](unsigned bar) {
    __syncwarp();
    asm volatile("bar.arrive %0, 288;" ::"r"(1 + team * 4 + bar) : "memory");
  };
  unsigned which = 0;

  if (mate < kWarps) {
    unsigned s = 0, phase = 0;
    bool first = true, gave_up = false;
#pragma unroll 1
    for (unsigned tile = first_tile; tile < tiles; tile += step) {
      float sum[kEights][4];
#pragma unroll
      for (int t = 0; t < kEights; ++t) sum[t][0] = sum[t][1] = sum[t][2] = sum[t][3] = 0.f;
#pragma unroll 1
      for (unsigned at = begin, left = tile + set < tiles ? count : 0; left > 0;) {
        if (!gave_up && !tc::mbar_wait(&bars[s], phase, status, kTimeout | s)) gave_up = true;
        __syncwarp();
        const unsigned held = min(chunk, left);
        const uint4* code_at = reinterpret_cast<const uint4*>(ring + s * slot_bytes) + lane;
        const unsigned char* scale_at = ring + s * slot_bytes + chunk * kBlockBytes + g * 4;
        const uint4* tokens_at = tokens + (at - part0) * kEights * 32 + lane;
        const int4* offs_at = offs + (at - part0) * kHalves * kEights * 4 + t4;
        const float2* units_at = reinterpret_cast<const float2*>(units + (at - part0) * kEights * 8) + t4;
        // of groups of 128 columns a block has half of one: the first or, with `odd`, the second
        const unsigned odd = kGroup == 128 ? (at & 1) * 32 : 0;
        // block b of those at the pointers: its codes times its tokens
        auto multiply = [&](int b) {
          const uint4 c = code_at[b * 32];
          uint4 v[kEights];
#pragma unroll
          for (int t = 0; t < kEights; ++t) v[t] = tokens_at[(b * kEights + t) * 32];
          int all[kEights][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const unsigned w0 = h ? c.z : c.x, w1 = h ? c.w : c.y, a0 = w0 & 0x0f0f0f0fu, a2 = w1 & 0x0f0f0f0fu;
#pragma unroll
            for (int t = 0; t < kEights; ++t) {
              const unsigned b0 = h ? v[t].z : v[t].x, b1 = h ? v[t].w : v[t].y;
              if (h == 0 || kGroup == 32) {
                const int4 off = offs_at[((b * int(kHalves) + h) * kEights + t) * 4];
                product(all[t], a0, w0, a2, w1, b0, b1, off.x, off.y, off.z, off.w);
              } else {
                product(all[t], a0, w0, a2, w1, b0, b1, all[t][0], all[t][1], all[t][2], all[t][3]);
              }
            }
            if (h == 0 && kGroup != 32) continue;
            const unsigned in_slot = kGroup == 32 ? (2 * b + h) * 32 : kGroup == 64 ? b * 32 : (b / 2) * 32 + (b % 2 ? odd : 0);
            const unsigned scale = *reinterpret_cast<const unsigned*>(scale_at + in_slot);
            const float low = __uint_as_float(scale << 16), high = __uint_as_float(scale & 0xffff0000u) * 0.0625f;
#pragma unroll
            for (int t = 0; t < kEights; ++t) {
              const float2 unit = units_at[(b * kEights + t) * 4];
              sum[t][0] = fmaf(float(all[t][0]), low * unit.x, sum[t][0]);
              sum[t][1] = fmaf(float(all[t][1]), low * unit.y, sum[t][1]);
              sum[t][2] = fmaf(float(all[t][2] - all[t][0]), high * unit.x, sum[t][2]);
              sum[t][3] = fmaf(float(all[t][3] - all[t][1]), high * unit.y, sum[t][3]);
            }
          }
        };
        constexpr unsigned kRowBytes = 32 * kBlock;      // of scales, a block: kRowBytes / kGroup
        unsigned todo = held;
#pragma unroll 1
        for (; todo >= 2; todo -= 2) {
#pragma unroll
          for (int b = 0; b < 2; ++b) multiply(b);
          code_at += 2 * 32;
          scale_at += 2 * kRowBytes / kGroup;
          tokens_at += 2 * kEights * 32;
          offs_at += 2 * kHalves * kEights * 4;
          units_at += 2 * kEights * 4;
        }
        if (todo) multiply(0);
        for (unsigned left_apart = __ballot_sync(0xffffffffu, lane < held && apart[at - part0 + lane]); left_apart; left_apart &= left_apart - 1) {
          const unsigned b = __ffs(left_apart) - 1, group0 = at * kBlock / kGroup;
          const uint4 c = reinterpret_cast<const uint4*>(ring + s * slot_bytes)[b * 32 + lane];
          // column g of the products is token g: columns 2 t .. and 2 t + 8 .. of two products are the lane's eight in a row of codes and tokens
          uint4 v[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
          if (g < live_tokens) {
            const uint4* const from = reinterpret_cast<const uint4*>(x + size_t(token0 + g) * ldx + (at + b) * kBlock + t4 * 8);
            v[0] = from[0];
            v[1] = from[4];
          }
          // 64 products of up to 8 times a value of 2^113 or more stay finite times 2^-10
          const bool huge = apart[at - part0 + b] == 2;
          const float back = huge ? 0x1p10f : 1.f;
          const bf162 small = __floats2bfloat162_rn(huge ? 0x1p-10f : 1.f, huge ? 0x1p-10f : 1.f);
          auto weights = [&](unsigned word, int i) {
            const unsigned pair = weights_of(word, i);
            const bf162 less = __hmul2(*reinterpret_cast<const bf162*>(&pair), small);
            return *reinterpret_cast<const unsigned*>(&less);
          };
          float all[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const unsigned w0 = h ? c.z : c.x, w1 = h ? c.w : c.y;
            skinny_mma_bf16(all, weights(w0, 0), weights(w0, 1), weights(w0, 2), weights(w0, 3), v[h].x, v[h].y);
            skinny_mma_bf16(all, weights(w1, 0), weights(w1, 1), weights(w1, 2), weights(w1, 3), v[h].z, v[h].w);
            if (h == 0 && kGroup != 32) continue;
            const unsigned group = ((at + b) * kBlock + h * 32) / kGroup - group0;
            const unsigned scale = *reinterpret_cast<const unsigned*>(ring + s * slot_bytes + chunk * kBlockBytes + group * 32 + g * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              sum[0][i] = fmaf(all[i] * __uint_as_float(i < 2 ? scale << 16 : scale & 0xffff0000u), back, sum[0][i]);
              all[i] = 0.f;
            }
          }
        }
        __syncwarp();       // the slot has been read
        if (lane == 0) ask(s);
        if (++s == stages) { s = 0; phase ^= 1; }
        at += held;
        left -= held;
      }
      if (!first) meet(2 + which);       // the sums that lay here have been taken
#pragma unroll
      for (unsigned t = 0; t < kColumns / 8; ++t)
#pragma unroll
        for (unsigned i = 0; i < 4; ++i)
          sums[team][which][mate][(t * 8 + 2 * t4 + (i & 1)) * kPitch + g + (i >> 1) * 8] = kEights == 1 ? sum[t][i] : sum[t][i] + sum[t + kEights / 2][i];
      pass(which);
      if (which) first = false;
      which ^= 1;
    }
    return;
  }

  // ---- the ninth warp: sums of the eight, parts of K, outputs ----
  const unsigned live = live_tokens * kTileRows;
#pragma unroll 1
  for (unsigned tile0 = first_tile; tile0 < tiles; tile0 += step) {
    meet(which);
#pragma unroll 1
    for (unsigned in = 0; in < sets; ++in) {
      const unsigned tile = tile0 + in;
      const float* const from = sums[team][which][in * ways];
      float* const to = partial + ((size_t(tile) * gridDim.y + blockIdx.y) * gridDim.z + blockIdx.z) * kOutputs;
#pragma unroll
      for (unsigned o = 0; o < kOutputs / 32; ++o) {
        const unsigned i = o * 32 + lane, m = token0 + i / kTileRows, n = tile * kTileRows + i % kTileRows;
        if (i >= live || n >= N) continue;
        float v = 0.f;
#pragma unroll 4
        for (unsigned w = 0; w < ways; ++w) {
          const float* const at = from + w * (kColumns * kPitch) + i / kTileRows * kPitch + i % kTileRows;
          v += kEights == 1 ? at[0] + at[kTokens * kPitch] : at[0];
        }
        if (gridDim.z == 1) gemm_store(v, m, n, y, ldy, bias, residual, 1.f, flags);
        else to[i] = v;
      }
    }
    // whoever writes here next waits for this; nobody does behind the last two rounds
    if (tile0 + 2 * step < tiles) pass(2 + which);
    which ^= 1;
    if (gridDim.z == 1) continue;
    __threadfence();
    __syncwarp();
    // a lane a tile: is this the last part?
    unsigned last = 0;
    if (lane < sets && tile0 + lane < tiles) last = atomicAdd(&counters[(tile0 + lane) * gridDim.y + blockIdx.y], 1u) == gridDim.z - 1;
    __threadfence();
    for (unsigned ready = __ballot_sync(0xffffffffu, last); ready; ready &= ready - 1) {
      const unsigned tile = tile0 + __ffs(ready) - 1;
      const float* const parts = partial + (size_t(tile) * gridDim.y + blockIdx.y) * gridDim.z * kOutputs;
#pragma unroll 1
      for (unsigned i = lane; i < live; i += 32) {
        const unsigned m = token0 + i / kTileRows, n = tile * kTileRows + i % kTileRows;
        if (n >= N) continue;
        float all = 0.f;
#pragma unroll 4
        for (unsigned z = 0; z < gridDim.z; ++z) all += __ldcg(parts + z * kOutputs + i);
        gemm_store(all, m, n, y, ldy, bias, residual, 1.f, flags);
      }
      if (lane == 0) counters[tile * gridDim.y + blockIdx.y] = 0;      // as the next launch expects it
    }
  }
}

}  // namespace w4

// grid = (CTAs that share the row tiles, tokens / 4 T, parts of K), block = 576, dynamic shared memory = 16 warps * stages * chunk * 576 and, for
// each 64 columns of a part, T * 608 (groups of 32: T * 672).  ways: 1, 2, 4 or 8; chunk: a multiple of 4; stages: at most 8.  K a multiple of
// 64 and of the group; ldx a multiple of 8.  counters: a word for each row tile and y of the grid, zero between launches.
#define AGI_GEMM_W4(T, GROUP)                                                                                                             \
  extern "C" __global__ void __launch_bounds__(w4::kThreads, 1)                                                                           \
  agi_gemm_w4_g##GROUP##_t##T(const bf16* x, const uint4* codes, const bf16* scales, bf16* y, const bf16* bias, const bf16* residual,     \
                              float* partial, unsigned* counters, unsigned* status, unsigned M, unsigned N, unsigned K, unsigned ldx,     \
                              unsigned ldy, unsigned flags, unsigned ways, unsigned chunk, unsigned stages, unsigned early) {             \
    w4::body<T, GROUP>(x, codes, scales, y, bias, residual, partial, counters, status, M, N, K, ldx, ldy, flags, ways, chunk, stages,     \
                       early);                                                                                                            \
  }
AGI_GEMM_W4(1, 32)
AGI_GEMM_W4(1, 64)
AGI_GEMM_W4(1, 128)
AGI_GEMM_W4(2, 32)
AGI_GEMM_W4(2, 64)
AGI_GEMM_W4(2, 128)
#undef AGI_GEMM_W4

// The weights as bf16, [N, K] in rows, for products of many tokens: (code - 8) * scale, rounded.  Bound by memory: a warp a tile of 16
// rows by 64 columns, a lane 16 bytes of codes, which leave through shared memory, four rows of 128 bytes a store (a store of eight
// rows' 64 bytes from the lanes that have them took the load and store unit 70 clocks: 1.5 TB/s).
// grid: any number of blocks, block = 256.
extern "C" __global__ void __launch_bounds__(256)
agi_dequantize_w4_bf16(const uint4* codes, const bf16* scales, bf16* out, unsigned* status, unsigned N, unsigned K, unsigned group, unsigned early) {
  constexpr unsigned kPitch = 144;       // bytes of a row of a tile: 128, and 16 against bank conflicts
  __shared__ __align__(16) unsigned char staged[8][w4::kTileRows * kPitch];
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3, blocks = K / w4::kBlock, groups = K / group;
  const unsigned tiles = (N + w4::kTileRows - 1) / w4::kTileRows, items = tiles * blocks, stride = gridDim.x * 8;
  const bool aligned = paged::aligned16(codes) && paged::aligned16(scales) && paged::aligned16(out);
  if (!early) grid_dependency_wait();
  unsigned item = blockIdx.x * 8 + warp;
  uint4 next = make_uint4(0u, 0u, 0u, 0u);
  if (aligned && item < items) next = w4::stream_load(codes + size_t(item) * 32 + lane);
  if (early) grid_dependency_wait();
  if (!aligned) {
    if (threadIdx.x == 0) paged::report(status, paged::kMisaligned);
    return;
  }
#pragma unroll 1
  for (; item < items; item += stride) {
    const unsigned tile = item / blocks, block = item - tile * blocks;
    const uint4 c = next;
    if (item + stride < items) next = w4::stream_load(codes + size_t(item + stride) * 32 + lane);
    const unsigned* const unit = reinterpret_cast<const unsigned*>(scales) + size_t(tile) * groups * 8 + g;
    const unsigned first = unit[block * w4::kBlock / group * 8], second = unit[(block * w4::kBlock + 32) / group * 8];
    __syncwarp();       // the tile before has left
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned word[2] = {h ? c.z : c.x, h ? c.w : c.y}, s = h ? second : first;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float by = __uint_as_float(half ? s & 0xffff0000u : s << 16);
        Bf16x8 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned pair = w4::weights_of(word[i >> 1], 2 * (i & 1) + half);
          v.v[i] = __floats2bfloat162_rn(__uint_as_float(pair << 16) * by, __uint_as_float(pair & 0xffff0000u) * by);
        }
        *reinterpret_cast<Bf16x8*>(staged[warp] + (g + half * 8) * kPitch + h * 64 + t4 * 16) = v;
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned row = i * 4 + lane / 8, n = tile * w4::kTileRows + row;
      if (n < N)
        *reinterpret_cast<uint4*>(out + size_t(n) * K + block * w4::kBlock + (lane & 7) * 8) =
            *reinterpret_cast<const uint4*>(staged[warp] + row * kPitch + (lane & 7) * 16);
    }
  }
}
