// Attention of few query rows (single tokens, short runs) over the 4-bit cache of kv4.cuh.
//
// out = softmax(scale * q K^T) V. A sequence's new tokens are the last of its cached ones: new token j of n at length L
// sees cache indices 0 .. L - n + j. One cluster of CTAs per (sequence, key head), for up to eight query rows; its warps
// take tiles of keys in turn, each with a running maximum, sum and output of its own (fp32), joined over the CTA and
// then over the cluster through distributed shared memory: no workspace, one launch.
//
// A row (token j, head h of the g that share the key head) is number j * g + h. Matrix products are
// mma.m16n8k16 with KEYS as the 16 rows and query rows as the 8 columns: for a few rows that wastes half as much as the
// other way round, and a lane's operand registers come straight from one aligned word of codes, see kv4.cuh:
//   word & 0x000f000f, word & 0x00f000f0 (and the same of word >> 8) are pairs of f16 subnormals n * 2^-24, n * 2^-20:
//   exact operands for one logical instruction per two codes. The factor 16 of every other pair is taken out of q
//   beforehand (scores) or out of the result (output).
// Scores: S = sum over groups of s_k * (q . n) + (c_k - 8 s_k) * sum(q), exact codes, q scaled to [1, 2) per row, fp32.
// Output: P' = p * s rounded to f16 once, times the codes; the centres' share p * c is summed in fp32. The products with n
// and with the offset 8 share the rounded P', so its rounding weighs on the centred codes only. p runs up to 8 (the
// maximum is taken 3 higher in log2; the sum carries the same factor): P' stays below 8 * 7648 < 65504 whatever the steps,
// and is a normal f16 number, with its full eleven bits, down to p s = 2^-17 of the largest p.
//
// COLS > 0 (rows x groups <= 4 COLS): a column belongs to one row and one GROUP of dims, with q zero outside it. One chain of
// products then leaves each group's part in a column of its own, every lane applies one group's step and centre instead
// of all, and the parts meet by one or two exchanges; likewise one set of P' columns serves all groups' output products.
// COLS = 1 keeps to the even columns, so a lane has one row instead of two.
// What is left is mostly the unpacking (88 of about 150 instructions per 16 tokens of 128 dims; about 250 without).
//
// Each warp has a ring of bulk copies to itself (no barrier among warps before the join): one copy per tile where a page
// holds whole tiles, else one per block. 128 registers, 16 warps per SM; 20 or 24 warps with fewer registers were no faster.
// Measured: 256 sequences of up to 1024 tokens, 12 heads of 64: 50 us = 3.8 TB/s (the slope from 512 to 1024 tokens is
// 5.5 TB/s; the rest is the start and the join of 256 x 12 short clusters); 4 sequences of 131k tokens, 32 heads on 8 of 128:
// 180 us = 3.0 TB/s, bound by issue (52 % of the slots; logical instructions run at half rate) on the SMs that have two
// CTAs of a cluster of eight. Clusters of 9 to 16 pack worse onto the GPU's partitions (204 - 231 us).
#pragma once
#include <type_traits>

#include "kv4.cuh"

namespace crl {

struct Kv4AttentionParams {
  const uint8_t* pages;
  Kv4Table table;
  const int32_t* lengths;     // [seqs] cached tokens, the new ones included
  const int32_t* cu;          // [seqs + 1] first query row of each sequence; null: one token each
  int32_t seqs, kv_heads, group;   // group: query heads per key head
  int32_t max_tokens;         // most new tokens of a sequence
  int32_t row_tiles;
  Kv4Divisor by_group;
  int64_t tokens;             // token rows of q and out
  const void* q;
  void* out;
  int64_t q_tok, q_head, o_tok, o_head;
  int32_t vec_q;
  int32_t pair_o, vec_o;      // output rows 4-byte / 16-byte aligned
  int32_t whole_tiles;        // pages hold whole tiles of the kernel
  float scale_log2;           // softmax scale * log2(e)
  int* status;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a b, without an accumulator to clear
__device__ __forceinline__ void mma_f16_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// number of this CTA's cluster along the grid's x axis
__device__ __forceinline__ uint32_t cluster_id_x() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size_x() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float cluster_ld_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], const uint8_t* p) {
  if constexpr (N == 1) w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (N == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
  else { const uint4 v = *reinterpret_cast<const uint4*>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
}

template <int HD, int WARPS>
struct Kv4AttnShape {
  static constexpr int kTile = HD == 128 ? 2 : 4;                  // blocks of a tile
  static constexpr int kStages = HD == 32 ? 4 : 2;                 // about 160 KB of an SM's shared memory for its 16 warps
  static constexpr int kStage = kTile * kv4_block_bytes(HD);
  static constexpr int kRows = 8;
  static constexpr int kRing = WARPS * kStages * kStage;
  static constexpr int kPart = kRows * (HD + 2) * 4;               // a warp's output, maximum and sum
  static constexpr int kJoin = (WARPS + 1) * kPart;                // the warps' and the CTA's
  static constexpr int kBytes = (kRing > kJoin ? kRing : kJoin) + WARPS * kStages * 8;
};

template <typename T, int HD, int COLS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS) kv4_attention_kernel(const Kv4AttentionParams p) {
  using Shape = Kv4AttnShape<HD, WARPS>;
  constexpr int STAGES = Shape::kStages, TB = Shape::kTile, KEYS = 16 * TB, ALL = (1 << TB) - 1;
  constexpr int G = HD / 32, MT = HD / 16, BB = kv4_block_bytes(HD), ROWS = Shape::kRows;
  constexpr bool PACKED = COLS != 0;
  constexpr int C = COLS == 1 ? 1 : 2;        // live columns of a lane: 2t, and 2t + 1
  constexpr int GA = PACKED ? 1 : G;          // groups that a lane applies steps and centres of
  constexpr int PER = PACKED ? 4 / G : 4;     // lanes t that share a group's columns
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int splits = cluster_size_x(), rank = cluster_ctarank();
  const int head = blockIdx.y, seq = blockIdx.z;
  uint8_t* ring = smem + warp * STAGES * Shape::kStage;
  const uint32_t bars = smem_u32(smem + Shape::kBytes - WARPS * STAGES * 8) + warp * STAGES * 8;
  const int my_group = PACKED ? t / PER : 0;             // of the columns 2t, 2t + 1
  const int col_row = C * (t % PER);                     // the row of column 2t; 2t + 1: the next

  // the first tiles' pages are asked for together with the sequence's length and its run of new tokens
  const int first = rank * WARPS + warp, step = splits * WARPS;
  const int32_t* pages_of = p.table.table + seq * p.table.stride;
  uint32_t ahead[STAGES];
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    ahead[s] = lane < (p.whole_tiles ? 1 : TB) ? kv4_block_of(p.table, pages_of, (first + s * step) * TB + lane) : kNoBlock;
  int len = p.lengths[seq];
  const int64_t q0 = p.cu != nullptr ? p.cu[seq] : seq;
  int run = p.cu != nullptr ? p.cu[seq + 1] - p.cu[seq] : 1;
  const int64_t room = static_cast<int64_t>(p.table.width) * p.table.blocks * kKv4Block;
  if (len > room) {
    if (threadIdx.x == 0) kv4_report(p.status, kDevKv4Table);
    len = static_cast<int>(room);
  }
  const int before = len - max(run, 0);      // cache indices in front of the new tokens
  if (q0 < 0 || run < 0 || q0 + run > p.tokens || run > p.max_tokens) {
    if (threadIdx.x == 0) kv4_report(p.status, kDevKv4Run);
    run = q0 < 0 || run < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(min(run, p.max_tokens)), max(p.tokens - q0, int64_t{0})));
  }
  const int live = run * p.group;                        // rows, at most eight
  if (live <= 0) return;                                 // the same for every CTA of the cluster
  const int seen_most = max(0, min(len, before + run)), seen_least = max(0, before + 1);
  const int tiles = (seen_most + KEYS - 1) / KEYS, blocks = (seen_most + kKv4Block - 1) / kKv4Block;

  if (lane < STAGES) mbar_init(bars + lane * 8, 1);
  mbar_fence_init();
  __syncwarp();

  uint32_t held = 0;      // four bits per stage: which blocks of the tile are there
  const uint8_t* head_pages = p.pages + static_cast<size_t>(head) * p.table.blocks * BB;
  // lane b looks block b of a tile up (well before it is wanted: the table lies in global memory) and copies it; where
  // pages hold whole tiles lane 0 does so for all
  const int lookers = p.whole_tiles ? 1 : TB;
  auto issue = [&](uint32_t at, int tile, int stage) {
    if (lane < min(lookers, blocks - tile * TB)) {
      if (at == kNoBlock) kv4_report(p.status, kDevKv4Table);
    } else {
      at = kNoBlock;
    }
    uint32_t there = __ballot_sync(0xffffffffu, at != kNoBlock);
    const uint32_t to = smem_u32(ring + stage * Shape::kStage), bar = bars + stage * 8;
    if (p.whole_tiles) {
      const int n = min(TB, blocks - tile * TB);
      there = there != 0 ? (1u << n) - 1 : 0u;
      if (lane == 0) {
        mbar_expect_tx(bar, there != 0 ? n * BB : 0);
        if (there != 0) bulk_load(to, head_pages + static_cast<size_t>(at) * BB, n * BB, bar);
      }
    } else {
      if (lane == 0) mbar_expect_tx(bar, __popc(there) * BB);
      __syncwarp();
      if (at != kNoBlock) bulk_load(to + lane * BB, head_pages + static_cast<size_t>(at) * BB, BB, bar);
    }
    held = (held & ~(15u << (4 * stage))) | (there << (4 * stage));
  };
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    if (first + s * step < tiles) issue(ahead[s], first + s * step, s);

  // queries as the B operand: this lane's column is r, scaled to [1, 2) by a power of two; nibbles 1, 3, 5, 7 of a word
  // come 16 times too large
  uint32_t qf[G][4];
  float qsum[2][GA], kcol[2];      // per column 2t, 2t + 1: sum(q) * 2^-24 of the groups and the factor of S, >= 0
  int limit[2];
  {
    const int row = PACKED ? C * ((r >> 1) % PER) + (r & 1) : r, its = PACKED ? (r >> 1) / PER : 0;
    const int tok = kv4_div(row, p.by_group);
    const bool on = row < live && (r & 1) < C;
    const T* src = static_cast<const T*>(p.q) + (q0 + tok) * p.q_tok + static_cast<int64_t>(head * p.group + row - tok * p.group) * p.q_head;
    float x[G][8], big = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (on) kv4_load8(src + 32 * g + 8 * t, p.vec_q, x[g]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!on) x[g][i] = 0.0f;
        big = fmaxf(big, fabsf(x[g][i]));
      }
    }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // exponent of the largest; 100 bounds the factors below (2^(24 + 100) is a finite fp32)
    const int e = big > 0.0f ? min(100, max(-100, static_cast<int>(__float_as_uint(big) >> 23) - 127)) : 0;
    // a negative scale is taken into q, so that the largest score is the largest product
    const float down = copysignf(__uint_as_float(static_cast<uint32_t>(127 - e) << 23), p.scale_log2);
    float sums[GA];
#pragma unroll
    for (int g = 0; g < GA; ++g) sums[g] = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const bool mine = !PACKED || g == its;
      float all = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[g][i] = mine ? x[g][i] * down : 0.0f;
        all += x[g][i];
      }
      sums[PACKED ? 0 : g] += all;
      qf[g][0] = pack_f16(x[g][0], x[g][4]);
      qf[g][1] = pack_f16(x[g][1] * 0.0625f, x[g][5] * 0.0625f);
      qf[g][2] = pack_f16(x[g][2], x[g][6]);
      qf[g][3] = pack_f16(x[g][3] * 0.0625f, x[g][7] * 0.0625f);
    }
#pragma unroll
    for (int g = 0; g < GA; ++g) {
      sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
      sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
    }
    // never zero, so that a hidden score stays at minus infinity
    const float factor = fmaxf(__uint_as_float(static_cast<uint32_t>(127 + 24 + e) << 23) * fabsf(p.scale_log2), 1e-35f);
    const int lim = on ? before + tok + 1 : 0;
    // lane (r, t) needs columns 2t and 2t + 1: lanes 4 * (2t) and 4 * (2t + 1) hold them
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int from = 4 * (2 * t + c);
      kcol[c] = __shfl_sync(0xffffffffu, factor, from);
      limit[c] = __shfl_sync(0xffffffffu, lim, from);
#pragma unroll
      for (int g = 0; g < GA; ++g) qsum[c][g] = __shfl_sync(0xffffffffu, sums[g], from) * (1.0f / 16777216.0f);
    }
  }

  // ones: -8 sum(P'). PACKED: elements 0, 1. Else of groups 2i (elements 0, 1) and 2i + 1 (2, 3)
  float acc[MT][4], ones[(GA + 1) / 2][4], centre[GA][2], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[m][i] = 0.0f;
#pragma unroll
  for (int g = 0; g < GA; ++g) {
    ones[g / 2][0] = ones[g / 2][1] = ones[g / 2][2] = ones[g / 2][3] = 0.0f;
    centre[g][0] = centre[g][1] = 0.0f;
  }

  const int kr = (r >> 1) + 4 * (r & 1);      // row of a block that operand row r stands for; r + 8: kr + 8
  // address of the (s, c) words that a lane applies, in a row of G of them
  auto scales = [&](uint32_t (&m)[GA], const uint8_t* row) {
    if constexpr (PACKED) m[0] = *reinterpret_cast<const uint32_t*>(row + my_group * 4);
    else lds_words<GA>(m, row);
  };
  bool fine = true;
  uint32_t phase = 0;

  auto consume = [&](auto masked_tag, int tile, int stage) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const uint8_t* base = ring + stage * Shape::kStage;
    // scores of the tile: keys kr, kr + 8 of each block, columns 2t, 2t + 1
    float sc[TB][4];
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      const uint8_t* blk = base + b * BB;
      uint32_t w0[G], w1[G], m0[GA], m1[GA];
      lds_words<G>(w0, blk + kr * (HD / 2) + t * (G * 4));
      lds_words<G>(w1, blk + (kr + 8) * (HD / 2) + t * (G * 4));
      scales(m0, blk + 8 * HD + kr * (G * 4));
      scales(m1, blk + 8 * HD + (kr + 8) * (G * 4));
      float d[4];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t x0 = w0[g] & 0x000f000fu, x1 = w1[g] & 0x000f000fu, x2 = w0[g] & 0x00f000f0u, x3 = w1[g] & 0x00f000f0u;
        if (!PACKED || g == 0) mma_f16_16816_first(d, x0, x1, x2, x3, qf[g][0], qf[g][1]);
        else mma_f16_16816(d, x0, x1, x2, x3, qf[g][0], qf[g][1]);
        mma_f16_16816(d, (w0[g] >> 8) & 0x000f000fu, (w1[g] >> 8) & 0x000f000fu, (w0[g] >> 8) & 0x00f000f0u,
                      (w1[g] >> 8) & 0x00f000f0u, qf[g][2], qf[g][3]);
        if (PACKED && g + 1 < G) continue;
        const int ga = PACKED ? 0 : g;
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&m0[ga]));
        const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&m1[ga]));
        const float ca = fmaf(-8.0f, a.x, a.y), cc = fmaf(-8.0f, c.x, c.y);
#pragma unroll
        for (int i = 0; i < 4; i += 3 - C) {
          const float s = i < 2 ? a.x : c.x, o = i < 2 ? ca : cc;
          sc[b][i] = fmaf(s, d[i], ga == 0 ? o * qsum[i & 1][ga] : fmaf(o, qsum[i & 1][ga], sc[b][i]));
        }
      }
      if constexpr (PACKED && G > 1) {
#pragma unroll
        for (int i = 0; i < 4; i += 3 - C) {
          if (G == 4) sc[b][i] += __shfl_xor_sync(0xffffffffu, sc[b][i], 1);
          sc[b][i] += __shfl_xor_sync(0xffffffffu, sc[b][i], 2);
        }
      }
    }
    const uint32_t there = (held >> (4 * stage)) & ALL;
    // running maximum per column
    float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int i = 0; i < 4; i += 3 - C) {
        if (MASKED) {
          const int key = tile * KEYS + b * 16 + kr + (i >> 1) * 8;
          if (key >= limit[i & 1] || !((there >> b) & 1u)) sc[b][i] = -INFINITY;
        }
        most[i & 1] = fmaxf(most[i & 1], sc[b][i]);
      }
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int m = 4; m < 32; m <<= 1) most[c] = fmaxf(most[c], __shfl_xor_sync(0xffffffffu, most[c], m));
      most[c] = fmaxf(top[c], fmaf(most[c], kcol[c], -3.0f));      // the maximum in log2 units, less 3
    }
    if (__any_sync(0xffffffffu, most[0] > top[0] || (C == 2 && most[1] > top[1]))) {
      float alpha[2];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        alpha[c] = top[c] == -INFINITY ? 0.0f : exp2_approx(top[c] - most[c]);
        top[c] = most[c];
        sum[c] *= alpha[c];
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; i += 3 - C) acc[m][i] *= alpha[i & 1];
#pragma unroll
      for (int g = 0; g < GA; ++g)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          ones[g / 2][2 * (g & 1) + c] *= alpha[c];
          centre[g][c] *= alpha[c];
        }
    }
    const float off[2] = {top[0] == -INFINITY ? 0.0f : top[0], top[1] == -INFINITY ? 0.0f : top[1]};
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int i = 0; i < 4; i += 3 - C) {
        sc[b][i] = exp2_approx(fmaf(sc[b][i], kcol[i & 1], -off[i & 1]));
        sum[i & 1] += sc[b][i];
      }
    // output
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      uint32_t pf[GA][2], v0[GA], v1[GA];
      scales(v0, base + b * BB + 18 * HD + kr * (G * 4));
      scales(v1, base + b * BB + 18 * HD + (kr + 8) * (G * 4));
#pragma unroll
      for (int g = 0; g < GA; ++g) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v0[g]));
        const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&v1[g]));
        const float* x = sc[b];
        float y[4] = {x[0] * a.x, C == 2 ? x[1] * a.x : 0.0f, x[2] * c.x, C == 2 ? x[3] * c.x : 0.0f};
        float z[4] = {a.y, a.y, c.y, c.y};
        if (MASKED) {      // a hidden key's row may hold anything
#pragma unroll
          for (int i = 0; i < 4; i += 3 - C) {
            const int key = tile * KEYS + b * 16 + kr + (i >> 1) * 8;
            if (key >= limit[i & 1] || !((there >> b) & 1u)) y[i] = z[i] = 0.0f;
          }
        }
        centre[g][0] = fmaf(x[0], z[0], fmaf(x[2], z[2], centre[g][0]));
        if (C == 2) centre[g][1] = fmaf(x[1], z[1], fmaf(x[3], z[3], centre[g][1]));
        pf[g][0] = transpose_8x8(pack_f16(y[0], y[1]));
        pf[g][1] = transpose_8x8(pack_f16(y[2], y[3]));
        if (g & 1) mma_f16_16816(ones[g / 2], 0u, 0x80088008u, 0u, 0x80088008u, pf[g][0], pf[g][1]);
        else mma_f16_16816(ones[g / 2], 0x80088008u, 0u, 0x80088008u, 0u, pf[g][0], pf[g][1]);
      }
      const uint8_t* blk = base + b * BB + 10 * HD;
      if constexpr (HD == 32) {
        const uint16_t* rowp = reinterpret_cast<const uint16_t*>(blk) + r;
        const uint32_t x = rowp[t * 8] | (static_cast<uint32_t>(rowp[(t + 4) * 8]) << 16);
        const uint32_t y = rowp[(t + 8) * 8] | (static_cast<uint32_t>(rowp[(t + 12) * 8]) << 16);
        mma_f16_16816(acc[0], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, pf[0][0], pf[0][1]);
        mma_f16_16816(acc[1], (x >> 8) & 0x000f000fu, (x >> 8) & 0x00f000f0u, (y >> 8) & 0x000f000fu, (y >> 8) & 0x00f000f0u, pf[0][0],
                      pf[0][1]);
      } else {
        constexpr int W = HD / 64;
        uint32_t wa[W], wb[W], wc[W], wd[W];
        lds_words<W>(wa, blk + t * (HD / 2) + r * (W * 4));
        lds_words<W>(wb, blk + (t + 4) * (HD / 2) + r * (W * 4));
        lds_words<W>(wc, blk + (t + 8) * (HD / 2) + r * (W * 4));
        lds_words<W>(wd, blk + (t + 12) * (HD / 2) + r * (W * 4));
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t x = __byte_perm(wa[w], wb[w], half ? 0x7632 : 0x5410);
            const uint32_t y = __byte_perm(wc[w], wd[w], half ? 0x7632 : 0x5410);
            const int m = 4 * w + 2 * half, g = PACKED ? 0 : m / 2;
            mma_f16_16816(acc[m], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, pf[g][0], pf[g][1]);
            mma_f16_16816(acc[m + 1], (x >> 8) & 0x000f000fu, (x >> 8) & 0x00f000f0u, (y >> 8) & 0x000f000fu, (y >> 8) & 0x00f000f0u,
                          pf[g][0], pf[g][1]);
          }
      }
    }
  };

  int stage = 0;
  for (int tile = first; tile < tiles; tile += step) {
    const int next = tile + STAGES * step;
    const uint32_t then = next < tiles && lane < lookers ? kv4_block_of(p.table, pages_of, next * TB + lane) : kNoBlock;
    if (!mbar_wait(bars + stage * 8, (phase >> stage) & 1u)) { fine = false; break; }
    phase ^= 1u << stage;
    if (tile * KEYS + KEYS > seen_least || ((held >> (4 * stage)) & ALL) != ALL) consume(std::true_type{}, tile, stage);
    else consume(std::false_type{}, tile, stage);
    __syncwarp();
    if (next < tiles) issue(then, next, stage);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  if (!fine) {      // give up; the copies still under way end before their shared memory is used for something else
    if (lane == 0) kv4_report(p.status, kDevKv4Timeout);
    for (int s = 0; s < STAGES; ++s) mbar_wait(bars + s * 8, (phase >> s) & 1u);
  }

  // join the warps: each leaves (maximum, sum, output) per row; the ring is free once every warp is here
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem) + warp * (Shape::kPart / 4);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float s = sum[c], ce[GA];
#pragma unroll
    for (int m = 4; m < 32; m <<= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
#pragma unroll
    for (int g = 0; g < GA; ++g) {
      ce[g] = centre[g][c];
#pragma unroll
      for (int m = 4; m < 32; m <<= 1) ce[g] += __shfl_xor_sync(0xffffffffu, ce[g], m);
    }
    const int row = col_row + c;
    if (row >= live) continue;
    if (r == 0 && my_group == 0) {
      // a NaN sum must survive the join even where no score was a number
      part[ROWS * HD + row] = s != s ? INFINITY : top[c];
      part[ROWS * HD + ROWS + row] = s;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (PACKED && m / 2 != my_group) continue;
      const int g = PACKED ? 0 : m / 2;
      const float eight = ones[g / 2][2 * (g & 1) + c];
      part[row * HD + 16 * m + r] = fmaf(acc[m][c] + eight, 16777216.0f, ce[g]);
      part[row * HD + 16 * m + 8 + r] = fmaf(fmaf(acc[m][c + 2], 0.0625f, eight), 16777216.0f, ce[g]);
    }
  }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(smem);
  float* mine = reinterpret_cast<float*>(smem) + WARPS * (Shape::kPart / 4);
  auto store = [&](int row, int d, float o, float s) {
    const int tok = kv4_div(row, p.by_group);
    // a row that sees nothing is zero (its sum is the only one that can be)
    static_cast<T*>(p.out)[(q0 + tok) * p.o_tok + static_cast<int64_t>(head * p.group + row - tok * p.group) * p.o_head + d] =
        kv4_from_float<T>(s == 0.0f ? 0.0f : o / s);
  };
  for (int i = threadIdx.x; i < live * HD; i += WARPS * 32) {
    const int row = i / HD;
    float most = -INFINITY, o = 0.0f, s = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) most = fmaxf(most, all[w * (Shape::kPart / 4) + ROWS * HD + row]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float* a = all + w * (Shape::kPart / 4);
      const float m = a[ROWS * HD + row];
      if (m == -INFINITY) continue;
      const float f = exp2_approx(m - most);
      o = fmaf(f, a[i], o);
      s = fmaf(f, a[ROWS * HD + ROWS + row], s);
    }
    if (splits == 1) {
      store(row, i % HD, o, s);
    } else {
      mine[i] = o;
      if (i % HD == 0) {
        mine[ROWS * HD + row] = most;
        mine[ROWS * HD + ROWS + row] = s;
      }
    }
  }
  if (splits == 1) return;
  __syncwarp();
  cluster_sync();
  const uint32_t mine_at = smem_u32(mine);
  for (int i = rank * WARPS * 32 + threadIdx.x; i < live * HD; i += splits * WARPS * 32) {
    const int row = i / HD;
    float most = -INFINITY, o = 0.0f, s = 0.0f;
    for (int c = 0; c < splits; ++c) most = fmaxf(most, cluster_ld_f32(mapa_u32(mine_at + (ROWS * HD + row) * 4, c)));
    for (int c = 0; c < splits; ++c) {
      const float m = cluster_ld_f32(mapa_u32(mine_at + (ROWS * HD + row) * 4, c));
      if (m == -INFINITY) continue;
      const float f = exp2_approx(m - most);
      o = fmaf(f, cluster_ld_f32(mapa_u32(mine_at + i * 4, c)), o);
      s = fmaf(f, cluster_ld_f32(mapa_u32(mine_at + (ROWS * HD + ROWS + row) * 4, c)), s);
    }
    store(row, i % HD, o, s);
  }
  __syncwarp();
  cluster_sync();      // nobody leaves while its shared memory is read
}

}  // namespace crl
