// Attention of more than eight query rows per key head (runs of tokens, prompts) over the 4-bit cache of kv4.cuh.
//
// Same contract as kv4_attention_kernel. Here query rows are the 16 rows of mma.m16n8k16: RW warps of a CTA take 16 rows
// each, KW groups of warps take key tiles of 64 in turn (RW * KW = 4: a tile of 16, 32 or 64 rows keeps four warps busy),
// each with a running maximum, sum and output, joined over the CTA and the cluster at the end as there. A key group's
// tiles arrive by one bulk copy per block in a ring that its RW warps share.
//
// Codes become operands by one logical and two arithmetic f16x2 instructions per pair: 1024 + n is f16 with n in its low
// bits, minus 1032 (or through 1/16 for the nibbles that stand four bits higher) gives n - 8 exactly, times the step is
// exact too (eight significant bits times three). The centres come in as one more step of the products: for the scores
// sixteen columns that hold c_g against the row's sum of q over group g (in two f16 parts), for the output one more
// column block that collects sum p c_g. So only the weights p are rounded (f16), as a 16-bit cache would do as well.
//
// Bound by latency at the sizes it is for: 64-token prompts of 256 sequences, 12 heads of 64: 45 us (256 x 12 CTAs of one tile
// each, four to an SM; issue slots 48 % used), 5-token runs of 33 sequences at 1000 tokens, 16 heads on 4 of 32: 11.4 us.
// At 4096-token prompts it reaches 153 TFLOP/s where the kernel of kv4_prompt.cuh reaches 670.
#pragma once
#include "kv4_attention.cuh"

namespace crl {

template <int HD, int RW, int KW>
struct Kv4RowsShape {
  static constexpr int kStages = 2;
  static constexpr int kStage = 4 * kv4_block_bytes(HD);
  static constexpr int kRing = KW * kStages * kStage;
  static constexpr int kPart = 16 * (HD + 2) * 4;
  static constexpr int kJoin = (RW * KW + RW) * kPart;
  static constexpr int kBytes = (kRing > kJoin ? kRing : kJoin) + KW * kStages * 20;
};

__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t as_word(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }

// two codes at the low nibbles of both halves of w (HIGH: the second nibbles), minus 8, times s
template <bool HIGH>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, __half2 s) {
  const uint32_t x = (w & (HIGH ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;
  const __half2 n = HIGH ? __hfma2(as_half2(x), __float2half2_rn(0.0625f), __float2half2_rn(-72.0f))
                         : __hadd2(as_half2(x), __float2half2_rn(-1032.0f));
  return as_word(__hmul2(n, s));
}

template <typename T, int HD, int RW, int KW>
__global__ void __launch_bounds__(RW * KW * 32, HD == 128 ? 2 : 4) kv4_rows_kernel(const Kv4AttentionParams p) {
  using Shape = Kv4RowsShape<HD, RW, KW>;
  constexpr int G = HD / 32, DT = HD / 8, BB = kv4_block_bytes(HD), ROWS = 16 * RW, ST = Shape::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int kw = warp / RW, rw = warp % RW;
  const int splits = cluster_size_x(), rank = cluster_ctarank();
  const int head = blockIdx.y, row_tile = p.row_tiles - 1 - static_cast<int>(cluster_id_x()), seq = blockIdx.z;   // long rows first
  uint8_t* ring = smem + kw * ST * Shape::kStage;
  const uint32_t full = smem_u32(smem + Shape::kBytes - KW * ST * 20) + kw * ST * 16, empty = full + ST * 8;
  // which blocks of a stage's tile there are, left by the warp that copies them
  uint32_t* held = reinterpret_cast<uint32_t*>(smem + Shape::kBytes - KW * ST * 4) + kw * ST;

  // the first tiles' pages are asked for together with the sequence's length and its run of new tokens
  const int first = rank * KW + kw, step = splits * KW;
  const int32_t* pages_of = p.table.table + seq * p.table.stride;
  const int lookers = p.whole_tiles ? 1 : 4;
  uint32_t ahead[ST];
#pragma unroll
  for (int s = 0; s < ST; ++s)
    ahead[s] = rw == 0 && lane < lookers ? kv4_block_of(p.table, pages_of, (first + s * step) * 4 + lane) : kNoBlock;
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
  const int row0 = row_tile * ROWS, rows = run * p.group - row0;
  if (rows <= 0) return;      // the same for every CTA of the cluster
  const int last_tok = kv4_div(min(row0 + ROWS - 1, run * p.group - 1), p.by_group);
  const int seen_most = max(0, min(len, before + last_tok + 1));
  const int tiles = (seen_most + 63) / 64, blocks = (seen_most + kKv4Block - 1) / kKv4Block;

  if (threadIdx.x < KW * ST) {
    const uint32_t at = smem_u32(smem + Shape::kBytes - KW * ST * 20) + (threadIdx.x / ST) * ST * 16 + (threadIdx.x % ST) * 8;
    mbar_init(at, 1);
    mbar_init(at + ST * 8, RW);
  }
  mbar_fence_init();
  __syncthreads();

  // lane b of a key group's first warp looks block b of a tile up (well before it is wanted) and copies it; where pages
  // hold whole tiles lane 0 does so for all
  const uint8_t* head_pages = p.pages + static_cast<size_t>(head) * p.table.blocks * BB;
  auto issue = [&](uint32_t at, int tile, int stage) {
    const int n = min(4, blocks - tile * 4);
    if (lane < min(lookers, n)) {
      if (at == kNoBlock) kv4_report(p.status, kDevKv4Table);
    } else {
      at = kNoBlock;
    }
    uint32_t there = __ballot_sync(0xffffffffu, at != kNoBlock);
    const uint32_t to = smem_u32(ring + stage * Shape::kStage), bar = full + stage * 8;
    if (p.whole_tiles) there = there != 0 ? (1u << n) - 1 : 0u;
    if (lane == 0) {
      held[stage] = there;
      mbar_expect_tx(bar, __popc(there) * BB);
      if (p.whole_tiles && there != 0) bulk_load(to, head_pages + static_cast<size_t>(at) * BB, n * BB, bar);
    }
    __syncwarp();
    if (!p.whole_tiles && at != kNoBlock) bulk_load(to + lane * BB, head_pages + static_cast<size_t>(at) * BB, BB, bar);
  };
  if (rw == 0)
#pragma unroll
    for (int s = 0; s < ST; ++s)
      if (first + s * step < tiles) issue(ahead[s], first + s * step, s);

  // queries as the A operand, rows r and r + 8 of this warp, scaled to [1, 2) by a power of two
  uint32_t qf[G][2][4], qsum[2] = {0, 0};     // [group][half of the group][register]; sums: rows r, r + 8
  float factor[2];
  int limit[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = row0 + rw * 16 + r + 8 * h, tok = kv4_div(row, p.by_group);
    const bool live = tok < run;
    const T* src = static_cast<const T*>(p.q) + (q0 + tok) * p.q_tok + static_cast<int64_t>(head * p.group + row - tok * p.group) * p.q_head;
    float x[G][8], big = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (live) kv4_load8(src + 32 * g + 8 * t, p.vec_q, x[g]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!live) x[g][i] = 0.0f;
        big = fmaxf(big, fabsf(x[g][i]));
      }
    }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const int e = big > 0.0f ? min(120, max(-120, static_cast<int>(__float_as_uint(big) >> 23) - 127)) : 0;
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    factor[h] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * p.scale_log2;
    limit[h] = live ? before + tok + 1 : 0;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[g][i] *= down;
        sum += x[g][i];
      }
      qf[g][0][h] = pack_f16(x[g][0], x[g][4]);
      qf[g][0][2 + h] = pack_f16(x[g][1], x[g][5]);
      qf[g][1][h] = pack_f16(x[g][2], x[g][6]);
      qf[g][1][2 + h] = pack_f16(x[g][3], x[g][7]);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      // columns of the centres' step: g holds the sum's leading part, 4 + g the rest; lane t has columns 2t, 2t + 1
      const __half hi = __float2half_rn(sum);
      const __half mine = t == g / 2 ? hi : __float2half_rn(sum - __half2float(hi));
      if (t == g / 2 || t == 2 + g / 2)
        qsum[h] |= static_cast<uint32_t>(__half_as_ushort(mine)) << (16 * (g & 1));
    }
  }

  float acc[DT][4], cen[4] = {0, 0, 0, 0}, top[2] = {-INFINITY, -INFINITY}, sum[2] = {0, 0};
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[d][i] = 0.0f;

  const int kr = (r >> 1) + 4 * (r & 1);     // key of a half block that column r stands for
  // the tile's keys that every row of this warp sees, and those that any does
  const int warp_row = row0 + rw * 16, most_row = min(warp_row + 15, run * p.group - 1);
  const int see_all = before + kv4_div(warp_row, p.by_group) + 1;
  const int see_any = warp_row < run * p.group ? min(len, before + kv4_div(most_row, p.by_group) + 1) : 0;

  auto consume = [&](auto masked_tag, int tile, int stage, uint32_t there) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const uint8_t* base = ring + stage * Shape::kStage;
    float sc[8][4];
    // blocks of the tile that any of the warp's rows sees
    const int seen = MASKED ? min(4, (see_any - tile * 64 + 15) / 16) : 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (MASKED && j / 2 >= seen) {
        sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = -INFINITY;
        continue;
      }
      const uint8_t* blk = base + (j >> 1) * BB;
      const int key = kr + 8 * (j & 1);
      uint32_t w[G], m[G];
      lds_words<G>(w, blk + key * (HD / 2) + t * (G * 4));
      lds_words<G>(m, blk + 8 * HD + key * (G * 4));
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[j][i] = 0.0f;
      // centres: columns 0..G-1 and 4..4+G-1 of the step, lane t has columns 2t, 2t + 1
      uint32_t c = 0;
      if constexpr (G == 1) c = (t & 1) == 0 ? m[0] >> 16 : 0u;
      else if constexpr (G == 2) c = (t & 1) == 0 ? __byte_perm(m[0], m[1], 0x7632) : 0u;
      else c = (t & 1) == 0 ? __byte_perm(m[0], m[1], 0x7632) : __byte_perm(m[2], m[3], 0x7632);
      mma_f16_16816(sc[j], qsum[0], qsum[1], 0u, 0u, c, 0u);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const __half2 s = __low2half2(as_half2(m[g]));
        mma_f16_16816(sc[j], qf[g][0][0], qf[g][0][1], qf[g][0][2], qf[g][0][3], code_pair<false>(w[g], s), code_pair<true>(w[g], s));
        mma_f16_16816(sc[j], qf[g][1][0], qf[g][1][1], qf[g][1][2], qf[g][1][3], code_pair<false>(w[g] >> 8, s),
                      code_pair<true>(w[g] >> 8, s));
      }
    }
    float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = sc[j][i] * factor[i >> 1];
        if (MASKED) {
          const int key = tile * 64 + j * 8 + t + 4 * (i & 1);
          if (key >= limit[i >> 1] || !((there >> (j >> 1)) & 1u)) x = -INFINITY;
        }
        sc[j][i] = x;
        most[i >> 1] = fmaxf(most[i >> 1], x);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 1));
      most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 2));
      most[h] = fmaxf(most[h], top[h]);
    }
    if (__any_sync(0xffffffffu, most[0] > top[0] || most[1] > top[1])) {
      float alpha[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        alpha[h] = top[h] == -INFINITY ? 0.0f : exp2_approx(top[h] - most[h]);
        top[h] = most[h];
        sum[h] *= alpha[h];
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[d][i] *= alpha[i >> 1];
#pragma unroll
      for (int i = 0; i < 4; ++i) cen[i] *= alpha[i >> 1];
    }
    const float off[2] = {top[0] == -INFINITY ? 0.0f : top[0], top[1] == -INFINITY ? 0.0f : top[1]};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[j][i] = exp2_approx(sc[j][i] - off[i >> 1]);
        sum[i >> 1] += sc[j][i];
      }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (MASKED && b >= seen) break;
      const uint8_t* blk = base + b * BB + 10 * HD;
      const uint32_t a0 = pack_f16(sc[2 * b][0], sc[2 * b][1]), a1 = pack_f16(sc[2 * b][2], sc[2 * b][3]);
      const uint32_t a2 = pack_f16(sc[2 * b + 1][0], sc[2 * b + 1][1]), a3 = pack_f16(sc[2 * b + 1][2], sc[2 * b + 1][3]);
      uint32_t m[4][G];
#pragma unroll
      for (int k = 0; k < 4; ++k) lds_words<G>(m[k], blk + 8 * HD + (t + 4 * k) * (G * 4));
      if (MASKED) {
        // rows that no query sees may hold anything; a NaN that some rows see and others do not must not reach the
        // others through 0 * NaN in the product: it is taken out and given to the rows that see it
        __half2 probe = __float2half2_rn(0.0f);      // 0 * m is NaN for a NaN or an infinity
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool gone = tile * 64 + b * 16 + t + 4 * k >= see_any || !((there >> b) & 1u);
#pragma unroll
          for (int g = 0; g < G; ++g) {
            if (gone) m[k][g] = 0u;
            probe = __hfma2(as_half2(m[k][g]), __float2half2_rn(0.0f), probe);
          }
        }
        if (__any_sync(0xffffffffu, (as_word(probe) & 0x7fff7fffu) != 0)) {
          uint32_t bad[4] = {0, 0, 0, 0};
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int g = 0; g < G; ++g)
              if ((m[k][g] & 0x7c00u) == 0x7c00u || (m[k][g] & 0x7c000000u) == 0x7c000000u) {
                bad[k] |= 1u << g;
                m[k][g] = 0u;
              }
          uint32_t lost[2] = {0, 0};
          for (int key = 0; key < 16; ++key) {
            const uint32_t mine = key / 4 == 0 ? bad[0] : key / 4 == 1 ? bad[1] : key / 4 == 2 ? bad[2] : bad[3];
            const uint32_t them = __shfl_sync(0xffffffffu, mine, (lane & ~3) + (key & 3));
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (tile * 64 + b * 16 + key < limit[h]) lost[h] |= them;
          }
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if ((lost[i >> 1] >> (d / 4)) & 1u) acc[d][i] = __int_as_float(0x7fc00000);
        }
      }
      // centres: column g of one more block
      uint32_t c0 = 0, c1 = 0;
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (r == g) {
          c0 = __byte_perm(m[0][g], m[1][g], 0x7632);
          c1 = __byte_perm(m[2][g], m[3][g], 0x7632);
        }
      mma_f16_16816(cen, a0, a1, a2, a3, c0, c1);
      __half2 s0[G], s1[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        s0[g] = as_half2(__byte_perm(m[0][g], m[1][g], 0x5410));
        s1[g] = as_half2(__byte_perm(m[2][g], m[3][g], 0x5410));
      }
      if constexpr (HD == 32) {
        const uint16_t* rowp = reinterpret_cast<const uint16_t*>(blk) + r;
        const uint32_t x = rowp[t * 8] | (static_cast<uint32_t>(rowp[(t + 4) * 8]) << 16);
        const uint32_t y = rowp[(t + 8) * 8] | (static_cast<uint32_t>(rowp[(t + 12) * 8]) << 16);
        mma_f16_16816(acc[0], a0, a1, a2, a3, code_pair<false>(x, s0[0]), code_pair<false>(y, s1[0]));
        mma_f16_16816(acc[1], a0, a1, a2, a3, code_pair<true>(x, s0[0]), code_pair<true>(y, s1[0]));
        mma_f16_16816(acc[2], a0, a1, a2, a3, code_pair<false>(x >> 8, s0[0]), code_pair<false>(y >> 8, s1[0]));
        mma_f16_16816(acc[3], a0, a1, a2, a3, code_pair<true>(x >> 8, s0[0]), code_pair<true>(y >> 8, s1[0]));
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
            const int d = 8 * w + 4 * half, g = d / 4;
            mma_f16_16816(acc[d], a0, a1, a2, a3, code_pair<false>(x, s0[g]), code_pair<false>(y, s1[g]));
            mma_f16_16816(acc[d + 1], a0, a1, a2, a3, code_pair<true>(x, s0[g]), code_pair<true>(y, s1[g]));
            mma_f16_16816(acc[d + 2], a0, a1, a2, a3, code_pair<false>(x >> 8, s0[g]), code_pair<false>(y >> 8, s1[g]));
            mma_f16_16816(acc[d + 3], a0, a1, a2, a3, code_pair<true>(x >> 8, s0[g]), code_pair<true>(y >> 8, s1[g]));
          }
      }
    }
  };

  int stage = 0;
  uint32_t phase = 0;
  bool fine = true;
  for (int tile = first; tile < tiles; tile += step) {
    const bool more = rw == 0 && tile + ST * step < tiles;
    const uint32_t then = more && lane < lookers ? kv4_block_of(p.table, pages_of, (tile + ST * step) * 4 + lane) : kNoBlock;
    if (!mbar_wait(full + stage * 8, phase)) { fine = false; break; }
    const uint32_t there = held[stage];
    if (tile * 64 < see_any) {
      if (tile * 64 + 64 > see_all || there != 15u) consume(std::true_type{}, tile, stage, there);
      else consume(std::false_type{}, tile, stage, there);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + stage * 8);
    if (more) {
      if (!mbar_wait(empty + stage * 8, phase)) { fine = false; break; }
      issue(then, tile + ST * step, stage);
    }
    if (++stage == ST) {
      stage = 0;
      phase ^= 1u;
    }
  }
  if (!fine) {      // give up; the copies still under way end before their shared memory is used for something else
    if (lane == 0) kv4_report(p.status, kDevKv4Timeout);
    for (int s = 0; s < ST; ++s) mbar_wait(full + s * 8, s < stage ? phase ^ 1u : phase);
  }

  if (KW == 1 && splits == 1) {      // nothing to join: from the registers
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      const int at = row0 + rw * 16 + r + 8 * h, tok = kv4_div(at, p.by_group);
      const float inv = sum[h] == 0.0f ? 0.0f : 1.0f / sum[h];      // a row that sees nothing is zero
      T* out = static_cast<T*>(p.out) + (q0 + tok) * p.o_tok + static_cast<int64_t>(head * p.group + at - tok * p.group) * p.o_head + 2 * t;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float c = __shfl_sync(0xffffffffu, cen[2 * h + (g & 1)], (lane & ~3) + g / 2);
        if (tok >= run) continue;
#pragma unroll
        for (int d = 4 * g; d < 4 * g + 4; ++d) {
          T two[2] = {kv4_from_float<T>((acc[d][2 * h] + c) * inv), kv4_from_float<T>((acc[d][2 * h + 1] + c) * inv)};
          if (p.pair_o) {
            *reinterpret_cast<uint32_t*>(out + 8 * d) = *reinterpret_cast<const uint32_t*>(two);
          } else {
            out[8 * d] = two[0];
            out[8 * d + 1] = two[1];
          }
        }
      }
    }
    return;
  }
  // join over the key groups, then over the cluster
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem) + warp * (Shape::kPart / 4);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    const int row = r + 8 * h;
    if (t == 0) {
      part[16 * HD + row] = sum[h] != sum[h] ? INFINITY : top[h];     // a NaN sum must survive the join
      part[16 * HD + 16 + row] = sum[h];
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float c = __shfl_sync(0xffffffffu, cen[2 * h + (g & 1)], (lane & ~3) + g / 2);
#pragma unroll
      for (int d = 4 * g; d < 4 * g + 4; ++d)
        *reinterpret_cast<float2*>(part + row * HD + 8 * d + 2 * t) = make_float2(acc[d][2 * h] + c, acc[d][2 * h + 1] + c);
    }
  }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(smem);
  float* mine = reinterpret_cast<float*>(smem) + RW * KW * (Shape::kPart / 4);
  constexpr int P4 = Shape::kPart / 4, THREADS = RW * KW * 32;
  const int live = min(rows, ROWS);
  if (KW > 1 || splits > 1) {
    for (int i = threadIdx.x; i < live * HD; i += THREADS) {
      const int row = i / HD, w = row / 16, in = row % 16, d = i - row * HD;
      float most = -INFINITY, o = 0.0f, s = 0.0f;
#pragma unroll
      for (int k = 0; k < KW; ++k) most = fmaxf(most, all[(k * RW + w) * P4 + 16 * HD + in]);
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const float* a = all + (k * RW + w) * P4;
        const float m = a[16 * HD + in];
        if (m == -INFINITY) continue;
        const float f = exp2_approx(m - most);
        o = fmaf(f, a[in * HD + d], o);
        s = fmaf(f, a[16 * HD + 16 + in], s);
      }
      mine[w * P4 + in * HD + d] = o;
      if (d == 0) {
        mine[w * P4 + 16 * HD + in] = most;
        mine[w * P4 + 16 * HD + 16 + in] = s;
      }
    }
    __syncwarp();
    if (splits > 1) cluster_sync(); else __syncthreads();
  }
  const float* whole = KW > 1 || splits > 1 ? mine : all;
  const uint32_t whole_at = smem_u32(whole);
  for (int i = rank * THREADS + threadIdx.x; i < live * HD / 2; i += splits * THREADS) {
    const int row = i / (HD / 2), w = row / 16, in = row % 16, d = 2 * (i - row * (HD / 2));
    float o0, o1, s;
    if (splits == 1) {
      const float2 o = *reinterpret_cast<const float2*>(whole + w * P4 + in * HD + d);
      o0 = o.x;
      o1 = o.y;
      s = whole[w * P4 + 16 * HD + 16 + in];
    } else {
      float most = -INFINITY;
      for (int c = 0; c < splits; ++c) most = fmaxf(most, cluster_ld_f32(mapa_u32(whole_at + (w * P4 + 16 * HD + in) * 4, c)));
      o0 = o1 = s = 0.0f;
      for (int c = 0; c < splits; ++c) {
        const float m = cluster_ld_f32(mapa_u32(whole_at + (w * P4 + 16 * HD + in) * 4, c));
        if (m == -INFINITY) continue;
        const float f = exp2_approx(m - most);
        o0 = fmaf(f, cluster_ld_f32(mapa_u32(whole_at + (w * P4 + in * HD + d) * 4, c)), o0);
        o1 = fmaf(f, cluster_ld_f32(mapa_u32(whole_at + (w * P4 + in * HD + d + 1) * 4, c)), o1);
        s = fmaf(f, cluster_ld_f32(mapa_u32(whole_at + (w * P4 + 16 * HD + 16 + in) * 4, c)), s);
      }
    }
    const int at = row0 + row, tok = kv4_div(at, p.by_group);
    const float inv = s == 0.0f ? 0.0f : 1.0f / s;      // a row that sees nothing is zero
    T* out = static_cast<T*>(p.out) + (q0 + tok) * p.o_tok + static_cast<int64_t>(head * p.group + at - tok * p.group) * p.o_head + d;
    if (p.pair_o) {
      T two[2] = {kv4_from_float<T>(o0 * inv), kv4_from_float<T>(o1 * inv)};
      *reinterpret_cast<uint32_t*>(out) = *reinterpret_cast<const uint32_t*>(two);
    } else {
      out[0] = kv4_from_float<T>(o0 * inv);
      out[1] = kv4_from_float<T>(o1 * inv);
    }
  }
  __syncwarp();
  if (splits > 1) cluster_sync();      // nobody leaves while its shared memory is read
}

}  // namespace crl
