// Attention of many query rows (prompts) over the 4-bit cache of kv4.cuh, on the 5th-generation tensor cores.
//
// Same contract as kv4_attention_kernel. A CTA takes 256 query rows of a (sequence, key head) as two tiles of 128 and walks
// the keys in tiles of KT. Its warps:
//   0-3, 4-7   softmax of the first / second row tile: a thread owns a row
//   8-14       unpack: warp 8 + b turns block b of a key tile into matrix operands in shared memory
//   15         one thread issues the tcgen05.mma products; the warp owns the tensor memory
// The softmax warps take registers over from the others (168 and 88 of the 128 at launch), so that a row's 112 scores are
// read from tensor memory once and stay in registers.
// Tensor memory: scores S [128 x KT] fp32 per row tile, over which the weights P are written back as f16 (the left
// operand of the output product), and the outputs O [128 x (hd + 16)] fp32: 512 columns in all at hd 128, KT 112.
// The two row tiles are half a step apart: while one's softmax runs, the other's products do.
//
// Operands are exact: n - 8 times the step (eight significant bits) is an f16 number. The centres come in as 16 more
// columns of the products: for the scores c_g against the row's sum of q over group g, in two f16 parts; for the output
// the extra columns collect sum p c_g. Queries are scaled to [1, 2) per row by a power of two. So the only rounding
// before the result's is that of P to f16, as in the other kernels.
//
// Shared memory holds operands as 8 x 16-byte core matrices (no swizzle): element (row, k) lies at
// (k / 8) * lead + (row / 8) * 128 + (row % 8) * 16 + (k % 8) * 2. Unpacking writes 16-byte pieces that fall on distinct
// banks (keys: the lead has 32 bytes of padding; dims of a piece in the order 0 4 1 5 2 6 3 7 that the codes come in, q
// alike). Values are stored dim by dim along the keys: two keys' words give pairs of adjacent keys.
//
// A row's running maximum is only moved when it grows by more than 2^8 (P <= 256 stays well inside f16), so O is
// rarely rescaled.
//
// Measured: two prompts of up to 4096 tokens, 32 heads on 8 of 128, bf16: 384 us = 670 TFLOP/s, 41 % of the measured matrix
// rate. A step of a row tile (112 keys) takes about 3500 cycles against 2230 of products for both tiles: the softmax
// of one (2000) and the chain last weight -> output product -> scores (1500) follow one another, and two row tiles are
// all that tensor memory holds at hd 128. The scores wait for the output product before them because they overwrite its weights.
// Tried: taking turns with the exponentials (541 against 513 us then), reading the scores twice instead of keeping
// them (503 against 406), issuing whichever row tile is ready first (501 against 390): none kept.
#pragma once
#include "kv4_rows.cuh"

namespace crl {

template <int HD>
struct Kv4PromptShape {
  static constexpr int kKeys = 112;      // the most that S and O leave room for in tensor memory at hd 128
  static constexpr int kBlocks = kKeys / 16;
  static constexpr int kWide = HD + 16;                   // dims and the centres' columns
  static constexpr int kLeadQ = 128 * 16, kLeadK = kKeys * 16 + 32, kLeadV = kWide * 16;
  static constexpr int kQ = kWide / 8 * kLeadQ, kK = kWide / 8 * kLeadK, kV = kKeys / 8 * kLeadV;
  static constexpr int kOffK = 2 * kQ, kOffV = kOffK + 2 * kK;
  static constexpr int kOffFlags = kOffV + 2 * kV;                 // 4 x 8 words of block flags
  static constexpr int kOffBad = kOffFlags + 4 * 8 * 4;            // 4 x kKeys bytes: groups of a key's value that are NaN
  static constexpr int kOffBars = (kOffBad + 4 * kKeys + 15) / 16 * 16;
  static constexpr int kBytes = kOffBars + 22 * 8;
  static constexpr int kRow = HD * 2 + 16;                // a row of q or out on its way, padded onto distinct banks
  static constexpr int kThreads = 16 * 32;
  static constexpr int kColS = 0, kColO = 2 * kKeys;      // tensor memory columns: S_a, S_b, O_a, O_b
};

// shared-memory matrix descriptor, no swizzle, K-major (see above): `lead` bytes between core matrices along k, 128 along
// the rows
__device__ __forceinline__ uint64_t umma_desc_plain(uint32_t addr, uint32_t lead) {
  return static_cast<uint64_t>((addr & 0x3FFFF) >> 4) | static_cast<uint64_t>(lead >> 4) << 16 | static_cast<uint64_t>(128 >> 4) << 32 |
         static_cast<uint64_t>(1) << 46;
}
// D[tmem] (+)= A[tmem] * B[smem]^T, f16
__device__ __forceinline__ void umma_f16_ta(uint32_t d, uint32_t a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
               "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <typename T, int HD>
__global__ void __launch_bounds__(Kv4PromptShape<HD>::kThreads, 1) kv4_prompt_kernel(const Kv4AttentionParams p) {
  using Shape = Kv4PromptShape<HD>;
  constexpr int G = HD / 32, BB = kv4_block_bytes(HD), KT = Shape::kKeys, NB = Shape::kBlocks;
  constexpr int kHalf = 4;      // blocks of a tile whose weights are handed over early
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.y, row_tile = p.row_tiles - 1 - static_cast<int>(blockIdx.x), seq = blockIdx.z;   // long rows first

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
  const int row0 = row_tile * 256, live = run * p.group - row0;     // rows of this CTA: min(live, 256)
  if (live <= 0) return;
  const int last_tok = kv4_div(row0 + min(live, 256) - 1, p.by_group);
  const int seen_most = max(0, min(len, before + last_tok + 1));
  const int tiles = (seen_most + KT - 1) / KT;

  uint32_t* flags = reinterpret_cast<uint32_t*>(smem + Shape::kOffFlags);
  uint8_t* bad_keys = smem + Shape::kOffBad;
  const uint32_t bars = smem_u32(smem + Shape::kOffBars);
  // full / free per operand stage, then per row tile: scores there, weights there, output product done
  const uint32_t k_full = bars, k_free = bars + 16, v_full = bars + 32, v_free = bars + 48, s_full = bars + 64, p_full = bars + 80,
                 o_done = bars + 96, p_half = bars + 112, q_full = bars + 128, q_raw = bars + 144;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Shape::kOffBars + 160);

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(k_full + 8 * s, NB);
      mbar_init(k_free + 8 * s, 1);
      mbar_init(v_full + 8 * s, NB);
      mbar_init(v_free + 8 * s, 1);
      mbar_init(q_full + 8 * s, 4);
      mbar_init(q_raw + 8 * s, 1);
      mbar_init(s_full + 8 * s, 2);      // the products' commit and the issuing thread
      mbar_init(p_half + 8 * s, 4);
      mbar_init(p_full + 8 * s, 4);
      mbar_init(o_done + 8 * s, 1);
    }
    mbar_fence_init();
  }
  if (warp == 15) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  // both stages' extra columns: those that no group has are zero for good, one of the values' is one: it collects the
  // rows' sums of P
  constexpr int kSumRow = 4;
  for (int i = threadIdx.x; i < 2 * 2 * KT; i += Shape::kThreads) {
    const int stage = i / (2 * KT), c = i / KT % 2, row = i % KT;
    *reinterpret_cast<uint4*>(smem + Shape::kOffK + stage * Shape::kK + (HD / 8 + c) * Shape::kLeadK + row * 16) = make_uint4(0, 0, 0, 0);
  }
  for (int i = threadIdx.x; i < 2 * (KT / 8) * 16; i += Shape::kThreads) {
    const int stage = i / (KT / 8 * 16), c = i / 16 % (KT / 8), row = i % 16;
    const uint32_t one = row == kSumRow ? 0x3c003c00u : 0u;
    *reinterpret_cast<uint4*>(smem + Shape::kOffV + stage * Shape::kV + c * Shape::kLeadV + (HD + row) * 16) = make_uint4(one, one, one, one);
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool fine = true;
  if (warp >= 8) {
    // registers: 256 x 168 + 256 x 88 = 512 x 128
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 15) {
    // ---- products ---------------------------------------------------------------------------------------------------
    if (lane == 0 && tiles > 0) {
      const uint32_t idesc_s = umma_idesc(128, KT, 0, 1), idesc_o = umma_idesc(128, Shape::kWide, 0, 1);
      const uint32_t sm = smem_u32(smem);
      auto scores = [&](int x, int i) {      // S_x = Q_x K(i)^T
        const uint32_t q = sm + x * Shape::kQ, k = sm + Shape::kOffK + (i & 1) * Shape::kK;
#pragma unroll
        for (int s = 0; s < Shape::kWide / 16; ++s)
          umma<kKindF16>(tmem + Shape::kColS + x * KT, umma_desc_plain(q + 2 * s * Shape::kLeadQ, Shape::kLeadQ),
                         umma_desc_plain(k + 2 * s * Shape::kLeadK, Shape::kLeadK), idesc_s, s > 0);
        tc_commit(s_full + 8 * x);
        mbar_arrive(s_full + 8 * x);         // hands on what the unpacking warps left beside the operands
        if (x == 1) tc_commit(k_free + 8 * (i & 1));
      };
      fine = mbar_wait(k_full, 0);
      for (int x = 0; x < 2 && fine; ++x) {
        fine = mbar_wait(q_full + 8 * x, 0);
        tc_fence_after();
        if (fine) scores(x, 0);
      }
      for (int i = 0; i < tiles && fine; ++i) {
#pragma unroll 1
        for (int x = 0; x < 2 && fine; ++x) {
          fine = mbar_wait(p_half + 8 * x, i & 1) && (x == 1 || mbar_wait(v_full + 8 * (i & 1), (i >> 1) & 1));
          if (!fine) break;
          tc_fence_after();
          const uint32_t v = sm + Shape::kOffV + (i & 1) * Shape::kV, o = tmem + Shape::kColO + x * Shape::kWide;
#pragma unroll
          for (int s = 0; s < kHalf; ++s)
            umma_f16_ta(o, tmem + Shape::kColS + x * KT + 8 * s, umma_desc_plain(v + 2 * s * Shape::kLeadV, Shape::kLeadV), idesc_o,
                        i > 0 || s > 0);
          fine = mbar_wait(p_full + 8 * x, i & 1);
          if (!fine) break;
          tc_fence_after();
#pragma unroll
          for (int s = kHalf; s < KT / 16; ++s)
            umma_f16_ta(o, tmem + Shape::kColS + x * KT + 8 * s, umma_desc_plain(v + 2 * s * Shape::kLeadV, Shape::kLeadV), idesc_o, 1);
          tc_commit(o_done + 8 * x);
          if (x == 1) tc_commit(v_free + 8 * (i & 1));
          if (i + 1 < tiles) {
            // the next scores overwrite the weights: their product has to be through
            fine = (x == 1 || mbar_wait(k_full + 8 * ((i + 1) & 1), ((i + 1) >> 1) & 1)) && mbar_wait(o_done + 8 * x, i & 1);
            if (!fine) break;
            tc_fence_after();
            scores(x, i + 1);
          }
        }
      }
      // every product has ended before tensor memory is given back
      for (int x = 0; x < 2; ++x) fine = mbar_wait(o_done + 8 * x, (tiles - 1) & 1) && fine;
    }
    __syncwarp();
    } else {
    // ---- unpack -----------------------------------------------------------------------------------------------------
    const int b = warp - 8;
    {
      const int32_t* pages_of = p.table.table + seq * p.table.stride;
      const uint8_t* head_pages = p.pages + static_cast<size_t>(head) * p.table.blocks * BB;
      const int kt = lane & 3, kn = lane >> 2;                 // keys kn, kn + 8, quarter kt
      const int vr = lane & 7, vu = lane >> 3, vc = vu >> 1, vh = vu & 1;   // values: dims vr mod 8, keys 8 vc .. + 7, half vh
      constexpr int VN = HD / 16;                              // nibbles of a lane's part of a value row
      constexpr int VG = HD == 128 ? 2 : 1;                    // groups they belong to
      const int vg = HD == 128 ? 2 * vh : HD == 64 ? vh : 0;   // the first of them
      uint32_t kw[2][G], km[2][G], vw[8], vm[8][VG];
      const uint8_t* from = nullptr;
      auto look = [&](int i) -> const uint8_t* {
        if (i * KT + b * 16 >= seen_most) return nullptr;
        const uint32_t at = kv4_block_of(p.table, pages_of, i * NB + b);
        if (at == kNoBlock) {
          if (lane == 0) kv4_report(p.status, kDevKv4Table);
          return nullptr;
        }
        return head_pages + static_cast<size_t>(at) * BB;
      };
      auto load_keys = [&]() {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int g = 0; g < G; ++g) kw[h][g] = km[h][g] = 0;
        if (from == nullptr) return;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          lds_words<G>(kw[h], from + (kn + 8 * h) * (HD / 2) + kt * (G * 4));
          lds_words<G>(km[h], from + 8 * HD + (kn + 8 * h) * (G * 4));
        }
      };
      auto load_values = [&]() {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          vw[j] = 0;
#pragma unroll
          for (int g = 0; g < VG; ++g) vm[j][g] = 0;
          if (from == nullptr) continue;
          const uint8_t* row = from + 10 * HD + (8 * vc + j) * (HD / 2) + vr * (HD / 16) + vh * (HD / 32);
          if constexpr (HD == 128) vw[j] = *reinterpret_cast<const uint32_t*>(row);
          else if constexpr (HD == 64) vw[j] = *reinterpret_cast<const uint16_t*>(row);
          else vw[j] = *row;
          lds_words<VG>(vm[j], from + 18 * HD + (8 * vc + j) * (G * 4) + vg * 4);
        }
      };
      // the table is read two tiles ahead, the codes one
      from = tiles > 0 ? look(0) : nullptr;
      if (tiles > 0) {
        load_keys();
        load_values();
      }
      bool there = from != nullptr;
      const uint8_t* then = tiles > 1 ? look(1) : nullptr;
      for (int i = 0; i < tiles; ++i) {
        const int stage = i & 1;
        from = then;
        then = i + 2 < tiles ? look(i + 2) : nullptr;
        if (i >= 2 && !mbar_wait(k_free + 8 * stage, ((i >> 1) & 1) ^ 1)) { fine = false; break; }
        uint8_t* k = smem + Shape::kOffK + stage * Shape::kK;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = b * 16 + kn + 8 * h;
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const __half2 s = __low2half2(as_half2(km[h][g]));
            const uint32_t w = kw[h][g];
            *reinterpret_cast<uint4*>(k + (4 * g + kt) * Shape::kLeadK + n * 16) =
                make_uint4(code_pair<false>(w, s), code_pair<true>(w, s), code_pair<false>(w >> 8, s), code_pair<true>(w >> 8, s));
          }
          if (kt == 0) {
            uint32_t c0 = G > 1 ? __byte_perm(km[h][0], km[h][G > 1 ? 1 : 0], 0x7632) : km[h][0] >> 16;
            uint32_t c1 = G > 2 ? __byte_perm(km[h][G > 2 ? 2 : 0], km[h][G > 2 ? 3 : 0], 0x7632) : 0u;
            *reinterpret_cast<uint4*>(k + HD / 8 * Shape::kLeadK + n * 16) = make_uint4(c0, c1, c0, c1);
          }
        }
        load_keys();
        // a value row that no query sees may hold anything; one that is NaN must not reach the rows that do not see it
        // through 0 * NaN: it is taken out here and given to the rows that see it by the softmax warps
        if (!there || i * KT + b * 16 + 16 > seen_most) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int g = 0; g < VG; ++g)
              if (!there || i * KT + b * 16 + 8 * vc + j >= seen_most) vm[j][g] = 0;
        }
        __half2 probe = __float2half2_rn(0.0f);      // 0 * m is NaN for a NaN or an infinity
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int g = 0; g < VG; ++g) probe = __hfma2(as_half2(vm[j][g]), __float2half2_rn(0.0f), probe);
        const bool some = __any_sync(0xffffffffu, (as_word(probe) & 0x7fff7fffu) != 0);
        if (some) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t bad = 0;
#pragma unroll
            for (int g = 0; g < VG; ++g)
              if ((vm[j][g] & 0x7c00u) == 0x7c00u || (vm[j][g] & 0x7c000000u) == 0x7c000000u) {
                bad |= 1u << (vg + g);
                vm[j][g] = 0;
              }
            bad |= __shfl_xor_sync(0xffffffffu, bad, 8);      // the other half's groups
            if (vr == 0 && vh == 0) bad_keys[(i & 3) * KT + b * 16 + 8 * vc + j] = static_cast<uint8_t>(bad);
          }
        }
        if (lane == 0) flags[(i & 3) * 8 + b] = (there ? 1u : 0u) | (some ? 2u : 0u);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(k_full + 8 * stage);

        if (i >= 2 && !mbar_wait(v_free + 8 * stage, ((i >> 1) & 1) ^ 1)) { fine = false; break; }
        uint8_t* v = smem + Shape::kOffV + stage * Shape::kV + (2 * b + vc) * Shape::kLeadV;
        uint32_t piece[VN][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {      // keys 2j, 2j + 1 of the eight
          __half2 s[VG];
#pragma unroll
          for (int g = 0; g < VG; ++g) s[g] = as_half2(__byte_perm(vm[2 * j][g], vm[2 * j + 1][g], 0x5410));
          if constexpr (HD == 128) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t x = __byte_perm(vw[2 * j], vw[2 * j + 1], half ? 0x7632 : 0x5410);
              piece[4 * half][j] = code_pair<false>(x, s[half % VG]);
              piece[4 * half + 1][j] = code_pair<true>(x, s[half % VG]);
              piece[4 * half + 2][j] = code_pair<false>(x >> 8, s[half % VG]);
              piece[(4 * half + 3) % VN][j] = code_pair<true>(x >> 8, s[half % VG]);
            }
          } else {
            const uint32_t x = vw[2 * j] | (vw[2 * j + 1] << 16);
            piece[0][j] = code_pair<false>(x, s[0]);
            piece[1][j] = code_pair<true>(x, s[0]);
            if constexpr (HD == 64) {
              piece[2][j] = code_pair<false>(x >> 8, s[0]);
              piece[3][j] = code_pair<true>(x >> 8, s[0]);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < VN; ++n)
          *reinterpret_cast<uint4*>(v + (vh * VN + n) * 128 + vr * 16) = make_uint4(piece[n][0], piece[n][1], piece[n][2], piece[n][3]);
        if (vr < VG && (HD != 32 || vh == 0)) {
          uint32_t c[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            c[j] = VG == 2 && vr == 1 ? __byte_perm(vm[2 * j][VG - 1], vm[2 * j + 1][VG - 1], 0x7632) : __byte_perm(vm[2 * j][0], vm[2 * j + 1][0], 0x7632);
          *reinterpret_cast<uint4*>(v + (HD + vg + vr) * 16) = make_uint4(c[0], c[1], c[2], c[3]);
        }
        load_values();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full + 8 * stage);
        there = from != nullptr;
      }
    }
    }
  } else {
    // ---- softmax: thread = row --------------------------------------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const int x = warp >> 2, row = threadIdx.x & 127, mine = x * 128 + row, at = row0 + mine;
    const int tok = kv4_div(at, p.by_group);
    const bool on = mine < live;
    const int limit = on ? before + tok + 1 : 0;
    float factor;
    {
      // the row's queries, by one bulk copy into the place of the operands, from there into registers (16-byte loads from
      // global memory by row took four times as long)
      const T* src = static_cast<const T*>(p.q) + (q0 + tok) * p.q_tok + static_cast<int64_t>(head * p.group + at - tok * p.group) * p.q_head;
      uint8_t* place = smem + x * Shape::kQ + row * Shape::kRow;
      uint4 raw[HD / 8];
      if (p.vec_q) {
        if (row == 0) mbar_expect_tx(q_raw + 8 * x, max(0, min(live - x * 128, 128)) * HD * 2);
        if (on) bulk_load(smem_u32(place), src, HD * 2, q_raw + 8 * x);
        if (!mbar_wait(q_raw + 8 * x, 0)) fine = false;
      }
#pragma unroll
      for (int c = 0; c < HD / 8; ++c)
        raw[c] = !on ? make_uint4(0, 0, 0, 0) : p.vec_q ? *reinterpret_cast<const uint4*>(place + 16 * c) : kv4_raw8(src + 8 * c, false);
      asm volatile("bar.sync %0, 128;" ::"r"(1 + x) : "memory");      // the four warps of the row tile have read
      float big = 0.0f;
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) {
        float y[8];
        kv4_floats8<T>(raw[c], y);
#pragma unroll
        for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(y[i]));
      }
      const int e = big > 0.0f ? min(120, max(-120, static_cast<int>(__float_as_uint(big) >> 23) - 127)) : 0;
      // a negative scale is taken into q, so that the largest score is the largest product
      const float down = copysignf(__uint_as_float(static_cast<uint32_t>(127 - e) << 23), p.scale_log2);
      // never zero, so that a hidden score stays at minus infinity
      factor = fmaxf(__uint_as_float(static_cast<uint32_t>(127 + e) << 23) * fabsf(p.scale_log2), 1e-35f);
      uint8_t* q = smem + x * Shape::kQ + row * 16;
      uint32_t lead[2] = {0, 0}, rest[2] = {0, 0};
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float sum = 0.0f;
#pragma unroll
        for (int c = 4 * g; c < 4 * g + 4; ++c) {
          float y[8];
          kv4_floats8<T>(raw[c], y);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y[i] *= down;
            sum += y[i];
          }
          *reinterpret_cast<uint4*>(q + c * Shape::kLeadQ) =
              make_uint4(pack_f16(y[0], y[4]), pack_f16(y[1], y[5]), pack_f16(y[2], y[6]), pack_f16(y[3], y[7]));
        }
        const __half hi = __float2half_rn(sum);
        lead[g / 2] |= static_cast<uint32_t>(__half_as_ushort(hi)) << (16 * (g & 1));
        rest[g / 2] |= static_cast<uint32_t>(__half_as_ushort(__float2half_rn(sum - __half2float(hi)))) << (16 * (g & 1));
      }
      *reinterpret_cast<uint4*>(q + HD / 8 * Shape::kLeadQ) = make_uint4(lead[0], lead[1], rest[0], rest[1]);
      *reinterpret_cast<uint4*>(q + (HD / 8 + 1) * Shape::kLeadQ) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full + 8 * x);
    }
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;      // 32 tensor memory lanes a warp
    const uint32_t s_at = tmem + lanes + Shape::kColS + x * KT, o_at = tmem + lanes + Shape::kColO + x * Shape::kWide;
    float top = -INFINITY;                  // maximum in use, log2 units
    uint32_t lost = 0;                      // groups that a NaN value has reached
    for (int i = 0; i < tiles; ++i) {
      if (!mbar_wait(s_full + 8 * x, i & 1)) { fine = false; break; }
      tc_fence_after();
      const uint32_t flag = lane < NB ? flags[(i & 3) * 8 + lane] : 1u;
      const uint32_t there = __ballot_sync(0xffffffffu, (flag & 1u) != 0), broken = __ballot_sync(0xffffffffu, (flag & 2u) != 0);
      // the keys that every row of the warp sees need no mask
      const bool masked = __any_sync(0xffffffffu, (i + 1) * KT > limit) || there != 0xffffffffu;
      if (broken != 0) {
        for (int k = 0; k < KT; ++k)
          if (((broken >> (k >> 4)) & 1u) && i * KT + k < limit) lost |= bad_keys[(i & 3) * KT + k];
        __syncwarp();
      }
      uint32_t v[NB][16];
#pragma unroll
      for (int c = 0; c < NB; ++c) tmem_ld_x16(s_at + 16 * c, v[c]);
      tmem_ld_wait();
      if (masked) {
#pragma unroll
        for (int c = 0; c < NB; ++c) {      // 16 columns = one block
          const int first = ((there >> c) & 1u) ? i * KT + 16 * c : INT32_MAX - 16;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (first + j >= limit) v[c][j] = 0xff800000u;
        }
      }
      float high[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int j = 0; j < 16; j += 2) high[j / 2 % 4] = max3(high[j / 2 % 4], __uint_as_float(v[c][j]), __uint_as_float(v[c][j + 1]));
      const float most = fmaxf(max3(high[0], high[1], high[2]), high[3]);
      const float next = most * factor;
      if (i == 0) {
        top = next;
      } else if (__any_sync(0xffffffffu, next > top + 8.0f || (top == -INFINITY && next > top))) {
        // the output product of the step before is through (the scores were issued after it)
        const float now = fmaxf(top, next), alpha = top == -INFINITY ? 0.0f : exp2_approx(top - now);
        top = now;
#pragma unroll 1
        for (int c = 0; c < Shape::kWide; c += 16) {
          uint32_t o[16];
          tmem_ld_x16(o_at + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
          tmem_st_x16(o_at + c, o);
        }
      }
      const float off = top == -INFINITY ? 0.0f : top;
      const uint64_t factor2 = pack_f32x2(factor, factor), off2 = pack_f32x2(-off, -off);
#pragma unroll
      for (int c = 0; c < NB; ++c) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          float e0, e1;
          unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[c][j]), __uint_as_float(v[c][j + 1])), factor2, off2), e0, e1);
          w[j / 2] = pack_f16(exp2_approx(e0), exp2_approx(e1));
        }
        tmem_st_x8(s_at + 8 * c, w);
        if (c == kHalf - 1) {      // the output product can start on these
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_half + 8 * x);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + 8 * x);
    }
    if (fine && tiles > 0) {
      fine = mbar_wait(o_done + 8 * x, (tiles - 1) & 1);
      tc_fence_after();
    }
    T* out = static_cast<T*>(p.out) + (q0 + tok) * p.o_tok + static_cast<int64_t>(head * p.group + at - tok * p.group) * p.o_head;
    T* place = reinterpret_cast<T*>(smem + x * Shape::kQ + row * Shape::kRow);      // the queries' place: their products are through
    uint32_t cen[16];
    if (fine && tiles > 0) {
      tmem_ld_x16(o_at + HD, cen);
      tmem_ld_wait();
    }
    const float sum = tiles > 0 ? __uint_as_float(cen[kSumRow]) : 0.0f, inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // 0: sees nothing
#pragma unroll
    for (int c = 0; c < HD; c += 16) {
      uint32_t v[16];
      __syncwarp();
      if (fine && tiles > 0) {
        tmem_ld_x16(o_at + c, v);
        tmem_ld_wait();
      }
      if (!on) continue;
      const bool nan = (lost >> (c / 32)) & 1u;
      float y[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        y[j] = nan ? __int_as_float(0x7fc00000) : inv == 0.0f ? 0.0f : (__uint_as_float(v[j]) + __uint_as_float(cen[c / 32])) * inv;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float z[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = y[8 * h + j];
        kv4_store8(p.vec_o ? place + c + 8 * h : out + c + 8 * h, p.vec_o, z);
      }
    }
    if (p.vec_o && on) {      // the row leaves by one bulk copy
      fence_proxy_async_smem();
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(out), "r"(smem_u32(place)), "r"(HD * 2) : "memory");
      bulk_commit();
      bulk_wait_read0();
    }
  }
  if (!fine && lane == 0) kv4_report(p.status, kDevKv4Timeout);
  tc_fence_before();
  __syncthreads();
  if (warp == 15) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace crl
