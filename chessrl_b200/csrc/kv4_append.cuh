// Appending to and reading from the 4-bit cache (layout: kv4.cuh).
//
// A CTA takes a few tokens: where each goes (its sequence, page and row of the rotation table) is looked up once. A row
// (a token's head of q, k or v) is worked on by hd / 8 neighbouring lanes of a warp, eight values each: a 16-byte load,
// the rotation, the group's extremes over four lanes by two shuffles, one 32-bit word of codes per lane. Key words are
// stored as they are; value words are the transpose of 8 lanes x 8 nibbles, three exchanges away.
//
// Bound by instruction issue for prompts (the rotation is 13 instructions a value, see kv4_turn; the codes 6): 19k prompt
// tokens of 32 + 2 x 8 heads of 128, half of each head rotated, appended and read back in 178 us (2.9 TB/s of the 6.5 that
// a copy reaches; 201 with 64 registers and four CTAs per SM instead of 40 and six, 190 with half-rotated query rows like
// all others). Single tokens are bound by the launch:
// 4.6 us for one, 6.2 us for 256 sequences, append and read together.
#pragma once
#include "kv4.cuh"

namespace crl {

struct Kv4AppendParams {
  uint8_t* pages;
  Kv4Table table;
  const int32_t* starts;      // [seqs] cache indices held before the call
  const int32_t* cu;          // [seqs + 1] first token row of each sequence; null: one token each
  int32_t seqs, kv_heads, heads;   // heads: rows of q to rotate per token (0: none)
  int64_t tokens;
  const void *q, *k, *v;
  void* q_out;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;   // strides in elements
  const float2* rope;         // [positions][rot / 2] (cos, sin), or null
  int64_t rope_positions;
  int32_t rot, interleaved;
  int32_t vec_q, vec_k, vec_v, vec_o;    // rows 16-byte aligned
  int32_t per_cta;            // tokens of a CTA, at most kKv4CtaTokens
  uint32_t over_rows;         // ceil(2^32 / rows per token), to divide a CTA's row numbers
  int* status;
};

// the rotated values of dims 8 * part .. + 7 of a row
template <typename T>
__device__ __forceinline__ void kv4_rotate(const T* row, bool vec, const float2* rope, int rot, bool interleaved, int part,
                                           float (&x)[8]) {
  const int d0 = part * 8;
  if (rope == nullptr || d0 >= rot) return;
  const int half = rot >> 1;
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (d0 + i >= rot) break;
      const float2 cs = rope[(d0 + i) >> 1];
      const float a = x[i], b = x[i + 1];
      x[i] = kv4_turn(a, cs.x, b, cs.y);
      x[i + 1] = kv4_turn(b, cs.x, -a, cs.y);
    }
  } else if ((half & 7) == 0) {
    const bool first = d0 < half;
    const int base = first ? d0 : d0 - half;
    float o[8];
    kv4_load8(row + (first ? d0 + half : d0 - half), vec, o);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 cs = rope[base + i];
      x[i] = kv4_turn(x[i], cs.x, first ? o[i] : -o[i], cs.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = d0 + i;
      if (d >= rot) break;
      const bool first = d < half;
      const float o = kv4_to_float(row[first ? d + half : d - half]);
      const float2 cs = rope[first ? d : d - half];
      x[i] = kv4_turn(x[i], cs.x, first ? o : -o, cs.y);
    }
  }
}

// A query row of which half is rotated: every lane takes two pairs and four of the dims that stay, where eight neighbouring
// dims to a lane would have half of the lanes do the arithmetic (rows 16-byte aligned).
template <typename T, int HD>
__device__ __forceinline__ void kv4_rotate_half_row(const T* row, T* out, const float2* rope, bool interleaved, int part) {
  constexpr int ROT = HD / 2, APART = ROT / 2;
  const uint2 stay = *reinterpret_cast<const uint2*>(row + ROT + 4 * part);
  const float2 c0 = rope[2 * part], c1 = rope[2 * part + 1];
  T x[4];      // interleaved: a0 b0 a1 b1; halves: a0 a1 b0 b1
  if (interleaved) {
    *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(row + 4 * part);
  } else {
    *reinterpret_cast<uint32_t*>(x) = *reinterpret_cast<const uint32_t*>(row + 2 * part);
    *reinterpret_cast<uint32_t*>(x + 2) = *reinterpret_cast<const uint32_t*>(row + APART + 2 * part);
  }
  const float a0 = kv4_to_float(x[0]), b0 = kv4_to_float(interleaved ? x[1] : x[2]);
  const float a1 = kv4_to_float(interleaved ? x[2] : x[1]), b1 = kv4_to_float(x[3]);
  const T y0 = kv4_from_float<T>(kv4_turn(a0, c0.x, b0, c0.y)), z0 = kv4_from_float<T>(kv4_turn(b0, c0.x, -a0, c0.y));
  const T y1 = kv4_from_float<T>(kv4_turn(a1, c1.x, b1, c1.y)), z1 = kv4_from_float<T>(kv4_turn(b1, c1.x, -a1, c1.y));
  x[0] = y0;
  x[1] = interleaved ? z0 : y1;
  x[2] = interleaved ? y1 : z0;
  x[3] = z1;
  if (interleaved) {
    *reinterpret_cast<uint2*>(out + 4 * part) = *reinterpret_cast<const uint2*>(x);
  } else {
    *reinterpret_cast<uint32_t*>(out + 2 * part) = *reinterpret_cast<const uint32_t*>(x);
    *reinterpret_cast<uint32_t*>(out + APART + 2 * part) = *reinterpret_cast<const uint32_t*>(x + 2);
  }
  *reinterpret_cast<uint2*>(out + ROT + 4 * part) = stay;
}

constexpr int kKv4CtaTokens = 8, kKv4Threads = 256;

struct Kv4Place {
  uint32_t block;     // block of head 0 that the token's row lies in, kNoBlock: none
  int32_t row;        // its row there
  int32_t ok;         // the token belongs to a sequence (and has a place in the rotation table)
  const float2* rope;
};

// Where the CTA's tokens go. Rows behind the last sequence have ok = 0.
template <typename P>
__device__ __forceinline__ Kv4Place kv4_place(const P& p, int64_t tok, const float2* rope, int64_t positions, int half) {
  Kv4Place w{kNoBlock, 0, 0, nullptr};
  if (tok >= p.tokens) return w;
  int seq = static_cast<int>(tok);
  int64_t offset = 0;
  if (p.cu != nullptr) {
    seq = kv4_seq_of(p.cu, p.seqs, tok);
    offset = tok - p.cu[seq];
    if (tok >= p.cu[p.seqs] || offset < 0) return w;
  } else if (tok >= p.seqs) {
    return w;
  }
  const int64_t index = p.starts[seq] + offset;
  if (rope != nullptr) {
    if (index < 0 || index >= positions) {
      kv4_report(p.status, kDevKv4Rope);
      return w;
    }
    w.rope = rope + index * half;
  }
  w.ok = 1;
  w.row = static_cast<int32_t>(index & 15);
  if (index >= 0 && index <= INT32_MAX)
    w.block = kv4_block_of(p.table, p.table.table + seq * p.table.stride, static_cast<int>(index >> 4));
  if (w.block == kNoBlock) kv4_report(p.status, kDevKv4Table);
  return w;
}

// Transposes the 8 x 8 nibbles of eight neighbouring lanes: nibble j of lane i becomes nibble i of lane j.
__device__ __forceinline__ uint32_t transpose_nibbles(uint32_t w, int lane) {
  uint32_t o = __shfl_xor_sync(0xffffffffu, w, 4);
  w = __byte_perm(w, o, (lane & 4) ? 0x3276 : 0x5410);
  o = __shfl_xor_sync(0xffffffffu, w, 2);
  w = __byte_perm(w, o, (lane & 2) ? 0x3715 : 0x6240);
  o = __shfl_xor_sync(0xffffffffu, w, 1);
  const uint32_t keep = (lane & 1) ? 0xf0f0f0f0u : 0x0f0f0f0fu;
  return (w & keep) | (((lane & 1) ? o >> 4 : o << 4) & ~keep);
}

// hd 32: eight lanes hold two rows of four. After the transpose lane r has part r of the first row in its low half and of
// the second in its high half; a row's lane takes its two parts from their lanes.
__device__ __forceinline__ uint32_t pair_rows(uint32_t w, int lane) {
  const int from = (lane & ~7) + 2 * (lane & 3);
  const uint32_t a = __shfl_sync(0xffffffffu, w, from), b = __shfl_sync(0xffffffffu, w, from + 1);
  return __byte_perm(a, b, (lane & 4) ? 0x7632 : 0x5410);
}
// and back: a lane's word holds parts 2 l, 2 l + 1 of its row; the transpose wants part r of both rows in lane r
__device__ __forceinline__ uint32_t unpair_rows(uint32_t w, int lane) {
  const int r = lane & 7, from = (lane & ~7) + r / 2;
  const uint32_t a = __shfl_sync(0xffffffffu, w, from), b = __shfl_sync(0xffffffffu, w, from + 4);
  return __byte_perm(a, b, (r & 1) ? 0x7632 : 0x5410);
}
// The word of a value row that lane `part` holds the transpose of: lane 8 w + r has nibble r of lanes 8 w .. 8 w + 7.
template <int HD>
__device__ __forceinline__ int value_word(int part) {
  return HD == 32 ? part : (part & 7) * (HD / 64) + part / 8;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kKv4Threads, 6) kv4_append_kernel(const Kv4AppendParams p) {
  constexpr int LANES = HD / 8, G = HD / 32, AT_ONCE = kKv4Threads / LANES;
  __shared__ Kv4Place places[kKv4CtaTokens];
  const int lane = threadIdx.x & 31, part = lane % LANES;
  const int64_t tok0 = static_cast<int64_t>(blockIdx.x) * p.per_cta;
  if (threadIdx.x < p.per_cta) places[threadIdx.x] = kv4_place(p, tok0 + threadIdx.x, p.rope, p.rope_positions, p.rot >> 1);
  __syncthreads();
  const uint32_t per_token = p.heads + 2 * p.kv_heads, rows = per_token * p.per_cta;
  for (uint32_t base = 0; base < rows; base += AT_ONCE) {
    const uint32_t unit = base + threadIdx.x / LANES;
    const uint32_t mine = min(unit, rows - 1), local = __umulhi(mine, p.over_rows);
    int h = static_cast<int>(mine - local * per_token);
    const Kv4Place& w = places[local];
    const int64_t tok = tok0 + local;
    const bool live = unit < rows && w.ok != 0, is_q = h < p.heads;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (live && is_q) {
      const T* row = static_cast<const T*>(p.q) + tok * p.q_tok + h * p.q_head;
      T* out = static_cast<T*>(p.q_out) + tok * p.o_tok + h * p.o_head;
      if (w.rope != nullptr && p.rot == HD / 2 && p.vec_q && p.vec_o) {
        kv4_rotate_half_row<T, HD>(row, out, w.rope, p.interleaved, part);
      } else {
        kv4_load8(row + part * 8, p.vec_q, x);
        kv4_rotate(row, p.vec_q, w.rope, p.rot, p.interleaved, part, x);
        kv4_store8(out + part * 8, p.vec_o, x);
      }
    }
    const bool ok = live && !is_q && w.block != kNoBlock;
    if (!__any_sync(0xffffffffu, ok)) continue;
    h -= p.heads;
    const bool is_k = h < p.kv_heads;
    if (!is_k) h -= p.kv_heads;
    if (ok) {
      const T* row = is_k ? static_cast<const T*>(p.k) + tok * p.k_tok + h * p.k_head
                          : static_cast<const T*>(p.v) + tok * p.v_tok + h * p.v_head;
      const bool vec = is_k ? p.vec_k : p.vec_v;
      kv4_load8(row + part * 8, vec, x);
      if (is_k) kv4_rotate(row, vec, w.rope, p.rot, p.interleaved, part, x);
    }
    // every lane of the warp takes part in the exchanges below
    float lo = INFINITY, hi = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      nan |= x[i] != x[i];
      x[i] = fminf(fmaxf(x[i], -kKv4Limit), kKv4Limit);
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
    }
    if (nan) hi = INFINITY;      // the clamp leaves nothing this large: it marks a group with a NaN
#pragma unroll
    for (int m = 1; m < 4; m <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    }
    if (hi == INFINITY) lo = hi = __int_as_float(0x7fc00000);      // such a group is NaN as a whole
    const __half s16 = __float2half_rn(__bfloat162float(__float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f))));
    const float s = __half2float(s16);
    const __half c16 = __float2half_rn(__fadd_rn(lo, __fmul_rn(8.0f, s)));
    const float c = __half2float(c16);
    const float inv = s > 0.0f ? __frcp_rn(s) : 0.0f;
    // n - 8 is clamped first and rounded to even by adding 1.5 * 2^23; with 8 more the low bits of the sum are n, and
    // the eight sums are strung together as base-16 digits (the constant part of the digits comes off at the end)
    uint32_t word = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      const float n = fminf(fmaxf(__fmul_rn(__fsub_rn(x[i], c), inv), -8.0f), 7.0f);
      word = word * 16u + __float_as_uint(n + 12582920.0f);
    }
    word -= 0x4b400000u * 0x11111111u;
    uint32_t turned = transpose_nibbles(word, lane);
    if constexpr (HD == 32) turned = pair_rows(turned, lane);
    if (!ok) continue;
    uint8_t* at = p.pages + static_cast<size_t>(w.block + h * p.table.blocks) * kv4_block_bytes(HD) + (is_k ? 0 : 10 * HD);
    const int g = part / 4, t = part % 4;
    uint8_t* codes = at + w.row * (HD / 2);
    reinterpret_cast<uint32_t*>(codes)[is_k ? t * G + g : value_word<HD>(part)] = is_k ? word : turned;
    if (t == 0) reinterpret_cast<__half2*>(at + 8 * HD + w.row * (HD / 8))[g] = __halves2half2(s16, c16);
  }
}

struct Kv4ReadParams {
  const uint8_t* pages;
  Kv4Table table;
  const int32_t* starts;
  const int32_t* cu;
  int32_t seqs, kv_heads;
  int64_t tokens;
  void *k, *v;
  int64_t k_tok, k_head, v_tok, v_head;
  int32_t vec_k, vec_v;
  int32_t per_cta;
  uint32_t over_rows;
  int* status;
};

template <typename T, int HD>
__global__ void __launch_bounds__(kKv4Threads) kv4_read_kernel(const Kv4ReadParams p) {
  constexpr int LANES = HD / 8, G = HD / 32, AT_ONCE = kKv4Threads / LANES;
  __shared__ Kv4Place places[kKv4CtaTokens];
  const int lane = threadIdx.x & 31, part = lane % LANES, g = part / 4, t = part % 4;
  const int64_t tok0 = static_cast<int64_t>(blockIdx.x) * p.per_cta;
  if (threadIdx.x < p.per_cta) places[threadIdx.x] = kv4_place(p, tok0 + threadIdx.x, static_cast<const float2*>(nullptr), 0, 0);
  __syncthreads();
  const uint32_t per_token = 2 * p.kv_heads, rows = per_token * p.per_cta;
  for (uint32_t base = 0; base < rows; base += AT_ONCE) {
    const uint32_t unit = base + threadIdx.x / LANES;
    const uint32_t mine = min(unit, rows - 1), local = __umulhi(mine, p.over_rows);
    int h = static_cast<int>(mine - local * per_token);
    const bool is_k = h < p.kv_heads;
    if (!is_k) h -= p.kv_heads;
    const Kv4Place& w = places[local];
    const int64_t tok = tok0 + local;
    uint32_t word = 0;
    float s = 0.0f, c = 0.0f;      // a row that is not there is zero
    if (w.block != kNoBlock) {
      const uint8_t* at = p.pages + static_cast<size_t>(w.block + h * p.table.blocks) * kv4_block_bytes(HD) + (is_k ? 0 : 10 * HD);
      word = reinterpret_cast<const uint32_t*>(at + w.row * (HD / 2))[is_k ? t * G + g : value_word<HD>(part)];
      const float2 sc = __half22float2(reinterpret_cast<const __half2*>(at + 8 * HD + w.row * (HD / 8))[g]);
      s = sc.x;
      c = sc.y;
    }
    uint32_t turned = word;
    if constexpr (HD == 32) turned = unpair_rows(turned, lane);
    turned = transpose_nibbles(turned, lane);
    if (!is_k) word = turned;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)      // 2^23 + n as a bit pattern, minus 2^23 + 8
      x[i] = __fmaf_rn(__uint_as_float(((word >> (4 * i)) & 15u) | 0x4b000000u) - 8388616.0f, s, c);
    if (unit >= rows || tok >= p.tokens) continue;
    T* out = is_k ? static_cast<T*>(p.k) + tok * p.k_tok + h * p.k_head : static_cast<T*>(p.v) + tok * p.v_tok + h * p.v_head;
    kv4_store8(out + part * 8, is_k ? p.vec_k : p.vec_v, x);
  }
}

}  // namespace crl
