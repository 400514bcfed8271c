// Appending to and reading from the 4-bit cache (layout: kv4.cuh).
//
// One row (a token's head of q, k or v) is worked on by hd / 8 neighbouring lanes of a warp, eight values each: a
// 16-byte load, the rotation, the group's extremes over four lanes by two shuffles, one 32-bit word of codes per lane.
// Key words are stored as they are; value words are the transpose (8 lanes x 8 nibbles) taken by shuffles.
// Bound by memory for prompts and by the launch for single tokens.
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

template <typename T, int HD>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4AppendParams p) {
  constexpr int LANES = HD / 8, G = HD / 32;
  const int lane = threadIdx.x & 31, part = lane % LANES;
  const int per_token = p.heads + 2 * p.kv_heads;
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / LANES;
  const int64_t total = p.tokens * per_token;
  const bool live = unit < total;
  const int64_t tok = live ? unit / per_token : 0;
  int h = live ? static_cast<int>(unit - tok * per_token) : 0;
  // which sequence, which cache index
  int seq = 0;
  int64_t offset = 0;
  bool ok = live;
  if (p.cu == nullptr) {
    seq = static_cast<int>(tok);
    ok = ok && tok < p.seqs;
  } else if (ok) {
    seq = kv4_seq_of(p.cu, p.seqs, tok);
    offset = tok - p.cu[seq];
    ok = tok < p.cu[p.seqs] && offset >= 0;      // rows behind the last sequence are left alone
  }
  int64_t index = 0;
  const float2* rope = nullptr;
  if (ok) {
    index = p.starts[seq] + offset;
    if (p.rope != nullptr) {
      if (index < 0 || index >= p.rope_positions) {
        kv4_report(p.status, kDevKv4Rope);
        ok = false;
      } else {
        rope = p.rope + index * (p.rot >> 1);
      }
    }
  }
  const bool is_q = h < p.heads;
  h -= p.heads;
  const bool is_k = h < p.kv_heads;
  if (!is_q && !is_k) h -= p.kv_heads;
  float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (ok && is_q) {
    const T* row = static_cast<const T*>(p.q) + tok * p.q_tok + static_cast<int64_t>(h + p.heads) * p.q_head;
    kv4_load8(row + part * 8, p.vec_q, x);
    kv4_rotate(row, p.vec_q, rope, p.rot, p.interleaved, part, x);
    kv4_store8(static_cast<T*>(p.q_out) + tok * p.o_tok + static_cast<int64_t>(h + p.heads) * p.o_head + part * 8, p.vec_o, x);
    ok = false;
  }
  int64_t block = -1;
  if (ok) {
    block = index < 0 || index > INT32_MAX ? -1 : kv4_block_of(p.table, p.kv_heads, seq, static_cast<int>(index >> 4));
    if (block < 0) {
      kv4_report(p.status, kDevKv4Table);
      ok = false;
    }
  }
  if (ok) {
    const T* row = is_k ? static_cast<const T*>(p.k) + tok * p.k_tok + static_cast<int64_t>(h) * p.k_head
                        : static_cast<const T*>(p.v) + tok * p.v_tok + static_cast<int64_t>(h) * p.v_head;
    const bool vec = is_k ? p.vec_k : p.vec_v;
    kv4_load8(row + part * 8, vec, x);
    if (is_k) kv4_rotate(row, vec, rope, p.rot, p.interleaved, part, x);
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
#pragma unroll
  for (int m = 1; m < 4; m <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    nan |= __shfl_xor_sync(0xffffffffu, static_cast<int>(nan), m) != 0;
  }
  if (nan) lo = hi = __int_as_float(0x7fc00000);      // a NaN makes its whole group NaN
  const __half s16 = __float2half_rn(__bfloat162float(__float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f))));
  const float s = __half2float(s16);
  const __half c16 = __float2half_rn(__fadd_rn(lo, __fmul_rn(8.0f, s)));
  const float c = __half2float(c16);
  const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float n = rintf(__fmul_rn(__fsub_rn(x[i], c), inv)) + 8.0f;
    n = fminf(fmaxf(n, 0.0f), 15.0f);
    word |= static_cast<uint32_t>(n) << (4 * i);
  }
  // value rows: nibble position 8 * part + m of the row = (r, i) holds nibble r of lane i's word
  uint32_t turned = 0;
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    const int pos = part * 8 + m, r = pos / LANES, i = pos % LANES;
    const uint32_t w = __shfl_sync(0xffffffffu, word, (lane - part) + i);
    turned |= ((w >> (4 * r)) & 15u) << (4 * m);
  }
  if (!ok) return;
  uint8_t* at = p.pages + (block + static_cast<int64_t>(h) * p.table.blocks) * kv4_block_bytes(HD) + (is_k ? 0 : 10 * HD);
  const int row = static_cast<int>(index & 15);
  const int g = part / 4, t = part % 4;
  reinterpret_cast<uint32_t*>(at + row * (HD / 2))[is_k ? t * G + g : part] = is_k ? word : turned;
  if (t == 0) reinterpret_cast<__half2*>(at + 8 * HD + row * (HD / 8))[g] = __halves2half2(s16, c16);
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
  int* status;
};

template <typename T, int HD>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadParams p) {
  constexpr int LANES = HD / 8, G = HD / 32;
  const int lane = threadIdx.x & 31, part = lane % LANES;
  const int per_token = 2 * p.kv_heads;
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / LANES;
  const bool live = unit < p.tokens * per_token;
  bool ok = live;
  const int64_t tok = ok ? unit / per_token : 0;
  int h = ok ? static_cast<int>(unit - tok * per_token) : 0;
  int seq = 0;
  int64_t offset = 0;
  if (p.cu == nullptr) {
    seq = static_cast<int>(tok);
    ok = ok && tok < p.seqs;
  } else if (ok) {
    seq = kv4_seq_of(p.cu, p.seqs, tok);
    offset = tok - p.cu[seq];
    ok = tok < p.cu[p.seqs] && offset >= 0;
  }
  const bool is_k = h < p.kv_heads;
  if (!is_k) h -= p.kv_heads;
  int64_t index = 0, block = -1;
  if (ok) {
    index = p.starts[seq] + offset;
    block = index < 0 || index > INT32_MAX ? -1 : kv4_block_of(p.table, p.kv_heads, seq, static_cast<int>(index >> 4));
    if (block < 0) {
      kv4_report(p.status, kDevKv4Table);
      ok = false;
    }
  }
  const int g = part / 4, t = part % 4;
  uint32_t word = 0;
  float s = 0.0f, c = 0.0f;
  if (ok) {
    const uint8_t* at = p.pages + (block + static_cast<int64_t>(h) * p.table.blocks) * kv4_block_bytes(HD) + (is_k ? 0 : 10 * HD);
    const int row = static_cast<int>(index & 15);
    word = reinterpret_cast<const uint32_t*>(at + row * (HD / 2))[is_k ? t * G + g : part];
    const float2 sc = __half22float2(reinterpret_cast<const __half2*>(at + 8 * HD + row * (HD / 8))[g]);
    s = sc.x;
    c = sc.y;
  }
  float x[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int pos = r * LANES + part;        // values: nibble position of dim 8 * part + r
    const uint32_t w = __shfl_sync(0xffffffffu, word, (lane - part) + pos / 8);
    const uint32_t n = is_k ? word >> (4 * r) : w >> (4 * (pos % 8));
    x[r] = __fmaf_rn(static_cast<float>(static_cast<int>(n & 15u) - 8), s, c);      // no row: s = c = 0
  }
  if (!live) return;
  T* out = is_k ? static_cast<T*>(p.k) + tok * p.k_tok + static_cast<int64_t>(h) * p.k_head
                : static_cast<T*>(p.v) + tok * p.v_tok + static_cast<int64_t>(h) * p.v_head;
  kv4_store8(out + part * 8, is_k ? p.vec_k : p.vec_v, x);
}

}  // namespace crl
