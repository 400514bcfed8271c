// Next-token logits: penalties for tokens already said, biases, bit masks; one pass over the rows.
//
//   z = logits[row, v] (fp32);  n = how often v stands in the row's history
//   n > 0:  z = z > 0 ? z / repetition : z * repetition;  z = z - (frequency * n + presence)
//   z = z + bias of v (where an id is given more than once, its last entry counts)
//   mask bit v of the row clear:  z = masked_value
// each operation rounded once, the result once more to the row's type. A CTA takes one tile of one row: the history and
// the biases that fall into the tile are entered into a table in shared memory (integers, so the order in which they
// arrive does not matter) while its rows' pieces are under way. Measured: 4096 rows of 1929 fp32 with legal-move masks 13.6 us =
// 4.8 TB/s (of 6.5 that a copy reaches), 64 rows of 50304 f16 with histories of 1024: 6.9 us, one row 3.0 us (the launch).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace crl {

enum LogitsStatus : int { kDevLogitsMaskRow = 131 };      // a row asks for a mask that the table does not have

struct LogitsParams {
  const void* in;
  void* out;
  int64_t in_stride, out_stride;
  int64_t rows;
  int32_t vocab, tile, tiles;
  const int32_t* history;      // [rows, history_len], entries outside the vocabulary are padding; null: none
  int64_t history_stride;
  int32_t history_len;
  const float *repetition, *frequency, *presence;   // [rows]; null: 1, 0, 0
  const int32_t* bias_ids;     // [rows, biases]; entries outside the vocabulary are padding
  const float* bias_values;
  int64_t bias_stride, value_stride;
  int32_t biases;
  const uint8_t* mask;         // [mask_count, mask_stride] bit v of a row: v allowed; null: no mask
  int64_t mask_stride;
  int32_t mask_count;
  const int32_t* mask_rows;    // [rows] which mask a row takes, negative: none; null: its own number
  float masked_value;
  int32_t same_phase;          // in and out rows have the same offset from a 16-byte boundary
  int* status;
};

template <typename T> __device__ __forceinline__ float logit_to(T x);
template <> __device__ __forceinline__ float logit_to(float x) { return x; }
template <> __device__ __forceinline__ float logit_to(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float logit_to(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T logit_from(float x);
template <> __device__ __forceinline__ float logit_from(float x) { return x; }
template <> __device__ __forceinline__ __half logit_from(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 logit_from(float x) { return __float2bfloat16_rn(x); }

// table entry: how often the token was said (low 20 bits), 1 + the number of its last bias entry (high 12)
constexpr int kLogitsMaxHistory = (1 << 20) - 1, kLogitsMaxBiases = (1 << 12) - 2;
constexpr int kLogitsThreads = 256, kLogitsAhead = 2;

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) adjust_logits_kernel(const LogitsParams p) {
  extern __shared__ __align__(16) uint32_t room[];
  constexpr int VEC = 16 / sizeof(T);
  const int64_t row = blockIdx.x / p.tiles;
  const int tile = static_cast<int>(blockIdx.x - row * p.tiles);
  const int v0 = tile * p.tile, n = min(p.tile, p.vocab - v0);
  const bool marks = p.history != nullptr || p.biases > 0;
  const T* in = static_cast<const T*>(p.in) + row * p.in_stride + v0;
  T* out = static_cast<T*>(p.out) + row * p.out_stride + v0;
  const float* values = p.bias_values + (p.biases > 0 ? row * p.value_stride : 0);
  // 16-byte pieces from the first boundary on, single elements around them; a thread's pieces are under way while the
  // table is made
  const int lead = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(in) & 15)) & 15) / static_cast<int>(sizeof(T));
  const int head = p.same_phase ? min(lead, n) : n;
  const int pieces = (n - head) / VEC;
  uint32_t* table = room + ((4 - (head & 3)) & 3);      // a piece's entries start on a 16-byte boundary
  uint4 ahead[kLogitsAhead];
#pragma unroll
  for (int u = 0; u < kLogitsAhead; ++u) {
    const int q = threadIdx.x + u * kLogitsThreads;
    ahead[u] = q < pieces ? *reinterpret_cast<const uint4*>(in + head + q * VEC) : make_uint4(0, 0, 0, 0);
  }
  const float rep = p.repetition != nullptr ? p.repetition[row] : 1.0f;
  const float freq = p.frequency != nullptr ? p.frequency[row] : 0.0f;
  const float pres = p.presence != nullptr ? p.presence[row] : 0.0f;
  const uint8_t* bits = nullptr;
  if (p.mask != nullptr) {
    const int64_t m = p.mask_rows != nullptr ? p.mask_rows[row] : row;
    if (m >= p.mask_count) {
      if (threadIdx.x == 0 && p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kDevLogitsMaskRow));
    } else if (m >= 0) {
      bits = p.mask + m * p.mask_stride;
    }
  }
  if (marks) {
    for (int i = threadIdx.x; i < (n + 6) / 4; i += kLogitsThreads) reinterpret_cast<uint4*>(room)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int32_t* ids = p.bias_ids + (p.biases > 0 ? row * p.bias_stride : 0);
    for (int i = threadIdx.x; i < p.biases; i += kLogitsThreads) {
      const int64_t at = static_cast<int64_t>(ids[i]) - v0;
      if (at >= 0 && at < n) atomicMax(&table[at], static_cast<uint32_t>(i + 1) << 20);
    }
    if (p.biases > 0) __syncthreads();
    if (p.history != nullptr) {
      const int32_t* said = p.history + row * p.history_stride;
      for (int i = threadIdx.x; i < p.history_len; i += kLogitsThreads) {
        const int64_t at = static_cast<int64_t>(said[i]) - v0;
        if (at >= 0 && at < n) atomicAdd(&table[at], 1u);
      }
    }
    __syncthreads();
  }
  const T masked = logit_from<T>(p.masked_value);
  auto adjusted = [&](T x, uint32_t mark) -> T {
    float z = logit_to<T>(x);
    const uint32_t count = mark & 0xfffffu, last = mark >> 20;
    if (count != 0) {
      z = z > 0.0f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
      z = __fsub_rn(z, __fadd_rn(__fmul_rn(freq, static_cast<float>(count)), pres));
    }
    if (last != 0) z = __fadd_rn(z, values[last - 1]);
    return logit_from<T>(z);
  };
  auto allowed = [&](int i) { return bits == nullptr || ((bits[(v0 + i) >> 3] >> ((v0 + i) & 7)) & 1) != 0; };
  auto piece = [&](int q, const uint4& raw) {
    const int i = head + q * VEC;
    T x[VEC];
    *reinterpret_cast<uint4*>(x) = raw;
    uint32_t m = ~0u;
    if (bits != nullptr) {
      const int v = v0 + i, b = v >> 3;
      m = bits[b];
      if ((v & 7) + VEC > 8) m |= static_cast<uint32_t>(bits[b + 1]) << 8;
      m >>= v & 7;
    }
    if (marks) {
      uint32_t mark[VEC], any = 0;
#pragma unroll
      for (int j = 0; j < VEC; j += 4) *reinterpret_cast<uint4*>(mark + j) = *reinterpret_cast<const uint4*>(table + i + j);
#pragma unroll
      for (int j = 0; j < VEC; ++j) any |= mark[j];
      if (any != 0) {
        // marked entries are few and most of them masked: one after the other rather than all eight alike
        uint32_t left = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) left |= mark[j] != 0 ? 1u << j : 0u;
        for (left &= m; left != 0; left &= left - 1) {
          const int at = __ffs(left) - 1;
          T y = x[0];
#pragma unroll
          for (int j = 1; j < VEC; ++j) y = at == j ? x[j] : y;
          y = adjusted(y, table[i + at]);
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[j] = at == j ? y : x[j];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = (m >> j) & 1u ? x[j] : masked;
    *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(x);
  };
#pragma unroll
  for (int u = 0; u < kLogitsAhead; ++u)
    if (threadIdx.x + u * kLogitsThreads < pieces) piece(threadIdx.x + u * kLogitsThreads, ahead[u]);
  for (int q = threadIdx.x + kLogitsAhead * kLogitsThreads; q < pieces; q += kLogitsThreads)
    piece(q, *reinterpret_cast<const uint4*>(in + head + q * VEC));
  const int tail = head + pieces * VEC, singles = head + n - tail;
  for (int q = threadIdx.x; q < singles; q += kLogitsThreads) {
    const int i = q < head ? q : tail + q - head;
    const T x = in[i];
    out[i] = !allowed(i) ? masked : marks && table[i] != 0 ? adjusted(x, table[i]) : x;
  }
}

}  // namespace crl
