// The 4-bit key/value cache: layout of a page, quantisation, and what the kernels that touch it share.
//
// A (token, head) row of head_dim values is cut into groups of 32. A group is held as two f16 numbers, the step s and
// the centre c, and one 4-bit code n per value, which stands for (n - 8) * s + c. With lo / hi the group's extremes
//     s = f16(bf16((hi - lo) * (1 / 15))),  c = f16(lo + 8 s),  n = clamp(rint((x - c) * (1 / s)) + 8, 0, 15),  n = 8 where s = 0
// in fp32 (1 / 15 and 1 / s rounded to fp32 first). The step keeps eight significant bits (the detour over bf16), so (n - 8) * s has at most eleven and is exact
// in f16: the attention kernels feed codes to the tensor cores without a further rounding. The rounding of the step
// costs under 2^-9 of a step per code, against half a step of the code itself.
//
// Pages: [num_pages][kv_heads][page_size / 16] blocks of 16 tokens; a block is
//     key codes [16][hd / 2] | key (s, c) [16][hd / 32] | value codes [16][hd / 2] | value (s, c) [16][hd / 32]
// = 20 hd bytes, a multiple of 16 bytes for one bulk copy. Nibble p of a row (low half of a byte first) holds
//     keys:    p = (t, g, i), t < 4, g < hd / 32, i < 8  ->  dim 32 g + 8 t + i
//     values:  p = (r, i), r < 8, i < hd / 8             ->  dim 8 i + r
// which is the order in which a warp's lanes want them as matrix operands (lane 4 r + t): one aligned load per lane and
// row, no exchange between lanes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "ptx.cuh"

namespace crl {

constexpr float kKv4Limit = 57344.0f;   // |value| beyond this is held as this: (n - 8) * s + c stays inside f16
constexpr int kKv4Block = 16;           // tokens of a block

enum Kv4Status : int {
  kDevKv4Table = 121,     // a cache index past its sequence's row of the block table, or a page number outside the pool
  kDevKv4Run = 122,       // a sequence has more new tokens than the call allows for, or token rows past the tensor
  kDevKv4Rope = 123,      // a position past the rotation table
  kDevKv4Timeout = 124,   // a bounded wait on a block's copy ran out
};

__host__ __device__ constexpr int kv4_block_bytes(int hd) { return 20 * hd; }

__device__ __forceinline__ void kv4_report(int* status, int code) {
  if (status != nullptr) atomicCAS(status, 0, code);
}

// Where the block of cache index `index` of a sequence lies: its number in [num_pages][kv_heads][blocks per page] for
// head 0, or kNoBlock for an index that the table does not cover or a page that the pool does not have. Block numbers
// are 32-bit (2^32 blocks of 640 bytes or more are more than a GPU holds; the host checks).
struct Kv4Table {
  const int32_t* table;   // [seqs][stride]
  int64_t stride;
  int32_t width;          // pages a sequence can have
  int32_t blocks;         // 16-token blocks per page
  int32_t shift;          // its logarithm where it is a power of two, else -1
  uint32_t num_pages;
  uint32_t page_blocks;   // kv_heads * blocks
};
constexpr uint32_t kNoBlock = 0xffffffffu;
__device__ __forceinline__ uint32_t kv4_block_of(const Kv4Table& t, const int32_t* row, int block) {
  const int slot = t.shift >= 0 ? block >> t.shift : block / t.blocks;
  if (static_cast<uint32_t>(slot) >= static_cast<uint32_t>(t.width)) return kNoBlock;
  const uint32_t page = static_cast<uint32_t>(row[slot]);
  if (page >= t.num_pages) return kNoBlock;
  return page * t.page_blocks + static_cast<uint32_t>(block - slot * t.blocks);
}

// The sequence that token row `row` belongs to: the last one whose first row is not behind it (cu ascending, cu[0] = 0).
__device__ __forceinline__ int kv4_seq_of(const int32_t* cu, int seqs, int64_t row) {
  int lo = 0, hi = seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= row) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// n / d for a divisor that the host knows: one multiplication while n * d < 2^32
struct Kv4Divisor {
  uint32_t d, mul;      // mul = ceil(2^32 / d), 0 where the bound does not hold (or d is 1)
};
__device__ __forceinline__ int kv4_div(int n, const Kv4Divisor& v) {
  if (v.mul != 0) return static_cast<int>(__umulhi(static_cast<uint32_t>(n), v.mul));
  return v.d == 1 ? n : n / static_cast<int>(v.d);
}

template <typename T> __device__ __forceinline__ float kv4_to_float(T x);
template <> __device__ __forceinline__ float kv4_to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float kv4_to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T kv4_from_float(float x);
template <> __device__ __forceinline__ __half kv4_from_float(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 kv4_from_float(float x) { return __float2bfloat16_rn(x); }

// eight consecutive values as they are; `vec`: 16-byte aligned
template <typename T>
__device__ __forceinline__ uint4 kv4_raw8(const T* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  return make_uint4(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16, h[4] | static_cast<uint32_t>(h[5]) << 16,
                    h[6] | static_cast<uint32_t>(h[7]) << 16);
}
template <typename T>
__device__ __forceinline__ void kv4_floats8(const uint4& raw, float (&x)[8]) {
  const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = kv4_to_float(t[i]);
}
template <typename T>
__device__ __forceinline__ void kv4_load8(const T* p, bool vec, float (&x)[8]) {
  kv4_floats8<T>(kv4_raw8(p, vec), x);
}
template <typename T>
__device__ __forceinline__ void kv4_store8(T* p, bool vec, const float (&x)[8]) {
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = kv4_from_float<T>(x[i]);
  if (vec) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(t);
  else
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = t[i];
}

// a * c - b * s in twice the working precision, rounded to fp32 once (products and the difference carry their rounding
// errors along): the codes of a rotated key then do not depend on how the rotation was evaluated.
__device__ __forceinline__ float kv4_turn(float a, float c, float b, float s) {
  const float p = __fmul_rn(a, c), pe = __fmaf_rn(a, c, -p);
  const float q = __fmul_rn(b, s), qe = __fmaf_rn(b, s, -q);
  const float d = __fsub_rn(p, q), z = __fsub_rn(d, p);
  const float de = __fsub_rn(__fsub_rn(p, __fsub_rn(d, z)), __fadd_rn(q, z));
  return __fadd_rn(d, __fadd_rn(de, __fsub_rn(pe, qe)));
}

}  // namespace crl
