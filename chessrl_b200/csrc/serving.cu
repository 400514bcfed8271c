// Entry points of the decoder-serving operators: the 4-bit key/value cache and next-token logits. See
// include/chessrl_b200.h for their contracts.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "../../include/chessrl_b200.h"
#include "kv4_append.cuh"
#include "kv4_attention.cuh"
#include "kv4_prompt.cuh"
#include "kv4_rows.cuh"
#include "logits.cuh"

using namespace crl;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// rows at multiples of these strides (in 16-bit elements) all start on a 16-byte boundary
bool rows_aligned(const void* p, int64_t tok, int64_t head) { return aligned16(p) && tok % 8 == 0 && head % 8 == 0; }

int check_cache(const crl_kv4_cache& c) {
  if (c.pages == nullptr || c.block_table == nullptr || c.num_pages <= 0 || c.kv_heads <= 0 || c.seqs < 0 || c.table_width <= 0 ||
      c.table_stride < c.table_width)
    return CRL_ERR_INVALID;
  if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128) return CRL_ERR_SHAPE;
  if (c.page_size <= 0 || c.page_size % kKv4Block != 0 || !aligned16(c.pages)) return CRL_ERR_SHAPE;
  // cache indices are 32-bit, with room for the last tile's end
  if (static_cast<int64_t>(c.table_width) * c.page_size > INT32_MAX - 1024 || c.num_pages > INT32_MAX ||
      c.num_pages > (int64_t{0xfffffffe} * kKv4Block) / (static_cast<int64_t>(c.kv_heads) * c.page_size))
    return CRL_ERR_SHAPE;
  return CRL_OK;
}
Kv4Table table_of(const crl_kv4_cache& c) {
  Kv4Table t;
  t.table = c.block_table;
  t.stride = c.table_stride;
  t.width = c.table_width;
  t.blocks = c.page_size / kKv4Block;
  t.shift = -1;
  for (int b = 0; b < 30; ++b)
    if (t.blocks == 1 << b) t.shift = b;
  t.num_pages = static_cast<uint32_t>(c.num_pages);
  t.page_blocks = static_cast<uint32_t>(c.kv_heads) * t.blocks;
  return t;
}
bool known16(int dtype) { return dtype == CRL_OUT_F16 || dtype == CRL_OUT_BF16; }

template <template <typename, int> class F, typename... A>
int by_type(int dtype, int hd, A&&... a) {
  if (dtype == CRL_OUT_F16)
    return hd == 32 ? F<__half, 32>::run(a...) : hd == 64 ? F<__half, 64>::run(a...) : F<__half, 128>::run(a...);
  return hd == 32 ? F<__nv_bfloat16, 32>::run(a...) : hd == 64 ? F<__nv_bfloat16, 64>::run(a...) : F<__nv_bfloat16, 128>::run(a...);
}

// SMs of the current device, asked once per device
int current_sms(int* sms) {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return CRL_ERR_CUDA;
  int n = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return CRL_ERR_CUDA;
    if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  }
  *sms = n;
  return CRL_OK;
}

// Tokens of a CTA and the grid for `rows` rows per token: few tokens get a CTA each, many share the look-up of theirs.
template <typename P>
int by_tokens(P* p, int64_t rows, unsigned* grid) {
  int sms = 0;
  if (const int rc = current_sms(&sms)) return rc;
  if (rows > 16384) return CRL_ERR_SHAPE;      // over_rows divides exactly up to here
  p->per_cta = static_cast<int32_t>(std::min<int64_t>(kKv4CtaTokens, std::max<int64_t>(1, p->tokens / (8 * sms))));
  p->over_rows = static_cast<uint32_t>(((uint64_t{1} << 32) + rows - 1) / rows);
  const int64_t blocks = (p->tokens + p->per_cta - 1) / p->per_cta;
  if (blocks > INT32_MAX) return CRL_ERR_SHAPE;
  *grid = static_cast<unsigned>(blocks);
  return CRL_OK;
}

template <typename T, int HD>
struct Append {
  static int run(Kv4AppendParams p, cudaStream_t s) {
    unsigned grid;
    if (const int rc = by_tokens(&p, static_cast<int64_t>(p.heads) + 2 * p.kv_heads, &grid)) return rc;
    kv4_append_kernel<T, HD><<<grid, kKv4Threads, 0, s>>>(p);
    return cudaGetLastError() == cudaSuccess ? CRL_OK : CRL_ERR_CUDA;
  }
};
template <typename T, int HD>
struct Read {
  static int run(Kv4ReadParams p, cudaStream_t s) {
    unsigned grid;
    if (const int rc = by_tokens(&p, int64_t{2} * p.kv_heads, &grid)) return rc;
    kv4_read_kernel<T, HD><<<grid, kKv4Threads, 0, s>>>(p);
    return cudaGetLastError() == cudaSuccess ? CRL_OK : CRL_ERR_CUDA;
  }
};

constexpr int kMaxSplits = 16;      // the largest cluster that the hardware takes (more than 8 are allowed kernel by kernel)

// What is known of an attention kernel on a device: how many clusters of 1 .. kMaxSplits CTAs are resident at once.
struct KernelFacts {
  std::atomic<int> clusters[kMaxSplits + 1];
};
template <typename K>
int facts_of(K* kernel, KernelFacts* all, int bytes, int threads, KernelFacts** out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return CRL_ERR_CUDA;
  KernelFacts& f = all[dev];
  if (f.clusters[0].load(std::memory_order_acquire) == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return CRL_ERR_CUDA;
    for (int n = 1; n <= kMaxSplits; ++n) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(n);
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = bytes;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = n;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      int many = 0;
      if (cudaOccupancyMaxActiveClusters(&many, kernel, &cfg) != cudaSuccess) return CRL_ERR_CUDA;
      f.clusters[n].store(many, std::memory_order_relaxed);      // 0: no GPC has room for as many
    }
    f.clusters[0].store(1, std::memory_order_release);
  }
  *out = &f;
  return CRL_OK;
}

// The number of CTAs that share the keys of a (row tile, key head, sequence): the one that makes the waves of clusters
// times the key tiles of the longest warp least (`fixed` tiles' worth of time goes to a CTA's start and join), for
// sequences as long as the table allows.
int split_keys(const KernelFacts& f, int64_t units, int64_t max_keys, int keys_at_once, int fixed, int64_t* total = nullptr) {
  int best = 1;
  int64_t least = INT64_MAX;
  for (int n = 1; n <= kMaxSplits; ++n) {
    const int64_t tiles = (max_keys + static_cast<int64_t>(n) * keys_at_once - 1) / (static_cast<int64_t>(n) * keys_at_once);
    const int64_t active = f.clusters[n].load(std::memory_order_relaxed);
    if (active == 0) break;
    const int64_t waves = (units + active - 1) / active;
    const int64_t cost = waves * (tiles + fixed + (n > 1 ? 1 : 0));
    if (cost < least) {
      least = cost;
      best = n;
    }
    if (tiles <= 1) break;
  }
  if (total != nullptr) *total = least;
  return best;
}

// One launch of an attention kernel: a cluster along the keys per (row tile, key head, sequence).
template <typename K>
int attend_launch(K* kernel, KernelFacts* all, int bytes, int threads, int tile_rows, int keys_at_once, Kv4AttentionParams p,
                  int64_t max_keys, cudaStream_t s) {
  KernelFacts* f = nullptr;
  if (const int rc = facts_of(kernel, all, bytes, threads, &f)) return rc;
  p.row_tiles = (p.max_tokens * p.group + tile_rows - 1) / tile_rows;
  const int64_t units = static_cast<int64_t>(p.seqs) * p.kv_heads * p.row_tiles;
  const int splits = split_keys(*f, units, max_keys, keys_at_once, 2);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(splits * p.row_tiles, p.kv_heads, p.seqs);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<const Kv4AttentionParams>(p)) == cudaSuccess ? CRL_OK : CRL_ERR_CUDA;
}
template <typename T, int HD, int COLS, int WARPS>
int attend_few(Kv4AttentionParams p, int64_t max_keys, cudaStream_t s) {
  using Shape = Kv4AttnShape<HD, WARPS>;
  static KernelFacts facts[64];
  p.whole_tiles = p.table.blocks % Shape::kTile == 0;
  return attend_launch(kv4_attention_kernel<T, HD, COLS, WARPS>, facts, Shape::kBytes, WARPS * 32, Shape::kRows, WARPS * Shape::kTile * 16,
                       p, max_keys, s);
}
template <typename T, int HD, int WARPS>
int attend_few_by_rows(const Kv4AttentionParams& p, int64_t rows, int64_t max_keys, cudaStream_t s) {
  if (rows * (HD / 32) <= 4) return attend_few<T, HD, 1, WARPS>(p, max_keys, s);
  if (HD == 32 || rows * (HD / 32) <= 8) return attend_few<T, HD, 2, WARPS>(p, max_keys, s);
  if constexpr (HD > 32) return attend_few<T, HD, 0, WARPS>(p, max_keys, s);
}
template <typename T, int HD, int RW>
KernelFacts rows_facts[64];
// What the two kernels for many rows would take for sequences as long as the table allows, in hundreds of cycles: a CTA of
// the first takes about 7000 per tile of 64 keys, one of the second 4400 per tile of 112 and 12000 to start and to end
// (both measured at 4096-token prompts, head_dim 128). The first splits the keys over a cluster, the second does not.
// First / second, measured: 32 new tokens at 60000, 12 heads on 1 of 64: 132 / 1176 us; 128-token prompts of 16 sequences,
// 12 heads of 64: 14 / 26 us; 200 new tokens at 5000 in 4 sequences, 32 heads on 8 of 128: 471 / 140 us; a 2048-token
// prompt of those heads: 375 / 84 us.
template <typename T, int HD>
bool prompt_is_faster(const Kv4AttentionParams& p, int64_t rows, int sms, int64_t max_keys) {
  using Shape = Kv4RowsShape<HD, 4, 1>;
  KernelFacts* f = nullptr;
  if (facts_of(kv4_rows_kernel<T, HD, 4, 1>, rows_facts<T, HD, 4>, Shape::kBytes, 128, &f) != CRL_OK) return false;
  const int64_t pairs = static_cast<int64_t>(p.seqs) * p.kv_heads, ctas = pairs * ((rows + 255) / 256);
  int64_t waves_tiles = 0;
  split_keys(*f, pairs * ((rows + 63) / 64), max_keys, 64, 2, &waves_tiles);
  return (ctas + sms - 1) / sms * ((max_keys + 111) / 112 * 44 + 120) < waves_tiles * 70;
}
template <typename T, int HD, int RW>
int attend_rows(Kv4AttentionParams p, int64_t max_keys, cudaStream_t s) {
  using Shape = Kv4RowsShape<HD, RW, 4 / RW>;
  p.whole_tiles = p.table.blocks % 4 == 0;
  return attend_launch(kv4_rows_kernel<T, HD, RW, 4 / RW>, rows_facts<T, HD, RW>, Shape::kBytes, 128, 16 * RW, 4 / RW * 64, p, max_keys, s);
}
template <typename T, int HD>
int attend_prompt(Kv4AttentionParams p, cudaStream_t s) {
  using Shape = Kv4PromptShape<HD>;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return CRL_ERR_CUDA;
  const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
  if ((ready.load(std::memory_order_relaxed) & bit) == 0) {      // once per device
    if (cudaFuncSetAttribute(kv4_prompt_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kBytes) != cudaSuccess)
      return CRL_ERR_CUDA;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  p.row_tiles = (p.max_tokens * p.group + 255) / 256;
  kv4_prompt_kernel<T, HD><<<dim3(p.row_tiles, p.kv_heads, p.seqs), Shape::kThreads, Shape::kBytes, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? CRL_OK : CRL_ERR_CUDA;
}
template <typename T, int HD>
struct Attend {
  static int run(const Kv4AttentionParams& p, int sms, int64_t max_keys, cudaStream_t s) {
    const int64_t rows = static_cast<int64_t>(p.max_tokens) * p.group;
    if (rows <= 8) {
      // two warps per CTA where there are enough (sequence, key head) pairs to fill the GPU, or so few keys that a CTA of
      // eight would idle (256 sequences of up to 1024 tokens, 12 heads of 64: 53 us with two, 56 with four, 70 with
      // eight; 4 sequences of 131k tokens, 8 heads of 128: 270 / 204 / 177 us)
      const int64_t units = static_cast<int64_t>(p.seqs) * p.kv_heads;
      if (units >= 2 * sms || max_keys <= 512) return attend_few_by_rows<T, HD, 2>(p, rows, max_keys, s);
      return attend_few_by_rows<T, HD, 8>(p, rows, max_keys, s);
    }
    if (rows <= 16) return attend_rows<T, HD, 1>(p, max_keys, s);
    if (rows <= 32) return attend_rows<T, HD, 2>(p, max_keys, s);
    if (rows > 64 && prompt_is_faster<T, HD>(p, rows, sms, max_keys)) return attend_prompt<T, HD>(p, s);
    return attend_rows<T, HD, 4>(p, max_keys, s);
  }
};

template <typename T>
int logits_rows(const LogitsParams& p, cudaStream_t s) {
  const int64_t grid = p.rows * p.tiles;
  if (grid > INT32_MAX) return CRL_ERR_SHAPE;
  adjust_logits_kernel<T><<<static_cast<unsigned>(grid), kLogitsThreads, (p.tile + 8) * 4, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? CRL_OK : CRL_ERR_CUDA;
}

}  // namespace

extern "C" {

size_t crl_kv4_page_bytes(int32_t page_size, int32_t kv_heads, int32_t head_dim) {
  if (page_size <= 0 || page_size % kKv4Block != 0 || kv_heads <= 0 || (head_dim != 32 && head_dim != 64 && head_dim != 128)) return 0;
  return static_cast<size_t>(kv_heads) * (page_size / kKv4Block) * kv4_block_bytes(head_dim);
}

int crl_kv4_append(const crl_kv4_append_args* a) {
  if (a == nullptr) return CRL_ERR_INVALID;
  if (const int rc = check_cache(a->cache)) return rc;
  const crl_kv4_cache& c = a->cache;
  if (a->k == nullptr || a->v == nullptr || a->starts == nullptr || a->tokens < 0 || a->heads < 0 || !known16(a->dtype)) return CRL_ERR_INVALID;
  if (a->heads > 0 && (a->q == nullptr || a->q_out == nullptr || a->q == a->q_out)) return CRL_ERR_INVALID;
  if (a->rope != nullptr && (a->rope_dim <= 0 || a->rope_dim % 2 != 0 || a->rope_dim > c.head_dim || a->rope_positions <= 0))
    return CRL_ERR_SHAPE;
  if (a->tokens == 0 || c.seqs == 0) return CRL_OK;
  Kv4AppendParams p{};
  p.pages = static_cast<uint8_t*>(c.pages);
  p.table = table_of(c);
  p.starts = a->starts; p.cu = a->cu_tokens; p.seqs = c.seqs; p.kv_heads = c.kv_heads; p.heads = a->heads; p.tokens = a->tokens;
  p.q = a->q; p.k = a->k; p.v = a->v; p.q_out = a->q_out;
  p.q_tok = a->q_token_stride; p.q_head = a->q_head_stride; p.k_tok = a->k_token_stride; p.k_head = a->k_head_stride;
  p.v_tok = a->v_token_stride; p.v_head = a->v_head_stride; p.o_tok = a->out_token_stride; p.o_head = a->out_head_stride;
  p.rope = reinterpret_cast<const float2*>(a->rope); p.rope_positions = a->rope_positions; p.rot = a->rope_dim;
  p.interleaved = a->rope_interleaved;
  p.vec_q = rows_aligned(a->q, p.q_tok, p.q_head); p.vec_k = rows_aligned(a->k, p.k_tok, p.k_head);
  p.vec_v = rows_aligned(a->v, p.v_tok, p.v_head); p.vec_o = rows_aligned(a->q_out, p.o_tok, p.o_head);
  p.status = a->device_status;
  return by_type<Append>(a->dtype, c.head_dim, p, static_cast<cudaStream_t>(a->stream));
}

int crl_kv4_read(const crl_kv4_read_args* a) {
  if (a == nullptr) return CRL_ERR_INVALID;
  if (const int rc = check_cache(a->cache)) return rc;
  const crl_kv4_cache& c = a->cache;
  if (a->k == nullptr || a->v == nullptr || a->starts == nullptr || a->tokens < 0 || !known16(a->dtype)) return CRL_ERR_INVALID;
  if (a->tokens == 0 || c.seqs == 0) return CRL_OK;
  Kv4ReadParams p{};
  p.pages = static_cast<const uint8_t*>(c.pages);
  p.table = table_of(c);
  p.starts = a->starts; p.cu = a->cu_tokens; p.seqs = c.seqs; p.kv_heads = c.kv_heads; p.tokens = a->tokens;
  p.k = a->k; p.v = a->v;
  p.k_tok = a->k_token_stride; p.k_head = a->k_head_stride; p.v_tok = a->v_token_stride; p.v_head = a->v_head_stride;
  p.vec_k = rows_aligned(a->k, p.k_tok, p.k_head); p.vec_v = rows_aligned(a->v, p.v_tok, p.v_head);
  p.status = a->device_status;
  return by_type<Read>(a->dtype, c.head_dim, p, static_cast<cudaStream_t>(a->stream));
}

int crl_kv4_attention(const crl_kv4_attention_args* a) {
  if (a == nullptr) return CRL_ERR_INVALID;
  if (const int rc = check_cache(a->cache)) return rc;
  const crl_kv4_cache& c = a->cache;
  if (a->q == nullptr || a->out == nullptr || a->lengths == nullptr || a->tokens < 0 || !known16(a->dtype) || a->heads <= 0 ||
      a->max_tokens < 0)
    return CRL_ERR_INVALID;
  if (a->heads % c.kv_heads != 0 || c.seqs > 65535 || c.kv_heads > 65535) return CRL_ERR_SHAPE;
  if (a->tokens == 0 || c.seqs == 0 || a->max_tokens == 0) return CRL_OK;
  int sms = 0;
  if (const int rc = current_sms(&sms)) return rc;
  Kv4AttentionParams p{};
  p.pages = static_cast<const uint8_t*>(c.pages);
  p.table = table_of(c);
  p.lengths = a->lengths; p.cu = a->cu_tokens; p.seqs = c.seqs; p.kv_heads = c.kv_heads; p.group = a->heads / c.kv_heads;
  p.max_tokens = a->cu_tokens != nullptr ? static_cast<int32_t>(std::min<int64_t>(a->max_tokens, a->tokens)) : 1;
  const int64_t rows = static_cast<int64_t>(p.max_tokens) * p.group + 256;      // a tile's last row
  if (rows > (int64_t{1} << 27)) return CRL_ERR_SHAPE;      // leaves the grid room for splits
  p.by_group.d = static_cast<uint32_t>(p.group);
  p.by_group.mul = p.group > 1 && rows * p.group < (int64_t{1} << 32) ? static_cast<uint32_t>(((uint64_t{1} << 32) + p.group - 1) / p.group) : 0;
  p.tokens = a->tokens;
  p.q = a->q; p.out = a->out;
  p.q_tok = a->q_token_stride; p.q_head = a->q_head_stride; p.o_tok = a->out_token_stride; p.o_head = a->out_head_stride;
  p.vec_q = rows_aligned(a->q, p.q_tok, p.q_head);
  p.pair_o = (reinterpret_cast<uintptr_t>(a->out) & 3) == 0 && p.o_tok % 2 == 0 && p.o_head % 2 == 0;
  p.vec_o = rows_aligned(a->out, p.o_tok, p.o_head);
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.status = a->device_status;
  return by_type<Attend>(a->dtype, c.head_dim, p, sms, static_cast<int64_t>(c.table_width) * c.page_size,
                         static_cast<cudaStream_t>(a->stream));
}

int crl_adjust_logits(const crl_logits_args* a) {
  if (a == nullptr || a->logits == nullptr || a->out == nullptr) return CRL_ERR_INVALID;
  if (a->dtype != CRL_OUT_F32 && !known16(a->dtype)) return CRL_ERR_INVALID;
  if (a->rows < 0 || a->vocab <= 0 || a->in_stride < a->vocab || a->out_stride < a->vocab || a->history_len < 0 || a->biases < 0)
    return CRL_ERR_INVALID;
  if ((a->history_len > 0 && (a->history == nullptr || a->history_stride < a->history_len)) ||
      (a->biases > 0 && (a->bias_ids == nullptr || a->bias_values == nullptr || a->bias_stride < a->biases || a->value_stride < a->biases)))
    return CRL_ERR_INVALID;
  if (a->history_len > kLogitsMaxHistory || a->biases > kLogitsMaxBiases || a->vocab > INT32_MAX - 65536) return CRL_ERR_SHAPE;
  if (a->mask != nullptr && (a->mask_count <= 0 || a->mask_stride < (static_cast<int64_t>(a->vocab) + 7) / 8)) return CRL_ERR_INVALID;
  if (a->mask != nullptr && a->mask_rows == nullptr && a->mask_count < a->rows) return CRL_ERR_INVALID;
  if (a->rows == 0) return CRL_OK;
  const int size = a->dtype == CRL_OUT_F32 ? 4 : 2;
  LogitsParams p{};
  p.in = a->logits; p.out = a->out; p.in_stride = a->in_stride; p.out_stride = a->out_stride; p.rows = a->rows; p.vocab = a->vocab;
  p.history = a->history_len > 0 ? a->history : nullptr; p.history_stride = a->history_stride; p.history_len = a->history_len;
  p.repetition = a->repetition; p.frequency = a->frequency; p.presence = a->presence;
  p.bias_ids = a->bias_ids; p.bias_values = a->bias_values; p.bias_stride = a->bias_stride; p.value_stride = a->value_stride;
  p.biases = a->biases;
  p.mask = a->mask; p.mask_stride = a->mask_stride; p.mask_count = static_cast<int32_t>(std::min<int64_t>(a->mask_count, INT32_MAX));
  p.mask_rows = a->mask_rows; p.masked_value = a->masked_value; p.status = a->device_status;
  const intptr_t ip = reinterpret_cast<intptr_t>(a->logits), op = reinterpret_cast<intptr_t>(a->out);
  p.same_phase = (ip - op) % 16 == 0 && ((a->in_stride - a->out_stride) * size) % 16 == 0 && ip % size == 0;
  p.tile = 4096;
  p.tiles = (p.vocab + p.tile - 1) / p.tile;
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  if (a->dtype == CRL_OUT_F32) return logits_rows<float>(p, s);
  if (a->dtype == CRL_OUT_F16) return logits_rows<__half>(p, s);
  return logits_rows<__nv_bfloat16>(p, s);
}

}  // extern "C"
