// torch tensors -> the serving entry points of the C ABI, for chessrl_b200/serving.py. A single-token call keeps the GPU
// busy for a few microseconds; looking at a dozen tensors from Python took longer than that (11 - 23 us a call), here it
// takes about one. Every rule about tensors is checked here: the C functions get raw pointers and see none of it. Their
// addresses come from the library that the Python side has loaded (bind), so nothing is linked against it.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <string>

#include "../../include/chessrl_b200.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;

decltype(&crl_kv4_append) append_fn = nullptr;
decltype(&crl_kv4_read) read_fn = nullptr;
decltype(&crl_kv4_attention) attention_fn = nullptr;
decltype(&crl_adjust_logits) logits_fn = nullptr;

[[noreturn]] void refuse(const std::string& why) { throw py::value_error(why); }
std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
const char* dtype_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "float32";
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    case at::kInt: return "int32";
    case at::kByte: return "uint8";
    default: return "another dtype";
  }
}
bool known(at::ScalarType t, int32_t* out) {
  if (t == at::kFloat) *out = CRL_OUT_F32;
  else if (t == at::kHalf) *out = CRL_OUT_F16;
  else if (t == at::kBFloat16) *out = CRL_OUT_BF16;
  else return false;
  return true;
}

// on GPU `dev`, of this many dimensions
void check_place(const char* name, const Tensor& t, int dev, int64_t dim) {
  if (!t.is_cuda() || t.get_device() != dev) refuse(std::string(name) + " must live on cuda:" + std::to_string(dev) + ", got " + t.device().str());
  if (t.dim() != dim) refuse(std::string(name) + " must have " + std::to_string(dim) + " dimensions, got shape " + shape_of(t));
}
void check_type(const char* name, const Tensor& t, at::ScalarType type) {
  if (t.scalar_type() != type) refuse(std::string(name) + " must have dtype " + dtype_name(type) + ", got " + dtype_name(t.scalar_type()));
}
void check_half(const char* name, const Tensor& t) {
  if (t.scalar_type() != at::kHalf && t.scalar_type() != at::kBFloat16)
    refuse(std::string(name) + " must have dtype float16 or bfloat16, got " + dtype_name(t.scalar_type()));
}
template <typename V>
V* vector_of(const char* name, const Tensor& t, int dev, at::ScalarType type, int64_t count) {
  check_place(name, t, dev, 1);
  check_type(name, t, type);
  if (t.size(0) != count || (count > 1 && t.stride(0) != 1))
    refuse(std::string(name) + " must hold " + std::to_string(count) + " contiguous " + dtype_name(type) + ", got shape " + shape_of(t));
  return static_cast<V*>(t.data_ptr());
}
int* status_of(const Maybe& t, int dev) {
  if (!t) return nullptr;
  check_place("status", *t, dev, 1);
  check_type("status", *t, at::kInt);
  if (t->size(0) < 1) refuse("status must hold an int32");
  return static_cast<int*>(t->data_ptr());
}
// [tokens, heads, dim] with contiguous rows; heads < 0: any
void check_rows(const char* name, const Tensor& t, int dev, int64_t heads, int64_t dim) {
  check_place(name, t, dev, 3);
  if (t.size(2) != dim || (heads >= 0 && t.size(1) != heads))
    refuse(std::string(name) + " must be [tokens, " + (heads < 0 ? "heads" : std::to_string(heads)) + ", " + std::to_string(dim) + "], got shape " + shape_of(t));
  if (t.stride(2) != 1) refuse(std::string("the last dimension of ") + name + " must be contiguous");
}
crl_kv4_cache cache_of(const Tensor& pages, const Tensor& table, int* dev) {
  if (!pages.is_cuda()) refuse("pages must be a tensor on the GPU (see kv4_pages)");
  *dev = pages.get_device();
  check_place("pages", pages, *dev, 4);
  check_type("pages", pages, at::kByte);
  const int64_t n = pages.size(0), heads = pages.size(1), blocks = pages.size(2), width = pages.size(3);
  if ((width != 640 && width != 1280 && width != 2560) || !pages.is_contiguous() || n * heads * blocks == 0 || heads > INT32_MAX || blocks > (1 << 26))
    refuse("pages must be contiguous [num_pages, kv_heads, page_size / 16, 20 * head_dim] with head_dim 32, 64 or 128");
  check_place("block_table", table, *dev, 2);
  check_type("block_table", table, at::kInt);
  const int64_t seqs = table.size(0), wide = table.size(1), stride = seqs > 1 ? table.stride(0) : wide;
  if (wide == 0 || (wide > 1 && table.stride(1) != 1) || stride < wide || wide > INT32_MAX || seqs > INT32_MAX)
    refuse("block_table must be [seqs, pages] with contiguous rows that do not overlap");
  crl_kv4_cache c;
  c.pages = pages.data_ptr();
  c.num_pages = n;
  c.page_size = static_cast<int32_t>(16 * blocks);
  c.kv_heads = static_cast<int32_t>(heads);
  c.head_dim = static_cast<int32_t>(width / 20);
  c.seqs = static_cast<int32_t>(seqs);
  c.block_table = static_cast<const int32_t*>(table.data_ptr());
  c.table_stride = stride;
  c.table_width = static_cast<int32_t>(wide);
  return c;
}
const int32_t* runs_of(const Maybe& cu, int dev, int64_t tokens, int64_t seqs) {
  if (cu) return vector_of<int32_t>("cu_tokens", *cu, dev, at::kInt, seqs + 1);
  if (tokens != seqs) refuse("without cu_tokens there is one token per sequence");
  return nullptr;
}
Tensor new_rows(const Tensor& like, int64_t a, int64_t b, int64_t c, at::ScalarType type) {
  return at::empty({a, b, c}, like.options().dtype(type));
}

template <typename F, typename A>
void call(const char* name, F* fn, A& args, int dev) {
  if (fn == nullptr) throw std::runtime_error("the serving functions are not bound to a library");
  args.stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
  int rc;
  {
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    rc = fn(&args);
  }
  if (rc != 0) {
    py::object error = py::module_::import("chessrl_b200._lib").attr("CrlError");
    py::object what = error(rc, name);
    PyErr_SetObject(error.ptr(), what.ptr());
    throw py::error_already_set();
  }
}

void bind(uintptr_t append, uintptr_t read, uintptr_t attention, uintptr_t logits) {
  append_fn = reinterpret_cast<decltype(append_fn)>(append);
  read_fn = reinterpret_cast<decltype(read_fn)>(read);
  attention_fn = reinterpret_cast<decltype(attention_fn)>(attention);
  logits_fn = reinterpret_cast<decltype(logits_fn)>(logits);
}

Maybe kv4_append(const Tensor& pages, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& starts, const Maybe& cu, const Maybe& q,
                 const Maybe& rope, bool interleaved, const Maybe& status) {
  int dev = 0;
  crl_kv4_append_args a{};
  a.cache = cache_of(pages, table, &dev);
  const int64_t hd = a.cache.head_dim, tokens = k.dim() == 3 ? k.size(0) : 0;
  check_rows("k", k, dev, a.cache.kv_heads, hd);
  check_half("k", k);
  check_rows("v", v, dev, a.cache.kv_heads, hd);
  check_type("v", v, k.scalar_type());
  if (q) {
    check_rows("q", *q, dev, -1, hd);
    check_type("q", *q, k.scalar_type());
  }
  if (v.size(0) != tokens || (q && q->size(0) != tokens)) refuse("q, k and v must have the same number of tokens");
  known(k.scalar_type(), &a.dtype);
  a.tokens = tokens;
  a.k = k.data_ptr(); a.k_token_stride = k.stride(0); a.k_head_stride = k.stride(1);
  a.v = v.data_ptr(); a.v_token_stride = v.stride(0); a.v_head_stride = v.stride(1);
  a.starts = vector_of<int32_t>("starts", starts, dev, at::kInt, a.cache.seqs);
  a.cu_tokens = runs_of(cu, dev, tokens, a.cache.seqs);
  Maybe out = q;
  if (rope) {
    check_place("rope", *rope, dev, 3);
    check_type("rope", *rope, at::kFloat);
    if (rope->size(2) != 2 || !rope->is_contiguous() || rope->size(1) < 1 || 2 * rope->size(1) > hd || rope->size(0) == 0)
      refuse("rope must be a contiguous [positions, rot_dim / 2, 2] table with rot_dim <= head_dim (see rope_table)");
    a.rope = static_cast<const float*>(rope->data_ptr());
    a.rope_positions = rope->size(0);
    a.rope_dim = static_cast<int32_t>(2 * rope->size(1));
    a.rope_interleaved = interleaved;
    if (q && q->size(1) > 0) {
      const int64_t heads = q->size(1);
      out = new_rows(*q, tokens, heads, hd, q->scalar_type());
      a.q = q->data_ptr(); a.q_token_stride = q->stride(0); a.q_head_stride = q->stride(1);
      a.q_out = out->data_ptr(); a.out_token_stride = heads * hd; a.out_head_stride = hd;
      a.heads = static_cast<int32_t>(heads);
    }
  }
  a.device_status = status_of(status, dev);
  if (tokens > 0) call("crl_kv4_append", append_fn, a, dev);
  return out;
}

std::pair<Tensor, Tensor> kv4_read(const Tensor& pages, const Tensor& table, const Tensor& starts, int64_t tokens, const Maybe& cu, bool bf16,
                                   const Maybe& status) {
  int dev = 0;
  crl_kv4_read_args a{};
  a.cache = cache_of(pages, table, &dev);
  if (tokens < 0) refuse("tokens must not be negative");
  const int64_t heads = a.cache.kv_heads, hd = a.cache.head_dim;
  a.dtype = bf16 ? CRL_OUT_BF16 : CRL_OUT_F16;
  a.tokens = tokens;
  a.starts = vector_of<int32_t>("starts", starts, dev, at::kInt, a.cache.seqs);
  a.cu_tokens = runs_of(cu, dev, tokens, a.cache.seqs);
  a.device_status = status_of(status, dev);
  Tensor k = new_rows(pages, tokens, heads, hd, bf16 ? at::kBFloat16 : at::kHalf), v = new_rows(pages, tokens, heads, hd, bf16 ? at::kBFloat16 : at::kHalf);
  a.k = k.data_ptr(); a.v = v.data_ptr();
  a.k_token_stride = a.v_token_stride = heads * hd;
  a.k_head_stride = a.v_head_stride = hd;
  if (tokens > 0) {
    if (a.cache.seqs == 0) {
      k.zero_();
      v.zero_();
    } else {
      call("crl_kv4_read", read_fn, a, dev);
    }
  }
  return {k, v};
}

Tensor kv4_attention(const Tensor& pages, const Tensor& q, const Tensor& table, const Tensor& lengths, const Maybe& cu, int64_t max_tokens,
                     std::optional<double> scale, const Maybe& into, const Maybe& status) {
  int dev = 0;
  crl_kv4_attention_args a{};
  a.cache = cache_of(pages, table, &dev);
  const int64_t hd = a.cache.head_dim;
  check_rows("q", q, dev, -1, hd);
  check_half("q", q);
  const int64_t tokens = q.size(0), heads = q.size(1);
  if (heads == 0 || heads % a.cache.kv_heads != 0)
    refuse("query heads must be a multiple of the cache's " + std::to_string(a.cache.kv_heads) + ", got " + std::to_string(heads));
  a.lengths = vector_of<int32_t>("lengths", lengths, dev, at::kInt, a.cache.seqs);
  a.cu_tokens = runs_of(cu, dev, tokens, a.cache.seqs);
  if (cu && max_tokens < 1) refuse("max_tokens must be at least 1");
  a.max_tokens = cu ? static_cast<int32_t>(std::min<int64_t>({max_tokens, tokens, INT32_MAX})) : 1;
  a.device_status = status_of(status, dev);
  Tensor out;
  if (into) {
    check_rows("out", *into, dev, heads, hd);
    check_type("out", *into, q.scalar_type());
    if (into->size(0) != tokens) refuse("out must have q's shape");
    const int64_t st = into->stride(0), sh = into->stride(1);
    const bool tokens_outside = st >= (heads - 1) * sh + hd && (heads == 1 || sh >= hd), heads_outside = sh >= (tokens - 1) * st + hd && (tokens == 1 || st >= hd);
    if (tokens > 1 ? !tokens_outside && !(heads > 1 && heads_outside) : heads > 1 && sh < hd) refuse("the rows of out must not overlap");
    out = *into;
  } else {
    out = new_rows(q, tokens, heads, hd, q.scalar_type());
  }
  known(q.scalar_type(), &a.dtype);
  a.heads = static_cast<int32_t>(heads);
  a.tokens = tokens;
  a.q = q.data_ptr(); a.q_token_stride = q.stride(0); a.q_head_stride = q.stride(1);
  a.out = out.data_ptr(); a.out_token_stride = out.stride(0); a.out_head_stride = out.stride(1);
  a.scale = scale ? static_cast<float>(*scale) : static_cast<float>(1.0 / std::sqrt(static_cast<double>(hd)));
  if (tokens > 0) call("crl_kv4_attention", attention_fn, a, dev);
  return out;
}

// [count, wide] with contiguous rows that do not overlap; count < 0: any
int64_t pitch_of(const char* name, const Tensor& t, int dev, int64_t count) {
  check_place(name, t, dev, 2);
  if (count >= 0 && t.size(0) != count) refuse(std::string(name) + " must have " + std::to_string(count) + " rows, got shape " + shape_of(t));
  const int64_t wide = t.size(1), stride = t.size(0) > 1 ? t.stride(0) : wide;
  if ((wide > 1 && t.stride(1) != 1) || stride < wide) refuse(std::string("the rows of ") + name + " must be contiguous and not overlap");
  return stride;
}

Tensor adjust_logits(const Tensor& logits, const Maybe& history, const Maybe& repetition, const Maybe& frequency, const Maybe& presence,
                     const Maybe& bias_ids, const Maybe& bias_values, const Maybe& mask, const Maybe& mask_rows, double masked_value, const Maybe& into,
                     const Maybe& status) {
  if (!logits.is_cuda()) refuse("logits must be a tensor on the GPU");
  const int dev = logits.get_device();
  crl_logits_args a{};
  a.in_stride = pitch_of("logits", logits, dev, -1);
  if (!known(logits.scalar_type(), &a.dtype)) refuse("logits must have dtype float32, float16 or bfloat16");
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  if (vocab == 0 || vocab > INT32_MAX) refuse("logits must have a vocabulary");
  a.rows = rows;
  a.vocab = static_cast<int32_t>(vocab);
  if (history) {
    a.history_stride = pitch_of("history", *history, dev, rows);
    check_type("history", *history, at::kInt);
    if (history->size(1) > INT32_MAX) refuse("history is too long");
    a.history = static_cast<const int32_t*>(history->data_ptr());
    a.history_len = static_cast<int32_t>(history->size(1));
  }
  if (repetition) a.repetition = vector_of<float>("repetition", *repetition, dev, at::kFloat, rows);
  if (frequency) a.frequency = vector_of<float>("frequency", *frequency, dev, at::kFloat, rows);
  if (presence) a.presence = vector_of<float>("presence", *presence, dev, at::kFloat, rows);
  if (bias_ids.has_value() != bias_values.has_value()) refuse("bias_ids and bias_values go together");
  if (bias_ids) {
    a.bias_stride = pitch_of("bias_ids", *bias_ids, dev, rows);
    check_type("bias_ids", *bias_ids, at::kInt);
    a.value_stride = pitch_of("bias_values", *bias_values, dev, rows);
    check_type("bias_values", *bias_values, at::kFloat);
    if (bias_ids->size(1) != bias_values->size(1) || bias_ids->size(1) > INT32_MAX) refuse("bias_ids and bias_values must have the same shape");
    a.bias_ids = static_cast<const int32_t*>(bias_ids->data_ptr());
    a.bias_values = static_cast<const float*>(bias_values->data_ptr());
    a.biases = static_cast<int32_t>(bias_ids->size(1));
  }
  if (mask_rows && !mask) refuse("mask_rows needs a mask");
  if (mask) {
    a.mask_stride = pitch_of("mask", *mask, dev, mask_rows ? -1 : rows);
    check_type("mask", *mask, at::kByte);
    if (mask->size(1) * 8 < vocab)
      refuse("mask rows hold " + std::to_string(mask->size(1)) + " bytes, the vocabulary needs " + std::to_string((vocab + 7) / 8));
    if (mask->size(0) == 0 && rows > 0) refuse("mask must have a row");
    a.mask = static_cast<const uint8_t*>(mask->data_ptr());
    a.mask_count = mask->size(0);
    if (mask_rows) a.mask_rows = vector_of<int32_t>("mask_rows", *mask_rows, dev, at::kInt, rows);
  }
  a.device_status = status_of(status, dev);
  Tensor out;
  if (into) {
    a.out_stride = pitch_of("out", *into, dev, rows);
    check_type("out", *into, logits.scalar_type());
    if (into->size(1) != vocab) refuse("out must have the shape of logits");
    out = *into;
  } else {
    out = at::empty({rows, vocab}, logits.options());
    a.out_stride = vocab;
  }
  a.logits = logits.data_ptr();
  a.out = out.data_ptr();
  a.masked_value = static_cast<float>(masked_value);
  if (rows > 0) call("crl_adjust_logits", logits_fn, a, dev);
  return out;
}

}  // namespace

PYBIND11_MODULE(_serving, m) {
  m.def("bind", &bind);
  m.def("kv4_append", &kv4_append);
  m.def("kv4_read", &kv4_read);
  m.def("kv4_attention", &kv4_attention);
  m.def("adjust_logits", &adjust_logits);
}
