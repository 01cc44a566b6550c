// The paged operators and the batched sampler for torch tensors: checks, outputs, workspaces and
// the current stream on one side, the C ABI (include/qdecode.h) on the other. These calls are
// made per layer or per token; from Python through ctypes the host side of one took 14 us, most
// of it the look-ups of a dozen tensors' attributes.
//
// Python module kernel_optimization_webgpu_b200._torch_calls; runtime.py documents the functions.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/qdecode.h"
#include "overlap.hpp"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace {

void need(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);  // ValueError
}

// Raises QdError(code, message) for a refused or failed C call.
void done(int rc) {
  if (rc == QD_OK) return;
  const char* msg = qd_last_error(nullptr);
  const py::object cls = py::module_::import("kernel_optimization_webgpu_b200._lib").attr("QdError");
  const py::object err = cls(rc, std::string(msg ? msg : ""));
  PyErr_SetObject(cls.ptr(), err.ptr());
  throw py::error_already_set();
}

int code(const Tensor& x, const char* what) {
  const auto t = x.scalar_type();
  if (t == at::kHalf) return QD_KV_F16;
  if (t == at::kFloat) return QD_KV_F32;
  if (t == at::kBFloat16) return QD_KV_BF16;
  throw std::invalid_argument(std::string(what) + " must be float16, bfloat16 or float32");
}

// Contiguous vector of n entries on `dev`; NULL where there is none.
template <typename T>
const T* vec(const Maybe& x, int64_t n, at::ScalarType type, c10::Device dev, const char* what) {
  if (!x) return nullptr;
  if (x->scalar_type() != type || x->dim() != 1 || x->size(0) != n || !x->is_contiguous() || x->device() != dev)
    throw std::invalid_argument(std::string(what) + " must be a contiguous " + c10::toString(type) + " vector of " +
                                std::to_string(n) + " entries on " + dev.str());
  return static_cast<const T*>(x->const_data_ptr());
}

// Row stride of a [rows, ...] tensor whose rows are `width` contiguous elements.
int64_t row_stride(const Tensor& x, int64_t width, const char* what) {
  int64_t inner = 1;
  bool ok = x.dim() >= 1;
  for (int64_t i = x.dim() - 1; i > 0; --i) {
    ok = ok && (x.size(i) == 1 || x.stride(i) == inner);
    inner *= x.size(i);
  }
  if (!ok || inner != width)
    throw std::invalid_argument(std::string(what) + " must have contiguous rows of " + std::to_string(width) + " elements");
  return x.size(0) > 1 ? x.stride(0) : width;
}

// The rows of a [rows, ...] tensor, `stride` elements apart (padding rows of a tensor are memory too).
qd::Rows rows_of(const Tensor& x, int64_t width, int64_t stride) {
  const int64_t size = x.element_size();
  return {x.const_data_ptr(), x.size(0), width * size, stride * size};
}

// As the C ABI takes it, where 0 stands for the default: a scale that f32 cannot hold must not become that.
float to_scale(double v) {
  need(v == 0.0 || (float)v != 0.0f, "scale is below what float32 holds");
  return (float)v;
}

int to_int(int64_t v, const char* what) {
  need(v >= INT32_MIN && v <= INT32_MAX, what);
  return (int)v;
}

qd_paged_kv paged(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens, const Maybe& status,
                  c10::Device dev) {
  need(dev.is_cuda(), "tensors must be on a CUDA device");
  need(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && k.is_contiguous() &&
           v.is_contiguous() && k.device() == dev && v.device() == dev,
       "k_pages and v_pages must be contiguous [pages][kv_heads][page_size][128] of one type, on the device of the "
       "other tensors");
  need(table.scalar_type() == at::kInt && table.dim() == 2 && table.device() == dev &&
           (table.size(1) <= 1 || table.stride(1) == 1),
       "block_table must be int32 [batch][pages] with contiguous rows, on the device of the other tensors");
  qd_paged_kv kv{};
  kv.k = k.data_ptr();
  kv.v = v.data_ptr();
  kv.dtype = code(k, "the cache");
  kv.num_pages = to_int(k.size(0), "too many pages");
  kv.kv_heads = to_int(k.size(1), "too many KV heads");
  kv.page_size = to_int(k.size(2), "page_size too large");
  kv.head_dim = to_int(k.size(3), "head_dim too large");
  kv.batch = to_int(table.size(0), "batch too large");
  kv.block_table = static_cast<const int32_t*>(table.const_data_ptr());
  kv.table_width = to_int(table.size(1), "block_table too wide");
  kv.table_stride = to_int(kv.batch > 1 ? table.stride(0) : table.size(1), "block_table too wide");
  kv.seq_lens = vec<int32_t>(lens, kv.batch, at::kInt, dev, "seq_lens");
  kv.status = const_cast<int32_t*>(vec<int32_t>(status, 1, at::kInt, dev, "status"));
  return kv;
}

// The device of a call's tensors made current, and its current stream. (What the call allocates
// belongs to that stream.)
struct Here {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit Here(c10::Device dev) : guard(dev), stream(c10::cuda::getCurrentCUDAStream(dev.index()).stream()) {}
};

// (straight from the allocator: through the dispatcher a call took 0.5 us more, of 5)
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
  return at::detail::empty_cuda(sizes, type, dev, std::nullopt);
}

Tensor workspace(const Maybe& given, size_t bytes, c10::Device dev) {
  if (!given) return fresh({(int64_t)bytes}, at::kByte, dev);
  need(given->device() == dev && given->is_contiguous() && given->nbytes() >= bytes,
       "workspace must be a contiguous tensor of at least the bytes that the call asks for, on its device");
  return *given;
}

Tensor paged_append(const Tensor& qkv, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens,
                    const Maybe& cos, const Maybe& sin, int64_t q_heads, const Maybe& q_norm, const Maybe& k_norm,
                    double eps, const Maybe& q_starts, const Maybe& q_out, std::optional<int64_t> rope_stride,
                    const Maybe& status) {
  const auto dev = qkv.device();
  const qd_paged_kv kv = paged(k, v, table, lens, status, dev);
  need(q_heads >= 0 && q_heads <= 65536, "bad q_heads");
  const int64_t stride = row_stride(qkv, (q_heads + 2 * kv.kv_heads) * 128, "qkv"), rows = qkv.size(0);
  int64_t rope_len = 0, step = rope_stride.value_or(0);
  for (const Maybe* x : {&cos, &sin})
    need(!*x || ((*x)->scalar_type() == at::kFloat && (*x)->device() == dev && (*x)->is_contiguous()),
         "cos and sin must be contiguous float32 tables on the device of the other tensors");
  if (cos && sin) {
    rope_len = std::min(cos->numel(), sin->numel());
    if (!rope_stride) {  // their own: 64 in a vector, else a row of both
      need(cos->sizes() == sin->sizes() &&
               (cos->dim() < 2 || (cos->size(-1) >= 64 && cos->numel() == cos->size(0) * cos->size(-1))),
           "cos and sin must be [positions][64 or more], of one shape, where no rope_stride is given");
      step = cos->dim() > 1 ? cos->size(-1) : 64;
    }
  }
  const Here here(dev);
  need(!q_out || (q_out->device() == dev && q_out->dim() >= 1 && q_out->size(0) == rows),
       "q_out must have a row for every row of qkv, on its device");
  const Tensor q = q_out ? *q_out : fresh({rows, q_heads * 128}, qkv.scalar_type(), dev);
  const int64_t q_stride = row_stride(q, q_heads * 128, "q_out");
  if (q_out) {
    const bool in_place = q.const_data_ptr() == qkv.const_data_ptr() && q.scalar_type() == qkv.scalar_type() &&
                          (q_stride == stride || rows == 1);
    need(in_place || qd::apart(rows_of(q, q_heads * 128, q_stride), rows_of(qkv, (q_heads + 2 * kv.kv_heads) * 128, stride)),
         "q_out overlaps qkv (it may be the first q_heads * 128 elements of its rows)");
  }
  done(qd_paged_append(&kv, qkv.const_data_ptr(), code(qkv, "qkv"), stride, to_int(rows, "too many rows"),
                       vec<int32_t>(q_starts, (int64_t)kv.batch + 1, at::kInt, dev, "q_starts"), (int)q_heads,
                       vec<float>(q_norm, 128, at::kFloat, dev, "q_norm"),
                       vec<float>(k_norm, 128, at::kFloat, dev, "k_norm"), (float)eps,
                       cos ? static_cast<const float*>(cos->const_data_ptr()) : nullptr,
                       sin ? static_cast<const float*>(sin->const_data_ptr()) : nullptr, rope_len, step, q.data_ptr(),
                       code(q, "q_out"), q_stride, here.stream));
  return q;
}

// The shared part of the two attention calls.
struct Attn {
  qd_paged_kv kv;
  int heads, dtype;
  int64_t width, q_stride;
  Attn(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens, const Maybe& status)
      : kv(paged(k, v, table, lens, status, q.device())) {
    need(q.dim() == 2 || q.dim() == 3, "q must be [rows][q_heads][128] or [rows][q_heads * 128]");
    width = q.dim() == 3 ? q.size(1) * q.size(2) : q.size(1);
    need(width % 128 == 0, "q must be [rows][q_heads][128] or [rows][q_heads * 128]");
    heads = to_int(width / 128, "too many heads");
    dtype = code(q, "q");
    q_stride = row_stride(q, width, "q");
  }
  Tensor out(const Tensor& q, const Maybe& y) const {
    if (!y) return fresh(q.sizes(), q.scalar_type(), q.device());
    need(y->scalar_type() == q.scalar_type() && y->sizes() == q.sizes() && y->device() == q.device(),
         "y must have q's type, shape and device");
    need(qd::apart(rows_of(*y, width, row_stride(*y, width, "y")), rows_of(q, width, q_stride)), "y overlaps q");
    return *y;
  }
};

Tensor paged_attn_decode(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens,
                         int64_t window, int64_t sinks, double scale, const Maybe& y_out, const Maybe& ws_in,
                         const Maybe& status) {
  const Attn a(q, k, v, table, lens, status);
  need(q.size(0) == a.kv.batch, "q must have one row per sequence");
  const Here here(q.device());
  const Tensor y = a.out(q, y_out);
  const Tensor ws = workspace(ws_in, qd_paged_attn_decode_workspace_bytes(a.kv.batch, a.heads), q.device());
  done(qd_paged_attn_decode(&a.kv, q.const_data_ptr(), a.dtype, a.q_stride, a.heads, to_int(window, "bad window"),
                            to_int(sinks, "bad sinks"), to_scale(scale), y.data_ptr(), row_stride(y, a.width, "y"),
                            ws.data_ptr(), here.stream));
  return y;
}

Tensor paged_attn_prompt(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens,
                         const Tensor& q_starts, int64_t window, int64_t sinks, double scale, const Maybe& y_out,
                         const Maybe& ws_in, const Maybe& status) {
  const Attn a(q, k, v, table, lens, status);
  const int rows = to_int(q.size(0), "too many rows");
  const Here here(q.device());
  const Tensor y = a.out(q, y_out);
  const Tensor ws =
      workspace(ws_in, qd_paged_attn_prompt_workspace_bytes(a.kv.batch, rows, a.heads, a.kv.kv_heads, a.dtype),
                q.device());
  done(qd_paged_attn_prompt(&a.kv, q.const_data_ptr(), a.dtype, a.q_stride, rows,
                            vec<int32_t>(q_starts, (int64_t)a.kv.batch + 1, at::kInt, q.device(), "q_starts"), a.heads,
                            to_int(window, "bad window"), to_int(sinks, "bad sinks"), to_scale(scale), y.data_ptr(),
                            row_stride(y, a.width, "y"), ws.data_ptr(), here.stream));
  return y;
}

std::pair<Tensor, Tensor> sample_rows(const Tensor& logits, const Tensor& u, const Maybe& temperature,
                                      const Maybe& top_k, const Maybe& top_p, const Maybe& min_p, const Maybe& ids_out,
                                      const Maybe& logprobs_out) {
  const auto dev = logits.device();
  need(logits.dim() == 2, "logits must be [rows][vocab]");
  need(dev.is_cuda(), "tensors must be on a CUDA device");
  const int64_t rows = logits.size(0), vocab = logits.size(1), stride = row_stride(logits, vocab, "logits");
  const Here here(dev);
  const Tensor ids = ids_out ? *ids_out : fresh({rows}, at::kInt, dev);
  const Tensor logprobs = logprobs_out ? *logprobs_out : fresh({rows}, at::kFloat, dev);
  need(vocab <= UINT32_MAX, "vocab too large");
  done(qd_sample_rows(logits.const_data_ptr(), code(logits, "logits"), to_int(rows, "too many rows"), (uint32_t)vocab,
                      stride, vec<float>(temperature, rows, at::kFloat, dev, "temperature"),
                      vec<int32_t>(top_k, rows, at::kInt, dev, "top_k"), vec<float>(top_p, rows, at::kFloat, dev, "top_p"),
                      vec<float>(min_p, rows, at::kFloat, dev, "min_p"), vec<float>(u, rows, at::kFloat, dev, "u"),
                      const_cast<int32_t*>(vec<int32_t>(ids, rows, at::kInt, dev, "ids")),
                      const_cast<float*>(vec<float>(logprobs, rows, at::kFloat, dev, "logprobs")), here.stream));
  return {ids, logprobs};
}

}  // namespace

PYBIND11_MODULE(_torch_calls, m) {
  m.def("paged_append", &paged_append);
  m.def("paged_attn_decode", &paged_attn_decode);
  m.def("paged_attn_prompt", &paged_attn_prompt);
  m.def("sample_rows", &sample_rows);
}
