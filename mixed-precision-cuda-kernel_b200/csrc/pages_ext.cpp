// The paged KV cache and the adjustment of logits as the `quant_cuda` module shows them (C ABI: include/cherryq.h).  As in
// quant_cuda_ext.cpp this file holds no device code: it checks the tensors and takes torch's current stream and device.
#include "pages_ext.h"

#include <cmath>

#include "tensor_checks.h"

namespace py = pybind11;

namespace {

using namespace checks;

// A pool of pages of keys and values in 16 bits; keeps its two tensors alive.
struct KVPages {
  torch::Tensor k, v;
  cq_pages c = {};
  c10::Device device;
  c10::cuda::CUDAStream home;

  KVPages(torch::Tensor k_pages, torch::Tensor v_pages)
      : k(std::move(k_pages)), v(std::move(v_pages)), device(k.device()), home(c10::cuda::getDefaultCUDAStream()) {
    TORCH_CHECK(k.scalar_type() == torch::kFloat16 || k.scalar_type() == torch::kBFloat16, "k must have dtype Half or BFloat16, got ",
                c10::toString(k.scalar_type()));
    check_tensor(k, "k", k.scalar_type(), device);
    check_tensor(v, "v", k.scalar_type(), device);
    home = c10::cuda::getCurrentCUDAStream(device.index());
    TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes(), "k and v must be (pages, KV heads, page size, D)");
    TORCH_CHECK(k.size(0) > 0 && k.size(0) <= INT32_MAX && k.size(1) > 0 && k.size(1) <= 16383, "1 to 2^31 - 1 pages, 1 to 16383 KV heads");
    TORCH_CHECK(k.size(2) == 16 || k.size(2) == 32 || k.size(2) == 64 || k.size(2) == 128 || k.size(2) == 256,
                "a page must have 16, 32, 64, 128 or 256 slots, not ", k.size(2));
    TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128, "heads must be 64 or 128 wide, not ", k.size(3));
    c.pages = (int)k.size(0);
    c.n_kv_heads = (int)k.size(1);
    c.page_size = (int)k.size(2);
    c.head_dim = (int)k.size(3);
    c.dtype = k.scalar_type() == torch::kFloat16 ? 0 : 2;
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    check_status(cq_pages_check(&c), "KVPages");
  }

  // zero-filled
  static KVPages empty(int64_t pages, int64_t n_kv_heads, int64_t page_size, int64_t head_dim, py::object dtype, const torch::Device& device) {
    TORCH_CHECK(pages > 0 && n_kv_heads > 0 && page_size > 0 && head_dim > 0, "sizes must be positive");
    const auto type = dtype.is_none() ? torch::kFloat16 : py::cast<c10::ScalarType>(dtype);
    auto kp = torch::zeros({pages, n_kv_heads, page_size, head_dim}, torch::TensorOptions().device(device).dtype(type)), vp = torch::zeros_like(kp);
    return KVPages(kp, vp);
  }

  // A launch on another stream than the one that the handle was made on is recorded with the allocator, so that the
  // tensors' memory is not given out before it ends.
  cq_stream_t use() const {
    const auto s = c10::cuda::getCurrentCUDAStream(device.index());
    if (s != home)
      for (const auto* t : {&k, &v}) c10::cuda::CUDACachingAllocator::recordStream(t->storage().data_ptr(), s);
    return (cq_stream_t)s.stream();
  }

  torch::Tensor fresh(c10::IntArrayRef shape, c10::ScalarType type) const { return fresh_on(device, shape, type); }

  cq_table check_table(const torch::Tensor& t) const {
    TORCH_CHECK(t.defined() && t.is_cuda() && t.device() == device, "table must be a CUDA tensor on ", device);
    TORCH_CHECK(t.scalar_type() == torch::kInt32, "table must have dtype Int, got ", c10::toString(t.scalar_type()));
    TORCH_CHECK(t.dim() == 2 && t.size(0) > 0 && t.size(0) <= 65535 && t.size(1) > 0 && (t.size(1) == 1 || t.stride(1) == 1),
                "table must be (sequences, pages of a sequence) with contiguous rows, of 1 to 65535 sequences");
    TORCH_CHECK(t.size(1) <= (1 << 30) / c.page_size, "a sequence may have 2^30 slots at most");
    return {(const int32_t*)t.const_data_ptr(), (int)t.size(0), (int)t.size(1), t.size(0) == 1 ? 0 : t.stride(0)};
  }
  // rows (rows, heads, D); heads < 0: any number
  cq_rows check_rows(const torch::Tensor& t, const char* name, int64_t rows, int64_t heads) const {
    TORCH_CHECK(t.defined() && t.is_cuda() && t.device() == device, name, " must be a CUDA tensor on ", device);
    TORCH_CHECK(t.scalar_type() == k.scalar_type(), name, " must have dtype ", c10::toString(k.scalar_type()), ", got ", c10::toString(t.scalar_type()));
    TORCH_CHECK(t.dim() == 3 && t.size(0) == rows && t.size(1) > 0 && (heads < 0 || t.size(1) == heads) && t.size(2) == c.head_dim, name,
                " must be (", rows, ", ", heads < 0 ? std::string("heads") : std::to_string(heads), ", ", c.head_dim, ")");
    const cq_rows r = {t.const_data_ptr(), t.size(0) == 1 ? 0 : t.stride(0), t.size(1) == 1 ? 0 : t.stride(1)};
    TORCH_CHECK(t.stride(2) == 1 && aligned16(t) && r.token_stride >= 0 && r.head_stride >= 0 && r.token_stride % 8 == 0 && r.head_stride % 8 == 0, name,
                " must have contiguous columns and 16-byte aligned rows");
    return r;
  }
  cq_rows check_queries(const torch::Tensor& q, int64_t rows) const {
    const cq_rows r = check_rows(q, "q", rows, -1);
    TORCH_CHECK(q.size(1) % c.n_kv_heads == 0 && q.size(1) <= INT32_MAX, "the query heads must be a multiple of the ", c.n_kv_heads, " KV heads");
    return r;
  }
  // the tables' rows; 0 without rotation
  int check_tables(const OptTensor& cos, const OptTensor& sin, const OptTensor& positions, int64_t rows) const {
    TORCH_CHECK(cos.has_value() == sin.has_value() && cos.has_value() == positions.has_value(), "cos, sin and positions come together");
    if (!cos.has_value()) return 0;
    check_tensor(*cos, "cos", torch::kFloat32, device);
    check_tensor(*sin, "sin", torch::kFloat32, device);
    TORCH_CHECK(cos->dim() == 2 && cos->size(0) > 0 && cos->size(0) <= INT32_MAX && cos->size(1) == c.head_dim / 2 && sin->sizes() == cos->sizes(),
                "cos / sin tables must be (positions, ", c.head_dim / 2, ")");
    whole_numbers(*positions, "positions", rows, device);
    return (int)cos->size(0);
  }

  OptTensor write(const OptTensor& q, const torch::Tensor& k_rows, const torch::Tensor& v_rows, const torch::Tensor& table, const torch::Tensor& first,
                  const OptTensor& cos, const OptTensor& sin, const OptTensor& positions, const OptTensor& starts) {
    const c10::cuda::CUDAGuard guard(device);
    const cq_table at = check_table(table);
    TORCH_CHECK(k_rows.dim() == 3 && k_rows.size(0) <= INT32_MAX, "k must be (rows, KV heads, D)");
    const int64_t rows = k_rows.size(0);
    TORCH_CHECK(starts.has_value() || rows % at.sequences == 0, "without starts the rows must be divided evenly among the ", at.sequences, " sequences");
    const long long* from = whole_numbers(first, "first", at.sequences, device);
    const long long* begin = starts.has_value() ? whole_numbers(*starts, "starts", at.sequences + 1, device) : nullptr;
    const cq_rows kr = check_rows(k_rows, "k", rows, c.n_kv_heads), vr = check_rows(v_rows, "v", rows, c.n_kv_heads);
    const cq_rows qr = q.has_value() ? check_queries(*q, rows) : cq_rows{};
    const int H = q.has_value() ? (int)q->size(1) : 0, tables = check_tables(cos, sin, positions, rows);
    OptTensor out;
    if (H) out = fresh({rows, H, c.head_dim}, k.scalar_type());
    if (rows == 0) return out;
    check_status(cq_pages_write(&c, &at, H ? &qr : nullptr, H ? out->data_ptr() : nullptr, &kr, &vr, tables ? cos->const_data_ptr<float>() : nullptr,
                                tables ? sin->const_data_ptr<float>() : nullptr, tables ? (const long long*)positions->const_data_ptr() : nullptr, tables,
                                from, begin, (int)rows, H, use()),
                 "KVPages.write");
    return out;
  }

  std::pair<torch::Tensor, torch::Tensor> read(const torch::Tensor& table, const torch::Tensor& first, int64_t count) {
    const c10::cuda::CUDAGuard guard(device);
    const cq_table at = check_table(table);
    TORCH_CHECK(count > 0 && count <= INT32_MAX, "count must be positive");
    const long long* from = whole_numbers(first, "first", at.sequences, device);
    auto to_k = fresh({at.sequences, count, c.n_kv_heads, c.head_dim}, k.scalar_type()), to_v = fresh(to_k.sizes(), k.scalar_type());
    check_status(cq_pages_read(&c, &at, from, (int)count, to_k.data_ptr(), to_v.data_ptr(), use()), "KVPages.read");
    return {to_k, to_v};
  }

  static float check_scale(c10::optional<double> scale, int head_dim) {
    const float s = (float)scale.value_or(1.0 / std::sqrt((double)head_dim));
    TORCH_CHECK(s > 0.f && std::isfinite(s), "scale must be positive");
    return s;
  }
  // undefined where a call needs none
  torch::Tensor workspace(const cq_table& at, int H, int64_t window, int64_t sinks) const {
    const int64_t bytes = (int64_t)cq_pages_attend_workspace_bytes(&c, &at, H, (int)window, (int)sinks);
    return bytes ? fresh({bytes}, torch::kUInt8) : torch::Tensor();
  }

  torch::Tensor attend(const torch::Tensor& q, const torch::Tensor& table, const torch::Tensor& length, int64_t window, int64_t sinks,
                       c10::optional<double> scale) {
    const c10::cuda::CUDAGuard guard(device);
    const cq_table at = check_table(table);
    const cq_rows qr = check_queries(q, at.sequences);
    check_mask(window, sinks);
    const float by = check_scale(scale, c.head_dim);
    const long long* n = whole_numbers(length, "length", at.sequences, device);
    const int H = (int)q.size(1);
    auto out = fresh(q.sizes(), k.scalar_type());
    auto ws = workspace(at, H, window, sinks);
    check_status(cq_pages_attend(&c, &at, &qr, n, out.data_ptr(), H, (int)window, (int)sinks, by, ws.defined() ? ws.data_ptr() : nullptr, use()),
                 "KVPages.attend");
    return out;
  }

  torch::Tensor step(const torch::Tensor& q, const torch::Tensor& k_rows, const torch::Tensor& v_rows, const OptTensor& cos, const OptTensor& sin,
                     const OptTensor& positions, const torch::Tensor& table, const torch::Tensor& length, int64_t window, int64_t sinks,
                     c10::optional<double> scale) {
    const c10::cuda::CUDAGuard guard(device);
    const cq_table at = check_table(table);
    const cq_rows qr = check_queries(q, at.sequences);
    const cq_rows kr = check_rows(k_rows, "k", at.sequences, c.n_kv_heads), vr = check_rows(v_rows, "v", at.sequences, c.n_kv_heads);
    check_mask(window, sinks);
    const float by = check_scale(scale, c.head_dim);
    const int tables = check_tables(cos, sin, positions, at.sequences), H = (int)q.size(1);
    const long long* n = whole_numbers(length, "length", at.sequences, device);
    auto out = fresh(q.sizes(), k.scalar_type());
    auto ws = workspace(at, H, window, sinks);
    check_status(cq_pages_step(&c, &at, &qr, &kr, &vr, tables ? cos->const_data_ptr<float>() : nullptr, tables ? sin->const_data_ptr<float>() : nullptr,
                               tables ? (const long long*)positions->const_data_ptr() : nullptr, tables, n, out.data_ptr(), H, (int)window, (int)sinks, by,
                               ws.defined() ? ws.data_ptr() : nullptr, use()),
                 "KVPages.step");
    return out;
  }
};

// ------------------------------------------------------------------ logits
// stride between the rows of a matrix (rows, columns) whose columns are contiguous
int64_t matrix(const torch::Tensor& t, const char* name, c10::ScalarType dtype, const c10::Device& device, int64_t rows) {
  TORCH_CHECK(t.defined() && t.is_cuda() && t.device() == device, name, " must be a CUDA tensor on ", device);
  TORCH_CHECK(t.scalar_type() == dtype, name, " must have dtype ", c10::toString(dtype), ", got ", c10::toString(t.scalar_type()));
  TORCH_CHECK(t.dim() == 2 && (rows < 0 || t.size(0) == rows) && (t.size(1) <= 1 || t.stride(1) == 1), name, " must be (",
              rows < 0 ? std::string("rows") : std::to_string(rows), ", columns) with contiguous columns");
  return t.size(0) <= 1 ? 0 : t.stride(0);
}
const float* numbers(const OptTensor& t, const char* name, int64_t n, const c10::Device& device) {
  if (!t.has_value()) return nullptr;
  check_tensor(*t, name, torch::kFloat32, device);
  TORCH_CHECK(t->numel() == n, name, " must have ", n, " entries");
  return t->const_data_ptr<float>();
}

std::pair<torch::Tensor, torch::Tensor> adjust_logits(const torch::Tensor& logits, const OptTensor& tokens, const OptTensor& length, const OptTensor& prompt,
                                                      const OptTensor& repetition, const OptTensor& presence, const OptTensor& frequency,
                                                      const OptTensor& bias_ids, const OptTensor& bias, const OptTensor& mask, const OptTensor& mask_rows,
                                                      const OptTensor& out) {
  TORCH_CHECK(logits.defined() && logits.is_cuda(), "logits must be a CUDA tensor");
  const auto type = logits.scalar_type();
  TORCH_CHECK(type == torch::kFloat16 || type == torch::kBFloat16 || type == torch::kFloat32, "logits must have dtype Half, BFloat16 or Float, got ",
              c10::toString(type));
  const c10::Device device = logits.device();
  const c10::cuda::CUDAGuard guard(device);
  cq_adjust a = {};
  a.logits_stride = matrix(logits, "logits", type, device, -1);
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  TORCH_CHECK(rows <= 65535 && vocab > 0 && vocab <= (1 << 30), "at most 65535 rows of 1 to 2^30 logits");
  a.dtype = type == torch::kFloat16 ? 0 : (type == torch::kFloat32 ? 1 : 2);
  a.logits = logits.const_data_ptr();
  TORCH_CHECK(tokens.has_value() || !(length.has_value() || prompt.has_value() || repetition.has_value() || presence.has_value() || frequency.has_value()),
              "length, prompt and penalties need tokens");
  if (tokens.has_value()) {
    a.tokens_stride = matrix(*tokens, "tokens", torch::kInt64, device, rows);
    TORCH_CHECK(tokens->size(1) < (1 << 30), "less than 2^30 tokens a row");
    a.tokens = (const long long*)tokens->const_data_ptr();
    a.width = tokens->size(1);
    if (length.has_value()) a.length = whole_numbers(*length, "length", rows, device);
    if (prompt.has_value()) a.prompt = whole_numbers(*prompt, "prompt", rows, device);
    a.repetition = numbers(repetition, "repetition", rows, device);
    a.presence = numbers(presence, "presence", rows, device);
    a.frequency = numbers(frequency, "frequency", rows, device);
    // without a penalty nothing depends on the history
    if (a.width == 0 || !(a.repetition || a.presence || a.frequency)) {
      a.tokens = a.length = a.prompt = nullptr;
      a.repetition = a.presence = a.frequency = nullptr;
    }
  }
  TORCH_CHECK(bias_ids.has_value() == bias.has_value(), "bias_ids and bias come together");
  if (bias.has_value()) {
    a.bias_ids_stride = matrix(*bias_ids, "bias_ids", torch::kInt64, device, rows);
    a.bias_stride = matrix(*bias, "bias", torch::kFloat32, device, rows);
    TORCH_CHECK(bias->size(1) == bias_ids->size(1) && bias->size(1) < (1 << 30), "bias_ids and bias must have the same shape, of less than 2^30 a row");
    a.biases = (int)bias->size(1);
    a.bias_ids = (const long long*)bias_ids->const_data_ptr();
    a.bias = bias->const_data_ptr<float>();
  }
  TORCH_CHECK(mask.has_value() || !mask_rows.has_value(), "mask_rows without mask");
  if (mask.has_value()) {
    a.mask_stride = matrix(*mask, "mask", torch::kInt32, device, -1);
    TORCH_CHECK(mask->size(1) >= (vocab + 31) / 32 && mask->size(0) > 0 && mask->size(0) <= INT32_MAX, "mask must be (masks, ", (vocab + 31) / 32,
                " or more words)");
    a.mask = (const uint32_t*)mask->const_data_ptr();
    a.masks = (int)mask->size(0);
    if (mask_rows.has_value()) a.mask_rows = whole_numbers(*mask_rows, "mask_rows", rows, device);
    else TORCH_CHECK(a.masks == rows, "without mask_rows mask must have ", rows, " rows");
  }
  torch::Tensor to;
  if (out.has_value()) {
    to = *out;
    a.out_stride = matrix(to, "out", type, device, rows);
    TORCH_CHECK(to.size(1) == vocab && (rows <= 1 || to.stride(0) >= vocab), "out must be (", rows, ", ", vocab, ") with rows apart from one another");
  } else {
    to = fresh_on(device, logits.sizes(), type);
    a.out_stride = vocab;
  }
  auto next = fresh_on(device, {rows}, torch::kInt64);
  if (rows == 0) return {to, next};
  a.out = to.data_ptr();
  a.next = (long long*)next.data_ptr();
  check_status(cq_adjust_logits(&a, (int)rows, (int)vocab, (cq_stream_t)c10::cuda::getCurrentCUDAStream().stream()), "adjust_logits");
  return {to, next};
}

}  // namespace

void register_pages(py::module_& m) {
  using py::arg;
  m.def("adjust_logits", &adjust_logits, "penalties, biases and a grammar's mask on logits: (adjusted logits, the token with the largest one)",
        arg("logits"), arg("tokens") = py::none(), arg("length") = py::none(), arg("prompt") = py::none(), arg("repetition") = py::none(),
        arg("presence") = py::none(), arg("frequency") = py::none(), arg("bias_ids") = py::none(), arg("bias") = py::none(), arg("mask") = py::none(),
        arg("mask_rows") = py::none(), arg("out") = py::none());
  py::class_<KVPages>(m, "KVPages")
      .def(py::init<torch::Tensor, torch::Tensor>(), arg("k"), arg("v"))
      .def_static("empty", &KVPages::empty, arg("pages"), arg("n_kv_heads"), arg("page_size"), arg("head_dim"), arg("dtype") = py::none(),
                  arg("device") = torch::Device(torch::kCUDA))
      .def("write", &KVPages::write, arg("q"), arg("k"), arg("v"), arg("table"), arg("first"), arg("cos") = py::none(), arg("sin") = py::none(),
           arg("positions") = py::none(), arg("starts") = py::none())
      .def("read", &KVPages::read, arg("table"), arg("first"), arg("count"))
      .def("attend", &KVPages::attend, arg("q"), arg("table"), arg("length"), arg("window") = 0, arg("sinks") = 0, arg("scale") = py::none())
      .def("step", &KVPages::step, arg("q"), arg("k"), arg("v"), arg("cos"), arg("sin"), arg("positions"), arg("table"), arg("length"),
           arg("window") = 0, arg("sinks") = 0, arg("scale") = py::none())
      .def_readonly("k", &KVPages::k)
      .def_readonly("v", &KVPages::v)
      .def_property_readonly("pages", [](const KVPages& s) { return s.c.pages; })
      .def_property_readonly("n_kv_heads", [](const KVPages& s) { return s.c.n_kv_heads; })
      .def_property_readonly("page_size", [](const KVPages& s) { return s.c.page_size; })
      .def_property_readonly("head_dim", [](const KVPages& s) { return s.c.head_dim; });
}
