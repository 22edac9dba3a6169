// The 4-bit KV cache and the attention of prompts as the `quant_cuda` module shows them (C ABI: include/cherryq.h).  As in
// quant_cuda_ext.cpp this file holds no device code: it checks the tensors and takes torch's current stream and device.
#include "kv4_ext.h"

#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>
#include <cmath>

#include "cherryq.h"

namespace py = pybind11;

namespace {

using OptTensor = c10::optional<torch::Tensor>;

void check_status(int rc, const char* what) {
  if (rc == CQ_OK) return;
  TORCH_CHECK(rc != CQ_ERR_CUDA, what, ": CUDA error ", cq_last_cuda_error());
  TORCH_CHECK(false, what, ": ", cq_strerror(rc));
}

void check_tensor(const torch::Tensor& t, const char* name, c10::ScalarType dtype, const c10::Device& device) {
  TORCH_CHECK(t.defined() && t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == dtype, name, " must have dtype ", c10::toString(dtype), ", got ", c10::toString(t.scalar_type()));
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.device() == device, name, " is on ", t.device(), ", not on ", device);
}

bool aligned16(const torch::Tensor& t) { return ((uintptr_t)t.const_data_ptr() & 15) == 0; }

void check_mask(int64_t window, int64_t sinks) {
  TORCH_CHECK(window >= 0 && window <= INT32_MAX && sinks >= 0 && sinks <= INT32_MAX, "window and sinks must not be negative");
}

const long long* whole_numbers(const torch::Tensor& t, const char* name, int64_t n, const c10::Device& device) {
  check_tensor(t, name, torch::kInt64, device);
  TORCH_CHECK(t.numel() == n, name, " must have ", n, " entries");
  return (const long long*)t.const_data_ptr();
}

// An output or workspace, straight from the allocator: short calls are bound by the host, and a trip through the dispatcher for
// each of them costs more than the rest of a call.  (Not where a dispatch mode watches.)
torch::Tensor fresh_on(const c10::Device& device, c10::IntArrayRef shape, c10::ScalarType type) {
  if (c10::impl::TorchDispatchModeTLS::any_modes_set()) return torch::empty(shape, torch::TensorOptions().device(device).dtype(type));
  return at::detail::empty_cuda(shape, type, device, c10::nullopt);
}

// KV cache of `sequences` sequences in 4 bits; keeps its four tensors alive.
struct KVCache4 {
  torch::Tensor k_codes, k_scales, v_codes, v_scales;
  cq_kv4 c = {};
  c10::Device device;
  c10::cuda::CUDAStream home;

  KVCache4(torch::Tensor kc, torch::Tensor ks, torch::Tensor vc, torch::Tensor vs)
      : k_codes(std::move(kc)), k_scales(std::move(ks)), v_codes(std::move(vc)), v_scales(std::move(vs)), device(k_codes.device()),
        home(c10::cuda::getDefaultCUDAStream()) {
    check_tensor(k_codes, "k_codes", torch::kUInt8, device);
    check_tensor(v_codes, "v_codes", torch::kUInt8, device);
    check_tensor(k_scales, "k_scales", torch::kFloat16, device);
    check_tensor(v_scales, "v_scales", torch::kFloat16, device);
    home = c10::cuda::getCurrentCUDAStream(device.index());
    TORCH_CHECK(k_codes.dim() == 4 && v_codes.sizes() == k_codes.sizes(), "codes must be (sequences, KV heads, slots, D / 2)");
    TORCH_CHECK(k_scales.dim() == 5 && v_scales.sizes() == k_scales.sizes() && k_scales.size(4) == 2 && k_scales.size(0) == k_codes.size(0) &&
                    k_scales.size(1) == k_codes.size(1) && k_scales.size(2) == k_codes.size(2),
                "scales must be (sequences, KV heads, slots, D / group, 2)");
    const int64_t D = 2 * k_codes.size(3), groups = k_scales.size(3);
    TORCH_CHECK(D == 64 || D == 128, "heads must be 64 or 128 wide, not ", D);
    TORCH_CHECK(groups > 0 && D % groups == 0 && (D / groups == 32 || D / groups == 64), "groups must have 32 or 64 columns");
    TORCH_CHECK(k_codes.size(2) > 0 && k_codes.size(2) % 32 == 0 && k_codes.size(2) <= (1 << 30), "slots must be a multiple of 32");
    TORCH_CHECK(k_codes.size(0) > 0 && k_codes.size(0) <= 65535 && k_codes.size(1) > 0 && k_codes.size(1) <= 32767, "1 to 65535 sequences, 1 to 32767 KV heads");
    c.sequences = (int)k_codes.size(0);
    c.n_kv_heads = (int)k_codes.size(1);
    c.slots = (int)k_codes.size(2);
    c.head_dim = (int)D;
    c.group = (int)(D / groups);
    c.k_codes = k_codes.data_ptr();
    c.k_scales = k_scales.data_ptr();
    c.v_codes = v_codes.data_ptr();
    c.v_scales = v_scales.data_ptr();
    check_status(cq_kv4_check(&c), "KVCache4");
  }

  // zero-filled; slots rounded up to a multiple of 32
  static KVCache4 empty(int64_t sequences, int64_t n_kv_heads, int64_t slots, int64_t head_dim, int64_t group, const torch::Device& device) {
    TORCH_CHECK(sequences > 0 && n_kv_heads > 0 && slots > 0 && head_dim > 0 && group > 0 && head_dim % group == 0,
                "sizes must be positive and the group divide the head");
    slots = (slots + 31) / 32 * 32;
    const auto codes = torch::TensorOptions().device(device).dtype(torch::kUInt8), scales = codes.dtype(torch::kFloat16);
    auto kc = torch::zeros({sequences, n_kv_heads, slots, head_dim / 2}, codes), vc = torch::zeros_like(kc);
    auto ks = torch::zeros({sequences, n_kv_heads, slots, head_dim / group, 2}, scales), vs = torch::zeros_like(ks);
    return KVCache4(kc, ks, vc, vs);
  }

  // A launch on another stream than the one that the handle was made on is recorded with the allocator, so that the
  // tensors' memory is not given out before it ends.
  cq_stream_t use() const {
    const auto s = c10::cuda::getCurrentCUDAStream(device.index());
    if (s != home)
      for (const auto* t : {&k_codes, &k_scales, &v_codes, &v_scales}) c10::cuda::CUDACachingAllocator::recordStream(t->storage().data_ptr(), s);
    return (cq_stream_t)s.stream();
  }

  torch::Tensor fresh(c10::IntArrayRef shape, c10::ScalarType type) const { return fresh_on(device, shape, type); }

  // rows (rows, heads, D) fp16; returns the number of heads
  int check_rows(const torch::Tensor& t, const char* name, int64_t rows, int64_t heads) const {
    check_tensor(t, name, torch::kFloat16, device);
    TORCH_CHECK(t.dim() == 3 && t.size(0) == rows && t.size(1) > 0 && (heads < 0 || t.size(1) == heads) && t.size(2) == c.head_dim, name,
                " must be (", rows, ", ", heads < 0 ? std::string("heads") : std::to_string(heads), ", ", c.head_dim, ")");
    TORCH_CHECK(aligned16(t), name, " must be 16-byte aligned");
    return (int)t.size(1);
  }
  int check_queries(const torch::Tensor& q, int64_t rows) const {
    const int H = check_rows(q, "q", rows, -1);
    TORCH_CHECK(H % c.n_kv_heads == 0, "the query heads must be a multiple of the ", c.n_kv_heads, " KV heads");
    return H;
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

  OptTensor write(const OptTensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& first, const OptTensor& cos,
                  const OptTensor& sin, const OptTensor& positions) {
    const c10::cuda::CUDAGuard guard(device);
    TORCH_CHECK(k.dim() == 3 && k.size(0) > 0 && k.size(0) % c.sequences == 0 && k.size(0) <= INT32_MAX,
                "k must be (sequences * tokens, KV heads, D)");
    const int64_t rows = k.size(0);
    check_rows(k, "k", rows, c.n_kv_heads);
    check_rows(v, "v", rows, c.n_kv_heads);
    const int H = q.has_value() ? check_queries(*q, rows) : 0;
    const int table = check_tables(cos, sin, positions, rows);
    const long long* at = whole_numbers(first, "first", c.sequences, device);
    OptTensor out;
    if (q.has_value()) out = fresh(q->sizes(), torch::kFloat16);
    check_status(cq_kv4_write(&c, H ? q->const_data_ptr() : nullptr, H ? out->data_ptr() : nullptr, k.const_data_ptr(), v.const_data_ptr(),
                              table ? cos->const_data_ptr<float>() : nullptr, table ? sin->const_data_ptr<float>() : nullptr,
                              table ? (const long long*)positions->const_data_ptr() : nullptr, table, at, (int)(rows / c.sequences), H, use()),
                 "KVCache4.write");
    return out;
  }

  std::pair<torch::Tensor, torch::Tensor> read(const torch::Tensor& first, int64_t count) {
    const c10::cuda::CUDAGuard guard(device);
    TORCH_CHECK(count > 0 && count <= INT32_MAX, "count must be positive");
    const long long* at = whole_numbers(first, "first", c.sequences, device);
    auto k = fresh({c.sequences, count, c.n_kv_heads, c.head_dim}, torch::kFloat16), v = fresh(k.sizes(), torch::kFloat16);
    check_status(cq_kv4_read(&c, at, (int)count, k.data_ptr(), v.data_ptr(), use()), "KVCache4.read");
    return {k, v};
  }

  // (in, out) of the accumulated weights, or nulls
  std::pair<const float*, float*> check_weights(const OptTensor& weights, const OptTensor& weights_out) const {
    if (!weights.has_value()) {
      TORCH_CHECK(!weights_out.has_value(), "weights_out without weights");
      return {nullptr, nullptr};
    }
    const torch::Tensor& out = weights_out.has_value() ? *weights_out : *weights;
    for (const auto* t : {&*weights, &out}) {
      check_tensor(*t, "weights", torch::kFloat32, device);
      TORCH_CHECK(t->dim() == 3 && t->size(0) == c.sequences && t->size(1) == c.n_kv_heads && t->size(2) == c.slots, "weights must be (",
                  c.sequences, ", ", c.n_kv_heads, ", ", c.slots, ")");
    }
    return {weights->const_data_ptr<float>(), out.data_ptr<float>()};
  }

  // undefined where a call needs none
  torch::Tensor workspace(int H, int64_t window, int64_t sinks, bool weights) const {
    const int64_t bytes = (int64_t)cq_kv4_attend_workspace_bytes(&c, H, (int)window, (int)sinks, weights);
    return bytes ? fresh({bytes}, torch::kUInt8) : torch::Tensor();
  }

  torch::Tensor attend(const torch::Tensor& q, const torch::Tensor& length, int64_t window, int64_t sinks, const OptTensor& weights,
                       const OptTensor& weights_out, c10::optional<double> scale) {
    const c10::cuda::CUDAGuard guard(device);
    const int H = check_queries(q, c.sequences);
    check_mask(window, sinks);
    const long long* n = whole_numbers(length, "length", c.sequences, device);
    const auto w = check_weights(weights, weights_out);
    auto out = fresh(q.sizes(), torch::kFloat16);
    auto ws = workspace(H, window, sinks, w.first);
    check_status(cq_kv4_attend(&c, q.const_data_ptr(), n, out.data_ptr(), H, (int)window, (int)sinks,
                               (float)scale.value_or(1.0 / std::sqrt((double)c.head_dim)), w.first, w.second, ws.defined() ? ws.data_ptr() : nullptr, use()),
                 "KVCache4.attend");
    return out;
  }

  torch::Tensor step(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const OptTensor& cos, const OptTensor& sin,
                     const OptTensor& positions, const torch::Tensor& length, int64_t window, int64_t sinks, const OptTensor& weights,
                     const OptTensor& weights_out, c10::optional<double> scale) {
    const c10::cuda::CUDAGuard guard(device);
    const int H = check_queries(q, c.sequences);
    check_rows(k, "k", c.sequences, c.n_kv_heads);
    check_rows(v, "v", c.sequences, c.n_kv_heads);
    check_mask(window, sinks);
    const int table = check_tables(cos, sin, positions, c.sequences);
    const long long* n = whole_numbers(length, "length", c.sequences, device);
    const auto w = check_weights(weights, weights_out);
    auto out = fresh(q.sizes(), torch::kFloat16);
    auto ws = workspace(H, window, sinks, w.first);
    check_status(cq_kv4_step(&c, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), table ? cos->const_data_ptr<float>() : nullptr,
                             table ? sin->const_data_ptr<float>() : nullptr, table ? (const long long*)positions->const_data_ptr() : nullptr,
                             table, n, out.data_ptr(), H, (int)window, (int)sinks,
                             (float)scale.value_or(1.0 / std::sqrt((double)c.head_dim)), w.first, w.second, ws.defined() ? ws.data_ptr() : nullptr, use()),
                 "KVCache4.step");
    return out;
  }

  std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> evict(const torch::Tensor& weights, const torch::Tensor& length, int64_t keep,
                                                                int64_t sinks, int64_t recent, KVCache4* out) {
    const c10::cuda::CUDAGuard guard(device);
    const auto w = check_weights(weights, c10::nullopt);
    const long long* n = whole_numbers(length, "length", c.sequences, device);
    const KVCache4& to = out ? *out : *this;
    TORCH_CHECK(to.device == device && to.c.sequences == c.sequences && to.c.n_kv_heads == c.n_kv_heads && to.c.head_dim == c.head_dim &&
                    to.c.group == c.group, "the caches must agree in all but their slots");
    TORCH_CHECK(keep > 0 && keep <= to.c.slots, "keep must be 1 to ", to.c.slots);
    TORCH_CHECK(sinks >= 0 && sinks <= INT32_MAX && recent >= 0 && recent <= INT32_MAX, "sinks and recent must be 0 or more");
    auto kept = fresh({c.sequences, c.n_kv_heads, keep}, torch::kInt32), left = fresh(kept.sizes(), torch::kFloat32), now = fresh(length.sizes(), torch::kInt64);
    torch::Tensor ws;
    if (to.c.k_codes == c.k_codes) ws = fresh({(int64_t)cq_kv4_evict_workspace_bytes(&c, (int)keep)}, torch::kUInt8);
    to.use();
    check_status(cq_kv4_evict(&c, &to.c, w.first, left.data_ptr<float>(), n, (long long*)now.data_ptr(), (int)keep, (int)sinks, (int)recent,
                              kept.data_ptr<int>(), ws.defined() ? ws.data_ptr() : nullptr, use()),
                 "KVCache4.evict");
    return {kept, left, now};
  }
};

// strides (sequence, token, head) of q, k or v (sequences, tokens, heads, D)
void strides_of(const torch::Tensor& t, const char* name, const c10::Device& device, int64_t (&to)[3]) {
  TORCH_CHECK(t.defined() && t.is_cuda() && t.device() == device, name, " must be a CUDA tensor on ", device);
  TORCH_CHECK(t.scalar_type() == torch::kFloat16, name, " must have dtype Half, got ", c10::toString(t.scalar_type()));
  TORCH_CHECK(t.dim() == 4 && t.numel() > 0, name, " must be (sequences, tokens, heads, D)");
  bool fits = t.stride(3) == 1 && aligned16(t);
  for (int i = 0; i < 3; ++i) {
    to[i] = t.size(i) == 1 ? 0 : t.stride(i);
    fits = fits && to[i] % 8 == 0 && to[i] >= 0;
  }
  TORCH_CHECK(fits, name, " must have contiguous columns and 16-byte aligned rows");
}

// one row for all tokens (an expanded tensor) is written out: the kernels' copies of tiles need a step from token to token
torch::Tensor rows_apart(const torch::Tensor& t) {
  return t.defined() && t.dim() == 4 && t.size(1) > 1 && t.stride(1) == 0 ? t.contiguous() : t;
}

cq_prompt prompt_of(const torch::Tensor& q, const torch::Tensor& k, int64_t window, int64_t sinks, const OptTensor& lengths,
                    c10::optional<double> scale, const long long** n) {
  cq_prompt s = {};
  TORCH_CHECK(q.defined() && q.is_cuda(), "q must be a CUDA tensor");
  strides_of(q, "q", q.device(), s.q_strides);
  strides_of(k, "k", q.device(), s.k_strides);
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(3) == k.size(3) && q.size(1) <= k.size(1) && q.size(2) % k.size(2) == 0,
              "q must be (sequences, queries, heads, D) and k (sequences, keys, KV heads, D), with no more queries than keys");
  TORCH_CHECK(q.size(3) == 64 || q.size(3) == 128, "heads must be 64 or 128 wide, not ", q.size(3));
  check_mask(window, sinks);
  TORCH_CHECK(q.size(0) <= 65535 && q.size(2) <= 65535 && k.size(1) <= (1 << 24), "too many sequences, heads or keys");
  s.sequences = (int)q.size(0);
  s.queries = (int)q.size(1);
  s.keys = (int)k.size(1);
  s.n_heads = (int)q.size(2);
  s.n_kv_heads = (int)k.size(2);
  s.head_dim = (int)q.size(3);
  s.window = (int)window;
  s.sinks = (int)sinks;
  s.scale = (float)scale.value_or(1.0 / std::sqrt((double)s.head_dim));
  TORCH_CHECK(s.scale > 0.f, "scale must be positive");
  *n = lengths.has_value() ? whole_numbers(*lengths, "lengths", s.sequences, q.device()) : nullptr;
  return s;
}

std::pair<torch::Tensor, torch::Tensor> attn_prefill(torch::Tensor q, torch::Tensor k, torch::Tensor v, int64_t window,
                                                     int64_t sinks, const OptTensor& lengths, c10::optional<double> scale) {
  const at::cuda::OptionalCUDAGuard guard(device_of(q));
  const long long* n;
  q = rows_apart(q), k = rows_apart(k), v = rows_apart(v);
  cq_prompt s = prompt_of(q, k, window, sinks, lengths, scale, &n);
  strides_of(v, "v", q.device(), s.v_strides);
  TORCH_CHECK(v.sizes() == k.sizes(), "v must have the shape of k");
  auto out = fresh_on(q.device(), q.sizes(), torch::kFloat16), lse = fresh_on(q.device(), {s.sequences, s.n_heads, s.queries}, torch::kFloat32);
  torch::Tensor ws;
  if (const size_t bytes = cq_attn_prefill_workspace_bytes(&s)) ws = fresh_on(q.device(), {(int64_t)bytes}, torch::kUInt8);
  check_status(cq_attn_prefill(&s, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), n, out.data_ptr(), lse.data_ptr<float>(),
                               ws.defined() ? ws.data_ptr() : nullptr, device_status(q.device()),
                               (cq_stream_t)c10::cuda::getCurrentCUDAStream().stream()),
               "attn_prefill");
  return {out, lse};
}

torch::Tensor attn_prefill_weights(torch::Tensor q, torch::Tensor k, const torch::Tensor& lse, int64_t window, int64_t sinks,
                                   const OptTensor& lengths, c10::optional<int64_t> observe, c10::optional<double> scale) {
  const at::cuda::OptionalCUDAGuard guard(device_of(q));
  const long long* n;
  q = rows_apart(q), k = rows_apart(k);
  const cq_prompt s = prompt_of(q, k, window, sinks, lengths, scale, &n);
  check_tensor(lse, "lse", torch::kFloat32, q.device());
  TORCH_CHECK(lse.dim() == 3 && lse.size(0) == s.sequences && lse.size(1) == s.n_heads && lse.size(2) == s.queries,
              "lse must be (sequences, heads, queries)");
  const int64_t last = observe.value_or(s.keys);
  TORCH_CHECK(last > 0, "observe must be positive");
  auto out = fresh_on(q.device(), {s.sequences, s.n_kv_heads, s.keys}, torch::kFloat32);
  auto ws = fresh_on(q.device(), {(int64_t)cq_attn_prefill_weights_workspace_bytes(&s, (int)std::min<int64_t>(last, s.keys))}, torch::kUInt8);
  check_status(cq_attn_prefill_weights(&s, q.const_data_ptr(), k.const_data_ptr(), lse.const_data_ptr<float>(), n,
                                       (int)std::min<int64_t>(last, s.keys), out.data_ptr<float>(), ws.data_ptr(),
                                       device_status(q.device()), (cq_stream_t)c10::cuda::getCurrentCUDAStream().stream()),
               "attn_prefill_weights");
  return out;
}

}  // namespace

void register_kv4(py::module_& m) {
  using py::arg;
  m.def("attn_prefill", &attn_prefill, "causal attention of prompts with a sliding window and sinks: (out, lse)", arg("q"), arg("k"), arg("v"),
        arg("window") = 0, arg("sinks") = 0, arg("lengths") = py::none(), arg("scale") = py::none());
  m.def("attn_prefill_weights", &attn_prefill_weights, "the weight that each key received from the last queries", arg("q"), arg("k"), arg("lse"),
        arg("window") = 0, arg("sinks") = 0, arg("lengths") = py::none(), arg("observe") = py::none(), arg("scale") = py::none());
  py::class_<KVCache4>(m, "KVCache4")
      .def(py::init<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>(), arg("k_codes"), arg("k_scales"), arg("v_codes"),
           arg("v_scales"))
      .def_static("empty", &KVCache4::empty, arg("sequences"), arg("n_kv_heads"), arg("slots"), arg("head_dim"), arg("group") = 32,
                  arg("device") = torch::Device(torch::kCUDA))
      .def("write", &KVCache4::write, arg("q"), arg("k"), arg("v"), arg("first"), arg("cos") = py::none(), arg("sin") = py::none(),
           arg("positions") = py::none())
      .def("read", &KVCache4::read, arg("first"), arg("count"))
      .def("attend", &KVCache4::attend, arg("q"), arg("length"), arg("window") = 0, arg("sinks") = 0, arg("weights") = py::none(),
           arg("weights_out") = py::none(), arg("scale") = py::none())
      .def("step", &KVCache4::step, arg("q"), arg("k"), arg("v"), arg("cos"), arg("sin"), arg("positions"), arg("length"), arg("window") = 0,
           arg("sinks") = 0, arg("weights") = py::none(), arg("weights_out") = py::none(), arg("scale") = py::none())
      .def("evict", &KVCache4::evict, arg("weights"), arg("length"), arg("keep"), arg("sinks") = 0, arg("recent") = 0, arg("out") = nullptr)
      .def_readonly("k_codes", &KVCache4::k_codes)
      .def_readonly("k_scales", &KVCache4::k_scales)
      .def_readonly("v_codes", &KVCache4::v_codes)
      .def_readonly("v_scales", &KVCache4::v_scales)
      .def_property_readonly("sequences", [](const KVCache4& s) { return s.c.sequences; })
      .def_property_readonly("n_kv_heads", [](const KVCache4& s) { return s.c.n_kv_heads; })
      .def_property_readonly("slots", [](const KVCache4& s) { return s.c.slots; })
      .def_property_readonly("head_dim", [](const KVCache4& s) { return s.c.head_dim; })
      .def_property_readonly("group", [](const KVCache4& s) { return s.c.group; });
}
