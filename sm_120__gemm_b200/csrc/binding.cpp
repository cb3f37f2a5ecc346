// Host path of the operators' Python entry points (linear.py, experts.py): the
// checks of their tensors, their outputs and workspaces, and the call of the
// C ABI. In Python the same work took 11-18 us a call, several times the
// kernels of a single token (routing 18.2 -> 7.3 us, combination 10.5 -> 5.5 us).
//
// Every function runs on the current device's current stream; the Python side
// makes the tensors' device and the caller's stream current first.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>
#include <torch/version.h>

#include <map>
#include <mutex>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/i4g.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

[[noreturn]] void bad_value(const std::string& text) { throw py::value_error(text); }
[[noreturn]] void bad_type(const std::string& text) { throw py::type_error(text); }

std::string shape_text(at::IntArrayRef s) {
  std::string t = "(";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + (s.size() == 1 ? ",)" : ")");
}

// `t` is a CUDA tensor of `dtype` on `device`, of `shape` unless that is empty.
void want(const Tensor& t, const char* name, at::ScalarType dtype, at::Device device,
          at::IntArrayRef shape = {}) {
  if (!t.is_cuda()) bad_type(std::string(name) + " must be a CUDA tensor");
  if (t.scalar_type() != dtype)
    bad_type(std::string(name) + " must be " + toString(dtype) + ", got " +
             toString(t.scalar_type()));
  if (t.device() != device)
    bad_value(std::string(name) + " is on " + t.device().str() + ", expected " + device.str());
  if (!shape.empty() && t.sizes() != shape)
    bad_value(std::string(name) + " must have shape " + shape_text(shape) + ", got " +
              shape_text(t.sizes()));
}

// As `want`, for memory that is used as it lies.
void want_flat(const Tensor& t, const char* name, at::ScalarType dtype, at::Device device,
               at::IntArrayRef shape) {
  want(t, name, dtype, device, shape);
  if (!t.is_contiguous()) bad_value(std::string(name) + " must be contiguous");
}

// A non-zero status becomes the package's I4GError.
void check(const char* name, int status) {
  if (status == I4G_OK) return;
  py::module_::import("sm_120__gemm_b200").attr("_check")(name, status);
}

const void* ptr(const Tensor& t) { return t.const_data_ptr(); }
const void* ptr(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }

Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, at::Device device) {
  return Tensor(at::detail::empty_cuda(shape, dtype, device, std::nullopt));
}

// Contiguous tensor of 32-bit values inside `whole`, from its next free value on
// (`at`, moved past it to a multiple of 16 bytes).
Tensor part(const Tensor& whole, at::IntArrayRef shape, at::ScalarType dtype, int64_t& at) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(
      c10::Storage(whole.storage()), whole.key_set(), c10::scalarTypeToTypeMeta(dtype));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  at += (t.numel() + 3) / 4 * 4;
  return t;
}

int narrow(int64_t v, const char* name) {
  if (v < 0 || v > INT32_MAX) bad_value(std::string(name) + " is out of range");
  return static_cast<int>(v);
}

// A workspace of at least `need` bytes with zeroed arrival counters for a
// launch on the current stream (undefined for 0). Calls on one stream share a
// buffer: their order keeps it theirs alone. While the stream is being captured
// into a graph each call takes its own from the graph's memory and clears its
// counters in the graph, so graphs share nothing with each other or with eager
// calls.
constexpr int64_t kCounterBytes = 4096;

struct Held {
  std::mutex mutex;
  std::map<std::pair<int, cudaStream_t>, Tensor> of;  // by device and stream
};
Held& held() {
  static Held& h = *new Held;  // lives as long as the process
  return h;
}

// A launch that gave up on a wait leaves counters behind: every buffer is
// dropped (its memory stays its stream's), the next call makes a zeroed one.
void reset_workspaces() {
  std::lock_guard<std::mutex> lock(held().mutex);
  held().of.clear();
}

std::vector<Tensor> workspaces() {
  std::lock_guard<std::mutex> lock(held().mutex);
  std::vector<Tensor> all;
  for (const auto& entry : held().of) all.push_back(entry.second);
  return all;
}

Tensor workspace(size_t need, at::Device device, cudaStream_t stream) {
  if (need == 0) return Tensor();
  const int64_t bytes = static_cast<int64_t>(need);
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
    Tensor ws = empty({bytes}, at::kByte, device);
    ws.narrow(0, 0, kCounterBytes).zero_();
    return ws;
  }
  std::lock_guard<std::mutex> lock(held().mutex);
  Tensor& ws = held().of[{device.index(), stream}];
  if (!ws.defined() || ws.numel() < bytes) {
    ws = empty({bytes}, at::kByte, device);
    ws.narrow(0, 0, kCounterBytes).zero_();
  }
  return ws;
}

struct Launch {
  at::Device device;
  cudaStream_t stream;
  explicit Launch(const Tensor& t) : device(t.device()), stream(nullptr) {
    if (!t.is_cuda()) bad_type("a CUDA tensor is needed");
    stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  }
};

Tensor gemm_epilogue(const Tensor& a_in, const Tensor& tiles, const Tensor& scales, int64_t K,
                     int64_t N, int64_t group, const OptTensor& bias_in, int64_t activation,
                     bool gated, const OptTensor& residual_in, const OptTensor& out_in,
                     bool fp32_out) {
  const Launch on(tiles);
  want(scales, "scales", at::kHalf, on.device);
  want(a_in, "A", at::kHalf, on.device);
  if (a_in.dim() != 2 || a_in.size(1) != K)
    bad_value("A must be float16 [M, " + std::to_string(K) + "]");
  const Tensor a = a_in.contiguous();
  const int64_t M = a.size(0), cols = gated ? N / 2 : N;
  const auto dtype = fp32_out ? at::kFloat : at::kHalf;
  i4g_epilogue_t e{};
  OptTensor bias, residual;
  if (bias_in) {
    want(*bias_in, "bias", at::kHalf, on.device, {N});
    bias = bias_in->contiguous();
    e.bias = ptr(bias);
  }
  if (residual_in) {
    want(*residual_in, "residual", at::kHalf, on.device, {M, cols});
    const bool rows = residual_in->stride(1) == 1 && residual_in->stride(0) >= cols &&
                      residual_in->stride(0) <= INT32_MAX;
    residual = rows ? *residual_in : residual_in->contiguous();
    e.residual = ptr(residual);
    e.ld_residual = static_cast<int>(M > 1 ? residual->stride(0) : cols);
  }
  Tensor out;
  if (out_in) {
    want_flat(*out_in, "out", dtype, on.device, {M, cols});
    out = *out_in;
  } else {
    out = empty({M, cols}, dtype, on.device);
  }
  e.activation = static_cast<int>(activation);
  e.gated = gated;
  e.fp32_out = fp32_out;
  const int m = narrow(M, "M");
  size_t need = 0;
  check("i4g_gemm_epilogue_workspace_size",
        i4g_gemm_epilogue_workspace_size(m, static_cast<int>(N), static_cast<int>(K), &need));
  const Tensor ws = workspace(need, on.device, on.stream);
  check("i4g_gemm_epilogue",
        i4g_gemm_epilogue(ptr(a), tiles.const_data_ptr<uint8_t>(), ptr(scales),
                          out.mutable_data_ptr(), m, static_cast<int>(N), static_cast<int>(K),
                          static_cast<int>(group), &e, need ? ws.mutable_data_ptr() : nullptr,
                          need ? static_cast<size_t>(ws.numel()) : 0, on.stream));
  return out;
}

Tensor experts_gemm(const Tensor& a_in, const Tensor& tiles, const Tensor& scales, int64_t E,
                    int64_t K, int64_t N, int64_t group, const Tensor& offsets,
                    const Tensor& rows, const Tensor& slots, bool gather,
                    const OptTensor& bias_in, int64_t activation, bool gated,
                    const OptTensor& out_in, bool fp32_out) {
  const Launch on(tiles);
  want(scales, "scales", at::kHalf, on.device);
  want(a_in, "A", at::kHalf, on.device);
  if (slots.dim() != 2) bad_value("routing.slots must be [T, top_k]");
  const int64_t T = slots.size(0), top_k = slots.size(1), pairs = T * top_k;
  want_flat(offsets, "routing.offsets", at::kInt, on.device, {E + 1});
  want_flat(rows, "routing.rows", at::kInt, on.device, {pairs});
  const int64_t a_rows = gather ? T : pairs;
  if (a_in.dim() != 2 || a_in.size(0) != a_rows || a_in.size(1) != K)
    bad_value("A must be float16 [" + std::to_string(a_rows) + ", " + std::to_string(K) + "]");
  const Tensor a = a_in.contiguous();
  const int64_t cols = gated ? N / 2 : N;
  const auto dtype = fp32_out ? at::kFloat : at::kHalf;
  i4g_epilogue_t e{};
  OptTensor bias;
  if (bias_in) {
    want(*bias_in, "bias", at::kHalf, on.device, {E, N});
    bias = bias_in->contiguous();
    e.bias = ptr(bias);
  }
  e.activation = static_cast<int>(activation);
  e.gated = gated;
  e.fp32_out = fp32_out;
  Tensor out;
  if (out_in) {
    want_flat(*out_in, "out", dtype, on.device, {pairs, cols});
    out = *out_in;
  } else {
    out = empty({pairs, cols}, dtype, on.device);
  }
  const int p = narrow(pairs, "T * top_k");
  size_t need = 0, copy = 0;
  check("i4g_experts_workspace_parts",
        i4g_experts_workspace_parts(p, static_cast<int>(E), static_cast<int>(N),
                                    static_cast<int>(K), &need, &copy));
  const Tensor ws = workspace(need, on.device, on.stream);
  if (!gather) copy = 0;
  Tensor scratch;  // the copied rows are this call's alone
  if (copy) scratch = empty({static_cast<int64_t>(copy)}, at::kByte, on.device);
  check("i4g_experts_gemm_parts",
        i4g_experts_gemm_parts(ptr(a), static_cast<int>(a_rows), tiles.const_data_ptr<uint8_t>(),
                               ptr(scales), out.mutable_data_ptr(), offsets.const_data_ptr<int>(),
                               gather ? rows.const_data_ptr<int>() : nullptr,
                               static_cast<int>(top_k > 0 ? top_k : 1), p, static_cast<int>(E),
                               static_cast<int>(N), static_cast<int>(K), static_cast<int>(group),
                               &e, need ? ws.mutable_data_ptr() : nullptr,
                               need ? static_cast<size_t>(ws.numel()) : 0,
                               copy ? scratch.mutable_data_ptr() : nullptr, copy, on.stream));
  return out;
}

py::tuple route(const Tensor& logits_in, int64_t top_k, int64_t scoring, const OptTensor& bias_in,
                int64_t n_group, int64_t topk_group, int64_t group_score, bool renormalize,
                double scale) {
  const auto dtype = logits_in.scalar_type();
  if (!logits_in.is_cuda()) bad_type("logits must be a CUDA tensor");
  if (dtype != at::kFloat && dtype != at::kHalf)
    bad_type(std::string("logits must be float32 or float16, got ") + toString(dtype));
  if (logits_in.dim() != 2) bad_value("logits must be [T, E]");
  const Launch on(logits_in);
  const int64_t T = logits_in.size(0), E = logits_in.size(1);
  const bool rows_ok = logits_in.stride(1) == 1 && logits_in.stride(0) >= E &&
                       logits_in.stride(0) <= INT32_MAX;
  const Tensor logits = rows_ok ? logits_in : logits_in.contiguous();
  OptTensor bias;
  if (bias_in) {
    want(*bias_in, "bias", at::kFloat, on.device, {E});
    bias = bias_in->contiguous();
  }
  const int t = narrow(T, "T"), experts = narrow(E, "E"), k = narrow(top_k, "top_k");
  const int64_t pairs = T * k;
  size_t need = 0;
  check("i4g_route_workspace_size", i4g_route_workspace_size(t, experts, &need));
  // the five results in one allocation: one token's call 9.4 -> 7.3 us
  int64_t at = 0;
  const Tensor whole = empty({4 * ((pairs + 3) / 4 * 4) + (E + 4) / 4 * 4}, at::kInt, on.device);
  Tensor ids = part(whole, {T, k}, at::kInt, at);
  Tensor weights = part(whole, {T, k}, at::kFloat, at);
  Tensor offsets = part(whole, {E + 1}, at::kInt, at);
  Tensor rows = part(whole, {pairs}, at::kInt, at);
  Tensor slots = part(whole, {T, k}, at::kInt, at);
  Tensor ws;  // for the counts; nothing is kept in it
  if (need) ws = empty({static_cast<int64_t>(need)}, at::kByte, on.device);
  i4g_route_t o{static_cast<int>(scoring),     narrow(n_group, "n_group"),
                narrow(topk_group, "topk_group"), static_cast<int>(group_score), renormalize,
                static_cast<float>(scale)};
  check("i4g_route",
        i4g_route(ptr(logits), dtype == at::kFloat, static_cast<int>(T > 1 ? logits.stride(0) : E),
                  static_cast<const float*>(ptr(bias)), t, experts, k, &o,
                  ids.mutable_data_ptr<int>(), weights.mutable_data_ptr<float>(),
                  offsets.mutable_data_ptr<int>(), rows.mutable_data_ptr<int>(),
                  slots.mutable_data_ptr<int>(), need ? ws.mutable_data_ptr() : nullptr, need,
                  on.stream));
  return py::make_tuple(std::move(ids), std::move(weights), std::move(offsets), std::move(rows),
                        std::move(slots));
}

Tensor combine(const Tensor& y_in, const Tensor& slots, const Tensor& weights,
               const OptTensor& residual_in, const OptTensor& out_in) {
  if (!y_in.is_cuda()) bad_type("y must be a CUDA tensor");
  const Launch on(y_in);
  want(y_in, "y", at::kHalf, on.device);
  if (y_in.dim() != 2 || slots.dim() != 2) bad_value("y must be [rows, N], slots [T, top_k]");
  const int64_t T = slots.size(0), top_k = slots.size(1), N = y_in.size(1);
  want_flat(slots, "routing.slots", at::kInt, on.device, {T, top_k});
  want_flat(weights, "routing.weights", at::kFloat, on.device, {T, top_k});
  const Tensor y = y_in.contiguous();
  OptTensor residual;
  if (residual_in) {
    want(*residual_in, "residual", at::kHalf, on.device, {T, N});
    residual = residual_in->contiguous();
  }
  Tensor out;
  if (out_in) {
    want_flat(*out_in, "out", at::kHalf, on.device, {T, N});
    out = *out_in;
  } else {
    out = empty({T, N}, at::kHalf, on.device);
  }
  check("i4g_experts_combine",
        i4g_experts_combine(ptr(y), narrow(y.size(0), "rows of y"), slots.const_data_ptr<int>(),
                            weights.const_data_ptr<float>(), ptr(residual),
                            out.mutable_data_ptr(), narrow(T, "T"), narrow(top_k, "top_k"),
                            narrow(N, "N"), on.stream));
  return out;
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
  m.attr("torch_version") = std::string(TORCH_VERSION);
  m.def("gemm_epilogue", &gemm_epilogue);
  m.def("experts_gemm", &experts_gemm);
  m.def("route", &route);
  m.def("combine", &combine);
  m.def("reset_workspaces", &reset_workspaces);
  m.def("workspaces", &workspaces);
}
