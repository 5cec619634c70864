// Python-facing side of the few-token experts and of the adapters' projection: checks,
// allocation and the autograd node in C++, so that a call costs little more on the host
// than its launches (a decode step has kernels of a few microseconds), and a backward
// pass runs without the interpreter.  The work is done by the C ABI of
// libmoe_overlap_b200.so, whose entry points the package hands over (bind).
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/extension.h>

#include <cstdlib>
#include <cstring>
#include <memory>
#include <sstream>
#include <unordered_set>
#include <vector>

#include "../../include/moe_overlap.h"

namespace {

using at::Tensor;
namespace py = pybind11;

struct {
  decltype(&moe_few_tokens) few_tokens;
  decltype(&moe_few_tokens_workspace) few_tokens_workspace;
  decltype(&moe_lora_forward) lora_forward;
  decltype(&moe_lora_backward) lora_backward;
  decltype(&moe_lora_kept_bytes) lora_kept_bytes;
} abi;

constexpr int kMaxDevices = 64;
int32_t* status_words[kMaxDevices] = {};  // pinned host words that the kernels write

void bind(uintptr_t few_tokens, uintptr_t few_tokens_workspace, uintptr_t lora_forward,
          uintptr_t lora_backward, uintptr_t lora_kept_bytes) {
  abi = {reinterpret_cast<decltype(&moe_few_tokens)>(few_tokens),
         reinterpret_cast<decltype(&moe_few_tokens_workspace)>(few_tokens_workspace),
         reinterpret_cast<decltype(&moe_lora_forward)>(lora_forward),
         reinterpret_cast<decltype(&moe_lora_backward)>(lora_backward),
         reinterpret_cast<decltype(&moe_lora_kept_bytes)>(lora_kept_bytes)};
}

void set_status_word(int64_t device, uintptr_t address) {
  if (device >= 0 && device < kMaxDevices) status_words[device] = reinterpret_cast<int32_t*>(address);
}

template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw py::value_error(s.str());
}

py::object lib() { return py::module_::import("moe_overlap_b200._lib"); }

// The device's status word; raises what an earlier kernel has recorded there.  (Both
// functions take the GIL where they need it: a backward pass runs without.)
int32_t* checked_status(c10::Device device) {
  int32_t*& word = status_words[device.index()];
  if (word == nullptr) {
    const py::gil_scoped_acquire gil;
    lib().attr("status_word")(py::cast(device));
  }
  if (*static_cast<volatile int32_t*>(word) != MOE_OK) {
    const py::gil_scoped_acquire gil;
    lib().attr("check_status")(py::cast(device));
  }
  return word;
}

void check_call(int32_t code, const char* where, c10::Device device) {
  if (code != MOE_OK) {
    const py::gil_scoped_acquire gil;
    lib().attr("check_call")(code, where);
  }
  // MOE_B200_SYNC_CHECK=1: wait for the kernels and raise what they have recorded
  const char* env = std::getenv("MOE_B200_SYNC_CHECK");
  if (env != nullptr && *env != 0 && std::strcmp(env, "0") != 0) {
    const py::gil_scoped_acquire gil;
    lib().attr("check_status")(py::cast(device), true);
  }
}

void* stream_of(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

int32_t dtype_code(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? MOE_DTYPE_BF16 : t.scalar_type() == at::kHalf ? MOE_DTYPE_F16 : -1;
}

bool on_16_bytes(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }

// Unit-stride rows that start on 16 bytes; of several matrices, one behind another.
bool rows_ok(const Tensor& t) {
  const auto st = t.strides(), sz = t.sizes();
  const size_t d = sz.size();
  if (st[d - 1] != 1 || st[d - 2] % 8 != 0 || st[d - 2] < sz[d - 1] || !on_16_bytes(t)) return false;
  return d < 3 || sz[0] <= 1 || (st[0] % 8 == 0 && st[0] >= st[1] * sz[1]);
}
Tensor with_rows(const Tensor& t) { return rows_ok(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// For calls, or inputs of them, that pass no gradient on: refused rather than lost without
// a word.
bool wants_gradient(const Tensor& t) {
  return t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined());
}
void forward_only(const char* op, std::initializer_list<Tensor> inputs) {
  for (const Tensor& t : inputs)
    if (wants_gradient(t))
      refuse(op, " is forward only: detach the inputs that require a gradient, or call it under no_grad");
}
// Neither does a forward-mode tangent pass lora_linear.
void no_tangent(std::initializer_list<Tensor> inputs) {
  for (const Tensor& t : inputs)
    if (t.defined() && t._fw_grad(0).defined()) refuse("lora_linear has no forward-mode derivative");
}

void* data(const Tensor& t) { return const_cast<void*>(t.const_data_ptr()); }

// ------------------------------------------------------------ few tokens --
constexpr int64_t kMaxFewTokens = 128, kMaxWidth = int64_t(1) << 30;

void check_weights(const char* name, const Tensor& t, const Tensor& x) {
  if (t.device() != x.device() || t.scalar_type() != x.scalar_type())
    refuse(name, " must be a ", x.scalar_type(), " tensor on ", x.device());
  if (!rows_ok(t)) refuse(name, " needs unit-stride rows that start on 16 bytes, one matrix behind another");
}

Tensor few(const Tensor& x_in, const Tensor* router_w, const Tensor* router_bias, const Tensor& w1,
           const Tensor& w2, int64_t top_k, bool renormalize, const Tensor& idx, const Tensor& w,
           const std::optional<Tensor>& out_in) {
  const int64_t tokens = x_in.size(0), hidden = x_in.size(1), experts = w1.size(0), ffn = w1.size(1);
  check_weights("w1", w1, x_in);
  check_weights("w2", w2, x_in);
  const Tensor x = with_rows(x_in);
  Tensor out;
  if (out_in.has_value()) {
    out = *out_in;
    if (out.dim() != 2 || out.size(0) != tokens || out.size(1) != hidden) refuse("out must be [T, H]");
    check_weights("out", out, x);
    // what autograd has saved of it is not what it was
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
  } else {
    out = at::empty({tokens, hidden}, x.options());
  }
  const c10::Device dev = x.device();
  int32_t* status = checked_status(dev);
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const int64_t bytes = abi.few_tokens_workspace(tokens, hidden, ffn, experts, top_k);
  const Tensor ws = at::empty({bytes}, x.options().dtype(at::kByte));
  const int32_t rc = abi.few_tokens(
      data(x), x.stride(0), router_w != nullptr ? data(*router_w) : nullptr,
      router_w != nullptr ? router_w->stride(0) : 0,
      router_bias != nullptr ? static_cast<const float*>(data(*router_bias)) : nullptr, data(w1), w1.stride(0),
      w1.stride(1), data(w2), w2.stride(0), w2.stride(1), dtype_code(x), tokens, hidden, ffn, experts, top_k,
      renormalize, static_cast<int64_t*>(data(idx)), static_cast<float*>(data(w)), data(out), out.stride(0),
      data(ws), bytes, status, stream_of(dev));
  check_call(rc, "moe_few_tokens", dev);
  return out;
}

void check_few(const Tensor& x, const Tensor& w1, const Tensor& w2, int64_t top_k) {
  if (!x.is_cuda()) refuse("few-token experts need CUDA tensors");
  const char* shapes = "Shapes must be x [T, H], w1 [E, F, H], w2 [E, H, F].";
  if (x.dim() != 2 || w1.dim() != 3 || w2.dim() != 3) refuse(shapes);
  const int64_t hidden = x.size(1), experts = w1.size(0), ffn = w1.size(1);
  if (dtype_code(x) < 0) refuse("x must be bf16/fp16");
  if (w1.size(2) != hidden || w2.size(0) != experts || w2.size(1) != hidden || w2.size(2) != ffn) refuse(shapes);
  if (hidden % 8 != 0 || ffn % 8 != 0 || hidden == 0 || ffn == 0)
    refuse("hidden and ffn sizes must be multiples of 8");
  if (hidden > kMaxWidth || ffn > kMaxWidth) refuse("hidden and ffn sizes go up to 2^30");
  if (x.size(0) > kMaxFewTokens)
    refuse("at most ", kMaxFewTokens, " tokens: use MoELayer.forward for larger batches");
  if (top_k < 1 || top_k > 16 || top_k > experts || experts > 256)
    refuse("top_k must be in 1..min(16, E), and E at most 256");
}

std::tuple<Tensor, Tensor, Tensor> moe_few_tokens_op(const Tensor& x, const Tensor& router_w, const Tensor& w1,
                                                     const Tensor& w2, int64_t top_k,
                                                     const std::optional<Tensor>& router_bias, bool renormalize,
                                                     const std::optional<Tensor>& out) {
  forward_only("moe_few_tokens", {x, router_w, w1, w2, router_bias.value_or(Tensor()), out.value_or(Tensor())});
  if (router_w.dim() != 2 || w1.dim() != 3 || x.dim() < 1 || router_w.size(0) != w1.size(0) ||
      router_w.size(1) != x.size(-1))
    refuse("router_w must be [E, H]");
  check_few(x, w1, w2, top_k);
  check_weights("router_w", router_w, x);
  Tensor bias;
  if (router_bias.has_value()) {
    if (router_bias->dim() != 1 || router_bias->size(0) != router_w.size(0)) refuse("router bias must be [E]");
    bias = router_bias->to(x.device(), at::kFloat).contiguous();
  }
  const Tensor idx = at::empty({x.size(0), top_k}, x.options().dtype(at::kLong));
  const Tensor w = at::empty({x.size(0), top_k}, x.options().dtype(at::kFloat));
  Tensor y = few(x, &router_w, bias.defined() ? &bias : nullptr, w1, w2, top_k, renormalize, idx, w, out);
  return {y, idx, w};
}

Tensor experts_few_tokens_op(const Tensor& x, const Tensor& w1, const Tensor& w2, const Tensor& topk_idx,
                             const Tensor& topk_w, const std::optional<Tensor>& out) {
  forward_only("experts_few_tokens", {x, w1, w2, topk_w, out.value_or(Tensor())});
  if (topk_idx.dim() != 2 || x.dim() < 1 || topk_idx.size(0) != x.size(0) || topk_w.sizes() != topk_idx.sizes())
    refuse("topk_idx and topk_w must be [T, k]");
  if (topk_idx.device() != x.device() || topk_w.device() != x.device())
    refuse("topk_idx and topk_w must be on ", x.device());
  if (topk_idx.scalar_type() != at::kLong && topk_idx.scalar_type() != at::kInt)
    refuse("topk_idx must be int64 or int32");
  check_few(x, w1, w2, topk_idx.size(1));
  return few(x, nullptr, nullptr, w1, w2, topk_idx.size(1), false, topk_idx.to(at::kLong).contiguous(),
             topk_w.to(at::kFloat).contiguous(), out);
}

// ---------------------------------------------------------------- adapters --
struct Sizes {
  int64_t m, k, n, adapters, rank;
  Sizes(const Tensor& x, const Tensor& weight, const Tensor& a)
      : m(x.size(0)), k(x.size(1)), n(weight.size(0)), adapters(a.size(0)), rank(a.size(1)) {}
};

const float* scale_data(const Tensor& scale) {
  return scale.defined() ? static_cast<const float*>(data(scale)) : nullptr;
}

// y, and the buffer that the backward needs.  Holds the GIL (errors are Python's).
std::pair<Tensor, Tensor> lora_forward(const Tensor& x, const Tensor& weight, const Tensor& a, const Tensor& b,
                                       const Tensor& ids, const std::optional<Tensor>& scale,
                                       double scale_all, bool for_backward) {
  const Sizes z(x, weight, a);
  const c10::Device dev = x.device();
  int32_t* status = checked_status(dev);
  const c10::cuda::OptionalCUDAGuard guard(dev);
  Tensor y = at::empty({z.m, z.n}, x.options());
  Tensor kept = at::empty({abi.lora_kept_bytes(z.m, z.adapters, z.rank)},
                          x.options().dtype(at::kByte));
  const int32_t rc = abi.lora_forward(
      data(x), x.stride(0), data(weight), weight.stride(0), data(a), a.stride(0), a.stride(1), data(b),
      b.stride(0), b.stride(1), data(ids), ids.scalar_type() == at::kLong,
      scale_data(scale.value_or(Tensor())), static_cast<float>(scale_all), dtype_code(x), z.m, z.k, z.n, z.adapters, z.rank, for_backward, data(y),
      z.n, data(kept), status, stream_of(dev));
  check_call(rc, "moe_lora_forward", dev);
  return {y, kept};
}

// A leaf's gradient accumulator belongs to the stream that it was made on and lives as
// long as any graph of the leaf.  Under capture, one from another stream would pull that
// stream into the captured backward and break the capture in the autograd engine.
bool capturing() {
  return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
}
void refuse_foreign(torch::autograd::Node& accumulator) {
  const auto stream = accumulator.stream();
  if (!stream.has_value() || *stream == c10::cuda::getCurrentCUDAStream(stream->device_index()).unwrap()) return;
  // (the legacy stream is never captured, and may not be asked)
  const cudaStream_t raw = c10::cuda::CUDAStream(*stream).stream();
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (raw != nullptr && cudaStreamIsCapturing(raw, &status) == cudaSuccess && status == cudaStreamCaptureStatusActive)
    return;
  throw std::runtime_error(
      "lora_linear: a gradient accumulator of the captured step's inputs belongs to a stream outside the capture: "
      "a graph of the same leaves from before is alive, or something else (a hook, a data-parallel wrapper) holds "
      "the accumulator; drop it before capturing a training step");
}
// In the forward the inputs that are leaves, whatever the pass will ask for.
void refuse_foreign_graphs(const Tensor& leaf) {
  if (!leaf.requires_grad() || !leaf.is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (node != nullptr) refuse_foreign(*node);
}
// In the backward those that this pass will come to behind its inputs (adapters cast from
// the leaves that are trained).
void refuse_foreign_graphs_behind(const std::shared_ptr<torch::autograd::Node>& node) {
  const auto* run = torch::autograd::get_current_graph_task_exec_info();
  std::vector<torch::autograd::Node*> next{node.get()};
  std::unordered_set<torch::autograd::Node*> seen{node.get()};
  while (!next.empty()) {
    torch::autograd::Node* at = next.back();
    next.pop_back();
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(at) != nullptr) refuse_foreign(*at);
    for (const auto& edge : at->next_edges()) {
      torch::autograd::Node* to = edge.function.get();
      if (to == nullptr || !seen.insert(to).second) continue;
      if (run != nullptr && !run->empty()) {
        const auto it = run->find(to);
        if (it == run->end() || !it->second.should_execute()) continue;
      }
      next.push_back(to);
    }
  }
}

// x [M, K], a [L, r, K], b [L, N, r] -> y [M, N]; the weight, the ids and the scale get no
// gradient.
struct LoraLinear : torch::autograd::Function<LoraLinear> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const Tensor& a, const Tensor& b, const Tensor& ids,
                        const std::optional<Tensor>& scale, double scale_all) {
    auto [y, kept] = lora_forward(x, weight, a, b, ids, scale, scale_all, true);
    ctx->save_for_backward({x, weight, a, b, kept, scale.value_or(Tensor())});
    ctx->saved_data["scale"] = scale_all;
    return y;
  }

  // Runs in an autograd thread, without the GIL.
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "lora_linear can be differentiated once: its backward takes no create_graph");
    if (capturing()) refuse_foreign_graphs_behind(torch::autograd::get_current_node());
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &a = saved[2], &b = saved[3], &kept = saved[4],
                 &scale = saved[5];
    const Sizes z(x, weight, a);
    const Tensor dy = with_rows(grads[0]);
    const c10::Device dev = x.device();
    int32_t* status = checked_status(dev);
    const c10::cuda::OptionalCUDAGuard guard(dev);
    Tensor dx, da, db;
    if (ctx->needs_input_grad(0)) dx = at::empty({z.m, z.k}, x.options());
    if (ctx->needs_input_grad(2)) da = at::empty({z.adapters, z.rank, z.k}, x.options());
    if (ctx->needs_input_grad(3)) db = at::empty({z.adapters, z.n, z.rank}, x.options());
    const int32_t rc = abi.lora_backward(
        data(dy), dy.stride(0), data(x), x.stride(0), data(weight), weight.stride(0), data(a), a.stride(0),
        a.stride(1), data(b), b.stride(0), b.stride(1), scale_data(scale),
        static_cast<float>(ctx->saved_data["scale"].toDouble()), dtype_code(x), z.m, z.k, z.n, z.adapters,
        z.rank, data(kept), dx.defined() ? data(dx) : nullptr, z.k, da.defined() ? data(da) : nullptr,
        db.defined() ? data(db) : nullptr, status, stream_of(dev));
    check_call(rc, "moe_lora_backward", dev);
    return {dx, Tensor(), da, db, Tensor(), Tensor(), Tensor()};
  }
};

Tensor pad(const Tensor& t, int64_t last, int64_t before_last) {
  return last == 0 && before_last == 0 ? t : at::constant_pad_nd(t, {0, last, 0, before_last}, 0);
}

Tensor lora_linear_op(const Tensor& x, const Tensor& weight, const Tensor& lora_a, const Tensor& lora_b,
                      const Tensor& adapter_ids, const std::optional<Tensor>& scale_in, double scale_all) {
  no_tangent({x, weight, lora_a, lora_b, scale_in.value_or(Tensor())});
  if (!x.is_cuda()) refuse("lora_linear requires CUDA tensors.");
  const char* shapes = "Shapes must be x [M, K], weight [N, K], lora_a [L, r, K], lora_b [L, N, r].";
  if (x.dim() != 2 || weight.dim() != 2 || lora_a.dim() != 3 || lora_b.dim() != 3) refuse(shapes);
  const Sizes z(x, weight, lora_a);
  if (weight.size(1) != z.k || lora_a.size(2) != z.k || lora_b.size(0) != z.adapters || lora_b.size(1) != z.n ||
      lora_b.size(2) != z.rank)
    refuse(shapes);
  if (z.k == 0 || z.n == 0 || z.rank < 1 || z.rank > 128 || z.adapters < 1 || z.adapters > 1024)
    refuse("ranks go from 1 to 128, adapters from 1 to 1024, and K and N must not be 0");
  if (dtype_code(x) < 0) refuse("x dtype must be bf16/fp16.");
  auto like_x = [&](const char* name, const Tensor& t) {
    if (t.device() != x.device() || t.scalar_type() != x.scalar_type())
      refuse(name, " must be a ", x.scalar_type(), " tensor on ", x.device());
  };
  like_x("weight", weight);
  like_x("lora_a", lora_a);
  like_x("lora_b", lora_b);
  if (adapter_ids.dim() != 1 || adapter_ids.size(0) != z.m || adapter_ids.device() != x.device() ||
      (adapter_ids.scalar_type() != at::kInt && adapter_ids.scalar_type() != at::kLong))
    refuse("adapter_ids must be an int32 or int64 tensor [M] on ", x.device());
  const bool grad_mode = at::GradMode::is_enabled();
  if (grad_mode && weight.requires_grad())
    refuse("the shared weight is frozen: lora_linear gives it no gradient");
  std::optional<Tensor> scale;
  if (scale_in.has_value()) {
    if (scale_in->dim() != 1 || scale_in->size(0) != z.adapters || !scale_in->is_floating_point())
      refuse("scale must be a number or a float tensor [L]");
    if (grad_mode && scale_in->requires_grad()) refuse("lora_linear gives the scale no gradient");
    scale = scale_in->to(x.device(), at::kFloat).contiguous();
  }
  const int64_t pk = (8 - z.k % 8) % 8, pn = (8 - z.n % 8) % 8, pr = (8 - z.rank % 8) % 8;
  const Tensor xr = with_rows(pad(x, pk, 0)), wr = with_rows(pad(weight, pk, pn)),
               ar = with_rows(pad(lora_a, pk, pr)), br = with_rows(pad(lora_b, pr, pn)),
               ids = adapter_ids.contiguous();
  Tensor y;
  if (grad_mode && (x.requires_grad() || lora_a.requires_grad() || lora_b.requires_grad())) {
    if (capturing()) {
      refuse_foreign_graphs(x);
      refuse_foreign_graphs(lora_a);
      refuse_foreign_graphs(lora_b);
    }
    y = LoraLinear::apply(xr, wr, ar, br, ids, scale, scale_all);
  } else {
    y = lora_forward(xr, wr, ar, br, ids, scale, scale_all, false).first;
  }
  return pn == 0 ? y : y.slice(1, 0, z.n);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("set_status_word", &set_status_word);
  m.def("moe_few_tokens", &moe_few_tokens_op);
  m.def("experts_few_tokens", &experts_few_tokens_op);
  m.def("lora_linear", &lora_linear_op);
}
