// torch side of layer norm, rotary positions and attention to a shared prefix: checks of arguments, outputs and
// workspaces from torch's allocator, the current stream, and autograd nodes, around the C ABI of libnatten_b200.so.
//
// These operators take 3 to 60 microseconds on the device at everyday sizes.  Called through ctypes, with autograd
// functions in Python, a layer norm of one token took 11.5 us and a forward and backward pass 111 us on the host; an
// autograd node in C++ runs its backward without waiting for the interpreter.  The library is not linked: its symbols
// come from the handle that the package has loaded, so that there is one copy of its state.
#include <dlfcn.h>
#include <torch/csrc/autograd/edge.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <memory>
#include <mutex>
#include <vector>

#include "../../include/natten_b200.h"

namespace {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<at::Tensor> OptTensor;

struct Library {
  decltype(&natten_b200_last_error) last_error;
  decltype(&natten_b200_layer_norm_forward) layer_norm_forward;
  decltype(&natten_b200_layer_norm_backward) layer_norm_backward;
  decltype(&natten_b200_layer_norm_backward_scratch_bytes) layer_norm_scratch;
  decltype(&natten_b200_rotary) rotary;
  decltype(&natten_b200_prefix_scratch_bytes) prefix_scratch;
  decltype(&natten_b200_prefix_forward) prefix_forward;
} lib = {};

template <typename F>
void bind(void* handle, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(handle, name));
  TORCH_CHECK(f != nullptr, "libnatten_b200.so has no ", name);
}

void init(const std::string& path) {
  void* handle = dlopen(path.c_str(), RTLD_NOW | RTLD_NOLOAD);
  TORCH_CHECK(handle != nullptr, path, " is not loaded");
  bind(handle, "natten_b200_last_error", lib.last_error);
  bind(handle, "natten_b200_layer_norm_forward", lib.layer_norm_forward);
  bind(handle, "natten_b200_layer_norm_backward", lib.layer_norm_backward);
  bind(handle, "natten_b200_layer_norm_backward_scratch_bytes", lib.layer_norm_scratch);
  bind(handle, "natten_b200_rotary", lib.rotary);
  bind(handle, "natten_b200_prefix_scratch_bytes", lib.prefix_scratch);
  bind(handle, "natten_b200_prefix_forward", lib.prefix_forward);
}

// What the C ABI refuses is a ValueError, what fails at launch a RuntimeError.
void check(int rc) {
  if (rc == NATTEN_B200_OK) return;
  TORCH_CHECK_VALUE(rc != NATTEN_B200_EINVAL, lib.last_error());
  TORCH_CHECK(false, "natten_b200 error ", rc, ": ", lib.last_error());
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return NATTEN_B200_F32;
    case at::kHalf: return NATTEN_B200_F16;
    case at::kBFloat16: return NATTEN_B200_BF16;
    default: return -1;
  }
}

void check_cuda(const at::Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "natten_mlx_b200 runs on CUDA tensors only (there is no CPU path)");
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad(); }

// There are no formulas for forward-mode differentiation: a tangent is refused, not dropped.
template <typename... Tensors>
void check_no_tangent(const char* name, const Tensors&... ts) {
  const bool any = ((ts.defined() && ts._fw_grad(/*level=*/0).defined()) || ...);
  TORCH_CHECK(!any, name, " does not support forward-mode differentiation");
}

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Results of a backward pass that is recorded itself (create_graph): usable, but not to be differentiated again.
variable_list once(variable_list&& grads) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", (int)grads.size());
  for (auto& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  return (*error)(std::move(grads));
}

// The axes `n` of a tensor as few (size, stride) pairs, outermost first: axes of one step are joined, those of size 1
// dropped.  False when there are more than `most`.
struct Steps {
  int count = 0;
  int64_t size[2], stride[2];
};
bool join_axes(const at::Tensor& t, int64_t n, int most, Steps* s) {
  const auto sizes = t.sizes();
  const auto strides = t.strides();
  for (int64_t i = 0; i < n; ++i) {
    if (sizes[i] == 1) continue;
    if (s->count > 0 && s->stride[s->count - 1] == sizes[i] * strides[i]) {
      s->size[s->count - 1] *= sizes[i];
      s->stride[s->count - 1] = strides[i];
    } else {
      if (s->count == most) return false;
      s->size[s->count] = sizes[i];
      s->stride[s->count++] = strides[i];
    }
  }
  return true;
}

// ---------------------------------------------------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------------------------------------------------

// x itself when its rows follow one or two strides, else a dense copy.
at::Tensor norm_rows(const at::Tensor& x, natten_b200_rows* r) {
  const int64_t c = x.size(-1);
  *r = {};
  r->rows = x.numel() / c;
  r->channels = (int32_t)c;
  r->inner = 1;
  r->outer_stride = c;
  if (x.is_contiguous()) return x;
  Steps s;
  if ((x.stride(-1) == 1 || c == 1) && join_axes(x, x.dim() - 1, 2, &s)) {
    if (s.count > 0) r->outer_stride = s.stride[0];
    if (s.count == 2) {
      r->inner = s.size[1];
      r->inner_stride = s.stride[1];
    }
    return x;
  }
  return x.contiguous();
}

int weight_code(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b) {
  return dtype_code(w.defined() ? w : b.defined() ? b : x);
}

struct LayerNormBackward : public Node {
  SavedVariable x_, weight_, bias_;
  at::Tensor stats_;

  std::string name() const override { return "LayerNormB200Backward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    x_.reset_data();
    weight_.reset_data();
    bias_.reset_data();
    stats_.reset();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list out(3);
    at::Tensor x, weight, bias, stats;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      x = x_.unpack();
      weight = weight_.unpack();
      bias = bias_.unpack();
      stats = stats_;
    }
    if (!grads[0].defined()) return out;
    const bool want[3] = {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)};
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::cuda::CUDAGuard guard(x.device());
      const auto opts = x.options();
      if (want[0]) out[0] = at::empty(x.sizes(), opts);
      if (want[1]) out[1] = at::empty_like(weight);
      if (want[2]) out[2] = at::empty_like(bias);
      natten_b200_rows rows;
      const at::Tensor xr = norm_rows(x, &rows), grad = grads[0].contiguous();
      at::Tensor scratch;
      size_t bytes = 0;
      if (want[1] || want[2]) {
        bytes = lib.layer_norm_scratch(rows.rows, rows.channels);
        scratch = at::empty({(int64_t)bytes}, opts.dtype(at::kByte));
      }
      const float* mean = stats.data_ptr<float>();
      check(lib.layer_norm_backward(dtype_code(x), weight_code(x, weight, bias), &rows, ptr(xr), ptr(weight), mean, mean + rows.rows,
                                    ptr(grad), ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(scratch), bytes, stream_of(x)));
    }
    return once(std::move(out));
  }
};

void check_vector(const char* name, const at::Tensor& t, const at::Tensor& x) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(-1), name, " must have shape (", x.size(-1), ",), got ", t.sizes());
  TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, name,
                    " must have the input's dtype ", x.scalar_type(), " or float32, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " must be on the input's device ", x.device(), ", got ", t.device());
}

at::Tensor layer_norm(const at::Tensor& x, const OptTensor& weight_opt, const OptTensor& bias_opt, double eps) {
  const at::Tensor weight = weight_opt.value_or(at::Tensor()), bias = bias_opt.value_or(at::Tensor());
  check_no_tangent("layer_norm", x, weight, bias);
  check_cuda(x);
  TORCH_CHECK_VALUE(dtype_code(x) >= 0, "unsupported dtype ", x.scalar_type(), "; expected float32, float16 or bfloat16");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "layer_norm expects [..., C] with C >= 1, got ", x.sizes());
  TORCH_CHECK_VALUE(x.size(-1) <= INT32_MAX, "layer_norm expects fewer than 2^31 channels");
  TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(eps), "eps must be finite and not negative, got ", eps);
  if (weight.defined()) check_vector("weight", weight, x);
  if (bias.defined()) check_vector("bias", bias, x);
  TORCH_CHECK_VALUE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
                    "weight and bias must have one dtype");
  const bool record = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias));
  at::Tensor y, stats;
  // a backward reads the weights as they are laid out here
  const at::Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(x.device());
    natten_b200_rows rows;
    const at::Tensor xr = norm_rows(x, &rows);
    y = at::empty(x.sizes(), x.options());
    if (record) stats = at::empty({2, rows.rows}, x.options().dtype(at::kFloat));
    float* mean = record ? stats.data_ptr<float>() : nullptr;
    if (rows.rows > 0)
      check(lib.layer_norm_forward(dtype_code(x), weight_code(x, w, b), &rows, ptr(xr), ptr(w), ptr(b), (float)eps, ptr(y), mean,
                                   record ? mean + rows.rows : nullptr, stream_of(x)));
  }
  if (record) {
    std::shared_ptr<LayerNormBackward> node(new LayerNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    node->x_ = SavedVariable(x, false);
    node->weight_ = SavedVariable(w, false);
    node->bias_ = SavedVariable(b, false);
    node->stats_ = stats;
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---------------------------------------------------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------------------------------------------------

struct RotarySpec {
  std::vector<int32_t> axis_dims;
  std::vector<uint64_t> phases;
  bool interleaved;
};
typedef std::shared_ptr<RotarySpec> Spec;

// t itself when one stride leads through its tokens, else a dense copy.
at::Tensor token_rows(const at::Tensor& t, int64_t* token, int64_t* head) {
  const int64_t n = t.dim(), d = t.size(n - 1), heads = t.size(n - 2);
  *token = heads * d;
  *head = d;
  if (t.is_contiguous()) return t;
  Steps s;
  if ((t.stride(n - 1) == 1 || d == 1) && join_axes(t, n - 2, 1, &s)) {
    if (s.count > 0) *token = s.stride[0];
    if (heads > 1) *head = t.stride(n - 2);
    return t;
  }
  return t.contiguous();
}

struct Turn {
  Spec spec;
  std::vector<int64_t> origin;
  at::Tensor offsets, positions;    // at most one of them
};

std::pair<at::Tensor, at::Tensor> turn(const at::Tensor& q, const at::Tensor& k, const Turn& t, bool inverse) {
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
  if (q.numel() == 0) return {yq, yk};
  natten_b200_rotary_geom g = {};
  const at::Tensor qr = token_rows(q, &g.q_token_stride, &g.q_head_stride), kr = token_rows(k, &g.k_token_stride, &g.k_head_stride);
  g.dtype = dtype_code(q);
  g.rank = (int32_t)q.dim() - 3;
  g.batch = q.size(0);
  for (int i = 0; i < g.rank; ++i) {
    g.extent[i] = (int32_t)q.size(1 + i);
    g.origin[i] = t.origin.empty() ? 0 : t.origin[i];
  }
  g.heads_q = (int32_t)q.size(-2);
  g.heads_k = (int32_t)k.size(-2);
  g.head_dim = (int32_t)q.size(-1);
  g.n_axes = (int32_t)t.spec->axis_dims.size();
  for (int i = 0; i < g.n_axes; ++i) g.axis_dims[i] = t.spec->axis_dims[i];
  g.interleaved = t.spec->interleaved;
  const at::Tensor& pos = t.positions.defined() ? t.positions : t.offsets;
  g.position_kind = t.positions.defined() ? NATTEN_B200_POS_GIVEN : t.offsets.defined() ? NATTEN_B200_POS_OFFSET : NATTEN_B200_POS_GRID;
  g.position_bits = pos.defined() && pos.scalar_type() == at::kLong ? 64 : 32;
  g.position_batch = t.positions.defined() && t.positions.size(0) == q.size(0);
  g.positions = ptr(pos);
  g.phases = t.spec->phases.data();
  check(lib.rotary(&g, ptr(qr), ptr(kr), ptr(yq), ptr(yk), inverse, stream_of(q)));
  return {yq, yk};
}

// The gradient of a turn is the turn back, so only the positions are kept.
struct RotaryBackward : public Node {
  Spec spec_;
  std::vector<int64_t> origin_;
  SavedVariable offsets_, positions_;
  std::vector<int64_t> q_sizes_, k_sizes_;
  at::TensorOptions options_;

  std::string name() const override { return "RotaryB200Backward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    offsets_.reset_data();
    positions_.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    Turn t;
    t.spec = spec_;
    t.origin = origin_;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      t.offsets = offsets_.unpack();
      t.positions = positions_.unpack();
    }
    variable_list out(2);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const at::Tensor gq = grads[0].defined() ? grads[0] : at::zeros(q_sizes_, options_);
      const at::Tensor gk = grads[1].defined() ? grads[1] : at::zeros(k_sizes_, options_);
      std::tie(out[0], out[1]) = turn(gq, gk, t, true);
    }
    for (int i = 0; i < 2; ++i)
      if (!task_should_compute_output(i)) out[i].reset();
    return once(std::move(out));
  }
};

at::Tensor check_positions(const char* name, const at::Tensor& t, const at::Tensor& q) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be an int32 or int64 tensor, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == q.device(), name, " must be on the query's device ", q.device(), ", got ", t.device());
  return t.contiguous();
}

std::pair<at::Tensor, at::Tensor> rotary(const at::Tensor& q, const at::Tensor& k, const Spec& spec, const std::vector<int64_t>& origin,
                                         const OptTensor& offsets, const OptTensor& positions) {
  const int64_t nd = q.dim(), rank = nd - 3;
  TORCH_CHECK_VALUE(rank >= 1 && rank <= 3 && k.dim() == nd, "rotary expects query and key with one of the shapes "
                    "[B, L, heads, dim], [B, H, W, heads, dim], [B, D, H, W, heads, dim]");
  TORCH_CHECK_VALUE(q.sizes().slice(0, nd - 2) == k.sizes().slice(0, nd - 2), "Batch and spatial dimensions must match: Q=",
                    q.sizes(), ", K=", k.sizes(), ".");
  TORCH_CHECK_VALUE(q.size(-1) == k.size(-1), "Head dim must match: Q has ", q.size(-1), ", K has ", k.size(-1), ".");
  TORCH_CHECK_VALUE(dtype_code(q) >= 0 && q.scalar_type() == k.scalar_type(),
                    "query and key must share a dtype of float32, float16 or bfloat16, got ", q.scalar_type(), " and ", k.scalar_type());
  TORCH_CHECK_VALUE(q.size(-2) >= 1 && k.size(-2) >= 1, "query and key must have heads, got ", q.size(-2), " and ", k.size(-2));
  for (int64_t i = 1; i < nd; ++i)
    TORCH_CHECK_VALUE(q.size(i) <= INT32_MAX && k.size(i) <= INT32_MAX, "rotary expects sizes below 2^31, got ", q.sizes(), " and ", k.sizes());
  check_no_tangent("rotary", q, k);
  check_cuda(q);
  TORCH_CHECK_VALUE(k.device() == q.device(), "query and key must be on one device");
  const int64_t axes = (int64_t)spec->axis_dims.size();
  Turn t;
  t.spec = spec;
  t.origin = origin;
  if (positions.has_value()) {
    t.positions = check_positions("positions", *positions, q);
    const auto got = t.positions.sizes();
    bool ok = t.positions.dim() == rank + 2 && (got[0] == 1 || got[0] == q.size(0)) && got[rank + 1] == axes;
    for (int64_t i = 1; ok && i <= rank; ++i) ok = got[i] == q.size(i);
    TORCH_CHECK_VALUE(ok, "positions must have shape [", q.size(0), " or 1, the spatial sizes, ", axes, "], got ", got);
  } else {
    TORCH_CHECK_VALUE(axes == rank, "axis_dims must have an entry for each of the ", rank, " spatial axes, got ", axes);
    if (offsets.has_value()) {
      t.offsets = check_positions("offsets", *offsets, q);
      TORCH_CHECK_VALUE(t.offsets.dim() == 2 && t.offsets.size(0) == q.size(0) && t.offsets.size(1) == rank,
                        "offsets must have shape [", q.size(0), ", ", rank, "], got ", t.offsets.sizes());
    }
  }
  std::pair<at::Tensor, at::Tensor> y;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    y = turn(q, k, t, false);
  }
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k))) {
    std::shared_ptr<RotaryBackward> node(new RotaryBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q, k));
    node->spec_ = spec;
    node->origin_ = origin;
    node->offsets_ = SavedVariable(t.offsets, false);
    node->positions_ = SavedVariable(t.positions, false);
    node->q_sizes_ = q.sizes().vec();
    node->k_sizes_ = k.sizes().vec();
    node->options_ = q.options();
    torch::autograd::set_history(variable_list{y.first, y.second}, node);
  }
  return y;
}

// ---------------------------------------------------------------------------------------------------------------------
// attention to a shared prefix
// ---------------------------------------------------------------------------------------------------------------------

// As token_rows, but a dense copy unless the address and the strides are positive multiples of 16 bytes.
at::Tensor aligned_rows(const at::Tensor& t, int64_t* token, int64_t* head) {
  const at::Tensor r = token_rows(t, token, head);
  const int64_t step = 16 / r.element_size();
  const bool strides = r.is_contiguous() || (*token % step == 0 && *head % step == 0);
  if ((reinterpret_cast<uintptr_t>(r.data_ptr()) & 15) == 0 && *token > 0 && *head > 0 && strides) return r;
  *token = t.size(-2) * t.size(-1);
  *head = t.size(-1);
  return r.clone(at::MemoryFormat::Contiguous);
}

at::Tensor aligned_dense(const at::Tensor& t) {
  const at::Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0 ? c : c.clone(at::MemoryFormat::Contiguous);
}

std::pair<at::Tensor, at::Tensor> prefix(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, std::optional<double> scale,
                                         const OptTensor& lens_opt, const OptTensor& window_out, const OptTensor& window_lse, int path) {
  const int64_t nd = q.dim(), rank = nd - 3;
  TORCH_CHECK_VALUE(rank >= 1 && rank <= 3, "prefix_attention expects a query of shape [B, spatial..., heads, dim] with 1 to 3 spatial axes.");
  TORCH_CHECK_VALUE(k.dim() == 3 && v.dim() == 3, "prefix_keys/prefix_values must be 3D: [P, heads_kv, dim].");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "prefix_keys and prefix_values must have one shape, got ", k.sizes(), " and ", v.sizes(), ".");
  const int64_t heads = q.size(-2), d = q.size(-1);
  TORCH_CHECK_VALUE(k.size(2) == d, "Head dim must match: Q has ", d, ", the prefix has ", k.size(2), ".");
  TORCH_CHECK_VALUE(d >= 1 && d <= 256, "prefix_attention takes head dims from 1 to 256, got ", d, ".");
  TORCH_CHECK_VALUE(k.size(1) >= 1 && heads >= 1 && heads % k.size(1) == 0, "heads_q (", heads, ") must be divisible by heads_kv (", k.size(1), ").");
  TORCH_CHECK_VALUE(dtype_code(q) >= 0 && q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
                    "query, prefix_keys and prefix_values must share a dtype of float32, float16 or bfloat16.");
  TORCH_CHECK_VALUE(window_out.has_value() == window_lse.has_value(), "window must be (output, lse).");
  bool grad = wants_grad(q) || wants_grad(k) || wants_grad(v);
  if (window_out.has_value()) {
    TORCH_CHECK_VALUE(window_out->sizes() == q.sizes() && window_lse->sizes() == q.sizes().slice(0, nd - 1), "window must have the shapes ",
                      q.sizes(), " and ", q.sizes().slice(0, nd - 1), ", got ", window_out->sizes(), " and ", window_lse->sizes(), ".");
    TORCH_CHECK_VALUE(window_out->scalar_type() == q.scalar_type(), "the window's output must have the query's dtype ", q.scalar_type(),
                      ", got ", window_out->scalar_type(), ".");
    grad = grad || wants_grad(*window_out) || wants_grad(*window_lse);
  }
  TORCH_CHECK_VALUE(!scale.has_value() || (*scale > 0.0 && std::isfinite(*scale)), "scale must be positive and finite, got ", scale.value_or(0.0), ".");
  check_no_tangent("prefix_attention", q, k, v, window_out.value_or(at::Tensor()), window_lse.value_or(at::Tensor()));
  TORCH_CHECK(!(at::GradMode::is_enabled() && grad),
              "prefix_attention computes no gradients: call it under torch.no_grad(), or detach its inputs");
  check_cuda(q);
  TORCH_CHECK_VALUE(k.device() == q.device() && v.device() == q.device() &&
                    (!window_out.has_value() || (window_out->device() == q.device() && window_lse->device() == q.device())),
                    "all tensors must be on one device");
  const at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor lens;
  if (lens_opt.has_value()) {
    lens = *lens_opt;
    TORCH_CHECK_VALUE(lens.scalar_type() == at::kInt || lens.scalar_type() == at::kLong, "prefix_lens must be an int32 or int64 tensor.");
    TORCH_CHECK_VALUE(lens.dim() == 1 && lens.size(0) == q.size(0), "prefix_lens must have shape (", q.size(0), ",), got ", lens.sizes(), ".");
    TORCH_CHECK_VALUE(lens.device() == q.device(), "prefix_lens must be on the query's device");
    lens = lens.scalar_type() == at::kInt ? lens.contiguous() : lens.clamp(0, k.size(0)).to(at::kInt).contiguous();
  }
  at::Tensor out = at::empty(q.sizes(), q.options()), lse = at::empty(q.sizes().slice(0, nd - 1), q.options().dtype(at::kFloat));
  if (q.numel() == 0) return {out, lse};
  natten_b200_prefix_geom g = {};
  const at::Tensor qr = aligned_rows(q, &g.q_token_stride, &g.q_head_stride), kr = aligned_rows(k, &g.k_token_stride, &g.k_head_stride),
                   vr = aligned_rows(v, &g.v_token_stride, &g.v_head_stride);
  at::Tensor wo, wl;
  if (window_out.has_value()) {
    wo = aligned_dense(*window_out);
    wl = window_lse->to(at::kFloat).contiguous();
  }
  g.dtype = dtype_code(q);
  TORCH_CHECK_VALUE(heads <= INT32_MAX, "too many heads");
  g.heads_q = (int32_t)heads;
  g.heads_kv = (int32_t)k.size(1);
  g.head_dim = (int32_t)d;
  g.batch = q.size(0);
  g.tokens = q.numel() / (g.batch * heads * d);
  g.prefix = k.size(0);
  g.scale = scale.has_value() ? (float)*scale : (float)(1.0 / std::sqrt((double)d));
  g.path = path;
  g.lens = static_cast<const int32_t*>(ptr(lens));
  const size_t bytes = lib.prefix_scratch(&g);
  at::Tensor scratch;
  if (bytes > 0) scratch = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check(lib.prefix_forward(&g, ptr(qr), ptr(kr), ptr(vr), ptr(wo), static_cast<const float*>(ptr(wl)), ptr(out), lse.data_ptr<float>(),
                           ptr(scratch), bytes, stream_of(q)));
  return {out, lse};
}

}  // namespace

PYBIND11_MODULE(_torch_binding, m) {
  m.def("init", &init);
  m.def("layer_norm", &layer_norm);
  py::class_<RotarySpec, Spec>(m, "RotarySpec")
      .def(py::init([](std::vector<int32_t> dims, std::vector<uint64_t> phases, bool interleaved) {
        auto s = std::make_shared<RotarySpec>();
        s->axis_dims = std::move(dims);
        s->phases = std::move(phases);
        s->interleaved = interleaved;
        int64_t sum = 0;
        for (int32_t d : s->axis_dims) sum += d;
        TORCH_CHECK_VALUE(s->axis_dims.size() >= 1 && s->axis_dims.size() <= 3 && sum == 2 * (int64_t)s->phases.size(),
                          "a phase for each pair of channels, 1 to 3 axes");
        return s;
      }))
      .def_readonly("phases", &RotarySpec::phases);
  m.def("rotary", &rotary);
  m.def("prefix", &prefix);
}
