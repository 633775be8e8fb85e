// The group norm and the 8-bit activation checkpoints as PyTorch operators (their schemas and fake
// implementations are in spio_b200/functional).
//
// In C++ because of what a call costs on the host: a Python operator takes 20 to 50 us in eager mode and about
// 200 us with its backward pass, many times what the kernels of a small tensor take; these take 5 to 10.
// The device work is that of the C ABI (include/spio_b200.h), on torch's current stream.
#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/spio_b200.h"

namespace {

using at::Tensor;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return SPIO_TYPE_F16;
    case at::kBFloat16: return SPIO_TYPE_BF16;
    case at::kFloat: return SPIO_TYPE_F32;
    default: TORCH_CHECK_VALUE(false, "expected float16, bfloat16 or float32, got ", t);
  }
}

constexpr int kActivations = 4;
constexpr c10::string_view kActivationNames[kActivations] = {"none", "relu", "silu", "gelu"};  // by SPIO_ACT_*

int activation_code(c10::string_view name) {
  for (int i = 0; i < kActivations; ++i)
    if (name == kActivationNames[i]) return i;
  TORCH_CHECK_VALUE(false, "activation must be one of none, relu, silu, gelu, got ", std::string(name));
}

void check_call(int rc, const char* what) {
  TORCH_CHECK_VALUE(rc == 0, spio_b200_last_error(), " [", what, "]");
}

void check_image(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda(), "spio ", what, " runs on CUDA devices only (no CPU implementation)");
  TORCH_CHECK_VALUE(t.dim() == 4, "spio ", what, ": expected an NCHW tensor");
}

// `t` in channels_last order at a 16-byte boundary (itself if it is already).
Tensor kernel_layout(const Tensor& t) {
  const Tensor c = t.contiguous(at::MemoryFormat::ChannelsLast);
  if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0) return c;
  return c.clone(at::MemoryFormat::ChannelsLast);
}

// Allocated without the dispatcher: these calls are below it, and a backward pass allocates four tensors.
Tensor empty(at::IntArrayRef size, const Tensor& like, at::ScalarType type, at::MemoryFormat format = at::MemoryFormat::Contiguous) {
  return Tensor(at::detail::empty_cuda(size, type, like.device(), format));
}
Tensor empty_image(at::IntArrayRef size, const Tensor& like, at::ScalarType type) {
  return empty(size, like, type, at::MemoryFormat::ChannelsLast);
}
Tensor empty_vector(int64_t n, const Tensor& like, at::ScalarType type) { return empty({n}, like, type); }

void* pointer(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return static_cast<float*>(pointer(t)); }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

std::tuple<Tensor, Tensor> empty_codes(const Tensor& x) {
  return {empty_image(x.sizes(), x, at::kChar), empty_image({x.size(0), x.size(1) / 8, x.size(2), x.size(3)}, x, at::kByte)};
}

// ---------------------------------------------------------------- 8-bit checkpoints

std::tuple<Tensor, Tensor> checkpoint8_pack(const Tensor& x_) {
  check_image(x_, "checkpoint8_pack");
  const int type = type_code(x_.scalar_type());
  TORCH_CHECK_VALUE(x_.size(1) % 8 == 0, "Number of channels must be a multiple of 8.");
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = kernel_layout(x_);
  auto [codes, exponents] = empty_codes(x);
  check_call(spio_checkpoint8_pack(pointer(codes), pointer(exponents), pointer(x), x.numel() / 8, type, stream()),
             "checkpoint8_pack");
  return {codes, exponents};
}

Tensor checkpoint8_unpack(const Tensor& codes_, const Tensor& exponents_, at::ScalarType dtype) {
  check_image(codes_, "checkpoint8_unpack");
  const int type = type_code(dtype);
  const int64_t n = codes_.size(0), c = codes_.size(1), h = codes_.size(2), w = codes_.size(3);
  TORCH_CHECK_VALUE(codes_.scalar_type() == at::kChar && exponents_.scalar_type() == at::kByte,
                    "codes are int8 and exponents uint8");
  TORCH_CHECK_VALUE(exponents_.device() == codes_.device(), "codes and exponents must be on one device");
  TORCH_CHECK_VALUE(c % 8 == 0 && exponents_.sizes() == at::IntArrayRef({n, c / 8, h, w}),
                    "exponents must be (n, c / 8, h, w)");
  const c10::cuda::CUDAGuard guard(codes_.device());
  const Tensor codes = kernel_layout(codes_), exponents = kernel_layout(exponents_);
  const Tensor x = empty_image(codes.sizes(), codes, dtype);
  check_call(spio_checkpoint8_unpack(pointer(x), pointer(codes), pointer(exponents), x.numel() / 8, type, stream()),
             "checkpoint8_unpack");
  return x;
}

// ---------------------------------------------------------------- group norm

// (No sizes: these may be symbolic while a call is traced.)
void check_parameter_types(const Tensor& x, const OptTensor& weight, const OptTensor& bias) {
  const auto both = [&](at::ScalarType type) {
    return (!weight.has_value() || weight->scalar_type() == type) && (!bias.has_value() || bias->scalar_type() == type);
  };
  TORCH_CHECK_VALUE(both(at::kFloat) || both(x.scalar_type()), "weight and bias are both fp32 or both of the data's type");
}

spio_groupnorm_2d_desc describe(const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t num_groups,
                                double eps, c10::string_view activation) {
  check_image(x, "groupnorm_2d");
  const int64_t c = x.size(1);
  TORCH_CHECK_VALUE(c > 0 && c % 8 == 0, "Number of channels must be a multiple of 8.");
  TORCH_CHECK_VALUE(num_groups > 0 && c % num_groups == 0, "Number of channels must be divisible by the number of groups.");
  TORCH_CHECK_VALUE(c <= (1 << 20), "GroupNorm2d supports at most 2^20 channels");
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative");
  check_parameter_types(x, weight, bias);
  for (const OptTensor* t : {&weight, &bias})
    TORCH_CHECK_VALUE(!t->has_value() || ((*t)->dim() == 1 && (*t)->numel() == c && (*t)->device() == x.device()),
                      "weight and bias are vectors of the channels on the data's device");
  spio_groupnorm_2d_desc d;
  d.n = x.size(0);
  d.pixels = x.size(2) * x.size(3);
  d.c = (int)c;
  d.groups = (int)num_groups;
  d.type = type_code(x.scalar_type());
  d.activation = activation_code(activation);
  d.eps = (float)eps;
  return d;
}

// In fp32, as the kernels take them (a 16-bit vector is exact in it).
OptTensor fp32(const OptTensor& t) { return t.has_value() ? OptTensor(t->to(at::kFloat)) : std::nullopt; }
Tensor vector_of(const OptTensor& t) { return t.has_value() ? t->to(at::kFloat).contiguous() : Tensor(); }

Tensor scratch_of(size_t bytes, const Tensor& like) {
  return bytes > 0 ? empty_vector((int64_t)bytes, like, at::kByte) : Tensor();
}

// y; stats, codes and exponents where wanted
std::tuple<Tensor, Tensor, Tensor, Tensor> forward(const Tensor& x_, const OptTensor& weight_, const OptTensor& bias_,
                                                   int64_t num_groups, double eps, c10::string_view activation,
                                                   bool want_stats, bool want_codes) {
  const spio_groupnorm_2d_desc desc = describe(x_, weight_, bias_, num_groups, eps, activation);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = kernel_layout(x_), weight = vector_of(weight_), bias = vector_of(bias_);
  const Tensor y = empty_image(x.sizes(), x, x.scalar_type());
  Tensor stats, codes, exponents;
  if (want_stats) stats = empty({x.size(0), num_groups, 2}, x, at::kFloat);
  if (want_codes) std::tie(codes, exponents) = empty_codes(x);
  const size_t bytes = spio_groupnorm_2d_fwd_scratch_bytes(&desc);
  const Tensor scratch = scratch_of(bytes, x);
  check_call(spio_groupnorm_2d_fwd(pointer(y), floats(stats), pointer(codes), pointer(exponents), pointer(x), floats(weight),
                                   floats(bias), &desc, pointer(scratch), bytes, stream()),
             "groupnorm_2d");
  return {y, stats, codes, exponents};
}

Tensor groupnorm_2d(const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t num_groups, double eps,
                    c10::string_view activation, bool) {
  return std::get<0>(forward(x, weight, bias, num_groups, eps, activation, false, false));
}

std::tuple<Tensor, Tensor, Tensor, Tensor> groupnorm_2d_forward(const Tensor& x, const OptTensor& weight,
                                                                const OptTensor& bias, int64_t num_groups, double eps,
                                                                c10::string_view activation, bool checkpoint8) {
  auto r = forward(x, weight, bias, num_groups, eps, activation, true, checkpoint8);
  if (!checkpoint8) {
    std::get<2>(r) = empty_vector(0, x, at::kChar);
    std::get<3>(r) = empty_vector(0, x, at::kByte);
  }
  return r;
}

std::tuple<Tensor, Tensor, Tensor> groupnorm_2d_backward(const Tensor& dy_, const OptTensor& x_, const OptTensor& codes_,
                                                         const OptTensor& exponents_, const Tensor& stats_,
                                                         const OptTensor& weight_, const OptTensor& bias_,
                                                         int64_t num_groups, c10::string_view activation,
                                                         bool needs_input_grad, bool needs_weight_grad,
                                                         bool needs_bias_grad) {
  const spio_groupnorm_2d_desc desc = describe(dy_, weight_, bias_, num_groups, 0., activation);
  const int64_t n = dy_.size(0), c = dy_.size(1);
  const c10::cuda::CUDAGuard guard(dy_.device());
  Tensor x, codes, exponents;
  if (x_.has_value()) {
    TORCH_CHECK_VALUE(x_->scalar_type() == dy_.scalar_type() && x_->sizes() == dy_.sizes() && x_->device() == dy_.device(),
                      "x must have the type, the size and the device of grad_output");
    x = kernel_layout(*x_);
  } else {
    TORCH_CHECK_VALUE(codes_.has_value() && exponents_.has_value(), "backward needs x or its 8-bit form");
    TORCH_CHECK_VALUE(codes_->scalar_type() == at::kChar && codes_->sizes() == dy_.sizes() && codes_->device() == dy_.device(),
                      "codes must be int8, of the size and on the device of grad_output");
    TORCH_CHECK_VALUE(exponents_->scalar_type() == at::kByte && exponents_->device() == dy_.device() &&
                          exponents_->sizes() == at::IntArrayRef({n, c / 8, dy_.size(2), dy_.size(3)}),
                      "exponents must be uint8 (n, c / 8, h, w) on the device of grad_output");
    codes = kernel_layout(*codes_), exponents = kernel_layout(*exponents_);
  }
  TORCH_CHECK_VALUE(stats_.scalar_type() == at::kFloat && stats_.sizes() == at::IntArrayRef({n, num_groups, 2}) &&
                        stats_.device() == dy_.device(),
                    "stats must be fp32 (n, groups, 2) on the device of grad_output");
  const Tensor dy = kernel_layout(dy_), weight = vector_of(weight_), bias = vector_of(bias_);
  Tensor stats = stats_.contiguous();
  if (reinterpret_cast<uintptr_t>(stats.data_ptr()) % 8 != 0) stats = stats.clone();
  const Tensor dx = needs_input_grad ? empty_image(dy.sizes(), dy, dy.scalar_type()) : empty_vector(0, dy, dy.scalar_type());
  const Tensor dw = empty_vector(needs_weight_grad ? c : 0, dy, at::kFloat);
  const Tensor db = empty_vector(needs_bias_grad ? c : 0, dy, at::kFloat);
  const size_t bytes = spio_groupnorm_2d_bwd_scratch_bytes(&desc);
  const Tensor scratch = scratch_of(bytes, dy);
  check_call(spio_groupnorm_2d_bwd(pointer(dx), floats(dw), floats(db), pointer(dy), pointer(x), pointer(codes),
                                   pointer(exponents), floats(stats), floats(weight), floats(bias), &desc,
                                   pointer(scratch), bytes, stream()),
             "groupnorm_2d backward");
  return {dx, dw, db};
}

// ---------------------------------------------------------------- autograd

auto forward_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("spio::groupnorm_2d_forward", "")
                             .typed<decltype(groupnorm_2d_forward)>();
  return op;
}
auto backward_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("spio::groupnorm_2d_backward", "")
                             .typed<decltype(groupnorm_2d_backward)>();
  return op;
}
auto infer_op() {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("spio::groupnorm_2d", "").typed<decltype(groupnorm_2d)>();
  return op;
}

OptTensor optional_of(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
Tensor tensor_of(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

// Forward-mode derivatives: refused, or the result would seem constant.
void check_no_tangent(const Tensor& t, const char* what = "groupnorm_2d") {
  TORCH_CHECK(!t._fw_grad(0).defined(), "spio ", what, " has no forward-mode derivative");
}
void check_no_tangent(const OptTensor& t) {
  if (t.has_value()) check_no_tangent(*t);
}

// The backward operator refuses a derivative of its own instead of returning values that seem constant.  `origin`: a
// tensor at the place in the graph of what the gradients depend on besides.
struct GroupNormBackward : torch::autograd::Function<GroupNormBackward> {
  static variable_list forward(torch::autograd::AutogradContext*, const Tensor& dy, const OptTensor& x,
                               const OptTensor& codes, const OptTensor& exponents, const Tensor& stats,
                               const OptTensor& weight, const OptTensor& bias,
                               int64_t num_groups, std::string activation, bool needs_input_grad,
                               bool needs_weight_grad, bool needs_bias_grad, const OptTensor&) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dx, dw, db] = backward_op().call(dy, x, codes, exponents, stats, weight, bias, num_groups, activation,
                                           needs_input_grad, needs_weight_grad, needs_bias_grad);
    return {dx, dw, db};
  }
  static variable_list backward(torch::autograd::AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "spio groupnorm_2d cannot be differentiated twice");
  }
};

// An empty tensor at the place in the graph of the first input of the backward node that is running (where that requires
// a gradient).
OptTensor origin_of_input() {
  const auto node = torch::autograd::get_current_node();
  TORCH_CHECK(node, "spio groupnorm_2d cannot be differentiated twice");
  const torch::autograd::Edge edge = node->next_edge(0);
  if (!edge.is_valid()) return std::nullopt;
  const Tensor t = at::empty({0});
  torch::autograd::impl::set_gradient_edge(t, edge);
  return t;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& weight,
                        const OptTensor& bias, int64_t num_groups, double eps, std::string activation, bool checkpoint8) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, stats, codes, exponents] = forward_op().call(x, weight, bias, num_groups, eps, activation, checkpoint8);
    if (checkpoint8)
      ctx->save_for_backward({Tensor(), codes, exponents, stats, tensor_of(weight), tensor_of(bias)});
    else
      ctx->save_for_backward({x, Tensor(), Tensor(), stats, tensor_of(weight), tensor_of(bias)});
    ctx->saved_data["call"] = num_groups * kActivations + activation_code(activation);
    return y;
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list result(7);
    if (!grads[0].defined()) return result;
    check_no_tangent(grads[0]);
    // (an absent weight or bias has no edge in the graph)
    size_t edge = 0;
    const bool want_x = ctx->needs_input_grad(edge++);
    const bool want_weight = saved[4].defined() && ctx->needs_input_grad(edge++);
    const bool want_bias = saved[5].defined() && ctx->needs_input_grad(edge++);
    const bool want[3] = {want_x, want_weight, want_bias};
    const int64_t call = ctx->saved_data["call"].toInt();
    if (at::GradMode::is_enabled()) {  // a derivative of the gradients may be asked for, which the node refuses;
      // the 8-bit form of x is no part of the graph, x itself is
      const variable_list r = GroupNormBackward::apply(
          grads[0], optional_of(saved[0]), optional_of(saved[1]), optional_of(saved[2]), saved[3], optional_of(saved[4]),
          optional_of(saved[5]), call / kActivations, std::string(kActivationNames[call % kActivations]), want[0], want[1],
          want[2], saved[1].defined() ? origin_of_input() : std::nullopt);
      for (int i = 0; i < 3; ++i)
        if (want[i]) result[i] = r[i];
      return result;
    }
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dx, dw, db] = backward_op().call(
        grads[0], optional_of(saved[0]), optional_of(saved[1]), optional_of(saved[2]), saved[3], optional_of(saved[4]),
        optional_of(saved[5]), call / kActivations, kActivationNames[call % kActivations], want[0], want[1], want[2]);
    if (want[0]) result[0] = dx;
    if (want[1]) result[1] = dw;
    if (want[2]) result[2] = db;
    return result;
  }
};

bool requires_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }

Tensor groupnorm_2d_autograd(const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t num_groups,
                             double eps, c10::string_view activation, bool checkpoint8) {
  check_no_tangent(x), check_no_tangent(weight), check_no_tangent(bias);
  if (at::GradMode::is_enabled() && (x.requires_grad() || requires_grad(weight) || requires_grad(bias))) {
    check_parameter_types(x, weight, bias);
    // 16-bit parameters: their gradients are rounded to their type once, by the derivative of this conversion
    return GroupNorm::apply(x, fp32(weight), fp32(bias), num_groups, eps, std::string(activation), checkpoint8);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return infer_op().call(x, weight, bias, num_groups, eps, activation, checkpoint8);
}

std::tuple<Tensor, Tensor, Tensor> groupnorm_2d_backward_autograd(
    const Tensor& dy, const OptTensor& x, const OptTensor& codes, const OptTensor& exponents, const Tensor& stats,
    const OptTensor& weight, const OptTensor& bias, int64_t num_groups, c10::string_view activation,
    bool needs_input_grad, bool needs_weight_grad, bool needs_bias_grad) {
  check_no_tangent(dy), check_no_tangent(x), check_no_tangent(weight), check_no_tangent(bias);
  if (at::GradMode::is_enabled() && (dy.requires_grad() || requires_grad(x) || requires_grad(weight) || requires_grad(bias))) {
    const variable_list r =
        GroupNormBackward::apply(dy, x, codes, exponents, stats, weight, bias, num_groups, std::string(activation),
                                 needs_input_grad, needs_weight_grad, needs_bias_grad, std::nullopt);
    return {r[0], r[1], r[2]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return backward_op().call(dy, x, codes, exponents, stats, weight, bias, num_groups, activation, needs_input_grad,
                            needs_weight_grad, needs_bias_grad);
}

// ---------------------------------------------------------------- autocast

// The data keeps its type; weight and bias are taken in fp32.
Tensor groupnorm_2d_autocast(const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t num_groups,
                             double eps, c10::string_view activation, bool checkpoint8) {
  const c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::AutocastCUDA);
  return infer_op().call(x, fp32(weight), fp32(bias), num_groups, eps, activation, checkpoint8);
}

// ---------------------------------------------------------------- convolution with an 8-bit checkpoint
//
// The eager form of spio::conv2d_gw8_checkpoint8 for kernels built into the library.  `tunes` holds the tile
// configurations (spio_gw8_tune) of the forward, input-gradient and weight-gradient kernels, which the
// package's kernel factories have chosen for these sizes.

struct Conv {
  spio_gw8_shape shape;
  spio_gw8_tune fprop, dgrad, wgrad;
};

constexpr size_t kTunes = 3 * sizeof(spio_gw8_tune) / sizeof(int);

Conv conv_of(at::IntArrayRef size, const Tensor& weight, int64_t pad_y, int64_t pad_x, at::IntArrayRef tunes) {
  TORCH_CHECK_VALUE(tunes.size() == kTunes, "three tile configurations expected");
  Conv c;
  c.shape = {(int)size[0], (int)size[1], (int)size[2], (int)size[3], (int)weight.size(2), (int)weight.size(3),
             (int)pad_y, (int)pad_x};
  spio_gw8_tune* tune[3] = {&c.fprop, &c.dgrad, &c.wgrad};
  for (size_t i = 0; i < kTunes; ++i) reinterpret_cast<int*>(tune[i / (kTunes / 3)])[i % (kTunes / 3)] = (int)tunes[i];
  return c;
}

Conv checked_conv(const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t pad_y, int64_t pad_x,
                  at::IntArrayRef tunes) {
  check_image(x, "conv2d_gw8_checkpoint8");
  TORCH_CHECK_VALUE(x.scalar_type() == at::kHalf && weight.scalar_type() == at::kHalf && weight.dim() == 4,
                    "conv2d_gw8 takes float16 data and weights");
  TORCH_CHECK_VALUE(weight.size(0) == x.size(1) && weight.size(1) == 8, "weight must be (c, 8, r, s)");
  TORCH_CHECK_VALUE(weight.device() == x.device(), "weight must be on the data's device");
  TORCH_CHECK_VALUE(!bias.has_value() || (bias->scalar_type() == at::kFloat && bias->dim() == 1 &&
                                          bias->size(0) == x.size(1) && bias->device() == x.device()),
                    "bias must be an fp32 vector of the channels on the data's device");
  return conv_of(x.sizes(), weight, pad_y, pad_x, tunes);
}

Tensor conv_forward(const Conv& c, const Tensor& x, const Tensor& weight, const OptTensor& bias_) {
  const c10::cuda::CUDAGuard guard(x.device());
  const spio_gw8_shape& s = c.shape;
  const Tensor bias = vector_of(bias_), w = kernel_layout(weight);
  const Tensor y = empty_image({s.n, s.c, s.h + 2 * s.pad_h - s.r + 1, s.w + 2 * s.pad_w - s.s + 1}, x, at::kHalf);
  check_call(spio_conv2d_gw8_fprop(pointer(y), pointer(x), pointer(w), floats(bias), &s, &c.fprop, stream()), "conv2d_gw8");
  return y;
}

Tensor conv2d_gw8_checkpoint8_planned(const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t pad_y,
                                      int64_t pad_x, at::IntArrayRef tunes) {
  return conv_forward(checked_conv(x, weight, bias, pad_y, pad_x, tunes), kernel_layout(x), weight, bias);
}

struct ConvCheckpoint8 : torch::autograd::Function<ConvCheckpoint8> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x_, const Tensor& weight,
                        const OptTensor& bias, int64_t pad_y, int64_t pad_x, std::vector<int64_t> tunes) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Conv c = checked_conv(x_, weight, bias, pad_y, pad_x, tunes);
    const Tensor x = kernel_layout(x_);
    const Tensor y = conv_forward(c, x, weight, bias);
    Tensor codes, exponents;  // nothing but the weight's gradient reads the input's values again
    if (weight.requires_grad()) std::tie(codes, exponents) = checkpoint8_pack(x);
    ctx->save_for_backward({codes, exponents, weight, tensor_of(bias)});
    for (const int64_t v : {pad_y, pad_x, x.size(0), x.size(1), x.size(2), x.size(3)}) tunes.push_back(v);
    ctx->saved_data["call"] = std::move(tunes);
    return y;
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grads) {
    // (what is launched here has no derivative of its own)
    TORCH_CHECK(!at::GradMode::is_enabled(), "spio conv2d_gw8_checkpoint8 cannot be differentiated twice");
    const variable_list saved = ctx->get_saved_variables();
    variable_list result(6);
    if (!grads[0].defined()) return result;
    check_no_tangent(grads[0], "conv2d_gw8_checkpoint8");
    const Tensor &codes = saved[0], &exponents = saved[1], &weight = saved[2];
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    const bool want_b = saved[3].defined() && ctx->needs_input_grad(2);
    const c10::cuda::CUDAGuard guard(weight.device());
    const std::vector<int64_t> call = ctx->saved_data["call"].toIntVector();  // tunes, padding, the input's size
    const at::IntArrayRef tunes = at::IntArrayRef(call).slice(0, kTunes), size = at::IntArrayRef(call).slice(kTunes + 2, 4);
    const Conv c = conv_of(size, weight, call[kTunes], call[kTunes + 1], tunes);
    Tensor x;
    if (want_w) x = checkpoint8_unpack(codes, exponents, at::kHalf);
    const Tensor dy = kernel_layout(grads[0]), w = kernel_layout(weight);
    Tensor dx, dw, db;
    if (want_x) dx = empty_image(size, dy, at::kHalf);
    if (want_w) dw = empty_image(weight.sizes(), dy, at::kHalf);
    // with an odd number of taps the weight-gradient kernel sums dy in a spare half of its last product
    const bool with_taps = want_b && want_w && (c.shape.r * c.shape.s) % 2 == 1;
    if (with_taps) db = empty_vector(c.shape.c, dy, at::kFloat);
    else if (want_b) db = dy.sum({0, 2, 3}, false, at::kFloat);
    if (want_w) {
      const size_t bytes = spio_conv2d_gw8_wgrad_scratch_bytes(&c.shape, &c.wgrad);
      const Tensor scratch = scratch_of(bytes, dy);  // of this call: two captured graphs share none
      spio_gw8_backward_opts opts{};
      opts.dw_f16 = 1;  // the weight's own type: the fp32 sums are rounded once
      check_call(spio_conv2d_gw8_backward_ex(pointer(dx), static_cast<float*>(pointer(dw)), with_taps ? floats(db) : nullptr,
                                             pointer(x), pointer(dy), pointer(w), &c.shape, &c.dgrad, &c.wgrad,
                                             pointer(scratch), bytes, stream(), nullptr, &opts),
                 "conv2d_gw8_checkpoint8 backward");
    } else if (want_x) {
      check_call(spio_conv2d_gw8_dgrad(pointer(dx), pointer(dy), pointer(w), &c.shape, &c.dgrad, stream()),
                 "conv2d_gw8_checkpoint8 backward");
    }
    result[0] = dx, result[1] = dw, result[2] = db;
    return result;
  }
};

Tensor conv2d_gw8_checkpoint8_planned_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                               int64_t pad_y, int64_t pad_x, at::IntArrayRef tunes) {
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || requires_grad(bias)))
    return ConvCheckpoint8::apply(x, weight, bias, pad_y, pad_x, tunes.vec());
  at::AutoDispatchBelowADInplaceOrView below;
  return conv2d_gw8_checkpoint8_planned(x, weight, bias, pad_y, pad_x, tunes);
}

}  // namespace

TORCH_LIBRARY_IMPL(spio, CUDA, m) {
  m.impl("groupnorm_2d", groupnorm_2d);
  m.impl("groupnorm_2d_forward", groupnorm_2d_forward);
  m.impl("groupnorm_2d_backward", groupnorm_2d_backward);
  m.impl("checkpoint8_pack", checkpoint8_pack);
  m.impl("checkpoint8_unpack", checkpoint8_unpack);
  m.impl("conv2d_gw8_checkpoint8_planned", conv2d_gw8_checkpoint8_planned);
}

// (these refuse CPU tensors by name)
TORCH_LIBRARY_IMPL(spio, CPU, m) {
  m.impl("groupnorm_2d", groupnorm_2d);
  m.impl("groupnorm_2d_forward", groupnorm_2d_forward);
  m.impl("groupnorm_2d_backward", groupnorm_2d_backward);
  m.impl("checkpoint8_pack", checkpoint8_pack);
  m.impl("checkpoint8_unpack", checkpoint8_unpack);
  m.impl("conv2d_gw8_checkpoint8_planned", conv2d_gw8_checkpoint8_planned);
}

TORCH_LIBRARY_IMPL(spio, Autograd, m) {
  m.impl("groupnorm_2d", groupnorm_2d_autograd);
  m.impl("groupnorm_2d_backward", groupnorm_2d_backward_autograd);
  m.impl("conv2d_gw8_checkpoint8_planned", conv2d_gw8_checkpoint8_planned_autograd);
}

TORCH_LIBRARY_IMPL(spio, AutocastCUDA, m) { m.impl("groupnorm_2d", groupnorm_2d_autocast); }
