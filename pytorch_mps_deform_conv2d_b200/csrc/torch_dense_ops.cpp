// torch_dense_ops.cpp -- PyTorch operators of the orthogonalised updates and
// of the 8-bit products, beside those of torch_ops.cpp in the same namespace.
// As there, each validates, allocates outputs and scratch through PyTorch's
// caching allocator and calls the C ABI on the current CUDA stream of its
// tensors' device.
#include <ATen/ATen.h>
#include <ATen/Context.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <iterator>
#include <utility>
#include <vector>

#include "dcn_b200.h"

namespace {

uint32_t resolve_math(int64_t math) {
  if (math >= 0) return static_cast<uint32_t>(math);
  return at::globalContext().allowTF32CuBLAS() ? DCN_MATH_TF32 : DCN_MATH_FP32;
}

void check_rc(int rc) { TORCH_CHECK(rc == DCN_OK, dcn_last_error()); }

bool float_type(at::ScalarType t) {
  return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf;
}

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return DCN_TYPE_F32;
    case at::kBFloat16: return DCN_TYPE_BF16;
    case at::kHalf: return DCN_TYPE_F16;
    default: return DCN_TYPE_I8;
  }
}

std::vector<float> step_coefficients(c10::ArrayRef<double> c, int64_t steps, const char* op) {
  TORCH_CHECK(steps >= 1 && steps <= 32, op, ": steps must be 1 to 32, got ", steps);
  TORCH_CHECK(c.size() == 3 || (int64_t)c.size() == 3 * steps, op,
              ": coefficients must be one triple or one for each of the ", steps, " steps");
  std::vector<float> v(3 * steps);
  for (int64_t i = 0; i < 3 * steps; ++i) v[i] = (float)c[c.size() == 3 ? i % 3 : i];
  return v;
}

// Bytes for the current stream of the current device, given back at the end of
// the call: a later allocation of the same stream may have them, other streams
// not before.
c10::DataPtr scratch(size_t bytes) {
  return c10::cuda::CUDACachingAllocator::get()->allocate(std::max<size_t>(bytes, 1));
}

// Contiguous, on `like`'s device.
at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

at::Tensor newton_schulz(const at::Tensor& update, int64_t steps, at::ArrayRef<double> coefficients,
                         double eps, int64_t math) {
  TORCH_CHECK(update.device().is_cuda(), "newton_schulz: update must be a CUDA tensor");
  TORCH_CHECK(float_type(update.scalar_type()),
              "newton_schulz: update must be float32, bfloat16 or float16");
  TORCH_CHECK(update.dim() >= 2, "newton_schulz: update must have at least two dimensions, got ",
              update.dim());
  const auto coef = step_coefficients(coefficients, steps, "newton_schulz");
  c10::cuda::CUDAGuard guard(update.device());
  auto x = update.contiguous();
  auto out = make(x.sizes(), x.scalar_type(), x);
  if (x.numel() == 0) return out;
  const int64_t rows = x.size(-2), cols = x.size(-1), count = x.numel() / (rows * cols);
  const int type = type_code(x.scalar_type());
  const uint32_t flags = resolve_math(math);
  const size_t bytes =
      dcn_newton_schulz_workspace_size(count, rows, cols, type, (int)steps, flags);
  auto ws = scratch(bytes);
  check_rc(dcn_newton_schulz(count, rows, cols, type, x.data_ptr(), out.data_ptr(), (int)steps,
                             coef.data(), (float)eps, flags, ws.get(), bytes,
                             at::cuda::getCurrentCUDAStream().stream()));
  return out;
}

// Rows of the flattened parameter lie one after another, in whatever order of
// the trailing dimensions: permuting the columns of an update permutes those
// of its orthogonalised form, so a channels-last weight is taken as it lies.
bool rows_outermost(const at::Tensor& t) {
  return t.is_non_overlapping_and_dense() &&
         (t.size(0) <= 1 || t.stride(0) * t.size(0) == t.numel());
}

void muon_update_(at::TensorList params, at::TensorList grads, at::TensorList momenta, double lr,
                  double momentum, bool nesterov, double weight_decay, int64_t steps,
                  at::ArrayRef<double> coefficients, double eps, bool match_rms, int64_t groups,
                  int64_t math) {
  TORCH_CHECK(params.size() == grads.size() && params.size() == momenta.size(),
              "muon_update_: as many grads and momenta as params are needed, got ",
              params.size(), ", ", grads.size(), " and ", momenta.size());
  const auto coef = step_coefficients(coefficients, steps, "muon_update_");
  TORCH_CHECK(groups > 0, "muon_update_: groups must be positive, got ", groups);
  TORCH_CHECK(momentum >= 0.0 && momentum < 1.0, "muon_update_: momentum must be in [0, 1), got ",
              momentum);
  if (params.empty()) return;
  const uint32_t flags = resolve_math(math);
  std::vector<at::Tensor> aligned(params.size());  // gradients in their parameter's layout
  std::vector<std::pair<const char*, const char*>> written;  // dense, so ranges of bytes
  for (size_t i = 0; i < params.size(); ++i) {
    const auto &p = params[i], &g = grads[i], &m = momenta[i];
    TORCH_CHECK(p.device().is_cuda() && p.device() == params[0].device() &&
                    g.device() == p.device() && m.device() == p.device(),
                "muon_update_: params, grads and momenta must be on one CUDA device");
    TORCH_CHECK(float_type(p.scalar_type()) && g.scalar_type() == p.scalar_type(),
                "muon_update_: params must be float32, bfloat16 or float16, and grads of the "
                "same type");
    TORCH_CHECK(m.scalar_type() == at::kFloat, "muon_update_: momenta must be float32");
    TORCH_CHECK(p.layout() == at::kStrided && g.layout() == at::kStrided,
                "muon_update_: sparse tensors are not supported");
    TORCH_CHECK(p.dim() >= 2, "muon_update_: params must have at least two dimensions, got ",
                p.dim());
    TORCH_CHECK(g.sizes() == p.sizes() && m.sizes() == p.sizes(),
                "muon_update_: grads and momenta must have their parameter's shape ", p.sizes(),
                ", got ", g.sizes(), " and ", m.sizes());
    TORCH_CHECK(p.size(0) % groups == 0, "muon_update_: rows (", p.size(0),
                ") not divisible by groups (", groups, ")");
    TORCH_CHECK(p.numel() == 0 || (rows_outermost(p) && m.strides() == p.strides()),
                "muon_update_: params must be dense with dimension 0 outermost, momenta of the "
                "same strides");
    if (p.numel() == 0) continue;
    // a size that is refused is refused before any parameter is written
    TORCH_CHECK(dcn_muon_update_workspace_size(1, p.size(0) / groups, p.numel() / p.size(0),
                                               type_code(p.scalar_type()), (int)steps, flags) > 0,
                dcn_last_error());
    const char *pb = static_cast<const char*>(p.data_ptr()),
               *mb = static_cast<const char*>(m.data_ptr());
    written.emplace_back(pb, pb + p.nbytes());
    written.emplace_back(mb, mb + m.nbytes());
  }
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    TORCH_CHECK(written[i].first >= written[i - 1].second,
                "muon_update_: params and momenta must not overlap (the same parameter or "
                "momentum is given twice?)");
  for (size_t i = 0; i < grads.size(); ++i) {  // read after the first of them are written
    const auto& g = grads[i];
    if (g.numel() == 0) continue;
    int64_t span = 1;
    for (int64_t d = 0; d < g.dim(); ++d) span += (g.size(d) - 1) * g.stride(d);
    const char* gb = static_cast<const char*>(g.data_ptr());
    const char* ge = gb + span * g.element_size();
    const auto next = std::lower_bound(written.begin(), written.end(), std::make_pair(gb, gb));
    TORCH_CHECK((next == written.end() || next->first >= ge) &&
                    (next == written.begin() || std::prev(next)->second <= gb),
                "muon_update_: grads must not overlap params or momenta");
  }
  c10::cuda::CUDAGuard guard(params[0].device());
  std::vector<bool> done(params.size(), false);
  const auto stream = at::cuda::getCurrentCUDAStream().stream();
  for (size_t i = 0; i < params.size(); ++i) {
    if (done[i] || params[i].numel() == 0) continue;
    const auto& first = params[i];
    const int64_t rows = first.size(0) / groups, cols = first.numel() / first.size(0);
    const int type = type_code(first.scalar_type());
    std::vector<void*> p;
    std::vector<const void*> g;
    std::vector<float*> m;
    for (size_t j = i; j < params.size(); ++j) {  // all of this shape and type in one call
      if (done[j] || params[j].numel() != first.numel() || params[j].size(0) != first.size(0) ||
          params[j].scalar_type() != first.scalar_type())
        continue;
      done[j] = true;
      aligned[j] = grads[j].strides() == params[j].strides()
                       ? grads[j]
                       : at::empty_like(params[j]).copy_(grads[j]);
      const size_t es = first.element_size();
      for (int64_t k = 0; k < groups; ++k) {
        p.push_back(static_cast<char*>(params[j].data_ptr()) + k * rows * cols * es);
        g.push_back(static_cast<const char*>(aligned[j].data_ptr()) + k * rows * cols * es);
        m.push_back(momenta[j].data_ptr<float>() + k * rows * cols);
      }
    }
    const double big = (double)std::max(rows, cols);
    const double scale = match_rms ? 0.2 * std::sqrt(big)
                                   : std::sqrt(std::max(1.0, (double)rows / (double)cols));
    const size_t bytes = dcn_muon_update_workspace_size((int64_t)p.size(), rows, cols, type,
                                                        (int)steps, flags);
    auto ws = scratch(bytes);
    check_rc(dcn_muon_update_f64((int64_t)p.size(), rows, cols, type, p.data(), g.data(), m.data(),
                                 lr, momentum, nesterov ? 1 : 0, weight_decay, scale, (int)steps,
                                 coef.data(), (float)eps, flags, ws.get(), bytes, stream));
  }
  for (size_t i = 0; i < params.size(); ++i) {  // written through raw pointers
    params[i].unsafeGetTensorImpl()->bump_version();
    momenta[i].unsafeGetTensorImpl()->bump_version();
  }
}

std::tuple<at::Tensor, at::Tensor> quantize_int8(const at::Tensor& x) {
  TORCH_CHECK(x.device().is_cuda(), "quantize_int8: x must be a CUDA tensor");
  TORCH_CHECK(float_type(x.scalar_type()),
              "quantize_int8: x must be float32, bfloat16 or float16");
  TORCH_CHECK(x.dim() >= 1, "quantize_int8: x must have at least one dimension");
  c10::cuda::CUDAGuard guard(x.device());
  auto xc = x.contiguous();
  auto q = make(xc.sizes(), at::kChar, xc);
  auto sizes = xc.sizes().slice(0, xc.dim() - 1);
  const int64_t cols = xc.size(-1);
  if (cols == 0) return std::make_tuple(q, at::zeros(sizes, xc.options().dtype(at::kFloat)));
  auto scale = make(sizes, at::kFloat, xc);
  if (xc.numel() == 0) return std::make_tuple(q, scale);
  check_rc(dcn_quantize_int8(xc.numel() / cols, cols, type_code(xc.scalar_type()), xc.data_ptr(),
                             q.data_ptr<int8_t>(), scale.data_ptr<float>(),
                             at::cuda::getCurrentCUDAStream().stream()));
  return std::make_tuple(q, scale);
}

// Weight scale (one fp32 value an output channel) and bias, checked.
at::Tensor channel_scale(const at::Tensor& scale, const at::Tensor& weight, const char* op) {
  TORCH_CHECK(scale.device() == weight.device() && scale.scalar_type() == at::kFloat &&
                  scale.dim() == 1 && scale.size(0) == weight.size(0),
              op, ": weight_scale must be float32 of ", weight.size(0),
              " elements on the weight's device, got ", scale.sizes());
  return scale.contiguous();
}
at::Tensor channel_bias(const c10::optional<at::Tensor>& bias, const at::Tensor& weight,
                        const char* op) {
  if (!bias.has_value() || !bias->defined()) return at::Tensor();
  TORCH_CHECK(bias->device() == weight.device() && float_type(bias->scalar_type()) &&
                  bias->dim() == 1 && bias->size(0) == weight.size(0),
              op, ": bias must be float32, bfloat16 or float16 of ", weight.size(0),
              " elements on the weight's device, got ", bias->sizes());
  return bias->contiguous();
}

at::Tensor int8_linear(const at::Tensor& x, const at::Tensor& weight,
                       const at::Tensor& weight_scale, const c10::optional<at::Tensor>& bias,
                       const c10::optional<at::Tensor>& x_scale,
                       c10::optional<at::ScalarType> out_dtype, int64_t flags) {
  TORCH_CHECK(x.device().is_cuda() && weight.device() == x.device(),
              "int8_linear: x and weight must be on one CUDA device");
  const bool given = x.scalar_type() == at::kChar;
  TORCH_CHECK(given || float_type(x.scalar_type()),
              "int8_linear: x must be int8, float32, bfloat16 or float16");
  TORCH_CHECK(weight.scalar_type() == at::kChar && weight.dim() == 2,
              "int8_linear: weight must be int8 (out_features, in_features)");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) == weight.size(1), "int8_linear: x must end in ",
              weight.size(1), " features, got ", x.sizes());
  TORCH_CHECK(weight.size(1) > 0, "int8_linear: at least one input feature is needed");
  const bool has_scale = x_scale.has_value() && x_scale->defined();
  TORCH_CHECK(given == has_scale,
              "int8_linear: x_scale comes with an int8 x, and only then");
  const auto odt = out_dtype.has_value() ? *out_dtype : (given ? at::kFloat : x.scalar_type());
  TORCH_CHECK(float_type(odt), "int8_linear: out_dtype must be float32, bfloat16 or float16");
  auto ws_ = channel_scale(weight_scale, weight, "int8_linear");
  auto b = channel_bias(bias, weight, "int8_linear");
  c10::cuda::CUDAGuard guard(x.device());
  auto xc = x.contiguous();
  auto w = weight.contiguous();
  at::Tensor xs;
  if (given) {
    TORCH_CHECK(x_scale->device() == x.device() && x_scale->scalar_type() == at::kFloat &&
                    x_scale->sizes() == x.sizes().slice(0, x.dim() - 1),
                "int8_linear: x_scale must be float32 with x's leading shape, got ",
                x_scale->sizes());
    xs = x_scale->contiguous();
  }
  auto sizes = xc.sizes().vec();
  sizes.back() = w.size(0);
  auto out = make(sizes, odt, xc);
  if (out.numel() == 0) return out;
  const int64_t in = w.size(1), tokens = xc.numel() / in;
  const int xt = type_code(xc.scalar_type());
  const size_t bytes = dcn_int8_linear_workspace_size(tokens, in, w.size(0), xt);
  auto call = [&](void* ws) {
    return dcn_int8_linear(tokens, in, w.size(0), xt, xc.data_ptr(),
                           given ? xs.data_ptr<float>() : nullptr, w.data_ptr<int8_t>(),
                           ws_.data_ptr<float>(), b.defined() ? b.data_ptr() : nullptr,
                           b.defined() ? type_code(b.scalar_type()) : 0, out.data_ptr(),
                           type_code(odt), (uint32_t)flags, ws, ws != nullptr ? bytes : 0,
                           at::cuda::getCurrentCUDAStream().stream());
  };
  // a few tokens take no workspace where their rows allow it
  int rc = dcn_int8_linear_few_tokens(tokens, in, w.size(0), xt) ? call(nullptr)
                                                                 : DCN_ERR_WORKSPACE;
  if (rc == DCN_ERR_WORKSPACE) {
    auto ws = scratch(bytes);
    rc = call(ws.get());
  }
  check_rc(rc);
  return out;
}

at::Tensor deform_conv2d_int8(const at::Tensor& input, const at::Tensor& weight,
                              const at::Tensor& weight_scale, const at::Tensor& offset,
                              const c10::optional<at::Tensor>& mask,
                              const c10::optional<at::Tensor>& bias, int64_t stride_h,
                              int64_t stride_w, int64_t pad_h, int64_t pad_w, int64_t dilation_h,
                              int64_t dilation_w, int64_t groups, int64_t deformable_groups,
                              c10::optional<at::ScalarType> out_dtype, int64_t flags) {
  TORCH_CHECK(input.device().is_cuda() && weight.device() == input.device() &&
                  offset.device() == input.device(),
              "deform_conv2d_int8: input, weight and offset must be on one CUDA device");
  const auto dt = input.scalar_type();
  TORCH_CHECK(float_type(dt) && offset.scalar_type() == dt,
              "deform_conv2d_int8: input and offset must both be float32, bfloat16 or float16");
  TORCH_CHECK(input.dim() == 4, "input must be 4-D (N, C, H, W), got ", input.dim());
  TORCH_CHECK(weight.scalar_type() == at::kChar && weight.dim() == 4,
              "deform_conv2d_int8: weight must be int8 (outC, C/groups, kh, kw)");
  TORCH_CHECK(offset.dim() == 4, "offset must be 4-D (N, 2*dg*kh*kw, oh, ow), got ",
              offset.dim());
  TORCH_CHECK(groups > 0 && weight.size(1) * groups == input.size(1),
              "weight shape mismatch: expected in-channels ", input.size(1), ", got ",
              weight.size(1) * groups);
  const bool has_mask = mask.has_value() && mask->defined();
  const auto odt = out_dtype.has_value() ? *out_dtype : dt;
  TORCH_CHECK(float_type(odt),
              "deform_conv2d_int8: out_dtype must be float32, bfloat16 or float16");
  auto wscale = channel_scale(weight_scale, weight, "deform_conv2d_int8");
  auto b = channel_bias(bias, weight, "deform_conv2d_int8");
  dcn_shape s;
  s.batch = input.size(0);
  s.in_channels = input.size(1);
  s.height = input.size(2);
  s.width = input.size(3);
  s.out_channels = weight.size(0);
  s.kernel_h = weight.size(2);
  s.kernel_w = weight.size(3);
  s.stride_h = stride_h;
  s.stride_w = stride_w;
  s.pad_h = pad_h;
  s.pad_w = pad_w;
  s.dilation_h = dilation_h;
  s.dilation_w = dilation_w;
  s.groups = groups;
  s.deformable_groups = deformable_groups;
  int64_t oh = 0, ow = 0;
  check_rc(dcn_output_size(&s, &oh, &ow));
  const int64_t taps = s.kernel_h * s.kernel_w * deformable_groups;
  TORCH_CHECK(offset.size(0) == s.batch && offset.size(1) == 2 * taps && offset.size(2) == oh &&
                  offset.size(3) == ow,
              "offset shape mismatch: expected (", s.batch, ", ", 2 * taps, ", ", oh, ", ", ow,
              "), got ", offset.sizes());
  if (has_mask) {
    TORCH_CHECK(mask->device() == input.device() && mask->scalar_type() == dt,
                "deform_conv2d_int8: mask must have the input's device and type");
    TORCH_CHECK(mask->dim() == 4 && mask->size(0) == s.batch && mask->size(1) == taps &&
                    mask->size(2) == oh && mask->size(3) == ow,
                "mask shape mismatch: expected (", s.batch, ", ", taps, ", ", oh, ", ", ow,
                "), got ", mask->sizes());
  }
  c10::cuda::CUDAGuard guard(input.device());
  const bool nhwc =
      !input.is_contiguous() && input.is_contiguous(at::MemoryFormat::ChannelsLast);
  auto x = nhwc ? input : input.contiguous();
  auto w = weight.permute({0, 2, 3, 1}).contiguous();  // no copy for a channels-last weight
  auto off = offset.contiguous();
  auto msk = has_mask ? mask->contiguous() : at::Tensor();
  auto out = make({s.batch, s.out_channels, oh, ow}, odt, x);
  if (out.numel() == 0) return out;
  const uint32_t fl = (uint32_t)flags | (nhwc ? DCN_INPUT_NHWC : 0u);
  const int type = type_code(dt);
  const size_t bytes = dcn_deform_int8_workspace_size(&s, type, fl);
  auto ws = scratch(bytes);
  check_rc(dcn_deform_int8(&s, type, x.numel() ? x.data_ptr() : nullptr, w.data_ptr<int8_t>(),
                           wscale.data_ptr<float>(), off.data_ptr(),
                           has_mask ? msk.data_ptr() : nullptr,
                           b.defined() ? b.data_ptr() : nullptr,
                           b.defined() ? type_code(b.scalar_type()) : 0, out.data_ptr(),
                           type_code(odt), fl, ws.get(), bytes,
                           at::cuda::getCurrentCUDAStream().stream()));
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(deform_conv2d_b200, m) {
  m.def(
      "newton_schulz(Tensor update, int steps, float[] coefficients, float eps, int math=-1) "
      "-> Tensor");
  m.def(
      "muon_update_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] momenta, float lr, "
      "float momentum, bool nesterov, float weight_decay, int steps, float[] coefficients, "
      "float eps, bool match_rms=False, int groups=1, int math=-1) -> ()");
  m.def("quantize_int8(Tensor x) -> (Tensor, Tensor)");
  m.def(
      "int8_linear(Tensor x, Tensor weight, Tensor weight_scale, Tensor? bias=None, "
      "Tensor? x_scale=None, ScalarType? out_dtype=None, int flags=0) -> Tensor");
  m.def(
      "deform_conv2d_int8(Tensor input, Tensor weight, Tensor weight_scale, Tensor offset, "
      "Tensor? mask, Tensor? bias, int stride_h, int stride_w, int pad_h, int pad_w, "
      "int dilation_h, int dilation_w, int groups, int deformable_groups, "
      "ScalarType? out_dtype=None, int flags=0) -> Tensor");
}

TORCH_LIBRARY_IMPL(deform_conv2d_b200, CUDA, m) {
  m.impl("newton_schulz", TORCH_FN(newton_schulz));
  m.impl("muon_update_", TORCH_FN(muon_update_));
  m.impl("quantize_int8", TORCH_FN(quantize_int8));
  m.impl("int8_linear", TORCH_FN(int8_linear));
  m.impl("deform_conv2d_int8", TORCH_FN(deform_conv2d_int8));
}
