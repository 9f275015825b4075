// dcn_capi_dense.cu -- extern "C" entry points of the orthogonalised updates
// and of the 8-bit products (declared in include/dcn_b200.h): validation,
// workspace carving, dispatch.  As in dcn_capi.cu nothing allocates device
// memory or waits for the device.
#include <cmath>
#include <cstring>

#include "dcn_capi_util.h"
#include "dcn_gemm.h"
#include "dcn_int8.h"
#include "dcn_kernels.h"
#include "dcn_launch.h"
#include "dcn_ortho.h"

using namespace dcn::capi;

namespace {

// Chunk of matrices an orthogonalisation keeps in its workspace at a time: up
// to 64, and no more than fit 1 GB (one always does).
constexpr size_t kOrthoChunkBytes = size_t(1) << 30;
// Sampled 8-bit columns kept at a time.
constexpr size_t kColumnBytes = size_t(256) << 20;
// |sum| <= K * 128 * 128 stays inside int32
constexpr int64_t kInt8MaxK = 131071;
// Rows and columns of a product: the kernels round them up to whole tiles, of
// 256 at most, in int
constexpr int64_t kMaxSide = (int64_t(1) << 31) - 256;

int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
size_t type_bytes(int t) { return t == DCN_TYPE_F32 ? 4 : t == DCN_TYPE_I8 ? 1 : 2; }
bool float_type(int t) { return t == DCN_TYPE_F32 || t == DCN_TYPE_BF16 || t == DCN_TYPE_F16; }
static_assert(DCN_TYPE_F32 == dcn::kF32 && DCN_TYPE_BF16 == dcn::kBF16T &&
                  DCN_TYPE_F16 == dcn::kF16T,
              "one numbering");

long long wait_limit(uint32_t flags) {
  return flags & DCN_TEST_WAIT_TIMEOUT ? dcn::kTestWaitLimit : dcn::kWaitLimit;
}

struct Carve {
  char* at;
  explicit Carve(void* p)
      : at(reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p) + kAlign - 1) &
                                   ~(uintptr_t)(kAlign - 1))) {}
  template <class T>
  T* take(size_t bytes) {
    T* p = reinterpret_cast<T*>(at);
    at += align_up(bytes);
    return p;
  }
};

// The polynomial a + b S + c S S is summed in fp32 and its values are stored in
// fp16 (up to 16): those on [0, 1] have to fit, b and c by themselves need not.
bool polynomial_fits(const float* abc) {
  const double a = abc[0], b = abc[1], c = abc[2], most = 15.0;
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c) || std::fabs(a) > most)
    return false;
  if (std::fabs(b) <= most && std::fabs(c) <= most) return true;
  const double turn = c != 0.0 ? -b / (2.0 * c) : -1.0;  // of the parabola
  return std::fabs(a + b + c) <= most &&
         (turn <= 0.0 || turn >= 1.0 || std::fabs(a + 0.5 * b * turn) <= most);
}

// fp16 terms by what the result can hold: bf16 keeps 8 bits, so X between two
// runs is rounded to fp16's 11 once; fp16 and fp32 results take both terms
// there.  fp32 tensors under DCN_MATH_TF32 ask for 11 bits.
int ortho_shape(int64_t rows, int64_t cols, int type, int steps, const float* coef, float eps,
                uint32_t flags, bool muon, dcn::OrthoShape& s, const char* op) {
  DCN_CHECK(rows >= 0 && cols >= 0, "%s: matrix sizes must be non-negative", op);
  DCN_CHECK(float_type(type), "%s: matrices must be float32, bfloat16 or float16", op);
  DCN_CHECK(steps >= 1 && steps <= dcn::kOrthoMaxSteps, "%s: steps must be 1 to %d, got %d", op,
            dcn::kOrthoMaxSteps, steps);
  DCN_CHECK(eps >= 0.f, "%s: eps must be non-negative", op);
  const int64_t small = rows < cols ? rows : cols, large = rows < cols ? cols : rows;
  if (small > 32768 || large > kMaxSide || small * large >= (int64_t(1) << 31))
    return fail(DCN_ERR_UNSUPPORTED, "%s: matrices of 2^31 elements and more, with a side beyond "
                "2^31 - 256 or with both sides beyond 32768, are not supported", op);
  const uint32_t math = flags & 0xff;
  const bool f32 = type == DCN_TYPE_F32;
  s.rows = (int)rows;
  s.cols = (int)cols;
  s.type = type;
  s.first_terms = f32 && math != DCN_MATH_TF32 ? 2 : 1;
  s.later_terms = (f32 && math != DCN_MATH_TF32) || (type == DCN_TYPE_F16 && !muon) ? 2 : 1;
  s.steps = steps;
  s.eps = eps;
  if (coef != nullptr) {
    std::memcpy(s.coef, coef, sizeof(float) * 3 * steps);
    for (int i = 0; i < steps; ++i)
      DCN_CHECK(polynomial_fits(coef + 3 * i),
                "%s: coefficients (a, b, c) must be finite, a at most 15 in size, and b and c, or "
                "the values of a + b s + c s^2 for s in [0, 1], too", op);
  }
  return DCN_OK;
}

int ortho_chunk(const dcn::OrthoShape& s, int64_t count) {
  int64_t n = count < dcn::kGemmMaxList ? count : dcn::kGemmMaxList;
  while (n > 1 && dcn::ortho_workspace_bytes(s, (int)n) > kOrthoChunkBytes) n = (n + 1) / 2;
  return (int)n;
}

struct DeformInt8 {
  dcn::Geom g;
  int64_t kg, kp;  // columns a group, padded
  int64_t chunk;   // pixels at a time
  bool pack;       // the weight's rows need the padded pitch
  bool nhwc;       // the image is sampled where it lies
  size_t stage_bytes, col_bytes, scale_bytes, weight_bytes, total;
};

int deform_int8_plan(const dcn_shape* shape, int type, uint32_t flags, DeformInt8& d,
                     const char* op) {
  const int rc = make_geom(shape, true, true, d.g, op);
  if (rc != DCN_OK) return rc;
  DCN_CHECK(float_type(type), "%s: input, offset and mask must be float32, bfloat16 or float16",
            op);
  const dcn::Geom& g = d.g;
  if (!(flags & DCN_INPUT_NHWC) && g.N > 65535)
    return fail(DCN_ERR_UNSUPPORTED, "%s: more than 65535 NCHW images are not supported", op);
  if (g.Og > kMaxSide)
    return fail(DCN_ERR_UNSUPPORTED, "%s: more than %lld output channels a group are not supported",
                op, (long long)kMaxSide);
  d.kg = (int64_t)g.Cg * g.kk;
  if (d.kg > kInt8MaxK)
    return fail(DCN_ERR_UNSUPPORTED, "%s: more than %lld columns a group are not supported", op,
                (long long)kInt8MaxK);
  d.kp = up16(d.kg);
  d.pack = d.kp != d.kg;
  const int64_t a_pixel = d.kp * g.G;
  d.chunk = g.NP;
  const int64_t fit = (int64_t)(kColumnBytes / (size_t)(a_pixel > 0 ? a_pixel : 1)) / 128 * 128;
  if (d.chunk > fit) d.chunk = fit > 128 ? fit : 128;
  // (images without pixels may have no address: theirs is the row of zeros that
  // the staging kernels append)
  d.nhwc = (flags & DCN_INPUT_NHWC) && g.HW > 0;
  d.stage_bytes = d.nhwc ? 0 : align_up(((size_t)g.N * g.HW * g.C + g.C) * type_bytes(type));
  d.col_bytes = align_up((size_t)d.chunk * a_pixel);
  d.scale_bytes = align_up((size_t)d.chunk * g.G * sizeof(float));
  d.weight_bytes = align_up((size_t)g.outC * d.kp);  // for rows off their pitch or alignment
  d.total = d.stage_bytes + d.col_bytes + d.scale_bytes + d.weight_bytes + kAlign;
  return DCN_OK;
}

struct LinearPlan {
  bool quantize, pack_x, pack_w;
  int64_t kp;
  size_t x_bytes, scale_bytes, w_bytes, total;
};

LinearPlan linear_plan(int64_t tokens, int64_t in, int64_t out, int x_type) {
  LinearPlan p;
  p.quantize = x_type != DCN_TYPE_I8;
  p.kp = up16(in);
  // rows of other lengths, or an 8-bit operand off a 16-byte boundary, are
  // copied to rows TMA can step over; the workspace always has room
  p.pack_x = p.pack_w = p.kp != in;
  p.x_bytes = align_up((size_t)tokens * p.kp);
  p.scale_bytes = align_up((size_t)tokens * sizeof(float));
  p.w_bytes = align_up((size_t)out * p.kp);
  p.total = p.x_bytes + p.scale_bytes + p.w_bytes + kAlign;
  return p;
}

dcn::GemmOperand rows_i8(const signed char* base, int64_t rows, int64_t inner, int64_t pitch,
                         int64_t batch) {
  dcn::GemmOperand o{base, rows, inner, pitch, 1, 0, (int)batch, rows * pitch, false};
  return o;
}

}  // namespace

extern "C" {

DCN_API size_t dcn_newton_schulz_workspace_size(int64_t count, int64_t rows, int64_t cols,
                                                int type, int steps, uint32_t flags) {
  dcn::OrthoShape s;
  if (count <= 0 || rows <= 0 || cols <= 0 ||
      ortho_shape(rows, cols, type, steps, nullptr, 0.f, flags, false, s,
                  "dcn_newton_schulz") != DCN_OK)
    return 0;
  return dcn::ortho_workspace_bytes(s, ortho_chunk(s, count));
}

DCN_API int dcn_newton_schulz(int64_t count, int64_t rows, int64_t cols, int type,
                              const void* input, void* output, int steps,
                              const float* coefficients, float eps, uint32_t flags,
                              void* workspace, size_t workspace_bytes, void* stream_) {
  g_last_error.clear();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  dcn::OrthoShape s;
  DCN_CHECK(coefficients != nullptr, "dcn_newton_schulz: coefficients must not be NULL");
  int rc = ortho_shape(rows, cols, type, steps, coefficients, eps, flags, false, s,
                       "dcn_newton_schulz");
  if (rc != DCN_OK) return rc;
  DCN_CHECK(count >= 0, "dcn_newton_schulz: count must be non-negative");
  if (count == 0 || rows == 0 || cols == 0) return DCN_OK;
  DCN_CHECK(input != nullptr && output != nullptr,
            "dcn_newton_schulz: input and output must not be NULL");
  const int chunk = ortho_chunk(s, count);
  if (workspace == nullptr || workspace_bytes < dcn::ortho_workspace_bytes(s, chunk))
    return fail(DCN_ERR_WORKSPACE, "dcn_newton_schulz: workspace too small");
  const size_t one = (size_t)rows * cols * type_bytes(type);
  dcn::OrthoChunk c{};
  for (int64_t b = 0; b < count; b += chunk) {
    c.count = (int)(count - b < chunk ? count - b : chunk);
    for (int i = 0; i < c.count; ++i) {
      c.in[i] = static_cast<const char*>(input) + (b + i) * one;
      c.out[i] = static_cast<char*>(output) + (b + i) * one;
    }
    const char* stage = "";
    const cudaError_t e = dcn::launch_ortho(s, c, workspace, wait_limit(flags),
                                            flags & DCN_TEST_WAIT_TIMEOUT ? 1 : 0, stream, &stage);
    if (e != cudaSuccess) return cuda_fail(e, stage);
  }
  return DCN_OK;
}

DCN_API size_t dcn_muon_update_workspace_size(int64_t count, int64_t rows, int64_t cols, int type,
                                              int steps, uint32_t flags) {
  dcn::OrthoShape s;
  if (count <= 0 || rows <= 0 || cols <= 0 ||
      ortho_shape(rows, cols, type, steps, nullptr, 0.f, flags, true, s, "dcn_muon_update") !=
          DCN_OK)
    return 0;
  return dcn::ortho_workspace_bytes(s, ortho_chunk(s, count));
}

DCN_API int dcn_muon_update(int64_t count, int64_t rows, int64_t cols, int type,
                            void* const* params, const void* const* grads, float* const* momenta,
                            float lr, float momentum, int nesterov, float weight_decay,
                            float update_scale, int steps, const float* coefficients, float eps,
                            uint32_t flags, void* workspace, size_t workspace_bytes,
                            void* stream) {
  return dcn_muon_update_f64(count, rows, cols, type, params, grads, momenta, lr, momentum,
                             nesterov, weight_decay, update_scale, steps, coefficients, eps, flags,
                             workspace, workspace_bytes, stream);
}

DCN_API int dcn_muon_update_f64(int64_t count, int64_t rows, int64_t cols, int type,
                                void* const* params, const void* const* grads,
                                float* const* momenta, double lr, double momentum, int nesterov,
                                double weight_decay, double update_scale, int steps,
                                const float* coefficients, float eps, uint32_t flags,
                                void* workspace, size_t workspace_bytes, void* stream_) {
  g_last_error.clear();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  dcn::OrthoShape s;
  DCN_CHECK(coefficients != nullptr, "dcn_muon_update: coefficients must not be NULL");
  int rc = ortho_shape(rows, cols, type, steps, coefficients, eps, flags, true, s,
                       "dcn_muon_update");
  if (rc != DCN_OK) return rc;
  DCN_CHECK(count >= 0, "dcn_muon_update: count must be non-negative");
  DCN_CHECK(momentum >= 0.0 && momentum < 1.0, "dcn_muon_update: momentum must be in [0, 1)");
  if (count == 0 || rows == 0 || cols == 0) return DCN_OK;
  DCN_CHECK(params != nullptr && grads != nullptr && momenta != nullptr,
            "dcn_muon_update: params, grads and momenta must not be NULL");
  const int chunk = ortho_chunk(s, count);
  if (workspace == nullptr || workspace_bytes < dcn::ortho_workspace_bytes(s, chunk))
    return fail(DCN_ERR_WORKSPACE, "dcn_muon_update: workspace too small");
  for (int64_t i = 0; i < count; ++i)
    DCN_CHECK(params[i] != nullptr && grads[i] != nullptr && momenta[i] != nullptr,
              "dcn_muon_update: params, grads and momenta must not be NULL");
  dcn::OrthoChunk c{};
  c.muon = true;
  c.nesterov = nesterov != 0;
  c.beta = (float)momentum;
  c.rest = (float)(1.0 - momentum);
  c.keep = (float)(1.0 - lr * weight_decay);
  c.step = (float)(-lr * update_scale);
  for (int64_t b = 0; b < count; b += chunk) {
    c.count = (int)(count - b < chunk ? count - b : chunk);
    for (int i = 0; i < c.count; ++i) {
      c.in[i] = grads[b + i];
      c.out[i] = params[b + i];
      c.momentum[i] = momenta[b + i];
    }
    const char* stage = "";
    const cudaError_t e = dcn::launch_ortho(s, c, workspace, wait_limit(flags),
                                            flags & DCN_TEST_WAIT_TIMEOUT ? 1 : 0, stream, &stage);
    if (e != cudaSuccess) return cuda_fail(e, stage);
  }
  return DCN_OK;
}

DCN_API int dcn_quantize_int8(int64_t rows, int64_t cols, int type, const void* input,
                              int8_t* codes, float* scale, void* stream_) {
  g_last_error.clear();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  DCN_CHECK(rows >= 0 && cols >= 0, "dcn_quantize_int8: sizes must be non-negative");
  DCN_CHECK(float_type(type), "dcn_quantize_int8: input must be float32, bfloat16 or float16");
  if (rows >= (int64_t(1) << 31) || cols >= (int64_t(1) << 30))
    return fail(DCN_ERR_UNSUPPORTED, "dcn_quantize_int8: 2^31 rows or 2^30 columns and more are "
                "not supported");
  if (rows == 0) return DCN_OK;
  DCN_CHECK(scale != nullptr && (cols == 0 || (input != nullptr && codes != nullptr)),
            "dcn_quantize_int8: input, codes and scale must not be NULL");
  DCN_CUDA(dcn::launch_quantize_rows(input, type, rows, (int)cols, cols,
                                     reinterpret_cast<signed char*>(codes), cols, scale, stream),
           "quantize_rows");
  return DCN_OK;
}

DCN_API size_t dcn_int8_linear_workspace_size(int64_t tokens, int64_t in_features,
                                              int64_t out_features, int x_type) {
  if (tokens <= 0 || in_features <= 0 || out_features <= 0) return 0;
  return linear_plan(tokens, in_features, out_features, x_type).total;
}

DCN_API int dcn_int8_linear_few_tokens(int64_t tokens, int64_t in_features,
                                       int64_t out_features, int x_type) {
  return tokens > 0 && in_features > 0 && out_features > 0 &&
                 dcn::few_tokens_fit(tokens, in_features) &&
                 dcn::few_tokens_pay(x_type, tokens, in_features, out_features)
             ? 1
             : 0;
}

DCN_API int dcn_int8_linear(int64_t tokens, int64_t in_features, int64_t out_features, int x_type,
                            const void* x, const float* x_scale, const int8_t* weight,
                            const float* weight_scale, const void* bias, int bias_type,
                            void* output, int out_type, uint32_t flags, void* workspace,
                            size_t workspace_bytes, void* stream_) {
  g_last_error.clear();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  DCN_CHECK(tokens >= 0 && in_features > 0 && out_features >= 0,
            "dcn_int8_linear: sizes must be positive (tokens and outputs may be 0)");
  DCN_CHECK(float_type(x_type) || x_type == DCN_TYPE_I8,
            "dcn_int8_linear: x must be float32, bfloat16, float16 or int8");
  DCN_CHECK(float_type(out_type) && (bias == nullptr || float_type(bias_type)),
            "dcn_int8_linear: output and bias must be float32, bfloat16 or float16");
  if (in_features > kInt8MaxK || tokens > kMaxSide || out_features > kMaxSide)
    return fail(DCN_ERR_UNSUPPORTED, "dcn_int8_linear: more than %lld input features (sums past "
                "int32), or than %lld tokens or outputs, are not supported", (long long)kInt8MaxK,
                (long long)kMaxSide);
  if (tokens == 0 || out_features == 0) return DCN_OK;
  DCN_CHECK(x != nullptr && weight != nullptr && weight_scale != nullptr && output != nullptr &&
                ((x_type == DCN_TYPE_I8) == (x_scale != nullptr)),
            "dcn_int8_linear: x, weight, weight_scale and output must not be NULL; x_scale comes "
            "with int8 x and only then");
  LinearPlan p = linear_plan(tokens, in_features, out_features, x_type);
  if (workspace != nullptr && workspace_bytes < p.total)
    return fail(DCN_ERR_WORKSPACE, "dcn_int8_linear: workspace too small");
  if (dcn::few_tokens_fit(tokens, in_features) && aligned16(x) && aligned16(weight) &&
      (workspace == nullptr ||
       dcn::few_tokens_pay(x_type, tokens, in_features, out_features))) {
    DCN_CUDA(dcn::launch_few_tokens(x, x_type, x_scale, (int)tokens, (int)in_features,
                                    (int)out_features,
                                    reinterpret_cast<const signed char*>(weight), weight_scale,
                                    bias, bias_type, output, out_type, stream),
             "few_tokens");
    return DCN_OK;
  }
  if (workspace == nullptr)
    return fail(DCN_ERR_WORKSPACE, "dcn_int8_linear: these operands need a workspace");
  if (!aligned16(x)) p.pack_x = true;
  if (!aligned16(weight)) p.pack_w = true;
  Carve ws(workspace);
  signed char* xq = ws.take<signed char>(p.x_bytes);
  float* xs = ws.take<float>(p.scale_bytes);
  signed char* wq = ws.take<signed char>(p.w_bytes);
  const signed char* a = xq;
  const float* as = xs;
  if (p.quantize) {
    DCN_CUDA(dcn::launch_quantize_rows(x, x_type, tokens, (int)in_features, in_features, xq, p.kp,
                                       xs, stream),
             "quantize_rows");
  } else {
    as = x_scale;
    if (p.pack_x)
      DCN_CUDA(dcn::launch_repack_i8(static_cast<const signed char*>(x), tokens,
                                     (int)in_features, xq, p.kp, stream),
               "repack_i8");
    else
      a = static_cast<const signed char*>(x);
  }
  const signed char* b = reinterpret_cast<const signed char*>(weight);
  if (p.pack_w) {
    DCN_CUDA(dcn::launch_repack_i8(b, out_features, (int)in_features, wq, p.kp, stream),
             "repack_i8");
    b = wq;
  }
  dcn::GemmProblem g{};
  g.a = rows_i8(a, tokens, in_features, p.kp, 1);
  g.b = rows_i8(b, out_features, in_features, p.kp, 1);
  g.M = (int)tokens;
  g.N = (int)out_features;
  g.K = (int)in_features;
  g.batch = 1;
  g.int8 = true;
  g.epi.mode = dcn::kEpiRows;
  g.epi.out = output;
  g.epi.out_type = out_type;
  g.epi.wide_ok =
      out_features * (int64_t)type_bytes(out_type) % 16 == 0 && aligned16(output) ? 1 : 0;
  g.epi.row_scale = as;
  g.epi.col_scale = weight_scale;
  g.epi.bias = bias;
  g.epi.bias_type = bias_type;
  g.wait_limit = wait_limit(flags);
  g.no_async = flags & DCN_TEST_WAIT_TIMEOUT ? 1 : 0;
  DCN_CUDA(dcn::launch_gemm(g, stream), "int8_gemm");
  return DCN_OK;
}

DCN_API size_t dcn_deform_int8_workspace_size(const dcn_shape* shape, int type, uint32_t flags) {
  DeformInt8 d;
  return deform_int8_plan(shape, type, flags, d, "dcn_deform_int8") == DCN_OK ? d.total : 0;
}

DCN_API int dcn_deform_int8(const dcn_shape* shape, int type, const void* input,
                            const int8_t* weight, const float* weight_scale, const void* offset,
                            const void* mask, const void* bias, int bias_type, void* output,
                            int out_type, uint32_t flags, void* workspace, size_t workspace_bytes,
                            void* stream_) {
  g_last_error.clear();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  DeformInt8 d;
  const int rc = deform_int8_plan(shape, type, flags, d, "dcn_deform_int8");
  if (rc != DCN_OK) return rc;
  dcn::Geom& g = d.g;
  g.use_mask = mask != nullptr;
  g.use_bias = bias != nullptr;
  g.mask_logits = (flags & DCN_MASK_LOGITS) && mask != nullptr ? 1 : 0;
  apply_test_flags(g, flags);
  DCN_CHECK(float_type(out_type) && (bias == nullptr || float_type(bias_type)),
            "dcn_deform_int8: output and bias must be float32, bfloat16 or float16");
  DCN_CHECK(g.C > 0, "dcn_deform_int8: at least one input channel is needed");
  if (g.NP == 0 || g.outC == 0) return DCN_OK;
  DCN_CHECK((input != nullptr || g.HW == 0) && weight != nullptr && weight_scale != nullptr &&
                offset != nullptr && output != nullptr,
            "dcn_deform_int8: input, weight, weight_scale, offset and output must not be NULL");
  if (workspace == nullptr || workspace_bytes < d.total)
    return fail(DCN_ERR_WORKSPACE, "dcn_deform_int8: workspace too small");
  Carve ws(workspace);
  void* xt = ws.take<void>(d.stage_bytes);
  signed char* col = ws.take<signed char>(d.col_bytes);
  float* scale = ws.take<float>(d.scale_bytes);
  signed char* wp = ws.take<signed char>(d.weight_bytes);
  const void* x = input;
  if (!d.nhwc) {
    if (type == DCN_TYPE_F32)
      DCN_CUDA(dcn::launch_nchw_to_nhwc(static_cast<const float*>(input), static_cast<float*>(xt),
                                        g.N, g.C, g.HW, true, nullptr, stream),
               "nchw_to_nhwc");
    else
      DCN_CUDA(dcn::launch_nchw_to_nhwc_bf16(input, xt, g.N, g.C, g.HW, true, stream),
               "nchw_to_nhwc");
    x = xt;
  }
  const signed char* w = reinterpret_cast<const signed char*>(weight);
  if (d.pack || !aligned16(w)) {
    DCN_CUDA(dcn::launch_repack_i8(w, g.outC, (int)d.kg, wp, d.kp, stream), "repack_i8");
    w = wp;
  }
  for (int64_t p0 = 0; p0 < g.NP; p0 += d.chunk) {
    const int np = (int)(g.NP - p0 < d.chunk ? g.NP - p0 : d.chunk);
    DCN_CUDA(dcn::launch_sample_i8(g, x, type, offset, mask, p0, np, col, (int)d.kp, scale,
                                   stream),
             "sample_i8");
    dcn::GemmProblem q{};
    q.a = rows_i8(col, np, d.kg, d.kp, g.G);
    q.b = rows_i8(w, g.Og, d.kg, d.kp, g.G);
    q.M = np;
    q.N = g.Og;
    q.K = (int)d.kg;
    q.batch = g.G;
    q.int8 = true;
    q.epi.mode = dcn::kEpiPlanes;
    q.epi.out = output;
    q.epi.out_type = out_type;
    q.epi.row_scale = scale;
    q.epi.row_scale_batch = np;
    q.epi.col_scale = weight_scale;
    q.epi.bias = bias;
    q.epi.bias_type = bias_type;
    q.epi.pixels = g.P;
    q.epi.channels = g.outC;
    q.epi.m_base = (int)p0;
    q.epi.pixel_pairs = np % 2 == 0 && p0 % 2 == 0 && g.P % 2 == 0 &&
                        (reinterpret_cast<uintptr_t>(output) & 3) == 0;
    q.wait_limit = g.wait_limit;
    q.no_async = g.no_async;
    DCN_CUDA(dcn::launch_gemm(q, stream), "int8_gemm");
  }
  return DCN_OK;
}

}  // extern "C"
