// dcn_capi_util.h -- what the C entry points share: the error message of the
// calling thread, argument checks, the kernel profiler, geometry validation.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <string>
#include <vector>

#include "dcn_b200.h"
#include "dcn_common.cuh"
#include "dcn_tc.h"

namespace dcn {
namespace capi {

inline thread_local std::string g_last_error;

inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

inline int cuda_fail(cudaError_t e, const char* where) {
  return fail(DCN_ERR_CUDA, "%s: CUDA error %d (%s)", where, (int)e, cudaGetErrorString(e));
}

#define DCN_CHECK(cond, ...)                                  \
  do {                                                        \
    if (!(cond)) return fail(DCN_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
  } while (0)

// ---- kernel profiler: a CUDA event pair around every launch when enabled --
// (tracing for the bench and for users; off by default, one branch per
// launch when off).
struct ProfRecord {
  const char* name;
  cudaEvent_t start, stop;
};
inline std::mutex g_prof_mu;
inline bool g_prof_on = false;
inline std::vector<ProfRecord> g_prof_recs;
inline std::vector<cudaEvent_t> g_prof_pool;

inline cudaEvent_t prof_event() {
  if (!g_prof_pool.empty()) {
    cudaEvent_t e = g_prof_pool.back();
    g_prof_pool.pop_back();
    return e;
  }
  cudaEvent_t e = nullptr;
  if (cudaEventCreate(&e) != cudaSuccess) return nullptr;
  return e;
}

struct ProfScope {
  const char* name;
  cudaStream_t stream;
  cudaEvent_t start = nullptr;
  ProfScope(const char* n, cudaStream_t s) : name(n), stream(s) {
    if (!g_prof_on) return;
    std::lock_guard<std::mutex> lk(g_prof_mu);
    start = prof_event();
    if (start) cudaEventRecord(start, stream);
  }
  void done() {
    if (!start) return;
    std::lock_guard<std::mutex> lk(g_prof_mu);
    cudaEvent_t stop = prof_event();
    if (stop) {
      cudaEventRecord(stop, stream);
      g_prof_recs.push_back({name, start, stop});
    } else {
      g_prof_pool.push_back(start);
    }
  }
};

#define DCN_CUDA(expr, where)                             \
  do {                                                    \
    ProfScope ps_(where, stream);                         \
    cudaError_t e_ = (expr);                              \
    ps_.done();                                           \
    if (e_ != cudaSuccess) return cuda_fail(e_, where);   \
  } while (0)

#define DCN_CUDA_ON(strm, expr, where)                    \
  do {                                                    \
    ProfScope ps_(where, strm);                           \
    cudaError_t e_ = (expr);                              \
    ps_.done();                                           \
    if (e_ != cudaSuccess) return cuda_fail(e_, where);   \
  } while (0)

constexpr size_t kAlign = 256;
inline size_t align_up(size_t v) { return (v + kAlign - 1) / kAlign * kAlign; }

// DCN_TEST_WAIT_TIMEOUT: the tensor-core kernels' TMA producers issue
// nothing and every wait gives up after a short budget.
inline void apply_test_flags(dcn::Geom& g, uint32_t flags) {
  if (flags & DCN_TEST_WAIT_TIMEOUT) {
    g.no_async = 1;
    g.wait_limit = dcn::kTestWaitLimit;
  }
}

// Validation shared by forward and backward (.mm:202-267, :693-760).
inline int make_geom(const dcn_shape* s, bool use_mask, bool use_bias, dcn::Geom& g,
              const char* op) {
  DCN_CHECK(s != nullptr, "%s: shape must not be NULL", op);
  DCN_CHECK(s->batch >= 0 && s->in_channels >= 0 && s->height >= 0 && s->width >= 0 &&
                s->out_channels >= 0,
            "%s: tensor dimensions must be non-negative", op);
  DCN_CHECK(s->kernel_h > 0 && s->kernel_w > 0, "kernel dims must be positive");
  DCN_CHECK(s->groups > 0, "groups must be positive, got %lld", (long long)s->groups);
  DCN_CHECK(s->stride_h > 0 && s->stride_w > 0, "stride must be positive");
  DCN_CHECK(s->dilation_h > 0 && s->dilation_w > 0, "dilation must be positive");
  DCN_CHECK(s->pad_h >= 0 && s->pad_w >= 0, "padding must be non-negative");
  DCN_CHECK(s->in_channels % s->groups == 0, "channels (%lld) not divisible by groups (%lld)",
            (long long)s->in_channels, (long long)s->groups);
  DCN_CHECK(s->out_channels % s->groups == 0,
            "out_channels (%lld) not divisible by groups (%lld)", (long long)s->out_channels,
            (long long)s->groups);
  const int64_t Ho = (s->height + 2 * s->pad_h - s->dilation_h * (s->kernel_h - 1) - 1) / s->stride_h + 1;
  const int64_t Wo = (s->width + 2 * s->pad_w - s->dilation_w * (s->kernel_w - 1) - 1) / s->stride_w + 1;
  DCN_CHECK(Ho > 0 && Wo > 0, "calculated output size (%lldx%lld) is non-positive",
            (long long)Ho, (long long)Wo);
  DCN_CHECK(s->deformable_groups > 0, "deformable_groups must be positive, got %lld",
            (long long)s->deformable_groups);
  DCN_CHECK(s->in_channels % s->deformable_groups == 0,
            "channels (%lld) not divisible by deformable_groups (%lld)",
            (long long)s->in_channels, (long long)s->deformable_groups);
  const int64_t kk = s->kernel_h * s->kernel_w;
  const int64_t lim = (int64_t)1 << 31;
  // per-image element counts are indexed in int32 inside the kernels
  if (s->in_channels * s->height * s->width >= lim || s->out_channels * Ho * Wo >= lim ||
      2 * s->deformable_groups * kk * Ho * Wo >= lim || s->batch * Ho * Wo >= lim ||
      s->out_channels * (s->in_channels / s->groups) * kk >= lim || s->height * s->width > 65535LL * 32)
    return fail(DCN_ERR_UNSUPPORTED, "%s: per-image tensor sizes beyond 2^31 elements are not supported", op);
  g.N = (int)s->batch; g.C = (int)s->in_channels; g.H = (int)s->height; g.W = (int)s->width;
  g.outC = (int)s->out_channels; g.kh = (int)s->kernel_h; g.kw = (int)s->kernel_w;
  g.sh = (int)s->stride_h; g.sw = (int)s->stride_w; g.ph = (int)s->pad_h; g.pw = (int)s->pad_w;
  g.dh = (int)s->dilation_h; g.dw = (int)s->dilation_w;
  g.G = (int)s->groups; g.dg = (int)s->deformable_groups;
  g.Ho = (int)Ho; g.Wo = (int)Wo;
  g.use_mask = use_mask ? 1 : 0; g.use_bias = use_bias ? 1 : 0;
  g.mask_logits = 0;
  g.oy0 = 0;
  g.wait_limit = dcn::kWaitLimit;
  g.no_async = 0;
  g.Cg = g.C / g.G; g.Og = g.outC / g.G; g.cpg = g.dg ? g.C / g.dg : 0;
  g.kk = g.kh * g.kw; g.P = g.Ho * g.Wo; g.HW = g.H * g.W;
  g.NP = (long long)g.N * g.P;
  return DCN_OK;
}

}  // namespace capi
}  // namespace dcn
