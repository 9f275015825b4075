// dcn_ortho.cu -- Newton-Schulz orthogonalisation of a batch of matrices, and
// the momentum optimiser step that uses it.
//
// X <- a X + (b S + c S S) X with S = X X^T, some steps over, starting from
// G / (|G| + eps).  Each step multiplies X by a polynomial of S, and all those
// polynomials commute, so a run of steps needs X only at its ends:
//   S = X X^T;  each step: P = a I + b S + c S S;  Q <- P Q;  S <- P (P S);
//   then X <- Q X.
// For m x n with n = 9 m (a layer of 3 x 3 taps) two runs for five steps take
// 68 m^3 flops of symmetric and plain products, the recurrence as written 140.
//
// A run cannot be long.  The rounding of S, 2^-22 of its largest value with
// two fp16 terms, is a larger relative error of the small singular values'
// part of it, and every further step of the run multiplies that by a^2 while
// those values grow.  A run ends before the product of its a^2 passes 150:
// three steps of the usual 3.4445, two runs for five steps; results of 16 bits
// do not see the difference (squarer matrices: run_length below).  For fp32
// results the first run, where one direction can hold nearly all of |X|, ends
// before 12: two steps; so does every run of more than 256 directions.
// Emulated in 64 bits on 64 x 576 with a few strong directions, the relative
// error is 5e-7 with runs (2, 3) and 4.6e-6 with (3, 2), fp32 products as
// written 1.4e-6; one run of five steps diverges on steep spectra.
#include "dcn_ortho.h"

#include <cmath>

#include "dcn_capi_util.h"
#include "dcn_dense_common.cuh"
#include "dcn_launch.h"
#include "dcn_ortho_chain.h"

namespace dcn {

namespace {

// Powers of two that bring fp16 into the middle of its range: S (at most 1.5
// in a run of the usual steps, 8 at most), P (its coefficients, 16 at most),
// Q (products of at most 150^(1/2) with room for 256).
constexpr float kScaleS = 8192.f, kScaleP = 4096.f, kScaleQ = 256.f;
constexpr int kPartials = 256;  // sums of squares a matrix, at most
constexpr float kRunLimit = 150.f, kShortRunLimit = 12.f;

struct PrepArgs {
  const void* in[kGemmMaxList];
  float* momentum[kGemmMaxList];
  double* partial;  // [count][kPartials]
  float* r1;        // [count] true X = r1 * stored X
  float* r2;        // [count] r1 squared
  unsigned short* x;
  long long numel, pitch, term_stride, batch_stride;
  int rows, cols, type, terms, target;  // |stored X| lies in [2^target, 2^(target + 1))
  int muon, nesterov, vec, partials;
  float beta, rest, eps;
};

template <int T>
__device__ __forceinline__ float load1(const void* p, long long i) {
  if constexpr (T == kF32) return static_cast<const float*>(p)[i];
  else if constexpr (T == kBF16T)
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  else return __half2float(static_cast<const __half*>(p)[i]);
}
// Eight values from i, a multiple of eight behind a 16-byte aligned pointer.
template <int T>
__device__ __forceinline__ void load8(const void* p, long long i, float (&v)[8]) {
  if constexpr (T == kF32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = q[0], b = q[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a =
        *reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p) + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = dense::unpack2<T>(w[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}

// The update's value from the gradient and the new momentum.
__device__ __forceinline__ float update_of(const PrepArgs& a, float g, float m) {
  return a.nesterov ? a.rest * g + a.beta * m : m;
}

// New momentum, and sums of squares of the update in 64 bits: any fp32 input
// keeps its norm, and the partial sums' fixed order keeps the result.  Bound
// by HBM (a step reads the gradient, reads and writes the momentum).
template <int T>
__global__ void __launch_bounds__(256) ortho_norm_kernel(const __grid_constant__ PrepArgs a) {
  const int b = blockIdx.y;
  const void* in = a.in[b];
  float* mom = a.momentum[b];
  const long long step = (long long)gridDim.x * 256;
  const long long first = (long long)blockIdx.x * 256 + threadIdx.x;
  double s = 0.0;
  const long long vecs = a.vec ? a.numel / 8 : 0;
  for (long long q = first; q < vecs; q += step) {
    float v[8];
    load8<T>(in, 8 * q, v);
    if (a.muon) {
      float m[8];
      load8<kF32>(mom, 8 * q, m);
#pragma unroll
      for (int j = 0; j < 8; ++j) m[j] = a.beta * m[j] + a.rest * v[j];
      float4* o = reinterpret_cast<float4*>(mom + 8 * q);
      o[0] = make_float4(m[0], m[1], m[2], m[3]);
      o[1] = make_float4(m[4], m[5], m[6], m[7]);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = update_of(a, v[j], m[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (double)v[j] * (double)v[j];
  }
  for (long long i = 8 * vecs + first; i < a.numel; i += step) {
    float v = load1<T>(in, i);
    if (a.muon) {
      const float m = a.beta * mom[i] + a.rest * v;
      mom[i] = m;
      v = update_of(a, v, m);
    }
    s += (double)v * (double)v;
  }
  __shared__ double red[8];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) s += red[w];
    a.partial[b * kPartials + blockIdx.x] = s;
  }
}

// X as fp16 terms of the update times a power of two: exact for 16-bit inputs
// (but for what lies 2^-24 below the largest), and 1 / (norm + eps) is left to
// the products' epilogues in fp32.
template <int T>
__global__ void __launch_bounds__(256) ortho_scale_kernel(const __grid_constant__ PrepArgs a) {
  const int b = blockIdx.y;
  __shared__ float f1, f2;
  dense::grid_launch_dependents();
  dense::grid_wait();
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int i = threadIdx.x; i < a.partials; i += 32) s += a.partial[b * kPartials + i];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) {
      const double norm = sqrt(s);
      int k = 0;
      if (norm > 0.0 && isfinite(norm)) k = a.target - ilogb(norm);
      f1 = (float)ldexp(1.0, k / 2);
      f2 = (float)ldexp(1.0, k - k / 2);
      if (blockIdx.x == 0) {
        // a norm that is not finite leaves nothing to scale by; a matrix of zeros
        // is its own answer, whatever 1 / eps (squared for the Gram matrix) is
        const float r = !isfinite(norm) ? __int_as_float(0x7fc00000)
                        : norm == 0.0   ? 0.f
                                        : (float)ldexp(1.0 / (norm + (double)a.eps), -k);
        a.r1[b] = r;
        a.r2[b] = r * r;
      }
    }
  }
  __syncthreads();
  const void* in = a.in[b];
  const float* mom = a.momentum[b];
  const float c1 = f1, c2 = f2;
  const int chunks = (int)(a.pitch / 8);
  const bool vec = a.vec && a.cols % 8 == 0;
  const long long total = (long long)a.rows * chunks;
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < total;
       q += (long long)gridDim.x * 256) {
    const int row = (int)(q / chunks), c = (int)(q - (long long)row * chunks) * 8;
    const long long i = (long long)row * a.cols + c;
    float v[8];
    if (vec) {
      load8<T>(in, i, v);
      if (a.muon) {
        float m[8];
        load8<kF32>(mom, i, m);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = update_of(a, v[j], m[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = 0.f;
        if (c + j < a.cols) {
          v[j] = load1<T>(in, i + j);
          if (a.muon) v[j] = update_of(a, v[j], mom[i + j]);
        }
      }
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      dense::split2(dense::pair(v[2 * j] * c1 * c2, v[2 * j + 1] * c1 * c2), hi[j], lo[j]);
    unsigned short* x = a.x + (long long)b * a.batch_stride + (long long)row * a.pitch + c;
    *reinterpret_cast<uint4*>(x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (a.terms == 2)
      *reinterpret_cast<uint4*>(x + a.term_stride) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

constexpr size_t align_up(size_t v) { return (v + 255) / 256 * 256; }

struct Layout {
  int m, n;  // smaller and larger side
  bool wide;
  long long xpitch, xterm;  // elements
  long long spitch, sterm;
  size_t x_bytes, s_bytes;  // one matrix, both terms of a slot / as many as needed
  int x_terms;
  size_t scalars, partials, total;
};

Layout layout_of(const OrthoShape& s, int count) {
  Layout l;
  l.wide = s.rows <= s.cols;
  l.m = l.wide ? s.rows : s.cols;
  l.n = l.wide ? s.cols : s.rows;
  auto up8 = [](long long v) { return (v + 7) / 8 * 8; };
  l.xpitch = up8(s.cols);
  l.xterm = l.xpitch * s.rows;
  l.spitch = up8(l.m);
  l.sterm = l.spitch * l.m;
  l.x_terms = s.first_terms > s.later_terms ? s.first_terms : s.later_terms;
  l.x_bytes = align_up((size_t)count * l.x_terms * l.xterm * 2);
  l.s_bytes = align_up((size_t)count * 2 * l.sterm * 2);
  l.partials = align_up((size_t)count * kPartials * sizeof(double));
  l.scalars = align_up((size_t)count * 2 * sizeof(float));
  l.total = l.partials + l.scalars + 2 * l.x_bytes + 5 * l.s_bytes;
  return l;
}

int run_length(const OrthoShape& s, int first) {
  // Matrices near enough to square gain nothing from longer runs (X costs
  // little more than S) and lose launches: 1024 x 1024 float32 251 us in single
  // steps, 294 in runs of 2 and 3; 1024 x 4096 531 and 413.  With X of one
  // term its rounding comes after a run of two, and single steps of one-term
  // squares follow: 1024 x 2048 bf16 207 us, 254 in runs of 3 and 2; 1024 x
  // 4096 274 and 293, which no longer pays for the rounding.
  const int m = s.rows < s.cols ? s.rows : s.cols, n = s.rows < s.cols ? s.cols : s.rows;
  const bool square = m > kChainMax && n < (s.later_terms == 1 ? 3LL : 2LL) * m;
  if (square && (first > 0 || s.later_terms == 2)) return 1;
  // The more directions, and the squarer the matrix, the more of them are still
  // small in the second run: up to 256 that run may be long, where the error stays
  // below twice that of fp32 products as written.  From some 350 on it would
  // pass that, for a twentieth of the time at best.  Relative errors (largest of
  // three gradients of rank m / 16 under noise) and us with runs (2, 3), with (2, 2, 1), and the
  // error of fp32 products:
  //   128 x 1152  0.80e-6  79    0.99e-6  90   1.05e-6  (the chain kernel's)
  //   192 x 400   2.2e-6  110    1.7e-6  106   1.6e-6
  //   256 x 520   3.5e-6  127    2.1e-6  130   1.9e-6
  //   256 x 2304  2.8e-6  132    2.7e-6  136   1.8e-6
  //   300 x 700   4.1e-6  136    2.3e-6  135   2.2e-6
  //   300 x 2700  3.4e-6  146    3.0e-6  148   2.1e-6
  //   384 x 1600  5.2e-6  157    3.1e-6  160   2.7e-6
  //   512 x 4608  6.7e-6  196    3.7e-6  206   3.4e-6
  //   1400 x 2900 9.0e-6  594    1.6e-6  611   2.8e-6
  const bool f32 = s.first_terms == 2 && s.later_terms == 2;
  const bool few = f32 ? first == 0 || m > 256 || n < 2LL * m : square;
  const float limit = few ? kShortRunLimit : kRunLimit;
  float grown = 1.f;
  int k = first;
  while (k + 1 < s.steps) {
    const float a = s.coef[3 * k];
    grown *= a * a > 1.f ? a * a : 1.f;
    if (!(grown <= limit)) break;
    ++k;
  }
  return k + 1 - first;
}

int log2_floor(double v) {
  int e = 0;
  while (v >= 2.0) {
    v *= 0.5;
    ++e;
  }
  return e;
}

}  // namespace

size_t ortho_workspace_bytes(const OrthoShape& s, int count) {
  return layout_of(s, count).total + 256;
}

cudaError_t launch_ortho(const OrthoShape& s, const OrthoChunk& c, void* workspace,
                         long long wait_limit, int no_async, cudaStream_t stream,
                         const char** stage) {
  const Layout l = layout_of(s, c.count);
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(workspace) + 255) &
                                     ~(uintptr_t)255);
  double* partial = reinterpret_cast<double*>(ws);
  float* r1 = reinterpret_cast<float*>(ws + l.partials);
  float* r2 = r1 + c.count;
  char* at = ws + l.partials + l.scalars;
  auto take = [&](size_t bytes) {
    unsigned short* p = reinterpret_cast<unsigned short*>(at);
    at += bytes;
    return p;
  };
  unsigned short* x[2] = {take(l.x_bytes), take(l.x_bytes)};
  unsigned short *S = take(l.s_bytes), *P = take(l.s_bytes), *C = take(l.s_bytes);
  unsigned short* Q[2] = {take(l.s_bytes), take(l.s_bytes)};

  // |X| = 1: entries of about 1 on average, and 2^15 at the most
  const double area = (double)s.rows * s.cols;
  int target = log2_floor(area) / 2;
  if (target > 14) target = 14;
  // between runs |X| is up to sqrt(m), entries about n^-1/2 and 1.5 at the most
  int later = log2_floor((double)l.n) / 2 + 4;
  if (later > 14) later = 14;
  const float later_scale = (float)(1 << later);

  PrepArgs p;
  for (int i = 0; i < c.count; ++i) {
    p.in[i] = c.in[i];
    p.momentum[i] = c.momentum[i];
  }
  p.partial = partial;
  p.r1 = r1;
  p.r2 = r2;
  p.x = x[0];
  p.numel = (long long)s.rows * s.cols;
  p.pitch = l.xpitch;
  p.term_stride = l.xterm;
  p.batch_stride = l.xterm * s.first_terms;
  p.rows = s.rows;
  p.cols = s.cols;
  p.type = s.type;
  p.terms = s.first_terms;
  p.target = target;
  p.muon = c.muon;
  p.nesterov = c.nesterov;
  p.beta = c.beta;
  p.rest = c.rest;
  p.eps = s.eps;
  p.vec = 1;
  for (int i = 0; i < c.count; ++i)
    if ((reinterpret_cast<uintptr_t>(c.in[i]) | reinterpret_cast<uintptr_t>(c.momentum[i])) & 15)
      p.vec = 0;
  // 4096 values a block at least, and some eight blocks an SM over all matrices
  long long parts = (p.numel + 4095) / 4096;
  const long long most = (8LL * device_sm_count() + c.count - 1) / c.count;
  if (parts > most) parts = most;
  p.partials = (int)(parts < kPartials ? parts : kPartials);
  *stage = "ortho_norm";
  auto norm = s.type == kF32 ? ortho_norm_kernel<kF32>
              : s.type == kBF16T ? ortho_norm_kernel<kBF16T> : ortho_norm_kernel<kF16T>;
  capi::ProfScope norm_scope(*stage, stream);
  norm<<<dim3(p.partials, c.count), 256, 0, stream>>>(p);
  norm_scope.done();
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  *stage = "ortho_scale";
  const long long chunks = s.rows * (l.xpitch / 8);
  long long blocks = (chunks + 511) / 512;
  if (blocks > most) blocks = most;
  auto scale = s.type == kF32 ? ortho_scale_kernel<kF32>
               : s.type == kBF16T ? ortho_scale_kernel<kBF16T> : ortho_scale_kernel<kF16T>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, (unsigned)c.count);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  capi::ProfScope scale_scope(*stage, stream);
  e = cudaLaunchKernelEx(&cfg, scale, p);
  scale_scope.done();
  if (e != cudaSuccess) return e;

  int sq_terms = 2;  // of the square matrices
  auto square = [&](const unsigned short* base) {
    GemmOperand o{base, l.m, l.m, l.spitch, sq_terms, l.sterm, c.count, 2 * l.sterm, false};
    return o;
  };
  auto product = [&](const char* name, const GemmOperand& a, const GemmOperand& b, int M, int N,
                     int K, GemmEpiArgs epi, bool sym) {
    GemmProblem g{};
    g.a = a;
    g.b = b;
    g.M = M;
    g.N = N;
    g.K = K;
    g.batch = c.count;
    g.sym = sym;
    g.fine = s.type == kF32;
    g.coarse = s.later_terms == 1;
    g.after_ours = true;
    g.epi = epi;
    g.wait_limit = wait_limit;
    g.no_async = no_async;
    *stage = name;
    capi::ProfScope scope(name, stream);
    const cudaError_t err = launch_gemm(g, stream);
    scope.done();
    return err;
  };
  auto to_square = [&](unsigned short* out, float factor) {
    GemmEpiArgs q{};
    q.mode = kEpiTerms;
    q.factor = factor;
    q.out16 = out;
    q.out_terms = sq_terms;
    q.pitch = l.spitch;
    q.term_stride = l.sterm;
    q.batch_stride = 2 * l.sterm;
    return q;
  };

  int terms = s.first_terms, cur = 0;
  for (int k = 0; k < s.steps;) {
    const int run = run_length(s, k);
    const bool first = k == 0, last = k + run == s.steps;
    // Where X keeps 11 bits between runs, so do S and P of a later run of one
    // step: they meet no direction that is still small but with a factor of at
    // most a, once a step (longer runs multiply S into itself, and earlier
    // ones have more steps to come).  1024 x 1024 bf16, relative error before
    // the result's rounding 0.6e-3 -> 1.1e-3, behind it 1.76e-3 -> 1.96e-3
    // (1.66e-3 for an exact result); half of the operations of those steps.
    // What S loses reaches P times |b| + 2 |c|, 8.9 for the usual coefficients;
    // larger ones keep two terms (4.125, -11.75, 8.5 on 300 x 500 bf16: 4.5e-3
    // with one).  So do few directions: the chain kernel takes two.
    const float* abc0 = s.coef + 3 * k;
    const bool mild = std::fabs(abc0[1]) + 2.f * std::fabs(abc0[2]) <= 9.f;
    sq_terms = l.m > kChainMax && s.later_terms == 1 && run == 1 && !first && mild ? 1 : 2;
    const GemmOperand X{x[cur], s.rows, s.cols, l.xpitch, terms, l.xterm, c.count,
                        terms * l.xterm, !l.wide};
    const float xs = first ? 1.f : 1.f / later_scale;
    GemmEpiArgs q = to_square(S, xs * xs * kScaleS);
    if (first) q.scale = r2;
    e = product("ortho_gram", X, X, l.m, l.m, l.n, q, true);
    if (e != cudaSuccess) return e;
    unsigned short* prod = nullptr;  // Q so far
    if (l.m <= kChainMax) {  // the run's products in one launch
      ChainArgs a;
      a.m = l.m;
      a.run = run;
      for (int i = 0; i < 3 * run; ++i) a.coef[i] = s.coef[3 * k + i];
      a.scale_s = kScaleS;
      a.scale_p = kScaleP;
      a.scale_q = kScaleQ;
      a.out = prod = Q[0];
      a.pitch = l.spitch;
      a.term_stride = l.sterm;
      a.batch_stride = 2 * l.sterm;
      *stage = "ortho_chain";
      capi::ProfScope scope(*stage, stream);
      e = launch_ortho_chain(a, square(S), c.count, wait_limit, no_async, stream);
      scope.done();
      if (e != cudaSuccess) return e;
    }
    for (int i = 0; l.m > kChainMax && i < run; ++i) {
      const float* abc = s.coef + 3 * (k + i);
      unsigned short* poly = prod == nullptr ? Q[0] : P;
      const float to = prod == nullptr ? kScaleQ : kScaleP;
      q = to_square(poly, abc[2] * to / (kScaleS * kScaleS));
      q.mode = kEpiPoly;
      q.diag = abc[0] * to;
      q.lin = abc[1] * to / kScaleS;
      q.lin16 = S;
      e = product("ortho_poly", square(S), square(S), l.m, l.m, l.m, q, true);
      if (e != cudaSuccess) return e;
      if (i + 1 < run) {  // S <- P (P S)
        e = product("ortho_square", square(poly), square(S), l.m, l.m, l.m,
                    to_square(C, 1.f / to), true);
        if (e != cudaSuccess) return e;
        e = product("ortho_square", square(poly), square(C), l.m, l.m, l.m,
                    to_square(S, 1.f / to), true);
        if (e != cudaSuccess) return e;
      }
      if (prod == nullptr) {
        prod = poly;
      } else {
        unsigned short* next = prod == Q[0] ? Q[1] : Q[0];
        e = product("ortho_join", square(poly), square(prod), l.m, l.m, l.m,
                    to_square(next, 1.f / to), true);
        if (e != cudaSuccess) return e;
        prod = next;
      }
    }
    GemmEpiArgs o{};
    o.factor = xs / kScaleQ;
    if (first) o.scale = r1;
    if (last) {
      o.mode = c.muon ? kEpiAxpy : kEpiOut;
      if (c.muon) {
        o.factor *= c.step;
        o.keep = c.keep;
      }
      o.out_type = s.type;
      const int es = s.type == kF32 ? 4 : 2;
      o.wide_ok = (long long)s.cols * es % 16 == 0;
      for (int i = 0; i < c.count; ++i) {
        o.list[i] = c.out[i];
        if (reinterpret_cast<uintptr_t>(c.out[i]) % 16 != 0) o.wide_ok = 0;
      }
    } else {
      o.mode = kEpiTerms;
      o.factor *= later_scale;
      o.out16 = x[cur ^ 1];
      o.out_terms = s.later_terms;
      o.pitch = l.xpitch;
      o.term_stride = l.xterm;
      o.batch_stride = s.later_terms * l.xterm;
    }
    // Q X with X's rows along K, or X Q with X as it lies
    GemmOperand t = X;
    t.k_rows = l.wide;
    e = l.wide ? product("ortho_apply", square(prod), t, l.m, l.n, l.m, o, false)
               : product("ortho_apply", t, square(prod), l.n, l.m, l.m, o, false);
    if (e != cudaSuccess) return e;
    cur ^= 1;
    terms = s.later_terms;
    k += run;
  }
  return cudaSuccess;
}

}  // namespace dcn
