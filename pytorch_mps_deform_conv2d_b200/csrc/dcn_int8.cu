// dcn_int8.cu -- 8-bit codes of rows and of sampled columns (see dcn_int8.h).
#include "dcn_int8.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dcn_launch.h"

namespace dcn {

namespace {

template <int T>
__device__ __forceinline__ float ld(const void* p, long long i) {
  if constexpr (T == kF32) return __ldg(static_cast<const float*>(p) + i);
  else if constexpr (T == kBF16T)
    return __uint_as_float((uint32_t)__ldg(static_cast<const unsigned short*>(p) + i) << 16);
  else
    return __half2float(
        __ushort_as_half(__ldg(static_cast<const unsigned short*>(p) + i)));
}

// |v| as bits: ordered like the values, NaN above infinity, so a plain integer
// maximum keeps either.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A row's scale and the code of v under it.  Divisions, not products with a
// reciprocal: the codes are those of the formula.
__device__ __forceinline__ float scale_of(unsigned top) {
  return __fdiv_rn(__uint_as_float(top), 127.f);
}
__device__ __forceinline__ int code_of(float v, float scale, bool usable) {
  if (!usable) return 0;
  const float q = rintf(__fdiv_rn(v, scale));
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}
__device__ __forceinline__ bool usable_scale(float s) { return s > 0.f && s <= 3.402823466e38f; }

template <int T>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const void* __restrict__ x, int cols, long long ldx,
                     signed char* __restrict__ q, long long ldq, float* __restrict__ scale) {
  const long long row = blockIdx.x;
  unsigned top = 0;
  for (int c = threadIdx.x; c < cols; c += 256) top = max(top, abs_bits(ld<T>(x, row * ldx + c)));
  __shared__ unsigned red[8];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < 8; ++w) top = max(top, red[w]);
  const float s = scale_of(top);
  const bool ok = usable_scale(s);
  if (threadIdx.x == 0) scale[row] = s;
  for (int c = threadIdx.x; c < cols; c += 256)
    q[row * ldq + c] = (signed char)code_of(ld<T>(x, row * ldx + c), s, ok);
}

__global__ void __launch_bounds__(256)
repack_i8_kernel(const signed char* __restrict__ in, long long rows, int cols,
                 signed char* __restrict__ out, long long ldo) {
  const long long n = rows * cols;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n;
       i += (long long)gridDim.x * 256) {
    const long long r = i / cols;
    out[r * ldo + (i - r * cols)] = in[i];
  }
}

// One warp per (pixel, group).  The taps' samples are made in fp32, in shared
// memory (STAGED) or, for columns that do not fit there, made twice.
template <int T, bool STAGED>
__global__ void __launch_bounds__(256)
sample_i8_kernel(Geom g, const void* __restrict__ x, const void* __restrict__ off,
                 const void* __restrict__ mask, long long p0, int np,
                 signed char* __restrict__ col, int kp, float* __restrict__ scale) {
  extern __shared__ float stage[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * (blockDim.x >> 5) + warp;
  if (item >= (long long)np * g.G) return;
  const int gi = (int)(item / np), lp = (int)(item - (long long)gi * np);
  const long long pix = p0 + lp;
  const int n = (int)(pix / g.P), p = (int)(pix - (long long)n * g.P);
  const int oy = p / g.Wo, ox = p - oy * g.Wo;
  const int K = g.kk * g.Cg;
  float* mine = stage + (size_t)warp * K;
  signed char* out = col + ((long long)gi * np + lp) * kp;
  const long long img = (long long)n * g.HW * g.C;
  unsigned top = 0;
  float s = 0.f;
  bool ok = false;
  for (int pass = 0; pass < (STAGED ? 1 : 2); ++pass) {
    if (pass == 1) {
      top = __reduce_max_sync(0xffffffffu, top);
      s = scale_of(top);
      ok = usable_scale(s);
    }
    for (int k = 0; k < g.kk; ++k) {
      const int ki = k / g.kw, kj = k - ki * g.kw;
      for (int c0 = 0; c0 < g.Cg;) {  // the channels of one deformable group
        const int ch = gi * g.Cg + c0, dgi = ch / g.cpg;
        const int run = min(g.Cg - c0, (dgi + 1) * g.cpg - ch);
        const long long oi = off_h_index(g, n, dgi, k, p);
        float h, w;
        sample_pos(g, oy, ox, ki, kj, ld<T>(off, oi), ld<T>(off, oi + g.P), h, w);
        float m = 1.f;
        if (g.use_mask) {
          m = ld<T>(mask, mask_index(g, n, dgi, k, p));
          if (g.mask_logits) m = 1.f / (1.f + expf(-m));
        }
        const Sample sp = make_sample(h, w, g.H, g.W);
        const float w1 = sp.w1 * m, w2 = sp.w2 * m, w3 = sp.w3 * m, w4 = sp.w4 * m;
        for (int c = lane; c < run; c += 32) {
          float v = 0.f;
          // dropped corners are not read: what lies there must not matter
          if (sp.live & 1u) v += w1 * ld<T>(x, img + (long long)sp.i1 * g.C + ch + c);
          if (sp.live & 2u) v += w2 * ld<T>(x, img + (long long)sp.i2 * g.C + ch + c);
          if (sp.live & 4u) v += w3 * ld<T>(x, img + (long long)sp.i3 * g.C + ch + c);
          if (sp.live & 8u) v += w4 * ld<T>(x, img + (long long)sp.i4 * g.C + ch + c);
          const int at = k * g.Cg + c0 + c;
          if (STAGED) mine[at] = v;
          if (pass == 0) top = max(top, abs_bits(v));
          else out[at] = (signed char)code_of(v, s, ok);
        }
        c0 += run;
      }
    }
  }
  if (STAGED) {
    top = __reduce_max_sync(0xffffffffu, top);
    s = scale_of(top);
    ok = usable_scale(s);
    __syncwarp();
    for (int i = lane; i < K; i += 32) out[i] = (signed char)code_of(mine[i], s, ok);
  }
  if (lane == 0) scale[(long long)gi * np + lp] = s;
}

template <int T>
cudaError_t sample_type(const Geom& g, const void* x, const void* off, const void* mask,
                        long long p0, int np, signed char* col, int kp, float* scale,
                        cudaStream_t stream) {
  const long long items = (long long)np * g.G;
  const size_t one = (size_t)g.kk * g.Cg * sizeof(float);
  if (one <= 200 * 1024) {
    int warps = 8;
    while (warps > 1 && one * warps > 100 * 1024) warps >>= 1;
    auto kern = sample_i8_kernel<T, true>;
    const size_t smem = one * warps;
    cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), (int)smem);
    if (e != cudaSuccess) return e;
    kern<<<(unsigned)((items + warps - 1) / warps), warps * 32, smem, stream>>>(
        g, x, off, mask, p0, np, col, kp, scale);
  } else {
    sample_i8_kernel<T, false><<<(unsigned)((items + 7) / 8), 256, 0, stream>>>(
        g, x, off, mask, p0, np, col, kp, scale);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize_rows(const void* x, int type, long long rows, int cols, long long ldx,
                                 signed char* q, long long ldq, float* scale,
                                 cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  if (rows > (1LL << 31) - 1) return cudaErrorInvalidValue;
  auto kern = type == kF32 ? quantize_rows_kernel<kF32>
              : type == kBF16T ? quantize_rows_kernel<kBF16T>
                               : quantize_rows_kernel<kF16T>;
  kern<<<(unsigned)rows, 256, 0, stream>>>(x, cols, ldx, q, ldq, scale);
  return cudaGetLastError();
}

cudaError_t launch_repack_i8(const signed char* in, long long rows, int cols, signed char* out,
                             long long ldo, cudaStream_t stream) {
  const long long n = rows * cols, blocks = (n + 255) / 256;
  if (n <= 0) return cudaSuccess;
  repack_i8_kernel<<<(unsigned)(blocks < 2368 ? blocks : 2368), 256, 0, stream>>>(in, rows, cols,
                                                                                 out, ldo);
  return cudaGetLastError();
}

cudaError_t launch_sample_i8(const Geom& g, const void* x, int type, const void* off,
                             const void* mask, long long p0, int np, signed char* col, int kp,
                             float* scale, cudaStream_t stream) {
  if (type == kF32) return sample_type<kF32>(g, x, off, mask, p0, np, col, kp, scale, stream);
  if (type == kBF16T) return sample_type<kBF16T>(g, x, off, mask, p0, np, col, kp, scale, stream);
  return sample_type<kF16T>(g, x, off, mask, p0, np, col, kp, scale, stream);
}

}  // namespace dcn
