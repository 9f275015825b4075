// dcn_int8.cu -- 8-bit codes of rows and of sampled columns (see dcn_int8.h).
#include "dcn_int8.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dcn_dense_common.cuh"
#include "dcn_launch.h"

namespace dcn {

namespace {

using dense::fma2;
using dense::pair;
using dense::unpair;

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

// Rows of any length and alignment: the first 256 * KEEP values of a row wait
// in registers for their scale.
template <int T>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const void* __restrict__ x, int cols, long long ldx,
                     signed char* __restrict__ q, long long ldq, float* __restrict__ scale) {
  constexpr int KEEP = 8;
  const long long row = blockIdx.x;
  float v[KEEP];
  unsigned top = 0;
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int c = threadIdx.x + 256 * k;
    v[k] = c < cols ? ld<T>(x, row * ldx + c) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < KEEP; ++k) top = max(top, abs_bits(v[k]));
  for (int c = threadIdx.x + 256 * KEEP; c < cols; c += 256)
    top = max(top, abs_bits(ld<T>(x, row * ldx + c)));
  __shared__ unsigned red[8];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < 8; ++w) top = max(top, red[w]);
  const float s = scale_of(top);
  const bool ok = usable_scale(s);
  if (threadIdx.x == 0) scale[row] = s;
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int c = threadIdx.x + 256 * k;
    if (c < cols) q[row * ldq + c] = (signed char)code_of(v[k], s, ok);
  }
  for (int c = threadIdx.x + 256 * KEEP; c < cols; c += 256)
    q[row * ldq + c] = (signed char)code_of(ld<T>(x, row * ldx + c), s, ok);
}

// Eight consecutive values (16-byte aligned) as fp32.
template <int T>
__device__ __forceinline__ void ld8(const void* p, long long i, float (&v)[8]) {
  if constexpr (T == kF32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 r = __ldg(
        reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p) + i));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (T == kBF16T) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
    }
  }
}
// The codes of eight values, the first in the lowest byte.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float s, bool ok) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    w[j >> 2] |= (uint32_t)(code_of(v[j], s, ok) & 255) << (8 * (j & 3));
  return make_uint2(w[0], w[1]);
}

// Rows of a multiple of eight values at 16-byte aligned addresses.  A row is
// read once: the first 8 * 256 * KEEP of its values wait in registers for
// their scale.  Bound by HBM.
template <int T>
__global__ void __launch_bounds__(256)
quantize_rows8_kernel(const void* __restrict__ x, int vecs, long long ldx,
                      signed char* __restrict__ q, long long ldq, float* __restrict__ scale) {
  constexpr int KEEP = 4;
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, nt = blockDim.x;
  float v[KEEP][8];
  unsigned top = 0;
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int c = tid + k * nt;
    if (c < vecs) {
      ld8<T>(x, row * ldx + 8LL * c, v[k]);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[k][j]));
    }
  }
  for (int c = tid + KEEP * nt; c < vecs; c += nt) {
    float u[8];
    ld8<T>(x, row * ldx + 8LL * c, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, abs_bits(u[j]));
  }
  __shared__ unsigned red[8];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
  for (int w = 0; w < nt / 32; ++w) top = max(top, red[w]);
  const float s = scale_of(top);
  const bool ok = usable_scale(s);
  if (tid == 0) scale[row] = s;
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int c = tid + k * nt;
    if (c < vecs) *reinterpret_cast<uint2*>(q + row * ldq + 8LL * c) = codes8(v[k], s, ok);
  }
  for (int c = tid + KEEP * nt; c < vecs; c += nt) {
    float u[8];
    ld8<T>(x, row * ldx + 8LL * c, u);
    *reinterpret_cast<uint2*>(q + row * ldq + 8LL * c) = codes8(u, s, ok);
  }
}

// A warp a row: 16 bytes a lane from wherever the row starts (two aligned
// words around each), 16-byte stores.
__global__ void __launch_bounds__(256)
repack_i8_kernel(const signed char* __restrict__ in, long long rows, int cols,
                 signed char* __restrict__ out, long long ldo) {
  const int lane = threadIdx.x & 31;
  const long long total = rows * cols;
  for (long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows;
       r += (long long)gridDim.x * 8) {
    const long long at = r * cols;
    const uintptr_t start = reinterpret_cast<uintptr_t>(in + at);
    const uint32_t* word = reinterpret_cast<const uint32_t*>(start & ~(uintptr_t)3);
    const int shift = (int)(start & 3) * 8;
    // words that begin before the end of the matrix may be read whole: they
    // share an aligned word with a byte of it
    const long long left = (total - at + (start & 3) + 3) / 4;
    for (int c = 16 * lane; c < cols; c += 512) {
      uint32_t w[5];
#pragma unroll
      for (int j = 0; j < 5; ++j) w[j] = c / 4 + j < left ? __ldg(word + c / 4 + j) : 0u;
      uint4 v;
      v.x = __funnelshift_r(w[0], w[1], shift);
      v.y = __funnelshift_r(w[1], w[2], shift);
      v.z = __funnelshift_r(w[2], w[3], shift);
      v.w = __funnelshift_r(w[3], w[4], shift);
      // (what follows the row's end in its last 16 bytes is never read)
      *reinterpret_cast<uint4*>(out + r * ldo + c) = v;
    }
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

__device__ __forceinline__ float max_abs_nan(float top, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(v)));
  return r;
}
// VEC values as they lie in memory, and the j-th pair of them as fp32.
template <int T, int VEC>
struct Raw {
  static constexpr int WORDS = VEC * (T == kF32 ? 4 : 2) / 4;
  uint32_t w[WORDS];
};
template <int T, int VEC>
__device__ __forceinline__ Raw<T, VEC> ld_raw(const void* p) {
  Raw<T, VEC> r;
  constexpr int N = Raw<T, VEC>::WORDS;
  if constexpr (N >= 4) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      const uint4 u = __ldg(static_cast<const uint4*>(p) + k / 4);
      r.w[k] = u.x, r.w[k + 1] = u.y, r.w[k + 2] = u.z, r.w[k + 3] = u.w;
    }
  } else if constexpr (N == 2) {
    const uint2 u = __ldg(static_cast<const uint2*>(p));
    r.w[0] = u.x, r.w[1] = u.y;
  } else {
    r.w[0] = __ldg(static_cast<const uint32_t*>(p));
  }
  return r;
}
template <int T, int VEC>
__device__ __forceinline__ uint64_t raw_pair(const Raw<T, VEC>& r, int j) {
  if constexpr (T == kF32) {
    return pair(__uint_as_float(r.w[2 * j]), __uint_as_float(r.w[2 * j + 1]));
  } else {
    const uint32_t w = r.w[j];
    if constexpr (T == kBF16T)
      return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return pair(f.x, f.y);
  }
}
// The low bytes of two words, and of four.
__device__ __forceinline__ uint32_t low2(uint32_t a, uint32_t b) {
  return __byte_perm(a, b, 0x0040);
}
__device__ __forceinline__ uint32_t low4(const uint32_t* b) {
  return __byte_perm(low2(b[0], b[1]), low2(b[2], b[3]), 0x5410);
}

// Channels in vectors of VEC (eight, four or two: as groups and deformable
// groups divide).  WPP warps share an item (a pixel and group), so that each
// lane holds at most NV vectors of samples in registers from the gather to
// their codes: the input is gathered once and only codes are written.  A block
// first makes the sampling plans (corner offsets, weights with the mask) of all
// its items in shared memory, neighbouring lanes on neighbouring pixels; then
// its warps work through the items without waiting for one another, the corners
// of one vector on their way while the last one's are used.  The neck's columns
// take 75 us (100 with the plans made item by item): 7.5 TB/s of corners (four
// of 16 bytes for eight codes), 40% of them from L1.  Bound by the instructions
// and latencies of four warps a scheduler, which issue in 60% of the cycles:
// more corners on their way, with the samples in shared memory instead of
// registers, took 95 us, more warps with fewer vectors each 89; a walk through
// the pixels in tiles of 8 x 4 changed nothing.
struct alignas(16) PlanI8 {
  int at[4];      // element offsets of the corners within the image
  uint64_t w[4];  // their weights, twice each: operands of packed multiply-adds
};

template <int T, int VEC, int NV>
__global__ void __launch_bounds__(256, NV > 5 && VEC == 8 ? 2 : 3)
sample_vec_i8_kernel(Geom g, const void* __restrict__ x, const void* __restrict__ off,
                     const void* __restrict__ mask, long long p0, int np,
                     signed char* __restrict__ col, int kp, float* __restrict__ scale, int wpp,
                     int gdg, int ib) {
  extern __shared__ PlanI8 plans[];  // [npl][ib]
  __shared__ unsigned red[2][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = warp / wpp, part = warp - slot * wpp, slots = 8 / wpp;
  const long long first = (long long)blockIdx.x * ib, items = (long long)np * g.G;
  const int mine = (int)min((long long)ib, items - first), npl = g.kk * gdg;
  for (int i = threadIdx.x; i < ib * npl; i += 256) {
    const int pl = i / ib, it = i - pl * ib;
    if (it >= mine) continue;
    const long long item = first + it;
    const int gi = (int)(item / np);
    const long long pix = p0 + (item - (long long)gi * np);
    const int n = (int)(pix / g.P), p = (int)(pix - (long long)n * g.P);
    const int oy = p / g.Wo, ox = p - oy * g.Wo;
    const int k = pl / gdg, dgi = gi * g.Cg / g.cpg + pl - k * gdg;
    const int ki = k / g.kw, kj = k - ki * g.kw;
    const long long oi = off_h_index(g, n, dgi, k, p);
    float h, w;
    sample_pos(g, oy, ox, ki, kj, ld<T>(off, oi), ld<T>(off, oi + g.P), h, w);
    float m = 1.f;
    if (g.use_mask) {
      m = ld<T>(mask, mask_index(g, n, dgi, k, p));
      if (g.mask_logits) m = 1.f / (1.f + expf(-m));
    }
    const Sample sp = make_sample(h, w, g.H, g.W);
    // A dropped corner has weight 0 (whatever the mask is) and reads one that is
    // not dropped; without any, the first offset is -1 and the sample 0.
    const int corner[4] = {sp.i1, sp.i2, sp.i3, sp.i4};
    const float weight[4] = {sp.w1, sp.w2, sp.w3, sp.w4};
    int some = -1;
#pragma unroll
    for (int c = 3; c >= 0; --c)
      if (sp.live >> c & 1u) some = corner[c] * g.C;
    PlanI8 q;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bool live = sp.live >> c & 1u;
      const float wc = live ? weight[c] * m : 0.f;
      q.at[c] = live ? corner[c] * g.C : some;
      q.w[c] = pair(wc, wc);
    }
    plans[i] = q;
  }
  __syncthreads();
  constexpr int PAIRS = VEC / 2;
  constexpr int SIZE = T == kF32 ? 4 : 2;
  const int cvec = g.Cg / VEC, nvec = g.kk * cvec;
  // vectors of a deformable group, and a reciprocal (exact: products below 2^32)
  const unsigned cpv = g.cpg / VEC, cpv_inv = 0xffffffffu / cpv + 1;
  int turn = 0;
#pragma unroll 1
  for (int it = slot; it < mine; it += slots, turn ^= 1) {
    const long long item = first + it;
    const int gi = (int)(item / np), lp = (int)(item - (long long)gi * np);
    const int n = (int)((p0 + lp) / g.P);
    const long long img = (long long)n * g.HW * g.C;
    uint64_t v[NV][PAIRS];  // of fp32
    float top = 0.f;        // NaN stays
    // (tap, vector of the tap) of the lane's next vector, and their step
    const int start = part * 32 + lane, stride = 32 * wpp;
    int k = start / cvec, cv = start - k * cvec;
    const int dk = stride / cvec, dc = stride - dk * cvec;
    // the next vector's corners are on their way while the last one's are used
    Raw<T, VEC> raw[2][4];
    uint64_t w[2][4];
    bool live[2];
    const char* base = static_cast<const char*>(x) + (img + gi * g.Cg) * SIZE;
    auto fetch = [&](int i) {
      const bool inside = start + i * stride < nvec;
      const int sub = gdg > 1 ? (cpv == 1 ? cv : (int)__umulhi((unsigned)cv, cpv_inv)) : 0;
      const PlanI8& q = plans[(inside ? k * gdg + sub : 0) * ib + it];
      const int4 at = *reinterpret_cast<const int4*>(q.at);
      live[i & 1] = inside && at.x >= 0;
      const char* ch = base + cv * (VEC * SIZE);
      const int o[4] = {at.x, at.y, at.z, at.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        raw[i & 1][c] = ld_raw<T, VEC>(ch + (long long)max(o[c], 0) * SIZE);
        w[i & 1][c] = q.w[c];
      }
      k += dk;
      cv += dc;
      if (cv >= cvec) {
        cv -= cvec;
        ++k;
      }
    };
    fetch(0);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i + 1 < NV) fetch(i + 1);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) v[i][j] = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < PAIRS; ++j)
          v[i][j] = fma2(raw_pair<T, VEC>(raw[i & 1][c], j), w[i & 1][c], v[i][j]);
      if (!live[i & 1]) {
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) v[i][j] = 0;
      }
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const float2 f = unpair(v[i][j]);
        top = max_abs_nan(max_abs_nan(top, f.x), f.y);
      }
    }
    unsigned bits = __reduce_max_sync(0xffffffffu, abs_bits(top));
    if (wpp > 1) {  // the item's warps agree on its largest value
      if (lane == 0) red[turn][warp] = bits;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(32 * wpp) : "memory");
      for (int o = 0; o < wpp; ++o) bits = max(bits, red[turn][slot * wpp + o]);
    }
    const float s = scale_of(bits);
    const bool ok = usable_scale(s);
    // one reciprocal for the item: the samples are rounded sums already, so the
    // codes are within those roundings of the formula's
    // (a scale whose reciprocal could overflow divides; one that is not usable
    // gives zeros)
    const bool fast = ok && s > 1e-35f;
    const float inv = fast ? 1.f / s : 0.f;
    signed char* out = col + ((long long)gi * np + lp) * kp;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = part * 32 + lane + i * 32 * wpp;
      if (idx < nvec) {
        // v inv + 1.5 * 2^23: rounded to the nearest whole number, its low byte
        // the code (|v inv| is 127 at most, up to a rounding)
        uint32_t b[VEC];
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
          const float2 f = unpair(v[i][j]);
          b[2 * j] = __float_as_uint(fmaf(f.x, inv, 12582912.f));
          b[2 * j + 1] = __float_as_uint(fmaf(f.y, inv, 12582912.f));
        }
        if (!fast) {
          float u[VEC];
#pragma unroll
          for (int j = 0; j < PAIRS; ++j) {
            const float2 f = unpair(v[i][j]);
            u[2 * j] = f.x;
            u[2 * j + 1] = f.y;
          }
#pragma unroll
          for (int j = 0; j < VEC; ++j) b[j] = (uint32_t)code_of(u[j], s, ok);
        }
        signed char* o = out + VEC * idx;
        if constexpr (VEC == 8)
          *reinterpret_cast<uint2*>(o) = make_uint2(low4(b), low4(b + 4));
        else if constexpr (VEC == 4)
          *reinterpret_cast<uint32_t*>(o) = low4(b);
        else
          *reinterpret_cast<unsigned short*>(o) = (unsigned short)low2(b[0], b[1]);
      }
    }
    if (part == 0 && lane == 0) scale[(long long)gi * np + lp] = s;
  }
}

template <int T, int VEC, int NV>
cudaError_t sample_vec_form(const Geom& g, const void* x, const void* off, const void* mask,
                            long long p0, int np, signed char* col, int kp, float* scale,
                            int wpp, int gdg, cudaStream_t stream) {
  const long long items = (long long)np * g.G;
  const int slots = 8 / wpp;
  // items a block: 32, fewer where their plans would take more than 32 KB or
  // the blocks would not fill the SMs three times over
  const int one = (int)sizeof(PlanI8) * g.kk * gdg;
  int ib = 32;
  while (ib > slots && (ib * one > 32 * 1024 || items < (long long)ib * 3 * device_sm_count()))
    ib /= 2;
  const int smem = one * ib;
  auto kern = sample_vec_i8_kernel<T, VEC, NV>;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  kern<<<(unsigned)((items + ib - 1) / ib), 256, smem, stream>>>(
      g, x, off, mask, p0, np, col, kp, scale, wpp, gdg, ib);
  return cudaGetLastError();
}

// Products of up to NT tokens: a token does not fill a tensor-core tile, and
// the weight is read once whatever the tokens are, so this is a matter of
// reading it at full width.  A block codes the tokens for itself (they lie in
// L2; a launch of its own would cost as much as the whole product), keeps the
// codes in shared memory and gives each warp ROWS rows of the weight: lane l
// multiplies 16-byte vectors l, l + 32, ... with the four-way integer dot
// product.  The first vectors are on their way while the tokens are coded.
// (Where it is the faster way: few_tokens_pay.)
constexpr int kFewAhead = 8;  // 16-byte weight vectors a lane has on its way

template <int T, int NT, int ROWS>
__global__ void __launch_bounds__(256)
few_tokens_kernel(const void* __restrict__ x, const float* __restrict__ x_scale, int tokens,
                  int K, int N, const signed char* __restrict__ w,
                  const float* __restrict__ w_scale, const void* __restrict__ bias, int bias_type,
                  void* __restrict__ out, int out_type) {
  extern __shared__ uint4 xq[];  // [NT][K / 16]
  __shared__ unsigned red[NT][8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vecs = K / 16;
  const int row0 = (blockIdx.x * 8 + warp) * ROWS;
  constexpr int AHEAD = kFewAhead / ROWS;
  // the first 8 * 256 * KEEP values of each token are asked for before the
  // weight is, or they would wait for it
  constexpr int KEEP = T == 3 || NT > 2 ? 0 : 2 / NT;
  Raw<T == 3 ? 0 : T, 8> raw[NT][KEEP > 0 ? KEEP : 1];
  if constexpr (KEEP > 0) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < KEEP; ++k)
        if (t < tokens && tid + 256 * k < K / 8)
          raw[t][k] = ld_raw<T, 8>(static_cast<const char*>(x) +
                                   ((long long)t * K + 8LL * (tid + 256 * k)) * (T == kF32 ? 4 : 2));
        else
          raw[t][k] = {};
  }
  uint4 wv[ROWS][AHEAD];
  const uint4* wr[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    wr[r] = reinterpret_cast<const uint4*>(w + (long long)min(row0 + r, N - 1) * K);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (lane + 32 * u < vecs) wv[r][u] = __ldg(wr[r] + lane + 32 * u);
  }
  float scale[NT];
  if constexpr (T == 3) {
    const uint4* xv = static_cast<const uint4*>(x);
    for (int i = tid; i < NT * vecs; i += 256)
      xq[i] = i < tokens * vecs ? __ldg(xv + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < NT; ++t) scale[t] = t < tokens ? __ldg(x_scale + t) : 0.f;
    __syncthreads();
  } else {
    auto kept = [&](int t, int k, float(&v)[8]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpair(raw_pair<T, 8>(raw[t][k], j));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
    };
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      unsigned top = 0;
      auto take = [&](const float(&u)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, abs_bits(u[j]));
      };
      if (t < tokens) {
#pragma unroll
        for (int k = 0; k < KEEP; ++k) {
          float u[8];
          kept(t, k, u);
          take(u);
        }
        for (int c = tid + 256 * KEEP; c < K / 8; c += 256) {
          float u[8];
          ld8<T>(x, (long long)t * K + 8LL * c, u);
          take(u);
        }
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) red[t][warp] = top;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, red[t][i]);
      const float s = scale_of(top);
      const bool ok = usable_scale(s);
      scale[t] = s;
      uint2* dst = reinterpret_cast<uint2*>(xq + (long long)t * vecs);
      if (t < tokens) {
#pragma unroll
        for (int k = 0; k < KEEP; ++k) {
          const int c = tid + 256 * k;
          float u[8];
          kept(t, k, u);
          if (c < K / 8) dst[c] = codes8(u, s, ok);
        }
        for (int c = tid + 256 * KEEP; c < K / 8; c += 256) {
          float u[8];
          ld8<T>(x, (long long)t * K + 8LL * c, u);
          dst[c] = codes8(u, s, ok);
        }
      } else {
        for (int c = tid; c < K / 8; c += 256) dst[c] = make_uint2(0, 0);
      }
    }
    __syncthreads();
  }
  if (row0 >= N) return;
  int acc[ROWS][NT];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[r][t] = 0;
  for (int c0 = 0; c0 < vecs; c0 += 32 * AHEAD) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int c = c0 + 32 * u + lane;
      if (c < vecs) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint4 xv = xq[t * vecs + c];
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            acc[r][t] = __dp4a((int)wv[r][u].x, (int)xv.x, acc[r][t]);
            acc[r][t] = __dp4a((int)wv[r][u].y, (int)xv.y, acc[r][t]);
            acc[r][t] = __dp4a((int)wv[r][u].z, (int)xv.z, acc[r][t]);
            acc[r][t] = __dp4a((int)wv[r][u].w, (int)xv.w, acc[r][t]);
          }
        }
        const int next = c + 32 * AHEAD;
        if (next < vecs) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r) wv[r][u] = __ldg(wr[r] + next);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = row0 + r;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int sum = __reduce_add_sync(0xffffffffu, acc[r][t]);
      if (lane == t && t < tokens && row < N) {
        float y = (float)sum * scale[t] * __ldg(w_scale + row);
        if (bias != nullptr)
          y += bias_type == kF32 ? ld<kF32>(bias, row)
               : bias_type == kBF16T ? ld<kBF16T>(bias, row) : ld<kF16T>(bias, row);
        const long long at = (long long)t * N + row;
        if (out_type == kF32) static_cast<float*>(out)[at] = y;
        else if (out_type == kBF16T) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(y);
        else static_cast<__half*>(out)[at] = __float2half_rn(y);
      }
    }
  }
}

template <int T, int NT, int ROWS>
cudaError_t few_form(const void* x, const float* x_scale, int tokens, int K, int N,
                     const signed char* w, const float* w_scale, const void* bias, int bias_type,
                     void* out, int out_type, cudaStream_t stream) {
  auto kern = few_tokens_kernel<T, NT, ROWS>;
  const int smem = NT * K;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  kern<<<(N + 8 * ROWS - 1) / (8 * ROWS), 256, smem, stream>>>(
      x, x_scale, tokens, K, N, w, w_scale, bias, bias_type, out, out_type);
  return cudaGetLastError();
}

template <int T>
cudaError_t few_type(const void* x, const float* x_scale, int tokens, int K, int N,
                     const signed char* w, const float* w_scale, const void* bias, int bias_type,
                     void* out, int out_type, cudaStream_t stream) {
  auto form = tokens <= 1 ? few_form<T, 1, 1> : tokens <= 2 ? few_form<T, 2, 1>
              : tokens <= 4 ? few_form<T, 4, 2> : few_form<T, 8, 2>;
  return form(x, x_scale, tokens, K, N, w, w_scale, bias, bias_type, out, out_type, stream);
}

// Runs the vector kernel where VEC channels divide each group and deformable
// group (one within the other), and registers and plans hold the items.
template <int T, int VEC>
bool sample_vec(const Geom& g, const void* x, const void* off, const void* mask, long long p0,
                int np, signed char* col, int kp, float* scale, cudaStream_t stream,
                cudaError_t& e) {
  const int gdg = g.Cg >= g.cpg ? g.Cg / g.cpg : 1;
  const bool nested = g.Cg % g.cpg == 0 || g.cpg % g.Cg == 0;
  const long long nvec = (long long)g.kk * g.Cg / VEC;
  if (g.HW == 0 || g.Cg % VEC != 0 || g.cpg % VEC != 0 || !nested || nvec > 5 * 32 * 8 ||
      (reinterpret_cast<uintptr_t>(x) & 15) != 0 ||
      sizeof(PlanI8) * g.kk * gdg * 8 > 96 * 1024)
    return false;
  // one warp an item up to nine vectors a lane (no warp waits for another:
  // neck 89 -> 81 us), else several with five at most (three blocks an SM
  // instead of two: the 512-channel sweep 95 us against 99)
  int wpp = 1;
  if (nvec > 9 * 32)
    while (nvec > 5LL * 32 * wpp) wpp *= 2;
  const long long nv = (nvec + 32 * wpp - 1) / (32 * wpp);
  auto form = nv <= 1 ? sample_vec_form<T, VEC, 1> : nv <= 3 ? sample_vec_form<T, VEC, 3>
              : nv <= 5 ? sample_vec_form<T, VEC, 5> : sample_vec_form<T, VEC, 9>;
  e = form(g, x, off, mask, p0, np, col, kp, scale, wpp, gdg, stream);
  return true;
}

template <int T>
cudaError_t sample_type(const Geom& g, const void* x, const void* off, const void* mask,
                        long long p0, int np, signed char* col, int kp, float* scale,
                        cudaStream_t stream) {
  const long long items = (long long)np * g.G;
  cudaError_t e = cudaSuccess;
  if (sample_vec<T, 8>(g, x, off, mask, p0, np, col, kp, scale, stream, e)) return e;
  if (sample_vec<T, 4>(g, x, off, mask, p0, np, col, kp, scale, stream, e)) return e;
  if (sample_vec<T, 2>(g, x, off, mask, p0, np, col, kp, scale, stream, e)) return e;
  const size_t one = (size_t)g.kk * g.Cg * sizeof(float);
  if (one <= 200 * 1024) {
    int warps = 8;
    while (warps > 1 && one * warps > 100 * 1024) warps >>= 1;
    auto kern = sample_i8_kernel<T, true>;
    const size_t smem = one * warps;
    e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), (int)smem);
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
  const int es = type == kF32 ? 4 : 2;
  if (cols % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ldx * es % 16 == 0 &&
      (reinterpret_cast<uintptr_t>(q) & 7) == 0 && ldq % 8 == 0) {
    auto kern8 = type == kF32 ? quantize_rows8_kernel<kF32>
                 : type == kBF16T ? quantize_rows8_kernel<kBF16T>
                                  : quantize_rows8_kernel<kF16T>;
    // (rows without columns take a warp too: their scale is 0)
    const int vecs = cols / 8, need = (vecs + 31) / 32, warps = need < 1 ? 1 : need < 8 ? need : 8;
    kern8<<<(unsigned)rows, 32 * warps, 0, stream>>>(x, vecs, ldx, q, ldq, scale);
    return cudaGetLastError();
  }
  auto kern = type == kF32 ? quantize_rows_kernel<kF32>
              : type == kBF16T ? quantize_rows_kernel<kBF16T>
                               : quantize_rows_kernel<kF16T>;
  kern<<<(unsigned)rows, 256, 0, stream>>>(x, cols, ldx, q, ldq, scale);
  return cudaGetLastError();
}

bool few_tokens_fit(int64_t tokens, int64_t K) {
  const int64_t nt = tokens <= 1 ? 1 : tokens <= 2 ? 2 : tokens <= 4 ? 4 : 8;
  return tokens <= 8 && K % 16 == 0 && nt * K <= 96 * 1024;
}

// Against the coder and the tensor-core product behind it, in a graph (us, that
// way in brackets; 9 tokens stand for it).  Every block codes the tokens, so
// floating ones cost it tokens * K: 4 of K = 1024 to 4096 outputs 8.2 (8.9), of
// K = 2304 to 256 10.0 (9.2), of K = 4096 to 1024 14.4 (11.8); 2 of 4096 x 4096
// 13.8 (15.0); 5 of K = 256 to 256 9.8 (6.3), 8 of 4096 x 4096 26.9 (15.0).  8
// int8 tokens of 4096 x 4096 10.7 (11.3).  Beyond some 32 MB of weight the dot
// products lose to the tensor core: 4096 x 16384 with 2 floating tokens 33.9
// (26.5), with 4 int8 ones 22.2 (22.2), with 8 33.9 (22.2); 8192 x 8192 with 2
// int8 ones 19.6 (25.2).
bool few_tokens_pay(int x_type, int64_t tokens, int64_t K, int64_t N) {
  const bool small = K * N <= (int64_t(32) << 20);
  if (x_type == 3) return tokens <= 2 || small;
  return tokens <= 1 || (small && (tokens <= 2 || (tokens <= 4 && tokens * K <= 8192)));
}

cudaError_t launch_few_tokens(const void* x, int x_type, const float* x_scale, int tokens, int K,
                              int N, const signed char* w, const float* w_scale, const void* bias,
                              int bias_type, void* out, int out_type, cudaStream_t stream) {
  auto run = x_type == kF32 ? few_type<kF32> : x_type == kBF16T ? few_type<kBF16T>
             : x_type == kF16T ? few_type<kF16T> : few_type<3>;
  return run(x, x_scale, tokens, K, N, w, w_scale, bias, bias_type, out, out_type, stream);
}

cudaError_t launch_repack_i8(const signed char* in, long long rows, int cols, signed char* out,
                             long long ldo, cudaStream_t stream) {
  const long long blocks = (rows + 7) / 8;
  if (rows <= 0 || cols <= 0) return cudaSuccess;
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
