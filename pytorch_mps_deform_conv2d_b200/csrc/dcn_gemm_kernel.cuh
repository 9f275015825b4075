// dcn_gemm_kernel.cuh -- batched dense products on tcgen05: the kernel and its
// launch, instantiated by dcn_gemm.cu (8 bits), dcn_gemm_f16.cu and
// dcn_gemm_f16x2.cu.
//
// D[m, n] = sum_k A[m, k] B[n, k].  A CTA (or a pair of CTAs on two SMs) works
// through tiles: one warp feeds K slices of 128 bytes to shared memory by TMA,
// one elected lane issues the products into tensor-memory accumulators, eight warps
// drain them.  So loads, products and the epilogue of different moments run at
// once.  Three tilings:
//   pairs    256 x 256 on two SMs (cta_group::2), each holding half of both
//            operands: 64 bytes of loads an SM for every 64 K of a value, half
//            of what a 128 x 128 tile takes.  L2 -> SM loads are what bounds
//            large products (about 70 bytes a nanosecond and SM, measured);
//   128 x 128 where pairs would leave SMs idle;
//   128 x 64 and 64 x 64 for small products, K split over a cluster of up to
//            eight CTAs, whose partial sums meet in distributed shared memory:
//            with few tiles the time is that of one SM's loads.
//
// fp16 operands of two terms, x = hi + lo with lo = fp16(x - hi), carry 22
// bits.  A K slice brings both terms of both operands once and the tensor core
// forms hi hi + hi lo + lo hi; lo lo lies below the 22 bits.  Three products
// for two thirds of the loads that separate passes would take.
//
// The tensor core rounds its fp32 accumulator towards zero after every 16
// values of K.  Measured here (128 x 128, both terms in one accumulator): a sum
// of K = 16 comes out 1.7 units of 2^-24 too small on average, K = 256 24 units,
// K = 4096 470; the steps of an orthogonalisation multiply that by about 100.
// So an accumulator only ever holds a short run of K (a unit), and the epilogue
// warps add the units in registers, rounding to nearest.  For fp32 results
// units of 32 values, the cross terms (2^-11 as large, and so are their losses)
// before hi hi; what is lost on average, 1.1 units of 2^-24 (0.8 for terms of
// both signs, 1.4 for squares), is added back.  For 16-bit results units of 256, for
// those of 11 bits and less units of 1024 where tensor memory is busiest (a
// drain of 256 columns takes it from the products: 4096 x 4096 x 4096 126 us in
// units of 256, 98 us whole; a sum of 1024 loses 6e-6 of its size).
#pragma once

#include "dcn_dense_common.cuh"
#include "dcn_gemm.h"
#include "dcn_launch.h"
#include "dcn_tc_common.cuh"
#include "dcn_tma.h"

namespace dcn {

namespace {

using namespace dense;

__device__ int g_gemm_status = 0;

constexpr int EPI_WARP0 = 2, EPI_WARPS = 8;
constexpr int THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
constexpr int kSmemMax = 227 * 1024;
constexpr int kStageWarp = 32 * 17 * 4;  // a warp's transposition buffer
// alignment, barriers, channel scales, transposition
constexpr int kMiscBytes = 1024 + 256 + 2048 + EPI_WARPS * kStageWarp;

struct GemmArgs {
  int M, N, K;
  int a_shared, b_shared;
  int mt, nt, per_batch, tiles;  // tiles: mt x nt, or the upper triangle of them
  int sym;
  int split;  // CTAs of a cluster that share a tile's K
  GemmEpiArgs e;
  long long wait_limit;
  int no_async;
};

// I8: int8 operands.  TA, TB: terms.  AT, BT: the operand's rows run along K.
// BM: rows of A in a CTA.  UNIT: K of a unit in steps of 16 (0: all of K, int32
// sums are exact).  PAIR: two CTAs a tile.
template <bool I8, int TA, int TB, bool AT, bool BT, int BM, int BN, int UNIT, bool PAIR>
struct Form {
  static constexpr int BK = I8 ? 128 : 64;  // 128 bytes of K
  static constexpr int TM = PAIR ? 2 * BM : BM;     // rows of a tile
  static constexpr int WROWS = BM / 4;              // rows in a quarter of the lanes
  static constexpr int BROWS = PAIR ? BN / 2 : BN;  // rows of B in this CTA
  static constexpr int A_TERM = BM * 128, B_TERM = BROWS * 128;
  static constexpr int STAGE = TA * A_TERM + TB * B_TERM;
  static constexpr int FIT = (kSmemMax - kMiscBytes) / STAGE;
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int SMEM = STAGES * STAGE + kMiscBytes;
  static_assert(STAGES >= 3, "three stages at least");
  static constexpr int BUFS = BN == 256 || UNIT == 0 ? 2 : 4;  // accumulators
  static constexpr int TMEM = BUFS * BN;
  static_assert((2 * STAGES + 2 * BUFS + 2) * 8 <= 256, "room for the barriers");
  static constexpr int COLS = BN / 2;  // of an epilogue warp
  static constexpr int PART_PITCH = BN + 4;  // floats a row of a partial sum
  static_assert(BN != 64 || STAGES * STAGE >= BM * PART_PITCH * 4, "room for a partial sum");
};

template <bool I8, bool PAIR>
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                     uint32_t accumulate) {
#define DCN_UMMA(group, kind)                                                \
  asm volatile(                                                              \
      "{\n.reg .pred p;\n"                                                   \
      "setp.ne.b32 p, %4, 0;\n"                                              \
      "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n}\n" ::"r"(d), \
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)                            \
      : "memory")
  if constexpr (I8 && PAIR) DCN_UMMA("2", "i8");
  else if constexpr (I8) DCN_UMMA("1", "i8");
  else if constexpr (PAIR) DCN_UMMA("2", "f16");
  else DCN_UMMA("1", "f16");
#undef DCN_UMMA
}
// Arrives on `bar` (of both CTAs of a pair) when the products issued so far are
// done.
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(tc::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    tc::umma_commit(bar);
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     tc::smem_u32(slot)),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tc::tmem_alloc(slot, cols);
    tc::tmem_relinquish();
  }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
  if constexpr (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols)
                 : "memory");
  else
    tc::tmem_dealloc(addr, cols);
}

// ---- clusters ----
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// A shared-memory address of this CTA in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr)
               : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();  // the barrier takes whole warps
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
// Instruction descriptors: fp16 x fp16 -> fp32 (bits 15 / 16: the operand's
// rows run along K), and signed 8-bit -> int32.
template <bool I8, bool AT, bool BT>
__device__ constexpr uint32_t idesc(int M, int N) {
  const uint32_t shape = ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
  if (I8) return (2u << 4) | (1u << 7) | (1u << 10) | shape;
  return (1u << 4) | (AT ? 1u << 15 : 0u) | (BT ? 1u << 16 : 0u) | shape;
}
// Descriptor of an operand whose rows run along K: blocks of 64 M (or N)
// values by 64 K rows, 128-byte swizzle; blocks 8192 bytes apart, groups of
// eight K rows 1024 bytes apart.
__device__ __forceinline__ uint64_t sdesc_k_rows(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(8192 >> 4) << 16) | (64ull << 32) |
         (1ull << 46) | (2ull << 61);
}

struct Tile {
  int b, m0, n0;  // m0 of this CTA's rows
  bool mirrored;
};
// Tile t of the launch.  `sym` (square tiles): those on and above the diagonal.
template <class F, bool PAIR>
__device__ __forceinline__ Tile tile_of(const GemmArgs& g, int t, int rank) {
  Tile r;
  r.b = t / g.per_batch;
  int i = t - r.b * g.per_batch, tm = 0, tn = 0;
  if (!g.sym) {
    tn = i / g.mt;
    tm = i - tn * g.mt;
    r.mirrored = false;
  } else {
    while (i >= g.nt - tm) i -= g.nt - tm++;
    tn = tm + i;
    r.mirrored = tn != tm;
  }
  r.m0 = tm * F::TM + (PAIR ? rank * (F::TM / 2) : 0);
  r.n0 = tn * (F::COLS * 2);
  return r;
}

template <int T>
__device__ __forceinline__ float load_f(const void* p, long long i) {
  if constexpr (T == kF32) return static_cast<const float*>(p)[i];
  else if constexpr (T == kBF16T)
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  else return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ float load_as_f32(const void* p, int type, long long i) {
  return type == kF32 ? load_f<kF32>(p, i)
         : type == kBF16T ? load_f<kBF16T>(p, i) : load_f<kF16T>(p, i);
}
template <int T>
__device__ __forceinline__ void store_f(void* p, long long i, float v) {
  if constexpr (T == kF32) static_cast<float*>(p)[i] = v;
  else if constexpr (T == kBF16T) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
// ---- epilogues: eight consecutive columns n .. n + 7 of row m < M ----

// fp16 terms.  The pitch is a multiple of eight, so a chunk that starts inside
// the row fits.  lh, ll: the terms of the linear part (kEpiPoly); hi / lo return
// what was stored.
__device__ __forceinline__ uint4 linear8(const GemmArgs& g, int term, int b, int m, int n) {
  const GemmEpiArgs& e = g.e;
  // (the linear part has the terms of the result)
  if (e.mode != kEpiPoly || term >= e.out_terms || m >= g.M || n >= g.N)
    return make_uint4(0, 0, 0, 0);
  return *reinterpret_cast<const uint4*>(e.lin16 + term * e.term_stride +
                                         (long long)b * e.batch_stride +
                                         (long long)m * e.pitch + n);
}
__device__ __forceinline__ void terms8(const GemmArgs& g, const float (&v)[8], int b, int m,
                                       int n, const uint4& lh, const uint4& ll,
                                       uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  const GemmEpiArgs& e = g.e;
  const long long at = (long long)b * e.batch_stride + (long long)m * e.pitch + n;
  uint64_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = pair(v[2 * j], v[2 * j + 1]);
  if (e.mode == kEpiPoly) {
    const uint64_t lin = pair(e.lin, e.lin);
    w[0] = fma2(join2(lh.x, ll.x), lin, w[0]);
    w[1] = fma2(join2(lh.y, ll.y), lin, w[1]);
    w[2] = fma2(join2(lh.z, ll.z), lin, w[2]);
    w[3] = fma2(join2(lh.w, ll.w), lin, w[3]);
    const int d = m - n;
    if (d >= 0 && d < 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = add2(w[j], pair(d == 2 * j ? e.diag : 0.f, d == 2 * j + 1 ? e.diag : 0.f));
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) split2(w[j], hi[j], lo[j]);
  *reinterpret_cast<uint4*>(e.out16 + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  if (e.out_terms == 2)
    *reinterpret_cast<uint4*>(e.out16 + e.term_stride + at) =
        make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

__device__ __forceinline__ void* out_base(const GemmEpiArgs& e, int b) {
  return e.out != nullptr ? e.out : e.list[b];
}

// Dense rows of N, 16-byte stores (N and the base allow them; N % 8 == 0 is not
// needed for fp32, so `left` counts).
template <int T>
__device__ __forceinline__ void rows8_wide(const GemmArgs& g, const float (&v)[8], void* base,
                                           int m, int n) {
  const GemmEpiArgs& e = g.e;
  const long long at = (long long)m * g.N + n;
  const bool axpy = e.mode == kEpiAxpy;
  if constexpr (T == kF32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (n + 4 * c >= g.N) return;
      float4 y = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
      if (axpy) {
        const float4 p = o[c];
        y.x += e.keep * p.x;
        y.y += e.keep * p.y;
        y.z += e.keep * p.z;
        y.w += e.keep * p.w;
      }
      o[c] = y;
    }
  } else {
    uint4* o = reinterpret_cast<uint4*>(static_cast<unsigned short*>(base) + at);
    float2 p[4];
    if (axpy) {
      const uint4 q = *o;
      p[0] = unpack2<T>(q.x);
      p[1] = unpack2<T>(q.y);
      p[2] = unpack2<T>(q.z);
      p[3] = unpack2<T>(q.w);
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = axpy ? pack2<T>(v[2 * j] + e.keep * p[j].x, v[2 * j + 1] + e.keep * p[j].y)
                  : pack2<T>(v[2 * j], v[2 * j + 1]);
    *o = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <int T>
__device__ __forceinline__ void rows1(const GemmArgs& g, float v, void* base, int m, int n) {
  const long long at = (long long)m * g.N + n;
  store_f<T>(base, at, g.e.mode == kEpiAxpy ? v + g.e.keep * load_f<T>(base, at) : v);
}
template <int T>
__device__ __forceinline__ void rows8(const GemmArgs& g, const float (&v)[8], void* base, int m,
                                      int n) {
  if (g.e.wide_ok) {
    rows8_wide<T>(g, v, base, m, n);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (n + j < g.N) rows1<T>(g, v[j], base, m, n + j);
}

// ---- epilogues: 32 columns n0 .. of the rows of a warp's 32 lanes ----

__device__ __forceinline__ void terms32(const GemmArgs& g, float (&v)[32], const Tile& T, int m,
                                        int n0) {
  const GemmEpiArgs& e = g.e;
  if (m >= g.M) return;
  uint4 lh[4], ll[4];  // on their way together
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    lh[c] = linear8(g, 0, T.b, m, n0 + 8 * c);
    ll[c] = linear8(g, 1, T.b, m, n0 + 8 * c);
  }
#pragma unroll
  for (int c = 0; c < 32; c += 8) {
    const int n = n0 + c;
    if (n >= g.N) return;
    float u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = v[c + j];
    uint32_t hi[4], lo[4];
    terms8(g, u, T.b, m, n, lh[c / 8], ll[c / 8], hi, lo);
    if (T.mirrored) {  // lanes hold neighbouring columns of the mirrored rows
      unsigned short* out =
          e.out16 + (long long)T.b * e.batch_stride + (long long)n * e.pitch + m;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (n + j < g.N) {
          out[j * e.pitch] = (unsigned short)(hi[j >> 1] >> (16 * (j & 1)));
          if (e.out_terms == 2)
            out[e.term_stride + j * e.pitch] = (unsigned short)(lo[j >> 1] >> (16 * (j & 1)));
        }
      }
    }
  }
}

// Rows that do not take 16-byte stores go through the warp's transposition
// buffer, so that its lanes write neighbouring columns.
template <int T>
__device__ __forceinline__ void rows32(const GemmArgs& g, const float (&v)[32], void* base, int m,
                                       int n0, float* stage, int lane, int first, int rows) {
  if (g.e.wide_ok) {
    if (m >= g.M) return;
#pragma unroll
    for (int c = 0; c < 32; c += 8) {
      if (n0 + c >= g.N) return;
      float u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = v[c + j];
      rows8_wide<T>(g, u, base, m, n0 + c);
    }
    return;
  }
#pragma unroll
  for (int h = 0; h < 32; h += 16) {  // 16 columns at a time, two rows a store
#pragma unroll
    for (int j = 0; j < 16; ++j) stage[lane * 17 + j] = v[h + j];
    __syncwarp();
    const int n = n0 + h + (lane & 15);
    if (n < g.N)
      for (int r = lane >> 4; r < rows; r += 2)
        rows1<T>(g, stage[r * 17 + (lane & 15)], base, first + r, n);
    __syncwarp();
  }
}

// 32 channels of one pixel into NCHW planes: a warp's first `rows` lanes hold
// neighbouring pixels (m < M).
template <int T>
__device__ __forceinline__ void planes32(const GemmArgs& g, const float (&v)[32], int b, int m,
                                         int n0, int rows) {
  const GemmEpiArgs& e = g.e;
  if (m >= g.M) return;
  const int pixel = e.m_base + m, img = pixel / e.pixels, px = pixel - img * e.pixels;
  const long long at = ((long long)img * e.channels + (long long)b * g.N + n0) * e.pixels + px;
  if constexpr (T != kF32) {
    // Pixels in pairs (both of one image, both < M): lanes 2 i and 2 i + 1
    // trade a value, the even one stores channel c of both pixels, the odd one
    // channel c + 1
    if (e.pixel_pairs) {
      const unsigned lanes = rows >= 32 ? 0xffffffffu : (1u << rows) - 1;
      const bool odd = pixel & 1;
      unsigned short* out = static_cast<unsigned short*>(e.out) + (odd ? at - 1 + e.pixels : at);
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        const float other = __shfl_xor_sync(lanes, odd ? v[c] : v[c + 1], 1);
        const uint32_t w = odd ? pack2<T>(other, v[c + 1]) : pack2<T>(v[c], other);
        if (n0 + c + odd < g.N)
          *reinterpret_cast<uint32_t*>(out + (long long)c * e.pixels) = w;
      }
      return;
    }
  }
#pragma unroll
  for (int c = 0; c < 32; ++c)
    if (n0 + c < g.N) store_f<T>(e.out, at + (long long)c * e.pixels, v[c]);
}

template <bool I8>
__device__ __forceinline__ void finish32(const GemmArgs& g, float (&v)[32], const Tile& T, int m,
                                         int n0, float* stage, int lane, int first, int rows) {
  // lanes hold rows m = first + lane, the first `rows` of them
  const int type = g.e.out_type;
  if constexpr (I8) {
    if (g.e.mode == kEpiPlanes) {
      if (type == kF32) planes32<kF32>(g, v, T.b, m, n0, rows);
      else if (type == kBF16T) planes32<kBF16T>(g, v, T.b, m, n0, rows);
      else planes32<kF16T>(g, v, T.b, m, n0, rows);
      return;
    }
  } else {
    if (g.e.mode <= kEpiPoly) {
      terms32(g, v, T, m, n0);
      return;
    }
  }
  void* base = out_base(g.e, T.b);
  if (type == kF32) rows32<kF32>(g, v, base, m, n0, stage, lane, first, rows);
  else if (type == kBF16T) rows32<kBF16T>(g, v, base, m, n0, stage, lane, first, rows);
  else rows32<kF16T>(g, v, base, m, n0, stage, lane, first, rows);
}

template <bool I8, int TA, int TB, bool AT, bool BT, int BM, int BN, int UNIT, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
gemm_tc_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
               const __grid_constant__ GemmArgs g) {
  using F = Form<I8, TA, TB, AT, BT, BM, BN, UNIT, PAIR>;
  constexpr int STAGES = F::STAGES, COLS = F::COLS;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw);
  unsigned char* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t s0 = tc::smem_u32(smem);
  float* stages_f = reinterpret_cast<float*>(smem);
  float* staging = reinterpret_cast<float*>(smem + STAGES * F::STAGE);
  // scale and bias of the tile's channels (int8)
  float2* chan = reinterpret_cast<float2*>(smem + STAGES * F::STAGE + EPI_WARPS * kStageWarp);
  uint64_t* full = reinterpret_cast<uint64_t*>(chan + 256);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + F::BUFS;
  uint64_t* drain = acc_empty + F::BUFS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const tc::Watch watch{abort_flag, &g_gemm_status, kStatusDense, g.wait_limit};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool clustered = PAIR || g.split > 1;
  const int rank = clustered ? (int)cluster_rank() : 0;
  // tiles of this CTA (of its cluster), and its part of their K
  const int group = PAIR ? 2 : g.split;
  const int first_tile = blockIdx.x / group, tile_step = gridDim.x / group;
  const int all_ksteps = (g.K + F::BK - 1) / F::BK;
  const int k0 = PAIR ? 0 : (int)((long long)all_ksteps * rank / g.split);
  const int k1 = PAIR ? all_ksteps : (int)((long long)all_ksteps * (rank + 1) / g.split);
  const int ksteps = k1 - k0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tc::mbar_init(&full[s], 1);
      tc::mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < F::BUFS; ++a) {
      tc::mbar_init(&acc_full[a], 1);
      tc::mbar_init(&acc_empty[a], EPI_WARPS * (PAIR ? 2 : 1));
    }
    tc::mbar_init(drain, 1);
    *abort_flag = 0;
    tc::fence_mbar_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&amap)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&bmap)) : "memory");
  }
  if (warp == 1) tmem_alloc<PAIR>(tmem_slot, F::TMEM);
  tc::tc_fence_before();
  __syncthreads();
  if (clustered) cluster_sync();  // the barriers of every CTA are there
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_launch_dependents();
  grid_wait();

  if (warp == 0) {
    // ------------------------------ loads ------------------------------
    if (elect_one() && !g.no_async) {
      int it = 0;
      bool ok = true;
      for (int t = first_tile; t < g.tiles && ok; t += tile_step) {
        const Tile T = tile_of<F, PAIR>(g, t, rank);
        const int ba = g.a_shared ? 0 : T.b;
        const int bb = g.b_shared ? 0 : T.b;
        const int bn0 = T.n0 + (PAIR ? rank * F::BROWS : 0);
        for (int k = k0; k < k1; ++k, ++it) {
          const int st = it % STAGES, u = it / STAGES;
          if (u > 0 && !tc::wait(watch, &empty[st], (u - 1) & 1)) {
            ok = false;
            break;
          }
          // a pair's bytes all count on its first CTA's barrier
          uint32_t bar = tc::smem_u32(&full[st]);
          if (!PAIR || rank == 0)
            tc::mbar_arrive_expect_tx(&full[st], F::STAGE * (PAIR ? 2 : 1));
          if constexpr (PAIR) bar = map_to(bar, 0);
          uint32_t dst = s0 + st * F::STAGE;
#pragma unroll
          for (int q = 0; q < TA; ++q, dst += F::A_TERM) {
            if constexpr (AT) {
              for (int j = 0; j < BM / 64; ++j)
                tma_load_4d<PAIR>(dst + j * 8192, &amap, T.m0 + j * 64, k * F::BK, q, ba, bar);
            } else {
              tma_load_4d<PAIR>(dst, &amap, k * F::BK, T.m0, q, ba, bar);
            }
          }
#pragma unroll
          for (int q = 0; q < TB; ++q, dst += F::B_TERM) {
            if constexpr (BT) {
              for (int j = 0; j < F::BROWS / 64; ++j)
                tma_load_4d<PAIR>(dst + j * 8192, &bmap, bn0 + j * 64, k * F::BK, q, bb, bar);
            } else {
              tma_load_4d<PAIR>(dst, &bmap, k * F::BK, bn0, q, bb, bar);
            }
          }
        }
      }
      // after a wait that ran out the copies in flight land before the CTA leaves
      if (tc::aborted(watch) && (!PAIR || rank == 0))
        for (int i = it > STAGES ? it - STAGES : 0; i < it; ++i)
          tc::drain_wait(&full[i % STAGES], (i / STAGES) & 1, g.wait_limit);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------ products ------------------------------
    if (!PAIR || rank == 0) {
      constexpr uint32_t id = idesc<I8, AT, BT>(F::TM, BN);
      // 16 K values (32 of int8): 32 bytes along a row, or 16 rows of 128
      constexpr uint64_t ka = AT ? 2048 >> 4 : 32 >> 4, kb = BT ? 2048 >> 4 : 32 >> 4;
      constexpr uint64_t la = F::A_TERM >> 4, lb = F::B_TERM >> 4;
      constexpr int RUN = UNIT == 2 ? 2 : 4;  // steps of 16 issued at once
      int it = 0, n = 0, unit = 0;
      bool ok = true;
      for (int t = first_tile; t < g.tiles && ok; t += tile_step, ++n) {
        uint32_t d = 0;
        int steps = 0;  // of 16 values of K in the current unit
        for (int k = 0; k < ksteps; ++k, ++it) {
          const int st = it % STAGES;
          ok = wait_warp(watch, &full[st], (it / STAGES) & 1);
          if (!ok) break;
          tc::tc_fence_after();
          const uint32_t sa = s0 + st * F::STAGE, sb = sa + TA * F::A_TERM;
          const uint64_t da = AT ? sdesc_k_rows(sa) : tc::sdesc_sw128(sa);
          const uint64_t db = BT ? sdesc_k_rows(sb) : tc::sdesc_sw128(sb);
#pragma unroll
          for (int j = 0; j < 4; j += RUN) {
            if (steps == 0) {
              const int buf = unit % F::BUFS, use = unit / F::BUFS;
              if (use > 0) ok = wait_warp(watch, &acc_empty[buf], (use - 1) & 1);
              if (!ok) break;
              tc::tc_fence_after();
              d = tmem + (uint32_t)(buf * BN);
            }
            const bool last = j + RUN == 4;
            const bool unit_done = steps + RUN == UNIT || (last && k + 1 == ksteps);
            if (elect_one()) {
              if constexpr (TA + TB > 2) {  // the small terms first
#pragma unroll
                for (int i = j; i < j + RUN; ++i) {
                  if constexpr (TB == 2)
                    umma<I8, PAIR>(d, da + i * ka, db + lb + i * kb, id,
                                   steps + i - j != 0 ? 1u : 0u);
                  if constexpr (TA == 2)
                    umma<I8, PAIR>(d, da + la + i * ka, db + i * kb, id,
                                   TB == 2 || steps + i - j != 0 ? 1u : 0u);
                }
              }
#pragma unroll
              for (int i = j; i < j + RUN; ++i)
                umma<I8, PAIR>(d, da + i * ka, db + i * kb, id,
                               TA + TB > 2 || steps + i - j != 0 ? 1u : 0u);
              if (unit_done) commit<PAIR>(&acc_full[unit % F::BUFS]);
              if (last) commit<PAIR>(&empty[st]);
            }
            __syncwarp();
            steps += RUN;
            if (unit_done) {
              ++unit;
              steps = 0;
            }
          }
          if (!ok) break;
        }
      }
      if (!ok && elect_one()) {  // every product issued so far completes before the CTA leaves
        commit<PAIR>(drain);
        tc::drain_wait(drain, 0, g.wait_limit);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ epilogue ------------------------------
    // Warp w of eight reads the tensor-memory lanes of its quarter (w % 4),
    // half of the columns (w / 4).
    const int q = warp & 3, half = (warp - EPI_WARP0) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * COLS);
    float* stage = staging + (warp - EPI_WARP0) * (kStageWarp / 4);
    const int units = UNIT == 0 ? 1 : (ksteps * 4 + UNIT - 1) / (UNIT == 0 ? 1 : UNIT);
    auto release = [&](uint64_t* bar) {
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) arrive_at(map_to(tc::smem_u32(bar), 0));
        else tc::mbar_arrive(bar);
      }
    };
    int unit = 0;
    // int8: false once a wait of this warp has run out.  Such a warp touches no
    // accumulator any more, but still meets the other seven at the named barrier
    // of every tile left: one of them may have found the accumulators complete a
    // moment later, and that barrier has no limit.
    bool live = true;
    for (int t = first_tile; t < g.tiles; t += tile_step) {
      const Tile T = tile_of<F, PAIR>(g, t, rank);
      // (64 rows of A lie in the first 16 lanes of each quarter)
      const int first = T.m0 + q * F::WROWS, rows = min(F::WROWS, g.M - first);
      const int m = lane < F::WROWS ? first + lane : g.M, n0 = T.n0 + half * COLS;
      if constexpr (I8) {
        const float rs = m < g.M ? __ldg(g.e.row_scale + T.b * g.e.row_scale_batch + m) : 0.f;
        // the epilogue warps alone: named barrier 1
        asm volatile("bar.sync 1, %0;" ::"n"(EPI_WARPS * 32) : "memory");
        for (int c = threadIdx.x - EPI_WARP0 * 32; c < BN; c += EPI_WARPS * 32) {
          const int col = T.n0 + c;
          const long long at = (long long)T.b * g.N + col;
          chan[c] = col < g.N ? make_float2(__ldg(g.e.col_scale + at),
                                            g.e.bias != nullptr
                                                ? load_as_f32(g.e.bias, g.e.bias_type, at)
                                                : 0.f)
                              : make_float2(0.f, 0.f);
        }
        asm volatile("bar.sync 1, %0;" ::"n"(EPI_WARPS * 32) : "memory");
        const int buf = unit % F::BUFS;
        // (whole warps: the loads of tensor memory that follow take all lanes)
        live = live && wait_warp(watch, &acc_full[buf], (unit / F::BUFS) & 1);
        if (!live) continue;
        ++unit;
        tc::tc_fence_after();
        if (g.split > 1) {
          int* part = reinterpret_cast<int*>(stages_f) +
                      (q * F::WROWS + lane) * F::PART_PITCH + half * COLS;
#pragma unroll 1
          for (int c = 0; c < COLS; c += 32) {
            uint32_t r[32];
            tmem_ld32(lanes + (uint32_t)(buf * BN + c), r);
            tc::tmem_ld_wait();
            if (lane < F::WROWS) {
#pragma unroll
              for (int j = 0; j < 32; j += 4)
                *reinterpret_cast<uint4*>(part + c + j) =
                    make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
            }
          }
          break;  // one tile a cluster: summed below
        }
#pragma unroll 1
        for (int c = 0; c < COLS && n0 + c < g.N; c += 32) {
          uint32_t r[32];
          tmem_ld32(lanes + (uint32_t)(buf * BN + c), r);
          tc::tmem_ld_wait();
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float2 s = chan[half * COLS + c + j];
            v[j] = (float)(int)r[j] * rs * s.x + s.y;
          }
          finish32<I8>(g, v, T, m, n0 + c, stage, lane, first, rows);
        }
        release(&acc_empty[buf]);
      } else {
        // written by a kernel of the same chain of launches: past L1
        const float f = g.e.factor * (g.e.scale != nullptr ? __ldcg(g.e.scale + T.b) : 1.f);
        uint64_t acc[COLS / 2];
#pragma unroll
        for (int c = 0; c < COLS / 2; ++c) acc[c] = 0;
        bool ok = true;
#pragma unroll 1
        for (int u = 0; u < units; ++u, ++unit) {
          const int buf = unit % F::BUFS;
          ok = wait_warp(watch, &acc_full[buf], (unit / F::BUFS) & 1);
          if (!ok) break;
          tc::tc_fence_after();
#pragma unroll
          for (int c = 0; c < COLS; c += 32) {
            uint32_t r[32];
            tmem_ld32(lanes + (uint32_t)(buf * BN + c), r);
            tc::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j)
              acc[c / 2 + j] = add2(acc[c / 2 + j], pair(__uint_as_float(r[2 * j]),
                                                         __uint_as_float(r[2 * j + 1])));
          }
          release(&acc_empty[buf]);
        }
        if (!ok) break;
        if constexpr (UNIT == 2) {
          const float lost = g.K <= 16 ? kStepLoss : kUnitLoss;
          const uint64_t loss = pair(lost, lost);
#pragma unroll
          for (int c = 0; c < COLS / 2; ++c) acc[c] = fma2(acc[c], loss, acc[c]);
        }
        if (g.split > 1) {
          float* part = stages_f + (q * F::WROWS + lane) * F::PART_PITCH + half * COLS;
          if (lane < F::WROWS) {
#pragma unroll
            for (int c = 0; c < COLS; c += 4) {
              const float2 a = unpair(acc[c / 2]), b = unpair(acc[c / 2 + 1]);
              *reinterpret_cast<float4*>(part + c) = make_float4(a.x, a.y, b.x, b.y);
            }
          }
          break;  // one tile a cluster: summed below
        }
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          if (n0 + c >= g.N) break;
          float v[32];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 a = unpair(acc[c / 2 + j]);
            v[2 * j] = a.x * f;
            v[2 * j + 1] = a.y * f;
          }
          finish32<I8>(g, v, T, m, n0 + c, stage, lane, first, rows);
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if constexpr (BN == 64) {
    if (g.split > 1) {
      // The cluster's partial sums meet: each CTA adds its rows of all of them,
      // in the order of the ranks, and finishes those.
      cluster_sync();
      const bool gave_up = tc::aborted(watch);  // then the sums are not there
      const int rows = BM / g.split;
      const Tile T = tile_of<F, PAIR>(g, first_tile, rank);
      if (!gave_up && warp >= EPI_WARP0 && first_tile < g.tiles) {
        for (int i = threadIdx.x - EPI_WARP0 * 32; i < rows * (BN / 8); i += EPI_WARPS * 32) {
          const int row = rank * rows + i / (BN / 8), c = i % (BN / 8) * 8;
          const int m = T.m0 + row, n = T.n0 + c;
          if (m >= g.M || n >= g.N) continue;
          const uint32_t at = s0 + (uint32_t)(row * F::PART_PITCH + c) * 4;
          float v[8];
          if constexpr (I8) {
            int s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            for (int r = 0; r < g.split; ++r) {
              const float4 x = ld_cluster_f4(map_to(at, r)), y = ld_cluster_f4(map_to(at + 16, r));
              const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
              for (int j = 0; j < 8; ++j) s[j] += __float_as_int(w[j]);
            }
            const float rs = __ldg(g.e.row_scale + T.b * g.e.row_scale_batch + m);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (float)s[j] * rs * chan[c + j].x + chan[c + j].y;
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
            for (int r = 0; r < g.split; ++r) {
              const float4 x = ld_cluster_f4(map_to(at, r)), y = ld_cluster_f4(map_to(at + 16, r));
              const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] += w[j];
            }
            const float f = g.e.factor * (g.e.scale != nullptr ? __ldcg(g.e.scale + T.b) : 1.f);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= f;
          }
          if (!I8 && g.e.mode <= kEpiPoly) {
            uint32_t hi[4], lo[4];
            terms8(g, v, T.b, m, n, linear8(g, 0, T.b, m, n), linear8(g, 1, T.b, m, n), hi, lo);
          } else if (I8 && g.e.mode == kEpiPlanes) {
            const GemmEpiArgs& e = g.e;
            const int pixel = e.m_base + m, img = pixel / e.pixels, px = pixel - img * e.pixels;
            const long long o =
                ((long long)img * e.channels + (long long)T.b * g.N + n) * e.pixels + px;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (n + j >= g.N) break;
              const long long at1 = o + (long long)j * e.pixels;
              if (e.out_type == kF32) store_f<kF32>(e.out, at1, v[j]);
              else if (e.out_type == kBF16T) store_f<kBF16T>(e.out, at1, v[j]);
              else store_f<kF16T>(e.out, at1, v[j]);
            }
          } else {
            void* base = out_base(g.e, T.b);
            if (g.e.out_type == kF32) rows8<kF32>(g, v, base, m, n);
            else if (g.e.out_type == kBF16T) rows8<kBF16T>(g, v, base, m, n);
            else rows8<kF16T>(g, v, base, m, n);
          }
        }
      }
    }
  }
  // nothing of a cluster's CTA goes before its neighbours are done with it
  if (clustered) cluster_sync();
  if (warp == 1) tmem_dealloc<PAIR>(tmem, F::TMEM);
}

inline cudaError_t make_map(CUtensorMap* map, const GemmOperand& o, bool int8, int box_rows) {
  return make_tmap_4d(map, o.base, int8, (uint64_t)o.inner, (uint64_t)o.rows, (uint64_t)o.pitch,
                      (uint64_t)o.terms,
                      (uint64_t)(o.terms > 1 ? o.term_stride : o.pitch * o.rows),
                      (uint64_t)o.batch,
                      (uint64_t)(o.batch > 1 ? o.batch_stride : o.pitch * o.rows),
                      o.k_rows ? 64u : (uint32_t)box_rows);
}

template <bool I8, int TA, int TB, bool AT, bool BT, int BM, int BN, int UNIT, bool PAIR>
cudaError_t launch_form(const GemmProblem& p, int split, cudaStream_t stream) {
  using F = Form<I8, TA, TB, AT, BT, BM, BN, UNIT, PAIR>;
  GemmArgs g;
  g.M = p.M;
  g.N = p.N;
  g.K = p.K;
  g.a_shared = p.a.batch == 1;
  g.b_shared = p.b.batch == 1;
  g.mt = (p.M + F::TM - 1) / F::TM;
  g.nt = (p.N + BN - 1) / BN;
  // halves of a symmetric product only in large square tiles: small ones are
  // there for their latency, and SMs are free
  g.sym = p.sym && F::TM == BN && BN > 64;
  const long long per =
      g.sym ? (long long)g.nt * (g.nt + 1) / 2 : (long long)g.mt * g.nt;
  if (per * p.batch > (1LL << 29)) return cudaErrorInvalidValue;
  g.per_batch = (int)per;
  g.tiles = (int)(per * p.batch);
  g.split = split;
  g.e = p.epi;
  g.wait_limit = p.wait_limit;
  g.no_async = p.no_async;
  CUtensorMap amap, bmap;
  cudaError_t e = make_map(&amap, p.a, I8, BM);
  if (e == cudaSuccess) e = make_map(&bmap, p.b, I8, F::BROWS);
  if (e != cudaSuccess) return e;
  auto kern = gemm_tc_kernel<I8, TA, TB, AT, BT, BM, BN, UNIT, PAIR>;
  e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), F::SMEM);
  if (e != cudaSuccess) return e;
  const int sms = device_sm_count();
  cudaLaunchConfig_t cfg = {};
  const int group = PAIR ? 2 : split;
  const int most = sms / group;
  cfg.gridDim = dim3((unsigned)(group * (split > 1 || g.tiles < most ? g.tiles : most)));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = F::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (group > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)group;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (p.after_ours) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kern, amap, bmap, g);
}

// What a tiling costs, in microseconds: `base` for a launch, `slice` for a K
// slice (128 bytes of K) of one round of tiles, measured on products of 256 to
// 8192 rows.
struct TilingCost {
  double base, slice;
};
enum Operands { kOne, kMixed, kTwo, kTwoFine, kInt8 };
// 256 x 256 on two SMs, 128 x 128, 128 x 64, 64 x 64.  In units of 32 values
// (kTwoFine) a pair's accumulators wait for drains on the other SM: 2.4 us a
// slice against 0.81 of its products, so that 128 x 128 wins at every size and
// pairs are not built for them.
constexpr TilingCost kTilingCost[5][4] = {
    {{6.0, 0.60}, {4.2, 0.50}, {3.5, 0.375}, {3.2, 0.27}},
    {{6.0, 0.90}, {4.2, 0.68}, {3.5, 0.50}, {3.2, 0.34}},
    {{6.0, 1.24}, {4.2, 0.83}, {3.5, 0.60}, {3.2, 0.42}},
    {{1e9, 2.40}, {4.2, 1.02}, {3.5, 0.74}, {3.2, 0.60}},
    {{6.0, 0.38}, {4.2, 0.42}, {3.5, 0.33}, {3.2, 0.27}},
};
// K over a cluster divides the slices of the small tilings and costs its
// barriers and the partial sums' way; of clusters of 4 and 8 some 33 and 15 fit
// the SMs' groups at a time.
constexpr double kClusterCost = 2.5;

template <bool I8, int TA, int TB, bool AT, bool BT, int UNIT>
cudaError_t launch_tiling(const GemmProblem& p, cudaStream_t stream) {
  constexpr int KIND = I8 ? kInt8 : TA + TB == 2 ? kOne : TA + TB == 3 ? kMixed
                       : UNIT == 2 ? kTwoFine : kTwo;
  const long long sms = device_sm_count();
  const int ksteps = (p.K + (I8 ? 127 : 63)) / (I8 ? 128 : 64);
  const int tm[4] = {256, 128, 128, 64}, tn[4] = {256, 128, 64, 64};
  using Small = Form<I8, TA, TB, AT, BT, 64, 64, UNIT, false>;
  const void* small =
      reinterpret_cast<const void*>(gemm_tc_kernel<I8, TA, TB, AT, BT, 64, 64, UNIT, false>);
  const cudaError_t e = ensure_dynamic_smem(small, Small::SMEM);
  if (e != cudaSuccess) return e;
  double best = 1e30;
  int form = 0, split = 1;
  for (int f = 0; f < 4; ++f) {
    const long long mt = (p.M + tm[f] - 1) / tm[f], nt = (p.N + tn[f] - 1) / tn[f];
    const long long tiles = (p.sym && f < 2 ? mt * (mt + 1) / 2 : mt * nt) * p.batch;
    const TilingCost c = kTilingCost[KIND][f];
    for (int s = 1; s <= (f < 2 ? 1 : 8) && s <= ksteps; s *= 2) {
      const long long slots =
          f == 0 ? sms / 2
                 : s == 1 ? sms : device_cluster_slots(small, THREADS, Small::SMEM, s);
      if (s > 1 && tiles > slots) continue;  // a cluster has one tile
      const double rounds = (double)((tiles + slots - 1) / slots);
      const double cost = c.base + (s > 1 ? kClusterCost : 0.0) +
                          rounds * c.slice * ((ksteps + s - 1) / s);
      if (cost < best) {
        best = cost;
        form = f;
        split = s;
      }
    }
  }
  if (form == 3) return launch_form<I8, TA, TB, AT, BT, 64, 64, UNIT, false>(p, split, stream);
  if (form == 2) return launch_form<I8, TA, TB, AT, BT, 128, 64, UNIT, false>(p, split, stream);
  if constexpr (KIND != kTwoFine) {
    if constexpr (!I8 && TA + TB < 4)
      if (form == 0 && p.coarse)
        return launch_form<I8, TA, TB, AT, BT, 128, 256, 64, true>(p, 1, stream);
    if (form == 0) return launch_form<I8, TA, TB, AT, BT, 128, 256, UNIT, true>(p, 1, stream);
  }
  return launch_form<I8, TA, TB, AT, BT, 128, 128, UNIT, false>(p, 1, stream);
}

inline cudaError_t read_status(int* status, bool clear, cudaStream_t stream) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_gemm_status, sizeof(int), 0,
                                            cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e == cudaSuccess && clear && v != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_gemm_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice,
                                stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  }
  *status = v;
  return e;
}

}  // namespace

}  // namespace dcn
