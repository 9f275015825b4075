// dcn_gemm.cu -- batched dense products on tcgen05 (see dcn_gemm.h).
//
// D[m, n] = sum_k A[m, k] B[n, k].  A CTA keeps to one SM and works through
// tiles of 128 x BN: one warp feeds K slices of 128 bytes to shared memory by
// TMA, one lane issues the products into one of two tensor-memory
// accumulators, eight warps drain the other one.  So loads, products and the
// epilogue of three different moments run at once.
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
// warps add the units in registers, rounding to nearest.  Two terms: units of
// 32 for hi hi, the cross terms (2^-11 as large) in an accumulator of their own;
// what 32 lose on average, 1.1 units of 2^-24 (0.8 for terms of both signs, 1.4
// for squares), is added back.  One term (results of 16 bits): units of 256.
#include "dcn_gemm.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dcn_launch.h"
#include "dcn_tc_common.cuh"
#include "dcn_tma.h"

namespace dcn {

namespace {

__device__ int g_gemm_status = 0;

constexpr int BM = 128;
constexpr int EPI_WARP0 = 2, EPI_WARPS = 8;
constexpr int THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
constexpr int kSmemMax = 227 * 1024;
constexpr int kMiscBytes = 1024 + 512;  // alignment, barriers

struct GemmArgs {
  int M, N, K, batch;
  int a_mod, a_shared, b_shared;
  int mt, nt, per_batch, tiles;  // tiles: mt x nt, or those reaching the upper triangle
  int sym;
  GemmEpiArgs e;
  long long wait_limit;
  int no_async;
};

template <bool I8, int TA, int TB, bool AT, bool BT, int BN>
struct Cfg {
  static constexpr int BK = I8 ? 128 : 64;  // 128 bytes of K
  static constexpr int A_TERM = BM * 128, B_TERM = BN * 128;
  static constexpr int STAGE = TA * A_TERM + TB * B_TERM;
  static constexpr int FIT = (kSmemMax - kMiscBytes) / STAGE;
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int SMEM = STAGES * STAGE + kMiscBytes;
  static_assert(STAGES >= 2, "two stages at least");
  // units of K, in steps of 16 (0: all of K, int32 sums are exact), and the
  // accumulators that hold them beside the one of the cross terms
  static constexpr bool CROSS = TA == 2 && TB == 2;
  static constexpr int UNIT = I8 ? 0 : CROSS ? 2 : 16;
  static constexpr int BUFS = CROSS ? 3 : 2;
  static constexpr int TMEM = (BUFS + (CROSS ? 1 : 0)) * BN;
  static_assert(TMEM == 256 || TMEM == 512, "a power of two of columns");
};
// 1.1 units of 2^-24 (see the top of the file)
constexpr float kUnitLoss = 6.5565e-8f;

// 4-D tiled TMA load (no multicast): box at (x, y, term, matrix).
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(tc::smem_u32(bar))
      : "memory");
}

template <bool I8>
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                     uint32_t accumulate) {
  if constexpr (I8)
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    tc::umma_bf16(d, a, b, idesc, accumulate);
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

// 32 lanes x 32-bit, 32 consecutive columns.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

struct Tile {
  int b, m0, n0;
};
// Tile t of the launch.  `sym`: of each row of tiles only those that reach the
// diagonal or lie above it.
template <int BN>
__device__ __forceinline__ Tile tile_of(const GemmArgs& g, int t) {
  Tile r;
  r.b = t / g.per_batch;
  int i = t - r.b * g.per_batch;
  if (!g.sym) {
    r.n0 = i / g.mt * BN;
    r.m0 = i % g.mt * BM;
    return r;
  }
  int row = 0, first = 0;
  for (;; ++row) {
    first = row * BM / BN;
    if (i < g.nt - first) break;
    i -= g.nt - first;
  }
  r.m0 = row * BM;
  r.n0 = (first + i) * BN;
  return r;
}

__device__ __forceinline__ float load_as_f32(const void* p, int type, long long i) {
  if (type == kF32) return static_cast<const float*>(p)[i];
  if (type == kBF16T) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void* p, int type, long long i, float v) {
  if (type == kF32) static_cast<float*>(p)[i] = v;
  else if (type == kBF16T) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
__device__ __forceinline__ uint32_t pack2(int type, float a, float b) {
  if (type == kBF16T) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float half_lo(uint32_t w) {
  return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu)));
}
__device__ __forceinline__ float half_hi(uint32_t w) {
  return __half2float(__ushort_as_half((unsigned short)(w >> 16)));
}

// 32 columns of one row of an accumulator, fp16-term outputs.
__device__ __forceinline__ void epi_terms(const GemmArgs& g, const float (&w)[32], int b,
                                          int m, int n0) {
  const GemmEpiArgs& e = g.e;
  const long long base = (long long)b * e.batch_stride;
  const bool row = m < g.M;
#pragma unroll
  for (int c = 0; c < 32; c += 8) {
    const int n = n0 + c;
    if (n >= g.N) break;  // the same for the whole warp
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = w[c + j];
    const long long at = base + (long long)m * e.pitch + n;
    if (e.mode == kEpiPoly && row) {
      const uint4 h = *reinterpret_cast<const uint4*>(e.lin16 + at);
      const uint4 l = *reinterpret_cast<const uint4*>(e.lin16 + e.term_stride + at);
      const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] += e.lin * (half_lo(hw[j]) + half_lo(lw[j]));
        v[2 * j + 1] += e.lin * (half_hi(hw[j]) + half_hi(lw[j]));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n + j == m) v[j] += e.diag;
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      hi[j] = pack2(kF16T, v[2 * j], v[2 * j + 1]);
      lo[j] = pack2(kF16T, v[2 * j] - half_lo(hi[j]), v[2 * j + 1] - half_hi(hi[j]));
    }
    const bool two = e.out_terms == 2;
    if (row && (!g.sym || n >= m)) {  // pitch is a multiple of 8: the chunk fits
      *reinterpret_cast<uint4*>(e.out16 + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if (two)
        *reinterpret_cast<uint4*>(e.out16 + e.term_stride + at) =
            make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    if (g.sym && row) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned short h = (unsigned short)(hi[j >> 1] >> (16 * (j & 1)));
        const unsigned short l = (unsigned short)(lo[j >> 1] >> (16 * (j & 1)));
        if (n < m && n + j >= m) {  // the chunk that holds the diagonal, up to N
          if (n + j < g.N) {
            e.out16[at + j] = h;
            if (two) e.out16[e.term_stride + at + j] = l;
          }
        }
        if (n + j > m && n + j < g.N) {  // mirrored: lanes hold neighbouring columns
          const long long tr = base + (long long)(n + j) * e.pitch + m;
          e.out16[tr] = h;
          if (two) e.out16[e.term_stride + tr] = l;
        }
      }
    }
  }
}

// 32 columns of one row into dense rows of N (`out`, or out = keep out + v).
__device__ __forceinline__ void epi_rows(const GemmArgs& g, const float (&v)[32], int b, int m,
                                         int n0) {
  const GemmEpiArgs& e = g.e;
  if (m >= g.M) return;
  char* out = static_cast<char*>(e.out != nullptr ? e.out : e.list[b]);
  const long long at = (e.out != nullptr ? (long long)b * e.out_batch : 0) +
                       (long long)m * g.N + n0;
  const int left = g.N - n0 < 32 ? g.N - n0 : 32;
  const bool axpy = e.mode == kEpiAxpy;
  if (e.wide_ok && left == 32) {
    if (e.out_type == kF32) {
      float4* o = reinterpret_cast<float4*>(out + at * 4);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
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
      uint4* o = reinterpret_cast<uint4*>(out + at * 2);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[4];
        uint4 p = make_uint4(0, 0, 0, 0);
        if (axpy) p = o[c];
        const uint32_t pw[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float a = v[8 * c + 2 * j], d = v[8 * c + 2 * j + 1];
          if (axpy) {
            const bool bf = e.out_type == kBF16T;
            a += e.keep * (bf ? __uint_as_float(pw[j] << 16) : half_lo(pw[j]));
            d += e.keep * (bf ? __uint_as_float(pw[j] & 0xffff0000u) : half_hi(pw[j]));
          }
          w[j] = pack2(e.out_type, a, d);
        }
        o[c] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < 32; ++c)
    if (c < left)
      store_from_f32(out, e.out_type, at + c,
                     axpy ? v[c] + e.keep * load_as_f32(out, e.out_type, at + c) : v[c]);
}

// 32 channels of one pixel into NCHW planes: a warp's lanes hold neighbouring
// pixels.
__device__ __forceinline__ void epi_planes(const GemmArgs& g, const float (&v)[32], int b, int m,
                                           int n0) {
  const GemmEpiArgs& e = g.e;
  if (m >= g.M) return;
  const int pixel = e.m_base + m, img = pixel / e.pixels, px = pixel - img * e.pixels;
  const long long at = ((long long)img * e.channels + (long long)b * g.N + n0) * e.pixels + px;
#pragma unroll
  for (int c = 0; c < 32; ++c)
    if (n0 + c < g.N) store_from_f32(e.out, e.out_type, at + (long long)c * e.pixels, v[c]);
}

template <bool I8, int TA, int TB, bool AT, bool BT, int BN>
__global__ void __launch_bounds__(THREADS, 1)
gemm_tc_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
               const __grid_constant__ GemmArgs g) {
  using C = Cfg<I8, TA, TB, AT, BT, BN>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw);
  unsigned char* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t s0 = tc::smem_u32(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + C::BUFS;
  uint64_t* cross_full = acc_empty + C::BUFS;
  uint64_t* cross_empty = cross_full + 1;
  uint64_t* drain = cross_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const tc::Watch watch{abort_flag, &g_gemm_status, kStatusDense, g.wait_limit};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ksteps = (g.K + C::BK - 1) / C::BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tc::mbar_init(&full[s], 1);
      tc::mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < C::BUFS; ++a) {
      tc::mbar_init(&acc_full[a], 1);
      tc::mbar_init(&acc_empty[a], EPI_WARPS);
    }
    tc::mbar_init(cross_full, 1);
    tc::mbar_init(cross_empty, EPI_WARPS);
    tc::mbar_init(drain, 1);
    *abort_flag = 0;
    tc::fence_mbar_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, C::TMEM);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------ loads ------------------------------
    if (lane == 0 && !g.no_async) {
      int it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < g.tiles && ok; t += gridDim.x) {
        const Tile T = tile_of<BN>(g, t);
        const int ba = g.a_shared ? 0 : (g.a_mod ? T.b % g.a_mod : T.b);
        const int bb = g.b_shared ? 0 : T.b;
        for (int k = 0; k < ksteps; ++k, ++it) {
          const int st = it % STAGES, u = it / STAGES;
          if (u > 0 && !tc::wait(watch, &empty[st], (u - 1) & 1)) {
            ok = false;
            break;
          }
          tc::mbar_arrive_expect_tx(&full[st], C::STAGE);
          uint32_t dst = s0 + st * C::STAGE;
#pragma unroll
          for (int q = 0; q < TA; ++q, dst += C::A_TERM) {
            if constexpr (AT) {
              for (int j = 0; j < BM / 64; ++j)
                tma_load_4d(dst + j * 8192, &amap, T.m0 + j * 64, k * C::BK, q, ba, &full[st]);
            } else {
              tma_load_4d(dst, &amap, k * C::BK, T.m0, q, ba, &full[st]);
            }
          }
#pragma unroll
          for (int q = 0; q < TB; ++q, dst += C::B_TERM) {
            if constexpr (BT) {
              for (int j = 0; j < BN / 64; ++j)
                tma_load_4d(dst + j * 8192, &bmap, T.n0 + j * 64, k * C::BK, q, bb, &full[st]);
            } else {
              tma_load_4d(dst, &bmap, k * C::BK, T.n0, q, bb, &full[st]);
            }
          }
        }
      }
      if (tc::aborted(watch))  // the copies in flight land before the CTA leaves
        for (int i = it > STAGES ? it - STAGES : 0; i < it; ++i)
          tc::drain_wait(&full[i % STAGES], (i / STAGES) & 1, g.wait_limit);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------ products ------------------------------
    if (lane == 0) {
      constexpr uint32_t id = idesc<I8, AT, BT>(BM, BN);
      const uint32_t cross = tmem + (uint32_t)(C::BUFS * BN);
      int it = 0, n = 0, unit = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < g.tiles && ok; t += gridDim.x, ++n) {
        uint32_t d = 0;
        int steps = 0;  // of 16 values of K in the current unit
        for (int k = 0; k < ksteps && ok; ++k, ++it) {
          const int st = it % STAGES;
          if (!tc::wait(watch, &full[st], (it / STAGES) & 1)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t sa = s0 + st * C::STAGE, sb = sa + TA * C::A_TERM;
          const uint64_t da = AT ? sdesc_k_rows(sa) : tc::sdesc_sw128(sa);
          const uint64_t db = BT ? sdesc_k_rows(sb) : tc::sdesc_sw128(sb);
          // 16 K values (32 of int8): 32 bytes along a row, or 16 rows of 128
          constexpr uint64_t ka = AT ? 2048 >> 4 : 32 >> 4, kb = BT ? 2048 >> 4 : 32 >> 4;
          constexpr uint64_t la = C::A_TERM >> 4, lb = C::B_TERM >> 4;
          if constexpr (C::CROSS) {
            if (k == 0 && n > 0 && !tc::wait(watch, cross_empty, (n - 1) & 1)) {
              ok = false;
              break;
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (C::CROSS) {
              if (j % 2 == 0) {  // a unit's cross terms before its accumulator is needed
#pragma unroll
                for (int i = j; i < j + 2; ++i) {
                  umma<I8>(cross, da + i * ka, db + lb + i * kb, id, (k | i) != 0 ? 1u : 0u);
                  umma<I8>(cross, da + la + i * ka, db + i * kb, id, 1u);
                }
              }
            }
            if (steps == 0) {
              const int buf = unit % C::BUFS, use = unit / C::BUFS;
              if (use > 0 && !tc::wait(watch, &acc_empty[buf], (use - 1) & 1)) {
                ok = false;
                break;
              }
              tc::tc_fence_after();
              d = tmem + (uint32_t)(buf * BN);
            }
            umma<I8>(d, da + j * ka, db + j * kb, id, steps != 0 ? 1u : 0u);
            if constexpr (!C::CROSS && TB == 2) umma<I8>(d, da + j * ka, db + lb + j * kb, id, 1u);
            if constexpr (!C::CROSS && TA == 2) umma<I8>(d, da + la + j * ka, db + j * kb, id, 1u);
            ++steps;
            if (steps == C::UNIT || (k + 1 == ksteps && j == 3)) {
              tc::umma_commit(&acc_full[unit % C::BUFS]);
              ++unit;
              steps = 0;
            }
          }
          if (ok) tc::umma_commit(&empty[st]);
        }
        if constexpr (C::CROSS)
          if (ok) tc::umma_commit(cross_full);
      }
      if (tc::aborted(watch)) {  // every product issued so far completes before the CTA leaves
        tc::umma_commit(drain);
        tc::drain_wait(drain, 0, g.wait_limit);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ epilogue ------------------------------
    // Warp w of eight reads the tensor-memory lanes of its quarter (w % 4),
    // half of the columns (w / 4).
    constexpr int COLS = BN / 2;
    const int q = warp & 3, half = (warp - EPI_WARP0) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * COLS);
    const int units = C::UNIT == 0 ? 1 : (ksteps * 4 + C::UNIT - 1) / C::UNIT;
    int n = 0, unit = 0;
    for (int t = blockIdx.x; t < g.tiles; t += gridDim.x, ++n) {
      const Tile T = tile_of<BN>(g, t);
      const int m = T.m0 + q * 32 + lane, n0 = T.n0 + half * COLS;
      if constexpr (I8) {
        const float rs =
            m < g.M ? __ldg(g.e.row_scale + T.b * g.e.row_scale_batch + m) : 0.f;
        const int buf = unit % C::BUFS;
        if (!tc::wait(watch, &acc_full[buf], (unit / C::BUFS) & 1)) break;
        ++unit;
        tc::tc_fence_after();
        for (int c = 0; c < COLS && n0 + c < g.N; c += 32) {
          uint32_t r[32];
          tmem_ld32(lanes + (uint32_t)(buf * BN + c), r);
          tc::tmem_ld_wait();
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const int col = n0 + c + j < g.N ? n0 + c + j : g.N - 1;
            const long long at = (long long)T.b * g.N + col;
            const float y = (float)(int)r[j] * rs * __ldg(g.e.col_scale + at);
            v[j] = g.e.bias != nullptr ? y + load_as_f32(g.e.bias, g.e.bias_type, at) : y;
          }
          if (g.e.mode == kEpiRows) epi_rows(g, v, T.b, m, n0 + c);
          else epi_planes(g, v, T.b, m, n0 + c);
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
      } else {
        const float f = g.e.factor * (g.e.scale != nullptr ? __ldg(g.e.scale + T.b) : 1.f);
        float acc[COLS];
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[c] = 0.f;
        bool ok = true;
        for (int u = 0; u < units; ++u, ++unit) {
          const int buf = unit % C::BUFS;
          if (!tc::wait(watch, &acc_full[buf], (unit / C::BUFS) & 1)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
#pragma unroll
          for (int c = 0; c < COLS; c += 32) {
            uint32_t r[32];
            tmem_ld32(lanes + (uint32_t)(buf * BN + c), r);
            tc::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[c + j] += __uint_as_float(r[j]);
          }
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
        }
        if (!ok) break;
        if constexpr (C::CROSS) {
          if (!tc::wait(watch, cross_full, n & 1)) break;
          tc::tc_fence_after();
#pragma unroll
          for (int c = 0; c < COLS; c += 32) {
            uint32_t r[32];
            tmem_ld32(lanes + (uint32_t)(C::BUFS * BN + c), r);
            tc::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j)
              acc[c + j] += fmaf(acc[c + j], kUnitLoss, __uint_as_float(r[j]));
          }
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(cross_empty);
        }
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          if (n0 + c >= g.N) break;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = acc[c + j] * f;
          if (g.e.mode <= kEpiPoly) epi_terms(g, v, T.b, m, n0 + c);
          else epi_rows(g, v, T.b, m, n0 + c);
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc(tmem, C::TMEM);
}

cudaError_t make_map(CUtensorMap* map, const GemmOperand& o, bool int8, int box_rows) {
  return make_tmap_4d(map, o.base, int8, (uint64_t)o.inner, (uint64_t)o.rows, (uint64_t)o.pitch,
                      (uint64_t)o.terms,
                      (uint64_t)(o.terms > 1 ? o.term_stride : o.pitch * o.rows),
                      (uint64_t)o.batch,
                      (uint64_t)(o.batch > 1 ? o.batch_stride : o.pitch * o.rows),
                      o.k_rows ? 64u : (uint32_t)box_rows);
}

template <bool I8, int TA, int TB, bool AT, bool BT, int BN>
cudaError_t launch_form(const GemmProblem& p, cudaStream_t stream) {
  using C = Cfg<I8, TA, TB, AT, BT, BN>;
  GemmArgs g;
  g.M = p.M;
  g.N = p.N;
  g.K = p.K;
  g.batch = p.batch;
  g.a_mod = p.a_batch_mod;
  g.a_shared = p.a.batch == 1;
  g.b_shared = p.b.batch == 1;
  g.mt = (p.M + BM - 1) / BM;
  g.nt = (p.N + BN - 1) / BN;
  g.sym = p.sym;
  long long per = (long long)g.mt * g.nt;
  if (p.sym) {
    per = 0;
    for (int r = 0; r < g.mt; ++r) per += g.nt - r * BM / BN;
  }
  if (per * p.batch > (1LL << 30)) return cudaErrorInvalidValue;
  g.per_batch = (int)per;
  g.tiles = (int)(per * p.batch);
  g.e = p.epi;
  g.wait_limit = p.wait_limit;
  g.no_async = p.no_async;
  CUtensorMap amap, bmap;
  cudaError_t e = make_map(&amap, p.a, I8, BM);
  if (e == cudaSuccess) e = make_map(&bmap, p.b, I8, BN);
  if (e != cudaSuccess) return e;
  auto kern = gemm_tc_kernel<I8, TA, TB, AT, BT, BN>;
  e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), C::SMEM);
  if (e != cudaSuccess) return e;
  const int sms = device_sm_count();
  kern<<<g.tiles < sms ? g.tiles : sms, THREADS, C::SMEM, stream>>>(amap, bmap, g);
  return cudaGetLastError();
}

template <bool I8, int TA, int TB, bool AT, bool BT>
cudaError_t launch_width(const GemmProblem& p, cudaStream_t stream) {
  // 256 columns a tile halve the loads of A; with fewer such tiles than SMs
  // the narrow ones spread over more of them
  // (two terms of both operands: the tensor memory holds four accumulators of
  // 128 columns)
  if constexpr (TA + TB < 4) {
    const long long wide = (long long)((p.M + BM - 1) / BM) * ((p.N + 255) / 256) * p.batch;
    if (wide >= device_sm_count()) return launch_form<I8, TA, TB, AT, BT, 256>(p, stream);
  }
  return launch_form<I8, TA, TB, AT, BT, 128>(p, stream);
}

}  // namespace

cudaError_t launch_gemm(const GemmProblem& p, cudaStream_t stream) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0 || p.batch <= 0) return cudaErrorInvalidValue;
  const int ta = p.a.terms, tb = p.b.terms;
  const bool at = p.a.k_rows, bt = p.b.k_rows;
  if (p.int8) return launch_width<true, 1, 1, false, false>(p, stream);
  if (!at && !bt) {
    if (ta == 1 && tb == 1) return launch_width<false, 1, 1, false, false>(p, stream);
    if (ta == 1 && tb == 2) return launch_width<false, 1, 2, false, false>(p, stream);
    if (ta == 2 && tb == 2) return launch_width<false, 2, 2, false, false>(p, stream);
  } else if (at && bt) {
    if (ta == 1 && tb == 1) return launch_width<false, 1, 1, true, true>(p, stream);
    if (ta == 2 && tb == 2) return launch_width<false, 2, 2, true, true>(p, stream);
  } else if (bt) {
    if (ta == 2 && tb == 1) return launch_width<false, 2, 1, false, true>(p, stream);
    if (ta == 2 && tb == 2) return launch_width<false, 2, 2, false, true>(p, stream);
  }
  return cudaErrorInvalidValue;
}

cudaError_t read_gemm_status(int* status, bool clear, cudaStream_t stream) {
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

}  // namespace dcn
