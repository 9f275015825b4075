// dcn_ortho_chain.cu -- the products of one run of Newton-Schulz steps on a
// matrix S of at most 128 x 128, by one CTA that keeps S, P and Q in shared
// memory:
//   P = a I + b S + c S S;  S <- P (P S);  Q <- P Q
// for each step of the run (Q the first P; the last step leaves S alone).  All
// are polynomials of one symmetric matrix: symmetric, and commuting, so every
// product is of rows with rows, and its result replaces the operand that it
// retires.
//
// Bound by latency: a run of three steps is nine products that wait for one
// another.  As launches of their own they take 5 us each at 128 x 128 (launch,
// TMA from L2, drain, store); here a product is 24 tensor-core instructions, a
// drain of the accumulators and 16-byte stores into the swizzled operands.
//
// Operands are two fp16 terms, sums are kept to fp32's accuracy as in
// dcn_gemm_kernel.cuh: units of 32 values of K, each in an accumulator of its
// own (four of 128 columns are all of tensor memory), are added in registers.
#include "dcn_ortho_chain.h"

#include "dcn_dense_common.cuh"
#include "dcn_launch.h"
#include "dcn_tma.h"

namespace dcn {

namespace {

using namespace dense;

__device__ int g_chain_status = 0;

constexpr int N = kChainMax;                 // rows and columns of the buffers
constexpr int TERM = N * N * 2;              // one term: two blocks of 64 columns
constexpr int BLOCK = N * 128;               // 128 rows of 128 bytes
constexpr int MATRIX = 2 * TERM;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (1 + EPI_WARPS);
constexpr int UNITS = N / 32;
constexpr int SMEM = 3 * MATRIX + 1024 + 256;

struct Args {
  ChainArgs c;
  long long wait_limit;
  int no_async;
};

// Byte offset of eight columns from c (a multiple of eight) of row r.
__device__ __forceinline__ uint32_t at(int r, int c) {
  return (uint32_t)((c >> 6) * BLOCK) + tc::sw128_offset(r, (c & 63) >> 3);
}

// The i-th product of a run of `run` steps: four a step (P, S twice, Q) less the
// S of the last and the Q of the first.
enum Kind { kP, kS, kQ };
struct Op {
  int step;
  Kind kind;
};
__device__ __forceinline__ Op op_of(int i, int run) {
  if (i < 3 && run > 1) return {0, i == 0 ? kP : kS};
  if (run == 1) return {0, kP};
  const int j = i - 3, step = 1 + j / 4, w = j % 4;  // P, S, S, Q
  if (w == 0) return {step, kP};
  return {step, step + 1 < run && w < 3 ? kS : kQ};
}
__device__ __forceinline__ int op_count(int run) { return run == 1 ? 1 : 4 * run - 3; }

__global__ void __launch_bounds__(THREADS, 1)
ortho_chain_kernel(const __grid_constant__ CUtensorMap smap, const __grid_constant__ Args g) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw);
  unsigned char* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  unsigned char *S = smem, *Q = smem + MATRIX, *P = smem + 2 * MATRIX;
  uint64_t* loaded = reinterpret_cast<uint64_t*>(smem + 3 * MATRIX);
  uint64_t* acc_full = loaded + 1;
  uint64_t* ready = acc_full + UNITS;
  uint64_t* drain = ready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const tc::Watch watch{abort_flag, &g_chain_status, kStatusDense, g.wait_limit};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m = g.c.m, run = g.c.run;
  const int cols = (m + 15) / 16 * 16, ksteps = cols / 16, units = (ksteps + 1) / 2;
  const int ops = op_count(run);

  if (threadIdx.x == 0) {
    tc::mbar_init(loaded, 1);
    for (int i = 0; i < UNITS; ++i) tc::mbar_init(&acc_full[i], 1);
    tc::mbar_init(ready, EPI_WARPS);
    tc::mbar_init(drain, 1);
    *abort_flag = 0;
    tc::fence_mbar_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&smap)) : "memory");
  }
  if (warp == 0) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_launch_dependents();
  grid_wait();

  if (warp == 0) {
    // ------------------------ the load, the products ------------------------
    if (elect_one() && !g.no_async) {
      tc::mbar_arrive_expect_tx(loaded, MATRIX);
#pragma unroll
      for (int i = 0; i < 4; ++i)  // (term, block); zeros beyond m
        tma_load_4d<false>(tc::smem_u32(S) + i * BLOCK, &smap, (i & 1) * 64, 0, i >> 1,
                           blockIdx.x, tc::smem_u32(loaded));
    }
    __syncwarp();
    bool ok = wait_warp(watch, loaded, 0);
    const uint32_t id = (1u << 4) | ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(N >> 4) << 24);
    // one body for every product: a launch meets its code cold
#pragma unroll 1
    for (int i = 0; i < ops && ok; ++i) {
      const Op op = op_of(i, run);
      const uint32_t a = tc::smem_u32(op.kind == kP ? S : op.step == 0 ? Q : P);
      const uint32_t b = tc::smem_u32(op.kind == kQ ? Q : S);
      if (i > 0) ok = wait_warp(watch, ready, (i - 1) & 1);
      if (!ok) break;
      tc::tc_fence_after();
      const uint64_t da = tc::sdesc_sw128(a), db = tc::sdesc_sw128(b);
      // (the wait above also says that the last results are out of the
      // accumulators)
      if (elect_one()) {
        constexpr uint64_t lo = TERM >> 4;  // a descriptor's address counts 16 bytes
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          if (u < units) {
            const uint32_t d = tmem + u * N;
#pragma unroll
            for (int k = 2 * u; k < 2 * u + 2; ++k) {  // the small terms first
              const uint64_t o = (uint64_t)(((k >> 2) * BLOCK + (k & 3) * 32) >> 4);
              if (k < ksteps) {
                tc::umma_bf16(d, da + o, db + o + lo, id, k != 2 * u ? 1u : 0u);
                tc::umma_bf16(d, da + o + lo, db + o, id, 1u);
              }
            }
#pragma unroll
            for (int k = 2 * u; k < 2 * u + 2; ++k) {
              const uint64_t o = (uint64_t)(((k >> 2) * BLOCK + (k & 3) * 32) >> 4);
              if (k < ksteps) tc::umma_bf16(d, da + o, db + o, id, 1u);
            }
            tc::umma_commit(&acc_full[u]);
          }
        }
      }
      __syncwarp();
    }
    if (!ok && elect_one()) {  // what was issued completes before the CTA leaves
      if (!g.no_async) tc::drain_wait(loaded, 0, g.wait_limit);
      tc::umma_commit(drain);
      tc::drain_wait(drain, 0, g.wait_limit);
    }
    __syncwarp();
  } else {
    // ------------------------------ results ------------------------------
    // Warp w reads the tensor-memory lanes of its quarter (w % 4), columns
    // [32 h, 32 h + 32) and [64 + 32 h, 96 + 32 h) with h = (w - 1) / 4.
    const int q = warp & 3, h = (warp - 1) >> 2;
    const int row = q * 32 + lane;
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    bool ok = wait_warp(watch, loaded, 0);
#pragma unroll 1
    for (int i = 0; i < ops && ok; ++i) {
      const Op op = op_of(i, run);
      const bool poly = op.kind == kP;
      const float to = op.step == 0 ? g.c.scale_q : g.c.scale_p;
      const float ca = g.c.coef[3 * op.step] * to;
      const float cb = g.c.coef[3 * op.step + 1] * to / g.c.scale_s;
      const float factor =
          poly ? g.c.coef[3 * op.step + 2] * to / (g.c.scale_s * g.c.scale_s) : 1.f / to;
      // the last result goes to global memory
      unsigned char* dst = i + 1 == ops ? nullptr
                           : op.kind == kS ? S : op.kind == kQ || op.step == 0 ? Q : P;
      // the last unit's commit covers the products of all
      ok = wait_warp(watch, &acc_full[units - 1], i & 1);
      if (!ok) break;
      tc::tc_fence_after();
      // (the rows from `cols` on are nobody's operand and hold anything)
      const float lost = ksteps == 1 ? kStepLoss : kUnitLoss;
      const uint64_t loss = pair(lost, lost), f2 = pair(factor, factor);
      const uint64_t cb2 = pair(cb, cb);
      if (q * 32 < cols) {
#pragma unroll 1
        for (int c0 = 32 * h; c0 < cols; c0 += 64) {
          uint64_t acc[16];
#pragma unroll
          for (int u = 0; u < UNITS; u += 2) {  // two units' columns at a time
            if (u >= units) continue;
            uint32_t r[2][32];
            tmem_ld32(tmem + lanes + u * N + c0, r[0]);
            if (u + 1 < units) tmem_ld32(tmem + lanes + (u + 1) * N + c0, r[1]);
            tc::tmem_ld_wait();
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              if (u + v >= units) continue;
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const uint64_t x =
                    pair(__uint_as_float(r[v][2 * e]), __uint_as_float(r[v][2 * e + 1]));
                acc[e] = u + v == 0 ? x : add2(acc[e], x);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            const int col = c0 + j;
            if (col >= cols) continue;
            uint64_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint64_t x = acc[j / 2 + e];
              v[e] = mul2(fma2(x, loss, x), f2);
            }
            if (poly) {  // + b S + a I
              const uint4 sh = *reinterpret_cast<const uint4*>(S + at(row, col));
              const uint4 sl = *reinterpret_cast<const uint4*>(S + TERM + at(row, col));
              v[0] = fma2(join2(sh.x, sl.x), cb2, v[0]);
              v[1] = fma2(join2(sh.y, sl.y), cb2, v[1]);
              v[2] = fma2(join2(sh.z, sl.z), cb2, v[2]);
              v[3] = fma2(join2(sh.w, sl.w), cb2, v[3]);
              const int d = row - col;
              if (d >= 0 && d < 8 && row < m) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  v[e] = add2(v[e], pair(d == 2 * e ? ca : 0.f, d == 2 * e + 1 ? ca : 0.f));
              }
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) split2(v[e], hi[e], lo[e]);
            const uint4 hv = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            const uint4 lv = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            if (dst != nullptr) {
              *reinterpret_cast<uint4*>(dst + at(row, col)) = hv;
              *reinterpret_cast<uint4*>(dst + TERM + at(row, col)) = lv;
            } else if (row < m && col < m) {  // the pitch is a multiple of eight
              unsigned short* o = g.c.out + (long long)blockIdx.x * g.c.batch_stride +
                                  (long long)row * g.c.pitch + col;
              *reinterpret_cast<uint4*>(o) = hv;
              *reinterpret_cast<uint4*>(o + g.c.term_stride) = lv;
            }
          }
        }
      }
      tc::fence_proxy_async();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(ready);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 0) tc::tmem_dealloc(tmem, 512);
}

}  // namespace

cudaError_t launch_ortho_chain(const ChainArgs& c, const GemmOperand& s, int count,
                               long long wait_limit, int no_async, cudaStream_t stream) {
  if (c.m <= 0 || c.m > kChainMax || c.run <= 0 || c.run > kChainMaxRun)
    return cudaErrorInvalidValue;
  CUtensorMap map;
  cudaError_t e = make_tmap_4d(&map, s.base, false, (uint64_t)s.inner, (uint64_t)s.rows,
                               (uint64_t)s.pitch, 2, (uint64_t)s.term_stride, (uint64_t)count,
                               (uint64_t)s.batch_stride, N);
  if (e != cudaSuccess) return e;
  const Args g{c, wait_limit, no_async};
  e = ensure_dynamic_smem(reinterpret_cast<const void*>(ortho_chain_kernel), SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)count);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, ortho_chain_kernel, map, g);
}

cudaError_t read_chain_status(int* status, bool clear, cudaStream_t stream) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_chain_status, sizeof(int), 0,
                                            cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e == cudaSuccess && clear && v != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_chain_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice,
                                stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  }
  *status = v;
  return e;
}

}  // namespace dcn
