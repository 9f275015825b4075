// dcn_dense_common.cuh -- helpers of the dense tcgen05 kernels (dcn_gemm_kernel.cuh,
// dcn_ortho_chain.cu): elected issue, programmatic launches, 4-D TMA loads,
// wide tensor-memory loads, 16-bit pairs.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dcn_gemm.h"
#include "dcn_tc_common.cuh"

namespace dcn {
namespace dense {

// The tensor core rounds its fp32 accumulator towards zero: a sum over 32
// values of K comes out 1.1 units of 2^-24 too small on average (0.8 for terms
// of both signs, 1.4 for squares; see dcn_gemm_kernel.cuh).  x + kUnitLoss x,
// rounded to nearest, is x or one place (2^-23 of its power of two) more, the
// latter for significands above 1.135: 1.1 units on average.
constexpr float kUnitLoss = 5.25e-8f;
// The same for sums over 16 values and less: 0.65 units, above 1.4.
constexpr float kStepLoss = 4.26e-8f;

// Two fp32 values side by side, and both at once.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// One lane of a converged warp.  The instructions below take their operands
// from uniform registers; under `lane == 0` the compiler does not know that one
// thread runs and wraps each in a loop over the active ones: 800 cycles a K
// slice, measured, against 512 of its products.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n.reg .pred p;\n"
      "elect.sync _|p, 0xFFFFFFFF;\n"
      "selp.b32 %0, 1, 0, p;\n}\n"
      : "=r"(r));
  return r != 0;
}
// A wait of the whole warp: all of its lanes come to the same answer.
__device__ __forceinline__ bool wait_warp(const tc::Watch& w, uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, tc::wait(w, bar, parity));
}

// 4-D tiled TMA load (no multicast): box at (x, y, term, matrix).  PAIR: the
// barrier may be the other CTA's.
template <bool PAIR>
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            int z, int w, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
        "bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

// ---- programmatic dependent launch: the prologue of a product runs beside the
// end of the launch before it ----
__device__ __forceinline__ void grid_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void grid_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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

template <int T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (T == kBF16T) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <int T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (T == kBF16T)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// A pair as two fp16 terms: hi, and what hi leaves.
__device__ __forceinline__ void split2(uint64_t v, uint32_t& hi, uint32_t& lo) {
  const float2 f = unpair(v);
  hi = pack2<kF16T>(f.x, f.y);
  const float2 h = unpack2<kF16T>(hi);
  lo = pack2<kF16T>(f.x - h.x, f.y - h.y);
}
// Two fp16 terms of a pair added up.
__device__ __forceinline__ uint64_t join2(uint32_t hi, uint32_t lo) {
  const float2 h = unpack2<kF16T>(hi), l = unpack2<kF16T>(lo);
  return add2(pair(h.x, h.y), pair(l.x, l.y));
}

}  // namespace dense
}  // namespace dcn
