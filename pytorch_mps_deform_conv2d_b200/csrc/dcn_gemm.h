// dcn_gemm.h -- batched dense products on tcgen05: fp16 operands of one or two
// terms with fp32 accumulators, and 8-bit integer operands with exact int32
// accumulators.  Used by the orthogonalised updates (dcn_ortho.cu) and the
// 8-bit products (dcn_int8.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dcn {

// A batch of matrices in device memory: `rows` x `inner`, `inner` contiguous.
// A two-term fp16 operand holds value = high + low, the low matrix
// `term_stride` elements after the high one.  `base` 16-byte aligned, strides
// multiples of 16 bytes; `batch` 1 with the product's batch larger: shared.
struct GemmOperand {
  const void* base;
  long long rows, inner, pitch;  // elements
  int terms;
  long long term_stride;   // elements, when terms == 2
  int batch;
  long long batch_stride;  // elements, when batch > 1
  // the operand's rows run along K (its `inner` along M or N): the tensor
  // core takes it as it lies, fp16 only
  bool k_rows;
};

enum GemmEpilogue {
  // v = acc * scale[b] * factor, stored as fp16 terms (`out16`); with `sym`
  // large products compute the upper triangle of tiles and mirror it
  kEpiTerms = 0,
  // the same of v = (diag on the diagonal) + lin * L + acc * factor, L the
  // matrix `lin16` of the same layout and terms
  kEpiPoly = 1,
  // v = acc * scale[b] * factor into `out` of type `out_type`, dense rows of N
  kEpiOut = 2,
  // out = keep * out + v, v as above (a parameter updated where it lies)
  kEpiAxpy = 3,
  // y = acc * row_scale[b][m] * col_scale[b][n] + bias[b][n] into `out`, rows
  // of N (int8 products)
  kEpiRows = 4,
  // the same into an NCHW image batch: m counts (image, pixel), n channels of
  // group b: out[(m / pixels)][b * N + n][m % pixels]
  kEpiPlanes = 5,
};

enum GemmType { kF32 = 0, kBF16T = 1, kF16T = 2 };

constexpr int kGemmMaxList = 64;

struct GemmEpiArgs {
  int mode;
  float factor;
  const float* scale;  // NULL: 1
  float diag, lin, keep;
  unsigned short* out16;  // terms, pitch / strides below (elements)
  const unsigned short* lin16;
  int out_terms;
  long long pitch, term_stride, batch_stride;
  void* out;  // NULL: list[matrix]
  int out_type;
  int wide_ok;  // rows of `out` take 16-byte stores
  const float* row_scale;
  long long row_scale_batch;
  const float* col_scale;
  const void* bias;  // of out_type's sibling `bias_type`
  int bias_type;
  int pixels, channels;  // kEpiPlanes: pixels an image, channels of all groups,
  int m_base;            // and the pixel that m = 0 stands for; pixel_pairs:
  int pixel_pairs;       // M, m_base and pixels are even, `out` 4-byte aligned
  void* list[kGemmMaxList];
};

struct GemmProblem {
  GemmOperand a, b;  // D[m, n] = sum_k A[m, k] B[n, k]
  int M, N, K, batch;
  bool int8, sym;
  bool fine;        // two-term operands: sums to fp32's accuracy
  bool coarse;      // results of 11 bits and less
  bool after_ours;  // the launch before is one of this library's products, or
                    // another kernel whose writes this one may wait for late
  GemmEpiArgs epi;
  long long wait_limit;
  int no_async;
};

// Enqueues the product.  cudaErrorInvalidValue: a form that is not built.
cudaError_t launch_gemm(const GemmProblem& p, cudaStream_t stream);

// Error word of the kernel above (kStatusDense when a bounded wait ran out).
constexpr int kStatusDense = 0x8;
cudaError_t read_gemm_status(int* status, bool clear, cudaStream_t stream);

}  // namespace dcn
