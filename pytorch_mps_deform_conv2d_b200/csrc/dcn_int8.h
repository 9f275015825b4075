// dcn_int8.h -- 8-bit codes of rows (a scale each), the sampled columns of a
// deformable convolution as such rows, and repacking for the products.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "dcn_common.cuh"
#include "dcn_gemm.h"

namespace dcn {

// x (rows, cols) of `type`, row pitch `ldx` elements -> q (rows, cols) with row
// pitch `ldq`, scale[row] = max |x| / 127, q = round(x / scale) (ties to even;
// zeros for a row of zeros).  A row with NaN or an infinity gets zeros and
// that value as its scale.
cudaError_t launch_quantize_rows(const void* x, int type, long long rows, int cols, long long ldx,
                                 signed char* q, long long ldq, float* scale,
                                 cudaStream_t stream);
// Whether a product of so few tokens can run as one kernel that codes the tokens
// itself, whether that is the faster way, and that kernel: x (tokens, K) of
// `x_type` (3: int8 with x_scale), weight (N, K), both dense and 16-byte aligned.
bool few_tokens_fit(int64_t tokens, int64_t K);
bool few_tokens_pay(int x_type, int64_t tokens, int64_t K, int64_t N);
cudaError_t launch_few_tokens(const void* x, int x_type, const float* x_scale, int tokens, int K,
                              int N, const signed char* w, const float* w_scale, const void* bias,
                              int bias_type, void* out, int out_type, cudaStream_t stream);
// 8-bit rows into rows of pitch `ldo`.
cudaError_t launch_repack_i8(const signed char* in, long long rows, int cols, signed char* out,
                             long long ldo, cudaStream_t stream);
// Columns of output pixels [p0, p0 + np) (counted over the batch) as 8-bit
// rows: col[group][pixel - p0][tap * Cg + channel] with row pitch `kp` and
// scale[group][pixel - p0].  `x` is NHWC; x, offset and mask are of `type`.
cudaError_t launch_sample_i8(const Geom& g, const void* x, int type, const void* off,
                             const void* mask, long long p0, int np, signed char* col, int kp,
                             float* scale, cudaStream_t stream);

}  // namespace dcn
