// dcn_gemm_f16x2.cu -- products of two-term fp16 operands (see
// dcn_gemm_kernel.cuh), for fp32 results and, in longer units, for 16-bit ones.
#include "dcn_gemm_kernel.cuh"

namespace dcn {

cudaError_t launch_gemm_f16x2(const GemmProblem& p, cudaStream_t stream) {
  const bool at = p.a.k_rows, bt = p.b.k_rows;
  if (!p.fine) {
    if (!at && !bt) return launch_tiling<false, 2, 2, false, false, 16>(p, stream);
    if (at && bt) return launch_tiling<false, 2, 2, true, true, 16>(p, stream);
    if (bt) return launch_tiling<false, 2, 2, false, true, 16>(p, stream);
  } else {
    if (!at && !bt) return launch_tiling<false, 2, 2, false, false, 2>(p, stream);
    if (at && bt) return launch_tiling<false, 2, 2, true, true, 2>(p, stream);
    if (bt) return launch_tiling<false, 2, 2, false, true, 2>(p, stream);
  }
  return cudaErrorInvalidValue;
}
cudaError_t read_gemm_f16x2_status(int* status, bool clear, cudaStream_t stream) {
  return read_status(status, clear, stream);
}

}  // namespace dcn
