// dcn_gemm_f16.cu -- products of one-term fp16 operands, and of a one-term with
// a two-term one (see dcn_gemm_kernel.cuh).
#include "dcn_gemm_kernel.cuh"

namespace dcn {

cudaError_t launch_gemm_f16(const GemmProblem& p, cudaStream_t stream) {
  const int ta = p.a.terms, tb = p.b.terms;
  const bool at = p.a.k_rows, bt = p.b.k_rows;
  if (!at && !bt) {
    if (ta == 1 && tb == 1) return launch_tiling<false, 1, 1, false, false, 16>(p, stream);
    if (ta == 1 && tb == 2) return launch_tiling<false, 1, 2, false, false, 16>(p, stream);
  }
  if (at && bt && ta == 1 && tb == 1) return launch_tiling<false, 1, 1, true, true, 16>(p, stream);
  if (!at && bt && ta == 1 && tb == 1) return launch_tiling<false, 1, 1, false, true, 16>(p, stream);
  if (!at && bt && ta == 2 && tb == 1) return launch_tiling<false, 2, 1, false, true, 16>(p, stream);
  return cudaErrorInvalidValue;
}
cudaError_t read_gemm_f16_status(int* status, bool clear, cudaStream_t stream) {
  return read_status(status, clear, stream);
}

}  // namespace dcn
