// dcn_gemm.cu -- int8 products, and the choice of the form (see
// dcn_gemm_kernel.cuh).
#include "dcn_gemm_kernel.cuh"
#include "dcn_ortho_chain.h"

namespace dcn {

cudaError_t launch_gemm_f16(const GemmProblem& p, cudaStream_t stream);
cudaError_t launch_gemm_f16x2(const GemmProblem& p, cudaStream_t stream);
cudaError_t read_gemm_f16_status(int* status, bool clear, cudaStream_t stream);
cudaError_t read_gemm_f16x2_status(int* status, bool clear, cudaStream_t stream);

cudaError_t launch_gemm(const GemmProblem& p, cudaStream_t stream) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0 || p.batch <= 0) return cudaErrorInvalidValue;
  if (p.int8) return launch_tiling<true, 1, 1, false, false, 0>(p, stream);
  return p.a.terms == 2 && p.b.terms == 2 ? launch_gemm_f16x2(p, stream)
                                          : launch_gemm_f16(p, stream);
}

cudaError_t read_gemm_status(int* status, bool clear, cudaStream_t stream) {
  int v[4] = {0, 0, 0, 0};
  cudaError_t e = read_status(&v[0], clear, stream);
  if (e == cudaSuccess) e = read_gemm_f16_status(&v[1], clear, stream);
  if (e == cudaSuccess) e = read_gemm_f16x2_status(&v[2], clear, stream);
  if (e == cudaSuccess) e = read_chain_status(&v[3], clear, stream);
  *status = v[0] | v[1] | v[2] | v[3];
  return e;
}

}  // namespace dcn
