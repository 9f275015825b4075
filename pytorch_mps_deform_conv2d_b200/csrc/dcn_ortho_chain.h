// dcn_ortho_chain.h -- a run of Newton-Schulz steps on small Gram matrices in
// one launch (dcn_ortho_chain.cu).
#pragma once

#include <cuda_runtime.h>

#include "dcn_gemm.h"

namespace dcn {

constexpr int kChainMax = 128, kChainMaxRun = 32;

struct ChainArgs {
  int m, run;                   // matrices are m x m; steps of the run
  float coef[3 * kChainMaxRun];
  float scale_s, scale_p, scale_q;  // what S, P, Q are stored times
  unsigned short* out;          // Q, two terms
  long long pitch, term_stride, batch_stride;
};

// `s`: the two-term Gram matrices, `count` of them.
cudaError_t launch_ortho_chain(const ChainArgs& c, const GemmOperand& s, int count,
                               long long wait_limit, int no_async, cudaStream_t stream);
cudaError_t read_chain_status(int* status, bool clear, cudaStream_t stream);

}  // namespace dcn
