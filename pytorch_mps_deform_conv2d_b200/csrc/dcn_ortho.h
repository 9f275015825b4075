// dcn_ortho.h -- orthogonalised updates (Newton-Schulz) and the optimiser
// step around them: plan, workspace and launch of one chunk of matrices.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

#include "dcn_gemm.h"

namespace dcn {

constexpr int kOrthoMaxSteps = 32;

struct OrthoShape {
  int rows, cols;    // of one matrix; the recurrence runs over the smaller side
  int type;          // GemmType of the tensors
  int first_terms;   // fp16 terms of the scaled input
  int later_terms;   // of the matrix between two phases
  int steps;
  float coef[3 * kOrthoMaxSteps];  // (a, b, c) of each step
  float eps;
};

// What one chunk of matrices is made from and turned into.
struct OrthoChunk {
  int count;  // matrices, at most kGemmMaxList
  const void* in[kGemmMaxList];   // dense (rows, cols)
  void* out[kGemmMaxList];        // dense (rows, cols)
  // optimiser step: `in` are gradients, `out` parameters, updated in place:
  // m = beta m + rest g, u = nesterov ? rest g + beta m : m,
  // p = keep p + step O(u); rest is 1 - beta, rounded by itself
  float* momentum[kGemmMaxList];
  bool muon, nesterov;
  float beta, rest, keep, step;
};

size_t ortho_workspace_bytes(const OrthoShape& s, int count);
// `stage` receives the name of a launch that failed.
cudaError_t launch_ortho(const OrthoShape& s, const OrthoChunk& c, void* workspace,
                         long long wait_limit, int no_async, cudaStream_t stream,
                         const char** stage);

}  // namespace dcn
