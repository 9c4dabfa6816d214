// Arguments of the log-probability launch (logprobs.cu).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace skinny {

constexpr int kLpMaxTop = 32;           // alternatives per row
constexpr int kLpMaxVocab = 1 << 27;    // logits per row

struct LogprobParams {
  const void* x;  // [rows, V], row stride ld
  long long ld;
  int rows, V, top;
  const int32_t* tokens;  // [rows]
  float *logprob, *entropy, *top_lp;
  int32_t* top_id;        // [rows, top]
};

size_t logprob_ws_bytes(int rows, int V, int top, int n_sm);
cudaError_t logprob_launch(const LogprobParams& prm, bool f32, void* ws, int n_sm, cudaStream_t stream);

}  // namespace skinny
