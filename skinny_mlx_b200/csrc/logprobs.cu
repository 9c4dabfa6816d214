// Log probabilities of given tokens, the entropy of each row and its most likely alternatives:
//
//   m = max x,  Z = sum e^(x - m),  lse = m + ln Z
//   logprob = x[token] - lse,  entropy = ln Z - (1/Z) sum e^(x - m) (x - m)
//   the n largest x - lse, by value, ties to the lowest index, a NaN above every number
//
// A logit of -inf has probability 0 and adds nothing; a row of nothing else has every logprob -inf
// and entropy 0; a row with a NaN or +inf has NaN sums.  A token outside the vocabulary has logprob
// -inf.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "logprobs.cuh"
#include "ptx.cuh"

namespace skinny {

// The order of a logit and its index as one number: larger value first, then the lower index.
__device__ __forceinline__ unsigned long long lp_key(float v, int i) {
  uint32_t b = v != v ? 0x7FFFFFFFu : __float_as_uint(v + 0.f);
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(b) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

template <typename T>
__global__ void __launch_bounds__(256) logprob_kernel(const __grid_constant__ LogprobParams p) {
  __shared__ float red[3][8];
  __shared__ unsigned long long keys[8];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = static_cast<const T*>(p.x) + row * p.ld;
  const auto at = [&](int i) { return static_cast<float>(x[i]); };
  float m = -INFINITY;
  for (int i = tid; i < p.V; i += 256) m = fmaxf(m, at(i));
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
  for (int w = 0; w < 8; ++w) m = fmaxf(m, red[0][w]);
  float z = 0.f, s = 0.f;
  for (int i = tid; i < p.V; i += 256) {
    const float v = at(i);
    if (v == -INFINITY) continue;
    const float d = v - m, e = expf(d);
    z += e;
    s += e * fmaxf(d, -1e30f);
  }
  for (int o = 16; o; o >>= 1) {
    z += __shfl_xor_sync(0xFFFFFFFFu, z, o);
    s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  }
  if (lane == 0) red[1][warp] = z, red[2][warp] = s;
  __syncthreads();
  z = s = 0.f;
  for (int w = 0; w < 8; ++w) z += red[1][w], s += red[2][w];
  const float lz = logf(z);
  const auto lp = [&](float v) { return v == -INFINITY && z == z ? -INFINITY : v - m - lz; };
  if (tid == 0) {
    const int t = p.tokens[row];
    p.logprob[row] = t < 0 || t >= p.V ? -INFINITY : lp(at(t));
    p.entropy[row] = m == -INFINITY && z == 0.f ? 0.f : lz - s / z;
  }
  unsigned long long prev = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < p.V; i += 256) {
      const unsigned long long key = lp_key(at(i), i);
      if ((k == 0 || key < prev) && key > best) best = key;
    }
    for (int o = 16; o; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xFFFFFFFFu, best, o);
      best = other > best ? other : best;
    }
    __syncthreads();
    if (lane == 0) keys[warp] = best;
    __syncthreads();
    for (int w = 0; w < 8; ++w) best = keys[w] > best ? keys[w] : best;
    prev = best;
    if (tid == 0) {
      const int i = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(best));
      p.top_id[static_cast<size_t>(row) * p.top + k] = i;
      p.top_lp[static_cast<size_t>(row) * p.top + k] = lp(at(i));
    }
  }
}

size_t logprob_ws_bytes(int, int, int, int) { return 16; }

cudaError_t logprob_launch(const LogprobParams& p, bool f32, void*, int, cudaStream_t stream) {
  if (f32) logprob_kernel<float><<<p.rows, 256, 0, stream>>>(p);
  else logprob_kernel<__nv_bfloat16><<<p.rows, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace skinny
