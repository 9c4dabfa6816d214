// Attention of 1..16 new tokens per sequence over a paged key-value cache:
//
//   o[b, t, h] = sum_j softmax_j(scale * q[b, t, h] . k_j) v_j     (query head h reads kv head h / rep)
//
// over the positions j <= lengths[b] + t of sequence b's pages (and j > lengths[b] + t - window).
// A row that sees nothing (an idle slot, t >= counts[b], every page bad) is zero, its lse -inf.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "paged.cuh"
#include "ptx.cuh"

namespace skinny {

// One warp per query row: lane l holds dims l, l + 32, ...
template <bool F8>
__global__ void __launch_bounds__(128) paged_attn_kernel(const __grid_constant__ PagedAttnParams p) {
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<long long>(p.seq.B) * p.seq.T * p.Hq) return;
  const int h = row % p.Hq, t = row / p.Hq % p.seq.T, b = row / p.Hq / p.seq.T;
  const int g = h / (p.Hq / p.Hkv), n = p.D / 32;
  int len, cnt;
  bool ok = p.seq.get(b, len, cnt);
  float q[8], o[8], m = -INFINITY, l = 0.f;
  for (int i = 0; i < n; ++i) {
    q[i] = __bfloat162float(p.q[b * p.qs[0] + t * p.qs[1] + h * p.qs[2] + lane + 32 * i]);
    o[i] = 0.f;
  }
  const float ks = F8 ? p.k_scale[g] : 1.f, vs = F8 ? p.v_scale[g] : 1.f;
  if (t < cnt) {
    const int end = len + t + 1, beg = p.window > 0 ? max(0, end - p.window) : 0;
    for (int j = beg; j < end; ++j) {
      const int page = p.seq.table[b * p.seq.table_stride + j / p.seq.page];
      if (page < 0 || page >= p.seq.n_pages) {
        ok = false;
        continue;
      }
      const long long in = (static_cast<long long>(g) * p.seq.page + j % p.seq.page) * p.D + lane;
      const auto at = [&](const void* base, long long off) {
        if (F8) {
          __nv_fp8_e4m3 x;
          x.__x = static_cast<const uint8_t*>(base)[off];
          return static_cast<float>(x);
        }
        return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[off]);
      };
      float s = 0.f;
      for (int i = 0; i < n; ++i) s = fmaf(q[i], at(p.kp, page * p.kps + in + 32 * i), s);
      for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, w);
      s *= p.scale * ks;
      const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
      const float f = expf(m - mu), e = expf(s - mu);
      l = l * f + e;
      for (int i = 0; i < n; ++i) o[i] = o[i] * f + e * at(p.vp, page * p.vps + in + 32 * i);
      m = mn;
    }
  }
  if (!ok && lane == 0) atomicOr(p.seq.err, kErrBitBadInput);
  for (int i = 0; i < n; ++i) p.out[row * p.D + lane + 32 * i] = __float2bfloat16_rn(l > 0.f || l != l ? o[i] * vs / l : 0.f);
  if (p.lse && lane == 0) p.lse[row] = m + logf(l);
}

size_t paged_attn_ws_bytes(int, int, int, int, int, int) { return 16; }

cudaError_t paged_attn_launch(const PagedAttnParams& p, bool f8, void*, int, cudaStream_t stream) {
  const long long rows = static_cast<long long>(p.seq.B) * p.seq.T * p.Hq;
  const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
  if (f8) paged_attn_kernel<true><<<grid, 128, 0, stream>>>(p);
  else paged_attn_kernel<false><<<grid, 128, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace skinny
