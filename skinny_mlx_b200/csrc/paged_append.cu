// Append a step's keys and values to a paged cache, rotating queries and keys on the way:
//
//   p        = lengths[b] + t                       (token t < counts[b] of sequence b)
//   x'[j]    = x[j] cos(p f_j) - x[j + h] sin(p f_j)
//   x'[j+h]  = x[j + h] cos(p f_j) + x[j] sin(p f_j)   j < h = rot / 2; dims >= rot unchanged
//   q_out[b, t] = bf16(q')                          (zero for t >= counts[b])
//   page table[b][p / page], slot p % page <- k', v   (bf16, or e4m3(x / scale[head]), saturating)
//
// Bound by the bytes moved: every input element is read once and every output written once, in
// 16-byte pieces.  A CTA owns one token (few tokens: a slice of one token's heads) so that the
// rotation table is computed once for all heads of the token.
//
// The angle p f_j is formed in f64: at p = 131072 an f32 product is off by up to 2^-24 * p, 0.008
// rad, four bf16 steps of the result.  The product of an integer below 2^29 and an f32 is exact in
// f64; as a count of turns, less its whole part, it is off by at most 2^-52 of itself, and the f32
// rounding of that fraction (2^-25 turns) is what remains.
#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "paged.cuh"
#include "ptx.cuh"

namespace skinny {

__device__ uint32_t g_paged_err;  // error bits of this device's paged calls

constexpr int kPaThreads = 128;
constexpr int kPaAhead = 2;      // pieces per thread whose loads are issued together (1: 41.4 us for 8191 tokens, 2: 39.4, 4: 42.5; back-to-back graph replays)
constexpr int kPaMaxHalf = 128;  // rotation pairs (head dim <= 256)

__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint4 r;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
  return r;
}

// 8 elements of a page: bf16, or e4m3 of the quotient (a true division, so that the rounding to
// 8 bits is the definition's; infinities saturate to 448, NaN stays NaN).
template <bool F8>
__device__ __forceinline__ void store8(void* base, long long off, const float (&x)[8], float scale) {
  if (F8) {
    uint2 r;
    __nv_fp8x2_storage_t* h = reinterpret_cast<__nv_fp8x2_storage_t*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[2 * i], scale), __fdiv_rn(x[2 * i + 1], scale)),
                                      __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(base) + off) = r;
  } else {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + off) = pack8(x);
  }
}

// One piece of a token: 8 dims of a head and, where they are rotated, the 8 they are paired with.
struct PagedPiece {
  uint4 x, y;
  int kind;  // 0 query, 1 key, 2 value; -1 none
  int h, d;
  bool pair;
};

template <bool F8>
__global__ void __launch_bounds__(kPaThreads) paged_append_kernel(const __grid_constant__ PagedAppendParams p) {
  // cos and sin of pair j at [j % 8][j / 8]: the lanes of a warp, at pairs 8 u + c, read neighbours
  __shared__ float2 cs[8][kPaMaxHalf / 8];
  const int tid = threadIdx.x;
  const int b = blockIdx.x / p.seq.T, t = blockIdx.x % p.seq.T;
  const int half = p.rot >> 1;
  // Per query or key head half/8 pairs of pieces, then (D - rot)/8 plain pieces; per value head D/8 plain ones.
  const int pairs = half >> 3, per = pairs + ((p.D - p.rot) >> 3), perv = p.D >> 3;
  const int nq = p.q ? p.Hq * per : 0, nk = p.Hkv * per, all = nq + nk + p.Hkv * perv;
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  int len, cnt;
  const bool ok = p.seq.get(b, len, cnt);
  const bool live = t < cnt;
  const int pos = len + t;
  // the token's rows; a piece's head by a multiplication (p.inv_per = ceil(2^32 / per), exact below 2^27 pieces)
  const __nv_bfloat16* const qt = p.q + b * p.qs[0] + t * p.qs[1];
  const __nv_bfloat16* const kt = p.k + b * p.ks[0] + t * p.ks[1];
  const __nv_bfloat16* const vt = p.v + b * p.vs[0] + t * p.vs[1];
  const auto load = [&](int e) {
    PagedPiece q;
    q.kind = e >= all ? -1 : e < nq ? 0 : e < nq + nk ? 1 : 2;
    int u;
    if (q.kind == 2) {
      q.h = (e - nq - nk) >> p.perv_log;
      u = (e - nq - nk) & (perv - 1);
      q.d = 8 * u;
      q.pair = false;
    } else {
      const int r = q.kind == 1 ? e - nq : e;
      q.h = p.inv_per ? static_cast<int>(__umulhi(static_cast<uint32_t>(r), p.inv_per)) : r;
      u = r - q.h * per;
      q.pair = u < pairs;
      q.d = q.pair ? 8 * u : p.rot + 8 * (u - pairs);
    }
    q.x = q.y = make_uint4(0u, 0u, 0u, 0u);
    if (live && q.kind >= 0) {
      const __nv_bfloat16* const src = (q.kind == 0   ? qt + q.h * p.qs[2]
                                        : q.kind == 1 ? kt + q.h * p.ks[2]
                                                      : vt + q.h * p.vs[2]) + q.d;
      q.x = *reinterpret_cast<const uint4*>(src);
      if (q.pair) q.y = *reinterpret_cast<const uint4*>(src + half);
    }
    return q;
  };
  const int step = gridDim.y * kPaThreads, e0 = blockIdx.y * kPaThreads + tid;
  PagedPiece q[kPaAhead];
#pragma unroll
  for (int i = 0; i < kPaAhead; ++i) q[i] = load(e0 + i * step);  // in flight while the table is made
  int page = -1;
  long long slot = 0;
  if (live) {
    const int at = pos / p.seq.page;
    page = p.seq.table[b * p.seq.table_stride + at];
    slot = pos - at * p.seq.page;
    if (page < 0 || page >= p.seq.n_pages) page = -1;
    for (int j = tid; j < half; j += kPaThreads) {
      const double turns = static_cast<double>(pos) * static_cast<double>(p.inv_freq[j]) * 0.15915494309189533577;
      float sn, c;
      sincospif(2.f * static_cast<float>(turns - rint(turns)), &sn, &c);
      cs[j & 7][j >> 3] = make_float2(c, sn);
    }
  }
  if (tid == 0 && blockIdx.y == 0 && (!ok || (live && page < 0))) atomicOr(p.seq.err, kErrBitBadInput);
  __syncthreads();
  for (int e = e0; e < all; e += kPaAhead * step) {
    if (e != e0)
#pragma unroll
      for (int i = 0; i < kPaAhead; ++i) q[i] = load(e + i * step);
#pragma unroll
    for (int i = 0; i < kPaAhead; ++i) {
      if (q[i].kind < 0) continue;
      float x[8], y[8];
      unpack8(q[i].x, x);
      unpack8(q[i].y, y);
      if (q[i].pair && live) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float2 w = cs[c][q[i].d >> 3];
          const float a = x[c] * w.x - y[c] * w.y;
          y[c] = y[c] * w.x + x[c] * w.y;
          x[c] = a;
        }
      }
      const int h = q[i].h, d = q[i].d;
      if (q[i].kind == 0) {  // (zero where the token is padding)
        __nv_bfloat16* dst = p.q_out + (static_cast<long long>(blockIdx.x) * p.Hq + h) * p.D + d;
        *reinterpret_cast<uint4*>(dst) = pack8(x);
        if (q[i].pair) *reinterpret_cast<uint4*>(dst + half) = pack8(y);
      } else if (live && page >= 0) {
        const bool isv = q[i].kind == 2;
        const long long off = page * (isv ? p.vps : p.kps) + (static_cast<long long>(h) * p.seq.page + slot) * p.D + d;
        const float sc = F8 ? (isv ? p.v_scale[h] : p.k_scale[h]) : 1.f;
        void* base = isv ? p.vp : p.kp;
        store8<F8>(base, off, x, sc);
        if (q[i].pair) store8<F8>(base, off + half, y, sc);
      }
    }
  }
}

cudaError_t paged_append_launch(const PagedAppendParams& params, bool f8, int n_sm, cudaStream_t stream) {
  PagedAppendParams prm = params;
  const long long tokens = static_cast<long long>(prm.seq.B) * prm.seq.T;
  const int half = prm.rot / 2, per = half / 8 + (prm.D - prm.rot) / 8;
  prm.inv_per = per == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + per - 1) / per);
  prm.perv_log = prm.D == 64 ? 3 : prm.D == 128 ? 4 : 5;
  const int pieces = ((prm.q ? prm.Hq : 0) + prm.Hkv) * per + prm.Hkv * (prm.D / 8);
  // With few tokens their heads are spread over the SMs (each CTA then repeats the rotation table).
  const long long want = (2ll * n_sm + tokens - 1) / tokens;
  const int most = (pieces + kPaThreads - 1) / kPaThreads;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tokens), static_cast<unsigned>(want < most ? want : most));
  cfg.blockDim = dim3(kPaThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, f8 ? paged_append_kernel<true> : paged_append_kernel<false>, prm);
}

// ---------------------------------------------------------------------------------------------
// the device's paged error word
// ---------------------------------------------------------------------------------------------
cudaError_t paged_error_word(int dev, uint32_t** word) {
  static std::atomic<uint32_t*> cached[64];
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  uint32_t* w = cached[dev].load(std::memory_order_acquire);
  if (!w) {
    void* a = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&a, g_paged_err);
    if (e != cudaSuccess) return e;
    w = static_cast<uint32_t*>(a);
    cached[dev].store(w, std::memory_order_release);
  }
  *word = w;
  return cudaSuccess;
}

}  // namespace skinny
