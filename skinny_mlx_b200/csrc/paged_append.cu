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

template <bool F8>
__global__ void __launch_bounds__(kPaThreads) paged_append_kernel(const __grid_constant__ PagedAppendParams p) {
  __shared__ float cs[kPaMaxHalf][2];
  const int tid = threadIdx.x;
  const int b = blockIdx.x / p.seq.T, t = blockIdx.x % p.seq.T;
  const int half = p.rot >> 1;
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  int len, cnt;
  const bool ok = p.seq.get(b, len, cnt);
  const bool live = t < cnt;
  const int pos = len + t;
  int page = -1;
  if (live) {
    page = p.seq.table[b * p.seq.table_stride + pos / p.seq.page];
    if (page < 0 || page >= p.seq.n_pages) page = -1;
  }
  if (tid == 0 && blockIdx.y == 0 && (!ok || (live && page < 0))) atomicOr(p.seq.err, kErrBitBadInput);
  if (live)
    for (int j = tid; j < half; j += kPaThreads) {
      const double turns = static_cast<double>(pos) * static_cast<double>(p.inv_freq[j]) * 0.15915494309189533577;
      float s, c;
      sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
      cs[j][0] = c;
      cs[j][1] = s;
    }
  __syncthreads();
  const long long slot = live ? pos % p.seq.page : 0;
  // Pieces of the token: per query or key head half/8 pairs of 8 dims, then (D - rot)/8 plain
  // pieces; per value head D/8 plain pieces.
  const int pairs = half >> 3, per = pairs + ((p.D - p.rot) >> 3), perv = p.D >> 3;
  const int nq = p.q ? p.Hq * per : 0, nk = p.Hkv * per, nv = p.Hkv * perv;
  for (int e = blockIdx.y * kPaThreads + tid; e < nq + nk + nv; e += gridDim.y * kPaThreads) {
    const bool isq = e < nq, isv = e >= nq + nk;
    const int r = isq ? e : isv ? e - nq - nk : e - nq;
    const int w = isv ? perv : per;
    const int h = r / w, u = r - h * w;
    const bool pair = !isv && u < pairs;
    const int d = isv ? 8 * u : pair ? 8 * u : p.rot + 8 * (u - pairs);
    const __nv_bfloat16* src = isq ? p.q + b * p.qs[0] + t * p.qs[1] + h * p.qs[2]
                               : isv ? p.v + b * p.vs[0] + t * p.vs[1] + h * p.vs[2]
                                     : p.k + b * p.ks[0] + t * p.ks[1] + h * p.ks[2];
    float x[8], y[8];
    if (live) {
      unpack8(*reinterpret_cast<const uint4*>(src + d), x);
      if (pair) {
        unpack8(*reinterpret_cast<const uint4*>(src + d + half), y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float c = cs[d + i][0], s = cs[d + i][1];
          const float a = x[i] * c - y[i] * s;
          y[i] = y[i] * c + x[i] * s;
          x[i] = a;
        }
      }
    }
    if (isq) {
      if (!live) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
      }
      __nv_bfloat16* dst = p.q_out + (static_cast<long long>(blockIdx.x) * p.Hq + h) * p.D + d;
      *reinterpret_cast<uint4*>(dst) = pack8(x);
      if (pair) *reinterpret_cast<uint4*>(dst + half) = pack8(y);
    } else if (live && page >= 0) {
      const long long off = page * (isv ? p.vps : p.kps) + (static_cast<long long>(h) * p.seq.page + slot) * p.D + d;
      const float sc = F8 ? (isv ? p.v_scale[h] : p.k_scale[h]) : 1.f;
      void* base = isv ? p.vp : p.kp;
      store8<F8>(base, off, x, sc);
      if (pair) store8<F8>(base, off + half, y, sc);
    }
  }
}

cudaError_t paged_append_launch(const PagedAppendParams& prm, bool f8, int n_sm, cudaStream_t stream) {
  const long long tokens = static_cast<long long>(prm.seq.B) * prm.seq.T;
  const int half = prm.rot / 2, per = half / 8 + (prm.D - prm.rot) / 8;
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
