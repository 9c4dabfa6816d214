// Log probabilities of given tokens, the entropy of each row and its most likely alternatives:
//
//   m = max x,  Z = sum e^(x - m),  lse = m + ln Z
//   logprob = x[token] - lse,  entropy = ln Z - (1/Z) sum e^(x - m) (x - m)
//   the n largest x - lse, by value, ties to the lowest index, a NaN above every number
//
// A logit of -inf has probability 0 and adds nothing; a row of nothing else has every logprob -inf
// and entropy 0; a row with a NaN or +inf has NaN sums.  A token outside the vocabulary has logprob
// -inf.
//
// One pass over the logits: every thread keeps a running maximum and the two sums relative to it in
// f32 (renewed when a 16-byte piece exceeds it).  Bound by the bytes of the logits; next comes the
// exponential unit (16 per clock and SM, where a bf16 stream at full bandwidth wants 12).
//
// Alternatives.  A logit and its index form one 64-bit key whose order is the order wanted; keys are
// all different.  The first pieces of four runs that a CTA's part of the row is read in (up to 8192 logits, in
// registers) give a threshold that at least n keys reach: the n-th largest of the maxima of 64 groups.  After that, a
// piece costs one comparison; what reaches the threshold, some n * (part / sample) logits, is put on a
// list in shared memory, which is cut down by the same group maxima and ranked.  Rows whose order
// defeats the threshold (rising logits) overflow the list: the part is then read again to find the
// n-th key 12 bits at a time (a histogram per pass), which no input makes longer than 6 passes.
//
// Few rows: a row is cut into parts, one CTA each, and a second launch joins their sums and lists.
#include <algorithm>
#include <cstdint>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "logprobs.cuh"
#include "ptx.cuh"

namespace skinny {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpGroups = 64;      // groups whose maxima give a threshold (at least kLpMaxTop)
constexpr int kLpList = 2048;      // keys a CTA's list holds
constexpr int kLpRank = 128;       // keys that are ranked against each other
constexpr int kLpSample = 4;       // 16-byte pieces per thread of the sample
constexpr int kLpRadix = 12;       // bits per pass of the search for the n-th key
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLpLow = -3.402823466e38f;

static_assert(kLpGroups >= kLpMaxTop && kLpGroups * 4 == kLpThreads, "groups of 4 threads");

// The order of a logit and its index as one number: larger value first, then the lower index; NaN
// above every number, -0 and 0 alike.  Never 0.
__device__ __forceinline__ unsigned long long lp_key(float v, int i) {
  uint32_t b = v != v ? 0x7FFFFFFFu : __float_as_uint(v + 0.f);
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(b) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int lp_index(unsigned long long key) {
  return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}
// The value a key was made of (NaN for every NaN).
__device__ __forceinline__ float lp_value(unsigned long long key) {
  const uint32_t b = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}

__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The larger; NaN if either is (an ordinary maximum drops it).
__device__ __forceinline__ float lp_max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Running maximum (of numbers) and sums of e = e^(x - m) and e (x - m).
struct LpSums {
  float m = kLpLow, z = 0.f, s = 0.f;
  // to maximum n >= m: z -> z f, s -> f (s + z (m - n)), f = e^(m - n)
  __device__ __forceinline__ void renew(float n) {
    const float d = m - n, f = lp_exp2(d * kLog2e);
    s = z == 0.f ? 0.f : f == 0.f && z == z && s == s ? 0.f : f * fmaf(z, d, s);
    z *= f;
    m = n;
  }
  __device__ __forceinline__ void join(float om, float oz, float os) {
    LpSums o;
    o.m = om, o.z = oz, o.s = os;
    const float n = fmaxf(m, om);
    renew(n);
    o.renew(n);
    z += o.z;
    s += o.s;
  }
};

// The logits of one 16-byte piece: 8 bf16 or 4 f32.
template <bool F32>
struct LpPiece {
  static constexpr int kN = F32 ? 4 : 8;
  float x[kN];
  __device__ __forceinline__ explicit LpPiece(const uint4& w) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (F32) {
        x[i] = __uint_as_float(u[i]);
      } else {
        x[(F32 ? 0 : 2) * i] = __uint_as_float(u[i] << 16);
        x[(F32 ? 0 : 2) * i + (F32 ? 0 : 1)] = __uint_as_float(u[i] & 0xFFFF0000u);
      }
    }
  }
  // The largest, NaN above every number.
  __device__ __forceinline__ float top() const {
    float t = x[0];
#pragma unroll
    for (int i = 1; i < kN; ++i) t = lp_max_nan(t, x[i]);
    return t;
  }
  __device__ __forceinline__ void add(LpSums& a, float top) const {
    if (top > a.m) a.renew(top);
    // d is bounded below so that 0 times an infinite d (a logit of -inf) is 0; NaN stays NaN
    uint64_t z2 = f2_pack(0.f, 0.f), s2 = z2;
    const uint64_t nm = f2_pack(-a.m, -a.m), one = f2_pack(1.f, 1.f), l2 = f2_pack(kLog2e, kLog2e);
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
      float d0, d1, a0, a1;
      f2_unpack(f2_fma(f2_pack(x[i], x[i + 1]), one, nm), d0, d1);
      const uint64_t d = f2_pack(lp_max_nan(d0, -1e4f), lp_max_nan(d1, -1e4f));
      f2_unpack(f2_mul(d, l2), a0, a1);
      const uint64_t e = f2_pack(lp_exp2(a0), lp_exp2(a1));
      z2 = f2_fma(e, one, z2);
      s2 = f2_fma(e, d, s2);
    }
    float a0, a1;
    f2_unpack(z2, a0, a1);
    a.z += a0 + a1;
    f2_unpack(s2, a0, a1);
    a.s += a0 + a1;
  }
};

struct LpPlan {
  int parts, part;            // CTAs per row, logits of one part
  unsigned long long* keys;   // [rows, parts, top]
  float* sums;                // [rows, parts, 4]: m, z, s
};

struct LpSmem {
  unsigned long long list[2][kLpList];
  unsigned long long group[kLpGroups];
  int count[2];
  int scan[kLpWarps];
  unsigned long long threshold;
};

// The n-th largest of the group maxima (each lane of a group of 4 threads brings a key): n keys at least
// reach it.  All threads call it; 0 when fewer than n groups have a key.
__device__ unsigned long long lp_threshold(LpSmem& sm, unsigned long long key, int n) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const unsigned long long x = __shfl_xor_sync(0xFFFFFFFFu, key, o);
    key = x > key ? x : key;
  }
  if ((tid & 3) == 0) sm.group[tid >> 2] = key;
  if (tid == 0) sm.threshold = 0;
  __syncthreads();
  if (tid < kLpGroups) {
    const unsigned long long mine = sm.group[tid];
    int above = 0;
    const ulonglong2* const all = reinterpret_cast<const ulonglong2*>(sm.group);
#pragma unroll 8
    for (int i = 0; i < kLpGroups / 2; ++i) {
      const ulonglong2 x = all[i];
      above += (x.x > mine) + (x.y > mine);
    }
    if (above == n - 1 && mine != 0) sm.threshold = mine;  // (keys differ: one thread)
  }
  __syncthreads();
  return sm.threshold;
}

// The n largest keys of list[0][0 .. cnt), in order, to out(rank, key).  All threads call it; fewer than n
// keys give as many.  A group's maxima cut the list to n groups' keys per turn.
template <typename Out>
__device__ void lp_rank(LpSmem& sm, int cnt, int n, Out out) {
  const int tid = threadIdx.x;
  int cur = 0;
  while (cnt > kLpRank) {
    unsigned long long best = 0;
    for (int i = tid; i < cnt; i += kLpThreads) best = sm.list[cur][i] > best ? sm.list[cur][i] : best;
    if (tid == 0) sm.count[cur ^ 1] = 0;
    const unsigned long long t = lp_threshold(sm, best, n);  // (cnt > 64 n / 32: every group has keys)
    for (int i = tid; i < cnt; i += kLpThreads)
      if (sm.list[cur][i] >= t) sm.list[cur ^ 1][atomicAdd(&sm.count[cur ^ 1], 1)] = sm.list[cur][i];
    __syncthreads();
    cur ^= 1;
    cnt = sm.count[cur];
    __syncthreads();
  }
  if (tid < cnt) {
    const unsigned long long mine = sm.list[cur][tid];
    int above = 0;
    for (int i = 0; i < cnt; ++i) above += sm.list[cur][i] > mine;
    if (above < n) out(above, mine);
  }
}

// A part that is read again after its list overflowed: the n-th largest key, kLpRadix bits at a time,
// from the top; then the list holds the keys that reach it, n in all.
template <bool F32>
__device__ __noinline__ void lp_search(LpSmem& sm, const void* row, int c0, int c1, int n) {
  const int tid = threadIdx.x;
  uint32_t* const hist = reinterpret_cast<uint32_t*>(&sm.list[0][0]);  // 2^kLpRadix bins
  const auto at = [&](int i) {
    return F32 ? static_cast<const float*>(row)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
  };
  unsigned long long prefix = 0;  // the bits found, at the top
  int want = n;                   // the rank among the keys with that prefix
  for (int left = 64; left > 0;) {
    const int bits = min(kLpRadix, left), shift = left - bits;
    __syncthreads();
    for (int i = tid; i < 1 << kLpRadix; i += kLpThreads) hist[i] = 0;
    __syncthreads();
    for (int i = c0 + tid; i < c1; i += kLpThreads) {
      const unsigned long long key = lp_key(at(i), i);
      if (left == 64 || key >> left == prefix >> left) atomicAdd(&hist[key >> shift & ((1u << bits) - 1u)], 1u);
    }
    __syncthreads();
    // the bin, from the largest down, in which the count passes `want`: thread i has 16 bins
    constexpr int kPer = (1 << kLpRadix) / kLpThreads;
    const int hi = (1 << kLpRadix) - 1 - tid * kPer, warp = tid >> 5, lane = tid & 31;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine += hist[hi - i];
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) sm.scan[warp] = incl;
    __syncthreads();
    for (int i = 0; i < warp; ++i) incl += sm.scan[i];
    if (incl - mine < want && want <= incl) {
      int rest = want - (incl - mine), bin = hi;
      for (; static_cast<int>(hist[bin]) < rest; --bin) rest -= hist[bin];
      sm.threshold = prefix | static_cast<unsigned long long>(bin) << shift;
      sm.count[0] = rest;
    }
    __syncthreads();
    prefix = sm.threshold;
    want = sm.count[0];
    left = shift;
  }
  __syncthreads();
  if (tid == 0) sm.count[0] = 0;
  __syncthreads();
  for (int i = c0 + tid; i < c1; i += kLpThreads) {
    const unsigned long long key = lp_key(at(i), i);
    if (key >= prefix) sm.list[0][atomicAdd(&sm.count[0], 1)] = key;
  }
  __syncthreads();
}

// What a row's sums and alternatives become.
__device__ __forceinline__ float lp_logprob(float v, float m, float z, float lz) {
  if (z != z) return v * 0.f + z;  // NaN
  return v == -INFINITY ? -INFINITY : v - m - lz;
}

template <bool F32>
__device__ __forceinline__ void lp_finish(const LogprobParams& p, int row, const void* x, const LpSums& a) {
  const float lz = logf(a.z);
  const int t = p.tokens[row];
  float v = -INFINITY;
  const bool in = t >= 0 && t < p.V;
  if (in) v = F32 ? static_cast<const float*>(x)[t] : __bfloat162float(static_cast<const __nv_bfloat16*>(x)[t]);
  p.logprob[row] = in ? lp_logprob(v, a.m, a.z, lz) : -INFINITY;
  p.entropy[row] = a.z == 0.f ? 0.f : lz - a.s / a.z;
}

__device__ __forceinline__ void lp_block_sums(float (&red)[3][kLpWarps], LpSums& a) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
#pragma unroll
  for (int o = 16; o; o >>= 1)
    a.join(__shfl_xor_sync(0xFFFFFFFFu, a.m, o), __shfl_xor_sync(0xFFFFFFFFu, a.z, o), __shfl_xor_sync(0xFFFFFFFFu, a.s, o));
  if (lane == 0) {
    red[0][warp] = a.m;
    red[1][warp] = a.z;
    red[2][warp] = a.s;
  }
  __syncthreads();
  a.m = red[0][0], a.z = red[1][0], a.s = red[2][0];
#pragma unroll
  for (int w = 1; w < kLpWarps; ++w) a.join(red[0][w], red[1][w], red[2][w]);
}

template <bool F32, bool TOP>
__global__ void __launch_bounds__(kLpThreads) logprob_part_kernel(const __grid_constant__ LogprobParams p,
                                                                  const __grid_constant__ LpPlan plan) {
  constexpr int kN = LpPiece<F32>::kN, kEs = F32 ? 4 : 2;
  __shared__ float red[3][kLpWarps];
  __shared__ __align__(16) typename std::conditional<TOP, LpSmem, int>::type smem;
  LpSmem& sm = reinterpret_cast<LpSmem&>(smem);  // (used where TOP)
  const int tid = threadIdx.x, row = blockIdx.y;
  const uint8_t* const x = static_cast<const uint8_t*>(p.x) + static_cast<long long>(row) * p.ld * kEs;
  const int c0 = blockIdx.x * plan.part, c1 = min(p.V, c0 + plan.part);
  pdl_launch_dependents();
  if (TOP && tid == 0) sm.count[0] = 0;
  pdl_wait_prior_grid();
  // [a0, a1): whole 16-byte pieces; what lies before and after them is read one by one, at most 2 kN - 2
  const int mis = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) + static_cast<size_t>(c0) * kEs) % 16) % 16) / kEs;
  const int a0 = min(c1, c0 + mis), pieces = (c1 - a0) / kN, a1 = a0 + pieces * kN;
  const uint4* const body = reinterpret_cast<const uint4*>(x + static_cast<size_t>(a0) * kEs);
  const int edge = tid < a0 - c0 ? c0 + tid : a1 + tid - (a0 - c0);  // this thread's odd logit, if any
  const bool has_edge = edge < c1 && (edge < a0 || edge >= a1);
  float ev = -INFINITY;
  if (has_edge) ev = F32 ? reinterpret_cast<const float*>(x)[edge] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(x)[edge]);
  LpSums sums;
  const uint4 none = F32 ? make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u)
                         : make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u);  // -inf
  // the part as kLpSample runs, read side by side: the first pieces of each are the sample
  const int runs = (pieces + kLpSample * kLpThreads - 1) / (kLpSample * kLpThreads) * kLpThreads;
  uint4 w[kLpSample];
  const auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < kLpSample; ++u) {
      const int i = u * runs + base + tid;
      w[u] = i < pieces ? __ldcs(body + i) : none;
    }
  };
  load(0);
  if (has_edge) {
    if (ev > sums.m) sums.renew(ev);
    const float d = lp_max_nan(ev - sums.m, -1e4f), e = lp_exp2(d * kLog2e);
    sums.z += e;
    sums.s = fmaf(e, d, sums.s);
  }
  unsigned long long threshold = 0;
  float level = 0.f;  // the threshold's value: a piece below it has nothing for the list
  bool any = true;    // the threshold is a NaN, or there is none
  const auto offer = [&](const LpPiece<F32>& q, int i, int stop) {
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const unsigned long long key = lp_key(q.x[e], a0 + i * kN + e);
      if (key >= threshold && i < stop) {
        const int at = atomicAdd(&sm.count[0], 1);
        if (at < kLpList) sm.list[0][at] = key;
      }
    }
  };
  if (TOP) {
    unsigned long long best = has_edge ? lp_key(ev, edge) : 0;
#pragma unroll
    for (int u = 0; u < kLpSample; ++u) {
      const int i = u * runs + tid;
      if (i >= pieces) break;
      const LpPiece<F32> q(w[u]);
      const float t = q.top();
      int at = kN;
#pragma unroll
      for (int e = kN - 1; e >= 0; --e)
        if (q.x[e] == t || (t != t && q.x[e] != q.x[e])) at = e;
      const unsigned long long key = lp_key(t, a0 + i * kN + at);
      best = key > best ? key : best;
    }
    threshold = lp_threshold(sm, best, p.top);
    level = lp_value(threshold);
    any = threshold == 0 || level != level;
    if (has_edge && lp_key(ev, edge) >= threshold) {
      const int at = atomicAdd(&sm.count[0], 1);
      if (at < kLpList) sm.list[0][at] = lp_key(ev, edge);
    }
  }
  for (int base = 0; base < runs; base += kLpThreads) {
    if (base > 0) load(base);
#pragma unroll
    for (int u = 0; u < kLpSample; ++u) {
      const LpPiece<F32> q(w[u]);
      const float t = q.top();
      if (TOP && (any || !(t < level))) offer(q, u * runs + base + tid, pieces);
      q.add(sums, t);
    }
  }
  const bool alone = plan.parts == 1;
  lp_block_sums(red, sums);
  if (tid == 0) {
    if (alone) lp_finish<F32>(p, row, x, sums);
    else *reinterpret_cast<float4*>(plan.sums + (static_cast<size_t>(row) * plan.parts + blockIdx.x) * 4) =
        make_float4(sums.m, sums.z, sums.s, 0.f);
  }
  if (TOP) {
    __syncthreads();
    int cnt = sm.count[0];
    if (cnt > kLpList) {
      lp_search<F32>(sm, x, c0, c1, p.top);
      cnt = sm.count[0];
    }
    const float lz = logf(sums.z);
    unsigned long long* const keys = plan.keys + (static_cast<size_t>(row) * plan.parts + blockIdx.x) * p.top;
    if (!alone && tid < p.top && tid >= cnt) keys[tid] = 0;  // a part of fewer logits than alternatives
    lp_rank(sm, cnt, p.top, [&](int rank, unsigned long long key) {
      if (alone) {
        p.top_id[static_cast<size_t>(row) * p.top + rank] = lp_index(key);
        p.top_lp[static_cast<size_t>(row) * p.top + rank] = lp_logprob(lp_value(key), sums.m, sums.z, lz);
      } else {
        keys[rank] = key;
      }
    });
  }
}

// Joins a row's parts: one CTA per row.
template <bool F32, bool TOP>
__global__ void __launch_bounds__(kLpThreads) logprob_join_kernel(const __grid_constant__ LogprobParams p,
                                                                  const __grid_constant__ LpPlan plan) {
  __shared__ float red[3][kLpWarps];
  __shared__ __align__(16) typename std::conditional<TOP, LpSmem, int>::type smem;
  LpSmem& sm = reinterpret_cast<LpSmem&>(smem);  // (used where TOP)
  const int tid = threadIdx.x, row = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  const int n = TOP ? plan.parts * p.top : 0;
  if (TOP)
    for (int i = tid; i < n; i += kLpThreads) sm.list[0][i] = __ldcg(plan.keys + static_cast<size_t>(row) * n + i);
  LpSums sums;
  if (tid < plan.parts) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(plan.sums) + static_cast<size_t>(row) * plan.parts + tid);
    sums.m = v.x, sums.z = v.y, sums.s = v.z;
  }
  lp_block_sums(red, sums);  // (a barrier: the list is there)
  if (tid == 0)
    lp_finish<F32>(p, row, static_cast<const uint8_t*>(p.x) + static_cast<long long>(row) * p.ld * (F32 ? 4 : 2), sums);
  if (TOP) {
    const float lz = logf(sums.z);
    lp_rank(sm, n, p.top, [&](int rank, unsigned long long key) {
      p.top_id[static_cast<size_t>(row) * p.top + rank] = lp_index(key);
      p.top_lp[static_cast<size_t>(row) * p.top + rank] = lp_logprob(lp_value(key), sums.m, sums.z, lz);
    });
  }
}

// Parts per row: as many as give every SM some CTAs, of at least 4096 logits, and no more than the join's
// list holds (and its threads read).
static void lp_parts(int rows, int V, int top, int n_sm, LpPlan& plan) {
  const int most = std::min({(V + 4095) / 4096, kLpThreads, top > 0 ? kLpList / top : kLpThreads});
  const int want = (4 * std::max(n_sm, 1) + rows - 1) / rows;
  plan.parts = std::max(1, std::min(most, want));
  plan.part = ((V + plan.parts - 1) / plan.parts + 63) / 64 * 64;
  plan.parts = (V + plan.part - 1) / plan.part;
}

static size_t lp_keys_bytes(int rows, int parts, int top) {
  return (static_cast<size_t>(rows) * parts * top * 8 + 15) / 16 * 16;
}

size_t logprob_ws_bytes(int rows, int V, int top, int n_sm) {
  LpPlan plan;
  lp_parts(rows, V, top, n_sm, plan);
  return lp_keys_bytes(rows, plan.parts, top) + static_cast<size_t>(rows) * plan.parts * 16;
}

template <bool F32, bool TOP>
static cudaError_t lp_launch(const LogprobParams& p, const LpPlan& plan, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // rows in grids of at most 65535
  for (int r0 = 0; r0 < p.rows; r0 += 65535) {
    LogprobParams q = p;
    LpPlan pl = plan;
    q.rows = std::min(65535, p.rows - r0);
    q.x = static_cast<const uint8_t*>(p.x) + static_cast<long long>(r0) * p.ld * (F32 ? 4 : 2);
    q.tokens += r0;
    q.logprob += r0;
    q.entropy += r0;
    q.top_lp += static_cast<size_t>(r0) * p.top;
    q.top_id += static_cast<size_t>(r0) * p.top;
    pl.keys += static_cast<size_t>(r0) * plan.parts * p.top;
    pl.sums += static_cast<size_t>(r0) * plan.parts * 4;
    cfg.gridDim = dim3(plan.parts, q.rows);
    cudaError_t e = cudaLaunchKernelEx(&cfg, logprob_part_kernel<F32, TOP>, q, pl);
    if (e == cudaSuccess && plan.parts > 1) {
      cfg.gridDim = dim3(q.rows);
      e = cudaLaunchKernelEx(&cfg, logprob_join_kernel<F32, TOP>, q, pl);
    }
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t logprob_launch(const LogprobParams& p, bool f32, void* ws, int n_sm, cudaStream_t stream) {
  LpPlan plan;
  lp_parts(p.rows, p.V, p.top, n_sm, plan);
  plan.keys = static_cast<unsigned long long*>(ws);
  plan.sums = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + lp_keys_bytes(p.rows, plan.parts, p.top));
  if (p.top > 0) return f32 ? lp_launch<true, true>(p, plan, stream) : lp_launch<false, true>(p, plan, stream);
  return f32 ? lp_launch<true, false>(p, plan, stream) : lp_launch<false, false>(p, plan, stream);
}

}  // namespace skinny
