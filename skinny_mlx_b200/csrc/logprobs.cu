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
// f32 (renewed when a 16-byte piece exceeds it).  With y = x log2(e) - M, M = fl(m log2(e)), e^(x - m) is 2^y
// up to one common factor, the rounding of M, which a thread takes back at its end.  So a logit costs an fma
// in f32, an exponential, an addition and an fma (pairs in one instruction each), half a maximum and half
// a bound (pairs of bf16) and its unpacking.  Bound by the bytes of the logits; the exponential unit (16 per
// clock and SM) would take 0.75 of that time.
//
// The bound: logits below -1e30 count as -1e30, so that 0 times y is 0 for a masked logit.  A part whose
// maximum is beyond 1e6 in size (nothing but masks, most likely) is summed again with x - m: M is off by
// up to 2^-24 of itself, and 2^y by as many powers of two.
//
// Alternatives.  A logit and its index form one 64-bit key whose order is the order wanted; keys are all
// different.  In the pass a thread only keeps its largest logit and where it was (three instructions
// per piece).  After it, the n-th largest of the maxima of 64 groups of threads is a threshold that at
// least n keys reach and hardly more do; only (thread, run) pairs whose maximum reaches it, some n of 1024,
// can hold such keys, and all threads together read those pairs' pieces again (2 % of the row at n = 20,
// mostly from L2), put what reaches the threshold on a list and rank it.  (A list filled in the pass, behind a threshold from a
// sample, cost 24 of 53 us at 509 rows and n = 20: half of a warp's steps had a logit for it.)
// Rows that defeat the threshold (a thread whose logits are all large) overflow the list, and rows with
// a NaN have no maxima to go by: the part is then read again to find the n-th key 12 bits at a time (a
// histogram per pass), which no input makes longer than 6 passes.
//
// Few rows: a row is cut into parts, one CTA each, and a second launch joins their sums and lists.
//
// Times in this file are per call of back-to-back graph replays, where the next launch fills the SMs that a launch's
// last CTAs leave.  A call alone, behind other data in L2, takes 3 to 7 us more: 1024 bf16 rows of 152064 logits 51 us
// (93 % of the copy bandwidth) and 56 (85 %), 600 f32 rows 59 and 64, 509 rows with 20 alternatives 36 and 43.
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
constexpr int kLpRuns = 4;         // 16-byte pieces per thread and step, from as many places of the part
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
__device__ __forceinline__ uint32_t lp_max_nan2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
constexpr float kLpMasked = -1e30f;               // the bound
constexpr uint32_t kLpMasked2 = 0xF14AF14Au;      // a pair of bf16 below it, -1.0003e30
constexpr float kLpFar = 1e6f;                    // maxima beyond it: M is too coarse

// Running maximum (of numbers) and the sums of e = e^(x - m) and e (x - m).
struct LpSums {
  float m = kLpLow, z = 0.f, s = 0.f;
  // to a maximum n >= m: z -> z f, s -> f (s + z (m - n)), f = e^(m - n); unit: how d becomes a power of two
  __device__ __forceinline__ void scale(float d, float unit) {
    const float f = lp_exp2(d * unit);
    s = z == 0.f ? 0.f : f == 0.f && z == z && s == s ? 0.f : f * fmaf(z, d, s);
    z *= f;
  }
  __device__ __forceinline__ void renew(float n) {
    scale(m - n, kLog2e);
    m = n;
  }
  // a logit, whatever it is; d is bounded below so that 0 times an infinite d is 0 (NaN stays NaN)
  __device__ __forceinline__ void add(float x) {
    if (x > m) renew(x);
    const float d = lp_max_nan(x - m, -1e4f), e = lp_exp2(d * kLog2e);
    z += e;
    s = fmaf(e, d, s);
  }
};

// The same in the loop: M = fl(m log2(e)), sums of 2^y and 2^y y, y = x log2(e) - M, of bounded logits, in
// two halves (even and odd logits).
struct LpFast {
  float m = -2.f * kLpFar, M = -2.f * kLpFar * kLog2e;
  uint64_t z = 0, s = 0;  // pairs of f32
  __device__ __forceinline__ void renew(float n) {
    const float N = n * kLog2e;
    LpSums a, b;
    f2_unpack(z, a.z, b.z);
    f2_unpack(s, a.s, b.s);
    a.scale(M - N, 1.f);
    b.scale(M - N, 1.f);
    z = f2_pack(a.z, b.z);
    s = f2_pack(a.s, b.s);
    m = n;
    M = N;
  }
  __device__ __forceinline__ LpSums sums() const {
    float z0, z1, s0, s1;
    f2_unpack(z, z0, z1);
    f2_unpack(s, s0, s1);
    const float r = fmaf(m, kLog2e, -M), f = lp_exp2(-r);  // 2^y = e^(x - m) 2^r
    LpSums b;
    b.m = m;
    b.z = (z0 + z1) * f;
    b.s = f * fmaf(z0 + z1, -r, s0 + s1) * 0.6931471805599453f;
    return b;
  }
};

// The logits of one 16-byte piece: 8 bf16 or 4 f32.
template <bool F32>
struct LpPiece {
  static constexpr int kN = F32 ? 4 : 8;
  uint32_t u[4];
  __device__ __forceinline__ explicit LpPiece(const uint4& w) : u{w.x, w.y, w.z, w.w} {}
  __device__ __forceinline__ static float half(uint32_t w, int hi) {
    return __uint_as_float(hi ? w & 0xFFFF0000u : w << 16);
  }
  __device__ __forceinline__ float at(int i) const { return F32 ? __uint_as_float(u[i & 3]) : half(u[i >> 1 & 3], i & 1); }
  // The same for an index that the compiler does not know.
  __device__ __forceinline__ float pick(int i) const {
    const int k = F32 ? i : i >> 1;
    const uint32_t w = k & 2 ? (k & 1 ? u[3] : u[2]) : (k & 1 ? u[1] : u[0]);
    return F32 ? __uint_as_float(w) : half(w, i & 1);
  }
  // The largest, NaN above every number.
  __device__ __forceinline__ float top() const {
    if (F32)
      return lp_max_nan(lp_max_nan(__uint_as_float(u[0]), __uint_as_float(u[1])),
                        lp_max_nan(__uint_as_float(u[2]), __uint_as_float(u[3])));
    const uint32_t t = lp_max_nan2(lp_max_nan2(u[0], u[1]), lp_max_nan2(u[2], u[3]));
    return lp_max_nan(half(t, 0), half(t, 1));
  }
  __device__ __forceinline__ LpPiece bounded() const {
    LpPiece b = *this;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      b.u[i] = F32 ? __float_as_uint(lp_max_nan(__uint_as_float(u[i]), kLpMasked)) : lp_max_nan2(u[i], kLpMasked2);
    return b;
  }
  // A bounded piece to the sums (whose maximum it does not exceed).
  __device__ __forceinline__ void add(LpFast& f) const {
    const uint64_t nm = f2_pack(-f.M, -f.M), one = f2_pack(1.f, 1.f), l2 = f2_pack(kLog2e, kLog2e);
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
      float y0, y1;
      const uint64_t y = f2_fma(f2_pack(at(i), at(i + 1)), l2, nm);
      f2_unpack(y, y0, y1);
      const uint64_t e = f2_pack(lp_exp2(y0), lp_exp2(y1));
      f.z = f2_fma(e, one, f.z);
      f.s = f2_fma(e, y, f.s);
    }
  }
};

struct LpPlan {
  int parts, part;            // CTAs per row, logits of one part
  int cap;                    // keys of one part: its n largest among them, 0 where there are fewer
  unsigned long long* keys;   // [rows, parts, cap]
  float* sums;                // [rows, parts, 4]: m, z, s
};

struct LpSmem {
  unsigned long long list[2][kLpList];
  unsigned long long group[kLpGroups];
  int count[2];
  int chosen[kLpRuns * kLpThreads];  // (run, thread) pairs whose pieces are read again
  int n_chosen;
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
  if (z != z) return z;
  return v == -INFINITY ? -INFINITY : v - m - lz;
}

// The given token's logit (asked for at a kernel's start: two dependent loads).
template <bool F32>
__device__ __forceinline__ float lp_token(const LogprobParams& p, int row, const void* x, bool& in) {
  const int t = p.tokens[row];
  in = t >= 0 && t < p.V;
  if (!in) return -INFINITY;
  return F32 ? static_cast<const float*>(x)[t] : __bfloat162float(static_cast<const __nv_bfloat16*>(x)[t]);
}

__device__ __forceinline__ void lp_finish(const LogprobParams& p, int row, float v, bool in, const LpSums& a) {
  const float lz = logf(a.z);
  p.logprob[row] = in ? lp_logprob(v, a.m, a.z, lz) : -INFINITY;
  p.entropy[row] = a.z == 0.f ? 0.f : lz - a.s / a.z;
}

// All threads' sums as one, in every thread.
__device__ __forceinline__ void lp_block_sums(float (&red)[3][kLpWarps], LpSums& a) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float m = a.m;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kLpWarps; ++w) m = fmaxf(m, red[0][w]);
  a.renew(m);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a.z += __shfl_xor_sync(0xFFFFFFFFu, a.z, o);
    a.s += __shfl_xor_sync(0xFFFFFFFFu, a.s, o);
  }
  if (lane == 0) {
    red[1][warp] = a.z;
    red[2][warp] = a.s;
  }
  __syncthreads();
  a.z = a.s = 0.f;
#pragma unroll
  for (int w = 0; w < kLpWarps; ++w) {
    a.z += red[1][w];
    a.s += red[2][w];
  }
}

// A part summed with x - m, logit by logit.
template <bool F32>
__device__ __noinline__ LpSums lp_careful(const void* row, int c0, int c1) {
  LpSums a;
  for (int i = c0 + threadIdx.x; i < c1; i += kLpThreads)
    a.add(F32 ? static_cast<const float*>(row)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]));
  return a;
}

template <bool F32, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4) logprob_part_kernel(const __grid_constant__ LogprobParams p,
                                                                  const __grid_constant__ LpPlan plan) {
  constexpr int kN = LpPiece<F32>::kN, kEs = F32 ? 4 : 2;
  __shared__ float red[3][kLpWarps];
  __shared__ __align__(16) typename std::conditional<TOP, LpSmem, int>::type smem;
  LpSmem& sm = reinterpret_cast<LpSmem&>(smem);  // (used where TOP)
  const int tid = threadIdx.x, row = blockIdx.y;
  const uint8_t* const x = static_cast<const uint8_t*>(p.x) + static_cast<long long>(row) * p.ld * kEs;
  const int c0 = blockIdx.x * plan.part, c1 = min(p.V, c0 + plan.part);
  pdl_launch_dependents();
  if (TOP && tid == 0) sm.count[0] = sm.n_chosen = 0;
  pdl_wait_prior_grid();
  const bool alone = plan.parts == 1;
  bool in = false;
  float tv = 0.f;
  if (alone && tid == 0) tv = lp_token<F32>(p, row, x, in);
  // [a0, a1): whole 16-byte pieces; what lies before and after them is read one by one, at most 2 kN - 2
  const int mis = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) + static_cast<size_t>(c0) * kEs) % 16) % 16) / kEs;
  const int a0 = min(c1, c0 + mis), pieces = (c1 - a0) / kN, a1 = a0 + pieces * kN;
  const uint4* const body = reinterpret_cast<const uint4*>(x + static_cast<size_t>(a0) * kEs);
  const int edge = tid < a0 - c0 ? c0 + tid : a1 + tid - (a0 - c0);  // this thread's odd logit, if any
  const bool has_edge = edge < c1 && (edge < a0 || edge >= a1);
  float ev = -INFINITY;
  if (has_edge) ev = F32 ? reinterpret_cast<const float*>(x)[edge] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(x)[edge]);
  LpFast fast;
  const uint4 none = F32 ? make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u)
                         : make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u);  // -inf
  // the part as kLpRuns runs, read side by side
  const int runs = (pieces + kLpRuns * kLpThreads - 1) / (kLpRuns * kLpThreads) * kLpThreads;
  uint4 w[kLpRuns];
  const auto load = [&](uint4 (&v)[kLpRuns], int base) {
#pragma unroll
    for (int u = 0; u < kLpRuns; ++u) {
      const int i = u * runs + base + tid;
      v[u] = i < pieces && base < runs ? __ldcs(body + i) : none;
    }
  };
  load(w, 0);
  float best = kLpMasked;  // this thread's largest logit above the bound, and its piece
  int best_at = tid;
  float run_best[kLpRuns];  // the same of its pieces of each run
#pragma unroll
  for (int u = 0; u < kLpRuns; ++u) run_best[u] = kLpMasked;
  const auto step = [&](const uint4 (&v)[kLpRuns], int base) {
    LpPiece<F32> b[kLpRuns] = {LpPiece<F32>(v[0]).bounded(), LpPiece<F32>(v[1]).bounded(), LpPiece<F32>(v[2]).bounded(),
                               LpPiece<F32>(v[3]).bounded()};
    float t[kLpRuns], most = kLpMasked;
#pragma unroll
    for (int u = 0; u < kLpRuns; ++u) {
      t[u] = b[u].top();
      most = fmaxf(most, t[u]);
      if (TOP && t[u] > best) {
        best = t[u];
        best_at = u * runs + base + tid;
      }
      if (TOP) run_best[u] = fmaxf(run_best[u], t[u]);
    }
    if (most > fast.m) fast.renew(most);
#pragma unroll
    for (int u = 0; u < kLpRuns; ++u) b[u].add(fast);
  };
  // The next step's pieces are in flight while one's are added, two steps per turn so that the buffers change roles
  // instead of being copied; then the steps that not every run fills.
  static_assert(kLpRuns == 4, "step()");
  uint4 next[kLpRuns];
  const auto load_full = [&](uint4 (&v)[kLpRuns], int base) {
#pragma unroll
    for (int u = 0; u < kLpRuns; ++u) v[u] = __ldcs(body + u * runs + base + tid);
  };
  const int full = pieces - (kLpRuns - 1) * runs;  // pieces of the last run, the shortest
  int base = 0;
  for (; base + 3 * kLpThreads <= full; base += 2 * kLpThreads) {
    load_full(next, base + kLpThreads);
    step(w, base);
    load_full(w, base + 2 * kLpThreads);
    step(next, base + kLpThreads);
  }
  for (; base < runs; base += kLpThreads) {
    load(next, base + kLpThreads);
    step(w, base);
#pragma unroll
    for (int u = 0; u < kLpRuns; ++u) w[u] = next[u];
  }
  LpSums sums = fast.sums();
  if (has_edge) sums.add(lp_max_nan(ev, kLpMasked));
  lp_block_sums(red, sums);
  if (!(sums.m > -kLpFar && sums.m < kLpFar)) {  // nothing but masks, or logits far from 0
    sums = lp_careful<F32>(x, c0, c1);
    __syncthreads();
    lp_block_sums(red, sums);
  }
  if (tid == 0) {
    if (alone) lp_finish(p, row, tv, in, sums);
    else *reinterpret_cast<float4*>(plan.sums + (static_cast<size_t>(row) * plan.parts + blockIdx.x) * 4) =
        make_float4(sums.m, sums.z, sums.s, 0.f);
  }
  if (TOP) {
    // The threshold, from a key each thread's logits reach: its largest logit at the end of its piece (a
    // thread of masked logits: -inf).
    const bool some = best_at < pieces, above = best > kLpMasked;
    unsigned long long low = some ? lp_key(above ? best : -INFINITY, a0 + best_at * kN + kN - 1) : 0;
    const unsigned long long edge_key = has_edge ? lp_key(ev, edge) : 0;
    low = edge_key > low ? edge_key : low;
    const unsigned long long threshold = lp_threshold(sm, low, p.top);
    const float level = threshold == 0 ? -INFINITY : lp_value(threshold);
    // what can hold keys reaching it: a thread's pieces of a run; all where masked logits reach it
#pragma unroll
    for (int u = 0; u < kLpRuns; ++u)
      if (u * runs + tid < pieces &&
          (level <= kLpMasked || (run_best[u] > kLpMasked && lp_key(run_best[u], a0 + (u * runs + tid) * kN) >= threshold)))
        sm.chosen[atomicAdd(&sm.n_chosen, 1)] = u * runs + tid;
    if (edge_key != 0 && edge_key >= threshold) sm.list[0][atomicAdd(&sm.count[0], 1)] = edge_key;
    __syncthreads();
    const bool search = sums.z != sums.z;  // a NaN
    const int steps = runs / kLpThreads, again = search ? 0 : sm.n_chosen * steps;
    for (int q0 = 0; q0 < again; q0 += kLpRuns * kLpThreads) {
      int at[kLpRuns];
#pragma unroll
      for (int u = 0; u < kLpRuns; ++u) {
        const int q = q0 + u * kLpThreads + tid, who = q / steps, step = q - who * steps;
        at[u] = q < again ? sm.chosen[who] + step * kLpThreads : pieces;
        w[u] = at[u] < pieces ? __ldg(body + at[u]) : none;
      }
#pragma unroll
      for (int u = 0; u < kLpRuns; ++u) {
        const LpPiece<F32> q(w[u]);
        if (at[u] >= pieces || q.top() < level) continue;
        uint32_t hits = 0;
#pragma unroll
        for (int e = 0; e < kN; ++e) hits |= static_cast<uint32_t>(!(q.at(e) < level)) << e;
        for (; hits; hits &= hits - 1) {
          const int e = __ffs(hits) - 1;
          const unsigned long long key = lp_key(q.pick(e), a0 + at[u] * kN + e);
          if (key >= threshold) {
            const int slot = atomicAdd(&sm.count[0], 1);
            if (slot < kLpList) sm.list[0][slot] = key;
          }
        }
      }
    }
    __syncthreads();
    int cnt = sm.count[0];
    if (search || cnt > kLpList) {
      lp_search<F32>(sm, x, c0, c1, p.top);
      cnt = sm.count[0];
    }
    if (!alone) {
      // the keys as they are where they are few; the join ranks them
      unsigned long long* const keys = plan.keys + (static_cast<size_t>(row) * plan.parts + blockIdx.x) * plan.cap;
      if (cnt <= plan.cap) {
        if (tid < plan.cap) keys[tid] = tid < cnt ? sm.list[0][tid] : 0;
      } else {
        if (tid >= p.top && tid < plan.cap) keys[tid] = 0;
        lp_rank(sm, cnt, p.top, [&](int rank, unsigned long long key) { keys[rank] = key; });
      }
      return;
    }
    const float lz = logf(sums.z);
    lp_rank(sm, cnt, p.top, [&](int rank, unsigned long long key) {
      p.top_id[static_cast<size_t>(row) * p.top + rank] = lp_index(key);
      p.top_lp[static_cast<size_t>(row) * p.top + rank] = lp_logprob(lp_value(key), sums.m, sums.z, lz);
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
  if (TOP && tid == 0) sm.count[0] = 0;
  if (TOP) __syncthreads();
  pdl_wait_prior_grid();
  bool in = false;
  float tv = 0.f;
  if (tid == 0)
    tv = lp_token<F32>(p, row, static_cast<const uint8_t*>(p.x) + static_cast<long long>(row) * p.ld * (F32 ? 4 : 2), in);
  LpSums sums;
  if (tid < plan.parts) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(plan.sums) + static_cast<size_t>(row) * plan.parts + tid);
    sums.m = v.x, sums.z = v.y, sums.s = v.z;
  }
  if (TOP) {
    const int n = plan.parts * plan.cap;
    const unsigned long long* const from = plan.keys + static_cast<size_t>(row) * n;
    for (int i = tid; i < n; i += kLpThreads) {
      const unsigned long long key = __ldcg(from + i);
      if (key != 0) sm.list[0][atomicAdd(&sm.count[0], 1)] = key;
    }
  }
  lp_block_sums(red, sums);  // (a barrier: the list is there)
  if (tid == 0) lp_finish(p, row, tv, in, sums);
  if (TOP) {
    const float lz = logf(sums.z);
    lp_rank(sm, sm.count[0], p.top, [&](int rank, unsigned long long key) {
      p.top_id[static_cast<size_t>(row) * p.top + rank] = lp_index(key);
      p.top_lp[static_cast<size_t>(row) * p.top + rank] = lp_logprob(lp_value(key), sums.m, sums.z, lz);
    });
  }
}

// Parts per row.  Fewer than three rows per SM are cut so that every SM has four CTAs (300 bf16 rows of 152064
// logits: one part 28.8 us, two 24.3, four 22.5), into parts of at least 4096 logits, no more than the join's list
// holds and its threads read.  From there on a row is one CTA (509 rows with 20 alternatives: one part 36 us, two 42,
// four 48: what a part and the join cost besides the logits), except that without alternatives, where the join is
// cheap, rows up to six per SM are cut into up to four parts of at least 32768 logits: whole rows, four to an SM, leave
// most SMs idle at the end (600 f32 rows of 152064: one part 68 us, four 59; 760 bf16 rows 44 and 45; at 1024 rows 51
// and 57, and 600 rows of 32000 logits 12 and 15).
static void lp_parts(int rows, int V, int top, int n_sm, LpPlan& plan) {
  plan.cap = top > 0 ? top + 32 : 0;
  const int sms = std::max(n_sm, 1);
  const int most = std::min({V / 4096 + (V % 4096 > 0), kLpThreads, top > 0 ? kLpList / plan.cap : kLpThreads});
  const int fill = rows >= 3 * sms ? 1 : (4 * sms + rows - 1) / rows;
  const int even = top == 0 && rows < 6 * sms ? std::min(4, V / 32768) : 1;
  const int want = std::max(fill, even);
  plan.parts = std::max(1, std::min(most, want));
  plan.part = ((V - 1) / plan.parts / 64 + 1) * 64;
  plan.parts = (V - 1) / plan.part + 1;
}

static size_t lp_keys_bytes(int rows, const LpPlan& plan) {
  return (static_cast<size_t>(rows) * plan.parts * plan.cap * 8 + 15) / 16 * 16;
}

size_t logprob_ws_bytes(int rows, int V, int top, int n_sm) {
  LpPlan plan;
  lp_parts(rows, V, top, n_sm, plan);
  return plan.parts == 1 ? 16 : lp_keys_bytes(rows, plan) + static_cast<size_t>(rows) * plan.parts * 16;
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
    pl.keys += static_cast<size_t>(r0) * plan.parts * plan.cap;
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
  plan.sums = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + lp_keys_bytes(p.rows, plan));
  if (p.top > 0) return f32 ? lp_launch<true, true>(p, plan, stream) : lp_launch<false, true>(p, plan, stream);
  return f32 ? lp_launch<true, false>(p, plan, stream) : lp_launch<false, false>(p, plan, stream);
}

}  // namespace skinny
