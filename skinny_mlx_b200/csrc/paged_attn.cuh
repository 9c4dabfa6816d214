// What the kernels of paged attention share: the line of all sequences' key tiles and a CTA's walk along its
// piece of it, the plan of a launch, tensor maps of a pool.
#pragma once
#include <algorithm>
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "paged.cuh"
#include "ptx.cuh"

namespace skinny {

constexpr float kPtMost = 256.f;          // how far p may exceed 1 before the maximum is renewed
constexpr float kPtNothing = -3.402823466e38f;  // the maximum of a row that has seen no key

struct PagedAttnPlan {
  int tile_log;    // keys of one tile, one block per warp (a power of two)
  int lead;        // what beginning an item costs, in tiles: counted on the line, so that the pieces balance
  int shift;       // log2 of the page size, or -1
  int box;         // positions of one copy: the largest power of two, up to a block, that divides the page size
  int nchunk;      // row chunks of 8 NB rows, one per warp (1, 2 or 4); the other warps split keys
  int groups;      // row groups of nchunk chunks per kv head
  int join_warps;  // warps per row of the join (a power of two up to 8)
  int rows;        // rows of one group: 8 NB nchunk
  int ctas;        // CTAs of the split launch
  long long* pre;  // [B + 1] where each sequence begins on the line
  float* ml;       // [2 ctas][rows][2] maximum (log2) and sum of a piece
  float* o;        // [2 ctas][rows][D]
  uint32_t rep_inv; // ceil(2^32 / rep), 0 for rep = 1: r / rep of rows r < 2^16

  __device__ __forceinline__ int token(int r) const { return rep_inv ? __umulhi(static_cast<uint32_t>(r), rep_inv) : r; }
};

// The positions some token of the sequence sees, and the tiles they make.
struct PagedSpan {
  int len, cnt, beg, end;
  int first, tiles;  // the tiles start at a multiple of 32: no box straddles two blocks
  int units;         // tiles and lead of one item on the line
};

__device__ __forceinline__ PagedSpan paged_span(const PagedAttnParams& p, const PagedAttnPlan& plan, int b,
                                                bool* ok = nullptr) {
  PagedSpan s;
  const bool good = p.seq.get(b, s.len, s.cnt);
  if (ok) *ok = good;
  s.end = s.len + s.cnt;
  s.beg = p.window > 0 && s.len >= p.window ? s.len - p.window + 1 : 0;
  s.first = s.beg & ~31;
  s.tiles = s.cnt > 0 ? ((s.end - s.first - 1) >> plan.tile_log) + 1 : 0;
  s.units = s.tiles ? s.tiles + plan.lead : 0;
  return s;
}

__device__ __forceinline__ float pt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// a / b of non-negative numbers, in 32 bits where they fit.
__device__ __forceinline__ long long pt_div(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// The line's pieces: `total` units over the CTAs, the first `rest` pieces one unit longer.
struct PtLine {
  long long total, each, rest;
  __device__ __forceinline__ PtLine(long long n, int ctas) : total(n), each(0), rest(0) {
    const long long parts = min(n, static_cast<long long>(ctas));
    if (parts > 0) {
      each = pt_div(n, parts);
      rest = n - each * parts;
    }
  }
  __device__ __forceinline__ long long start(int i) const { return i * each + min(static_cast<long long>(i), rest); }
  __device__ __forceinline__ int owner(long long u) const {
    const long long longer = rest * (each + 1);
    return static_cast<int>(u < longer ? pt_div(u, each + 1) : rest + pt_div(u - longer, each));
  }
};

__device__ __forceinline__ uint32_t pt_pack(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A CTA's place on its piece of the line: [u, u_end), `off` units into sequence b.
struct PtPart {
  PagedSpan sp;
  int seq, item, t0, t1;  // a sequence's item (kv head, row group) and its tiles [t0, t1)
};
struct PtWalk {
  int b;
  long long u, u_end, off;
  // The next part of the piece; false behind the last.
  __device__ __forceinline__ bool next(const PagedAttnParams& p, const PagedAttnPlan& plan, int items, PtPart& part) {
    while (u < u_end) {
      part.sp = paged_span(p, plan, b);
      if (part.sp.tiles == 0) {
        ++b;
        continue;
      }
      part.item = static_cast<int>(pt_div(off, part.sp.units));
      const int at = static_cast<int>(off - static_cast<long long>(part.item) * part.sp.units);
      const int take = static_cast<int>(min(static_cast<long long>(part.sp.units - at), u_end - u));
      part.t0 = max(at - plan.lead, 0);
      part.t1 = max(at + take - plan.lead, 0);
      part.seq = b;
      u += take;
      off += take;
      if (off == static_cast<long long>(part.sp.units) * items) {
        ++b;
        off = 0;
      }
      if (part.t1 > part.t0) return true;  // (else only an item's lead)
    }
    return false;
  }
};

// Finds this CTA's piece (all its threads call it); CTA 0 writes the join's copy of the line and reports
// sequences out of range.  False: the line is shorter than the grid and this CTA has nothing.
template <int kThreads>
__device__ __forceinline__ bool pt_begin(const PagedAttnParams& p, const PagedAttnPlan& plan, int items, long long* scan,
                                         long long* found, PtWalk& walk) {
  constexpr int kWarps = kThreads / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, B = p.seq.B;
  if (B <= 32) {  // one sequence per lane, every warp by itself
    bool ok = true;
    const long long mine =
        lane < B ? static_cast<long long>(paged_span(p, plan, lane, &ok).units) * items : 0;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += x;
    }
    const long long total = __shfl_sync(0xFFFFFFFFu, incl, 31);
    if (blockIdx.x == 0 && warp == 0) {
      if (lane < B) plan.pre[lane] = incl - mine;  // the join's copy of the line
      if (lane == 0) plan.pre[B] = total;
      if (!ok) atomicOr(p.seq.err, kErrBitBadInput);
    }
    if (blockIdx.x >= total) return false;
    const PtLine line(total, plan.ctas);
    walk.u = line.start(blockIdx.x);
    walk.u_end = line.start(blockIdx.x + 1);
    walk.b = __ffs(__ballot_sync(0xFFFFFFFFu, walk.u < incl)) - 1;
    walk.off = walk.u - __shfl_sync(0xFFFFFFFFu, incl - mine, walk.b);
    return true;
  }
  // thread i sums its run of sequences
  const int run = (B + kThreads - 1) / kThreads, b_lo = min(B, tid * run), b_hi = min(B, b_lo + run);
  long long mine = 0;
  bool all_ok = true;
  for (int i = b_lo; i < b_hi; ++i) {
    bool ok;
    mine += static_cast<long long>(paged_span(p, plan, i, &ok).units) * items;
    all_ok &= ok;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  long long total = 0, excl = incl - mine;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) excl += scan[w];
    total += scan[w];
  }
  if (blockIdx.x == 0) {
    long long at = excl;
    for (int i = b_lo; i < b_hi; ++i) {
      plan.pre[i] = at;
      at += static_cast<long long>(paged_span(p, plan, i).units) * items;
    }
    if (tid == 0) plan.pre[B] = total;
    if (!all_ok) atomicOr(p.seq.err, kErrBitBadInput);
  }
  if (blockIdx.x >= total) return false;
  const PtLine line(total, plan.ctas);
  walk.u = line.start(blockIdx.x);
  walk.u_end = line.start(blockIdx.x + 1);
  if (excl <= walk.u && walk.u < excl + mine) {
    long long at = excl;
    for (int i = b_lo; i < b_hi; ++i) {
      const long long n = static_cast<long long>(paged_span(p, plan, i).units) * items;
      if (walk.u < at + n) {
        found[0] = i;
        found[1] = walk.u - at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  walk.b = static_cast<int>(found[0]);
  walk.off = found[1];
  return true;
}

// A pool's rows of D elements: pages of a pool that interleaves others are further apart, the rows between are
// never asked for.
inline unsigned long long pt_rows(long long page_stride, const PagedAttnParams& p) {
  return static_cast<unsigned long long>(p.seq.n_pages - 1) * (page_stride / p.D) +
         static_cast<unsigned long long>(p.Hkv) * p.seq.page;
}
cudaError_t pt_encode(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
                      const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle);

// A tensor map of a pool, and the split launch of the tensor-memory kernel (paged_attn_tc.cu).
cudaError_t pt_map(CUtensorMap* map, const void* pool, long long page_stride, const PagedAttnParams& p, int es, int line,
                   int box, int lines);
cudaError_t paged_attn_tc_split(const PagedAttnParams& p, const PagedAttnPlan& plan, int dev, const cudaLaunchConfig_t& cfg);

}  // namespace skinny
