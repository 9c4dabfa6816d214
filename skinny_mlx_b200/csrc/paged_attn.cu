// Attention of 1..16 new tokens per sequence over a paged key-value cache:
//
//   o[b, t, h] = sum_j softmax_j(scale * q[b, t, h] . k_j) v_j     (query head h reads kv head h / rep)
//
// over the positions j <= lengths[b] + t of sequence b's pages (and j > lengths[b] + t - window).
// A row that sees nothing (an idle slot, t >= counts[b], every page bad) is zero, its lse -inf.
//
// One pass over the cache with a running maximum and sum, split over the cache's length and joined
// (online softmax).  Bound by the bytes of the keys and values: each is read once from memory, by
// one warp, straight into the registers that feed the matrix instructions.  Three choices make
// that possible without shared memory or barriers in the loop:
//
// * The keys are the 16-row operand and the query rows (t, head in the group; at most 8 NB of them)
//   the 8-column operand: S^T[key][row] = K q^T, then O^T[dim][row] += V^T P^T.  A decode step has
//   few rows, so 8-column tiles waste the least of the matrix unit, and O needs D / 16 * 4 registers
//   per 8 rows.
// * A dot product does not care in which order its dims come, so a thread's 16 consecutive bytes
//   of a key row serve as its operand pieces of two (e4m3: four) consecutive 16-dim steps, and the
//   query's fragments are loaded in the same order.  Likewise the 8 (16) consecutive dims a thread
//   reads of a value row are its rows of 4 (8) output tiles; pairs of keys are interleaved with
//   byte permutes.  Every load is 16 bytes and whole 32-byte sectors are used.
// * P^T as an operand is the transpose of the S^T accumulators, one movmatrix per 8 x 8 block.
//
// The maximum a row's exponentials refer to is renewed only when a score exceeds it by more than
// 8 (in powers of two): p stays below 256, which bf16 and f16 hold at the same relative precision,
// and the usual block needs one warp vote instead of shuffles and a rescaling of O.
// Roundings: scores, maxima, sums and O are f32; p is rounded to bf16 (bf16 pages, 2^-9 of p on
// average below the output's own rounding) or f16 (e4m3 pages: keys and values are exact in f16,
// and q is scaled per row by a power of two so that it is exact too).  The sum adds the p before
// that rounding, so the lse does not see it.
//
// Work split: the tiles of 64 keys of all (sequence, kv head, row group) items form one line that
// is cut into equal pieces, one per CTA (`kCtas` CTAs per SM), so that ragged lengths balance; the
// lengths are read on the device and the launch does not depend on them (a captured graph serves
// any).  A CTA whose piece covers an item writes its output; the others write (max, sum, O) to the
// workspace and the join launch adds them in order, so results do not depend on timing.
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "paged.cuh"
#include "ptx.cuh"

namespace skinny {

constexpr int kPtThreads = 128;
constexpr int kPtWarps = kPtThreads / 32;
constexpr int kPtTile = 64;               // keys of one unit of work: 16 per warp
constexpr uint32_t kPtNone = 0xFFFFFFFFu;  // no such key (past the end, or a page outside the pool)
constexpr float kPtSlack = 8.f;           // how far p may exceed 1, in powers of two

struct PagedAttnPlan {
  int nchunk;      // row chunks of 8 NB rows, one per warp (1, 2 or 4); the other warps split keys
  int groups;      // row groups of nchunk chunks per kv head
  int rows;        // rows of one group: 8 NB nchunk
  int ctas;        // CTAs of the split launch
  long long* pre;  // [B + 1] first tile of each sequence on the line
  float* ml;       // [2 ctas][rows][2] maximum (log2) and sum of a piece
  float* o;        // [2 ctas][rows][D]
};

// The positions some token of the sequence sees, and the tiles they make.
struct PagedSpan {
  int len, cnt, beg, end, tiles;
};

__device__ __forceinline__ PagedSpan paged_span(const PagedAttnParams& p, int b, bool* ok = nullptr) {
  PagedSpan s;
  const bool good = p.seq.get(b, s.len, s.cnt);
  if (ok) *ok = good;
  s.end = s.len + s.cnt;
  s.beg = p.window > 0 && s.len >= p.window ? s.len - p.window + 1 : 0;
  s.tiles = s.cnt > 0 ? (s.end - s.beg + kPtTile - 1) / kPtTile : 0;
  return s;
}

__device__ __forceinline__ float pt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pt_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <bool F16>
__device__ __forceinline__ void pt_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// WORDS 32-bit words at p, or zeros.  Volatile: the loads are issued where they stand.  (The pages
// are not written while the kernel runs: non-coherent loads.)
template <int WORDS>
__device__ __forceinline__ void pt_load(uint32_t* r, const uint8_t* p, bool pred) {
  if (WORDS == 4)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\t"
        "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
        "@q ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3])
        : "l"(p), "r"(static_cast<uint32_t>(pred)));
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %3, 0;\n\t"
        "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\t"
        "@q ld.global.nc.v2.u32 {%0, %1}, [%2];\n\t}"
        : "=&r"(r[0]), "=&r"(r[1])
        : "l"(p), "r"(static_cast<uint32_t>(pred)));
}

__device__ __forceinline__ uint32_t pt_cvt_e4m3x2(uint32_t pair) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair & 0xFFFFu), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | static_cast<uint32_t>(h.y) << 16;
}

template <bool F16>
__device__ __forceinline__ uint32_t pt_pack(float lo, float hi) {
  if (F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Sizes of one instance.  kCtas: CTAs per SM that the registers allow.
template <int D, int NB, bool F8>
struct PtShape {
  static constexpr int kQWords = D / 8;                   // query fragment words per thread and 8 rows
  static constexpr int kKWords = F8 ? D / 16 : D / 8;     // key words per thread and key (2 keys)
  static constexpr int kPiece = F8 && D == 64 ? 2 : 4;    // words of one value load
  static constexpr int kPieces = F8 ? (D + 127) / 128 : D / 64;  // value loads per thread and key (4 keys)
  static constexpr int kElems = F8 ? 4 * kPiece : 8;      // consecutive dims of one value load
  static constexpr int kTiles = D / 16;                   // output tiles of 16 dims
  static constexpr bool kQRegs = NB * D <= (F8 || D < 256 ? 256 : 0);  // query fragments stay in registers
  static constexpr int kCtas = NB * D <= 128 ? 3 : 2;
};

template <int D, int NB, bool F8>
__host__ __device__ constexpr int pt_o_floats() { return kPtWarps * 8 * NB * (D + 4); }

template <int D, int NB, bool F8>
__host__ __device__ constexpr int pt_smem_bytes() {
  using S = PtShape<D, NB, F8>;
  return pt_o_floats<D, NB, F8>() * 4 + (S::kQRegs ? 0 : kPtWarps * NB * S::kQWords * 32 * 4);
}

template <int D, int NB, bool F8>
__global__ void __launch_bounds__(kPtThreads, PtShape<D, NB, F8>::kCtas)
    paged_attn_split_kernel(const __grid_constant__ PagedAttnParams p, const __grid_constant__ PagedAttnPlan plan) {
  using S = PtShape<D, NB, F8>;
  constexpr int kEs = F8 ? 1 : 2;
  extern __shared__ __align__(16) uint8_t pt_smem[];
  float* const so = reinterpret_cast<float*>(pt_smem);                      // [warp][8 NB][D + 4]
  uint32_t* const sq = reinterpret_cast<uint32_t*>(so + pt_o_floats<D, NB, F8>());  // [warp][NB][kQWords / 4][lane][4]
  __shared__ float sml[kPtWarps][8 * NB][2];
  __shared__ long long scan[kPtWarps];
  __shared__ long long found[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cq = lane & 3;
  const int rep = p.Hq / p.Hkv, items = p.Hkv * plan.groups, B = p.seq.B;
  pdl_launch_dependents();
  pdl_wait_prior_grid();

  // ---- this CTA's piece of the line: thread i sums the tiles of its run of sequences
  const int run = (B + kPtThreads - 1) / kPtThreads, b_lo = min(B, tid * run), b_hi = min(B, b_lo + run);
  long long mine = 0;
  bool all_ok = true;
  for (int b = b_lo; b < b_hi; ++b) {
    bool ok;
    mine += static_cast<long long>(paged_span(p, b, &ok).tiles) * items;
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
  for (int w = 0; w < kPtWarps; ++w) {
    if (w < warp) excl += scan[w];
    total += scan[w];
  }
  const long long parts = min(static_cast<long long>(plan.ctas), total);
  if (blockIdx.x == 0) {  // the join's copy of the line
    long long at = excl;
    for (int b = b_lo; b < b_hi; ++b) {
      plan.pre[b] = at;
      at += static_cast<long long>(paged_span(p, b).tiles) * items;
    }
    if (tid == 0) plan.pre[B] = total;
    if (!all_ok) atomicOr(p.seq.err, kErrBitBadInput);
  }
  if (blockIdx.x >= parts) return;
  long long u = blockIdx.x * total / parts;
  const long long u_end = (blockIdx.x + 1ll) * total / parts;
  if (excl <= u && u < excl + mine) {
    long long at = excl;
    for (int b = b_lo; b < b_hi; ++b) {
      const long long n = static_cast<long long>(paged_span(p, b).tiles) * items;
      if (u < at + n) {
        found[0] = b;
        found[1] = u - at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  int b = static_cast<int>(found[0]);
  long long off = found[1];
  const int chunk = warp % plan.nchunk, slot = warp / plan.nchunk, slots = kPtWarps / plan.nchunk;
  const uint32_t kpr = static_cast<uint32_t>(p.kps / D), vpr = static_cast<uint32_t>(p.vps / D);
  uint32_t* const myq = sq + static_cast<size_t>(warp) * NB * S::kQWords * 32 + lane * 4;
  bool bad = false;

  for (int seg = 0; u < u_end; ++seg) {
    const PagedSpan sp = paged_span(p, b);
    if (sp.tiles == 0) {
      ++b;
      --seg;
      continue;
    }
    const int item = static_cast<int>(off / sp.tiles), t0 = static_cast<int>(off - static_cast<long long>(item) * sp.tiles);
    const int t1 = static_cast<int>(min(static_cast<long long>(sp.tiles), t0 + (u_end - u)));
    const int kvh = item / plan.groups, rbase = (item % plan.groups) * plan.rows;
    const int k0 = sp.beg + t0 * kPtTile, k1 = min(sp.end, sp.beg + t1 * kPtTile);
    const int r0 = rbase + chunk * 8 * NB;  // this warp's first row
    const int32_t* const table = p.seq.table + b * p.seq.table_stride;

    // ---- query fragments; sc: the factor that takes a score to powers of two
    uint32_t qr[S::kQRegs ? NB : 1][S::kQRegs ? S::kQWords : 1];
    float sc[F8 ? NB : 1][2];
    const float sc0 = p.scale * 1.4426950408889634f * (F8 ? p.k_scale[kvh] : 1.f);
    if (!F8) sc[0][0] = sc0;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = r0 + 8 * nb + g, t = r / rep, h = kvh * rep + r % rep;
      const bool live = t < sp.cnt;
      const uint8_t* const src =
          reinterpret_cast<const uint8_t*>(p.q + b * p.qs[0] + t * p.qs[1] + h * p.qs[2]) + cq * (F8 ? 32 : 16);
      uint32_t w[S::kQWords];
#pragma unroll
      for (int i = 0; i < S::kQWords / 4; ++i)
        pt_load<4>(w + 4 * i, src + (F8 ? (i >> 1) * 128 + (i & 1) * 16 : i * 64), live);
      if (F8) {  // to f16, the row's largest |q| to [1, 2)
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < S::kQWords; ++i) top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        const uint32_t ex = min(max(top >> 7, 1u), 253u);
        const float up = top >= 0x7F80u ? 1.f : __uint_as_float((254u - ex) << 23);
        const float down = top >= 0x7F80u ? 1.f : __uint_as_float(ex << 23);
#pragma unroll
        for (int i = 0; i < S::kQWords; ++i)
          w[i] = pt_pack<true>(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xFFFF0000u) * up);
        sc[nb][0] = sc0 * __shfl_sync(0xFFFFFFFFu, down, 8 * cq);  // rows 2 cq and 2 cq + 1: lanes g = row
        sc[nb][1] = sc0 * __shfl_sync(0xFFFFFFFFu, down, 8 * cq + 4);
      }
#pragma unroll
      for (int i = 0; i < S::kQWords; ++i) {
        if (S::kQRegs) qr[nb][i] = w[i];
        else myq[(nb * S::kQWords / 4 + i / 4) * 128 + i % 4] = w[i];
      }
    }

    // ---- one pass over the keys of the segment: 16-key blocks slot, slot + slots, ...
    float o[NB][S::kTiles][4], m[NB][2], l[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb][0] = m[nb][1] = -INFINITY;
      l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
      for (int i = 0; i < S::kTiles; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nb][i][e] = 0.f;
    }
    const int nblk = (k1 - k0 + 15) >> 4;
    uint32_t kw[2][S::kKWords], vw[4][S::kPieces * S::kPiece];
    // a block's page ids, one per lane (lanes 16..31 repeat), and from them its rows in the pools
    const auto page_id = [&](int i) {
      const int j = k0 + 16 * i + (lane & 15);
      return i < nblk && j < k1 ? __ldg(table + j / p.seq.page) : -1;
    };
    const auto row_of = [&](int i, int pid, uint32_t& rk, uint32_t& rv) {
      const int j = k0 + 16 * i + (lane & 15);
      const bool in = i < nblk && j < k1, ok = in && pid >= 0 && pid < p.seq.n_pages;
      bad |= in && !ok;
      const uint32_t in_page = static_cast<uint32_t>(kvh) * p.seq.page + static_cast<uint32_t>(j % p.seq.page);
      rk = ok ? static_cast<uint32_t>(pid) * kpr + in_page : kPtNone;
      rv = ok ? static_cast<uint32_t>(pid) * vpr + in_page : kPtNone;
    };
    const auto load_k = [&](uint32_t rk) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t r = __shfl_sync(0xFFFFFFFFu, rk, g + 8 * e);
        const uint8_t* const src = static_cast<const uint8_t*>(p.kp) + static_cast<size_t>(r) * (D * kEs) + cq * 16;
#pragma unroll
        for (int i = 0; i < S::kKWords / 4; ++i) pt_load<4>(kw[e] + 4 * i, src + i * 64, r != kPtNone);
      }
    };
    const auto load_v = [&](uint32_t rv) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t r = __shfl_sync(0xFFFFFFFFu, rv, 2 * cq + (e & 1) + 8 * (e >> 1));
        const uint8_t* const src =
            static_cast<const uint8_t*>(p.vp) + static_cast<size_t>(r) * (D * kEs) + g * (S::kElems * kEs);
#pragma unroll
        for (int i = 0; i < S::kPieces; ++i)
          pt_load<S::kPiece>(vw[e] + S::kPiece * i, src + i * (8 * S::kElems * kEs), r != kPtNone);
      }
    };
    uint32_t rk, rv, rk_next = kPtNone, rv_next = kPtNone;
    int pid = page_id(slot), pid_next = page_id(slot + slots);
    row_of(slot, pid, rk, rv);
    if (slot < nblk) {
      load_k(rk);
      load_v(rv);
    }
    for (int i = slot; i < nblk; i += slots) {
      const int j0 = k0 + 16 * i;
      row_of(i + slots, pid_next, rk_next, rv_next);
      pid_next = page_id(i + 2 * slots);
      // scores S^T = K q^T: s[nb] = (key g: rows 2 cq, 2 cq + 1; key g + 8: the same rows)
      float s[NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t a0, a1, a2, a3;
        if (F8) {
          a0 = pt_cvt_e4m3x2(kw[0][F8 ? ks : 0]);
          a1 = pt_cvt_e4m3x2(kw[1][F8 ? ks : 0]);
          a2 = pt_cvt_e4m3x2(kw[0][F8 ? ks : 0] >> 16);
          a3 = pt_cvt_e4m3x2(kw[1][F8 ? ks : 0] >> 16);
        } else {
          a0 = kw[0][F8 ? 0 : 2 * ks];
          a1 = kw[1][F8 ? 0 : 2 * ks];
          a2 = kw[0][F8 ? 0 : 2 * ks + 1];
          a3 = kw[1][F8 ? 0 : 2 * ks + 1];
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          uint32_t b0, b1;
          if (S::kQRegs) {
            b0 = qr[S::kQRegs ? nb : 0][S::kQRegs ? 2 * ks : 0];
            b1 = qr[S::kQRegs ? nb : 0][S::kQRegs ? 2 * ks + 1 : 0];
          } else {
            const uint2 q2 =
                *reinterpret_cast<const uint2*>(myq + (nb * S::kQWords / 4 + ks / 2) * 128 + (ks % 2) * 2);
            b0 = q2.x;
            b1 = q2.y;
          }
          pt_mma<F8>(s[nb], a0, a1, a2, a3, b0, b1);
        }
      }
      if (i + slots < nblk) load_k(rk_next);
      // a block that not every row sees whole: past some row's position, before some row's window,
      // or with keys that do not exist
      const bool edge = j0 + 15 > sp.len || (p.window > 0 && j0 <= sp.len + sp.cnt - 1 - p.window) ||
                        __any_sync(0xFFFFFFFFu, rk == kPtNone);
      const auto sees = [&](int nb, int e, int key) {  // row 2 cq + e of block nb, key of this block
        const int pos = sp.len + (r0 + 8 * nb + 2 * cq + e) / rep, j = j0 + key;
        return j <= pos && (p.window <= 0 || j > pos - p.window);
      };
      bool up = false;
      uint32_t have = 0;
      if (edge) have = __ballot_sync(0xFFFFFFFFu, rk != kPtNone);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nb][e] *= F8 ? sc[F8 ? nb : 0][e & 1] : sc[0][0];
          if (edge) {
            const int key = g + 8 * (e >> 1);
            if (!(have >> key & 1u) || !sees(nb, e & 1, key)) s[nb][e] = -INFINITY;
          }
        }
        up |= fmaxf(s[nb][0], s[nb][2]) > m[nb][0] + kPtSlack || fmaxf(s[nb][1], s[nb][3]) > m[nb][1] + kPtSlack;
      }
      if (__any_sync(0xFFFFFFFFu, up)) {  // renew the maxima, rescale the sums
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(m[nb][e], fmaxf(s[nb][e], s[nb][2 + e]));
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, w));
            const float f = m[nb][e] == x ? 1.f : pt_exp2(m[nb][e] - x);
            m[nb][e] = x;
            l[nb][e] *= f;
#pragma unroll
            for (int q = 0; q < S::kTiles; ++q) {
              o[nb][q][e] *= f;
              o[nb][q][2 + e] *= f;
            }
          }
      }
      uint32_t pb[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float m0 = m[nb][0] == -INFINITY ? 0.f : m[nb][0], m1 = m[nb][1] == -INFINITY ? 0.f : m[nb][1];
        s[nb][0] = pt_exp2(s[nb][0] - m0);
        s[nb][1] = pt_exp2(s[nb][1] - m1);
        s[nb][2] = pt_exp2(s[nb][2] - m0);
        s[nb][3] = pt_exp2(s[nb][3] - m1);
        l[nb][0] += s[nb][0] + s[nb][2];
        l[nb][1] += s[nb][1] + s[nb][3];
        pb[nb][0] = pt_transpose(pt_pack<F8>(s[nb][0], s[nb][1]));
        pb[nb][1] = pt_transpose(pt_pack<F8>(s[nb][2], s[nb][3]));
      }
      // An infinity or NaN among values that some row does not see would reach it as 0 * inf: such a
      // block (only where tokens of one draft see different keys) is added key by key instead.
      bool apart = false;
      if (edge && p.seq.T > 1) {
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i2 = 0; i2 < S::kPieces * S::kPiece; ++i2) {
            const uint32_t x = vw[e][i2];
            if (F8) odd |= __vcmpeq4(x & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0;
            else odd |= (x & 0x7F80u) == 0x7F80u || (x & 0x7F800000u) == 0x7F800000u;
          }
        apart = __any_sync(0xFFFFFFFFu, odd);
      }
      if (!apart) {  // O^T += V^T P^T
#pragma unroll
        for (int i2 = 0; i2 < S::kPieces * S::kPiece; ++i2) {
          const uint32_t v0 = vw[0][i2], v1 = vw[1][i2], v2 = vw[2][i2], v3 = vw[3][i2];
          if (F8) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const uint32_t x = __byte_perm(v0, v1, hf ? 0x7362 : 0x5140), y = __byte_perm(v2, v3, hf ? 0x7362 : 0x5140);
              const uint32_t a0 = pt_cvt_e4m3x2(x), a1 = pt_cvt_e4m3x2(x >> 16), a2 = pt_cvt_e4m3x2(y),
                             a3 = pt_cvt_e4m3x2(y >> 16);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) pt_mma<true>(o[nb][F8 ? 2 * i2 + hf : 0], a0, a1, a2, a3, pb[nb][0], pb[nb][1]);
            }
          } else {
            const uint32_t a0 = __byte_perm(v0, v1, 0x5410), a1 = __byte_perm(v0, v1, 0x7632),
                           a2 = __byte_perm(v2, v3, 0x5410), a3 = __byte_perm(v2, v3, 0x7632);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) pt_mma<false>(o[nb][F8 ? 0 : i2], a0, a1, a2, a3, pb[nb][0], pb[nb][1]);
          }
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < 4; ++c)  // keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9: held by the lanes (g, c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = 2 * c + (e & 1) + 8 * (e >> 1);
            float pk[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                pk[nb][q] = __shfl_sync(0xFFFFFFFFu, s[nb][(e >> 1) * 2 + q], (2 * c + (e & 1)) * 4 + cq);
                if (!(have >> key & 1u) || !sees(nb, q, key)) pk[nb][q] = -1.f;
              }
#pragma unroll
            for (int i2 = 0; i2 < S::kPieces * S::kPiece; ++i2) {
              const uint32_t x = __shfl_sync(0xFFFFFFFFu, vw[e][i2], g * 4 + c);
              float v[F8 ? 4 : 2];
              if (F8) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  const uint32_t hh = pt_cvt_e4m3x2(x >> (16 * q));
                  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hh));
                  v[F8 ? 2 * q : 0] = f.x;
                  v[F8 ? 2 * q + 1 : 1] = f.y;
                }
              } else {
                v[0] = __uint_as_float(x << 16);
                v[1] = __uint_as_float(x & 0xFFFF0000u);
              }
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int q = 0; q < 2; ++q)
                  if (pk[nb][q] >= 0.f || pk[nb][q] != pk[nb][q]) {
#pragma unroll
                    for (int d = 0; d < (F8 ? 4 : 2); ++d) {
                      float& acc = o[nb][F8 ? 2 * i2 + (d >> 1) : i2][2 * (d & 1) + q];
                      acc = fmaf(pk[nb][q], v[d], acc);
                    }
                  }
            }
          }
      }
      if (i + slots < nblk) load_v(rv_next);
      rk = rk_next;
      rv = rv_next;
    }

    // ---- the warps' results: (maximum, sum) and O to shared memory, joined by all threads
    __syncthreads();  // the previous segment's reads are done
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[nb][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nb][e], w);
        const int r = 8 * nb + 2 * cq + e;
        if (g == 0) {
          sml[warp][r][0] = m[nb][e];
          sml[warp][r][1] = l[nb][e];
        }
        float* const dst = so + (warp * 8 * NB + r) * (D + 4);
#pragma unroll
        for (int q = 0; q < S::kTiles; q += 2) {  // two tiles: 4 consecutive dims
          const int per = S::kElems / 2, piece = q / per, in = q % per;
          *reinterpret_cast<float4*>(dst + piece * 8 * S::kElems + g * S::kElems + 2 * in) =
              make_float4(o[nb][q][e], o[nb][q][2 + e], o[nb][q + 1][e], o[nb][q + 1][2 + e]);
        }
      }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == sp.tiles;
    const size_t piece = 2 * static_cast<size_t>(blockIdx.x) + (seg > 0);
    const float vs = F8 ? p.v_scale[kvh] : 1.f;
    const int live = min(plan.rows, sp.cnt * rep - rbase);  // rows of the group that exist
    for (int e = tid; e < live * (D / 4); e += kPtThreads) {
      const int r = e / (D / 4), d = (e % (D / 4)) * 4, c = r / (8 * NB), rr = r % (8 * NB);
      float mx = -INFINITY;
      for (int w = c; w < kPtWarps; w += plan.nchunk) mx = fmaxf(mx, sml[w][rr][0]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
      for (int w = c; w < kPtWarps; w += plan.nchunk) {
        const float f = sml[w][rr][0] == mx ? 1.f : pt_exp2(sml[w][rr][0] - mx);
        const float4 x = *reinterpret_cast<const float4*>(so + (w * 8 * NB + rr) * (D + 4) + d);
        sum = fmaf(f, sml[w][rr][1], sum);
        acc.x = fmaf(f, x.x, acc.x);
        acc.y = fmaf(f, x.y, acc.y);
        acc.z = fmaf(f, x.z, acc.z);
        acc.w = fmaf(f, x.w, acc.w);
      }
      if (whole) {
        const int t = (rbase + r) / rep, h = kvh * rep + (rbase + r) % rep;
        const size_t row = (static_cast<size_t>(b) * p.seq.T + t) * p.Hq + h;
        const float inv = sum == 0.f ? 0.f : vs / sum;
        uint2 w;
        w.x = pt_pack<false>(acc.x * inv, acc.y * inv);
        w.y = pt_pack<false>(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(p.out + row * D + d) = w;
        if (d == 0 && p.lse) p.lse[row] = (mx + log2f(sum)) * 0.6931471805599453f;
      } else {
        *reinterpret_cast<float4*>(plan.o + (piece * plan.rows + r) * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(plan.ml + (piece * plan.rows + r) * 2) = make_float2(mx, sum);
      }
    }
    const int done = t1 - t0;
    u += done;
    off += done;
    if (off == static_cast<long long>(sp.tiles) * items) {
      ++b;
      off = 0;
    }
  }
  if (__any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicOr(p.seq.err, kErrBitBadInput);
}

// Joins the pieces of the items that were split, one output row per CTA, and writes the rows that no
// piece covers (idle slots, padding).  Warp w adds pieces w, w + 4, ... and the four results are
// added in order.
template <int D>
__global__ void __launch_bounds__(kPtThreads)
    paged_attn_join_kernel(const __grid_constant__ PagedAttnParams p, const __grid_constant__ PagedAttnPlan plan) {
  constexpr int kPer = D / 32;
  constexpr int kAhead = 4;  // pieces whose loads are issued together
  __shared__ float so[kPtWarps][D], sml[kPtWarps][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rep = p.Hq / p.Hkv;
  const size_t row = blockIdx.x;
  const int h = static_cast<int>(row % p.Hq), t = static_cast<int>(row / p.Hq % p.seq.T),
            b = static_cast<int>(row / p.Hq / p.seq.T);
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  const PagedSpan sp = paged_span(p, b);
  if (t >= sp.cnt) {  // padding
    for (int d = tid; d < D / 8; d += kPtThreads)
      reinterpret_cast<uint4*>(p.out + row * D)[d] = make_uint4(0u, 0u, 0u, 0u);
    if (tid == 0 && p.lse) p.lse[row] = -INFINITY;
    return;
  }
  const int kvh = h / rep, r = t * rep + h % rep, item = kvh * plan.groups + r / plan.rows, rr = r % plan.rows;
  const long long total = __ldcg(plan.pre + p.seq.B);
  const long long parts = min(static_cast<long long>(plan.ctas), total);
  const long long beg = __ldcg(plan.pre + b) + static_cast<long long>(item) * sp.tiles, end = beg + sp.tiles;
  // the CTA that holds tile u: the last i with i * total / parts <= u
  const int first = static_cast<int>(((beg + 1) * parts - 1) / total), last = static_cast<int>((end * parts - 1) / total);
  if (first == last) return;  // one CTA had the whole item
  const auto piece = [&](int i) {  // where CTA i put this item: in its first piece unless it began another before
    return 2 * static_cast<size_t>(i) + (i * total / parts < beg);
  };
  float m = -INFINITY, l = 0.f, acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  for (int i0 = first + warp; i0 <= last; i0 += kPtWarps * kAhead) {
    float2 ml[kAhead];
    float x[kAhead][kPer];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int i = min(i0 + a * kPtWarps, last);
      const size_t at = piece(i) * plan.rows + rr;
      ml[a] = __ldcg(reinterpret_cast<const float2*>(plan.ml + at * 2));
#pragma unroll
      for (int q = 0; q < kPer; ++q) x[a][q] = __ldcg(plan.o + at * D + lane + 32 * q);
    }
    float mx = m;
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      if (i0 + a * kPtWarps <= last) mx = fmaxf(mx, ml[a].x);
    const float f = m == mx ? 1.f : pt_exp2(m - mx);
    m = mx;
    l *= f;
#pragma unroll
    for (int q = 0; q < kPer; ++q) acc[q] *= f;
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      if (i0 + a * kPtWarps <= last) {
        const float w = ml[a].x == mx ? 1.f : pt_exp2(ml[a].x - mx);
        l = fmaf(w, ml[a].y, l);
#pragma unroll
        for (int q = 0; q < kPer; ++q) acc[q] = fmaf(w, x[a][q], acc[q]);
      }
  }
#pragma unroll
  for (int q = 0; q < kPer; ++q) so[warp][lane + 32 * q] = acc[q];
  if (lane == 0) {
    sml[warp][0] = m;
    sml[warp][1] = l;
  }
  __syncthreads();
  float mx = -INFINITY, sum = 0.f, f[kPtWarps];
#pragma unroll
  for (int w = 0; w < kPtWarps; ++w) mx = fmaxf(mx, sml[w][0]);
#pragma unroll
  for (int w = 0; w < kPtWarps; ++w) {
    f[w] = sml[w][0] == mx ? 1.f : pt_exp2(sml[w][0] - mx);
    sum = fmaf(f[w], sml[w][1], sum);
  }
  const float inv = sum == 0.f ? 0.f : (p.v_scale ? p.v_scale[kvh] : 1.f) / sum;
  for (int d = 2 * tid; d < D; d += 2 * kPtThreads) {
    float a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int w = 0; w < kPtWarps; ++w) {
      a0 = fmaf(f[w], so[w][d], a0);
      a1 = fmaf(f[w], so[w][d + 1], a1);
    }
    *reinterpret_cast<uint32_t*>(p.out + row * D + d) = pt_pack<false>(a0 * inv, a1 * inv);
  }
  if (tid == 0 && p.lse) p.lse[row] = (mx + log2f(sum)) * 0.6931471805599453f;
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
namespace {

// 8-row blocks one warp may hold: as many as leave room for a block of keys and values in registers.
int pt_max_blocks(int D, bool f8) { return D <= 128 ? 4 : f8 ? 2 : 1; }

struct PtChoice {
  int nb, nchunk, groups, rows, ctas_per_sm;
};

PtChoice pt_choose(int T, int Hq, int Hkv, int D, bool f8) {
  const int blocks = (T * (Hq / Hkv) + 7) / 8, most = pt_max_blocks(D, f8);
  PtChoice c;
  c.nb = blocks >= 3 ? std::min(4, most) : std::min(blocks, most);
  const int chunks = (blocks + c.nb - 1) / c.nb;
  c.nchunk = chunks >= 3 ? 4 : chunks;
  c.groups = (chunks + c.nchunk - 1) / c.nchunk;
  c.rows = 8 * c.nb * c.nchunk;
  c.ctas_per_sm = c.nb * D <= 128 ? 3 : 2;
  return c;
}

size_t pt_round(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

template <int D, int NB, bool F8>
cudaError_t pt_split(const PagedAttnParams& p, const PagedAttnPlan& plan, int dev, cudaLaunchConfig_t cfg) {
  static std::atomic<bool> attr_set[64];
  const auto kernel = paged_attn_split_kernel<D, NB, F8>;
  constexpr int smem = pt_smem_bytes<D, NB, F8>();
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    attr_set[dev].store(true, std::memory_order_release);
  }
  cfg.dynamicSmemBytes = smem;
  return cudaLaunchKernelEx(&cfg, kernel, p, plan);
}

template <int D>
cudaError_t pt_launch(const PagedAttnParams& p, const PagedAttnPlan& plan, int nb, bool f8, int dev, cudaLaunchConfig_t cfg) {
  cudaError_t e = cudaErrorInvalidValue;
  if (nb == 1) e = f8 ? pt_split<D, 1, true>(p, plan, dev, cfg) : pt_split<D, 1, false>(p, plan, dev, cfg);
  if constexpr (D <= 128) {
    if (nb == 2) e = f8 ? pt_split<D, 2, true>(p, plan, dev, cfg) : pt_split<D, 2, false>(p, plan, dev, cfg);
    if (nb == 4) e = f8 ? pt_split<D, 4, true>(p, plan, dev, cfg) : pt_split<D, 4, false>(p, plan, dev, cfg);
  } else {
    if (nb == 2 && f8) e = pt_split<D, 2, true>(p, plan, dev, cfg);
  }
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<long long>(p.seq.B) * p.seq.T * p.Hq));
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<D>, p, plan);
}

}  // namespace

size_t paged_attn_ws_bytes(int B, int T, int Hq, int Hkv, int D, int n_sm) {
  size_t most = 0;
  for (int f8 = 0; f8 < 2; ++f8) {
    const PtChoice c = pt_choose(T, Hq, Hkv, D, f8);
    const size_t pieces = 2 * static_cast<size_t>(std::max(n_sm, 1)) * c.ctas_per_sm;
    most = std::max(most, pt_round(8 * (static_cast<size_t>(B) + 1)) + pt_round(pieces * c.rows * 8) + pieces * c.rows * D * 4);
  }
  return most;
}

cudaError_t paged_attn_launch(const PagedAttnParams& p, bool f8, void* ws, int n_sm, cudaStream_t stream) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || n_sm < 1) return cudaErrorInvalidDevice;
  const PtChoice c = pt_choose(p.seq.T, p.Hq, p.Hkv, p.D, f8);
  PagedAttnPlan plan;
  plan.nchunk = c.nchunk;
  plan.groups = c.groups;
  plan.rows = c.rows;
  plan.ctas = n_sm * c.ctas_per_sm;
  uint8_t* const base = static_cast<uint8_t*>(ws);
  const size_t n_pre = pt_round(8 * (static_cast<size_t>(p.seq.B) + 1));
  plan.pre = reinterpret_cast<long long*>(base);
  plan.ml = reinterpret_cast<float*>(base + n_pre);
  plan.o = reinterpret_cast<float*>(base + n_pre + pt_round(2 * static_cast<size_t>(plan.ctas) * c.rows * 8));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(plan.ctas);
  cfg.blockDim = dim3(kPtThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (p.D == 64) return pt_launch<64>(p, plan, c.nb, f8, dev, cfg);
  if (p.D == 128) return pt_launch<128>(p, plan, c.nb, f8, dev, cfg);
  return pt_launch<256>(p, plan, c.nb, f8, dev, cfg);
}

}  // namespace skinny
