// Attention of 1..16 new tokens per sequence over a paged key-value cache:
//
//   o[b, t, h] = sum_j softmax_j(scale * q[b, t, h] . k_j) v_j     (query head h reads kv head h / rep)
//
// over the positions j <= lengths[b] + t of sequence b's pages (and j > lengths[b] + t - window).
// A row that sees nothing (an idle slot, t >= counts[b], every page bad) is zero, its lse -inf.
//
// This file: the split launch for few rows per kv head, for 8-bit pages and for pages that are not eights of positions,
// and the join.  paged_attn_tc.cu: the split launch for more rows.
//
// One pass over the cache with a running maximum and sum, split over the cache's length and joined
// (online softmax).  Bound by the bytes of the keys and values: each is read once from memory, by
// the warp that multiplies it:
//
// * The keys are the 16-row operand and the query rows (t, head in the group; at most 8 NB of them)
//   the 8-column operand: S^T[key][row] = K q^T, then O^T[dim][row] += V^T P^T.  A decode step has
//   few rows, so 8-column tiles waste the least of the matrix unit, and O needs D / 16 * 4 registers
//   per 8 rows.
// * Keys and values come by TMA, in boxes of up to a block's consecutive positions of a page (the
//   largest power of two that divides the page size, so any page size works), in lines of 128 bytes,
//   swizzled, which makes the fragment loads below conflict-free.  The copy engine takes some 12 clocks per request
//   whatever its size: one request per 256-byte row held the kernel at 5.9 TB/s, per 128-byte row at
//   3.1.  A warp copies its own blocks and waits for them alone (one mbarrier per stage of keys and of
//   values): the loop has no CTA barrier.  Ordinary asynchronous copies (16 bytes per lane) stood in
//   the way of the shared-memory reads behind them in the same pipe: 4.3 TB/s.
// * K fragments are ldmatrix rows.  e4m3 rows are read as pairs: a lane then holds 4 consecutive dims,
//   two operand pieces of a 16-dim step in an order the query rows are stored in too (a dot product
//   does not care).  V fragments: the 8 (16) consecutive dims a lane reads of a value row are its rows
//   of 4 (8) output tiles; pairs of keys are interleaved with byte permutes.
// * P^T as an operand is the transpose of the S^T accumulators, one movmatrix per 8 x 8 block.
//
// The maximum a row's exponentials refer to is renewed only when a score exceeds it by more than
// 8 (in powers of two): p stays below 256, and the usual block needs one warp vote instead of shuffles and
// a rescaling of O.
// Roundings: scores, maxima, sums and O are f32; p is rounded to bf16 (half a step, as the output's own
// rounding), the same relative precision however far a key lies below the row's largest.  The sum adds the p
// before that rounding, so the lse does not see it.  e4m3 keys and values are exact in bf16 and converted in
// registers.  (f16 is one instruction nearer, but its smallest number is 2^-24: keys 17 nats below a dominating
// one, and elements of q far below the row's largest, were lost.  f16 against bf16: 64 sequences up to 4 K 73.5
// and 73 us, two of 131 K 95.5 and 93, 16 rows of 16 K 35 and 39, heads of 64 54.5 and 64.5, of 256 32.6 and 35.)
//
// Work split: the key tiles of all (sequence, kv head, row group) items form one line that is cut
// into equal pieces, one per CTA (`kCtas` CTAs per SM), so that ragged lengths balance; the
// lengths are read on the device and the launch does not depend on them (a captured graph serves
// any).  A CTA whose piece covers an item writes its output; the others write (max, sum, O) to the
// workspace and the join launch adds them in order, so results do not depend on timing.
//
// Times in this file are per call (both launches) of back-to-back graph replays over inputs larger than L2.
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda.h>
#include <cuda_runtime.h>

#include "mma_bf16.cuh"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "ptx.cuh"

namespace skinny {

constexpr int kPtThreads = 128;
constexpr int kPtWarps = kPtThreads / 32;
constexpr int kPtLead = 4;             // (0 to 8 tried: verify 31.6 us at 0, 26 at 4 and 6, 26.7 at 8; the others hardly move)
__device__ __forceinline__ uint32_t pt_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void pt_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void pt_lds4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void pt_lds2(uint32_t& x, uint32_t& y, uint32_t a) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(a) : "memory");
}

// Two pairs of e4m3 to two pairs of bf16 (exact, NaN stays NaN): by way of f16, of which bf16 is the upper half in f32.
__device__ __forceinline__ uint32_t pt_f16_to_bf16(uint32_t x) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
  return __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x7632);
}
__device__ __forceinline__ void pt_cvt_e4m3(uint32_t& lo, uint32_t& hi, uint32_t x) {
  uint32_t a, b;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(a), "=r"(b)
      : "r"(x));
  lo = pt_f16_to_bf16(a);
  hi = pt_f16_to_bf16(b);
}

// Sizes of one instance.
template <int D, int NB, bool F8>
struct PtShape {
  static constexpr int kEs = F8 ? 1 : 2;
  // Keys of one block: 16, or 32 where a block of 16 would be less than 8 KB (the block's fixed
  // instructions count for more then).
  static constexpr int kSub = 16 * 2 * D * kEs < 8192 ? 2 : 1;
  static constexpr int kKeys = 16 * kSub;
  static constexpr int kRow = D * kEs;                           // bytes of a key or value row
  static constexpr int kLine = kRow < 128 ? kRow : 128;          // bytes of it that one copy takes
  static constexpr int kLines = kRow / kLine;
  static constexpr int kQPad = 2 * D + 16;                       // bytes of a query row in shared memory (16-bit)
  static constexpr int kQLoads = D / 32;                         // query fragment loads (4 words) per lane and 8 rows
  static constexpr int kVBytes = F8 && D == 64 ? 8 : 16;         // bytes of one value fragment load
  static constexpr int kVLoads = kRow / (8 * kVBytes);           // value fragment loads per lane and key (4 keys per 16)
  static constexpr int kElems = kVBytes / kEs;                   // consecutive dims of one value load
  static constexpr int kTiles = D / 16;                          // output tiles of 16 dims
  static constexpr bool kQRegs = NB * D <= 256 && (F8 || D < 256);  // query fragments stay in registers
  static constexpr int kCtas = NB * D <= 128 ? 3 : 2;            // CTAs per SM
  static constexpr int kKBytes = kKeys * kRow;                   // keys (or values) of one block
  static constexpr int kStages = 16384 / (2 * kKBytes);
  static constexpr bool kJoint = kStages > 1;  // keys and values of a block on one barrier (else the one is fetched
                                               // again while the other is in use)
  static constexpr int kMaxNB = D <= 128 ? 4 : F8 ? 2 : 1;
  static constexpr int kChunks = NB == kMaxNB ? kPtWarps : 1;    // row chunks a CTA may hold
  static constexpr int kORow = D + 4;                            // floats of one row of O in shared memory
  // a warp's region: its ring, later its O
  static constexpr int kRing = kStages * 2 * kKBytes, kOBytes = 8 * NB * kORow * 4;
  static constexpr int kWarpBytes = ((kRing > kOBytes ? kRing : kOBytes) + 1023) / 1024 * 1024;
  static constexpr int kSmem = 1024 + kPtWarps * kWarpBytes + kChunks * 8 * NB * kQPad;
  static_assert(kStages >= 1 && kKBytes % 1024 == 0, "a block starts on a swizzle period");
};

template <int D, int NB, bool F8>
__global__ void __launch_bounds__(kPtThreads, PtShape<D, NB, F8>::kCtas)
    paged_attn_split_kernel(const __grid_constant__ PagedAttnParams p, const __grid_constant__ PagedAttnPlan plan,
                            const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using S = PtShape<D, NB, F8>;
  constexpr int kSub = S::kSub, kStages = S::kStages;
  extern __shared__ __align__(1024) uint8_t pt_raw[];
  uint8_t* const pt_smem = pt_raw + ((1024 - (smem_u32(pt_raw) & 1023)) & 1023);  // swizzle periods are 1 KB
  __shared__ uint64_t bars[kPtWarps][kStages][2];  // per warp and stage: the block (its keys, its values) is there
  __shared__ int gave_up;                          // a wait ran out
  __shared__ float sml[kPtWarps][8 * NB][2];
  __shared__ long long scan[kPtWarps];
  __shared__ long long found[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cq = lane & 3;
  const int rep = p.Hq / p.Hkv, items = p.Hkv * plan.groups;
  const uint32_t bar0 = smem_u32(&bars[warp][0][0]);
  pdl_launch_dependents();
  if (lane < kStages * 2) mbar_init(bar0 + 8 * lane, 1);
  if (tid == 0) gave_up = 0;
  fence_mbar_init();
  __syncthreads();

  PtWalk walk;
  if (!pt_begin<kPtThreads>(p, plan, items, scan, found, walk)) return;

  const int chunk = warp % plan.nchunk, slot = warp / plan.nchunk, slots = kPtWarps / plan.nchunk;
  const uint32_t kpr = static_cast<uint32_t>(p.kps / D), vpr = static_cast<uint32_t>(p.vps / D);
  const int boxes = S::kKeys / plan.box;  // of one block
  uint8_t* const region = pt_smem + warp * S::kWarpBytes;
  float* const so = reinterpret_cast<float*>(region);                  // [8 NB][kORow], after the loop
  const uint32_t ring = smem_u32(region);                               // [stage][keys | values][line][key][kLine], swizzled
  // Fragment addresses inside a block.  Swizzle: 16-byte piece c of a 128-byte line of key k lies at
  // c ^ (k & 7), of a 64-byte line at c ^ (k / 2 & 3).  K by ldmatrix: lanes 0-15 keys 0-15 at piece 2 i,
  // lanes 16-31 at 2 i + 1 (the piece's step is an xor).  V: keys 2 cq + (e & 1) + 8 (e >> 1), dims from 8 g
  // (16 g).
  const uint32_t kkey = lane & 15, kswz = S::kLine == 128 ? kkey & 7 : kkey >> 1 & 3;
  const uint32_t klane = kkey * S::kLine + ((static_cast<uint32_t>(lane >> 4) ^ kswz) << 4);
  const uint32_t vlane0 = S::kLine == 128 ? 2 * cq * 128 + ((g ^ (2 * cq)) << 4)
                                          : 2 * cq * 64 + (((g >> 1) ^ cq) << 4) + (g & 1) * 8;
  const uint32_t vlane1 = S::kLine == 128 ? (vlane0 ^ 16) + 128 : vlane0 + 64;  // the odd keys
  uint8_t* const sq = pt_smem + kPtWarps * S::kWarpBytes;               // [chunk][8 NB][kQPad]
  int stage = 0;                       // of the next block to multiply
  uint32_t pending = 0, parity = 0;    // per barrier (bit 2 stage + what): copies in flight, the phase they complete
  bool bad = false;

  PtPart part;
  for (int seg = 0; walk.next(p, plan, items, part);) {
    const PagedSpan sp = part.sp;
    const int item = part.item, cur = part.seq, t0 = part.t0, t1 = part.t1;
    const int kvh = item / plan.groups, rbase = (item % plan.groups) * plan.rows;
    const int k0 = sp.first + (t0 << plan.tile_log), k1 = min(sp.end, sp.first + (t1 << plan.tile_log));
    const int r0 = rbase + chunk * 8 * NB;  // this warp's first row
    const int32_t* const table = p.seq.table + cur * p.seq.table_stride;

    // ---- the query rows, 8 dims per thread at a time: asked for before the keys and values
    constexpr int kQBatch = NB * D / 128 < 1 ? 1 : NB * D / 128;  // pieces per thread of one chunk
    const auto q_load = [&](int e) {
      const int r = rbase + e / (D / 8), t = plan.token(r), h = kvh * rep + (r - t * rep);
      return t < sp.cnt ? __ldg(reinterpret_cast<const uint4*>(p.q + cur * p.qs[0] + t * p.qs[1] + h * p.qs[2]) + e % (D / 8))
                        : make_uint4(0u, 0u, 0u, 0u);
    };
    const int q_pieces = plan.rows * (D / 8);
    uint4 qw[kQBatch];
#pragma unroll
    for (int i = 0; i < kQBatch; ++i) {
      const int e = tid + i * kPtThreads;
      if (e < q_pieces) qw[i] = q_load(e);
    }

    // ---- this warp's blocks of keys: block n holds the keys from k0 + kKeys (n slots + slot)
    const int nblk_all = (k1 - k0 + S::kKeys - 1) / S::kKeys;
    const int nblk = nblk_all > slot ? (nblk_all - slot + slots - 1) / slots : 0;
    const auto first_key = [&](int n) { return k0 + S::kKeys * (n * slots + slot); };
    // a block's pages, one key per lane (16 keys: lanes 16..31 repeat), and from them its rows
    const auto page_of = [&](int n, int& in_page) {
      const int j = first_key(n) + (lane & (S::kKeys - 1));
      if (n >= nblk || j < sp.beg || j >= k1) return -2;
      const int q = plan.shift >= 0 ? j >> plan.shift : j / p.seq.page;
      in_page = j - q * p.seq.page;
      return __ldg(table + q);
    };
    uint32_t rk, rv;
    const auto rows_of = [&](int pid, int in_page) {  // -> the keys that exist, one bit each
      const bool ok = pid >= 0 && pid < p.seq.n_pages;
      bad |= !ok && pid != -2;
      const uint32_t in = static_cast<uint32_t>(kvh) * p.seq.page + static_cast<uint32_t>(in_page);
      rk = static_cast<uint32_t>(pid) * kpr + in;
      rv = static_cast<uint32_t>(pid) * vpr + in;
      return __ballot_sync(0xFFFFFFFFu, ok);
    };
    // The block whose pages were looked up last (one key per lane) into stage st, whose slots have been
    // read.  what: 0 keys, 1 values, 2 both (on the keys' barrier).  A box without a key that exists is
    // left out.
    const auto copy = [&](int st, int what, uint32_t exist) {
      const int bit = st * 2 + (what & 1);
      const uint32_t bar = bar0 + bit * 8, dst = ring + st * (2 * S::kKBytes);
      pending |= 1u << bit;
      if (boxes == 1) {  // one copy each, by lane 0
        const int src = exist ? __ffs(exist) - 1 : 0;
        const int row_k = static_cast<int>(__shfl_sync(0xFFFFFFFFu, rk, src)) - src;  // (orders the lanes' reads too)
        const int row_v = static_cast<int>(__shfl_sync(0xFFFFFFFFu, rv, src)) - src;
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, exist ? S::kKBytes * (what == 2 ? 2 : 1) : 0);
          if (exist) {
            if (what != 1) tma_load_3d(dst, &kmap, 0, row_k, 0, bar);
            if (what != 0) tma_load_3d(dst + S::kKBytes, &vmap, 0, row_v, 0, bar);
          }
        }
        return;
      }
      const uint32_t mask = (1u << plan.box) - 1u;  // one box per lane
      const int some = __popc(__ballot_sync(0xFFFFFFFFu, lane < boxes && (exist >> (lane * plan.box) & mask)));
      if (lane == 0) mbar_arrive_expect_tx(bar, some * plan.box * S::kRow * (what == 2 ? 2 : 1));
      __syncwarp();
      const int n = what == 2 ? 2 * boxes : boxes;
      for (int q0 = 0; q0 < n; q0 += 32) {
        const int q = q0 + lane, first = (q & (boxes - 1)) * plan.box, kv = what == 2 ? q >= boxes : what;
        const uint32_t here = q < n ? exist & mask << first : 0u;
        const int src = here ? __ffs(here) - 1 : 0;
        const uint32_t row_k = __shfl_sync(0xFFFFFFFFu, rk, src), row_v = __shfl_sync(0xFFFFFFFFu, rv, src);
        const uint32_t row = (kv ? row_v : row_k) - static_cast<uint32_t>(src - first);
        const uint32_t to = dst + kv * S::kKBytes + first * S::kLine;
        if (here) {
          if (S::kLine == 64 && plan.box == 1) {  // 64 bytes: less than a tiled copy's alignment
            const uint8_t* const from = static_cast<const uint8_t*>(kv ? p.vp : p.kp) + static_cast<size_t>(row) * S::kRow;
            for (int c = 0; c < 4; ++c) bulk_g2s(to + ((c ^ (first >> 1 & 3)) << 4), from + 16 * c, 16, bar);
          } else {
            // (a box of several lines would lay them out box by box: one line each)
#pragma unroll
            for (int c = 0; c < S::kLines; ++c)
              tma_load_3d(to + c * (S::kKeys * S::kLine), kv ? &vmap : &kmap, 0, static_cast<int>(row), c, bar);
          }
        }
      }
    };
    const auto arrived = [&](int bit) {  // bounded; the same answer in every lane
      const bool ok = mbar_wait(bar0 + bit * 8, parity >> bit & 1u, p.seq.err, kErrBitWaitFull, &gave_up);
      if (!__all_sync(0xFFFFFFFFu, ok)) return false;
      pending &= ~(1u << bit);
      parity ^= 1u << bit;
      return true;
    };
    uint32_t have[kStages];  // the keys that exist of the blocks in flight
    int pid_next, in_next = 0;
    {
      int pid[kStages], in[kStages];
#pragma unroll
      for (int st = 0; st < kStages; ++st) {
        in[st] = 0;
        pid[st] = page_of(st, in[st]);
      }
      pid_next = page_of(kStages, in_next);
      if (seg > 0) {
        fence_proxy_async_smem();  // the previous segment's O was written here by ordinary stores
        __syncthreads();           // and has been read
      }
#pragma unroll
      for (int st = 0; st < kStages; ++st) {
        have[st] = rows_of(pid[st], in[st]);
        if (st < nblk) {
          const int where = stage + st < kStages ? stage + st : stage + st - kStages;
          if (S::kJoint) {
            copy(where, 2, have[st]);
          } else {
            copy(where, 0, have[st]);
            copy(where, 1, have[st]);
          }
        }
      }
    }

    // ---- the query rows to shared memory
    const float sc = p.scale * 1.4426950408889634f * (F8 ? p.k_scale[kvh] : 1.f);
    const auto q_store = [&](int e, uint4 w) {
      const int row = e / (D / 8), u8 = e % (D / 8);
      uint8_t* const dst = sq + row * S::kQPad;
      if (F8) {  // pairs 0, 2, .. of 16 dims before pairs 1, 3, ..
        *reinterpret_cast<uint2*>(dst + (u8 >> 1) * 32 + (u8 & 1) * 8) = make_uint2(w.x, w.z);
        *reinterpret_cast<uint2*>(dst + (u8 >> 1) * 32 + 16 + (u8 & 1) * 8) = make_uint2(w.y, w.w);
      } else {
        reinterpret_cast<uint4*>(dst)[u8] = w;
      }
    };
#pragma unroll
    for (int i = 0; i < kQBatch; ++i) {
      const int e = tid + i * kPtThreads;
      if (e < q_pieces) q_store(e, qw[i]);
    }
    for (int e = tid + kQBatch * kPtThreads; e < q_pieces; e += kPtThreads) q_store(e, q_load(e));
    __syncthreads();
    // fragments by ldmatrix: rows 0-7 of a block at 16-byte pieces 4 i .. 4 i + 3
    const uint32_t qaddr = smem_u32(sq) + (chunk * 8 * NB + (lane & 7)) * S::kQPad + (lane >> 3) * 16;
    // and where they do not stay in registers, one 16-dim step of two blocks (of one block)
    const uint32_t qaddr_2 = smem_u32(sq) + (chunk * 8 * NB + (lane & 7) + 8 * (lane >> 4)) * S::kQPad + ((lane >> 3) & 1) * 16;
    const uint32_t qaddr_x2 = smem_u32(sq) + (chunk * 8 * NB + (lane & 7)) * S::kQPad + ((lane >> 3) & 1) * 16;
    uint32_t qr[S::kQRegs ? NB : 1][S::kQRegs ? S::kQLoads : 1][4];
    if (S::kQRegs) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < S::kQLoads; ++i) {
          uint32_t(&x)[4] = qr[S::kQRegs ? nb : 0][S::kQRegs ? i : 0];
          ldsm_x4(qaddr + nb * 8 * S::kQPad + i * 64, x[0], x[1], x[2], x[3]);
        }
    }
    // the tokens of this lane's rows, 4 bits each (rows past the last token: any)
    uint32_t tokens = 0;
    if (p.seq.T > 1) {
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) tokens |= min(15, plan.token(r0 + 8 * (i >> 1) + 2 * cq + (i & 1))) << (4 * i);
    }

    // ---- one pass over the blocks
    float o[NB][S::kTiles][4], m[NB][2], l[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb][0] = m[nb][1] = kPtNothing;
      l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
      for (int i = 0; i < S::kTiles; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nb][i][e] = 0.f;
    }
    const auto sees = [&](int t, int j) {  // does token t see position j
      const int pos = sp.len + t;
      return j <= pos && (p.window <= 0 || j > pos - p.window);
    };
    const auto is_edge = [&](int j0) {  // a block that some row sees only part of
      return j0 + S::kKeys - 1 > sp.len || (p.window > 0 && j0 <= sp.len + sp.cnt - 1 - p.window);
    };
    bool poison = false;
    for (int n = 0; n < nblk; ++n) {
      const int j0 = first_key(n);
      const uint32_t kaddr = ring + stage * (2 * S::kKBytes) + klane;
      const uint32_t vblock = ring + stage * (2 * S::kKBytes) + S::kKBytes;
      const uint32_t now = have[0];
      const uint32_t have_next = rows_of(pid_next, in_next);
      pid_next = page_of(n + kStages + 1, in_next);
      // scores S^T = K q^T: s[nb][sub] = (key g: rows 2 cq, 2 cq + 1; key g + 8: the same rows)
      float s[NB][kSub][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int sub = 0; sub < kSub; ++sub) s[nb][sub][0] = s[nb][sub][1] = s[nb][sub][2] = s[nb][sub][3] = 0.f;
      if (!arrived(stage * 2)) break;
      // (fragments of 4 steps asked for together: verify 26.4 -> 25.2 us, of 8 the same)
      constexpr int kSteps = S::kRow / 32, kBatch = kSteps < 4 ? kSteps : 4;
      uint32_t kb[kBatch][kSub][4];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {  // 32 bytes of 16 (32) keys: one 16-dim step, or two of e4m3
        if (i % kBatch == 0)
#pragma unroll
          for (int a = 0; a < kBatch; ++a)
#pragma unroll
            for (int sub = 0; sub < kSub; ++sub) {
              uint32_t(&x)[4] = kb[a][sub];
              ldsm_x4((kaddr ^ ((i + a) * 32 % S::kLine)) + (i + a) * 32 / S::kLine * (S::kKeys * S::kLine) + sub * 16 * S::kLine,
                      x[0], x[1], x[2], x[3]);
            }
        uint32_t(&kw)[kSub][4] = kb[i % kBatch];
#pragma unroll
        for (int c = 0; c < (F8 ? 2 : 1); ++c) {
          const int ks = F8 ? 2 * i + c : i;
          uint32_t bq[NB][2];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            if (S::kQRegs) {
              bq[nb][0] = qr[S::kQRegs ? nb : 0][S::kQRegs ? ks / 2 : 0][(ks & 1) * 2];
              bq[nb][1] = qr[S::kQRegs ? nb : 0][S::kQRegs ? ks / 2 : 0][(ks & 1) * 2 + 1];
            }
          }
          if (!S::kQRegs) {
            if (NB == 1) {
              ldsm_x2(qaddr_x2 + ks * 32, bq[0][0], bq[0][1]);
            } else {
#pragma unroll
              for (int nb = 0; nb < NB; nb += 2)
                ldsm_x4(qaddr_2 + nb * 8 * S::kQPad + ks * 32, bq[nb][0], bq[nb][1], bq[(nb + 1) % NB][0], bq[(nb + 1) % NB][1]);
            }
          }
#pragma unroll
          for (int sub = 0; sub < kSub; ++sub) {
            uint32_t a0, a1, a2, a3;  // (keys 0-7, 8-15) x (first, second half of the step)
            if (F8) {
              pt_cvt_e4m3(a0, a2, kw[sub][2 * c]);
              pt_cvt_e4m3(a1, a3, kw[sub][2 * c + 1]);
            } else {
              a0 = kw[sub][0];
              a1 = kw[sub][1];
              a2 = kw[sub][2];
              a3 = kw[sub][3];
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) pt_mma(s[nb][sub], a0, a1, a2, a3, bq[nb][0], bq[nb][1]);
          }
        }
      }
      if (!S::kJoint && n + kStages < nblk) copy(stage, 0, have_next);
      constexpr uint32_t kAll = 0xFFFFFFFFu;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int sub = 0; sub < kSub; ++sub)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nb][sub][e] *= sc;
      if (is_edge(j0) || now != kAll) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int t = tokens >> (4 * (2 * nb + e)) & 15u;
#pragma unroll
            for (int sub = 0; sub < kSub; ++sub)
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                const int key = 16 * sub + 8 * hf + g;
                if (!(now >> key & 1u) || !sees(t, j0 + key)) s[nb][sub][2 * hf + e] = -INFINITY;
              }
          }
      }
      // p = 2^(s - m), with the maximum of the blocks before
      float pr[NB][kSub][4];
      const auto exponentials = [&]() {
        float top = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int sub = 0; sub < kSub; ++sub)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              pr[nb][sub][e] = pt_exp2(s[nb][sub][e] - m[nb][e & 1]);
              top = fmaxf(top, pr[nb][sub][e]);
            }
        return top;
      };
      if (__any_sync(0xFFFFFFFFu, exponentials() > kPtMost)) {  // renew the maxima, rescale the sums
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = m[nb][e];
#pragma unroll
            for (int sub = 0; sub < kSub; ++sub)
              x = fmaxf(x, fmaxf(s[nb][sub][e], s[nb][sub][2 + e]));
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, w));
            const float f = pt_exp2(m[nb][e] - x);
            m[nb][e] = x;
            l[nb][e] *= f;
#pragma unroll
            for (int q = 0; q < S::kTiles; ++q) {
              o[nb][q][e] *= f;
              o[nb][q][2 + e] *= f;
            }
          }
        exponentials();
      }
      uint32_t pb[NB][kSub][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int sub = 0; sub < kSub; ++sub) {
          const float(&x)[4] = pr[nb][sub];
          l[nb][0] += x[0] + x[2];
          l[nb][1] += x[1] + x[3];
          pb[nb][sub][0] = pt_transpose(pt_pack(x[0], x[1]));
          pb[nb][sub][1] = pt_transpose(pt_pack(x[2], x[3]));
        }
      if (!S::kJoint && !arrived(stage * 2 + 1)) break;
      if (now != kAll) {  // keys that do not exist multiply zeros
        if (lane < S::kKeys && !(now >> lane & 1u))
#pragma unroll
          for (int c = 0; c < S::kLines; ++c)
#pragma unroll
            for (int i = 0; i < S::kLine; i += 16)
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vblock + (c * S::kKeys + lane) * S::kLine + i),
                           "r"(0u)
                           : "memory");
        fence_proxy_async_smem();  // (the slot's next copy is ordered after these stores)
        __syncwarp();
      }
      // An infinity or NaN among values that some row does not see would reach it as 0 * inf.  Such a
      // block (only where tokens of one draft see different keys) multiplies zeros in their place;
      // the rows that do see them get them after the loop.
      if (p.seq.T > 1 && is_edge(j0)) {
        bool odd = false;
#pragma unroll 1
        for (int q = lane * 8; q < S::kKeys * S::kRow; q += 256) {
          const uint32_t a = vblock + q;
          uint32_t x[2];
          pt_lds2(x[0], x[1], a);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t mask = F8 ? __vcmpeq4(x[c] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) : __vcmpeq2(x[c] & 0x7F807F80u, 0x7F807F80u);
            odd |= mask != 0;
            x[c] &= ~mask;
          }
          if (odd) asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(x[0]), "r"(x[1]) : "memory");
        }
        fence_proxy_async_smem();
        poison |= __any_sync(0xFFFFFFFFu, odd);
        __syncwarp();
      }
      // O^T += V^T P^T
#pragma unroll
      for (int sub = 0; sub < kSub; ++sub)
#pragma unroll
        for (int i = 0; i < S::kVLoads; ++i) {
          uint32_t v[4][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t a = vblock + (e & 1 ? vlane1 : vlane0) + ((e >> 1) * 8 + 16 * sub + i * S::kKeys) * S::kLine;
            if (S::kVBytes == 16) pt_lds4(v[e], a);
            else pt_lds2(v[e][0], v[e][1], a);
          }
#pragma unroll
          for (int c = 0; c < S::kVBytes / 4; ++c) {
            if (F8) {
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                uint32_t a0, a1, a2, a3;
                pt_cvt_e4m3(a0, a1, __byte_perm(v[0][c], v[1][c], hf ? 0x7362 : 0x5140));
                pt_cvt_e4m3(a2, a3, __byte_perm(v[2][c], v[3][c], hf ? 0x7362 : 0x5140));
                const int q = F8 ? 2 * (i * (S::kVBytes / 4) + c) + hf : 0;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) pt_mma(o[nb][q], a0, a1, a2, a3, pb[nb][sub][0], pb[nb][sub][1]);
              }
            } else {
              const uint32_t a0 = __byte_perm(v[0][c], v[1][c], 0x5410), a1 = __byte_perm(v[0][c], v[1][c], 0x7632),
                             a2 = __byte_perm(v[2][c], v[3][c], 0x5410), a3 = __byte_perm(v[2][c], v[3][c], 0x7632);
              const int q = F8 ? 0 : 4 * i + c;
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) pt_mma(o[nb][q], a0, a1, a2, a3, pb[nb][sub][0], pb[nb][sub][1]);
            }
          }
        }
      if (n + kStages < nblk) copy(stage, S::kJoint ? 2 : 1, have_next);
#pragma unroll
      for (int st = 0; st + 1 < kStages; ++st) have[st] = have[st + 1];
      have[kStages - 1] = have_next;
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    if (pending) {  // gave up: no copy may land after the CTA has left (bounded again)
      const uint64_t since = globaltimer_ns();
      for (int bit = 0; bit < 2 * kStages; ++bit)
        while ((pending >> bit & 1u) && !mbar_try_wait(bar0 + bit * 8, parity >> bit & 1u) &&
               globaltimer_ns() - since < SKINNY_WAIT_NS) {
        }
    }

    // ---- the warps' results: (maximum, sum) and O to shared memory, joined row by row
    __syncwarp();  // the ring's slots have been read
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
        float* const dst = so + r * S::kORow;
#pragma unroll
        for (int q = 0; q < S::kTiles; q += 2) {  // two tiles: 4 consecutive dims
          constexpr int per = S::kElems / 2;
          *reinterpret_cast<float4*>(dst + (q / per) * 8 * S::kElems + g * S::kElems + 2 * (q % per)) =
              make_float4(o[nb][q][e], o[nb][q][2 + e], o[nb][q + 1][e], o[nb][q + 1][2 + e]);
        }
      }
    if (poison) {  // the infinities and NaN that were left out, to the rows that see them
      __syncwarp();
#pragma unroll 1
      for (int n = 0; n < nblk; ++n) {
        const int j0 = first_key(n);
#pragma unroll 1
        for (int j = j0; is_edge(j0) && j < min(j0 + S::kKeys, k1); ++j) {
          const int pid = table[j / p.seq.page];
          if (j < sp.beg || pid < 0 || pid >= p.seq.n_pages) continue;
          const size_t where = pid * static_cast<size_t>(p.vps) + (static_cast<size_t>(kvh) * p.seq.page + j % p.seq.page) * D;
#pragma unroll 1
          for (int d = lane; d < D; d += 32) {
            float v;
            if (F8) {
              __nv_fp8_e4m3 x;
              x.__x = static_cast<const uint8_t*>(p.vp)[where + d];
              v = static_cast<float>(x);
            } else {
              v = __bfloat162float(static_cast<const __nv_bfloat16*>(p.vp)[where + d]);
            }
            if (!isfinite(v))
#pragma unroll 1
              for (int r = 0; r < 8 * NB; ++r)
                if (sees(plan.token(r0 + r), j)) so[r * S::kORow + d] += v;
          }
        }
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == sp.tiles;
    const size_t piece = 2 * static_cast<size_t>(blockIdx.x) + (seg > 0);
    const int live = min(plan.rows, sp.cnt * rep - rbase);  // rows of the group that exist
    // warp w finishes rows w, w + 4, ...: lane i first works out the weights of row w + 4 i
    float f[kPtWarps], inv = 0.f;
    int out_row = 0;
    {
      const int r = min(warp + kPtWarps * lane, plan.rows - 1), c = r / (8 * NB), rr = r % (8 * NB);
      float mx = kPtNothing, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kPtWarps; ++w)
        if (w < slots) mx = fmaxf(mx, sml[c + w * plan.nchunk][rr][0]);
#pragma unroll
      for (int w = 0; w < kPtWarps; ++w) {
        f[w] = 0.f;
        if (w < slots) {
          f[w] = pt_exp2(sml[c + w * plan.nchunk][rr][0] - mx);
          sum = fmaf(f[w], sml[c + w * plan.nchunk][rr][1], sum);
        }
      }
      const int t = plan.token(rbase + r), h = kvh * rep + (rbase + r - t * rep);
      out_row = (cur * p.seq.T + t) * p.Hq + h;
      inv = sum == 0.f ? 0.f : (F8 ? p.v_scale[kvh] : 1.f) / sum;
      if (warp + kPtWarps * lane < live) {
        if (!whole) *reinterpret_cast<float2*>(plan.ml + (piece * plan.rows + r) * 2) = make_float2(mx, sum);
        else if (p.lse) p.lse[out_row] = (mx + log2f(sum)) * 0.6931471805599453f;
      }
    }
#pragma unroll 2
    for (int i = 0; warp + kPtWarps * i < live; ++i) {
      const int r = warp + kPtWarps * i, c = r / (8 * NB), rr = r % (8 * NB);
      float fr[kPtWarps];
#pragma unroll
      for (int w = 0; w < kPtWarps; ++w) fr[w] = __shfl_sync(0xFFFFFFFFu, f[w], i);
      const float iv = __shfl_sync(0xFFFFFFFFu, inv, i);
      const size_t row = __shfl_sync(0xFFFFFFFFu, out_row, i);
#pragma unroll
      for (int d = 4 * lane; d < D; d += 128) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f), x[kPtWarps];
#pragma unroll
        for (int w = 0; w < kPtWarps; ++w)  // (together: no branch between the loads)
          x[w] = *reinterpret_cast<const float4*>(pt_smem + (w < slots ? c + w * plan.nchunk : c) * S::kWarpBytes +
                                                  (rr * S::kORow + d) * 4);
#pragma unroll
        for (int w = 0; w < kPtWarps; ++w) {
          const bool on = w < slots;  // (0 times an infinity is not 0)
          acc.x = fmaf(fr[w], on ? x[w].x : 0.f, acc.x);
          acc.y = fmaf(fr[w], on ? x[w].y : 0.f, acc.y);
          acc.z = fmaf(fr[w], on ? x[w].z : 0.f, acc.z);
          acc.w = fmaf(fr[w], on ? x[w].w : 0.f, acc.w);
        }
        if (whole)
          *reinterpret_cast<uint2*>(p.out + row * D + d) =
              make_uint2(pt_pack(acc.x * iv, acc.y * iv), pt_pack(acc.z * iv, acc.w * iv));
        else
          *reinterpret_cast<float4*>(plan.o + (piece * plan.rows + r) * D + d) = acc;
      }
    }
    ++seg;
    // A wait ran out: the results are void, the error word says so.  (The same for every thread: only waits write it,
    // and the next ones lie behind a barrier that all threads reach after this line.)
    if (*static_cast<volatile int*>(&gave_up)) break;
  }
  if (__any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicOr(p.seq.err, kErrBitBadInput);
}

// Joins the pieces of the items that were split and writes the rows that no piece covers (idle slots,
// padding).  plan.join_warps warps per output row: warp w of them adds pieces w, w + join_warps, ... and
// the results are added in order.
constexpr int kPtJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(32 * kPtJoinWarps)
    paged_attn_join_kernel(const __grid_constant__ PagedAttnParams p, const __grid_constant__ PagedAttnPlan plan) {
  constexpr int kPer = D / 32;
  constexpr int kAhead = 4;  // pieces whose loads are issued together
  __shared__ float so[kPtJoinWarps][D], sml[kPtJoinWarps][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, W = plan.join_warps, sub = warp & (W - 1);
  const int rep = p.Hq / p.Hkv;
  const int rows = p.seq.B * p.seq.T * p.Hq, row = blockIdx.x * (kPtJoinWarps / W) + warp / W;
  const int bt = row / p.Hq, h = row - bt * p.Hq, b = bt / p.seq.T, t = bt - b * p.seq.T;
  const int kvh = h / rep, r = t * rep + (h - kvh * rep), group = r / plan.rows, rr = r - group * plan.rows;
  const int item = kvh * plan.groups + group;
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  int first = 0, last = -1;  // the pieces' CTAs
  bool join = false;
  long long beg = 0;
  PtLine line(0, plan.ctas);
  if (row < rows) {
    const long long begins = __ldcg(plan.pre + b), total = __ldcg(plan.pre + p.seq.B);
    const PagedSpan sp = paged_span(p, plan, b);
    if (t >= sp.cnt) {  // padding
      if (lane < D / 8 && sub == 0)
        reinterpret_cast<uint4*>(p.out + static_cast<size_t>(row) * D)[lane] = make_uint4(0u, 0u, 0u, 0u);
      if (lane == 0 && sub == 0 && p.lse) p.lse[row] = -INFINITY;
    } else {
      line = PtLine(total, plan.ctas);
      beg = begins + static_cast<long long>(item) * sp.units;
      first = line.owner(beg + plan.lead);
      last = line.owner(beg + sp.units - 1);
      join = first != last;  // (else one CTA had the whole item)
    }
  }
  const auto piece = [&](int i) {  // where CTA i put this item: in its first piece unless it began another before
    return 2 * static_cast<size_t>(i) + (line.start(i) < beg);
  };
  float m = kPtNothing, l = 0.f, acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  for (int i0 = join ? first + sub : last + 1; i0 <= last; i0 += W * kAhead) {
    float2 ml[kAhead];
    float x[kAhead][kPer];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int i = i0 + a * W;
      ml[a] = make_float2(kPtNothing, 0.f);
#pragma unroll
      for (int q = 0; q < kPer; ++q) x[a][q] = 0.f;
      if (i <= last) {
        const size_t at = piece(i) * plan.rows + rr;
        ml[a] = __ldcg(reinterpret_cast<const float2*>(plan.ml + at * 2));
#pragma unroll
        for (int q = 0; q < kPer; ++q) x[a][q] = __ldcg(plan.o + at * D + lane + 32 * q);
      }
    }
    float mx = m;
#pragma unroll
    for (int a = 0; a < kAhead; ++a) mx = fmaxf(mx, ml[a].x);
    const float f = pt_exp2(m - mx);
    m = mx;
    l *= f;
#pragma unroll
    for (int q = 0; q < kPer; ++q) acc[q] *= f;
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const float w = pt_exp2(ml[a].x - mx);
      l = fmaf(w, ml[a].y, l);
#pragma unroll
      for (int q = 0; q < kPer; ++q) acc[q] = fmaf(w, x[a][q], acc[q]);
    }
  }
  const float vs = p.v_scale ? p.v_scale[kvh] : 1.f;
  if (W > 1) {
#pragma unroll
    for (int q = 0; q < kPer; ++q) so[warp][lane + 32 * q] = acc[q];
    if (lane == 0) {
      sml[warp][0] = m;
      sml[warp][1] = l;
    }
    __syncthreads();
    if (sub != 0) return;
    float mx = m;
    for (int w = 1; w < W; ++w) mx = fmaxf(mx, sml[warp + w][0]);
    const float f0 = pt_exp2(m - mx);
    l *= f0;
#pragma unroll
    for (int q = 0; q < kPer; ++q) acc[q] *= f0;
    for (int w = 1; w < W; ++w) {
      const float f = pt_exp2(sml[warp + w][0] - mx);
      l = fmaf(f, sml[warp + w][1], l);
#pragma unroll
      for (int q = 0; q < kPer; ++q) acc[q] = fmaf(f, so[warp + w][lane + 32 * q], acc[q]);
    }
    m = mx;
  }
  if (!join) return;
  const float inv = l == 0.f ? 0.f : vs / l;
#pragma unroll
  for (int q = 0; q < kPer; ++q)
    p.out[static_cast<size_t>(row) * D + lane + 32 * q] = __float2bfloat16_rn(acc[q] * inv);
  if (lane == 0 && p.lse) p.lse[row] = (m + log2f(l)) * 0.6931471805599453f;
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
cudaError_t pt_encode(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
                      const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> cached{nullptr};
  Encode encode = cached.load(std::memory_order_acquire);
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess) return e;
    if (!fn || found != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
    encode = reinterpret_cast<Encode>(fn);
    cached.store(encode, std::memory_order_release);
  }
  const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode(map, type, static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims, strides, box, steps,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// A pool as [line of 128 bytes][row of D elements][element], to be read in boxes of `lines` lines x `box` rows.
cudaError_t pt_map(CUtensorMap* map, const void* pool, long long page_stride, const PagedAttnParams& p, int es, int line,
                   int box, int lines) {
  const cuuint32_t elems = static_cast<cuuint32_t>(line / es);
  const cuuint64_t dims[3] = {elems, pt_rows(page_stride, p), static_cast<cuuint64_t>(p.D) / elems};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(p.D) * es, static_cast<cuuint64_t>(line)};
  const cuuint32_t boxes[3] = {elems, static_cast<cuuint32_t>(box), static_cast<cuuint32_t>(lines)};
  return pt_encode(map, es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, pool, dims, strides,
                   boxes, line == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

namespace {

struct PtChoice {
  int nb, nchunk, groups, rows, tile_log, ctas_per_sm;
  bool tc;  // the tensor-memory kernel
};

template <int D, int NB, bool F8>
PtChoice pt_sizes() {
  using S = PtShape<D, NB, F8>;
  return {NB, 1, 1, 8 * NB, S::kKeys == 32 ? 7 : 6, S::kCtas, false};
}

// As many 8-row blocks per warp as there are, up to what the registers hold; then one chunk of rows
// per warp (the chunks read the same keys), then several row groups.
template <int D, bool F8>
PtChoice pt_choose(int T, int Hq, int Hkv) {
  constexpr int most = PtShape<D, 1, F8>::kMaxNB;
  const int blocks = (T * (Hq / Hkv) + 7) / 8;
  const int nb = std::min(most, blocks >= 3 ? 4 : blocks);
  PtChoice c = nb == 4 ? pt_sizes<D, 4, F8>() : nb == 2 ? pt_sizes<D, 2, F8>() : pt_sizes<D, 1, F8>();
  const int chunks = (blocks + nb - 1) / nb;
  c.nchunk = chunks >= 3 ? 4 : chunks;
  c.groups = (chunks + c.nchunk - 1) / c.nchunk;
  c.rows = 8 * nb * c.nchunk;
  return c;
}

// More than 32 rows of bf16 pages (16 of heads of 256) go to the tensor-memory kernel, where its copies can be whole
// rows of 8 keys (`eights`): 128 rows of 16 K contexts 48 us against 104, 64 rows of 4 K contexts 28 against 41, 40
// rows 27 against 38, 64 rows of one context of 2 K 16 against 18; heads of 256, 4 K contexts: 64 rows 46 against 97,
// 20 rows 40 against 56.  With fewer the warps' matrix instructions do as well and begin sooner (32 rows of 8
// sequences of 4 K: 27.5 us against 27, a call alone 33 against 39; heads of 256, 16 rows: 39 against 42), and copies
// of single keys would take the other longer (32 rows, pages of 7: 315 us against 117).
PtChoice pt_choose(int T, int Hq, int Hkv, int D, bool f8, bool eights) {
  const int rows = T * (Hq / Hkv);
  if (!f8 && eights && rows > (D == 256 ? 16 : 32)) {
    const int chunks = (rows + 31) / 32, nchunk = chunks > 2 ? 4 : 2;
    return {4, nchunk, (chunks + nchunk - 1) / nchunk, 32 * nchunk, D == 256 ? 6 : 7, 1, true};
  }
  if (D == 64) return f8 ? pt_choose<64, true>(T, Hq, Hkv) : pt_choose<64, false>(T, Hq, Hkv);
  if (D == 128) return f8 ? pt_choose<128, true>(T, Hq, Hkv) : pt_choose<128, false>(T, Hq, Hkv);
  return f8 ? pt_choose<256, true>(T, Hq, Hkv) : pt_choose<256, false>(T, Hq, Hkv);
}

size_t pt_round(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

template <int D, int NB, bool F8>
cudaError_t pt_split(const PagedAttnParams& p, const PagedAttnPlan& plan, int dev, cudaLaunchConfig_t cfg) {
  using S = PtShape<D, NB, F8>;
  static std::atomic<bool> attr_set[64];
  const auto kernel = paged_attn_split_kernel<D, NB, F8>;
  constexpr int smem = PtShape<D, NB, F8>::kSmem;
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    attr_set[dev].store(true, std::memory_order_release);
  }
  CUtensorMap kmap, vmap;
  const int lines = plan.box == S::kKeys ? S::kLines : 1;
  cudaError_t e = pt_map(&kmap, p.kp, p.kps, p, S::kEs, S::kLine, plan.box, lines);
  if (e == cudaSuccess) e = pt_map(&vmap, p.vp, p.vps, p, S::kEs, S::kLine, plan.box, lines);
  if (e != cudaSuccess) return e;
  cfg.dynamicSmemBytes = smem;
  // Not a dependent launch: its CTAs would be placed around those of the kernel before, unevenly, for
  // their whole run (long context 183 us, else 170).
  cfg.numAttrs = 0;
  return cudaLaunchKernelEx(&cfg, kernel, p, plan, kmap, vmap);
}

template <int D>
cudaError_t pt_launch(const PagedAttnParams& p, const PagedAttnPlan& plan, int nb, bool tc, bool f8, int dev,
                      cudaLaunchConfig_t cfg) {
  cudaError_t e = cudaErrorInvalidValue;
  if (tc) {
    e = paged_attn_tc_split(p, plan, dev, cfg);
  } else if (nb == 1) {
    e = f8 ? pt_split<D, 1, true>(p, plan, dev, cfg) : pt_split<D, 1, false>(p, plan, dev, cfg);
  } else if constexpr (D <= 128) {
    if (nb == 2) e = f8 ? pt_split<D, 2, true>(p, plan, dev, cfg) : pt_split<D, 2, false>(p, plan, dev, cfg);
    if (nb == 4) e = f8 ? pt_split<D, 4, true>(p, plan, dev, cfg) : pt_split<D, 4, false>(p, plan, dev, cfg);
  } else {
    if (nb == 2 && f8) e = pt_split<D, 2, true>(p, plan, dev, cfg);
  }
  if (e != cudaSuccess) return e;
  const long long rows = static_cast<long long>(p.seq.B) * p.seq.T * p.Hq;
  cfg.gridDim = dim3(static_cast<unsigned>((rows * plan.join_warps + kPtJoinWarps - 1) / kPtJoinWarps));
  cfg.blockDim = dim3(32 * kPtJoinWarps);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<D>, p, plan);
}

}  // namespace

size_t paged_attn_ws_bytes(int B, int T, int Hq, int Hkv, int D, int n_sm) {
  size_t most = 0;
  for (int i = 0; i < 3; ++i) {
    const PtChoice c = pt_choose(T, Hq, Hkv, D, i == 2, i == 1);
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
  const bool eights = p.seq.page % 8 == 0 && p.kps / p.D % 8 == 0 && p.vps / p.D % 8 == 0;
  const PtChoice c = pt_choose(p.seq.T, p.Hq, p.Hkv, p.D, f8, eights);
  PagedAttnPlan plan;
  plan.tile_log = c.tile_log;
  plan.lead = kPtLead;
  plan.shift = -1;
  for (int i = 0; i < 31; ++i)
    if (p.seq.page == 1 << i) plan.shift = i;
  plan.box = c.tc ? 32 : 1 << (c.tile_log - 2);  // a block's keys
  while (p.seq.page % plan.box) plan.box /= 2;
  const uint32_t rep = static_cast<uint32_t>(p.Hq / p.Hkv);
  plan.rep_inv = rep == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + rep - 1) / rep);
  // Few rows are split among many CTAs each: up to 8 warps per row while all are on the GPU at once.
  const long long out_rows = static_cast<long long>(p.seq.B) * p.seq.T * p.Hq;
  plan.join_warps = kPtJoinWarps;
  while (plan.join_warps > 1 && out_rows * plan.join_warps > 32ll * n_sm) plan.join_warps /= 2;
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
  if (p.D == 64) return pt_launch<64>(p, plan, c.nb, c.tc, f8, dev, cfg);
  if (p.D == 128) return pt_launch<128>(p, plan, c.nb, c.tc, f8, dev, cfg);
  return pt_launch<256>(p, plan, c.nb, c.tc, f8, dev, cfg);
}

}  // namespace skinny
