// Paged attention of many query rows (tokens x heads of a kv head) on the tensor-memory matrix units: the split
// launch for bf16 pages whose items have many rows (the rule is pt_choose's); the line, its pieces and the join are
// those of paged_attn.cu.
//
// A tile is 128 keys (64 of heads of 256).  S = q K^T has the query rows in the 128 lanes of tensor memory and
// the keys in its columns, so a thread owns a row: its maximum, its sum and its part of O need no exchange.  q and P are
// operands in tensor memory, K (rows of D) and V (D in the other direction) come by TMA into a ring in shared
// memory and are read there as they lie.  With 64 rows per item the rows are repeated in both halves of the
// lanes, each of which exponentiates half of a tile's keys and multiplies zeros for the others: every warp has
// the same work, and the halves' O are joined at the item's end.  The matrix unit then repeats itself, which
// costs nothing: a tile of 128 keys takes it some 1600 clocks, the memory 2700 (64 KB at 1/148 of the copy
// bandwidth).  Measured per call of back-to-back graph replays: two sequences of 100 K and 64 rows 79 us (79 % of the
// copy bandwidth), four of 16 K and 128 rows 48 us (exponentials and the row maximum, some 2000 clocks a tile in one
// warp per scheduler; a CTA's beginning and end, some 10 us, weigh on shorter ones: eight of 4 K and 64 rows 28 us).
//
// Seven warps: four of softmax, one that issues the matrix instructions, one that copies keys, one values.
// S(n + 2) follows O += P(n) V(n), while the softmax works on S(n + 1).  The maximum of a row is renewed only when a
// score exceeds it by more than 8 (in powers of two), and only then O is read back and rescaled.
// Roundings as in paged_attn.cu: p to bf16, all else f32.
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "paged.cuh"
#include "paged_attn.cuh"
#include "ptx.cuh"

namespace skinny {

constexpr int kTcThreads = 224;
constexpr int kTcRingBytes = 163840;
constexpr int kTcInfo = 8;           // tiles whose flags are kept: keys are asked for at most 8 tiles ahead of the softmax
constexpr int kTcHalf = 64;          // dims of O that pass through shared memory at a time
constexpr int kTcORow = kTcHalf + 4;

template <int D>
struct TcShape {
  static constexpr int kKeys = D == 256 ? 64 : 128;         // of one tile
  static constexpr int kWords = kKeys / 32;
  static constexpr int kSlot = kKeys * D * 2;               // keys or values of a tile
  // Slots of the ring.  Keys are multiplied two tiles ahead and their slots freed; values stay until their P is there
  // (3 and 2: 84 us for two sequences of 100 K and 64 rows, 2 and 3: 79).
  static constexpr int kKSlots = D == 64 ? 5 : 2, kVSlots = D == 64 ? 5 : 3;
  static constexpr int kLines = D / 64;                     // lines of 128 bytes of a row: [key / 8][line][key % 8][128 B]
  static constexpr int kEight = 1024 * kLines;              // bytes of 8 keys
  static constexpr int kSmem = 1024 + kTcRingBytes + 128 * kTcORow * 4;
  // Columns of tensor memory: S (two tiles), O, q, P.  Heads of 256 fill it without P, which takes the place of its
  // S then (and S(n + 2) waits for P(n) V(n)).
  static constexpr bool kOver = D == 256;
  static constexpr uint32_t kS = 0, kO = 2 * kKeys, kQ = 384, kP = 448, kCols = 512;
  static_assert(kO + D <= kQ && kQ + D / 2 <= (kOver ? 512 : kP), "tensor memory");
  __device__ static __forceinline__ uint32_t p_col(int g) { return kOver ? kS + (g & 1) * kKeys : kP; }
};

struct TcShared {
  uint64_t full[10], empty[10];  // per slot of the ring: a tile is there, has been used
  uint64_t info[kTcInfo];    // a tile's `have` is written
  uint64_t s_full[2];        // S(n) is there
  uint64_t p_full;           // P(n) is there, O may be added to
  uint64_t pv_done;          // O has P(n) V(n)
  uint64_t q_full;           // a part's q is there
  uint64_t drain;
  alignas(16) uint32_t have[kTcInfo][4]; // the keys of a tile that exist
  uint32_t rows[2][128];     // the copying warps' own: where a tile's keys (values) lie
  float ml[128][2];          // per lane: maximum and sum
  float weight[4][128];      // per lane group and row: what its O counts
  float inv[128];
  int row_out[128];
  long long scan[kTcThreads / 32], found[2];
  uint32_t tmem;
  int gave_up;
  int poison;  // the last part whose values had infinities or NaN set to 0
  int stop[2];  // of a part (by its parity): leave behind it
};

// Operand B from a slot of the ring.  Keys as N (rows of 64 dims, the K direction contiguous): 8 keys are `eight`
// bytes further; the first stride is not used.  Values with N, the dims, contiguous: the next 64 dims are 1024
// bytes further, the next 8 keys `eight`.
__device__ __forceinline__ uint64_t tc_desc(uint32_t saddr, uint32_t eight) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>(1024 >> 4) << 16;
  d |= static_cast<uint64_t>(eight >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;  // 128-byte swizzle
  return d;
}

__device__ __forceinline__ void tc_softmax_barrier() {  // of the softmax warps, each whole behind it
  __syncwarp();
  asm volatile("bar.sync 1, 128;" ::: "memory");
  __syncwarp();
}

__device__ __forceinline__ void tc_lds4(uint32_t (&x)[4], uint32_t a) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(a) : "memory");
}

__device__ __forceinline__ void tc_store(uint32_t taddr, const uint32_t (&v)[16]) { tmem_st_x16(taddr, v); }
__device__ __forceinline__ void tc_store(uint32_t taddr, const uint32_t (&v)[32]) { tmem_st_x32(taddr, v); }

template <int N>
__device__ __forceinline__ void tc_load(uint32_t taddr, float (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 16) {
    float x[16];
    tmem_ld<16>(taddr + i, x);
#pragma unroll
    for (int e = 0; e < 16; ++e) s[i + e] = x[e];
  }
}

template <int D, int NC>
__global__ void __launch_bounds__(kTcThreads, 1)
    paged_attn_tc_kernel(const __grid_constant__ PagedAttnParams p, const __grid_constant__ PagedAttnPlan plan,
                         const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using S = TcShape<D>;
  // lane groups with the same rows, and the keys of a tile that each has
  constexpr int kKeys = S::kKeys, kSlots = 4 / NC, kCols = kKeys / kSlots;
  extern __shared__ __align__(1024) uint8_t tc_raw[];
  uint8_t* const smem = tc_raw + ((1024 - (smem_u32(tc_raw) & 1023)) & 1023);
  __shared__ TcShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rep = p.Hq / p.Hkv, items = p.Hkv * plan.groups;
  const uint32_t ring = smem_u32(smem);
  float* const so = reinterpret_cast<float*>(smem + kTcRingBytes);
  if (tid == 0) {
    for (int i = 0; i < S::kKSlots + S::kVSlots; ++i) {
      mbar_init(smem_u32(&sh.full[i]), 1);
      mbar_init(smem_u32(&sh.empty[i]), 1);
    }
    for (int i = 0; i < kTcInfo; ++i) mbar_init(smem_u32(&sh.info[i]), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&sh.s_full[i]), 1);
    mbar_init(smem_u32(&sh.p_full), 128);
    mbar_init(smem_u32(&sh.pv_done), 1);
    mbar_init(smem_u32(&sh.q_full), 128);
    mbar_init(smem_u32(&sh.drain), 1);
    sh.gave_up = 0;
    sh.poison = -1;
    fence_mbar_init();
  }
  if (warp >= 5) prefetch_tmap(warp == 5 ? &kmap : &vmap);
  pdl_wait_prior_grid();
  if (warp == 4) {
    tmem_alloc(smem_u32(&sh.tmem), S::kCols);
    tmem_relinquish();
  }
  PtWalk walk;
  const bool some = pt_begin<kTcThreads>(p, plan, items, sh.scan, sh.found, walk);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Only now: a kernel further down the stream may want tensor memory too, before it waits for this one.
  pdl_launch_dependents();
  const uint32_t tmem = sh.tmem;
  if (!some) {
    if (warp == 4) tmem_dealloc(tmem, S::kCols);
    return;
  }
  // bounded waits of a whole warp: the same answer in every lane
  const auto wait = [&](const uint64_t& bar, uint32_t parity) {
    const bool ok = mbar_wait(smem_u32(&bar), parity & 1u, p.seq.err, kErrBitWaitFull, &sh.gave_up);
    const bool all = __all_sync(0xFFFFFFFFu, ok) != 0;
    __syncwarp();
    return all;
  };
  // tile g's keys (values): their slot, and how often it has been used before
  const auto k_slot = [](int g) { return g % S::kKSlots; };
  const auto v_slot = [](int g) { return S::kKSlots + g % S::kVSlots; };
  const auto k_turn = [](int g) { return g / S::kKSlots; };
  const auto v_turn = [](int g) { return g / S::kVSlots; };
  PtPart part;

  if (warp >= 5) {
    // ---- copies: every tile's keys (one warp) and values (the other), as slots become free
    const int kv = warp - 5;
    const uint32_t per = static_cast<uint32_t>((kv ? p.vps : p.kps) / D);  // rows of D from page to page
    const CUtensorMap* const map = kv ? &vmap : &kmap;
    const int boxes = 32 / plan.box;  // of a row of 32 keys
    const uint32_t mask = plan.box == 32 ? 0xFFFFFFFFu : (1u << plan.box) - 1u;
    bool ok = true, bad = false;
    int tile = 0;
    while (ok && walk.next(p, plan, items, part)) {
      const PagedSpan sp = part.sp;
      const uint32_t head = static_cast<uint32_t>(part.item / plan.groups) * p.seq.page;
      const int nt = part.t1 - part.t0;
      const int k0 = sp.first + (part.t0 << plan.tile_log), k1 = min(sp.end, sp.first + (part.t1 << plan.tile_log));
      const int32_t* const table = p.seq.table + part.seq * p.seq.table_stride;
      int pid[S::kWords], in_page[S::kWords];
      const auto look = [&](int n) {  // tile n's pages, one key per lane and 32 keys
#pragma unroll
        for (int w = 0; w < S::kWords; ++w) {
          const int j = k0 + kKeys * n + 32 * w + lane;
          pid[w] = -2;
          in_page[w] = 0;
          if (n < nt && j >= sp.beg && j < k1) {
            const int q = plan.shift >= 0 ? j >> plan.shift : j / p.seq.page;
            in_page[w] = j - q * p.seq.page;
            pid[w] = __ldg(table + q);
          }
        }
      };
      look(0);
      for (int n = 0; n < nt; ++n, ++tile) {
        uint32_t ex[4] = {0u, 0u, 0u, 0u};
        __syncwarp();  // (the rows of the tile before have been read)
        int there = 0;  // boxes with a key that exists
#pragma unroll
        for (int w = 0; w < S::kWords; ++w) {
          const bool here = pid[w] >= 0 && pid[w] < p.seq.n_pages;
          bad |= !here && pid[w] != -2;
          sh.rows[kv][32 * w + lane] = static_cast<uint32_t>(pid[w]) * per + head + static_cast<uint32_t>(in_page[w]);
          ex[w] = __ballot_sync(0xFFFFFFFFu, here);
          there += __popc(__ballot_sync(0xFFFFFFFFu, lane < boxes && (ex[w] >> (lane * plan.box) & mask)));
        }
        look(n + 1);
        const int slot = kv ? v_slot(tile) : k_slot(tile), turn = kv ? v_turn(tile) : k_turn(tile);
        ok = turn == 0 || wait(sh.empty[slot], turn - 1);
        if (!ok) break;
        if (kv == 0 && lane < 4) sh.have[tile % kTcInfo][lane] = lane < 2 ? (lane ? ex[1] : ex[0]) : (lane == 2 ? ex[2] : ex[3]);
        __syncwarp();
        if (kv == 0 && lane == 0) mbar_arrive(smem_u32(&sh.info[tile % kTcInfo]));
        const uint32_t bar = smem_u32(&sh.full[slot]), dst = ring + slot * S::kSlot;
        if (lane == 0) mbar_arrive_expect_tx(bar, there * plan.box * 2 * D);
        __syncwarp();
        if (lane < S::kWords * boxes) {  // one copy per lane
          const int w = lane / boxes, first = (lane & (boxes - 1)) * plan.box;
          const uint32_t here = (w == 0 ? ex[0] : w == 1 ? ex[1] : w == 2 ? ex[2] : ex[3]) & mask << first;
          if (here) {
            const int src = __ffs(here) - 1;
            const int row = static_cast<int>(sh.rows[kv][32 * w + src] - static_cast<uint32_t>(src - first));
            tma_load_4d(dst + (4 * w + (first >> 3)) * S::kEight, map, 0, 0, 0, row >> 3, bar);
          }
        }
      }
    }
    if (__any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicOr(p.seq.err, kErrBitBadInput);
    // no copy may land after the CTA has left (they have all been waited for unless a wait ran out)
    const uint64_t since = globaltimer_ns();
    for (int n = max(0, tile - (kv ? S::kVSlots : S::kKSlots)); n < tile; ++n)
      while (!mbar_try_wait(smem_u32(&sh.full[kv ? v_slot(n) : k_slot(n)]), (kv ? v_turn(n) : k_turn(n)) & 1) &&
             globaltimer_ns() - since < SKINNY_WAIT_NS) {
      }
  } else if (warp == 4) {
    // ---- matrix instructions, issued by lane 0
    constexpr uint32_t kIdescS = idesc_bf16_f32(128, kKeys);
    constexpr uint32_t kIdescO = idesc_bf16_f32(128, D) | 1u << 16;  // (B's N direction is the contiguous one)
    bool ok = true;
    int tile = 0, seg = 0;
    const auto scores = [&](int g) {
      const int slot = k_slot(g);
      if (!wait(sh.full[slot], k_turn(g))) return false;
      tc_fence_after();
      if (lane == 0) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16_ts(tmem + S::kS + (g & 1) * kKeys, tmem + S::kQ + k * 8,
                      tc_desc(ring + slot * S::kSlot + (k / 4) * 1024 + (k % 4) * 32, S::kEight), kIdescS, k > 0);
        umma_commit(smem_u32(&sh.empty[slot]));
        umma_commit(smem_u32(&sh.s_full[g & 1]));
      }
      __syncwarp();
      return true;
    };
    while (ok && walk.next(p, plan, items, part)) {
      const int nt = part.t1 - part.t0;
      ok = wait(sh.q_full, seg);
      tc_fence_after();
      ok = ok && scores(tile);
      if (nt > 1) ok = ok && scores(tile + 1);
      for (int n = 0; ok && n < nt; ++n) {
        const int g = tile + n, slot = v_slot(g);
        ok = wait(sh.p_full, g) && wait(sh.full[slot], v_turn(g));
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            umma_f16_ts(tmem + S::kO, tmem + S::p_col(g) + k * 8,
                        tc_desc(ring + slot * S::kSlot + k * 2 * S::kEight, S::kEight), kIdescO, n > 0 || k > 0);
          umma_commit(smem_u32(&sh.empty[slot]));
          umma_commit(smem_u32(&sh.pv_done));
        }
        __syncwarp();
        // (every thread has read S(n): it brought P(n))
        if (n + 2 < nt) ok = (!S::kOver || wait(sh.pv_done, g)) && scores(g + 2);
      }
      tile += nt;
      ++seg;
    }
    // nothing of it may run after the tensor memory is given back
    if (lane == 0) umma_commit(smem_u32(&sh.drain));
    __syncwarp();
    const uint64_t since = globaltimer_ns();
    while (!mbar_try_wait(smem_u32(&sh.drain), 0) && globaltimer_ns() - since < SKINNY_WAIT_NS) {
    }
  } else {
    // ---- softmax: lane group `warp` has rows 32 chunk .. of the part, and its share of a tile's keys
    const int chunk = warp % NC, slot = warp / NC;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp) << 21);
    // to powers of two by a positive factor (a masked score stays -inf): q takes a negative scale's sign, and a
    // scale of 0 makes it 0
    const float sc = p.scale == 0.f ? 1.f : fabsf(p.scale) * 1.4426950408889634f;
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
    const uint32_t zeros[16] = {};
    const auto others = [&](int g) {  // zeros for the other half's keys
      if (kSlots > 1)
#pragma unroll
        for (int c = 0; c < kCols / 2; c += 16) tmem_st_x16(lanes + S::p_col(g) + (1 - slot) * (kCols / 2) + c, zeros);
    };
    if (!S::kOver) others(0);  // (they stay)
    int tile = 0;
    for (int seg = 0; walk.next(p, plan, items, part); ++seg) {
      const PagedSpan sp = part.sp;
      const int nt = part.t1 - part.t0, kvh = part.item / plan.groups, rbase = (part.item % plan.groups) * plan.rows;
      const int k0 = sp.first + (part.t0 << plan.tile_log), k1 = min(sp.end, sp.first + (part.t1 << plan.tile_log));
      const int r0 = rbase + 32 * chunk, r = r0 + lane, t = plan.token(r), h = kvh * rep + (r - t * rep);
      {
        const uint4* const src = reinterpret_cast<const uint4*>(p.q + part.seq * p.qs[0] + t * p.qs[1] + h * p.qs[2]);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          uint32_t x[32];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint4 w = t < sp.cnt && p.scale != 0.f ? __ldg(src + 8 * i + e) : make_uint4(0u, 0u, 0u, 0u);
            x[4 * e] = w.x ^ flip;
            x[4 * e + 1] = w.y ^ flip;
            x[4 * e + 2] = w.z ^ flip;
            x[4 * e + 3] = w.w ^ flip;
          }
          __syncwarp();
          tmem_st_x32(lanes + S::kQ + 32 * i, x);
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&sh.q_full));
      }
      const int last = sp.len + t, least = p.window > 0 ? last - p.window + 1 : 0;  // the positions this row sees
      const auto is_edge = [&](int j0) {  // a tile that some row sees only part of
        return j0 + kKeys - 1 > sp.len || (p.window > 0 && j0 <= sp.len + sp.cnt - 1 - p.window);
      };
      float m = kPtNothing, l = 0.f;
      bool ok = true;
      for (int n = 0; n < nt; ++n) {
        const int g = tile + n, j0 = k0 + kKeys * n;
        ok = wait(sh.s_full[g & 1], g >> 1) && wait(sh.info[g % kTcInfo], g / kTcInfo);
        if (!ok) break;
        tc_fence_after();
        float s[kCols];
        tc_load<kCols>(lanes + S::kS + (g & 1) * kKeys + slot * kCols, s);
        const uint4 have = *reinterpret_cast<const uint4*>(sh.have[g % kTcInfo]);
        const bool whole = (have.x & have.y & (S::kWords == 4 ? have.z & have.w : ~0u)) == ~0u, edge = is_edge(j0);
        // Values of keys that do not exist multiply zeros; so do infinities and NaN where some row must not have them
        // (0 * inf): among values that not every row sees, and with two lane groups anywhere, each of which has
        // zeros for the other's keys.  The rows that do see them get them after the loop.
        const uint32_t key = ring + v_slot(g) * S::kSlot + (tid >> 3) * S::kEight + (tid & 7) * 128;
        bool gone = false, odd = false;
        const auto look = [&]() {  // this thread's key, 16 bytes at a time, no two lanes of eight in one bank
          if (!wait(sh.full[v_slot(g)], v_turn(g))) return false;
          if (warp < S::kWords) {
            gone = !(sh.have[g % kTcInfo][warp] >> lane & 1u);
            const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
            __nv_bfloat162 nan[4] = {zero, zero, zero, zero};  // 0 x: NaN and stays so
#pragma unroll
            for (int c = 0; c < 8 * S::kLines; ++c) {
              uint32_t x[4];
              tc_lds4(x, key + (c >> 3) * 1024 + ((c + lane) & 7) * 16);
#pragma unroll
              for (int e = 0; e < 4; ++e) nan[e] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x[e]), zero, nan[e]);
            }
            const __nv_bfloat162 any = __hadd2(__hadd2(nan[0], nan[1]), __hadd2(nan[2], nan[3]));
            odd = !gone && (__hisnan(any.x) || __hisnan(any.y));
          }
          return true;
        };
        if ((kSlots > 1 || !whole || (p.seq.T > 1 && edge)) && !(ok = look())) break;  // (the scores are on their way)
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < kCols; ++i) asm volatile("" : "+f"(s[i]));  // (nothing of it is used before the wait)
        if (gone || odd) {
#pragma unroll 1
          for (int c = 0; c < 8 * S::kLines; ++c) {
            const uint32_t a = key + (c >> 3) * 1024 + ((c + lane) & 7) * 16;
            uint32_t x[4];
            tc_lds4(x, a);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] &= gone ? 0u : ~__vcmpgeu2(x[e] & 0x7FFF7FFFu, 0x7F807F80u);
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
          }
          fence_proxy_async_smem();
          if (odd) sh.poison = seg;
        }
        __syncwarp();  // (tensor memory is for whole warps)
        if (!whole || edge) {
#pragma unroll
          for (int i = 0; i < kCols; ++i) {
            const uint32_t word = sh.have[g % kTcInfo][slot * (kCols / 32) + i / 32];
            const int j = j0 + slot * kCols + i;
            if (!(word >> (i & 31) & 1u) || j > last || j < least) s[i] = -INFINITY;
          }
        }
        float tops[4] = {s[0], s[1], s[2], s[3]};  // (chains: one warp of this kind per scheduler)
#pragma unroll
        for (int i = 4; i < kCols; ++i) tops[i & 3] = fmaxf(tops[i & 3], s[i]);
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * sc;
        if (__any_sync(0xFFFFFFFFu, top > m + 8.f)) {  // renew the maxima, rescale the sums
          const float x = fmaxf(m, top), f = pt_exp2(m - x);
          m = x;
          l *= f;
          if (n > 0) {
            ok = wait(sh.pv_done, g - 1);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float o[16];
              uint32_t y[16];
              tmem_ld<16>(lanes + S::kO + c, o);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(o[e] * f);
              tmem_st_x16(lanes + S::kO + c, y);
            }
          }
        }
        uint32_t pk[kCols / 2];
        const uint64_t sc2 = f2_pack(sc, sc), m2 = f2_pack(-m, -m), one = f2_pack(1.f, 1.f);
        uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < kCols; i += 2) {
          float a, b;
          f2_unpack(f2_fma(f2_pack(s[i], s[i + 1]), sc2, m2), a, b);
          a = pt_exp2(a);
          b = pt_exp2(b);
          sum[i / 2 & 1] = f2_fma(f2_pack(a, b), one, sum[i / 2 & 1]);
          pk[i / 2] = pt_pack(a, b);
        }
        {
          float a, b, c, d;
          f2_unpack(sum[0], a, b);
          f2_unpack(sum[1], c, d);
          l += (a + b) + (c + d);
        }
        if (n > 0) {  // P(n - 1) has been used (and this warp cannot arrive twice at one turn of p_full)
          ok = wait(sh.pv_done, g - 1);
          if (!ok) break;
          tc_fence_after();
        }
        if (S::kOver) others(g);
        constexpr int kStore = kCols / 2 < 32 ? 16 : 32;
#pragma unroll
        for (int c = 0; c < kCols / 2; c += kStore) {
          uint32_t y[kStore];
#pragma unroll
          for (int e = 0; e < kStore; ++e) y[e] = pk[c + e];
          tc_store(lanes + S::p_col(g) + slot * (kCols / 2) + c, y);
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&sh.p_full));
      }
      tile += nt;

      // ---- the lane groups' results, joined row by row, half of O's dims at a time
      ok = ok && wait(sh.pv_done, tile - 1);
      tc_fence_after();
      const bool entire = part.t0 == 0 && part.t1 == sp.tiles;
      const size_t piece = 2 * static_cast<size_t>(blockIdx.x) + (seg > 0);
      const int live = min(plan.rows, sp.cnt * rep - rbase);  // rows of the group that exist
      sh.ml[tid][0] = m;
      sh.ml[tid][1] = l;
      if (tid == 0) sh.stop[seg & 1] = *static_cast<volatile int*>(&sh.gave_up);
#pragma unroll 1
      for (int d0 = 0; d0 < D; d0 += kTcHalf) {
        {
          float o[kTcHalf];
          tc_load<kTcHalf>(lanes + S::kO + d0, o);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < kTcHalf; e += 4)
            *reinterpret_cast<float4*>(so + tid * kTcORow + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
        tc_softmax_barrier();
        if (d0 == 0 && tid < 32 * NC) {  // row tid of the group: what the lane groups' parts count
          float mx = kPtNothing, sum = 0.f;
#pragma unroll
          for (int w = 0; w < kSlots; ++w) mx = fmaxf(mx, sh.ml[32 * NC * w + tid][0]);
#pragma unroll
          for (int w = 0; w < kSlots; ++w) {
            const float f = pt_exp2(sh.ml[32 * NC * w + tid][0] - mx);
            sum = fmaf(f, sh.ml[32 * NC * w + tid][1], sum);
            sh.weight[w][tid] = f;
          }
          // (row tid of the group is this thread's own row: slot 0 has the first 32 NC lanes)
          const int at = (part.seq * p.seq.T + t) * p.Hq + h;
          sh.row_out[tid] = at;
          sh.inv[tid] = sum == 0.f ? 0.f : 1.f / sum;
          if (tid < live) {
            if (!entire) *reinterpret_cast<float2*>(plan.ml + (piece * plan.rows + tid) * 2) = make_float2(mx, sum);
            else if (p.lse) p.lse[at] = (mx + log2f(sum)) * 0.6931471805599453f;
          }
        }
        if (sh.poison == seg) {  // the infinities and NaN that were left out, to the rows that see them
          // (of every tile: where none was left out, its infinity or NaN is in O already and once more changes nothing)
          const int32_t* const table = p.seq.table + part.seq * p.seq.table_stride;
#pragma unroll 1
          for (int n = 0; n < nt; ++n) {
            const int j0 = k0 + kKeys * n;
#pragma unroll 1
            for (int j = j0 + slot * kCols; j < min(j0 + (slot + 1) * kCols, k1); ++j) {
              const int pid = table[j / p.seq.page];
              if (j < sp.beg || pid < 0 || pid >= p.seq.n_pages) continue;
              const __nv_bfloat16* const src = static_cast<const __nv_bfloat16*>(p.vp) + pid * static_cast<size_t>(p.vps) +
                                               (static_cast<size_t>(kvh) * p.seq.page + j % p.seq.page) * D + d0;
#pragma unroll 1
              for (int d = lane; d < kTcHalf; d += 32) {
                const float v = __bfloat162float(src[d]);
                if (!isfinite(v))
#pragma unroll 1
                  for (int i = 0; i < 32; ++i) {
                    const int pos = sp.len + plan.token(r0 + i);
                    if (j <= pos && (p.window <= 0 || j > pos - p.window)) so[(32 * warp + i) * kTcORow + d] += v;
                  }
              }
            }
          }
        }
        tc_softmax_barrier();
        const int quad = 4 * (tid & 15);
#pragma unroll 4
        for (int q = tid >> 4; q < live; q += 8) {
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kSlots; ++w) {
            const float f = sh.weight[w][q];
            const float4 x = *reinterpret_cast<const float4*>(so + (32 * NC * w + q) * kTcORow + quad);
            acc.x = fmaf(f, x.x, acc.x);
            acc.y = fmaf(f, x.y, acc.y);
            acc.z = fmaf(f, x.z, acc.z);
            acc.w = fmaf(f, x.w, acc.w);
          }
          if (entire) {
            const float iv = sh.inv[q];
            *reinterpret_cast<uint2*>(p.out + static_cast<size_t>(sh.row_out[q]) * D + d0 + quad) =
                make_uint2(pt_pack(acc.x * iv, acc.y * iv), pt_pack(acc.z * iv, acc.w * iv));
          } else {
            *reinterpret_cast<float4*>(plan.o + (piece * plan.rows + q) * D + d0 + quad) = acc;
          }
        }
        if (d0 + kTcHalf < D) tc_softmax_barrier();
      }
      // (the next part's first O waits for every thread, so `so`, the weights and O are free by then)
      if (sh.stop[seg & 1]) break;  // a wait ran out: the results are void, the error word says so
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 4) tmem_dealloc(tmem, S::kCols);
}

// The pool as [8 positions][line][position][64 dims] (pages and pools consist of eights), to be read in boxes of
// whole rows.
static cudaError_t tc_map(CUtensorMap* map, const void* pool, long long page_stride, const PagedAttnParams& p,
                          int positions) {
  const cuuint64_t rows = pt_rows(page_stride, p);
  const cuuint64_t dims[4] = {64, 8, static_cast<cuuint64_t>(p.D / 64), rows / 8};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(p.D) * 2, 128, static_cast<cuuint64_t>(p.D) * 16};
  const cuuint32_t box[4] = {64, 8, static_cast<cuuint32_t>(p.D / 64), static_cast<cuuint32_t>(positions / 8)};
  return pt_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, pool, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D, int NC>
static cudaError_t tc_split(const PagedAttnParams& p, const PagedAttnPlan& plan, int dev, cudaLaunchConfig_t cfg) {
  using S = TcShape<D>;
  static std::atomic<bool> attr_set[64];
  const auto kernel = paged_attn_tc_kernel<D, NC>;
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    attr_set[dev].store(true, std::memory_order_release);
  }
  CUtensorMap kmap, vmap;
  cudaError_t e = tc_map(&kmap, p.kp, p.kps, p, plan.box);
  if (e == cudaSuccess) e = tc_map(&vmap, p.vp, p.vps, p, plan.box);
  if (e != cudaSuccess) return e;
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = S::kSmem;  // (one CTA per SM: a dependent launch places them evenly)
  return cudaLaunchKernelEx(&cfg, kernel, p, plan, kmap, vmap);
}

cudaError_t paged_attn_tc_split(const PagedAttnParams& p, const PagedAttnPlan& plan, int dev, const cudaLaunchConfig_t& cfg) {
  if (p.D == 64) return plan.nchunk == 2 ? tc_split<64, 2>(p, plan, dev, cfg) : tc_split<64, 4>(p, plan, dev, cfg);
  if (p.D == 128) return plan.nchunk == 2 ? tc_split<128, 2>(p, plan, dev, cfg) : tc_split<128, 4>(p, plan, dev, cfg);
  return plan.nchunk == 2 ? tc_split<256, 2>(p, plan, dev, cfg) : tc_split<256, 4>(p, plan, dev, cfg);
}

}  // namespace skinny
