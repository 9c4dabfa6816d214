// Paged key-value caches: what the append and the attention kernels share.
//
// A pool holds n_pages pages of `page` consecutive positions of ONE sequence: element
// [page id][kv head][slot][dim], so the keys of one head in one page are contiguous.  The rest of a
// page ([kv head][slot][dim]) is dense; pages may be further apart (page_stride elements), e.g. when
// a pool interleaves layers.  Sequence b's position j is slot j % page of page table[b][j / page].
// Elements are bf16, or e4m3 with one f32 scale per kv head (value = stored * scale).
//
// Everything a kernel reads from device memory to form an address is checked there: a sequence whose
// length or count is out of range takes no part in the call, a page id outside the pool is skipped
// (nothing written, its keys not seen); both set kErrBitBadInput in the device's paged error word.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "skinny_status.h"

namespace skinny {

constexpr int kPagedMaxTokens = 16;    // new tokens per sequence of one attention call
constexpr int kPagedMaxBatch = 8192;   // sequences per call
constexpr int kPagedMaxPositions = INT32_MAX - 4095;  // of a row of the table: the tile behind the last is still an int
constexpr int kPagedMaxGroup = 1024;   // query heads per kv head

struct PagedSeqs {
  const int32_t* lengths;  // [B] tokens in the cache before the step
  const int32_t* counts;   // [B] new tokens of the step (0 .. T), or null: T each
  const int32_t* table;    // [B, width] page ids
  long long table_stride;
  int width, page, n_pages, B, T;
  uint32_t* err;           // the device's paged error word (paged_error_word)

  // Length and count of sequence b; false (count 0) when they are out of range.
  __device__ __forceinline__ bool get(int b, int& len, int& cnt) const {
    len = lengths[b];
    cnt = counts ? counts[b] : T;
    const bool ok = len >= 0 && cnt >= 0 && cnt <= T &&
                    static_cast<long long>(len) + cnt <= static_cast<long long>(width) * page;
    if (!ok) len = cnt = 0;
    return ok;
  }
};

struct PagedAppendParams {
  PagedSeqs seq;
  const __nv_bfloat16 *q, *k, *v;  // [B, T, heads, D], element strides (batch, token, head)
  long long qs[3], ks[3], vs[3];
  __nv_bfloat16* q_out;            // [B, T, Hq, D] dense
  void *kp, *vp;
  long long kps, vps;              // page strides in elements
  const float *k_scale, *v_scale;  // [Hkv] (8-bit pages)
  const float* inv_freq;
  int rot, Hq, Hkv, D;
  uint32_t inv_per;                // (set by the launch) pieces per head: see the kernel
  int perv_log;
};

struct PagedAttnParams {
  PagedSeqs seq;
  const __nv_bfloat16* q;
  long long qs[3];                 // q element strides: batch, token, head
  const void *kp, *vp;
  long long kps, vps;              // page strides in elements
  const float *k_scale, *v_scale;  // [Hkv] (8-bit pages)
  float scale;
  int window, Hq, Hkv, D;
  __nv_bfloat16* out;              // [B, T, Hq, D] dense
  float* lse;                      // [B, T, Hq] or null
};

cudaError_t paged_error_word(int dev, uint32_t** word);
cudaError_t paged_append_launch(const PagedAppendParams& prm, bool f8, int n_sm, cudaStream_t stream);
size_t paged_attn_ws_bytes(int B, int T, int Hq, int Hkv, int D, int n_sm);
cudaError_t paged_attn_launch(const PagedAttnParams& prm, bool f8, void* ws, int n_sm, cudaStream_t stream);

}  // namespace skinny
