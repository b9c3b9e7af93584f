// A batch of sequences over a paged KV cache, as the kernels of paged_cache.cu and attn_paged.cu see it.
//
// New tokens of all sequences lie one behind the other: those of sequence b are rows cu[b] .. cu[b + 1] - 1 (no cu: row b alone). lens[b]
// keys are valid once they are appended, so new token i of n has position p = lens[b] - n + i, which is row p % page of the page
// table[b, p / page]. Everything that comes out of device memory is bounded before it is used as an address: page numbers and positions
// that are not there are reported in the status word (GF_ERR_BAD_ARG), never read or written.
#pragma once
#include "calls.h"
#include "gf_host.h"
#include "gf_ptx.cuh"

namespace gf {

struct PagedBatch {
  const int* table;       // [B, width], rows ld apart
  const int* lens;        // [B]
  const int* cu;          // [B + 1] or null
  int* status;
  int ld, width, page_shift, pages, B, T;

  __host__ __device__ __forceinline__ long long capacity() const { return (long long)width << page_shift; }
  __device__ __forceinline__ int first(int b) const { return cu ? max(0, min(cu[b], T)) : b; }
  __device__ __forceinline__ int end(int b) const { return cu ? max(0, min(cu[b + 1], T)) : b + 1; }
  __device__ __forceinline__ void bad() const {
    if (status) atomicCAS(status, 0, GF_ERR_BAD_ARG);
  }
};

// Whole warp: the sequence of new token t, B where it is behind the last one.
__device__ __forceinline__ int paged_seq_of(const PagedBatch& s, int t) {
  if (!s.cu) return min(t, s.B);
  const int lane = threadIdx.x & 31;
  int b = 0;
  for (int i = 0; i < s.B; i += 32) {
    const unsigned before = __ballot_sync(0xffffffffu, i + lane < s.B && s.cu[i + lane + 1] <= t);
    b += __popc(before);
    if (before != 0xffffffffu) break;
  }
  return b;
}

// Host: the batch of a call; false where the kernels do not take it: sizes, pages of other than a power of two from 16 rows, and rows of x, y
// and the pools that are not on 16-byte boundaries.
inline bool paged_batch(PagedBatch& s, const PagedCall& c) {
  constexpr long long MOST = 0x7fffffff;
  if (c.B <= 0 || c.B >= MOST || c.T <= 0 || c.T >= MOST || c.width < 0 || c.ld_table < 0 || c.ld_table > MOST || c.page < 16 ||
      (c.page & (c.page - 1)) || c.page > MOST || c.pages < 0 || c.pages * c.page > MOST || c.width > MOST / c.page || !c.lens ||
      (c.width > 0 && !c.table) || (!c.cu && c.T != c.B) || c.ldx % 8 || c.ldy % 8 || c.ldx < 0 || c.ldy < 0)
    return false;
  for (const void* p : {c.x, (const void*)c.y, (const void*)c.kpages, (const void*)c.vpages})
    if (!p || (reinterpret_cast<uintptr_t>(p) & 15)) return false;
  for (long long st : c.strides)
    if (st % 8 || st < 0) return false;
  s = {c.table, c.lens, c.cu, c.status, (int)c.ld_table, (int)c.width, __builtin_ctzll((unsigned long long)c.page), (int)c.pages, (int)c.B, (int)c.T};
  return true;
}

// attn_decode.cu: one new token of each sequence of a call (with cu: of those that have one), as gf_paged_attn_one. `chained`: behind a
// kernel of the same call that it does not depend on; it starts under it and ends behind it.
bool attn_paged_one_ok(const PagedCall& c, int splits, const float* scratch);
int attn_paged_one(const PagedCall& c, float scale, int splits, float* scratch, int chained, cudaStream_t st);

}  // namespace gf
