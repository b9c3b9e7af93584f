// A batch of sequences over a paged KV cache, as the kernels of paged_cache.cu and attn_paged.cu see it.
//
// New tokens of all sequences lie one behind the other: those of sequence b are rows cu[b] .. cu[b + 1] - 1 (no cu: row b alone). lens[b]
// keys are valid once they are appended, so new token i of n has position p = lens[b] - n + i, which is row p % page of the page
// table[b, p / page]. Everything that comes out of device memory is bounded before it is used as an address: page numbers and positions
// that are not there are reported in the status word (GF_ERR_BAD_ARG), never read or written.
#pragma once
#include "gf_host.h"
#include "gf_ptx.cuh"

namespace gf {

struct PagedBatch {
  const int* table;       // [B, width], rows ld apart
  const int* lens;        // [B]
  const int* cu;          // [B + 1] or null
  int* status;
  int ld, width, page_shift, pages, B, T;

  __device__ __forceinline__ long long capacity() const { return (long long)width << page_shift; }
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

// Host: fills `s` from what a caller gives; false where the kernels do not take it.
inline bool paged_batch(PagedBatch& s, const int* table, int ld, int width, const int* lens, const int* cu, int B, int T, int page,
                        int pages, int* status) {
  if (B <= 0 || T <= 0 || width < 0 || ld < 0 || page < 16 || (page & (page - 1)) || pages < 0 || !lens || (width > 0 && !table) ||
      (!cu && T != B) || (long long)pages * page > 0x7fffffffll || (long long)width * page > 0x7fffffffll)
    return false;
  s = {table, lens, cu, status, ld, width, __builtin_ctz((unsigned)page), pages, B, T};
  return true;
}

}  // namespace gf
