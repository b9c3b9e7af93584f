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

// 16 numbers of the cache times their row's power of two (twice, as f32x2), as bf16: exact but for what is below 2^-133, of rows of the two least units
__device__ __forceinline__ void bf16x16_of_e4m3(const uint4& in, uint64_t scale, uint4& lo, uint4& hi) {
  const uint32_t* four = reinterpret_cast<const uint32_t*>(&in);
  uint32_t out[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)(i & 1 ? four[i >> 1] >> 16 : four[i >> 1])));
    float a, b;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(a), "=f"(b) : "r"(h));
    const uint64_t x = f2_mul(pk2f(a, b), scale);
    out[i] = pack_bf16x2(lo2(x), hi2(x));
  }
  lo = make_uint4(out[0], out[1], out[2], out[3]);
  hi = make_uint4(out[4], out[5], out[6], out[7]);
}

// Pages of 8 bits. A row of a head is numbers of type e4m3 times 2^(b - 127), b the row's byte in the scales: the smallest power of two that leaves none of them
// above 448, the type's largest, so that none is cut off; and at least 2^-126. A power of two loses no bits in what it is multiplied with: a number of the
// cache has 4 bits, and is one of bf16 too, where it is not below 2^-133. It is off by 2^-4 of itself or, from 2^-6 of the unit on down, by 2^-10 of the unit. (A scale that brings the largest number to 448 itself gains nothing: the type's steps are
// relative.) Scales of a head lie one behind the other, so that 16 keys' are 16 bytes.
inline bool paged_scales(const PagedCall8& c8) {
  const PagedCall& c = c8.c;
  for (const void* p : {(const void*)c8.kscales, (const void*)c8.vscales})
    if (!p || (reinterpret_cast<uintptr_t>(p) & 15)) return false;
  for (long long st : c.strides)
    if (st % 16 || st > 0x7fffffff) return false;
  if (c.page <= 0 || c.strides[1] > 0x7fffffff / c.page || c.strides[4] > 0x7fffffff / c.page) return false;      // a page's rows are offsets of 32 bits
  return c.D % 16 == 0;
}

// attn_decode.cu: one new token of each sequence of a call (with cu: of those that have one), as gf_paged_attn_one. `chained`: behind a
// kernel of the same call that it does not depend on; it starts under it and ends behind it.
bool attn_paged_one_ok(const PagedCall& c, int splits, const float* scratch);
int attn_paged_one(const PagedCall& c, float scale, int splits, float* scratch, int chained, cudaStream_t st, const unsigned char* kscales = nullptr,
                   const unsigned char* vscales = nullptr);      // scales: pages of 8 bits

}  // namespace gf
