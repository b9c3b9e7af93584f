// What the entry points of the paged cache and of the logits take: tensors as addresses, sizes and strides in elements, 8 bytes each so that a caller
// in any language can pack them.
#pragma once

#include <initializer_list>

namespace gf {

struct PagedCall {
  const void* x;                 // new tokens: [T, heads, D], heads packed, rows ldx apart
  long long ldx;
  void* y;                       // result: [T, H, D], rows ldy apart
  long long ldy;
  void *kpages, *vpages;         // [pages, page, Hk, D]
  long long strides[6];          // pages, rows and heads of kpages, then of vpages
  const int* table;
  long long ld_table, width;
  const int *lens, *cu;
  long long B, T, H, Hk, D, page, pages;
  int* status;
};

// The same with pages of 8 bits, whose strides are of 16 bytes then: kscales and vscales [pages, Hk, page] dense, null where pages are bf16.
struct PagedCall8 {
  PagedCall c;
  const unsigned char *kscales, *vscales;
};

// Whether the scales lie outside the pools, from the first row to the last.
inline bool paged_scales_apart(const PagedCall8& r) {
  const PagedCall& c = r.c;
  for (int i = 0; i < 2; ++i) {
    const char* pool = (const char*)(i ? c.vpages : c.kpages);
    const char* end = pool + (c.pages - 1) * c.strides[3 * i] + (c.page - 1) * c.strides[3 * i + 1] + (c.Hk - 1) * c.strides[3 * i + 2] + c.D;
    for (const unsigned char* s : {r.kscales, r.vscales})
      if ((const char*)s < end && pool < (const char*)s + c.pages * c.Hk * c.page) return false;
  }
  return true;
}

struct LogitsCall {
  const void* x;                 // [B, V] of dtype (0 fp32, 1 bf16, 2 fp16), rows ldx apart
  long long ldx;
  void* y;                       // alike; may be x
  long long ldy, dtype, B, V;
  const void* tokens;            // the rest as in LogitsParams of logits.cu
  long long ldt, tokens64, L;
  const int *token_lens, *generated_from;
  const float *repetition, *presence, *frequency;
  double repetition0, presence0, frequency0;
  const float* bias;
  long long ldb;
  const unsigned* allowed;
  long long lda;
};

struct SampleCall {
  const void* x;                 // [B, V] of dtype (0 fp32, 1 bf16, 2 fp16), rows ldx apart
  long long ldx, dtype, B, V;
  const float* u;                // [B]; the rest as in SampleParams of sample.cu
  const float *temperature, *top_p, *min_p;
  const int* top_k;
  double temperature0, top_p0, min_p0;
  long long top_k0;
  long long* out;                // [B]
};

}  // namespace gf
