// What the entry points of the paged cache and of the logits take: tensors as addresses, sizes and strides in elements, 8 bytes each so that a caller
// in any language can pack them.
#pragma once

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

}  // namespace gf
