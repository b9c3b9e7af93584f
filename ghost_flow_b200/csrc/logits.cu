// What stands between a model's logits and the choice of a token: penalties for tokens that a sequence holds already, biases, and masks of
// the tokens that a grammar allows.
//
// The reference picks the largest logit whatever else is asked for (ghostflow-nn/src/gpt.rs:402-422).
//
// For entry v of a row, with c occurrences among the row's generated tokens and `seen` among all of them:
//   x = seen ? (x > 0 ? x / repetition : x repetition) : x
//   x = x - (c frequency + (c > 0) presence)
//   x = x + bias[v]
//   x = allowed ? x : -inf                                   all in 32 bits, rounded once
//
// One CTA has a slice of one row. Counts live in shared memory: a bit for each entry of the slice that says whether the row's tokens hold it,
// and a counter that only those entries use, so that nothing but the bits has to be cleared and the pass over the logits reads one bit
// more for an entry. Counters are whole numbers: the order of their atomics does not matter.
#include <cuda_fp16.h>

#include "gf_host.h"
#include "gf_ptx.cuh"

namespace gf {

constexpr int LG_THREADS = 256;
constexpr int LG_SLICE = 8192;   // entries of a CTA

struct LogitsParams {
  const void* x;
  void* y;
  long long ldx, ldy;
  const void* tokens;            // [B, L] int32 or int64, rows ldt apart; null: no penalties
  long long ldt;
  const int *token_lens, *generated_from;          // [B] or null: all L, from 0
  const float *repetition, *presence, *frequency;  // [B] or null: the numbers below
  float repetition0, presence0, frequency0;
  const float* bias;             // rows ldb apart (0: one for all); null: none
  long long ldb;
  const unsigned* allowed;       // rows lda words apart (0: one for all); null: all
  long long lda;
  int V, L, tokens64;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f(float& y, float x) { y = x; }
__device__ __forceinline__ void from_f(__nv_bfloat16& y, float x) { y = __float2bfloat16(x); }
__device__ __forceinline__ void from_f(__half& y, float x) { y = __float2half(x); }

template <typename T>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const __grid_constant__ LogitsParams p) {
  __shared__ unsigned seen[LG_SLICE / 32];
  __shared__ int count[LG_SLICE];
  const int row = blockIdx.y, v0 = blockIdx.x * LG_SLICE, v1 = min(v0 + LG_SLICE, p.V);
  const T* x = (const T*)p.x + row * p.ldx;
  T* y = (T*)p.y + row * p.ldy;
  if (p.tokens) {
    const int n = p.token_lens ? max(0, min(p.token_lens[row], p.L)) : p.L, from = p.generated_from ? p.generated_from[row] : 0;
    auto token = [&](int i) -> long long {
      return p.tokens64 ? ((const long long*)p.tokens)[row * p.ldt + i] : ((const int*)p.tokens)[row * p.ldt + i];
    };
    for (int i = threadIdx.x; i < LG_SLICE / 32; i += LG_THREADS) seen[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += LG_THREADS) {
      const long long t = token(i);
      if (t < v0 || t >= v1) continue;
      atomicOr(&seen[(t - v0) >> 5], 1u << ((t - v0) & 31));
      count[t - v0] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += LG_THREADS) {
      const long long t = token(i);
      if (t >= v0 && t < v1 && i >= from) atomicAdd(&count[t - v0], 1);
    }
    __syncthreads();
  }
  const float rep = p.repetition ? p.repetition[row] : p.repetition0, pres = p.presence ? p.presence[row] : p.presence0;
  const float freq = p.frequency ? p.frequency[row] : p.frequency0;
  for (int v = v0 + threadIdx.x; v < v1; v += LG_THREADS) {
    float a = to_f(x[v]);
    if (p.tokens && ((seen[(v - v0) >> 5] >> ((v - v0) & 31)) & 1)) {
      const int c = count[v - v0];
      a = a > 0.f ? a / rep : a * rep;
      a -= c * freq + (c > 0 ? pres : 0.f);
    }
    if (p.bias) a += p.bias[row * p.ldb + v];
    if (p.allowed && !((p.allowed[row * p.lda + (v >> 5)] >> (v & 31)) & 1)) a = -INFINITY;
    from_f(y[v], a);
  }
}

}  // namespace gf

using namespace gf;

// 8 bytes each, as in PagedCall.
struct LogitsCall {
  const void* x;                 // [B, V] of dtype (0 fp32, 1 bf16, 2 fp16), rows ldx apart
  long long ldx;
  void* y;                       // alike; may be x
  long long ldy, dtype, B, V;
  const void* tokens;
  long long ldt, tokens64, L;
  const int *token_lens, *generated_from;
  const float *repetition, *presence, *frequency;
  double repetition0, presence0, frequency0;
  const float* bias;
  long long ldb;
  const unsigned* allowed;
  long long lda;
};

GF_API int gf_process_logits(const LogitsCall* c, void* stream) {
  constexpr long long MOST = 0x7fffffff;
  if (!c || !c->x || !c->y || c->B <= 0 || c->V <= 0 || c->V > MOST || c->L < 0 || c->L > MOST || c->dtype < 0 || c->dtype > 2 ||
      c->B > 65535)
    return GFH_BAD_ARG;
  gf::enter();
  const LogitsParams p{c->x, c->y, c->ldx, c->ldy, c->L > 0 ? c->tokens : nullptr, c->ldt, c->token_lens, c->generated_from,
                       c->repetition, c->presence, c->frequency, (float)c->repetition0, (float)c->presence0, (float)c->frequency0,
                       c->bias, c->ldb, c->allowed, c->lda, (int)c->V, (int)c->L, (int)c->tokens64};
  const dim3 grid((unsigned)((c->V + LG_SLICE - 1) / LG_SLICE), (unsigned)c->B);
  cudaStream_t st = (cudaStream_t)stream;
  if (c->dtype == 0) logits_kernel<float><<<grid, LG_THREADS, 0, st>>>(p);
  else if (c->dtype == 1) logits_kernel<__nv_bfloat16><<<grid, LG_THREADS, 0, st>>>(p);
  else logits_kernel<__half><<<grid, LG_THREADS, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
}
