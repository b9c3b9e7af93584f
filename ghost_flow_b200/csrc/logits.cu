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
// One CTA has a slice of one row, which it reads and writes once, 16 bytes at a time. Which of its entries the row's tokens hold is a bit each in
// shared memory; an entry whose bit is set has a counter and a value, at its rank among the set bits (those of the words in front, counted
// once, and of its own word), so that there are no more of them than tokens and a slice may be long: a CTA looks at all tokens of its
// row, whatever its slice is. The penalties are worked out before the pass over the slice, a token to a thread; the pass itself only picks the
// values up where a bit is set (with the arithmetic in the pass, whose warps nearly all meet a set bit, 512 rows of 50257 in fp32 took 95 us).
// Counters are whole numbers, and a value is the same whichever of its tokens writes it: the order of the threads does not matter. The first
// logits are on their way all the while.
#include <cuda_fp16.h>

#include "gf_host.h"
#include "gf_ptx.cuh"

namespace gf {

constexpr int LG_THREADS = 256;
constexpr int LG_AHEAD = 4;      // vectors of a thread on their way together
constexpr int LG_TOKENS = 8;     // tokens of a thread that it looks up once
constexpr int LG_SLICE_MIN = 2048, LG_SLICE_MAX = 25600;

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
  int V, L, tokens64, slice, slices;               // slice: a multiple of 64
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f(float& y, float x) { y = x; }
__device__ __forceinline__ void from_f(__nv_bfloat16& y, float x) { y = __float2bfloat16(x); }
__device__ __forceinline__ void from_f(__half& y, float x) { y = __float2half(x); }

// 32 bits from bit `at` on; `more`: whether the bits that are wanted go on into the next word
__device__ __forceinline__ unsigned bits_at(const unsigned* words, int at, bool more) {
  const int s = at & 31;
  unsigned w = words[at >> 5] >> s;
  if (more && s) w |= words[(at >> 5) + 1] << (32 - s);
  return w;
}

template <typename T>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const __grid_constant__ LogitsParams p) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ unsigned shared[];
  __shared__ int warp_sum[LG_THREADS / 32];
  const int row = blockIdx.x / p.slices, v0 = (blockIdx.x - row * p.slices) * p.slice, v1 = min(v0 + p.slice, p.V), n_words = p.slice / 32;
  unsigned* seen = shared;                         // [n_words]
  int* before = (int*)(shared + n_words);          // [n_words]: set bits of the words in front
  int* count = before + n_words;                   // [min(L, slice)]
  float* value = (float*)(count + min(p.L, p.slice));
  const T* x = (const T*)p.x + row * p.ldx;
  T* y = (T*)p.y + row * p.ldy;
  // vector k has the entries from v0 - lead + k VEC on
  const int lead = (int)((reinterpret_cast<uintptr_t>(x + v0) & 15) / sizeof(T));
  const bool wide = (int)((reinterpret_cast<uintptr_t>(y + v0) & 15) / sizeof(T)) == lead;
  const int vectors = (v1 - v0 + lead + VEC - 1) / VEC;
  auto inside = [&](int k) {
    const int e = v0 - lead + k * VEC;
    return wide && e >= v0 && e + VEC <= v1;
  };
  uint4 in[LG_AHEAD];
  auto load = [&](int k0) {
#pragma unroll
    for (int i = 0; i < LG_AHEAD; ++i) {
      const int k = k0 + i * LG_THREADS;
      if (inside(k)) in[i] = *reinterpret_cast<const uint4*>(x + (v0 - lead + k * VEC));
    }
  };
  load(threadIdx.x);
  const float rep = p.repetition ? p.repetition[row] : p.repetition0, pres = p.presence ? p.presence[row] : p.presence0;
  const float freq = p.frequency ? p.frequency[row] : p.frequency0;
  int n = 0;
  if (p.tokens) n = p.token_lens ? max(0, min(p.token_lens[row], p.L)) : p.L;
  auto rank = [&](int v) { return before[v >> 5] + __popc(seen[v >> 5] & ((1u << (v & 31)) - 1)); };
  if (n > 0) {
    const int from = p.generated_from ? p.generated_from[row] : 0;
    // LG_TOKENS tokens of a thread from i0 on: their entries in the slice, -1 for one that is not in it
    auto tokens = [&](int i0, int (&v)[LG_TOKENS]) {
#pragma unroll
      for (int j = 0; j < LG_TOKENS; ++j) {
        const int i = i0 + j * LG_THREADS;
        const long long t = i >= n ? -1ll : p.tokens64 ? ((const long long*)p.tokens)[row * p.ldt + i] : ((const int*)p.tokens)[row * p.ldt + i];
        v[j] = t >= v0 && t < v1 ? (int)(t - v0) : -1;
      }
    };
    int mine[LG_TOKENS];                           // the first of them, for every round
    tokens(threadIdx.x, mine);
    auto each = [&](auto f) {
#pragma unroll
      for (int j = 0; j < LG_TOKENS; ++j)
        if (mine[j] >= 0) f(mine[j], (int)threadIdx.x + j * LG_THREADS);
      for (int i0 = threadIdx.x + LG_TOKENS * LG_THREADS; i0 < n; i0 += LG_TOKENS * LG_THREADS) {
        int v[LG_TOKENS];
        tokens(i0, v);
#pragma unroll
        for (int j = 0; j < LG_TOKENS; ++j)
          if (v[j] >= 0) f(v[j], i0 + j * LG_THREADS);
      }
    };
    for (int i = threadIdx.x; i < n_words; i += LG_THREADS) seen[i] = 0;
    for (int i = threadIdx.x; i < min(n, p.slice); i += LG_THREADS) count[i] = 0;
    __syncthreads();
    each([&](int v, int) { atomicOr(&seen[v >> 5], 1u << (v & 31)); });
    __syncthreads();
    // ranks: a thread sums up the words that are its own, one behind the other, then the threads' sums
    const int per = (n_words + LG_THREADS - 1) / LG_THREADS, w0 = min(threadIdx.x * per, n_words), w1 = min(w0 + per, n_words);
    int own = 0;
    for (int i = w0; i < w1; ++i) own += __popc(seen[i]);
    int incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if ((threadIdx.x & 31) >= o) incl += u;
    }
    if ((threadIdx.x & 31) == 31) warp_sum[threadIdx.x >> 5] = incl;
    __syncthreads();
    int at = incl - own;
#pragma unroll
    for (int i = 0; i < LG_THREADS / 32; ++i)
      if (i < (threadIdx.x >> 5)) at += warp_sum[i];
    for (int i = w0; i < w1; ++i) {
      before[i] = at;
      at += __popc(seen[i]);
    }
    __syncthreads();
    each([&](int v, int i) {
      if (i >= from) atomicAdd(&count[rank(v)], 1);
    });
    __syncthreads();
    each([&](int v, int) {
      const int r = rank(v), c = count[r];
      const float a = to_f(x[v0 + v]);
      value[r] = (a > 0.f ? a / rep : a * rep) - (c * freq + (c > 0 ? pres : 0.f));
    });
    __syncthreads();
  }
  const float* bias = p.bias ? p.bias + row * p.ldb : nullptr;
  const unsigned* allowed = p.allowed ? p.allowed + row * p.lda : nullptr;
  for (int k0 = threadIdx.x; k0 < vectors; k0 += LG_AHEAD * LG_THREADS) {
    if (k0 != threadIdx.x) load(k0);
#pragma unroll
    for (int i = 0; i < LG_AHEAD; ++i) {
      const int k = k0 + i * LG_THREADS, e = v0 - lead + k * VEC;
      if (k >= vectors) break;
      if (inside(k)) {
        const T* have = reinterpret_cast<const T*>(&in[i]);
        float a[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j] = to_f(have[j]);
        if (n > 0) {
          const unsigned hit = bits_at(seen, e - v0, ((e - v0) & 31) + VEC > 32) & ((1u << VEC) - 1);
          if (hit) {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
              if ((hit >> j) & 1) a[j] = value[rank(e - v0 + j)];
          }
        }
        if (bias) {
          if ((reinterpret_cast<uintptr_t>(bias + e) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < VEC; j += 4) {
              const float4 u = *reinterpret_cast<const float4*>(bias + e + j);
              a[j] += u.x; a[j + 1] += u.y; a[j + 2] += u.z; a[j + 3] += u.w;
            }
          } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] += bias[e + j];
          }
        }
        if (allowed) {
          const unsigned ok = bits_at(allowed, e, (e & 31) + VEC > 32);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (!((ok >> j) & 1)) a[j] = -INFINITY;
        }
        uint4 u;
        T* left = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int j = 0; j < VEC; ++j) from_f(left[j], a[j]);
        *reinterpret_cast<uint4*>(y + e) = u;
      } else {
        for (int v = max(e, v0); v < min(e + VEC, v1); ++v) {
          float a = to_f(x[v]);
          if (n > 0 && ((seen[(v - v0) >> 5] >> ((v - v0) & 31)) & 1)) a = value[rank(v - v0)];
          if (bias) a += bias[v];
          if (allowed && !((allowed[v >> 5] >> (v & 31)) & 1)) a = -INFINITY;
          from_f(y[v], a);
        }
      }
    }
  }
}

// A slice is as long as leaves about four CTAs to an SM, and at most LG_SLICE_MAX.
template <typename T>
static int launch_logits(LogitsParams& p, long long B, cudaStream_t st) {
  const long long want = ((long long)p.V * B + 4 * sm_count() - 1) / (4 * sm_count());
  long long slices = (p.V + max((long long)LG_SLICE_MIN, min(want, (long long)LG_SLICE_MAX)) - 1) / max((long long)LG_SLICE_MIN, min(want, (long long)LG_SLICE_MAX));
  p.slice = (int)(((p.V + slices - 1) / slices + 63) / 64 * 64);
  p.slices = (p.V + p.slice - 1) / p.slice;
  if (B * p.slices > 0x7fffffffll) return GFH_TOO_LARGE;
  const size_t smem = p.tokens ? p.slice / 4 + 8ll * min(p.L, p.slice) : 0;
  static gf::DeviceMax granted;
  auto kern = logits_kernel<T>;
  if (smem > 48 * 1024 && granted.get() < smem) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return GFH_CUDA;
    granted.set(smem);
  }
  kern<<<(unsigned)(B * p.slices), LG_THREADS, smem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
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
      c->B > MOST)
    return GFH_BAD_ARG;
  gf::enter();
  LogitsParams p{c->x, c->y, c->ldx, c->ldy, c->L > 0 ? c->tokens : nullptr, c->ldt, c->token_lens, c->generated_from,
                 c->repetition, c->presence, c->frequency, (float)c->repetition0, (float)c->presence0, (float)c->frequency0,
                 c->bias, c->ldb, c->allowed, c->lda, (int)c->V, (int)c->L, (int)c->tokens64, 0, 0};
  cudaStream_t st = (cudaStream_t)stream;
  return c->dtype == 0 ? launch_logits<float>(p, c->B, st) : c->dtype == 1 ? launch_logits<__nv_bfloat16>(p, c->B, st)
                                                                           : launch_logits<__half>(p, c->B, st);
}
