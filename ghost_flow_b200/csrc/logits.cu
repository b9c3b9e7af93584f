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
// One CTA has a slice of one row. The row's tokens, each with a thread, set a bit for the entry that they hold and count themselves; then a pass
// over the slice, 16 bytes at a time, does the arithmetic, whose first vectors were asked for before the tokens were looked at. An
// entry's counter, later what is taken off it, lies at its rank among the set bits (those of the words in front, counted once, and of its own word):
// there are no more of them than tokens, so that a slice may be long, and a CTA looks at all tokens of its row whatever its slice is; entries
// of one vector have ranks one behind the other. Counters are whole numbers: the order of the threads does not matter.
//
// What bounds it: issue slots, 73 % of them taken with fp32. 512 rows of 50257 with 2048 to 4096 tokens, a bias for all and a mask each take 52 us
// (4.1 TB/s); a pass without any of them 33 (6.2), the mask adds less than 1, the bias, from L2 once more for every row, 7 to 10, the tokens 7. One vector
// of a thread at a time, without the ring, took 95; two CTAs of 512 threads on an SM and longer rings 57. Small batches: 64 rows 11 us, two or three 4.
#include <cuda_fp16.h>

#include "calls.h"
#include "gf_host.h"
#include "gf_ptx.cuh"

namespace gf {

constexpr int LG_THREADS = 512;
constexpr int LG_CTAS = 3;       // on an SM
constexpr int LG_STAGES = 4;     // vectors of a thread on their way together
constexpr int LG_TOKENS = 8;     // tokens of a thread that it looks up once
constexpr int LG_SLICE_MIN = 4096, LG_SLICE_MAX = 25600;

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

template <typename T>
__global__ void __launch_bounds__(LG_THREADS, LG_CTAS) logits_kernel(const __grid_constant__ LogitsParams p) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) unsigned shared[];
  __shared__ int warp_sum[LG_THREADS / 32];
  const int row = blockIdx.x / p.slices, v0 = (blockIdx.x - row * p.slices) * p.slice, size = min(p.slice, p.V - v0), n_words = p.slice / 32;
  uint4* ring = reinterpret_cast<uint4*>(shared);  // [LG_STAGES][LG_THREADS]: a thread reads what it asked for itself
  unsigned* open = shared + 4 * LG_STAGES * LG_THREADS;          // [n_words]: allowed
  uint2* seen = reinterpret_cast<uint2*>(open + n_words);        // [n_words]: bits, and set bits of the words in front
  int* count = (int*)(seen + n_words);             // [min(L, slice)]
  const T* x = (const T*)p.x + row * p.ldx + v0;   // entry 0 of the slice
  T* y = (T*)p.y + row * p.ldy + v0;
  // whole vectors: `vectors` from entry `head` on, on 16-byte boundaries of x and y; none where the two begin on different ones
  const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)), size);
  const int vectors = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) ? 0 : (size - head) / VEC;
  const T* xv = x + head + threadIdx.x * VEC;
  const uint32_t slot = smem_u32(ring + threadIdx.x);
  auto ask = [&](int k, int st) {                  // vector k of the slice; one group each, empty ones behind the last
    if (k < vectors)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + st * (LG_THREADS * 16)), "l"(xv + (k - (int)threadIdx.x) * VEC)
                   : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const float* bias = p.bias ? p.bias + row * p.ldb + v0 : nullptr;
  auto begin = [&] {                               // what the pass needs first, on its way while the tokens are counted
#pragma unroll
    for (int i = 0; i < LG_STAGES; ++i) ask(threadIdx.x + i * LG_THREADS, i);
    if (p.allowed)
      for (int i = threadIdx.x; i < (size + 31) / 32; i += LG_THREADS) open[i] = __ldg(p.allowed + row * p.lda + (v0 >> 5) + i);
  };
  auto rank = [&](int v) {                         // of entry v if its bit is set, else of the next one whose is
    const uint2 w = seen[v >> 5];
    return (int)w.y + __popc(w.x & ~(0xffffffffu << (v & 31)));
  };
  int n = 0;
  const float rep = p.repetition ? p.repetition[row] : p.repetition0, less = 1.f / rep;
  auto penalised = [&](float a, int r) { return (a > 0.f ? a * less : a * rep) - __int_as_float(count[r]); };
  if (p.tokens) {
    const float pres = p.presence ? p.presence[row] : p.presence0, freq = p.frequency ? p.frequency[row] : p.frequency0;
    const int from = p.generated_from ? p.generated_from[row] : 0;
    n = p.token_lens ? max(0, min(p.token_lens[row], p.L)) : p.L;
    // LG_TOKENS tokens of a thread from i0 on: their entries, -1 for one that is not in the slice (or not there)
    auto tokens = [&](int i0, int (&v)[LG_TOKENS]) {
#pragma unroll
      for (int j = 0; j < LG_TOKENS; ++j) {
        const int i = i0 + j * LG_THREADS;
        long long t = -1;
        if (i < p.L) t = p.tokens64 ? ((const long long*)p.tokens)[row * p.ldt + i] : ((const int*)p.tokens)[row * p.ldt + i];
        t -= v0;
        v[j] = t >= 0 && t < size ? (int)t : -1;
      }
#pragma unroll
      for (int j = 0; j < LG_TOKENS; ++j)
        if (i0 + j * LG_THREADS >= n) v[j] = -1;
    };
    int mine[LG_TOKENS];                           // the first of them, for every round
    tokens(threadIdx.x, mine);
    begin();                                       // behind the tokens, which everything waits for
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
    for (int i = threadIdx.x; i < n_words; i += LG_THREADS) seen[i].x = 0;
    __syncthreads();
    each([&](int v, int) { atomicOr(&seen[v >> 5].x, 1u << (v & 31)); });
    __syncthreads();
    // ranks: a thread sums up the words that are its own, one behind the other, then the threads' sums
    const int per = (n_words + LG_THREADS - 1) / LG_THREADS, w0 = min(threadIdx.x * per, n_words), w1 = min(w0 + per, n_words);
    int own = 0;
    for (int i = w0; i < w1; ++i) own += __popc(seen[i].x);
    int incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if ((threadIdx.x & 31) >= o) incl += u;
    }
    if ((threadIdx.x & 31) == 31) warp_sum[threadIdx.x >> 5] = incl;
    __syncthreads();
    int at = incl - own, held = 0;                 // entries that the tokens hold
#pragma unroll
    for (int i = 0; i < LG_THREADS / 32; ++i) {
      if (i < (threadIdx.x >> 5)) at += warp_sum[i];
      held += warp_sum[i];
    }
    for (int i = threadIdx.x; i < held; i += LG_THREADS) count[i] = 0;
    for (int i = w0; i < w1; ++i) {
      seen[i].y = at;
      at += __popc(seen[i].x);
    }
    __syncthreads();
    each([&](int v, int i) {
      if (i >= from) atomicAdd(&count[rank(v)], 1);
    });
    __syncthreads();
    for (int i = threadIdx.x; i < held; i += LG_THREADS) {
      const int c = count[i];
      count[i] = __float_as_int(c * freq + (c > 0 ? pres : 0.f));
    }
  } else {
    begin();
  }
  __syncthreads();                                 // `open` and what is taken off
  // ---- the entries in front of the vectors and behind them, or all
  const int behind = head + vectors * VEC;
  for (int i = threadIdx.x; i < head + size - behind; i += LG_THREADS) {
    const int v = i < head ? i : i - head + behind;
    float a = to_f(x[v]);
    if (n > 0 && ((seen[v >> 5].x >> (v & 31)) & 1)) a = penalised(a, rank(v));
    if (bias) a += bias[v];
    if (p.allowed && !((open[v >> 5] >> (v & 31)) & 1)) a = -INFINITY;
    from_f(y[v], a);
  }
  // ---- the vectors
  const float* bv = bias ? bias + head + threadIdx.x * VEC : nullptr;
  const bool bias4 = (reinterpret_cast<uintptr_t>(bv) & 15) == 0;
  float add[VEC];
  auto bias_of = [&](int k) {                      // asked for a vector ahead
    if (!bias || k >= vectors) return;
    const float* from = bv + (k - (int)threadIdx.x) * VEC;
    if (bias4) {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(from + j));
        add[j] = u.x; add[j + 1] = u.y; add[j + 2] = u.z; add[j + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) add[j] = __ldg(from + j);
    }
  };
  const bool apart = head % VEC != 0;              // the bits of a vector may go on into the next word
  auto bits = [&](int l, auto word) {              // of the VEC entries from l on
    unsigned w = word(l >> 5) >> (l & 31);
    if (apart && (l & 31) + VEC > 32) w |= word((l >> 5) + 1) << (32 - (l & 31));
    return w & ((1u << VEC) - 1);
  };
  bias_of(threadIdx.x);
  T* to = y + head + threadIdx.x * VEC;
  for (int k0 = threadIdx.x; k0 < vectors; k0 += LG_STAGES * LG_THREADS) {
#pragma unroll
    for (int st = 0; st < LG_STAGES; ++st) {
      const int k = k0 + st * LG_THREADS;
      if (k >= vectors) break;
      asm volatile("cp.async.wait_group %0;" ::"n"(LG_STAGES - 1) : "memory");
      const uint4 in = ring[st * LG_THREADS + threadIdx.x];
      const T* have = reinterpret_cast<const T*>(&in);
      const int l = head + k * VEC;
      float a[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) a[j] = to_f(have[j]);
      if (n > 0) {
        const unsigned hit = bits(l, [&](int w) { return seen[w].x; });
        if (hit) {
          int r = rank(l);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if ((hit >> j) & 1) a[j] = penalised(a[j], r++);
        }
      }
      if (bias) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j] += add[j];
        bias_of(k + LG_THREADS);
      }
      if (p.allowed) {
        const unsigned ok = bits(l, [&](int w) { return open[w]; });
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!((ok >> j) & 1)) a[j] = -INFINITY;
      }
      uint4 u;
      T* left = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) from_f(left[j], a[j]);
      *reinterpret_cast<uint4*>(to + (k - (int)threadIdx.x) * VEC) = u;
      ask(k + LG_STAGES * LG_THREADS, st);
    }
  }
}

// Rows are cut into as many slices as run at one time, of LG_SLICE_MIN entries or more; more rows than that into slices of at most LG_SLICE_MAX (a CTA
// spends about half as long on its row's tokens as on such a slice: half as long ones took 62 us for 512 rows instead of 52, whole rows 61, because
// a fourth round of CTAs then has little to do).
template <typename T>
static int launch_logits(LogitsParams& p, long long B, cudaStream_t st) {
  const long long most = (p.V + LG_SLICE_MIN - 1) / LG_SLICE_MIN, least = (p.V + LG_SLICE_MAX - 1) / LG_SLICE_MAX;
  const long long slices = max(least, min(most, (long long)LG_CTAS * sm_count() / B));
  p.slice = (int)(((p.V + slices - 1) / slices + 63) / 64 * 64);
  p.slices = (p.V + p.slice - 1) / p.slice;
  if (B * p.slices > 0x7fffffffll) return GFH_TOO_LARGE;
  const size_t smem = 16 * LG_STAGES * LG_THREADS + p.slice / 8 + (p.tokens ? p.slice / 4 + 4ll * min(p.L, p.slice) : 0);
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
