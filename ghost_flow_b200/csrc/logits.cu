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
// x / repetition is x (1 / repetition), one rounding more: with a quotient the pass spills, 61 us for 55 (512 rows of 50257 in fp32, 4096 tokens, bias and
// mask). Callers bound the repetition so that the reciprocal is a normal number.
//
// One CTA has a slice of one row. The row's tokens, each with a thread, count themselves at the entry that they hold; then a pass over the slice, 16
// bytes at a time, does the arithmetic, whose first vectors were asked for before the tokens were looked at. Counters are whole numbers:
// the order of the threads does not matter. They lie in shared memory, 16 bits to an entry (32 where a row has 2^15 tokens or more), so that a
// vector's are one load; bits, with a counter at each set one's rank, are a third of that, but took 11.4 / 51 us for 64 / 512 rows instead of 8.0 / 47: two
// rounds over the tokens, ranks between them, and three looks for each vector.
//
// What bounds it: issue slots, 79 % of them taken: 512 rows of 50257 in fp32, 2048 to 4096 tokens, a bias for all and a mask each, take 47 us (4.5 TB/s); a pass without any of them 33 (6.2), with
// the mask 35, and the bias 43 (from L2 once more for every row; it comes by the same way as the tokens, 50 MB for three slices of a row), the mask and the
// tokens 44. One vector of a thread at a time, without the ring, took 95. Small batches: 64 rows 8.0 us, two or three 3.3. Three CTAs on an SM leave a thread
// 40 registers: enough for fp32 with 16-bit counters (36); the 16-bit types spill 28 bytes with counters and 8 without, fp32 with 32-bit counters 44.
#include <cuda_fp16.h>

#include "calls.h"
#include "gf_host.h"
#include "gf_ptx.cuh"

namespace gf {

constexpr int LG_THREADS = 512;
constexpr int LG_CTAS = 3;       // on an SM
constexpr int LG_TOKENS = 8;     // tokens of a thread on their way together
constexpr int LG_SLICE_MIN = 4096, LG_SLICE_MAX = 17408;

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

// Words of a slice's mask, which may begin up to 7 entries into the first: a multiple of 16 bytes.
__host__ __device__ constexpr int lg_words(int slice) { return (slice / 32 + 4) & ~3; }

// What the tokens say of an entry: that they hold it, in the highest bit (of a token of the prompt) or by the count below it (of generated ones).
// 16 bits to an entry where rows have fewer than 2^15 tokens; no bits where there are none.
template <int BITS>
struct LgCount {
  static constexpr int PER = BITS == 32 ? 1 : 2;                 // entries of a word
  static constexpr unsigned HELD = BITS == 32 ? 0x80000000u : 0x8000u;
  __device__ __forceinline__ static float number(unsigned c) {
    return BITS == 32 ? (float)c : __uint_as_float(0x4b000000u | c) - 8388608.f;        // 2^23 + c
  }
};
// Vectors of a thread on their way together. With counters in shared memory a fourth leaves the L1 too little: us, 3 / 4, 512 rows of 50257 with all
// there is 47 / 54, without tokens, bf16, 22 / 20.
__host__ __device__ constexpr int lg_stages(int bits) { return bits ? 3 : 4; }

template <typename T, int BITS>
__global__ void __launch_bounds__(LG_THREADS, LG_CTAS) logits_kernel(const __grid_constant__ LogitsParams p) {
  using Count = LgCount<BITS>;
  constexpr int VEC = 16 / sizeof(T), PER = Count::PER, WORDS = VEC / PER, STAGES = lg_stages(BITS);      // WORDS: counters' words of a vector
  constexpr unsigned FIELD = PER == 1 ? 0xffffffffu : 0xffffu;
  extern __shared__ __align__(16) unsigned shared[];
  const int row = blockIdx.x / p.slices, v0 = (blockIdx.x - row * p.slices) * p.slice, size = min(p.slice, p.V - v0);
  uint4* ring = reinterpret_cast<uint4*>(shared);  // [STAGES][LG_THREADS]: a thread reads what it asked for itself
  unsigned* open = shared + 4 * STAGES * LG_THREADS;          // allowed, 32 entries to a word
  unsigned* count = open + lg_words(p.slice);      // PER entries to a word
  const T* x = (const T*)p.x + row * p.ldx + v0;   // entry 0 of the slice
  T* y = (T*)p.y + row * p.ldy + v0;
  // whole vectors: `vectors` from entry `head` on, on 16-byte boundaries of x and y; none where the two begin on different ones
  const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)), size);
  const int vectors = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) ? 0 : (size - head) / VEC;
  const int shift = (VEC - head % VEC) % VEC;      // entry v is v + shift in shared memory, where vectors begin on their boundaries
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
    for (int i = 0; i < STAGES; ++i) ask(threadIdx.x + i * LG_THREADS, i);
    if (p.allowed) {
      const unsigned* from = p.allowed + row * p.lda + (v0 >> 5);
      const int words = (size + 31) / 32;
      for (int i = threadIdx.x; i < (size + shift + 31) / 32; i += LG_THREADS)
        open[i] = __funnelshift_l(i > 0 ? __ldg(from + i - 1) : 0u, i < words ? __ldg(from + i) : 0u, shift);
    }
  };
  int n = 0;
  float rep = 1.f, less = 1.f, pres = 0.f, freq = 0.f;
  if (BITS && p.tokens) {                          // (there are, with BITS; without the test the pass of fp32 is compiled to spill, 53 us for 47)
    int t[LG_TOKENS];                              // LG_TOKENS tokens of the thread from i0 on: their entries, -1 for what is not in the slice
    auto tokens = [&](int i0) {
#pragma unroll
      for (int j = 0; j < LG_TOKENS; ++j) {
        const int i = i0 + j * LG_THREADS;
        long long v = -1;
        if (i < p.L) v = p.tokens64 ? ((const long long*)p.tokens)[row * p.ldt + i] : ((const int*)p.tokens)[row * p.ldt + i];
        v -= v0;
        t[j] = v >= 0 && v < size ? (int)v + shift : -1;
      }
    };
    tokens(threadIdx.x);
    begin();                                       // behind the tokens, which everything waits for
    rep = p.repetition ? p.repetition[row] : p.repetition0;
    less = 1.f / rep;
    pres = p.presence ? p.presence[row] : p.presence0;
    freq = p.frequency ? p.frequency[row] : p.frequency0;
    const int from = p.generated_from ? p.generated_from[row] : 0;
    n = p.token_lens ? max(0, min(p.token_lens[row], p.L)) : p.L;
    for (int i = threadIdx.x; i < (p.slice + 8) / PER / 4; i += LG_THREADS) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < n;) {
#pragma unroll
      for (int j = 0; j < LG_TOKENS; ++j) {
        const int i = i0 + j * LG_THREADS;
        if (t[j] < 0 || i >= n) continue;
        unsigned* word = count + t[j] / PER;
        const int at = t[j] % PER * 16;
        if (i >= from)
          atomicAdd(word, 1u << at);
        else
          atomicOr(word, Count::HELD << at);
      }
      i0 += LG_TOKENS * LG_THREADS;
      if (i0 < n) tokens(i0);
    }
  } else {
    begin();
  }
  __syncthreads();                                 // `open` and `count`
  auto penalised = [&](float a, unsigned held) {   // held: not 0
    const unsigned c = held & (Count::HELD - 1);
    return (a > 0.f ? a * less : a * rep) - (Count::number(c) * freq + (c ? pres : 0.f));
  };
  // ---- the entries in front of the vectors and behind them, or all
  const int behind = head + vectors * VEC;
  for (int i = threadIdx.x; i < head + size - behind; i += LG_THREADS) {
    const int v = i < head ? i : i - head + behind, l = v + shift;
    float a = to_f(x[v]);
    if (BITS && n > 0) {
      const unsigned held = (count[l / PER] >> (l % PER * 16)) & FIELD;
      if (held) a = penalised(a, held);
    }
    if (bias) a += bias[v];
    if (p.allowed && !((open[l >> 5] >> (l & 31)) & 1)) a = -INFINITY;
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
  bias_of(threadIdx.x);
  T* to = y + head + threadIdx.x * VEC;
  const int first = head + shift;                  // of the vectors' entries in shared memory
  for (int k0 = threadIdx.x; k0 < vectors; k0 += STAGES * LG_THREADS) {
#pragma unroll
    for (int st = 0; st < STAGES; ++st) {
      const int k = k0 + st * LG_THREADS;
      if (k >= vectors) break;
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      const uint4 in = ring[st * LG_THREADS + threadIdx.x];
      const T* have = reinterpret_cast<const T*>(&in);
      const int l = first + k * VEC;
      float a[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) a[j] = to_f(have[j]);
      if (BITS && n > 0) {
        unsigned held[WORDS], any = 0;
        if constexpr (WORDS == 2) {
          const uint2 u = reinterpret_cast<const uint2*>(count)[l / VEC];
          held[0] = u.x; held[1] = u.y;
        } else {
#pragma unroll
          for (int w = 0; w < WORDS; w += 4) {
            const uint4 u = reinterpret_cast<const uint4*>(count)[(l / PER + w) / 4];
            held[w] = u.x; held[w + 1] = u.y; held[w + 2] = u.z; held[w + 3] = u.w;
          }
        }
#pragma unroll
        for (int w = 0; w < WORDS; ++w) any |= held[w];
        if (any) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const unsigned f = (held[j / PER] >> (j % PER * 16)) & FIELD;
            if (f) a[j] = penalised(a[j], f);
          }
        }
      }
      if (bias) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j] += add[j];
        bias_of(k + LG_THREADS);
      }
      if (p.allowed) {
        const unsigned ok = open[l >> 5] >> (l & 31);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!((ok >> j) & 1)) a[j] = -INFINITY;
      }
      uint4 u;
      T* left = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) from_f(left[j], a[j]);
      *reinterpret_cast<uint4*>(to + (k - (int)threadIdx.x) * VEC) = u;
      ask(k + STAGES * LG_THREADS, st);
    }
  }
}

// Rows are cut into two slices for every SM (with three 64 rows took 8.8 us instead of 8.0: every CTA looks at all tokens of its row), of LG_SLICE_MIN entries or
// more; many rows into slices of at most LG_SLICE_MAX, which leave the L1 room beside three CTAs' counters: 512 rows took 49 us with a quarter less, 54
// with half more. Without counters half more, with wide ones half of it.
template <typename T>
static int launch_logits(LogitsParams& p, long long B, cudaStream_t st) {
  const int bits = !p.tokens ? 0 : p.L < 1 << 15 ? 16 : 32;
  const long long longest = bits == 0 ? LG_SLICE_MAX * 3 / 2 : bits == 16 ? LG_SLICE_MAX : LG_SLICE_MAX / 2;
  const long long most = (p.V + LG_SLICE_MIN - 1) / LG_SLICE_MIN, least = (p.V + longest - 1) / longest;
  const long long slices = max(least, min(most, 2ll * sm_count() / B));
  p.slice = (int)(((p.V + slices - 1) / slices + 63) / 64 * 64);
  p.slices = (p.V + p.slice - 1) / p.slice;
  if (B * p.slices > 0x7fffffffll) return GFH_TOO_LARGE;
  const size_t smem = 16 * lg_stages(bits) * LG_THREADS + 4 * lg_words(p.slice) + (p.slice + 8) * bits / 8;
  static gf::SharedLimit limit[3];
  auto kern = bits == 0 ? logits_kernel<T, 0> : bits == 16 ? logits_kernel<T, 16> : logits_kernel<T, 32>;
  if (smem > 48 * 1024 && !limit[bits / 16].raise(kern, smem)) return GFH_CUDA;
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
