// The next token of every row of logits, from a random number of each row: temperature, the k likeliest, the likeliest that hold a share p, those of
// at least min_p of the likeliest's probability.
//
// The reference picks the largest logit (ghostflow-nn/src/gpt.rs:402-422).
//
// With m the row's largest logit, w[v] = exp((x[v] - m) / T). Of the order by (x down, v up) the first k stay, of these each in front of which less than p of
// their sum stands, of these those with w >= min_p. The result is the first v, in the order of the vocabulary, up to which the sum of what stays exceeds u
// times all of it.
//
// Weights are whole numbers of 64 bits, w 2^46 rounded (2^42 at the largest vocabulary): their sums do not depend on an order, so threads add them up as they come,
// and two runs agree to the bit. Exponentials are of 64 bits, as are shares and thresholds: with 32 the result of one row in some 10^4 would be another one's
// neighbour (a vocabulary of 50257 has that many borders, each off by some 2^-25). A weight below the last bit counts as one of it: u = 0 still takes the
// first token that stays.
//
// One CTA has a row, and reads it from L2 in every pass but the first: the largest entry; a histogram over bins of equal width of m - x, of numbers or of weights,
// that says in which bin the k-th entry or the share p ends; the entries of that bin, which are ranked among each other in shared memory (each thread has one
// and looks at all others). Bins of too many entries are cut further by the entries' bits, and entries that are all equal counted off in the order of
// the vocabulary. A last pass leaves the sums of every warp's pieces, among which u is looked up. Where all of the first k entries fit into shared memory the
// rest happens there, without that pass.
#include <cuda_fp16.h>

#include "calls.h"
#include "gf_host.h"
#include "gf_ptx.cuh"

namespace gf {

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32;
constexpr int SM_BINS = 2048;
constexpr int SM_LIST = SM_THREADS;      // entries that are ranked in shared memory
constexpr int SM_MOST = 1 << 20;         // entries of a row

typedef unsigned long long u64;

struct SampleParams {
  const void* x;
  long long ldx;
  const float* u;                                   // [B]
  const float *temperature, *top_p, *min_p;         // [B] or null: the numbers below
  const int* top_k;
  float temperature0, top_p0, min_p0;
  int top_k0;
  long long* out;                                   // [B]
  int V, bits;                                      // a weight of 1 is 2^bits
};

struct SampleShared {
  unsigned bin[2][SM_BINS];        // low and high words
  u64 entry[SM_LIST], weight[SM_LIST];
  u64 part[SM_WARPS];
  unsigned lo, hi;
  int n, first;
  u64 cut, above, total;
  unsigned critical;
};

__device__ __forceinline__ float sm_f(float x) { return x; }
__device__ __forceinline__ float sm_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float sm_f(__half x) { return __half2float(x); }

// Numbers in the order of the floats (zeros are one: -0 was made 0).
__device__ __forceinline__ unsigned sm_key(float x) {
  const unsigned b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
// An entry's place in the order by (x down, index up): the larger, the further in front.
__device__ __forceinline__ u64 sm_entry(float x, int v) { return (u64)sm_key(x) << 32 | (0xffffffffu - (unsigned)v); }
__device__ __forceinline__ int sm_index(u64 e) { return (int)(0xffffffffu - (unsigned)e); }
__device__ __forceinline__ float sm_value(u64 e) {
  const unsigned k = (unsigned)(e >> 32);
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ u64 sm_warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum of the lanes in front.
__device__ __forceinline__ u64 sm_warp_before(u64 v) {
  const int lane = threadIdx.x & 31;
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  return s - v;
}
// Whole CTA: the sum of the threads in front, and of all. `part` is free again behind the next barrier.
__device__ __forceinline__ u64 sm_before(u64 v, u64* part, u64& all) {
  const u64 in_warp = sm_warp_before(v), last = __shfl_sync(0xffffffffu, in_warp + v, 31);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = last;
  __syncthreads();
  u64 before = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < SM_WARPS; ++i) {
    if (i < (int)(threadIdx.x >> 5)) before += part[i];
    all += part[i];
  }
  return before + in_warp;
}

template <typename T>
struct SampleRow {
  static constexpr int VEC = 16 / sizeof(T);
  static constexpr int TILE = SM_THREADS * VEC;    // a vector to a thread
  static constexpr int AHEAD = sizeof(T) == 4 ? 4 : 2;         // vectors of a thread on their way together
  const T* x;
  int V, off, tiles;             // vector 0 begins `off` entries in front of the row, on a 16-byte boundary
  float m, per_bin;
  double per_t;                  // log2(e) / T
  double one;                    // 2^bits

  __device__ __forceinline__ void vector(int i, float (&a)[VEC]) const {
    const int v0 = i * VEC - off;
    if (v0 >= 0 && v0 + VEC <= V) {
      const uint4 in = __ldg(reinterpret_cast<const uint4*>(x + v0));
      const T* have = reinterpret_cast<const T*>(&in);
#pragma unroll
      for (int j = 0; j < VEC; ++j) a[j] = sm_f(have[j]) + 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) a[j] = v0 + j >= 0 && v0 + j < V ? sm_f(x[v0 + j]) + 0.f : -INFINITY;
    }
  }
  // f(entry, index) for all of them and, at the row's ends, for -inf at indices that are not there
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
    for (int t = 0; t < tiles; t += AHEAD) {
      float a[AHEAD][VEC];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) vector((t + k) * SM_THREADS + threadIdx.x, a[k]);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int v0 = ((t + k) * SM_THREADS + threadIdx.x) * VEC - off;
#pragma unroll
        for (int j = 0; j < VEC; ++j) f(a[k][j], v0 + j);
      }
    }
  }
  __device__ __forceinline__ bool there(int v) const { return (unsigned)v < (unsigned)V; }
  __device__ __forceinline__ int bin(float a) const { return min(SM_BINS - 1, __float2int_rz((m - a) * per_bin)); }
  __device__ __forceinline__ double weight(float a) const { return exp2(((double)a - (double)m) * per_t); }
  __device__ __forceinline__ u64 whole(double w) const {
    const u64 n = __double2ull_rn(w * one);
    return n == 0 && w > 0.0 ? 1 : n;
  }
};

// Where the order ends: the last entry (see sm_entry) that stays of those from `from` on, by numbers (the first `share` ones) or by weights (up to a `share` of
// their sum). `all_in_list`: by numbers, and the list has all entries from the first on, n of them, of which the first `share` are what stays.
template <bool WEIGHTS, typename T>
__device__ u64 sm_cut(const SampleRow<T>& row, SampleShared& s, u64 from, double share, bool& all_in_list) {
  const int tid = threadIdx.x;
  all_in_list = false;
  unsigned lo = 0, hi = 0xffffffffu;               // keys that are looked at
  int bin0 = -1;                                   // and, behind the first level, the bin
  unsigned top = 0;
  int shift = 0;
  u64 above = 0;
  double target = share;
  auto looked_at = [&](float a, int v) {
    if (!row.there(v) || sm_entry(a, v) < from) return false;
    if (bin0 < 0) return true;
    const unsigned k = sm_key(a);
    return row.bin(a) == bin0 && k >= lo && k <= hi;
  };
  while (true) {
    // ---- the bins
    for (int i = tid; i < 2 * SM_BINS; i += SM_THREADS) s.bin[0][i] = 0;
    if (tid == 0) s.n = 0;
    __syncthreads();
    row.each([&](float a, int v) {
      if (!looked_at(a, v)) return;
      const unsigned b = bin0 < 0 ? row.bin(a) : (top - sm_key(a)) >> shift;
      if (!WEIGHTS) {
        atomicAdd(&s.bin[0][b], 1u);
      } else {
        const u64 w = row.whole(row.weight(a));
        const unsigned low = (unsigned)w, old = atomicAdd(&s.bin[0][b], low), high = (unsigned)(w >> 32) + (old + low < old);
        if (high) atomicAdd(&s.bin[1][b], high);
      }
    });
    __syncthreads();
    constexpr int OWN = SM_BINS / SM_THREADS;
    u64 own[OWN], sum = 0, total;
#pragma unroll
    for (int i = 0; i < OWN; ++i) sum += own[i] = (u64)s.bin[1][tid * OWN + i] << 32 | s.bin[0][tid * OWN + i];
    u64 before = sm_before(sum, s.part, total) + above;
    if (WEIGHTS && bin0 < 0) target = share * (double)total;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      if ((double)before < target && (double)(before + own[i]) >= target) {
        s.critical = tid * OWN + i;
        s.above = before;
        s.total = before + own[i];
      }
      before += own[i];
    }
    __syncthreads();
    const unsigned b = s.critical;
    const u64 up_to = s.total;
    above = s.above;
    // ---- its entries, or all up to it
    all_in_list = !WEIGHTS && bin0 < 0 && up_to <= SM_LIST;
    if (bin0 < 0) {
      bin0 = (int)b;
    } else {
      hi = top - (b << shift);
      lo = hi - ((1u << shift) - 1);
    }
    row.each([&](float a, int v) {
      if (all_in_list ? row.there(v) && row.bin(a) <= bin0 : looked_at(a, v)) {
        const int at = atomicAdd(&s.n, 1);
        if (at < SM_LIST) s.entry[at] = sm_entry(a, v);
      }
    });
    __syncthreads();
    const int n = s.n;
    if (n <= SM_LIST) {
      if (all_in_list) return 0;
      if (WEIGHTS) {
        if (tid < n) s.weight[tid] = row.whole(row.weight(sm_value(s.entry[tid])));
        __syncthreads();
      }
      if (tid < n) {
        const u64 e = s.entry[tid];
        u64 front = above;
#pragma unroll 4
        for (int j = 0; j < n; ++j)
          if (s.entry[j] > e) front += WEIGHTS ? s.weight[j] : 1;
        if ((double)front < target && (double)(front + (WEIGHTS ? s.weight[tid] : 1)) >= target) s.cut = e;
      }
      __syncthreads();
      return s.cut;
    }
    // ---- too many: by the bits of those that there are
    if (tid == 0) {
      s.lo = 0xffffffffu;
      s.hi = 0;
    }
    __syncthreads();
    unsigned least = 0xffffffffu, most = 0;
    row.each([&](float a, int v) {
      if (!looked_at(a, v)) return;
      least = min(least, sm_key(a));
      most = max(most, sm_key(a));
    });
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if ((tid & 31) == 0) {
      atomicMin(&s.lo, least);
      atomicMax(&s.hi, most);
    }
    __syncthreads();
    lo = s.lo;
    hi = top = s.hi;
    if (lo == hi) break;
    shift = max(0, 32 - __clz(hi - lo) - 11);      // 2048 = 2^11 bins
    __syncthreads();
  }
  // ---- equal entries: as many of them as it takes, in the order of the vocabulary
  const u64 w = WEIGHTS ? row.whole(row.weight(sm_value((u64)hi << 32))) : 1;
  u64 take = (u64)fmax(1.0, ceil((target - (double)above) / (double)w));
  while (take > 1 && (double)(above + (take - 1) * w) >= target) --take;
  while ((double)(above + take * w) < target) ++take;
  u64 seen = 0;
  for (int t = 0; t < row.tiles; ++t) {            // a tile's entries stand in the threads' order
    float a[SampleRow<T>::VEC];
    const int v0 = (t * SM_THREADS + tid) * SampleRow<T>::VEC - row.off;
    row.vector(t * SM_THREADS + tid, a);
    unsigned hit = 0;
#pragma unroll
    for (int j = 0; j < SampleRow<T>::VEC; ++j)
      if (row.there(v0 + j) && sm_entry(a[j], v0 + j) >= from && sm_key(a[j]) == hi) hit |= 1u << j;
    u64 all, before = seen + sm_before(__popc(hit), s.part, all);
#pragma unroll
    for (int j = 0; j < SampleRow<T>::VEC; ++j)
      if (hit >> j & 1 && ++before == take) s.cut = sm_entry(a[j], v0 + j);
    seen += all;
    __syncthreads();
    if (seen >= take) break;
  }
  return s.cut;
}

// Whole CTA: the smallest index for which `f(entry)`; -1 where there is none.
template <typename T, typename F>
__device__ int sm_first(const SampleRow<T>& row, SampleShared& s, F f) {
  if (threadIdx.x == 0) s.first = 0x7fffffff;
  __syncthreads();
  int best = 0x7fffffff;
  row.each([&](float a, int v) {
    if (row.there(v) && f(a)) best = min(best, v);
  });
  best = __reduce_min_sync(0xffffffffu, best);
  if ((threadIdx.x & 31) == 0) atomicMin(&s.first, best);
  __syncthreads();
  return s.first == 0x7fffffff ? -1 : s.first;
}

template <typename T>
__global__ void __launch_bounds__(SM_THREADS, 2) sample_kernel(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) uint8_t raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(raw);
  u64* pieces = reinterpret_cast<u64*>(raw + sizeof(SampleShared));          // [tiles][warps]
  using Row = SampleRow<T>;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long b = blockIdx.x;
  Row row;
  row.x = (const T*)p.x + b * p.ldx;
  row.V = p.V;
  row.off = (int)((reinterpret_cast<uintptr_t>(row.x) & 15) / sizeof(T));
  row.tiles = (p.V + row.off + Row::TILE - 1) / Row::TILE;
  const float temperature = p.temperature ? p.temperature[b] : p.temperature0;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p0;
  const float min_p = fminf(p.min_p ? p.min_p[b] : p.min_p0, 1.f);
  const int top_k = p.top_k ? p.top_k[b] : p.top_k0;
  const float u = fminf(fmaxf(p.u[b], 0.f), 0x1.fffffep-1f);

  // ---- the largest entry, and the mean of those that are numbers
  float most = -INFINITY, sum = 0.f;
  int numbers = 0, none = 0;
  row.each([&](float a, int v) {
    none |= a != a;
    most = fmaxf(most, a);
    const bool number = fabsf(a) < 0x1p100f;
    sum += number ? a : 0.f;
    numbers += number;
  });
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  numbers = __reduce_add_sync(0xffffffffu, numbers);
  none = __any_sync(0xffffffffu, none);
  float* f = reinterpret_cast<float*>(s.entry);
  int* n = reinterpret_cast<int*>(s.weight);
  if (lane == 0) {
    f[warp] = most;
    f[SM_WARPS + warp] = sum;
    n[warp] = numbers;
    n[SM_WARPS + warp] = none;
  }
  __syncthreads();
  most = -INFINITY, sum = 0.f, numbers = none = 0;
#pragma unroll
  for (int i = 0; i < SM_WARPS; ++i) {
    most = fmaxf(most, f[i]);
    sum += f[SM_WARPS + i];
    numbers += n[i];
    none |= n[SM_WARPS + i];
  }
  // ---- rows without probabilities, and those whose likeliest entry is asked for
  if (none || !(temperature > 0.f) || top_k == 1 || top_p <= 0.f || fabsf(most) == INFINITY) {
    const int v = none                ? sm_first(row, s, [](float a) { return a != a; })
                  : most == -INFINITY ? -1
                                      : sm_first(row, s, [&](float a) { return a == most; });
    if (tid == 0) p.out[b] = v;
    return;
  }
  row.m = most;
  row.per_t = 1.4426950408889634 / (double)temperature;
  row.one = (double)(1ull << p.bits);
  // bins that reach twice as far as the mean; what is further away lies in the last
  const float reach = 2.f * (most - sum / (float)max(numbers, 1));
  row.per_bin = reach > 0x1p-60f && reach < 0x1p100f ? (float)SM_BINS / reach : 1.f;
  __syncthreads();

  u64 cut = 0;
  bool all_in_list;
  if (top_k > 0 && top_k < p.V) {
    cut = sm_cut<false>(row, s, 0, (double)top_k, all_in_list);
    if (all_in_list) {                             // the rest among these entries: a thread has one
      const int n = s.n;
      const u64 e = tid < n ? s.entry[tid] : 0;
      int rank = 0;
      if (tid < n) {
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += s.entry[j] > e;
      }
      const double w = tid < n && rank < top_k ? row.weight(sm_value(e)) : 0.0;
      const u64 mine = w > 0.0 ? row.whole(w) : 0;
      if (tid < n) s.weight[tid] = mine;
      u64 total;
      sm_before(mine, s.part, total);              // (its barrier is the one behind the weights too)
      u64 front = 0;
      if (top_p < 1.f && tid < n) {
#pragma unroll 4
        for (int j = 0; j < n; ++j) front += s.entry[j] > e ? s.weight[j] : 0;
      }
      const u64 stays = (!(top_p < 1.f) || (double)front < (double)top_p * (double)total) && !(w < (double)min_p) ? mine : 0;
      __syncthreads();
      if (tid < n) s.weight[tid] = stays;
      sm_before(stays, s.part, total);
      if (stays) {
        const u64 target = (u64)((double)u * (double)total);
        u64 before = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) before += (unsigned)s.entry[j] > (unsigned)e ? s.weight[j] : 0;      // of smaller indices
        if (before <= target && target < before + stays) p.out[b] = sm_index(e);
      }
      return;
    }
    __syncthreads();
  }
  if (top_p < 1.f) {
    cut = sm_cut<true>(row, s, cut, (double)top_p, all_in_list);
    __syncthreads();
  }
  // ---- sums of what stays, of every warp's vectors of a tile
  auto stays = [&](float a, int v) -> u64 {
    if (!row.there(v) || sm_entry(a, v) < cut) return 0;
    const double w = row.weight(a);
    return w < (double)min_p ? 0 : row.whole(w);
  };
#pragma unroll 1
  for (int t = 0; t < row.tiles; ++t) {
    float a[Row::VEC];
    row.vector(t * SM_THREADS + tid, a);
    u64 w = 0;
#pragma unroll
    for (int j = 0; j < Row::VEC; ++j) w += stays(a[j], (t * SM_THREADS + tid) * Row::VEC - row.off + j);
    w = sm_warp_sum(w);
    if (lane == 0) pieces[t * SM_WARPS + warp] = w;
  }
  __syncthreads();
  // ---- the piece in which u lies: a thread has some of them
  const int count = row.tiles * SM_WARPS, own = (count + SM_THREADS - 1) / SM_THREADS;
  u64 mine = 0, total;
  for (int i = 0; i < own; ++i) mine += tid * own + i < count ? pieces[tid * own + i] : 0;
  u64 before = sm_before(mine, s.part, total);
  const u64 target = (u64)((double)u * (double)total);
  for (int i = 0; i < own && tid * own + i < count; ++i) {
    const u64 w = pieces[tid * own + i];
    if (before <= target && target < before + w) {
      s.first = tid * own + i;
      s.above = before;
    }
    before += w;
  }
  __syncthreads();
  if (warp == 0) {
    float a[Row::VEC];
    const int i = s.first * 32 + lane;             // vectors of a tile stand in the threads' order
    row.vector(i, a);
    u64 w[Row::VEC], all = 0;
#pragma unroll
    for (int j = 0; j < Row::VEC; ++j) all += w[j] = stays(a[j], i * Row::VEC - row.off + j);
    u64 at = s.above + sm_warp_before(all);
#pragma unroll
    for (int j = 0; j < Row::VEC; ++j) {
      if (at <= target && target < at + w[j]) p.out[b] = i * Row::VEC - row.off + j;
      at += w[j];
    }
  }
}

template <typename T>
static int launch_sample(const SampleParams& p, long long B, cudaStream_t st) {
  constexpr int TILE = SampleRow<T>::TILE;
  const size_t smem = sizeof(SampleShared) + (size_t)((p.V + 16 + TILE - 1) / TILE) * SM_WARPS * sizeof(u64);
  static gf::SharedLimit limit;
  if (smem > 48 * 1024 && !limit.raise(sample_kernel<T>, smem)) return GFH_CUDA;
  sample_kernel<T><<<(unsigned)B, SM_THREADS, smem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
}

}  // namespace gf

using namespace gf;

GF_API int gf_sample_tokens(const SampleCall* c, void* stream) {
  if (!c || !c->x || !c->u || !c->out || c->B <= 0 || c->B > 0x7fffffff || c->V <= 0 || c->V > SM_MOST || c->dtype < 0 || c->dtype > 2) return GFH_BAD_ARG;
  gf::enter();
  int bits = 62;                                   // sums of V weights are below 2^62
  while (bits > 46 || (c->V >> (62 - bits)) > 0) --bits;
  const SampleParams p{c->x, c->ldx, c->u, c->temperature, c->top_p, c->min_p, c->top_k, (float)c->temperature0, (float)c->top_p0, (float)c->min_p0,
                       (int)c->top_k0, c->out, (int)c->V, bits};
  cudaStream_t st = (cudaStream_t)stream;
  return c->dtype == 0 ? launch_sample<float>(p, c->B, st) : c->dtype == 1 ? launch_sample<__nv_bfloat16>(p, c->B, st) : launch_sample<__half>(p, c->B, st);
}
