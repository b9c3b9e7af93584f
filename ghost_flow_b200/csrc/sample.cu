// The next token of every row of logits, from a random number of each row: temperature, the k likeliest, the likeliest that hold a share p, those of
// at least min_p of the likeliest's probability.
//
// The reference picks the largest logit (ghostflow-nn/src/gpt.rs:402-422).
//
// With m the row's largest logit, w[v] = exp((x[v] - m) / T). Of the order by (x down, v up) the first k stay, of these each in front of which less than p of
// their sum stands, of these those with w >= min_p. The result is the first v, in the order of the vocabulary, up to which the sum of what stays exceeds u
// times all of it.
//
// Weights are whole numbers of 64 bits, w 2^46 rounded (2^45 from 2^17 entries on, 2^43 at the largest vocabulary): their sums do not depend on an order, so threads add
// them up as they come, and two runs agree to the bit. A border, a sum of at most V weights, is off by V / 2 units at most (2^-31 of the likeliest one's weight for 50257
// entries, 2^-24 for 2^20), and by the series' 2^-42 of itself. Exponentials are of 64 bits, as are shares and thresholds: with 32 the result of one row in some 10^4 would be
// another one's neighbour (a vocabulary of 50257 has that many borders, each off by some 2^-25). What is less than half of the last bit counts as nothing; u = 0, which takes the
// first token that stays whatever its weight, looks for that one.
//
// One CTA has a row, or a cluster of them where there are few, and reads it from L2 in every pass but the first: the largest entry; a histogram over bins of equal width of m - x, which says in which bin the k-th
// entry lies, or about where the share p ends; then, with top-k, all entries up to that bin go to shared memory, are put in order there, and the rest is done
// among them. Without it a pass adds up the weights: all, those in front of the bins around the place where the share may end, the latter by 32 parts of
// the vocabulary too, and leaves the entries of those bins in shared memory, among which the last one that stays is found. u then tells the part, and the
// token in it. What does not fit (more than 1024 entries, as with equal ones) takes as many histograms as it wants, by weights and then by the entries' bits, and
// entries that are all equal are counted off in the order of the vocabulary.
//
// What bounds it: the instructions of an entry's weight (a table of 16 powers and a series, 64 bits), of its bin and its atomic addition, not the 6.6 TB/s that
// the first pass reaches. 512 rows of 50257 in bf16, of which memory wants 8 us: the likeliest 17 us, weights of all 60, k = 50 48, p = 0.9 128, p of the least
// 35; 32 bits, 16 us: 22, 54, 51, 109, 31. 64 rows in bf16: 6, 19, 18, 38, 15; 3 rows of 32000: 5, 12, 14, 26, 12.
#include <cfloat>
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "calls.h"
#include "gf_host.h"
#include "gf_ptx.cuh"

namespace gf {

constexpr int SM_BINS = 2048;
constexpr int SM_MOST = 1 << 20;         // entries of a row

typedef unsigned long long u64;

struct SampleParams {
  const void* x;
  long long ldx;
  const float* u;                                   // [B]
  const float *temperature, *top_p, *min_p;         // [B] or null: the numbers below
  const int* top_k;
  double temperature0, top_p0, min_p0;
  int top_k0;
  long long* out;                                   // [B]
  int V, bits;                                      // a weight of 1 is 2^bits
  double series[5];                                 // (log(2) / 16)^n / n!, n from 1: operands that an instruction takes from here, not from registers
};

constexpr int SM_LIST = 1024;    // entries that are ordered in shared memory
constexpr int SM_PARTS = 32;     // of the vocabulary, whose sums lead to the token
constexpr int SM_RANKS = 8;      // CTAs of a row

struct SampleShared {
  unsigned bin[2][SM_BINS];        // low and high words of sums; or numbers, and how many there are in front
  u64 entry[SM_LIST], sorted[SM_LIST];
  u64 part[SM_PARTS];
  unsigned kept[2][SM_PARTS];
  double power[16];                // 2^(i / 16) 2^bits
  unsigned lo, hi;
  int n, first;
  u64 cut, above, total;
  unsigned critical;
  int b0, b1;
  // of every CTA that has a part of the row: its largest entry, some entries' sum and number, and sums of weights
  float most[SM_RANKS], sum[SM_RANKS];
  int numbers[SM_RANKS];
  u64 everything[SM_RANKS], in_front[SM_RANKS];
  u64 own[32];                   // of this CTA's warps
};

__device__ __forceinline__ float sm_f(float x) { return x; }
__device__ __forceinline__ float sm_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float sm_f(__half x) { return __half2float(x); }
// The larger one; what is not a number before all others.
__device__ __forceinline__ float sm_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Numbers in the order of the floats (zeros are one).
__device__ __forceinline__ unsigned sm_key(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
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
template <int THREADS>
__device__ __forceinline__ u64 sm_before(u64 v, u64* part, u64& all) {
  const u64 in_warp = sm_warp_before(v), last = __shfl_sync(0xffffffffu, in_warp + v, 31);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = last;
  __syncthreads();
  u64 before = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    if (i < (int)(threadIdx.x >> 5)) before += part[i];
    all += part[i];
  }
  return before + in_warp;
}

// The CTAs of a row: all of them meet, and the shared memory of another one.
__device__ __forceinline__ void sm_meet() { cooperative_groups::this_cluster().sync(); }
__device__ __forceinline__ SampleShared& sm_of(SampleShared& s, int rank) { return *cooperative_groups::this_cluster().map_shared_rank(&s, rank); }

template <typename T, int THREADS>
struct SampleRow {
  static constexpr int VEC = 16 / sizeof(T);
  const T* x;
  int V, head, vectors;          // whole vectors from entry `head` on, on 16-byte boundaries; the few entries around them are threads' own
  int per_part;                  // vectors of a part; what is in front of them is the first part's, what is behind the last one's
  int part0, part1;              // parts of this CTA
  float m, per_bin;
  double per16;                  // 16 log2(e) / T
  float zero;                    // entries below have no weight
  const double* power;
  const SampleParams& p;

  __device__ __forceinline__ SampleRow(const SampleParams& p_) : p(p_) {}

  __device__ __forceinline__ void begin(const T* x_, int V_) {
    x = x_;
    V = V_;
    head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)), V);
    vectors = (V - head) / VEC;
    per_part = (vectors + SM_PARTS - 1) / SM_PARTS;
  }
  __device__ __forceinline__ void share(int rank, int ranks) {
    part0 = rank * (SM_PARTS / ranks);
    part1 = part0 + SM_PARTS / ranks;
  }
  static constexpr bool ALONE = THREADS < 1024;    // a smaller CTA has the whole row always
  __device__ __forceinline__ int first() const { return ALONE ? 0 : min(part0 * per_part, vectors); }
  __device__ __forceinline__ int end() const { return ALONE ? vectors : min(part1 * per_part, vectors); }
  __device__ __forceinline__ int part_of(int v) const {
    const int i = (v - head) / VEC;
    return v < head ? 0 : i >= vectors ? SM_PARTS - 1 : (int)((unsigned)i / (unsigned)per_part);
  }
  __device__ __forceinline__ int edges() const { return V - vectors * VEC; }
  __device__ __forceinline__ int edge(int i) const { return i < head ? i : i + vectors * VEC; }
  // f(entries, index of the first): an array of VEC of them, or of one at the row's ends
  template <typename F>
  __device__ __forceinline__ void one(int v, F f) const {
    const float a[1] = {sm_f(x[v])};
    f(a, v);
  }
  __device__ __forceinline__ uint4 raw(int i) const { return __ldg(reinterpret_cast<const uint4*>(x + head) + i); }
  template <typename F>
  __device__ __forceinline__ void vector(const uint4& in, int i, F f) const {
    const T* have = reinterpret_cast<const T*>(&in);
    float a[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) a[j] = sm_f(have[j]);
    f(a, head + i * VEC);
  }
  // ... for vectors first, first + step .. below `end`, so many of a thread on their way together; of much work, the next one
  template <int TOGETHER, typename F>
  __device__ __forceinline__ void range(int first, int step, int end, F f) const {
    if constexpr (TOGETHER == 1) {
      uint4 next = make_uint4(0, 0, 0, 0);
      if (first < end) next = raw(first);
#pragma unroll 1
      for (int i = first; i < end; i += step) {
        const uint4 in = next;
        if (i + step < end) next = raw(i + step);
        vector(in, i, f);
      }
    } else {
#pragma unroll 1
      for (int i = first; i < end; i += TOGETHER * step) {
        uint4 in[TOGETHER];
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k)
          if (i + k * step < end) in[k] = raw(i + k * step);
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k)
          if (i + k * step < end) vector(in[k], i + k * step, f);
      }
    }
  }
  // ... for all entries of this CTA
  template <int TOGETHER, typename F>
  __device__ __forceinline__ void each(F f) const {
    range<TOGETHER>(first() + threadIdx.x, THREADS, end(), f);
    if ((int)threadIdx.x < edges() && (ALONE || ((int)threadIdx.x < head ? part0 == 0 : part1 == SM_PARTS))) one(edge(threadIdx.x), f);
  }
  // ... for those of a part, of which `warps` have as many each
  template <typename F>
  __device__ __forceinline__ void of_part(int part, int warp, int warps, F f) const {
    const int lane = threadIdx.x & 31;
    range<1>(part * per_part + warp * 32 + lane, 32 * warps, min((part + 1) * per_part, vectors), f);
    if (warp) return;
    if (part == 0 && lane < head) one(lane, f);
    if (part == SM_PARTS - 1 && head + lane < edges()) one(edge(head + lane), f);
  }
  // Whole CTA: the sums of what `f` adds to `mine`, of each of its parts, into `to`. Behind the next barrier.
  template <typename F>
  __device__ __forceinline__ void sums(SampleShared& s, SampleShared& to, u64& mine, F f) const {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, parts = part1 - part0;
    if (!ALONE && parts < SM_PARTS) {              // a cluster's CTA: several warps to a part
      const int warps = THREADS / 32 / parts;
      mine = 0;
      of_part(part0 + warp / warps, warp % warps, warps, f);
      mine = sm_warp_sum(mine);
      if (lane == 0) s.own[warp] = mine;
      __syncthreads();
      if ((int)threadIdx.x >= parts) return;
      mine = 0;
      for (int i = 0; i < warps; ++i) mine += s.own[threadIdx.x * warps + i];
      to.kept[0][part0 + threadIdx.x] = (unsigned)mine;
      to.kept[1][part0 + threadIdx.x] = (unsigned)(mine >> 32);
      return;
    }
    for (int part = warp; part < SM_PARTS; part += THREADS / 32) {
      mine = 0;
      of_part(part, 0, 1, f);
      mine = sm_warp_sum(mine);
      if (lane == 0) {
        to.kept[0][part] = (unsigned)mine;
        to.kept[1][part] = (unsigned)(mine >> 32);
      }
    }
  }
  // bins of equal width, the further from the largest entry the higher
  __device__ __forceinline__ int bin(float a) const {
    const float t = fminf(fmaf(m - a, per_bin, 8388608.f), 8388608.f + (SM_BINS - 1));     // 2^23 + a whole number
    return __float_as_uint(t) & (SM_BINS - 1);
  }
  // w 2^bits, w = 2^((a - m) log2(e) / T), of entries from `zero` on: sixteenths of the exponent from a table, what is left of it, at most 2^-5, by the series of
  // the exponential function up to its fifth power (the sixth is 2^-42 of it), rounded to a whole number. Without branches: a chain of
  // a dozen operations of 64 bits is hidden by the other entries of a vector. The exponent ends at -52 (by its upper word: it is never above 0), not the entry at one of 32 bits:
  // at a small temperature numbers next to each other are further apart than that.
  __device__ __forceinline__ u64 weight(float a) const {
    constexpr double MAGIC = 6755399441055744.0;               // 1.5 2^52: what is added to it is a whole number in the low bits
    const double far = ((double)a - (double)m) * per16;                    // (0 of the largest, whose weight is 2^bits)
    const double t = __hiloint2double((int)min((unsigned)__double2hiint(far), 0xc08a0000u), __double2loint(far));       // -52 16 = -1.625 2^9
    const double n = t + MAGIC;
    const int i = __double2loint(n);
    const double r = t - (n - MAGIC);
    const double e = fma(fma(fma(fma(fma(p.series[4], r, p.series[3]), r, p.series[2]), r, p.series[1]), r, p.series[0]), r, 1.0) * power[i & 15];
    const double w = __hiloint2double(__double2hiint(e) + ((i & ~15) << 16), __double2loint(e)) + 4503599627370496.0;       // 2^52
    return __double_as_longlong(w) & 0xfffffffffffffull;
  }
  // The least entry with w >= p.
  __device__ __forceinline__ float least(double p, double temperature) const {
    return p > 0 ? fmaxf(__double2float_ru((double)m + temperature * log(p)), -INFINITY) : -INFINITY;      // (all, of an infinite temperature)
  }
};

// Where the order ends: the last entry (see sm_entry) that stays of those from `from` on (0: of all), by numbers (the first `share` ones) or by weights (up
// to a `share` of their sum).
template <bool WEIGHTS, typename T, int THREADS>
__device__ u64 sm_cut(const SampleRow<T, THREADS>& row, SampleShared& s, u64 from, double share) {
  constexpr int LIST = 256;                        // each of these is compared with all others
  const int tid = threadIdx.x;
  unsigned lo = 0, hi = 0xffffffffu;               // keys that are looked at
  int bin0 = -1;                                   // and, behind the first level, the bin
  unsigned top = 0;
  int shift = 0;
  u64 above = 0;
  double target = share;
  // what an earlier choice has left out, or has no weight
  const float from_value = fmaxf(from ? sm_value(from) : -INFINITY, WEIGHTS ? row.zero : -INFINITY);
  const int from_index = from && sm_value(from) == from_value ? sm_index(from) : 0x7fffffff;
  auto behind = [&](float a, int v) { return a <= from_value && (a < from_value || v > from_index); };
  auto looked_at = [&](float a, int v) {
    const unsigned k = sm_key(a);
    return !behind(a, v) && row.bin(a) == bin0 && k >= lo && k <= hi;
  };
  while (true) {
    // ---- the bins
    for (int i = tid; i < 2 * SM_BINS; i += THREADS) s.bin[0][i] = 0;
    if (tid == 0) s.n = 0;
    __syncthreads();
    auto count = [&](unsigned b, u64 w) {
      const unsigned low = (unsigned)w, old = atomicAdd(&s.bin[0][b], low), high = (unsigned)(w >> 32) + (old + low < old);
      if (high) atomicAdd(&s.bin[1][b], high);
    };
    if (bin0 < 0) {
      row.template each<WEIGHTS ? 1 : 2>([&](auto& a, int v0) {
        constexpr int N = sizeof(a) / sizeof(float);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const unsigned b = row.bin(a[j]);
          if constexpr (WEIGHTS) {
            const u64 w = row.weight(a[j]);
            if (!behind(a[j], v0 + j)) count(b, w);
          } else {
            if (b < SM_BINS - 1) atomicAdd(&s.bin[0][b], 1u);              // (those in the last bin are what is left)
          }
        }
      });
    } else {
      row.template each<1>([&](auto& a, int v0) {
#pragma unroll
        for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j)
          if (looked_at(a[j], v0 + j)) count((top - sm_key(a[j])) >> shift, WEIGHTS ? row.weight(a[j]) : 1);
      });
    }
    __syncthreads();
    constexpr int OWN = SM_BINS / THREADS;
    u64 own[OWN], sum = 0, total;
#pragma unroll
    for (int i = 0; i < OWN; ++i) sum += own[i] = (u64)s.bin[1][tid * OWN + i] << 32 | s.bin[0][tid * OWN + i];
    u64 before = sm_before<THREADS>(sum, s.part, total) + above;
    if (!WEIGHTS && bin0 < 0 && tid == THREADS - 1) own[OWN - 1] = row.V - total;
    if (WEIGHTS && bin0 < 0) target = share * (double)total;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      if ((double)before < target && (double)(before + own[i]) >= target) {
        s.critical = tid * OWN + i;
        s.above = before;
      }
      before += own[i];
    }
    __syncthreads();
    const unsigned b = s.critical;
    above = s.above;
    // ---- its entries
    if (bin0 < 0) {
      bin0 = (int)b;
    } else {
      hi = top - (b << shift);
      lo = hi - ((1u << shift) - 1);
    }
    row.template each<2>([&](auto& a, int v0) {
#pragma unroll
      for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j) {
        const int bin = row.bin(a[j]);
        if (bin == bin0 && looked_at(a[j], v0 + j)) {
          const int at = atomicAdd(&s.n, 1);
          if (at < LIST) s.entry[at] = sm_entry(a[j], v0 + j);
        }
      }
    });
    __syncthreads();
    const int n = s.n;
    if (n <= LIST) {
      if (WEIGHTS) {
        if (tid < n) s.sorted[tid] = row.weight(sm_value(s.entry[tid]));
        __syncthreads();
      }
      if (tid < n) {
        const u64 e = s.entry[tid];
        u64 front = above;
#pragma unroll 4
        for (int j = 0; j < n; ++j)
          if (s.entry[j] > e) front += WEIGHTS ? s.sorted[j] : 1;
        if ((double)front < target && (double)(front + (WEIGHTS ? s.sorted[tid] : 1)) >= target) s.cut = e;
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
    row.template each<2>([&](auto& a, int v0) {
#pragma unroll
      for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j) {
        if (!looked_at(a[j], v0 + j)) continue;
        least = min(least, sm_key(a[j]));
        most = max(most, sm_key(a[j]));
      }
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
  const float value = sm_value((u64)hi << 32);
  const u64 each = WEIGHTS ? row.weight(value) : 1;
  u64 take = (u64)fmax(1.0, ceil((target - (double)above) / (double)each));
  while (take > 1 && (double)(above + (take - 1) * each) >= target) --take;
  while ((double)(above + take * each) < target) ++take;
  // those in front of the vectors, then a vector to a thread at a time, then those behind
  u64 seen = 0;
  const int rounds = (row.vectors + THREADS - 1) / THREADS;
  for (int t = -1; t <= rounds && seen < take; ++t) {
    unsigned hit = 0;
    int first = 0;
    auto look = [&](auto& a, int v0) {
      first = v0;
#pragma unroll
      for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j)
        if (a[j] == value && !behind(a[j], v0 + j)) hit |= 1u << j;
    };
    if (t < 0) {
      if (tid < row.head) row.one(tid, look);
    } else if (t == rounds) {
      if (row.head + tid < row.edges()) row.one(row.edge(row.head + tid), look);
    } else if (t * THREADS + tid < row.vectors) {
      row.vector(row.raw(t * THREADS + tid), t * THREADS + tid, look);
    }
    u64 all, before = seen + sm_before<THREADS>(__popc(hit), s.part, all);
    for (; hit; hit &= hit - 1)
      if (++before == take) s.cut = sm_entry(value, first + __ffs(hit) - 1);
    seen += all;
    __syncthreads();
  }
  return s.cut;
}

// Whole warp: the part of the vocabulary that holds u of the sum of all parts, that number, and the sums in front of the part.
struct SamplePart {
  int part;
  u64 target, front;
  __device__ __forceinline__ SamplePart(const SampleShared& s, float u) {
    const int lane = threadIdx.x & 31;
    const u64 own = (u64)s.kept[1][lane] << 32 | s.kept[0][lane], before = sm_warp_before(own);
    target = (u64)((double)u * (double)__shfl_sync(0xffffffffu, before + own, 31));
    part = __ffs(__ballot_sync(0xffffffffu, before <= target && target < before + own)) - 1;
    front = __shfl_sync(0xffffffffu, before, part);
  }
};
static_assert(SM_PARTS == 32, "a lane has a part");

// Numbers of entries in every bin, and of those in front; the last bin, which reaches to the least entry, is not counted. In the first CTA of the row; the
// others have their own, and stay until the next barrier of all.
template <bool MANY, typename T, int THREADS>
__device__ void sm_count(const SampleRow<T, THREADS>& row, SampleShared& s, int rank, int ranks) {
  constexpr int OWN = SM_BINS / THREADS;
  const int tid = threadIdx.x;
  for (int i = tid; i < SM_BINS; i += THREADS) s.bin[0][i] = 0;
  __syncthreads();
  row.template each<2>([&](auto& a, int) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j) {
      const int b = row.bin(a[j]);
      if (b < SM_BINS - 1) atomicAdd(&s.bin[0][b], 1u);
    }
  });
  if (MANY && ranks > 1) sm_meet();
  else __syncthreads();
  if (MANY && rank) return;
  unsigned own[OWN], sum = 0;
#pragma unroll
  for (int i = 0; i < OWN; ++i) own[i] = s.bin[0][tid * OWN + i];
  for (int r = 1; MANY && r < ranks; ++r) {
#pragma unroll
    for (int i = 0; i < OWN; ++i) own[i] += sm_of(s, r).bin[0][tid * OWN + i];
  }
#pragma unroll
  for (int i = 0; i < OWN; ++i) sum += own[i];
  u64 all;
  unsigned before = (unsigned)sm_before<THREADS>(sum, s.part, all);
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    s.bin[0][tid * OWN + i] = own[i];
    s.bin[1][tid * OWN + i] = before;
    before += own[i];
  }
  __syncthreads();
}

// An entry of bins b0 .. b1, which have at most SM_LIST, into the list behind those of the bins in front.
template <typename T, int THREADS>
__device__ __forceinline__ void sm_keep(const SampleRow<T, THREADS>& row, SampleShared& s, float a, int v, int bin, int b0) {
  s.entry[s.bin[1][bin] - s.bin[1][b0] + atomicSub(&s.bin[0][bin], 1u) - 1] = sm_entry(a, v);        // (s: the first CTA's)
}
// Whole CTA: the list's n entries, from bin b0 on, in their order: an entry is compared with those of its bin.
template <typename T, int THREADS>
__device__ void sm_sort(const SampleRow<T, THREADS>& row, SampleShared& s, int n, int b0) {
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const u64 e = s.entry[i];
    const int b = row.bin(sm_value(e)), first = s.bin[1][b] - s.bin[1][b0], end = min(n, (int)(s.bin[1][b + 1] - s.bin[1][b0]));
    int rank = first;
    for (int j = first; j < end; ++j) rank += s.entry[j] > e;
    s.sorted[rank] = e;
  }
  __syncthreads();
}

// Whole CTA: the smallest index for which `f(entry, index)`; -1 where there is none.
template <typename T, int THREADS, typename F>
__device__ int sm_first(const SampleRow<T, THREADS>& row, SampleShared& s, F f) {
  if (threadIdx.x == 0) s.first = 0x7fffffff;
  __syncthreads();
  int best = 0x7fffffff;
  row.template each<2>([&](auto& a, int v0) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j)
      if (f(a[j], v0 + j)) best = min(best, v0 + j);
  });
  best = __reduce_min_sync(0xffffffffu, best);
  if ((threadIdx.x & 31) == 0) atomicMin(&s.first, best);
  __syncthreads();
  return s.first == 0x7fffffff ? -1 : s.first;
}

// A row has one CTA, or, where there are SMs for it, a cluster of them, each with as many of the row's parts: those help the first one with the passes over the
// row, leave what they find in its shared memory, and are done; what follows, and what is seldom wanted, is the first one's alone. They meet (sm_meet) as often
// as each other: what they go by is the same for all of them.
template <typename T, int THREADS, bool MANY>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) sample_kernel(const __grid_constant__ SampleParams p) {
  constexpr int WARPS = THREADS / 32;
  using Row = SampleRow<T, THREADS>;
  __shared__ SampleShared s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int rank = 0, ranks = 1;
  if (MANY) {
    rank = (int)cooperative_groups::this_cluster().block_rank();
    ranks = (int)cooperative_groups::this_cluster().num_blocks();
    cooperative_groups::this_cluster().barrier_arrive();
  }
  const long long b = blockIdx.x / ranks;
  Row row(p);
  row.begin((const T*)p.x + b * p.ldx, p.V);
  row.share(rank, ranks);
  const double temperature = p.temperature ? p.temperature[b] : p.temperature0;
  const double top_p = p.top_p ? p.top_p[b] : p.top_p0;
  const double min_p = fmin(p.min_p ? p.min_p[b] : p.min_p0, 1.0);
  const int top_k = p.top_k ? p.top_k[b] : p.top_k0;
  const float u = fminf(fmaxf(p.u[b], 0.f), 0x1.fffffep-1f);
  if (warp == WARPS - 1 && lane < 16) s.power[lane] = exp2(lane / 16.0) * (double)(1ull << p.bits);

  // ---- the largest entry, and the mean of some that are numbers
  float most = -INFINITY, sum = 0.f;
  int numbers = 0;
  row.template each<4>([&](auto& a, int) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j) most = sm_max(most, a[j]);
  });
  if (row.first() + tid < row.end()) row.vector(row.raw(row.first() + tid), row.first() + tid, [&](auto& a, int) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j) {
      const bool number = fabsf(a[j]) < 0x1p100f;
      sum += number ? a[j] : 0.f;
      numbers += number;
    }
  });
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    most = sm_max(most, __shfl_xor_sync(0xffffffffu, most, o));
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  numbers = __reduce_add_sync(0xffffffffu, numbers);
  float* f = reinterpret_cast<float*>(s.entry);
  int* n = reinterpret_cast<int*>(s.sorted);
  if (lane == 0) {
    f[warp] = most;
    f[WARPS + warp] = sum;
    n[warp] = numbers;
  }
  __syncthreads();
  most = -INFINITY, sum = 0.f, numbers = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    most = sm_max(most, f[i]);
    sum += f[WARPS + i];
    numbers += n[i];
  }
  if (MANY) {
    cooperative_groups::this_cluster().barrier_wait();               // (all of them run)
    if (tid < ranks) {
      SampleShared& to = sm_of(s, tid);
      to.most[rank] = most;
      to.sum[rank] = sum;
      to.numbers[rank] = numbers;
    }
    sm_meet();
    most = -INFINITY, sum = 0.f, numbers = 0;
    for (int i = 0; i < ranks; ++i) {
      most = sm_max(most, s.most[i]);
      sum += s.sum[i];
      numbers += s.numbers[i];
    }
  }
  SampleShared& s0 = MANY ? sm_of(s, 0) : s;          // the first CTA's
  // ---- rows without probabilities, and those whose likeliest entry is asked for
  if (!(fabsf(most) < INFINITY) || !(temperature > 0) || top_k == 1 || top_p <= 0) {
    if (MANY && rank) return;
    row.share(0, 1);
    const bool none = most != most;
    const int v = most == -INFINITY ? -1 : sm_first(row, s, [&](float a, int) { return none ? a != a : a == most; });
    if (tid == 0) p.out[b] = v;
    return;
  }
  row.m = most;
  row.per16 = fmax(16.0 * 1.4426950408889634 / temperature, 1e-300);        // (of an infinite one too: minus infinity stays so)
  // half of 2^-1074, the least number of 64 bits, is none: 1075 log(2). Minus infinity has no weight at any temperature.
  row.zero = fmaxf(__double2float_ru((double)most - 745.1332191019412 * temperature), -FLT_MAX);
  row.power = s.power;
  // Bins of numbers reach three quarters of the way to the mean, which some of the first entries stand for; those of weights twice as far. What is further away lies in
  // the last.
  const float reach = most - sum / (float)max(numbers, 1);
  const float per = reach > 0x1p-60f && reach < 0x1p100f ? (float)(SM_BINS - 1) / reach : 1.f;
  __syncthreads();

  u64 cut = 0;
  const float least_p = row.least(min_p, temperature);
  if (top_k > 0 && top_k < p.V) {
    row.per_bin = per * (4.f / 3.f);
    sm_count<MANY>(row, s, rank, ranks);
    // ---- the bin that the k-th entry lies in; -1 where there are more entries up to it than the list has room for
    if (rank == 0) {
      if (tid == 0) s.b1 = -1;
      if (tid < SM_PARTS) s.kept[0][tid] = s.kept[1][tid] = 0;
      __syncthreads();
      for (int i = tid; i < SM_BINS - 1; i += THREADS)
        if (s.bin[1][i] < (unsigned)top_k && s.bin[1][i + 1] >= (unsigned)top_k && s.bin[1][i + 1] <= SM_LIST) s.b1 = i;
    }
    if (MANY && ranks > 1) sm_meet();
    else __syncthreads();
    const int b1 = s0.b1;
    if (b1 >= 0) {
      // ---- all of them into the list; the rest happens there
      row.template each<2>([&](auto& a, int v0) {
#pragma unroll
        for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j) {
          const int bin = row.bin(a[j]);
          if (bin <= b1) sm_keep(row, s0, a[j], v0 + j, bin, 0);
        }
      });
      if (MANY && ranks > 1) sm_meet();
      if (MANY && rank) return;
      const int n = (int)s.bin[1][b1 + 1];
      sm_sort(row, s, n, 0);
      constexpr int OWN = SM_LIST / THREADS;       // a thread's entries, next to each other
      u64 e[OWN], w[OWN], sum = 0, total;
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int at = tid * OWN + i;
        e[i] = at < top_k && at < n ? s.sorted[at] : 0;
        w[i] = e[i] && sm_value(e[i]) >= row.zero ? row.weight(sm_value(e[i])) : 0;
        sum += w[i];
      }
      u64 before = sm_before<THREADS>(sum, s.part, total);
      const double target = top_p * (double)total;
      int lowest = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const u64 front = before;
        before += w[i];
        if (!e[i] || sm_value(e[i]) < row.zero || (top_p < 1 && !((double)front < target)) || sm_value(e[i]) < least_p) w[i] = 0;
        else lowest = min(lowest, sm_index(e[i]));
        if (w[i] == 0) continue;
        const int part = row.part_of(sm_index(e[i]));
        const unsigned low = (unsigned)w[i], old = atomicAdd(&s.kept[0][part], low), high = (unsigned)(w[i] >> 32) + (old + low < old);
        if (high) atomicAdd(&s.kept[1][part], high);
      }
      if (tid == 0) {
        s.n = 0;
        s.first = 0x7fffffff;
      }
      __syncthreads();
      if (u == 0.f) {                              // the first that stays
        atomicMin(&s.first, lowest);
        __syncthreads();
        if (tid == 0) p.out[b] = s.first;
        return;
      }
      const SamplePart at(s, u);
      // ---- the part's own: each is compared with all of them
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        if (w[i] == 0 || row.part_of(sm_index(e[i])) != at.part) continue;
        const int to = atomicAdd(&s.n, 1);
        s.entry[to] = e[i];
        s.sorted[to] = w[i];
      }
      __syncthreads();
      for (int i = tid; i < s.n; i += THREADS) {
        const int v = sm_index(s.entry[i]);
        u64 front = at.front;
        for (int j = 0; j < s.n; ++j) front += sm_index(s.entry[j]) < v ? s.sorted[j] : 0;
        if (front <= at.target && at.target < front + s.sorted[i]) p.out[b] = v;
      }
      return;
    }
    if (MANY && ranks > 1) sm_meet();                      // (its shared memory has been read)
    if (MANY && rank) return;
    row.share(0, 1);
    ranks = 1;
    cut = sm_cut<false>(row, s, 0, (double)top_k);
    __syncthreads();
  }
  u64 mine = 0;                                    // of this warp's part
  bool summed = false;
  if (top_p < 1) {
    row.per_bin = per * 0.5f;
    if (cut == 0) {
      // ---- by the bins' numbers and middles, about where the share ends
      sm_count<MANY>(row, s, rank, ranks);
      if (rank == 0) {
        constexpr int OWN = SM_BINS / THREADS;
        float own[OWN], sum = 0.f;
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
          const int at = tid * OWN + i;
          const float middle = row.m - at / row.per_bin;
          own[i] = at < SM_BINS - 1 ? (float)(s.bin[1][at + 1] - s.bin[1][at]) * exp2f((middle - row.m) * (float)(row.per16 / 16.0)) : 0.f;
          sum += own[i];
        }
        // (as whole numbers, of which the scan is)
        u64 all, before = sm_before<THREADS>((u64)(sum * 0x1p20f), s.part, all);
        const u64 target = (u64)(top_p * (double)all);
        if (tid == 0) s.critical = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
          const u64 upto = before + (u64)(own[i] * 0x1p20f);
          if (before <= target && target < upto) s.critical = tid * OWN + i;
          before = upto;
        }
        __syncthreads();
        // as many of them around it as there is room for, 31 on both sides at most (it is hardly ever that far off)
        const int about = min((int)s.critical, SM_BINS - 2), b0_ = max(about - lane, 0), b1_ = min(about + lane, SM_BINS - 2);
        const unsigned fits = __ballot_sync(0xffffffffu, s.bin[1][b1_ + 1] - s.bin[1][b0_] <= SM_LIST);
        const int wide = 31 - __clz(fits);
        if (tid == 0) {
          s.b0 = max(about - wide, 0);
          s.b1 = fits ? min(about + wide, SM_BINS - 2) : -1;
        }
      }
      if (MANY && ranks > 1) sm_meet();
      else __syncthreads();
      const int b0 = s0.b0, b1 = s0.b1;
      if (b1 < 0) {
        if (MANY && ranks > 1) sm_meet();                  // (as above)
        if (MANY && rank) return;
        row.share(0, 1);
        ranks = 1;
      } else {
        // ---- all weights, those in front of the list, those of each part; the list
        u64 everything = 0, in_front = 0;
        auto take = [&](auto& a, int v0) {
#pragma unroll 4
          for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j) {
            const u64 w = row.weight(a[j]);
            const int bin = row.bin(a[j]);
            if (a[j] >= row.zero) everything += w;
            if (bin < b0) {
              in_front += w;
              if (a[j] >= least_p) mine += w;
            } else if (bin <= b1) {
              sm_keep(row, s0, a[j], v0 + j, bin, b0);
            }
          }
        };
        row.sums(s, s0, mine, take);
        u64 total, front;
        sm_before<THREADS>(everything, s.part, total);
        __syncthreads();
        sm_before<THREADS>(in_front, s.part, front);
        if (MANY && ranks > 1) {
          if (tid == 0) {
            s0.everything[rank] = total;
            s0.in_front[rank] = front;
          }
          sm_meet();
          if (MANY && rank) return;
          total = front = 0;
          for (int i = 0; i < ranks; ++i) {
            total += s.everything[i];
            front += s.in_front[i];
          }
          row.share(0, 1);
          ranks = 1;
        }
        const int n = (int)(s.bin[1][b1 + 1] - s.bin[1][b0]);
        sm_sort(row, s, n, b0);
        // ---- the entry of the list at which the share ends
        constexpr int OWN_LIST = SM_LIST / THREADS;
        u64 w[OWN_LIST], sum = 0, list;
#pragma unroll
        for (int i = 0; i < OWN_LIST; ++i) {
          const int at = tid * OWN_LIST + i;
          w[i] = at < n && sm_value(s.sorted[at]) >= row.zero ? row.weight(sm_value(s.sorted[at])) : 0;
          sum += w[i];
        }
        u64 before = front + sm_before<THREADS>(sum, s.part, list);
        const double share = top_p * (double)total;
        if ((double)front < share && (double)(front + list) >= share) {      // else it lies elsewhere, and is looked for in another way
#pragma unroll
          for (int i = 0; i < OWN_LIST; ++i) {
            if (w[i] && (double)before < share) {
              const u64 e = s.sorted[tid * OWN_LIST + i];
              if ((double)(before + w[i]) >= share) s.cut = e;
              if (sm_value(e) >= least_p) {
                const int part = row.part_of(sm_index(e));
                const unsigned low = (unsigned)w[i], old = atomicAdd(&s.kept[0][part], low), high = (unsigned)(w[i] >> 32) + (old + low < old);
                if (high) atomicAdd(&s.kept[1][part], high);
              }
            }
            before += w[i];
          }
          summed = true;
        }
        __syncthreads();
        if (summed) cut = s.cut;
      }
    }
    if (!summed) {
      cut = sm_cut<true>(row, s, cut, (double)top_p);
      __syncthreads();
    }
  }
  // ---- sums of what stays, of every part
  const float cut_value = cut ? sm_value(cut) : -INFINITY, least = fmaxf(fmaxf(cut_value, row.zero), least_p);
  const int cut_index = cut && cut_value == least ? sm_index(cut) : 0x7fffffff;             // of entries as large as the last one, the last that stays
  const float next = sm_value((u64)(sm_key(least) + 1) << 32);
  auto from = [&](int v) { return v > cut_index ? next : least; };         // the least that stays
  auto add = [&](auto& a, int v0) {
    constexpr int N = sizeof(a) / sizeof(float);
    float largest = a[0];
#pragma unroll
    for (int j = 1; j < N; ++j) largest = fmaxf(largest, a[j]);
    if (largest < least) return;
#pragma unroll 4
    for (int j = 0; j < N; ++j) {
      const u64 w = row.weight(a[j]);
      if (a[j] >= from(v0 + j)) mine += w;
    }
  };
  if (!summed) {
    row.sums(s, s0, mine, add);
    if (MANY && ranks > 1) sm_meet();
    else __syncthreads();
    if (MANY && rank) return;
  }
  if (u == 0.f) {                                  // the first that stays
    row.share(0, 1);
    const int v = sm_first(row, s, [&](float a, int v) { return a >= from(v); });
    if (tid == 0) p.out[b] = v;
    return;
  }
  const SamplePart here(s, u);
  // ---- the part in which u lies, cut among all threads: vectors next to each other, the first thread with those in front of all vectors, the last with those
  // behind
  const int part = here.part, first = part * row.per_part, end = max(first, min(first + row.per_part, row.vectors)), own = (end - first + THREADS - 1) / THREADS;
  const int i0 = min(first + tid * own, end), i1 = min(i0 + own, end);
  auto walk = [&](auto f) {
    if (part == 0 && tid == 0)
      for (int v = 0; v < row.head; ++v) row.one(v, f);
    for (int i = i0; i < i1; ++i) row.vector(row.raw(i), i, f);
    if (part == SM_PARTS - 1 && tid == THREADS - 1)
      for (int i = row.head; i < row.edges(); ++i) row.one(row.edge(i), f);
  };
  mine = 0;
  walk(add);
  u64 all, before = here.front + sm_before<THREADS>(mine, s.part, all);
  if (before <= here.target && here.target < before + mine)
    walk([&](auto& a, int v0) {
#pragma unroll 1
      for (int j = 0; j < (int)(sizeof(a) / sizeof(float)); ++j) {
        const u64 x = a[j] >= from(v0 + j) ? row.weight(a[j]) : 0;
        if (before <= here.target && here.target < before + x) p.out[b] = v0 + j;
        before += x;
      }
    });
}

template <typename T>
static int launch_sample(const SampleParams& p, long long B, cudaStream_t st) {
  // Several CTAs to a row where it is long and there are SMs for them: clusters of 4 and 8 find room on seven and six of eight SMs. us with 1 / 2 / 4 / 8, the
  // weights of all entries wanted and a share of 0.9: 3 rows of 32000 15, 33 / 14, 30 / 13, 26 / 12, 26; 8 of 128256 34, 71 / 25, 52 / 18, 40 / 15, 35; 64 of
  // 50257 20, 43 / 18, 38; 4 of 16384 11, 23 / 13, 25 / 12, 25 / 12, 26. Where a cluster has to wait for another one: 16 of 128256 19, 40 with 4, 25, 54 with 8.
  const int sms = sm_count();
  if (B > sms) {
    sample_kernel<T, 512, false><<<(unsigned)B, 512, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
  }
  // The likeliest entries alone, one pass, gain nothing: 8 of 128256 10 with one, 12 with 8.
  const bool likeliest = !p.temperature && !(p.temperature0 > 0);
  int ranks = 1;
  while (!likeliest && ranks < SM_RANKS && p.V >= max(12000, 6000 * ranks) * 2 && 2 * ranks * B * 8 <= sms * (ranks == 4 ? 6 : ranks == 2 ? 7 : 8)) ranks *= 2;
  if (ranks == 1) {
    sample_kernel<T, 1024, false><<<(unsigned)B, 1024, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
  }
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * ranks));
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, sample_kernel<T, 1024, true>, p) != cudaSuccess) return GFH_CUDA;
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
}

}  // namespace gf

using namespace gf;

GF_API int gf_sample_tokens(const SampleCall* c, void* stream) {
  if (!c || !c->x || !c->u || !c->out || c->B <= 0 || c->B > 0x7fffffff || c->V <= 0 || c->V > SM_MOST || c->dtype < 0 || c->dtype > 2) return GFH_BAD_ARG;
  gf::enter();
  int bits = 46;                                   // sums of V weights are 2^63 at most
  while (c->V > 1ll << (63 - bits)) --bits;
  constexpr double C1 = 0.69314718055994530942 / 16;
  const SampleParams p{c->x, c->ldx, c->u, c->temperature, c->top_p, c->min_p, c->top_k, c->temperature0, c->top_p0, c->min_p0,
                       (int)c->top_k0, c->out, (int)c->V, bits, {C1, C1 * C1 / 2, C1 * C1 * C1 / 6, C1 * C1 * C1 * C1 / 24, C1 * C1 * C1 * C1 * C1 / 120}};
  cudaStream_t st = (cudaStream_t)stream;
  return c->dtype == 0 ? launch_sample<float>(p, c->B, st) : c->dtype == 1 ? launch_sample<__nv_bfloat16>(p, c->B, st) : launch_sample<__half>(p, c->B, st);
}
