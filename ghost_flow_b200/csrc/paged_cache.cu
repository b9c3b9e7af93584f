// New keys and values of a packed projection into a paged KV cache, with the rotation of q and k on the way.
//
// The reference has no KV cache (ghostflow-nn/src/gpt.rs:402-422 runs the whole prefix again for every token).
//
// q'[a] = q[a] cos(p f) - q[b] sin(p f), q'[b] = q[b] cos(p f) + q[a] sin(p f) for the pair (a, b) = (d, d + D / 2), or (2 d, 2 d + 1)
// where pairs lie next to each other; k alike, v is copied. In 32 bits from bf16, rounded once. Memory is all that counts: every row is
// read once and written once, and the rows of the tables once a token. One CTA has one token: a thread has the same 16 elements of every
// head it works on (8 pairs, two vectors), so it reads its part of the tables once, and all its loads are on their way before it knows where
// the token goes. 4500 tokens of five prompts, 32 / 32 heads of 128: 39 us, 5.9 TB/s; one token of each of 64 sequences 2.6 us, three looks into memory
// one behind the other (lengths, page, table rows). What a call costs is then its launch.
//
// Heads that are normed or rotated in part, and pages of 8 bits, have a kernel of their own (the one without them is as it was): the same CTA to a token, with
// D / 16 neighbouring lanes to a head (norm_rope.cuh), whose sum of squares, and largest number, are shuffles. Rows read back are written out as bf16, which
// has all of their bits from 2^-133 on. The same five prompts with norms into pages of 8 bits, and read back: 49 and 24 us (185 and 112 MB, of which 28 and 17; with the vectors of a lane far apart 81 together);
// 64 sequences of one token 3.0 and 2.5. Issue slots are 62 % taken: a number is normed, rotated, compared and rounded to 8 bits by itself.
#include <type_traits>

#include "norm_rope.cuh"
#include "paged.cuh"

namespace gf {

constexpr int PA_THREADS = 256;
constexpr int PA_AHEAD = 3;      // pieces of a thread whose loads are in flight together

struct PagedAppend {
  PagedBatch seqs;
  const __nv_bfloat16* qkv;      // [T, H + 2 Hk, D], rows ldx apart
  long long ldx;
  __nv_bfloat16 *q, *kp, *vp;    // [T, H, D] dense; [pages, page, Hk, D]
  long long kpage, krow, khead, vpage, vrow, vhead;   // strides
  const float *cos, *sin;        // [positions, D / 2]
  int H, Hk, D, positions, interleaved;
};

// 8 pairs: halves x, y (half-split), or 8 neighbours each (interleaved)
__device__ __forceinline__ void rotate16(uint4& x, uint4& y, const float (&c)[8], const float (&s)[8], bool interleaved) {
  uint32_t *a = reinterpret_cast<uint32_t*>(&x), *b = reinterpret_cast<uint32_t*>(&y);
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 u = unpack_bf16x2(a[i]), v = unpack_bf16x2(b[i]);
      a[i] = pack_bf16x2(u.x * c[i] - u.y * s[i], u.y * c[i] + u.x * s[i]);
      b[i] = pack_bf16x2(v.x * c[i + 4] - v.y * s[i + 4], v.y * c[i + 4] + v.x * s[i + 4]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 u = unpack_bf16x2(a[i]), v = unpack_bf16x2(b[i]);
      a[i] = pack_bf16x2(u.x * c[2 * i] - v.x * s[2 * i], u.y * c[2 * i + 1] - v.y * s[2 * i + 1]);
      b[i] = pack_bf16x2(v.x * c[2 * i] + u.x * s[2 * i], v.y * c[2 * i + 1] + u.y * s[2 * i + 1]);
    }
  }
}

__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const __grid_constant__ PagedAppend p) {
  const PagedBatch& S = p.seqs;
  const int t = blockIdx.x, per = p.D / 16;                      // pieces of a head
  const int step = PA_THREADS / per;                             // heads that the CTA works on at a time
  const int head0 = threadIdx.x / per, i = threadIdx.x - head0 * per, heads = p.H + 2 * p.Hk;
  const bool works = head0 < step;                               // D need not divide the threads
  const int at = p.interleaved ? 16 * i : 8 * i, far = p.interleaved ? 8 : p.D / 2;
  const __nv_bfloat16* row = p.qkv + (long long)t * p.ldx + at;
  uint4 x[PA_AHEAD], y[PA_AHEAD];
  auto load = [&](int h0) {
#pragma unroll
    for (int n = 0; n < PA_AHEAD; ++n) {
      const int h = h0 + n * step;
      if (works && h < heads) {
        x[n] = *reinterpret_cast<const uint4*>(row + (long long)h * p.D);
        y[n] = *reinterpret_cast<const uint4*>(row + (long long)h * p.D + far);
      }
    }
  };
  load(head0);
  const int b = paged_seq_of(S, t);
  if (b >= S.B) return;                                          // behind the last sequence
  const int first = S.first(b), end = S.end(b);
  if (t < first || t >= end) return;
  const int pos = S.lens[b] - (end - first) + (t - first);       // < 0: a sequence without this token (an empty slot of a batch)
  bool there = pos >= 0;
  if (there && (pos >= S.capacity() || pos >= p.positions)) {
    if (threadIdx.x == 0) S.bad();
    there = false;
  }
  int page = 0;
  if (there) page = S.table[(long long)b * S.ld + (pos >> S.page_shift)];
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    const long long off = (long long)pos * (p.D / 2) + 8 * i + e;
    const float4 u = there ? *reinterpret_cast<const float4*>(p.cos + off) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 v = there ? *reinterpret_cast<const float4*>(p.sin + off) : make_float4(0.f, 0.f, 0.f, 0.f);
    c[e] = u.x; c[e + 1] = u.y; c[e + 2] = u.z; c[e + 3] = u.w;
    s[e] = v.x; s[e + 1] = v.y; s[e + 2] = v.z; s[e + 3] = v.w;
  }
  const bool stored = there && page >= 0 && page < S.pages;
  if (there && !stored && threadIdx.x == 0) S.bad();
  const int r = pos & ((1 << S.page_shift) - 1);
  __nv_bfloat16* q = p.q + (long long)t * p.H * p.D + at;
  __nv_bfloat16* k = p.kp + page * p.kpage + r * p.krow + at;
  __nv_bfloat16* v = p.vp + page * p.vpage + r * p.vrow + at;
  for (int h0 = head0; h0 < heads; h0 += PA_AHEAD * step) {
    if (h0 != head0) load(h0);
#pragma unroll
    for (int n = 0; n < PA_AHEAD; ++n) {
      const int h = h0 + n * step;
      if (!works || h >= heads) continue;
      __nv_bfloat16* to;
      if (h < p.H + p.Hk) {
        rotate16(x[n], y[n], c, s, p.interleaved);
        if (!there) x[n] = y[n] = make_uint4(0, 0, 0, 0);        // not the products of what stands there
        to = h < p.H ? q + (long long)h * p.D : k + (h - p.H) * p.khead;
      } else {
        to = v + (h - p.H - p.Hk) * p.vhead;
      }
      if (h < p.H || stored) {
        *reinterpret_cast<uint4*>(to) = x[n];
        *reinterpret_cast<uint4*>(to + far) = y[n];
      }
    }
  }
}

struct PagedHeads {
  PagedAppend a;                 // pools and strides are of bytes where there are scales
  const __nv_bfloat16 *qw, *kw;  // [D]; null: no norms
  unsigned char *kscales, *vscales;
  float eps;
  int rotary;
};

// Where a new token's row is.
struct PagedRow {
  long long page;
  int pos, r;                    // position, row of the page
  bool there, stored;            // the token has a position; its row is in the pools
};
// Whole CTA; false for tokens behind the last sequence. `positions`: those that there are tables for.
__device__ __forceinline__ bool paged_row(const PagedBatch& S, int t, int positions, PagedRow& row) {
  const int b = paged_seq_of(S, t);
  if (b >= S.B) return false;
  const int first = S.first(b), end = S.end(b);
  if (t < first || t >= end) return false;
  row.pos = S.lens[b] - (end - first) + (t - first);
  row.there = row.pos >= 0;
  bool bad = row.there && (row.pos >= S.capacity() || row.pos >= positions);
  if (bad) row.there = false;
  row.page = row.there ? S.table[(long long)b * S.ld + (row.pos >> S.page_shift)] : 0;
  row.stored = row.there && row.page >= 0 && row.page < S.pages;
  bad |= row.there && !row.stored;
  if (bad && threadIdx.x == 0) S.bad();
  row.r = row.pos & ((1 << S.page_shift) - 1);
  return true;
}

__device__ __forceinline__ unsigned short e4m3x2(float lo, float hi) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// 8 numbers in a unit of `inv`^-1.
__device__ __forceinline__ uint2 e4m3x8(const uint64_t* x, float inv) {
  const uint64_t two = pk2f(inv, inv);
  unsigned short h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t y = f2_mul(x[i], two);
    h[i] = e4m3x2(lo2(y), hi2(y));
  }
  return make_uint2(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16);
}
template <int LANES>
__device__ __forceinline__ unsigned group_max(unsigned v) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// Whole warp: the byte of a row's power of two. What is not finite becomes NaN, which the type has, and counts for nothing.
template <int LANES>
__device__ __forceinline__ unsigned scale_byte(Head16& v) {
  constexpr unsigned INF = 0x7f800000u;
  float most = 0.f;                                // (what is not a number is passed over, and stays so in the conversion)
#pragma unroll
  for (int e = 0; e < 8; ++e) most = fmaxf(most, fmaxf(fabsf(lo2(v.x[e])), fabsf(hi2(v.x[e]))));
  unsigned m = group_max<LANES>(__float_as_uint(most));
  if (__any_sync(0xffffffffu, m >= INF)) {
    most = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = lo2(v.x[e]), b = hi2(v.x[e]);
      v.x[e] = pk2f(a + (a - a), b + (b - b));
      most = fmaxf(most, fmaxf(fabsf(lo2(v.x[e])), fabsf(hi2(v.x[e]))));
    }
    m = group_max<LANES>(__float_as_uint(most));
  }
  // m = 1.f 2^(E - 127), 448 = 1.75 2^8
  return (unsigned)max(1, (int)(m >> 23) - 8 + ((m & 0x7fffffu) > 0x600000u));
}

template <int LANES, bool BYTES>
__global__ void __launch_bounds__(PA_THREADS, 3) paged_append_heads_kernel(const __grid_constant__ PagedHeads p) {
  constexpr int D = 16 * LANES, STEP = PA_THREADS / LANES;
  const PagedAppend& A = p.a;
  const int t = blockIdx.x, head0 = threadIdx.x / LANES, i = threadIdx.x % LANES, heads = A.H + 2 * A.Hk;
  const HeadLane at(i, LANES, p.rotary, A.interleaved);
  const __nv_bfloat16* from = A.qkv + (long long)t * A.ldx;
  uint4 x[PA_AHEAD], y[PA_AHEAD];
  auto load = [&](int h0) {
#pragma unroll
    for (int n = 0; n < PA_AHEAD; ++n) {
      const int h = h0 + n * STEP;
      x[n] = y[n] = make_uint4(0, 0, 0, 0);
      if (h < heads) {
        x[n] = *reinterpret_cast<const uint4*>(from + (long long)h * D + at.x);
        y[n] = *reinterpret_cast<const uint4*>(from + (long long)h * D + at.y);
      }
    }
  };
  load(head0);
  PagedRow row;
  if (!paged_row(A.seqs, t, A.positions, row)) return;
  HeadTurn turn;
  const long long off = (long long)row.pos * (p.rotary / 2);
  turn.of(A.cos + off, A.sin + off, at, row.there);
  for (int base = 0; base < heads; base += PA_AHEAD * STEP) {              // (the same for all lanes of a warp)
    if (base) load(base + head0);
#pragma unroll
    for (int n = 0; n < PA_AHEAD; ++n) {
      const int h = base + head0 + n * STEP;
      const bool query = h < A.H, key = !query && h < A.H + A.Hk;
      if (!__any_sync(0xffffffffu, h < heads)) break;
      Head16 v;
      v.of(x[n], y[n]);
      if (p.qw) {
        const float r = rsqrtf(group_sum<LANES>(v.dot(v)) * (1.f / D) + p.eps);
        if (query || key) {
          Head16 w;
          const __nv_bfloat16* weight = query ? p.qw : p.kw;
          w.of(__ldg(reinterpret_cast<const uint4*>(weight + at.x)), __ldg(reinterpret_cast<const uint4*>(weight + at.y)));
          v.scale(r);
          v.scale(w);
        }
      }
      if (query || key) turn.turn<1>(v, at, A.interleaved);
      if (query) {
        v.to(x[n], y[n]);
        if (!row.there) x[n] = y[n] = make_uint4(0, 0, 0, 0);              // not the products of what stands there
        __nv_bfloat16* to = A.q + ((long long)t * A.H + h) * D;
        *reinterpret_cast<uint4*>(to + at.x) = x[n];
        *reinterpret_cast<uint4*>(to + at.y) = y[n];
        if constexpr (!BYTES) continue;
      }
      unsigned byte = 0;
      if constexpr (BYTES) {                       // (rows of queries have been written: what is not finite in them stays what it is)
        if (!__any_sync(0xffffffffu, !query)) continue;
        byte = scale_byte<LANES>(v);
      }
      if (query || !row.stored || h >= heads) continue;
      const int hk = h - A.H - (key ? 0 : A.Hk);
      const long long to = key ? row.page * A.kpage + row.r * A.krow + hk * A.khead : row.page * A.vpage + row.r * A.vrow + hk * A.vhead;
      if constexpr (BYTES) {
        unsigned char* pool = reinterpret_cast<unsigned char*>(key ? A.kp : A.vp) + to;
        const float inv = __uint_as_float((254u - byte) << 23);
        *reinterpret_cast<uint2*>(pool + at.x) = e4m3x8(v.x, inv);
        *reinterpret_cast<uint2*>(pool + at.y) = e4m3x8(v.x + 4, inv);
        if (i == 0) (key ? p.kscales : p.vscales)[((row.page * A.Hk + hk) << A.seqs.page_shift) + row.r] = (unsigned char)byte;
      } else {
        __nv_bfloat16* pool = (key ? A.kp : A.vp) + to;
        v.to(x[n], y[n]);
        *reinterpret_cast<uint4*>(pool + at.x) = x[n];
        *reinterpret_cast<uint4*>(pool + at.y) = y[n];
      }
    }
  }
}

struct PagedRead {
  PagedBatch seqs;
  const void *kp, *vp;
  const unsigned char *kscales, *vscales;
  __nv_bfloat16 *k, *v;          // [T, Hk, D] dense
  long long kpage, krow, khead, vpage, vrow, vhead;
  int Hk, D, shift;              // D = 16 << shift
};

template <bool BYTES>
__global__ void __launch_bounds__(PA_THREADS) paged_read_kernel(const __grid_constant__ PagedRead p) {
  const int t = blockIdx.x, all = 2 * p.Hk << p.shift;
  PagedRow row{};
  if (!paged_row(p.seqs, t, 0x7fffffff, row)) row.stored = false;
  for (int id = threadIdx.x; id < all; id += PA_THREADS) {
    const int i = id & ((1 << p.shift) - 1), head = id >> p.shift;
    const bool key = head < p.Hk;
    const int hk = key ? head : head - p.Hk;
    const long long from = key ? row.page * p.kpage + row.r * p.krow + hk * p.khead : row.page * p.vpage + row.r * p.vrow + hk * p.vhead;
    uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (row.stored) {
      if constexpr (BYTES) {
        const uint4 in = *reinterpret_cast<const uint4*>((const unsigned char*)(key ? p.kp : p.vp) + from + 16 * i);
        const unsigned byte = (key ? p.kscales : p.vscales)[((row.page * p.Hk + hk) << p.seqs.page_shift) + row.r];
        bf16x16_of_e4m3(in, pk2(byte << 23, byte << 23), x[0], x[1]);
      } else {
        const uint4* in = reinterpret_cast<const uint4*>((const __nv_bfloat16*)(key ? p.kp : p.vp) + from + 16 * i);
        x[0] = in[0];
        x[1] = in[1];
      }
    }
    uint4* to = reinterpret_cast<uint4*>((key ? p.k : p.v) + ((long long)t * p.Hk + hk) * p.D + 16 * i);
    to[0] = x[0];
    to[1] = x[1];
  }
}

}  // namespace gf

using namespace gf;

// x [T, H + 2 Hk, D], y [T, H, D] dense. GFH_OVERLAP where x shares memory with the pools. Tables fp32 [positions, D / 2] dense, on 16-byte boundaries.
GF_API int gf_paged_append(const PagedCall* c, const float* cos, const float* sin, int positions, int interleaved, void* stream) {
  PagedAppend p;
  if (!c || !paged_batch(p.seqs, *c)) return GFH_BAD_ARG;
  const long long H = c->H, Hk = c->Hk, D = c->D;
  if (H <= 0 || Hk <= 0 || H > 65535 || Hk > 65535 || D < 16 || D % 16 || D / 16 > PA_THREADS || positions < 0 || c->ldy != H * D ||
      !cos || !sin || ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15))
    return GFH_BAD_ARG;
  // new tokens are read while others are written to the pages
  const char *x0 = (const char*)c->x, *x1 = x0 + 2 * ((c->T - 1) * c->ldx + (H + 2 * Hk) * D);
  for (int i = 0; i < 2; ++i) {
    const long long* st = c->strides + 3 * i;
    const char* pool = (const char*)(i ? c->vpages : c->kpages);
    if (c->pages > 0 && x0 < pool + 2 * ((c->pages - 1) * st[0] + (c->page - 1) * st[1] + (Hk - 1) * st[2] + D) && pool < x1) return GFH_OVERLAP;
  }
  gf::enter();
  p.qkv = (const __nv_bfloat16*)c->x; p.ldx = c->ldx;
  p.q = (__nv_bfloat16*)c->y; p.kp = (__nv_bfloat16*)c->kpages; p.vp = (__nv_bfloat16*)c->vpages;
  p.kpage = c->strides[0]; p.krow = c->strides[1]; p.khead = c->strides[2];
  p.vpage = c->strides[3]; p.vrow = c->strides[4]; p.vhead = c->strides[5];
  p.cos = cos; p.sin = sin;
  p.H = (int)H; p.Hk = (int)Hk; p.D = (int)D; p.positions = positions; p.interleaved = interleaved;
  paged_append_kernel<<<p.seqs.T, PA_THREADS, 0, (cudaStream_t)stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
}

// The same with heads that are normed (qw, kw [D]; null: not) and of which `rotary` dims are rotated (tables [positions, rotary / 2]), into pages of bf16 (no
// scales) or of 8 bits. GFH_OVERLAP where x shares memory with the pools or scales, or these with each other. D of 32, 64, 128 or 256.
GF_API int gf_paged_append_heads(const PagedCall8* c8, const float* cos, const float* sin, int positions, int rotary, int interleaved, const void* qw,
                                 const void* kw, float eps, void* stream) {
  PagedHeads p{};
  if (!c8 || !paged_batch(p.a.seqs, c8->c) || !c8->kscales != !c8->vscales || (c8->kscales && !paged_scales(*c8))) return GFH_BAD_ARG;
  const PagedCall* c = &c8->c;
  const long long H = c->H, Hk = c->Hk, D = c->D, size = c8->kscales ? 1 : 2;
  if (H <= 0 || Hk <= 0 || H > 65535 || Hk > 65535 || (D != 32 && D != 64 && D != 128 && D != 256) || positions < 0 || c->ldy != H * D || rotary < 0 ||
      rotary > D || rotary % 16 || !qw != !kw || ((reinterpret_cast<uintptr_t>(qw) | reinterpret_cast<uintptr_t>(kw)) & 15) ||
      (rotary && (!cos || !sin)) || ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15))
    return GFH_BAD_ARG;
  // new tokens are read while others are written to the pages
  const char *x0 = (const char*)c->x, *x1 = x0 + 2 * ((c->T - 1) * c->ldx + (H + 2 * Hk) * D);
  for (int i = 0; i < 2; ++i) {
    const long long* st = c->strides + 3 * i;
    const char *pool = (const char*)(i ? c->vpages : c->kpages), *scales = (const char*)(i ? c8->vscales : c8->kscales);
    if (c->pages > 0 && x0 < pool + size * ((c->pages - 1) * st[0] + (c->page - 1) * st[1] + (Hk - 1) * st[2] + D) && pool < x1) return GFH_OVERLAP;
    if (scales && x0 < scales + c->pages * c->page * Hk && scales < x1) return GFH_OVERLAP;
  }
  if (c8->kscales && c->pages > 0 && !paged_scales_apart(*c8)) return GFH_OVERLAP;
  gf::enter();
  PagedAppend& a = p.a;
  a.qkv = (const __nv_bfloat16*)c->x; a.ldx = c->ldx;
  a.q = (__nv_bfloat16*)c->y; a.kp = (__nv_bfloat16*)c->kpages; a.vp = (__nv_bfloat16*)c->vpages;
  a.kpage = c->strides[0]; a.krow = c->strides[1]; a.khead = c->strides[2];
  a.vpage = c->strides[3]; a.vrow = c->strides[4]; a.vhead = c->strides[5];
  a.cos = cos; a.sin = sin;
  a.H = (int)H; a.Hk = (int)Hk; a.D = (int)D; a.positions = positions; a.interleaved = interleaved;
  p.qw = (const __nv_bfloat16*)qw; p.kw = (const __nv_bfloat16*)kw; p.eps = eps; p.rotary = rotary;
  p.kscales = (unsigned char*)c8->kscales; p.vscales = (unsigned char*)c8->vscales;
  auto of = [&](auto bytes) {
    constexpr bool B = decltype(bytes)::value;
    return D == 32 ? paged_append_heads_kernel<2, B> : D == 64 ? paged_append_heads_kernel<4, B> : D == 128 ? paged_append_heads_kernel<8, B>
                                                                                                           : paged_append_heads_kernel<16, B>;
  };
  auto kern = c8->kscales ? of(std::true_type{}) : of(std::false_type{});
  kern<<<a.seqs.T, PA_THREADS, 0, (cudaStream_t)stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
}

// Rows of the new tokens out of the pages: k, v [T, Hk, D] dense bf16, zeros for tokens that have none. x and y of the call are not looked at.
GF_API int gf_paged_read(const PagedCall8* c8, void* k, void* v, void* stream) {
  PagedRead p{};
  if (!c8 || !k || !v || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) return GFH_BAD_ARG;
  PagedCall c = c8->c;
  c.x = c.y = k;
  c.ldx = c.ldy = 0;
  if (!paged_batch(p.seqs, c) || !c8->kscales != !c8->vscales || (c8->kscales && !paged_scales(*c8)) || c.Hk <= 0 || c.Hk > 65535 || c.D < 16 || (c.D & (c.D - 1)) ||
      c.D > 4096)
    return GFH_BAD_ARG;
  gf::enter();
  p.kp = c.kpages; p.vp = c.vpages; p.kscales = c8->kscales; p.vscales = c8->vscales;
  p.k = (__nv_bfloat16*)k; p.v = (__nv_bfloat16*)v;
  p.kpage = c.strides[0]; p.krow = c.strides[1]; p.khead = c.strides[2];
  p.vpage = c.strides[3]; p.vrow = c.strides[4]; p.vhead = c.strides[5];
  p.Hk = (int)c.Hk; p.D = (int)c.D; p.shift = __builtin_ctz((unsigned)c.D) - 4;
  auto kern = c8->kscales ? paged_read_kernel<true> : paged_read_kernel<false>;
  kern<<<p.seqs.T, PA_THREADS, 0, (cudaStream_t)stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
}
