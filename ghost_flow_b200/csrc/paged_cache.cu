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
