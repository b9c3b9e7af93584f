// Attention of new tokens over a paged KV cache (see paged.cuh), grouped-query aware.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the keys j <= p of the token's sequence, p its position. One warp has one token and one query
// head, goes through the keys one by one and keeps the running maximum and sum.
#include "paged.cuh"

namespace gf {

struct PagedAttn {
  PagedBatch seqs;
  const __nv_bfloat16* q;        // [T, Hq, D], rows ldq apart
  long long ldq;
  const __nv_bfloat16 *kp, *vp;
  long long kpage, krow, khead, vpage, vrow, vhead;
  __nv_bfloat16* out;            // [T, Hq, D], rows ldo apart
  long long ldo;
  int Hq, Hkv;
  float scale_log2;
};

template <int D>
__global__ void __launch_bounds__(128) paged_attn_kernel(const __grid_constant__ PagedAttn p) {
  constexpr int E = D / 32;      // elements of a lane
  const PagedBatch& S = p.seqs;
  const int t = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int b = paged_seq_of(S, t);
  if (b >= S.B || h >= p.Hq) return;
  const int first = S.first(b), end = S.end(b);
  if (t < first || t >= end) return;
  const int len = S.lens[b], keys = (int)min((long long)max(len, 0), S.capacity());
  if (len != keys && lane == 0) S.bad();
  const int n = min(len - (end - first) + (t - first) + 1, keys), hk = h / (p.Hq / p.Hkv);
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(p.q[t * p.ldq + h * D + lane * E + e]);
    o[e] = 0.f;
  }
  for (int j = 0; j < n; ++j) {
    const int page = S.table[(long long)b * S.ld + (j >> S.page_shift)], r = j & ((1 << S.page_shift) - 1);
    const bool there = page >= 0 && page < S.pages;
    if (!there && lane == 0) S.bad();
    float x = 0.f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x += there ? q[e] * __bfloat162float(p.kp[page * p.kpage + r * p.krow + hk * p.khead + lane * E + e]) : 0.f;
      v[e] = there ? __bfloat162float(p.vp[page * p.vpage + r * p.vrow + hk * p.vhead + lane * E + e]) : 0.f;
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) x += __shfl_xor_sync(0xffffffffu, x, i);
    x *= p.scale_log2;
    const float mn = fmaxf(m, x), ref = mn == -INFINITY ? 0.f : mn, a = ex2_approx(m - ref), w = ex2_approx(x - ref);
    m = mn;
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * v[e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) p.out[t * p.ldo + h * D + lane * E + e] = __float2bfloat16(l > 0.f ? o[e] / l : 0.f);
}

}  // namespace gf

using namespace gf;

// q [T, Hq, D] and out alike, rows ldq and ldo elements apart; strides: pages, rows and heads of kpages, then of vpages, in elements.
GF_API int gf_paged_attn(const void* q, long long ldq, const void* kpages, const void* vpages, const long long* strides, const int* table,
                         int ld_table, int width, const int* lens, const int* cu, void* out, long long ldo, int B, int T, int Hq, int Hkv,
                         int D, int page, int pages, float scale, int* status, void* stream) {
  PagedAttn p;
  if (!paged_batch(p.seqs, table, ld_table, width, lens, cu, B, T, page, pages, status)) return GFH_BAD_ARG;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || (D != 64 && D != 128) || ldq % 8 || ldo % 8 || !strides) return GFH_BAD_ARG;
  for (const void* x : {q, kpages, vpages, (const void*)out})
    if (!x || (reinterpret_cast<uintptr_t>(x) & 15)) return GFH_BAD_ARG;
  for (int i = 0; i < 6; ++i)
    if (strides[i] % 8) return GFH_BAD_ARG;
  gf::enter();
  p.q = (const __nv_bfloat16*)q; p.ldq = ldq;
  p.kp = (const __nv_bfloat16*)kpages; p.vp = (const __nv_bfloat16*)vpages;
  p.kpage = strides[0]; p.krow = strides[1]; p.khead = strides[2];
  p.vpage = strides[3]; p.vrow = strides[4]; p.vhead = strides[5];
  p.out = (__nv_bfloat16*)out; p.ldo = ldo;
  p.Hq = Hq; p.Hkv = Hkv; p.scale_log2 = scale * 1.4426950408889634f;
  const dim3 grid(T, (Hq + 3) / 4);
  if (D == 128) paged_attn_kernel<128><<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  else paged_attn_kernel<64><<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
}
