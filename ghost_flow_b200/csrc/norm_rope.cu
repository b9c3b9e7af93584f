// RMS norms of the query and key heads of a packed projection with the rotation in the same pass, and their gradients.
//
// The reference normalises whole rows only (ghostflow-nn/src/llama.rs:154-185) and rotates in a pass of its own (llama.rs:208-252).
//
// y = rot(x r w), r = (mean x^2 + eps)^(-1/2), for each head of q and k. With g = rot^-1(dy) and d = g w: dx = r (d - x r mean(d x r)),
// dw = sum of g x r over all tokens and heads; the gradient of v is copied beside them. In 32 bits from bf16, rounded once; r is worked out again by the
// backward pass, which reads x anyway. Memory is all that counts: every row is read once and written once.
//
// A warp has a token and some of its heads, D / 16 lanes to a head (norm_rope.cuh), so it reads its rows of the tables once for all of them. dw: a warp of the
// backward pass keeps its sums in registers over all its tokens, a CTA leaves them in a row of a scratch buffer, and a second kernel, on the machine
// before the first one ends, adds the rows up in a fixed order.
#include "gf_host.h"
#include "norm_rope.cuh"

namespace gf {

constexpr int NR_THREADS = 256, NR_WARPS = NR_THREADS / 32;
constexpr int NR_ROWS = 2;       // of a lane on their way together
constexpr int NR_BWD_CTAS = 2;   // on an SM, which stay for all tokens

struct NormRope {
  const __nv_bfloat16* x;        // [T, H + 2 Hk, D], rows ldx apart
  long long ldx;
  const __nv_bfloat16 *qw, *kw;  // [D]; null: heads are rotated only
  const float *cos, *sin;        // [positions, rotary / 2]
  __nv_bfloat16 *q, *k;          // forward: [T, H, D], [T, Hk, D] dense
  const __nv_bfloat16 *dq, *dk, *dv;               // backward: rows ldq, ldk, ldv apart
  long long ldq, ldk, ldv;
  __nv_bfloat16* dx;             // [T, H + 2 Hk, D] dense
  float* part;                   // [CTAs][2][D]
  long long units;
  int H, Hk, S, pos0, rotary, interleaved, per, chunks;        // heads of a unit, units of a token
  float eps;
};

struct NrUnit {
  long long t;
  int h0, h1, pos;
};
__device__ __forceinline__ NrUnit nr_unit(const NormRope& p, long long u, int heads) {
  NrUnit n;
  n.t = u / p.chunks;
  n.h0 = (int)(u - n.t * p.chunks) * p.per;
  n.h1 = min(n.h0 + p.per, heads);
  n.pos = (int)(n.t % p.S) + p.pos0;
  return n;
}

template <int LANES>
__global__ void __launch_bounds__(NR_THREADS) norm_rope_kernel(const __grid_constant__ NormRope p) {
  constexpr int D = 16 * LANES, GROUPS = 32 / LANES;
  const int lane = threadIdx.x & 31, group = lane / LANES;
  const HeadLane at(lane % LANES, p.rotary, p.interleaved);
  const long long u = (long long)blockIdx.x * NR_WARPS + (threadIdx.x >> 5);
  if (u >= p.units) return;
  const NrUnit n = nr_unit(p, u, p.H + p.Hk);
  const __nv_bfloat16* row = p.x + n.t * p.ldx;
  float c[8], s[8];
  const long long off = (long long)n.pos * (p.rotary / 2) + at.t;
  table8(p.cos + off, at.turns, c);
  table8(p.sin + off, at.turns, s);
  for (int h0 = n.h0 + group; __any_sync(0xffffffffu, h0 < n.h1); h0 += NR_ROWS * GROUPS) {
    uint4 x[NR_ROWS], y[NR_ROWS];
#pragma unroll
    for (int i = 0; i < NR_ROWS; ++i) {
      const int h = h0 + i * GROUPS;
      x[i] = y[i] = make_uint4(0, 0, 0, 0);
      if (h < n.h1) {
        x[i] = *reinterpret_cast<const uint4*>(row + (long long)h * D + at.x);
        y[i] = *reinterpret_cast<const uint4*>(row + (long long)h * D + at.y);
      }
    }
#pragma unroll
    for (int i = 0; i < NR_ROWS; ++i) {
      const int h = h0 + i * GROUPS;
      Head16 v, w;
      v.of(x[i], y[i]);
      if (p.qw) {
        const __nv_bfloat16* weight = h < p.H ? p.qw : p.kw;
        w.of(__ldg(reinterpret_cast<const uint4*>(weight + at.x)), __ldg(reinterpret_cast<const uint4*>(weight + at.y)));
        const float r = rsqrtf(group_sum<LANES>(v.dot(v)) * (1.f / D) + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v.a[e] *= r * w.a[e];
          v.b[e] *= r * w.b[e];
        }
      }
      if (at.turns) v.turn<1>(c, s, p.interleaved);
      v.to(x[i], y[i]);
      if (h < n.h1) {
        __nv_bfloat16* to = h < p.H ? p.q + (n.t * p.H + h) * D : p.k + (n.t * p.Hk + h - p.H) * D;
        *reinterpret_cast<uint4*>(to + at.x) = x[i];
        *reinterpret_cast<uint4*>(to + at.y) = y[i];
      }
    }
  }
}

template <int LANES>
__global__ void __launch_bounds__(NR_THREADS, NR_BWD_CTAS) norm_rope_bwd_kernel(const __grid_constant__ NormRope p) {
  constexpr int D = 16 * LANES, GROUPS = 32 / LANES;
  __shared__ float sums[NR_WARPS][2][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = lane / LANES, heads = p.H + 2 * p.Hk;
  if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const HeadLane at(lane % LANES, p.rotary, p.interleaved);
  Head16 dw[2];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[0].a[e] = dw[0].b[e] = dw[1].a[e] = dw[1].b[e] = 0.f;
  for (long long u = (long long)blockIdx.x * NR_WARPS + warp; u < p.units; u += (long long)gridDim.x * NR_WARPS) {
    const NrUnit n = nr_unit(p, u, heads);
    const __nv_bfloat16* row = p.x + n.t * p.ldx;
    __nv_bfloat16* to = p.dx + n.t * heads * D;
    float c[8], s[8];
    const long long off = (long long)n.pos * (p.rotary / 2) + at.t;
    table8(p.cos + off, at.turns, c);
    table8(p.sin + off, at.turns, s);
    for (int h0 = n.h0 + group; __any_sync(0xffffffffu, h0 < n.h1); h0 += NR_ROWS * GROUPS) {
      uint4 x[NR_ROWS], y[NR_ROWS], gx[NR_ROWS], gy[NR_ROWS];
#pragma unroll
      for (int i = 0; i < NR_ROWS; ++i) {
        const int h = h0 + i * GROUPS;
        x[i] = y[i] = gx[i] = gy[i] = make_uint4(0, 0, 0, 0);
        if (h < n.h1) {
          const __nv_bfloat16* g = h < p.H ? p.dq + n.t * p.ldq + h * D : h < p.H + p.Hk ? p.dk + n.t * p.ldk + (h - p.H) * D
                                                                                        : p.dv + n.t * p.ldv + (h - p.H - p.Hk) * D;
          gx[i] = *reinterpret_cast<const uint4*>(g + at.x);
          gy[i] = *reinterpret_cast<const uint4*>(g + at.y);
          if (p.qw && h < p.H + p.Hk) {
            x[i] = *reinterpret_cast<const uint4*>(row + (long long)h * D + at.x);
            y[i] = *reinterpret_cast<const uint4*>(row + (long long)h * D + at.y);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NR_ROWS; ++i) {
        const int h = h0 + i * GROUPS;
        Head16 v, g, w;
        v.of(x[i], y[i]);
        g.of(gx[i], gy[i]);
        if (at.turns) g.turn<-1>(c, s, p.interleaved);
        if (p.qw) {
          const bool query = h < p.H;
          const __nv_bfloat16* weight = query ? p.qw : p.kw;
          w.of(__ldg(reinterpret_cast<const uint4*>(weight + at.x)), __ldg(reinterpret_cast<const uint4*>(weight + at.y)));
          const float r = rsqrtf(group_sum<LANES>(v.dot(v)) * (1.f / D) + p.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v.a[e] *= r;
            v.b[e] *= r;
            const float da = g.a[e] * v.a[e], db = g.b[e] * v.b[e];          // (of v, and of heads that are not there: zeros)
            dw[0].a[e] += query ? da : 0.f;
            dw[0].b[e] += query ? db : 0.f;
            dw[1].a[e] += query ? 0.f : da;
            dw[1].b[e] += query ? 0.f : db;
            g.a[e] *= w.a[e];
            g.b[e] *= w.b[e];
          }
          const float mean = group_sum<LANES>(g.dot(v)) * (1.f / D);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            g.a[e] = r * (g.a[e] - v.a[e] * mean);
            g.b[e] = r * (g.b[e] - v.b[e] * mean);
          }
        }
        if (h < p.H + p.Hk) g.to(gx[i], gy[i]);
        if (h < n.h1) {
          *reinterpret_cast<uint4*>(to + (long long)h * D + at.x) = gx[i];
          *reinterpret_cast<uint4*>(to + (long long)h * D + at.y) = gy[i];
        }
      }
    }
  }
  if (!p.qw) return;
  // ---- the weights' gradients: groups, then warps
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float v = e < 8 ? dw[i].a[e & 7] : dw[i].b[e & 7];
#pragma unroll
      for (int o = 16; o >= LANES; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (group == 0) sums[warp][i][(e < 8 ? at.x : at.y) + (e & 7)] = v;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += NR_THREADS) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NR_WARPS; ++w) v += sums[w][i / D][i % D];
    p.part[(long long)blockIdx.x * 2 * D + i] = v;
  }
}

// 32 columns to a CTA, 32 threads to a column.
__global__ void __launch_bounds__(1024) norm_rope_fold_kernel(const float* part, int rows, int D, __nv_bfloat16* dqw, __nv_bfloat16* dkw) {
  __shared__ float sums[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x % 32, first = threadIdx.x / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float v = 0.f;
#pragma unroll 4
  for (int r = first; r < rows; r += 32) v += part[(long long)r * 2 * D + col];
  sums[first][threadIdx.x % 32] = v;
  __syncthreads();
  v = sums[threadIdx.x % 32][first];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x % 32 == 0) {
    const int c = blockIdx.x * 32 + first;
    (c < D ? dqw : dkw)[c % D] = __float2bfloat16(v);
  }
}

// Units of a token: parts of its heads, so many that there are some warps for every place on the machine, each of four rounds at least where it has them.
static void nr_cut(NormRope& p, long long T, int heads, int lanes) {
  const int round = 32 / lanes * NR_ROWS;
  const long long rounds = (heads + round - 1) / round, want = (sm_count() * 64ll + T - 1) / T;
  const long long most = want > rounds / 4 ? want : rounds / 4;
  p.chunks = (int)(most < 1 ? 1 : most < rounds ? most : rounds);
  p.per = (int)((rounds + p.chunks - 1) / p.chunks) * round;
  p.chunks = (heads + p.per - 1) / p.per;
  p.units = T * p.chunks;
}

static bool nr_sizes(long long T, int S, int H, int Hk, int D, int rotary) {
  return T > 0 && T <= 0x7fffffff && S > 0 && T % S == 0 && H > 0 && Hk > 0 && H <= 65535 && Hk <= 65535 && (D == 32 || D == 64 || D == 128 || D == 256) &&
         rotary >= 0 && rotary <= D && rotary % 16 == 0;
}

static bool nr_weights(const void* qw, const void* kw) {
  return !qw == !kw && !((reinterpret_cast<uintptr_t>(qw) | reinterpret_cast<uintptr_t>(kw)) & 15);
}

}  // namespace gf

using namespace gf;

// x [T, H + 2 Hk, D] with rows ldx apart, T = sequences * S; q [T, H, D] and k [T, Hk, D] dense. Tables fp32 [positions, rotary / 2] dense, of which rows pos0 ..
// pos0 + S - 1 are there. All on 16-byte boundaries.
GF_API int gf_norm_rope_qkv(const void* x, long long ldx, const void* qw, const void* kw, const float* cos, const float* sin, void* q, void* k, long long T,
                            int S, int H, int Hk, int D, int rotary, int pos0, int interleaved, float eps, void* stream) {
  if (!nr_sizes(T, S, H, Hk, D, rotary) || pos0 < 0 || ldx % 8 || ldx < (H + Hk) * (long long)D) return GFH_BAD_ARG;
  for (const void* a : {x, (const void*)q, (const void*)k})
    if (!a || (reinterpret_cast<uintptr_t>(a) & 15)) return GFH_BAD_ARG;
  if (!nr_weights(qw, kw)) return GFH_BAD_ARG;
  if (rotary && (!cos || !sin || ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15))) return GFH_BAD_ARG;
  gf::enter();
  NormRope p{};
  p.x = (const __nv_bfloat16*)x; p.ldx = ldx; p.qw = (const __nv_bfloat16*)qw; p.kw = (const __nv_bfloat16*)kw; p.cos = cos; p.sin = sin;
  p.q = (__nv_bfloat16*)q; p.k = (__nv_bfloat16*)k;
  p.H = H; p.Hk = Hk; p.S = S; p.pos0 = pos0; p.rotary = rotary; p.interleaved = interleaved; p.eps = eps;
  nr_cut(p, T, H + Hk, D / 16);
  const long long ctas = (p.units + NR_WARPS - 1) / NR_WARPS;
  if (ctas > 0x7fffffffll) return GFH_TOO_LARGE;
  auto kern = D == 32 ? norm_rope_kernel<2> : D == 64 ? norm_rope_kernel<4> : D == 128 ? norm_rope_kernel<8> : norm_rope_kernel<16>;
  kern<<<(unsigned)ctas, NR_THREADS, 0, (cudaStream_t)stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
}

// Floats of scratch of the backward pass.
GF_API int gf_norm_rope_scratch(int D) {
  gf::bind();
  return sm_count() * NR_BWD_CTAS * 2 * D;
}

// dq [T, H, D], dk, dv [T, Hk, D] with rows lds[0 .. 2] apart, heads packed; dx [T, H + 2 Hk, D] dense; dqw, dkw [D] bf16. The rest as above.
GF_API int gf_norm_rope_qkv_bwd(const void* x, long long ldx, const void* qw, const void* kw, const float* cos, const float* sin, const void* dq,
                                const void* dk, const void* dv, const long long* lds, void* dx, void* dqw, void* dkw, float* scratch, long long T, int S,
                                int H, int Hk, int D, int rotary, int pos0, int interleaved, float eps, void* stream) {
  if (!nr_sizes(T, S, H, Hk, D, rotary) || pos0 < 0 || ldx % 8 || ldx < (H + Hk) * (long long)D || !lds) return GFH_BAD_ARG;
  for (const void* a : {x, dq, dk, dv, (const void*)dx})
    if (!a || (reinterpret_cast<uintptr_t>(a) & 15)) return GFH_BAD_ARG;
  if (!nr_weights(qw, kw) || (qw && (!scratch || !dqw || !dkw))) return GFH_BAD_ARG;
  if (rotary && (!cos || !sin || ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15))) return GFH_BAD_ARG;
  for (int i = 0; i < 3; ++i)
    if (lds[i] % 8 || lds[i] < (i ? Hk : H) * (long long)D) return GFH_BAD_ARG;
  gf::enter();
  NormRope p{};
  p.x = (const __nv_bfloat16*)x; p.ldx = ldx; p.qw = (const __nv_bfloat16*)qw; p.kw = (const __nv_bfloat16*)kw; p.cos = cos; p.sin = sin;
  p.dq = (const __nv_bfloat16*)dq; p.dk = (const __nv_bfloat16*)dk; p.dv = (const __nv_bfloat16*)dv;
  p.ldq = lds[0]; p.ldk = lds[1]; p.ldv = lds[2];
  p.dx = (__nv_bfloat16*)dx; p.part = scratch;
  p.H = H; p.Hk = Hk; p.S = S; p.pos0 = pos0; p.rotary = rotary; p.interleaved = interleaved; p.eps = eps;
  nr_cut(p, T, H + 2 * Hk, D / 16);
  const long long ctas = (p.units + NR_WARPS - 1) / NR_WARPS, places = (long long)sm_count() * NR_BWD_CTAS;
  const int grid = (int)(ctas < places ? ctas : places);
  auto kern = D == 32 ? norm_rope_bwd_kernel<2> : D == 64 ? norm_rope_bwd_kernel<4> : D == 128 ? norm_rope_bwd_kernel<8> : norm_rope_bwd_kernel<16>;
  cudaStream_t st = (cudaStream_t)stream;
  kern<<<grid, NR_THREADS, 0, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return GFH_CUDA;
  if (!qw) return GFH_OK;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * D / 32));
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, norm_rope_fold_kernel, (const float*)scratch, grid, D, (__nv_bfloat16*)dqw, (__nv_bfloat16*)dkw) != cudaSuccess) return GFH_CUDA;
  note_extra_launches(1);
  return GFH_OK;
}
