// RMS norms of the query and key heads of a packed projection with the rotation in the same pass, and their gradients.
//
// The reference normalises whole rows only (ghostflow-nn/src/llama.rs:154-185) and rotates in a pass of its own (llama.rs:208-252).
//
// y = rot(x r w), r = (mean x^2 + eps)^(-1/2), for each head of q and k. With g = rot^-1(dy) and d = g w: dx = r (d - x r mean(d x r)),
// dw = sum of g x r over all tokens and heads; the gradient of v is copied beside them. In 32 bits from bf16, rounded once; r is worked out again by the
// backward pass, which reads x anyway. Every row is read once and written once.
//
// A warp has a token and some of its heads, D / 16 lanes to a head (norm_rope.cuh), so it reads its rows of the tables once for all of them. What is on its way
// lies in shared memory, where a thread has a ring of its own for what it reads itself: NR_STAGES rows ahead, through the ends of tokens. The warps
// stay for all tokens. dw: a warp keeps its sums in registers, a CTA leaves them in a row of a scratch buffer, and a second kernel, on the machine before the first one ends, adds
// the rows up in a fixed order.
//
// 8192 tokens of 32 / 8 heads of 128: forward 33 us, 5.1 TB/s, backward 62 with the fold, 4.6 TB/s; 2987 of 32 / 32 heads, half of each rotated, 18.7, 5.2 TB/s. Issue slots
// are 60 to 63 % taken, DRAM 42 and 47 %: what is left is the latency of a row's chain (load, sum over lanes, product, store). Loads into registers, without rings,
// took 36 and 79, and with a head's halves in the same lane the rows of the third size 25; other numbers of stages and of CTAs to an SM were within the noise, weights
// kept in registers slower (a branch for each row).
#include "gf_host.h"
#include "norm_rope.cuh"

namespace gf {

constexpr int NR_THREADS = 256, NR_WARPS = NR_THREADS / 32;
constexpr int NR_STAGES = 4;
constexpr int NR_CTAS = 3, NR_BWD_CTAS = 2;        // on an SM

struct NormRope {
  const __nv_bfloat16* x;        // [T, H + 2 Hk, D], rows ldx apart
  unsigned ldx;
  const __nv_bfloat16 *qw, *kw;  // [D]; null: heads are rotated only
  const float *cos, *sin;        // [positions, rotary / 2]
  __nv_bfloat16 *q, *k;          // forward: [T, H, D], [T, Hk, D] dense
  const __nv_bfloat16 *dq, *dk, *dv;               // backward: rows ldq, ldk, ldv apart
  unsigned ldq, ldk, ldv;
  __nv_bfloat16* dx;             // [T, H + 2 Hk, D] dense
  float* part;                   // [CTAs][2][D]
  unsigned units;
  int H, Hk, S, pos0, rotary, interleaved, per, chunks;        // heads of a unit, units of a token
  unsigned step, step_t, step_chunk, step_pos;                 // from a warp's unit to its next one: units, whole tokens, units beyond those, positions
  float eps;
};

// A warp's place: heads h .. of a token, a group to each, up to h1.
struct NrAt {
  unsigned u, t, chunk, pos;
  int h, h1;
  __device__ __forceinline__ void heads(const NormRope& p, int all) {
    h = chunk * p.per;
    h1 = min(h + p.per, all);
  }
  __device__ __forceinline__ void begin(const NormRope& p, unsigned unit, int all) {
    u = unit;
    t = u / p.chunks;
    chunk = u - t * p.chunks;
    pos = t % p.S;
    heads(p, all);
  }
  // true where a unit begins
  __device__ __forceinline__ bool next(const NormRope& p, int groups, int all) {
    if ((h += groups) < h1) return false;
    u += p.step;
    chunk += p.step_chunk;
    const unsigned more = chunk >= (unsigned)p.chunks;
    chunk -= more ? p.chunks : 0;
    t += p.step_t + more;
    pos += p.step_pos + more;
    pos -= pos >= (unsigned)p.S ? p.S : 0;
    heads(p, all);
    return true;
  }
};

__device__ __forceinline__ void nr_copy(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

template <int LANES, bool BACK>
__global__ void __launch_bounds__(NR_THREADS, BACK ? NR_BWD_CTAS : NR_CTAS) norm_rope_kernel(const __grid_constant__ NormRope p) {
  constexpr int D = 16 * LANES, GROUPS = 32 / LANES, VECTORS = BACK ? 4 : 2;
  extern __shared__ uint4 ring[];                  // [stages][vectors][threads]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = lane / LANES, heads = p.H + (BACK ? 2 : 1) * p.Hk;
  if (BACK && threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const HeadLane at(lane % LANES, LANES, p.rotary, p.interleaved);
  const uint32_t mine = smem_u32(ring + threadIdx.x);
  NrAt now, ahead;
  now.begin(p, blockIdx.x * NR_WARPS + warp, heads);
  ahead = now;
  auto ask = [&](int st) {                         // one group of copies each, empty ones behind the last unit
    if (ahead.u < p.units) {
      const int h = ahead.h + group;
      if (h < ahead.h1) {
        const uint32_t to = mine + st * (VECTORS * NR_THREADS * 16);
        const __nv_bfloat16* x = p.x + (unsigned long long)ahead.t * p.ldx + h * D;
        if (!BACK || (p.qw && h < p.H + p.Hk)) {
          nr_copy(to, x + at.x);
          nr_copy(to + NR_THREADS * 16, x + at.y);
        }
        if constexpr (BACK) {
          const __nv_bfloat16* g = h < p.H ? p.dq + (unsigned long long)ahead.t * p.ldq + h * D : h < p.H + p.Hk ? p.dk + (unsigned long long)ahead.t * p.ldk + (h - p.H) * D
                                                                                            : p.dv + (unsigned long long)ahead.t * p.ldv + (h - p.H - p.Hk) * D;
          nr_copy(to + 2 * NR_THREADS * 16, g + at.x);
          nr_copy(to + 3 * NR_THREADS * 16, g + at.y);
        }
      }
      ahead.next(p, GROUPS, heads);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < NR_STAGES - 1; ++i) ask(i);
  Head16 dw[BACK ? 2 : 1];
#pragma unroll
  for (int i = 0; i < (BACK ? 2 : 1); ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i].x[e] = 0;
  HeadTurn turn;
  bool begins = true;
  for (int st = 0; now.u < p.units; st = st + 1 == NR_STAGES ? 0 : st + 1) {
    if (begins) {
      const long long off = (long long)(now.pos + p.pos0) * (p.rotary / 2);
      turn.of(p.cos + off, p.sin + off, at, true);
    }
    ask(st == 0 ? NR_STAGES - 1 : st - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(NR_STAGES - 1) : "memory");
    const uint4* in = ring + threadIdx.x + st * (VECTORS * NR_THREADS);
    const int h = now.h + group;
    const bool query = h < p.H, there = h < now.h1, normed = p.qw && there && h < p.H + p.Hk;
    Head16 w, v;
    const uint4 none = make_uint4(0, 0, 0, 0);
    if (normed) {
      const __nv_bfloat16* weight = query ? p.qw : p.kw;
      w.of(__ldg(reinterpret_cast<const uint4*>(weight + at.x)), __ldg(reinterpret_cast<const uint4*>(weight + at.y)));
    }
    uint4 x, y;
    if constexpr (!BACK) {
      v.of(there ? in[0] : none, there ? in[NR_THREADS] : none);
      if (p.qw) {
        v.scale(rsqrtf(group_sum<LANES>(v.dot(v)) * (1.f / D) + p.eps));
        v.scale(w);
      }
      turn.turn<1>(v, at, p.interleaved);
      v.to(x, y);
      if (there) {
        __nv_bfloat16* to = query ? p.q + ((unsigned long long)now.t * p.H + h) * D : p.k + ((unsigned long long)now.t * p.Hk + h - p.H) * D;
        *reinterpret_cast<uint4*>(to + at.x) = x;
        *reinterpret_cast<uint4*>(to + at.y) = y;
      }
    } else {
      x = there ? in[2 * NR_THREADS] : none;
      y = there ? in[3 * NR_THREADS] : none;
      Head16 g;
      g.of(x, y);
      turn.turn<-1>(g, at, p.interleaved);
      if (p.qw) {
        v.of(normed ? in[0] : none, normed ? in[NR_THREADS] : none);
        const float r = rsqrtf(group_sum<LANES>(v.dot(v)) * (1.f / D) + p.eps);
        v.scale(r);
        if (normed) {                              // sums of g x r of the query heads, and of the key heads
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (query == (i == 0)) {
#pragma unroll
              for (int e = 0; e < 8; ++e) dw[i].x[e] = f2_fma(g.x[e], v.x[e], dw[i].x[e]);
            }
          g.scale(w);
        }
        const float mean = group_sum<LANES>(normed ? g.dot(v) : 0.f) * (-1.f / D);
        const uint64_t two = pk2f(mean, mean);
#pragma unroll
        for (int e = 0; e < 8; ++e) g.x[e] = f2_fma(v.x[e], two, g.x[e]);
        g.scale(r);
      }
      if (h < p.H + p.Hk) g.to(x, y);
      if (there) {
        __nv_bfloat16* to = p.dx + ((unsigned long long)now.t * heads + h) * D;
        *reinterpret_cast<uint4*>(to + at.x) = x;
        *reinterpret_cast<uint4*>(to + at.y) = y;
      }
    }
    begins = now.next(p, GROUPS, heads);
  }
  if constexpr (BACK) {
    if (!p.qw) return;
    // ---- the weights' gradients: groups, then warps
    float* sums = reinterpret_cast<float*>(ring);  // [warps][2][D]
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float v = e & 1 ? hi2(dw[i].x[e >> 1]) : lo2(dw[i].x[e >> 1]);
#pragma unroll
        for (int o = 16; o >= LANES; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (group == 0) sums[(warp * 2 + i) * D + (e < 8 ? at.x : at.y) + (e & 7)] = v;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += NR_THREADS) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < NR_WARPS; ++w) v += sums[w * 2 * D + i];
      p.part[(long long)blockIdx.x * 2 * D + i] = v;
    }
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

// Units of a token: parts of its heads. A dozen for every warp, as those with one more than others are waited for, but of four rounds each at least (a unit's rows of the
// tables are not on their way before it begins) unless there are fewer units than warps.
static void nr_cut(NormRope& p, long long T, int heads, int lanes, int ctas) {
  const int groups = 32 / lanes;
  const long long rounds = (heads + groups - 1) / groups, warps = (long long)sm_count() * ctas * NR_WARPS;
  const long long room = 0x7fffffffll / T, many = (12 * warps + T - 1) / T, few = (warps + T - 1) / T, four = (rounds + 3) / 4;
  const long long wanted = many < four ? many : few > four ? few : four, want = wanted < room ? wanted : room;
  p.chunks = (int)(want < 1 ? 1 : want < rounds ? want : rounds);
  p.per = (int)((rounds + p.chunks - 1) / p.chunks) * groups;
  p.chunks = (heads + p.per - 1) / p.per;
  p.units = (unsigned)(T * p.chunks);
}

// Behind nr_cut: what a warp of `grid` CTAs adds up from unit to unit.
static void nr_step(NormRope& p, unsigned grid) {
  p.step = grid * NR_WARPS;
  p.step_t = p.step / p.chunks;
  p.step_chunk = p.step % p.chunks;
  p.step_pos = p.step_t % p.S;
}

template <bool BACK>
static int nr_launch(NormRope& p, int D, int grid, cudaStream_t st) {
  nr_step(p, grid);
  constexpr int SMEM = NR_STAGES * (BACK ? 4 : 2) * NR_THREADS * 16;
  auto kern = D == 32 ? norm_rope_kernel<2, BACK> : D == 64 ? norm_rope_kernel<4, BACK> : D == 128 ? norm_rope_kernel<8, BACK> : norm_rope_kernel<16, BACK>;
  static gf::SharedLimit limit[4];
  if (SMEM > 48 * 1024 && !limit[D == 32 ? 0 : D == 64 ? 1 : D == 128 ? 2 : 3].raise(kern, SMEM)) return GFH_CUDA;
  kern<<<grid, NR_THREADS, SMEM, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
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
  if (!nr_sizes(T, S, H, Hk, D, rotary) || pos0 < 0 || ldx % 8 || ldx < (H + Hk) * (long long)D || ldx > 0x7fffffff) return GFH_BAD_ARG;
  for (const void* a : {x, (const void*)q, (const void*)k})
    if (!a || (reinterpret_cast<uintptr_t>(a) & 15)) return GFH_BAD_ARG;
  if (!nr_weights(qw, kw)) return GFH_BAD_ARG;
  if (rotary && (!cos || !sin || ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15))) return GFH_BAD_ARG;
  gf::enter();
  NormRope p{};
  p.x = (const __nv_bfloat16*)x; p.ldx = (unsigned)ldx; p.qw = (const __nv_bfloat16*)qw; p.kw = (const __nv_bfloat16*)kw; p.cos = cos; p.sin = sin;
  p.q = (__nv_bfloat16*)q; p.k = (__nv_bfloat16*)k;
  p.H = H; p.Hk = Hk; p.S = S; p.pos0 = pos0; p.rotary = rotary; p.interleaved = interleaved; p.eps = eps;
  nr_cut(p, T, H + Hk, D / 16, NR_CTAS);
  const long long ctas = (p.units + NR_WARPS - 1) / NR_WARPS, places = (long long)sm_count() * NR_CTAS;
  return nr_launch<false>(p, D, (int)(ctas < places ? ctas : places), (cudaStream_t)stream);
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
  if (!nr_sizes(T, S, H, Hk, D, rotary) || pos0 < 0 || ldx % 8 || ldx < (H + Hk) * (long long)D || ldx > 0x7fffffff || !lds) return GFH_BAD_ARG;
  for (const void* a : {x, dq, dk, dv, (const void*)dx})
    if (!a || (reinterpret_cast<uintptr_t>(a) & 15)) return GFH_BAD_ARG;
  if (!nr_weights(qw, kw) || (qw && (!scratch || !dqw || !dkw))) return GFH_BAD_ARG;
  if (rotary && (!cos || !sin || ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15))) return GFH_BAD_ARG;
  for (int i = 0; i < 3; ++i)
    if (lds[i] % 8 || lds[i] < (i ? Hk : H) * (long long)D || lds[i] > 0x7fffffff) return GFH_BAD_ARG;
  gf::enter();
  NormRope p{};
  p.x = (const __nv_bfloat16*)x; p.ldx = (unsigned)ldx; p.qw = (const __nv_bfloat16*)qw; p.kw = (const __nv_bfloat16*)kw; p.cos = cos; p.sin = sin;
  p.dq = (const __nv_bfloat16*)dq; p.dk = (const __nv_bfloat16*)dk; p.dv = (const __nv_bfloat16*)dv;
  p.ldq = (unsigned)lds[0]; p.ldk = (unsigned)lds[1]; p.ldv = (unsigned)lds[2];
  p.dx = (__nv_bfloat16*)dx; p.part = scratch;
  p.H = H; p.Hk = Hk; p.S = S; p.pos0 = pos0; p.rotary = rotary; p.interleaved = interleaved; p.eps = eps;
  nr_cut(p, T, H + 2 * Hk, D / 16, NR_BWD_CTAS);
  const long long ctas = (p.units + NR_WARPS - 1) / NR_WARPS, places = (long long)sm_count() * NR_BWD_CTAS;
  const int grid = (int)(ctas < places ? ctas : places);
  cudaStream_t st = (cudaStream_t)stream;
  const int rc = nr_launch<true>(p, D, grid, st);
  if (rc) return rc;
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
