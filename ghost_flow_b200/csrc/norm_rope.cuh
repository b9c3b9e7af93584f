// A row of a head in a group of D / 16 lanes: RMS norm and rotation of its first `rotary` dims.
//
// A lane has 16 numbers, two vectors of 8, chosen so that both numbers of every pair are its own: with halves apart lane i of the first rotary / 16 has dims
// 8 i .. and rotary / 2 + 8 i .., with pairs side by side 16 i ..; lanes behind those have the dims that are not rotated.
#pragma once
#include "gf_ptx.cuh"

namespace gf {

struct HeadLane {
  int x, y;                      // first dims of the two vectors
  int t;                         // first entry in a row of the tables
  bool turns;
  __device__ __forceinline__ HeadLane(int i, int rotary, int interleaved) {
    turns = 16 * i < rotary;
    t = 8 * i;
    const bool apart = turns && !interleaved;
    x = apart ? 8 * i : 16 * i;
    y = apart ? rotary / 2 + 8 * i : 16 * i + 8;
  }
};

// Two neighbouring numbers to a register pair, whose products and sums are one instruction.
struct Head16 {
  uint64_t x[8];                 // the first vector in 0 .. 3, the second in 4 .. 7
  __device__ __forceinline__ void of(const uint4& first, const uint4& second) {
    const uint32_t *u = reinterpret_cast<const uint32_t*>(&first), *v = reinterpret_cast<const uint32_t*>(&second);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = pk2(u[i] << 16, u[i] & 0xffff0000u);
      x[4 + i] = pk2(v[i] << 16, v[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void to(uint4& first, uint4& second) const {
    uint32_t *u = reinterpret_cast<uint32_t*>(&first), *v = reinterpret_cast<uint32_t*>(&second);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = pack_bf16x2(lo2(x[i]), hi2(x[i]));
      v[i] = pack_bf16x2(lo2(x[4 + i]), hi2(x[4 + i]));
    }
  }
  __device__ __forceinline__ float dot(const Head16& o) const {
    uint64_t s = f2_mul(x[0], o.x[0]), t = f2_mul(x[1], o.x[1]);
#pragma unroll
    for (int i = 2; i < 8; i += 2) {
      s = f2_fma(x[i], o.x[i], s);
      t = f2_fma(x[i + 1], o.x[i + 1], t);
    }
    s = f2_add(s, t);
    return lo2(s) + hi2(s);
  }
  __device__ __forceinline__ void scale(const Head16& o) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = f2_mul(x[i], o.x[i]);
  }
  __device__ __forceinline__ void scale(float f) {
    const uint64_t two = pk2f(f, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = f2_mul(x[i], two);
  }
};

// A lane's 8 entries of a row of the tables, and the turn by them.
struct HeadTurn {
  uint64_t c[4], s[4];
  __device__ __forceinline__ void of(const float* cos, const float* sin, bool there) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const uint4 none = make_uint4(0, 0, 0, 0);
      const uint4 u = there ? __ldg(reinterpret_cast<const uint4*>(cos) + i / 2) : none, v = there ? __ldg(reinterpret_cast<const uint4*>(sin) + i / 2) : none;
      c[i] = pk2(u.x, u.y); c[i + 1] = pk2(u.z, u.w);
      s[i] = pk2(v.x, v.y); s[i + 1] = pk2(v.z, v.w);
    }
  }
  // a' = a c - b s, b' = b c + a s of every pair; SIGN -1: back
  template <int SIGN>
  __device__ __forceinline__ void turn(Head16& h, int interleaved) const {
    if (interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {                // the i-th pair goes by the i-th entry
        const float ci = i & 1 ? hi2(c[i >> 1]) : lo2(c[i >> 1]), si = i & 1 ? hi2(s[i >> 1]) : lo2(s[i >> 1]);
        h.x[i] = f2_fma(pk2f(hi2(h.x[i]), lo2(h.x[i])), pk2f(-SIGN * si, SIGN * si), f2_mul(h.x[i], pk2f(ci, ci)));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t minus = s[i] ^ 0x8000000080000000ull, a = h.x[i], b = h.x[4 + i];
        h.x[i] = f2_fma(b, SIGN > 0 ? minus : s[i], f2_mul(a, c[i]));
        h.x[4 + i] = f2_fma(a, SIGN > 0 ? s[i] : minus, f2_mul(b, c[i]));
      }
    }
  }
};

// Sum over a group of LANES (a power of two) neighbouring lanes.
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace gf
