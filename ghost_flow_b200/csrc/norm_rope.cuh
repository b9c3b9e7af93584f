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

struct Head16 {
  float a[8], b[8];
  __device__ __forceinline__ void of(const uint4& x, const uint4& y) {
    const uint32_t *u = reinterpret_cast<const uint32_t*>(&x), *v = reinterpret_cast<const uint32_t*>(&y);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_bf16x2(u[i]), g = unpack_bf16x2(v[i]);
      a[2 * i] = f.x; a[2 * i + 1] = f.y;
      b[2 * i] = g.x; b[2 * i + 1] = g.y;
    }
  }
  __device__ __forceinline__ void to(uint4& x, uint4& y) const {
    uint32_t *u = reinterpret_cast<uint32_t*>(&x), *v = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = pack_bf16x2(a[2 * i], a[2 * i + 1]);
      v[i] = pack_bf16x2(b[2 * i], b[2 * i + 1]);
    }
  }
  __device__ __forceinline__ float dot(const Head16& o) const {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += a[i] * o.a[i] + b[i] * o.b[i];
    return s;
  }
  // a' = a c - b s, b' = b c + a s of every pair; SIGN -1: back
  template <int SIGN>
  __device__ __forceinline__ void turn(const float (&c)[8], const float (&s)[8], int interleaved) {
    if (interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = a[2 * i], q = a[2 * i + 1], u = b[2 * i], v = b[2 * i + 1];
        a[2 * i] = p * c[i] - SIGN * q * s[i];
        a[2 * i + 1] = q * c[i] + SIGN * p * s[i];
        b[2 * i] = u * c[i + 4] - SIGN * v * s[i + 4];
        b[2 * i + 1] = v * c[i + 4] + SIGN * u * s[i + 4];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = a[i], q = b[i];
        a[i] = p * c[i] - SIGN * q * s[i];
        b[i] = q * c[i] + SIGN * p * s[i];
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

// 8 entries of a row of the tables.
__device__ __forceinline__ void table8(const float* row, bool there, float (&c)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    const float4 u = there ? __ldg(reinterpret_cast<const float4*>(row + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
    c[e] = u.x; c[e + 1] = u.y; c[e + 2] = u.z; c[e + 3] = u.w;
  }
}

}  // namespace gf
