// A row of a head in a group of D / 16 lanes: RMS norm and rotation of its first `rotary` dims.
//
// A lane has 16 numbers, two vectors of 8, chosen so that both numbers of every pair are its own and neighbouring lanes' vectors are neighbours: with halves apart lane
// i of the first n = rotary / 16 has dims 8 i .. and rotary / 2 + 8 i .., the m behind them, which are not rotated, vectors i - n and i - n + m of the rest;
// with pairs side by side all have vectors i and i + D / 16. (Two vectors next to each other, 16 i .., fill half of every 32 bytes with an access: 28 us for 21.)
#pragma once
#include "gf_ptx.cuh"

namespace gf {

struct HeadLane {
  int x, y;                      // first dims of the two vectors
  int t0, t1;                    // entries in a row of the tables: four from here, and four from there
  bool turns0, turns1;           // the vectors that those turn; with halves apart both together
  __device__ __forceinline__ HeadLane(int i, int lanes, int rotary, int interleaved) {
    const int n = rotary / 16, m = lanes - n;
    if (interleaved) {
      x = 8 * i;
      y = 8 * (i + lanes);
      turns0 = x < rotary;
      turns1 = y < rotary;
      t0 = x / 2;
      t1 = y / 2;
    } else {
      turns0 = turns1 = i < n;
      x = i < n ? 8 * i : rotary + 8 * (i - n);
      y = i < n ? rotary / 2 + 8 * i : rotary + 8 * (i - n + m);
      t0 = 8 * i;
      t1 = 8 * i + 4;
    }
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
  __device__ __forceinline__ void of(const float* cos, const float* sin, const HeadLane& at, bool there) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool turns = there && (i ? at.turns1 : at.turns0);
      const int t = i ? at.t1 : at.t0;
      const uint4 none = make_uint4(0, 0, 0, 0);
      const uint4 u = turns ? __ldg(reinterpret_cast<const uint4*>(cos + t)) : none, v = turns ? __ldg(reinterpret_cast<const uint4*>(sin + t)) : none;
      c[2 * i] = pk2(u.x, u.y); c[2 * i + 1] = pk2(u.z, u.w);
      s[2 * i] = pk2(v.x, v.y); s[2 * i + 1] = pk2(v.z, v.w);
    }
  }
  // a' = a c - b s, b' = b c + a s of every pair; SIGN -1: back
  template <int SIGN>
  __device__ __forceinline__ void turn(Head16& h, const HeadLane& at, int interleaved) const {
    if (interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {                // the i-th pair goes by the i-th entry
        if (!(i < 4 ? at.turns0 : at.turns1)) continue;
        const float ci = i & 1 ? hi2(c[i >> 1]) : lo2(c[i >> 1]), si = i & 1 ? hi2(s[i >> 1]) : lo2(s[i >> 1]);
        const float a = lo2(h.x[i]), b = hi2(h.x[i]);          // (as pairs of their own they would have to be moved first)
        h.x[i] = pk2f(a * ci - SIGN * b * si, b * ci + SIGN * a * si);
      }
    } else if (at.turns0) {
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
