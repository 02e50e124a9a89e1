// Rotary positions: the rotation itself, for the standalone kernel and the
// paged cache's writer (one arithmetic, so both round alike).
//
//   y1 = gain (x1 cos a - x2 sin a),  y2 = gain (x1 sin a + x2 cos a),
//   a = 2 pi frac(p f),  f in revolutions per position
//
// f is held as 64-bit fixed point (f 2^64), so p f mod 1 is one wrapping
// integer product, exact for any int32 position: at position 10^6 a 32-bit
// float angle is off by up to 0.03 radians, this by 10^-13. Cosine and sine are
// the Taylor polynomials of the nearest quarter turn's rest (at most pi / 4) in
// fp64, within 2^-40, rounded once to fp32 (v_cos_f32 and v_sin_f32, within
// 2^-20, put one result in 2000 on the wrong side of its rounding to bf16; this
// one in 10^5, and a token's angles serve all its heads). The products and
// their sum are fp32, each rounded, as the formula reads; fp64 products cost
// the rotation of 8192 tokens 49 us instead of 46.
#pragma once

#include "common.hpp"

namespace mtp {

struct RotSpec {
  const unsigned long long* table;   // [dims / 2] revolutions per position, 64-bit fixed point
  int dims, trad;
  float gain;
};

__device__ __forceinline__ float2 rot_angle(long long pos, unsigned long long f, float gain) {
  const unsigned long long ph = (unsigned long long)pos * f;
  const unsigned long long q = (ph + (1ull << 61)) >> 62;   // quarter turns, to the nearest (mod 4)
  const double x = (double)(long long)(ph - (q << 62)) * (6.283185307179586476925 / 18446744073709551616.0);
  const double z = x * x;
  double s = 1.0 / 6227020800.0, c = 1.0 / 479001600.0;
  s = fma(s, z, -1.0 / 39916800.0);
  c = fma(c, z, -1.0 / 3628800.0);
  s = fma(s, z, 1.0 / 362880.0);
  c = fma(c, z, 1.0 / 40320.0);
  s = fma(s, z, -1.0 / 5040.0);
  c = fma(c, z, -1.0 / 720.0);
  s = fma(s, z, 1.0 / 120.0);
  c = fma(c, z, 1.0 / 24.0);
  s = fma(s, z, -1.0 / 6.0);
  c = fma(c, z, -0.5);
  s = gain * fma(s * z, x, x);
  c = gain * fma(c, z, 1.0);
  const int n = (int)q;
  const float fs = (float)s, fc = (float)c;
  const float co = n & 1 ? fs : fc, si = n & 1 ? fc : fs;
  return make_float2((n + 1) & 2 ? -co : co, n & 2 ? -si : si);
}

__device__ __forceinline__ float rot_first(float x1, float x2, float2 cs) {
#pragma clang fp contract(off)
  return x1 * cs.x - x2 * cs.y;
}
__device__ __forceinline__ float rot_second(float x1, float x2, float2 cs) {
#pragma clang fp contract(off)
  return x1 * cs.y + x2 * cs.x;
}

// A head's row falls into items of 8 elements, or, where the halves of the
// rotated part are whole 8-element chunks, of a chunk and its partner chunk.
__host__ __device__ __forceinline__ bool rot_paired(int dims, int trad) { return !trad && dims > 0 && dims % 16 == 0; }
__host__ __device__ __forceinline__ int rot_items(int D, int dims, int trad) {
  return rot_paired(dims, trad) ? dims / 16 + (D - dims) / 8 : D / 8;
}

struct Chunk8 {
  float v[8];
};
__device__ __forceinline__ Chunk8 unpack8(uint4 r) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  Chunk8 c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c.v[2 * i] = __uint_as_float(w[i] << 16);
    c.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  return c;
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(f2bf2(v[0], v[1]), f2bf2(v[2], v[3]), f2bf2(v[4], v[5]), f2bf2(v[6], v[7]));
}

// Item `it` of one head's row (16-byte aligned), cs(i) its token's cos/sin of
// pair i; store(d, chunk) takes 8 finished elements from d on. An item
// reads all it needs before it stores, and only what it stores, unless the
// halves are no whole chunks (then partners are read from other items' rows).
template <class Angles, class Store>
__device__ __forceinline__ void rot_item(int it, const uint16_t* row, int dims, int trad, Angles cs, Store store) {
  if (rot_paired(dims, trad)) {
    const int np = dims / 16;
    if (it < np) {
      const int d = 8 * it, half = dims / 2;
      const Chunk8 a = unpack8(*reinterpret_cast<const uint4*>(row + d));
      const Chunk8 b = unpack8(*reinterpret_cast<const uint4*>(row + d + half));
      float y1[8], y2[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 w = cs(d + e);
        y1[e] = rot_first(a.v[e], b.v[e], w);
        y2[e] = rot_second(a.v[e], b.v[e], w);
      }
      store(d, pack8(y1));
      store(d + half, pack8(y2));
    } else {
      const int d = dims + 8 * (it - np);
      store(d, *reinterpret_cast<const uint4*>(row + d));
    }
    return;
  }
  const int d = 8 * it;
  const uint4 raw = *reinterpret_cast<const uint4*>(row + d);
  if (d >= dims) {
    store(d, raw);
    return;
  }
  const Chunk8 a = unpack8(raw);
  float y[8];
  if (trad) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {   // dims is even: a pair rotates or passes as a whole
      const bool in = d + e < dims;
      const float2 w = in ? cs((d + e) >> 1) : make_float2(1.f, 0.f);
      y[e] = in ? rot_first(a.v[e], a.v[e + 1], w) : a.v[e];
      y[e + 1] = in ? rot_second(a.v[e], a.v[e + 1], w) : a.v[e + 1];
    }
  } else {
    const int half = dims / 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int dd = d + e;
      if (dd >= dims)
        y[e] = a.v[e];
      else if (dd < half)
        y[e] = rot_first(a.v[e], bf2f(row[dd + half]), cs(dd));
      else
        y[e] = rot_second(bf2f(row[dd - half]), a.v[e], cs(dd - half));
    }
  }
  store(d, pack8(y));
}

}  // namespace mtp
