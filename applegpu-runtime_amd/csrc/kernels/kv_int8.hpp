// The append of rows to one block of a K/V cache held in 8 bits (kv_int8.hip
// has the definition), by one wave: the append's own kernel and the decode
// attention that appends its step's row share it.
#pragma once

#include "device.hpp"

namespace agpu {
namespace k {
namespace kv8 {
using namespace dev;

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, m, 64);
    v = o > v ? o : v;
  }
  return v;
}

// 8 consecutive values, raw.
template <typename T>
struct Raw8x {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = ((const uint4*)p)[i];
  }
  __device__ __forceinline__ void floats(float (&x)[8]) const {
    T e[8];
    __builtin_memcpy(e, v, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f(e[i]);
  }
};

// The largest magnitude so far as bits, of T or of a pair of 16-bit T.
template <typename T>
__device__ __forceinline__ uint32_t top_of(const Raw8x<T>& raw, uint32_t top) {
  typedef unsigned short u2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    const uint32_t w[4] = {raw.v[i].x, raw.v[i].y, raw.v[i].z, raw.v[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) {
        const uint32_t m = w[e] & 0x7fffffffu;
        top = m > top ? m : top;
      } else {
        top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u2, w[e] & 0x7fff7fffu),
                                                                     __builtin_bit_cast(u2, top)));
      }
    }
  }
  return top;
}

// The wave's largest magnitude.
template <typename T>
__device__ __forceinline__ float wave_top(uint32_t top) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(wave_umax(top));
  } else {
    const uint32_t hi = top >> 16, lo = top & 0xffffu;
    const uint16_t m = (uint16_t)wave_umax(hi > lo ? hi : lo);
    T t;
    __builtin_memcpy(&t, &m, 2);
    return to_f(t);
  }
}

// rint(x / s) of 8 values within 127 s as 8 bytes; 0 where the scale says
// nothing (0, infinite or NaN).  x / s is IEEE's; x times 1 / s is within 127
// (2^-23 + 2^-24) < 2.3e-5 of it, so only where that is nearer than 1e-4 to a
// half is the division done.  1.5 2^23 added rounds to a whole number, half to
// even, whose low byte is the code.  A scale that is subnormal or nearly so
// (1 / s past 1e30) may have been rounded below the largest / 127: its codes
// are clamped.  An append of 8 x 20 x 509 rows of 64 takes 11.3 us so, 13.7 with 8
// divisions, 12.7 with a clamp and a conversion of every value.
__device__ __forceinline__ uint2 codes_of(const float (&v)[8], float s, float inv, bool ok) {
  constexpr float kWhole = 12582912.f;
  float t[8];
  const bool tiny = !(inv < 1e30f);
  bool near = tiny;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = v[e] * inv;
    t[e] = q + kWhole;
    near |= fabsf(q - (t[e] - kWhole)) > 0.4999f;
  }
  if (near) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = v[e] / s;
      t[e] = (tiny ? fminf(fmaxf(q, -127.f), 127.f) : q) + kWhole;
    }
  }
  uint32_t u[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) u[e] = __float_as_uint(t[e]);
  uint2 w;
  w.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u), __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), 0x05040100u);
  w.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[7], u[6], 0x0c0c0400u), __builtin_amdgcn_perm(u[5], u[4], 0x0c0c0400u), 0x05040100u);
  return ok ? w : uint2{0, 0};
}

// Rows r0 .. r1 - 1 (at least one, x their first) of the block of rows from
// lo on; codes: the head's row 0; scale: the block's.  Returns its new scale
// (every lane).  NC > 0: the new rows are at most 64 NC chunks of 8 values and
// stay in registers between the search for the largest and the rounding; 0:
// any number, read twice.
template <typename T, int NC>
__device__ __forceinline__ float append_rows(const T* x, int64_t x_st, int8_t* codes, int64_t c_st, float* scale,
                                             int64_t lo, int64_t r0, int64_t r1, int lg_cpr, int lane) {
  int8_t* to = codes + r0 * c_st;
  const int cpr = 1 << lg_cpr;
  const int chunks = (int)(r1 - r0) << lg_cpr;

  uint32_t top = 0;
  Raw8x<T> keep[NC ? NC : 1];
  if constexpr (NC > 0) {
#pragma unroll
    for (int u = 0; u < NC; ++u) {
      const int i = lane + 64 * u;
#pragma unroll
      for (int e = 0; e < (int)sizeof(T) / 2; ++e) keep[u].v[e] = uint4{0, 0, 0, 0};
      if (i < chunks) keep[u].load(x + (i >> lg_cpr) * x_st + (i & (cpr - 1)) * 8);
    }
#pragma unroll
    for (int u = 0; u < NC; ++u) top = top_of(keep[u], top);
  } else {
    for (int i = lane; i < chunks; i += 64) {
      Raw8x<T> raw;
      raw.load(x + (i >> lg_cpr) * x_st + (i & (cpr - 1)) * 8);
      top = top_of(raw, top);
    }
  }
  uint32_t s_bits = __float_as_uint(wave_top<T>(top) / 127.f) & 0x7fffffffu;
  const uint32_t was = r0 > lo ? __float_as_uint(*scale) & 0x7fffffffu : 0u;
  if (was > s_bits) s_bits = was;
  const float s = __uint_as_float(s_bits);
  const bool ok = s > 0.f && s < INFINITY;
  const float inv = 1.f / s;

  if (s_bits != was) {  // rows before the append, if any, take the grown scale
    const int held = (int)(r0 - lo) << lg_cpr;
    const float rate = ok ? __uint_as_float(was) / s : 0.f;
    for (int i = lane; i < held; i += 64) {
      int8_t* q = codes + (lo + (i >> lg_cpr)) * c_st + (i & (cpr - 1)) * 8;
      const uint2 w = *(const uint2*)q;
      int8_t o[8];
      __builtin_memcpy(o, &w, 8);
      uint32_t n[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) n[e / 4] |= (uint32_t)((int)rintf((float)o[e] * rate) & 255) << (8 * (e % 4));
      *(uint2*)q = uint2{n[0], n[1]};
    }
  }
  auto put = [&](int i, const Raw8x<T>& raw) {
    float v[8];
    raw.floats(v);
    *(uint2*)(to + (i >> lg_cpr) * c_st + (i & (cpr - 1)) * 8) = codes_of(v, s, inv, ok);
  };
  if constexpr (NC > 0) {
#pragma unroll
    for (int u = 0; u < NC; ++u)
      if (lane + 64 * u < chunks) put(lane + 64 * u, keep[u]);
  } else {
    for (int i = lane; i < chunks; i += 64) {
      Raw8x<T> raw;
      raw.load(x + (i >> lg_cpr) * x_st + (i & (cpr - 1)) * 8);
      put(i, raw);
    }
  }
  if (lane == 0) *scale = s;
  return s;
}

}  // namespace kv8
}  // namespace k
}  // namespace agpu
