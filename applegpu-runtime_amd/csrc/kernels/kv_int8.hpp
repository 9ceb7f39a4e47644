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

__device__ __forceinline__ uint32_t top_of(const float (&v)[8], uint32_t top) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t m = __float_as_uint(v[e]) & 0x7fffffffu;
    top = m > top ? m : top;
  }
  return top;
}

// clamp(rint(x / s), -127, 127) of 8 values; 0 where the scale says nothing
// (0, infinite or NaN).  x / s is IEEE's; x times 1 / s is within 127 (2^-23 +
// 2^-24) < 2.3e-5 of it, so only where that is nearer than 1e-4 to a half is
// the division done (as 8 divisions a chunk the append of 8 x 20 x 509 rows
// of 64 takes 13.7 us, bound by them).
__device__ __forceinline__ void codes_of(const float (&v)[8], float s, float inv, bool ok, int (&c)[8]) {
  float r[8];
  bool near = !(inv < 1e30f);  // 1 / s overflows, or nearly
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = v[e] * inv;
    r[e] = rintf(q);
    near |= fabsf(fabsf(q - r[e]) - 0.5f) < 1e-4f;
  }
  if (near) {
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = rintf(v[e] / s);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = ok ? (int)fminf(fmaxf(r[e], -127.f), 127.f) : 0;
}

__device__ __forceinline__ void store_codes(int8_t* p, const int (&c)[8]) {
  uint2 w{0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w.x |= (uint32_t)(c[i] & 255) << (8 * i);
    w.y |= (uint32_t)(c[4 + i] & 255) << (8 * i);
  }
  *(uint2*)p = w;
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
    for (int u = 0; u < NC; ++u) {
      float v[8];
      keep[u].floats(v);
      top = top_of(v, top);
    }
  } else {
    for (int i = lane; i < chunks; i += 64) {
      Raw8x<T> raw;
      raw.load(x + (i >> lg_cpr) * x_st + (i & (cpr - 1)) * 8);
      float v[8];
      raw.floats(v);
      top = top_of(v, top);
    }
  }
  uint32_t s_bits = __float_as_uint(__uint_as_float(wave_umax(top)) / 127.f) & 0x7fffffffu;
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
      int cc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) cc[e] = (int)rintf((float)o[e] * rate);
      store_codes(q, cc);
    }
  }
  auto put = [&](int i, const Raw8x<T>& raw) {
    float v[8];
    raw.floats(v);
    int cc[8];
    codes_of(v, s, inv, ok, cc);
    store_codes(to + (i >> lg_cpr) * c_st + (i & (cpr - 1)) * 8, cc);
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
