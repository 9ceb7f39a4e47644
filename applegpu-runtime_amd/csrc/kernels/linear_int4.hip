// Linear layers with weights in 4 bits and a scale per row and group of
// columns: y = act(x W^T + bias), W[n, k] = (code + 8 - 8) scale[k / group, n].
//
// The codes are stored in tiles of 16 rows x 128 columns, 1 KB each, in the
// order in which a wave reads them: 16 bytes (32 codes) a lane, contiguous.
#include "device.hpp"

namespace agpu {
namespace k {
using namespace dev;

namespace {

// place of code i (0..7) among the nibbles of its 4-byte word
__device__ __forceinline__ int nibble_of(int i) { return (i >> 1) + 4 * (i & 1); }

// One thread per 4-byte word of the packed weights: eight codes of one row,
// all of one group.
template <typename T>
__global__ void __launch_bounds__(256) quantize_int4_kernel(const T* __restrict__ w, int64_t sn, int64_t sk, int64_t N,
                                                            int64_t K, int64_t group, const T* __restrict__ scales,
                                                            uint32_t* __restrict__ packed, int64_t words, int64_t steps) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
    const int word = (int)(i & 3), run = (int)(i >> 2) & 63;
    const int64_t tile = i >> 8, step = tile % steps;
    const int64_t n = tile / steps * 16 + (run & 15), k0 = step * 128 + (run >> 4) * 32 + word * 8;
    uint32_t v = 0x88888888u;
    if (n < N && k0 < K) {
      const float s = to_f(scales[k0 / group * N + n]);
      const bool ok = s > 0.f && s < INFINITY;
      v = 0;
      for (int e = 0; e < 8; ++e) {
        float r = 0.f;
        if (ok && k0 + e < K) r = rintf(to_f(w[n * sn + (k0 + e) * sk]) / s);
        v |= (uint32_t)((int)fminf(fmaxf(r, -7.f), 7.f) + 8) << (4 * nibble_of(e));
      }
    }
    packed[i] = v;
  }
}

// One thread per (group, row): scale = largest magnitude / 7.
template <typename T>
__global__ void __launch_bounds__(256) int4_scales_kernel(const T* __restrict__ w, int64_t sn, int64_t sk, int64_t N,
                                                          int64_t K, int64_t group, T* __restrict__ scales, int64_t n_s) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n_s; i += (int64_t)gridDim.x * 256) {
    const int64_t g = i / N, n = i % N;
    const int64_t k1 = (g + 1) * group < K ? (g + 1) * group : K;
    uint32_t top = 0;  // magnitudes by their bits: infinities and NaN are the largest
    for (int64_t k = g * group; k < k1; ++k) {
      const uint32_t m = __float_as_uint(to_f(w[n * sn + k * sk])) & 0x7fffffffu;
      top = m > top ? m : top;
    }
    scales[i] = from_f<T>(__uint_as_float(top) / 7.f);
  }
}

// One lane per byte run: 32 codes of a row, of one scale.  A wave reads 1 KB in
// a row and writes 64 bytes (16-bit types) of each of 16 rows four times over.
// VEC: rows are aligned and whole runs of 8 values are one store.  Columns K ..
// ld - 1 become 0.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dequantize_int4_kernel(const uint4* __restrict__ packed,
                                                              const T* __restrict__ scales, int64_t N, int64_t K,
                                                              int64_t group, T* __restrict__ out, int64_t ld,
                                                              int64_t runs, int64_t steps) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < runs; i += (int64_t)gridDim.x * 256) {
    const int run = (int)(i & 63);
    const int64_t tile = i >> 6, n = tile / steps * 16 + (run & 15), k0 = tile % steps * 128 + (run >> 4) * 32;
    if (n >= N || k0 >= ld) continue;
    const uint4 w = packed[i];  // (padding has code 0)
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    const float s = k0 < K ? to_f(scales[k0 / group * N + n]) : 0.f;
    T* o = out + n * ld + k0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      T v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = from_f<T>((float)((int)((ws[t] >> (4 * nibble_of(e))) & 15) - 8) * s);
      if (VEC && k0 + 8 * t + 8 <= ld) {
        uint4 raw[sizeof(T) / 2];
        __builtin_memcpy(raw, v, sizeof(v));
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; ++e) ((uint4*)(o + 8 * t))[e] = raw[e];
      } else {
        for (int e = 0; e < 8; ++e)
          if (k0 + 8 * t + e < ld) o[8 * t + e] = v[e];
      }
    }
  }
}

__device__ __forceinline__ float act_of(float v, int act) {
  if (act == kActRelu) return fmaxf(v, 0.f);  // (0 for NaN, as relu gives elsewhere)
  if (act == kActGelu) return gelu_tanh(v);
  if (act == kActGeluExact) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
  return v;
}

// ── few rows: codes straight into the matrix units ─────────────────────────
// Bound by the codes, N K / 2 bytes, and for small matrices by latency: 16 x
// 8192 x 8192 (bf16, groups of 64) 14.5 us, 2.5 TB/s of codes and scales; 1 x
// 1280 x 5120 (f16) 4.5 us.
//  - A wave instruction reads 1 KB of codes in a row and each byte is read
//    once; UN steps of them are under way before the first is multiplied.
//  - No conversion: a nibble becomes the mantissa of 16 + (code + 8) by a mask
//    and an or, and the 24 too many come off through one more product, of the
//    rows with a constant -24, which all tiles of columns share.  The products
//    and their difference are exact up to the fp32 sums, and a group's scale is
//    multiplied once, on its sum.  Where the difference is not a number (an
//    infinite x, or one next to fp32's largest) the sum is taken again from the
//    values, behind a test of 0 to 0.3 us.
//  - The waves of a block split K and add their sums through LDS.
// Two tiles of columns a wave (NT = 2) share the rows' loads where they leave
// enough blocks, and fewer waves a block where there are many (us, one row):
//   K = 1280, N = 50257   NT 2, 2 waves 12.3   NT 1, 10 waves 26.5
//   K = 1280, N = 5120    NT 2, 10 waves 4.1   NT 1 5.5
//   K = 5120, N = 1280    NT 1, 16 waves 5.4   NT 2 6.3
//   K = 8192, N = 8192    NT 2, 16 waves 12.1  NT 1 17.5
typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// The 16-bit type that the codes take, and the parts that a row's value is
// split into: fp32 rows become three bf16 (24 bits).
template <typename T> struct In4 {
  typedef b8 vec;
  static constexpr int P = sizeof(T) == 4 ? 3 : 1;
  // code + 24 of nibble i of a word: 16 + (code + 8), exact in 8 bits
  static constexpr uint32_t kMask = 0x00780078u, kBase = 0x41804180u;
  template <int I> static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    const uint32_t v = I == 0 ? w << 3 : w >> (4 * I - 3);
    return (v & kMask) | kBase;
  }
  static __device__ __forceinline__ f4 mfma(vec a, vec b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct In4<half_t> {
  typedef h8 vec;
  static constexpr int P = 1;
  static constexpr uint32_t kMask = 0x03c003c0u, kBase = 0x4c004c00u;
  template <int I> static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    const uint32_t v = I == 0 ? w << 6 : I == 1 ? w << 2 : w >> (4 * I - 6);
    return (v & kMask) | kBase;
  }
  static __device__ __forceinline__ f4 mfma(vec a, vec b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

template <typename T>
__device__ __forceinline__ typename In4<T>::vec codes24(uint32_t w) {
  const uint32_t r[4] = {In4<T>::template pair<0>(w), In4<T>::template pair<1>(w), In4<T>::template pair<2>(w),
                         In4<T>::template pair<3>(w)};
  typename In4<T>::vec o;
  __builtin_memcpy(&o, r, 16);
  return o;
}

// Rows of x [M, K] with zeros behind them, [M, ld].
template <typename T>
__global__ void __launch_bounds__(256) pad_rows_kernel(const T* __restrict__ x, int64_t sm, int64_t K,
                                                       T* __restrict__ out, int64_t ld) {
  const int64_t m = blockIdx.x;
  for (int64_t k = threadIdx.x; k < ld; k += 256) out[m * ld + k] = k < K ? x[m * sm + k] : (T)0.f;
}

struct L4Args {
  LinearInt4 a;
  int64_t steps;
  int nw;  // waves of a block
};

// What a wave keeps in flight: UN steps of 128 columns of codes, and the rows
// of XB steps (two where they fit the registers: those of the next step are
// loaded before this one is multiplied).
template <typename T, int MT, int NT, int G> struct InFlight {
  static constexpr int UN = NT == 1 ? 4 : 2;
  static constexpr int XB = sizeof(T) == 2 && MT <= 2 && !(MT == 1 && NT == 2 && G == 32) ? 2 : 1;
};

constexpr int kLnK = 2048, kLnX = 14336;  // row and elements of x that the normalising form holds (LDS: 64 KB with the sums)

// The rows of x normalised into LDS (row stride K + 8), a wave a row: the
// mean, then the mean square of the differences, from registers, rounded to T
// as layer_norm's own output is.  (gamma and beta loaded before the sums, or
// everything before the codes, take the registers that the codes are loaded
// into: 8.7 and 11.6 us a launch of a decode step against 7.4.)
template <typename T>
__device__ __forceinline__ void normalise_rows(const LinearInt4& a, T* xs, int K, int w, int nw, int lane) {
  const T* ga = (const T*)a.ln_gamma;
  const T* be = (const T*)a.ln_beta;
  for (int m = w; m < (int)a.M; m += nw) {
    const T* x = (const T*)a.x + m * a.x_sm;
    float v[kLnK / 512][8];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kLnK / 512; ++i) {
      const int k = (lane + 64 * i) * 8;
      T e[8];
      uint4 raw{0, 0, 0, 0};
      if (k < K) raw = *(const uint4*)(x + k);
      __builtin_memcpy(e, &raw, 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] = to_f(e[j]);
        sum += v[i][j];
      }
    }
    const float mean = wave_sum(sum) / (float)K;
    float var = 0.f;
#pragma unroll
    for (int i = 0; i < kLnK / 512; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = v[i][j] - mean;
        var += (lane + 64 * i) * 8 < K ? d * d : 0.f;
      }
    const float inv = 1.f / sqrtf(wave_sum(var) / (float)K + a.ln_eps);
#pragma unroll
    for (int i = 0; i < kLnK / 512; ++i) {
      const int k = (lane + 64 * i) * 8;
      if (k < K) {
        const uint4 gr = *(const uint4*)(ga + k), br = *(const uint4*)(be + k);
        T ge[8], bb[8], o[8];
        __builtin_memcpy(ge, &gr, 16);
        __builtin_memcpy(bb, &br, 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = from_f<T>(to_f(ge[j]) * (v[i][j] - mean) * inv + to_f(bb[j]));
        uint4 raw;
        __builtin_memcpy(&raw, o, 16);
        *(uint4*)(xs + m * (K + 8) + k) = raw;
      }
    }
  }
}

// A wave's share (steps w, w + nw, ..) of sum_k x[k] (code scale)[k] of one
// output, from the column's codes of its tile and its scales (N apart).
template <typename T, int G>
__device__ __forceinline__ float sum_of_values(const uint32_t* codes, const T* scales, const T* x, int64_t N,
                                                         int K, int w, int nw) {
  float v = 0.f;
#pragma unroll 1
  for (int k0 = 128 * w; k0 < K; k0 += 128 * nw) {
#pragma unroll 1
    for (int k = k0; k < k0 + 128 && k < K; k += 8) {
      const uint32_t word = codes[(int64_t)(k / 128) * 256 + (k % 128) / 32 * 64 + (k % 32) / 8];
      const float s = to_f(scales[k / G * N]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xe = k + e < K ? to_f(x[k + e]) : 0.f;
        if (k + e < K) v = fmaf(xe, (float)((int)((word >> (4 * nibble_of(e))) & 15) - 8) * s, v);
      }
      if (v != v) return v;
    }
  }
  return v;
}

// MT tiles of 16 rows of x by NT tiles of 16 columns of the output; the waves
// of a block take 128-deep steps of K in turn.  G: columns of a scale.  XVEC:
// K and the rows of x are such that 8 columns are one aligned load.  LN: the
// rows are normalised into LDS first, while the first codes are on their way.
template <typename T, int MT, int NT, int G, bool XVEC, bool LN>
__global__ void __launch_bounds__(MT == 1 ? 1024 : 512) linear_int4_mfma(L4Args g) {
  typedef In4<T> I;
  typedef typename I::vec V;
  constexpr int NG = 128 / G, UN = InFlight<T, MT, NT, G>::UN, XB = InFlight<T, MT, NT, G>::XB, XW = sizeof(T) / 2;
  static_assert(UN % XB == 0, "the rows' buffers follow the steps");
  static_assert(!LN || (XVEC && MT == 1 && sizeof(T) == 2), "few 16-bit rows of whole vectors");
  extern __shared__ float red[];  // [nw][MT][NT][16][16], then the normalised rows
  const LinearInt4& a = g.a;
  T* xs = (T*)(red + g.nw * MT * NT * 256);
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int steps = (int)g.steps, nw = g.nw, K = (int)a.K, groups = (K + G - 1) / G;
  const int64_t tiles = (a.N + 15) / 16, tile0 = (int64_t)blockIdx.x * NT, m0 = (int64_t)blockIdx.y * (16 * MT);
  const T* sc = (const T*)a.scales;

  V minus;  // -24: takes off what the codes are too large by
#pragma unroll
  for (int e = 0; e < 8; ++e) minus[e] = -24.f;

  const T* x[MT];
  bool row_ok[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = m0 + 16 * i + c;
    row_ok[i] = m < a.M;
    x[i] = (const T*)a.x + (row_ok[i] ? m : 0) * a.x_sm;
  }
  const uint4* wp[NT];
  int64_t col[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t t = tile0 + j < tiles ? tile0 + j : tiles - 1;
    wp[j] = (const uint4*)a.packed + t * steps * 64 + lane;
    col[j] = t * 16 + c < a.N ? t * 16 + c : a.N - 1;
  }

  uint4 wv[UN][NT];
  T sv[UN][NT];  // lane (c, q): the scale of column c for group q NG / 4 of the step
  auto load_w = [&](int u, int st) __attribute__((always_inline)) {
    st = st < steps ? st : steps - 1;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      wv[u][j] = wp[j][(int64_t)st * 64];
      const int gr = st * NG + q * NG / 4;
      sv[u][j] = sc[(int64_t)(gr < groups ? gr : groups - 1) * a.N + col[j]];
    }
  };
  // columns that word t of a lane's codes belongs to
  auto k_of = [&](int st, int t) __attribute__((always_inline)) {
    return st * 128 + (G < 128 ? 32 * t + 8 * q : 32 * q + 8 * t);
  };
  uint4 xr[XB][4][MT][XW];
  auto load_x = [&](int b, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int k = k_of(st, t);
#pragma unroll
        for (int e = 0; e < XW; ++e) xr[b][t][i][e] = uint4{0, 0, 0, 0};
        if constexpr (LN) {
          if (row_ok[i] && k < K) xr[b][t][i][0] = *(const uint4*)(xs + c * (K + 8) + k);
        } else if constexpr (XVEC) {
          if (row_ok[i] && k < K)
#pragma unroll
            for (int e = 0; e < XW; ++e) xr[b][t][i][e] = ((const uint4*)(x[i] + k))[e];
        } else {
          T v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = row_ok[i] && k + e < K ? x[i][k + e] : (T)0.f;
          __builtin_memcpy(xr[b][t][i], v, sizeof(v));
        }
      }
  };

  f4 tot[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) tot[i][j] = f4{0.f, 0.f, 0.f, 0.f};

  auto multiply = [&](int u, int b) __attribute__((always_inline)) {
    uint32_t word[NT][4];
    float sg[NT][NG];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      // each group's scale to all lanes of its column
      const uint32_t s1 = __float_as_uint(to_f(sv[u][j]));
      if constexpr (NG == 1) {
        sg[j][0] = __uint_as_float(s1);
      } else {
        const auto h = __builtin_amdgcn_permlane32_swap(s1, s1, false, false);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (NG == 2) {
            sg[j][i] = __uint_as_float(h[i]);
          } else {
            const auto r = __builtin_amdgcn_permlane16_swap(h[i], h[i], false, false);
            sg[j][2 * i] = __uint_as_float(r[0]);
            sg[j][2 * i + 1] = __uint_as_float(r[1]);
          }
        }
      }
      word[j][0] = wv[u][j].x; word[j][1] = wv[u][j].y; word[j][2] = wv[u][j].z; word[j][3] = wv[u][j].w;
      if constexpr (G < 128) {
        // lane (c, q) holds columns 32 q + 8 t of word t: exchanged between
        // the four lanes of a row so that word t holds 32 t + 8 q, and one
        // product covers 32 columns in a row, of one scale
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const auto r = __builtin_amdgcn_permlane32_swap(word[j][t], word[j][t + 2], false, false);
          word[j][t] = r[0]; word[j][t + 2] = r[1];
        }
#pragma unroll
        for (int t = 0; t < 4; t += 2) {
          const auto r = __builtin_amdgcn_permlane16_swap(word[j][t], word[j][t + 1], false, false);
          word[j][t] = r[0]; word[j][t + 1] = r[1];
        }
      }
    }
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      f4 acc[MT][NT], cor[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        cor[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int t = gr * 4 / NG; t < (gr + 1) * 4 / NG; ++t) {
        V wf[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) wf[j] = codes24<T>(word[j][t]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if constexpr (I::P == 1) {
            V xf;
            __builtin_memcpy(&xf, xr[b][t][i], 16);
            cor[i] = I::mfma(xf, minus, cor[i]);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = I::mfma(xf, wf[j], acc[i][j]);
          } else {
            float f[8];
            __builtin_memcpy(f, xr[b][t][i], 32);
#pragma unroll
            for (int p = 0; p < 3; ++p) {
              V xf;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                xf[e] = (__bf16)f[e];
                f[e] -= (float)xf[e];
              }
              cor[i] = I::mfma(xf, minus, cor[i]);
#pragma unroll
              for (int j = 0; j < NT; ++j) acc[i][j] = I::mfma(xf, wf[j], acc[i][j]);
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float s = sg[j][gr];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) tot[i][j][e] += s * (acc[i][j][e] + cor[i][e]);
      }
      // (the groups' products one after another: together their sums would
      // not fit the registers)
      if constexpr (NG > 1 && MT * NT > 1) __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (w < steps) {
#pragma unroll
    for (int u = 0; u < UN; ++u) load_w(u, w + u * nw);
  }
  if constexpr (LN) {
    normalise_rows<T>(a, xs, K, w, nw, lane);
    __syncthreads();
  }
  if constexpr (XB == 2)
    if (w < steps) load_x(0, w);
  for (int s0 = w; s0 < steps; s0 += nw * UN) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int st = s0 + u * nw;
      if (st >= steps) break;
      if constexpr (XB == 1) load_x(0, st);
      else if (st + nw < steps) load_x((u + 1) % 2, st + nw);
      multiply(u, u % XB);
      if (st + nw * UN < steps) load_w(u, st + nw * UN);
    }
  }

  // lane (c, q) holds rows 4 q + e, column c of each tile; the waves' sums
  // are added in wave order
  bool past = false;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        red[((w * MT + i) * NT + j) * 256 + (4 * q + e) * 16 + c] = tot[i][j][e];
        past |= !(fabsf(tot[i][j][e]) < INFINITY);
      }
  if (past) {
    // An infinity, and an x past 2^112, are infinities of both signs in the two
    // products and NaN in their sum (so is the first part of an fp32 x that
    // rounds up to 2^128): this lane's sums that are not finite are taken again
    // from the weights' values, and are then what the products give.
#pragma unroll 1
    for (int at = 0; at < MT * NT * 4; ++at) {
      const int e = at & 3, j = (at >> 2) % NT, i = (at >> 2) / NT;
      float* sum = red + ((w * MT + i) * NT + j) * 256 + (4 * q + e) * 16 + c;
      const int64_t m = m0 + 16 * i + 4 * q + e, n = (tile0 + j) * 16 + c;
      if (fabsf(*sum) < INFINITY || m >= a.M || n >= a.N) continue;
      const T* xm = LN ? xs + m * (K + 8) : (const T*)a.x + m * a.x_sm;
      *sum = sum_of_values<T, G>((const uint32_t*)a.packed + (tile0 + j) * steps * 256 + c * 4, sc + n, xm, a.N, K, w, nw);
    }
  }
  __syncthreads();
  for (int idx = tid; idx < MT * NT * 256; idx += 64 * g.nw) {
    const int cc = idx & 15, j = (idx >> 4) % NT, mm = idx / (16 * NT);
    const int64_t m = m0 + mm, n = (tile0 + j) * 16 + cc;
    if (m >= a.M || n >= a.N) continue;
    const int at = ((mm >> 4) * NT + j) * 256 + (mm & 15) * 16 + cc;
    float v = 0.f;
    for (int i = 0; i < g.nw; ++i) v += red[i * MT * NT * 256 + at];
    if (a.bias) v += to_f(((const T*)a.bias)[n]);
    v = act_of(v, a.act);
    if (a.residual) v += to_f(((const T*)a.residual)[m * a.N + n]);
    ((T*)a.out)[m * a.N + n] = from_f<T>(v);
  }
}

template <typename T, int MT, int NT, int G>
void launch_int4(const L4Args& g, bool xvec, hipStream_t s) {
  const int64_t tiles = (g.a.N + 15) / 16, bx = (tiles + NT - 1) / NT, by = (g.a.M + 16 * MT - 1) / (16 * MT);
  const dim3 grid((unsigned)bx, (unsigned)by);
  const size_t lds = (size_t)g.nw * MT * NT * 256 * sizeof(float);
  if constexpr (MT == 1 && sizeof(T) == 2) {
    if (g.a.ln_gamma) {
      hipLaunchKernelGGL((linear_int4_mfma<T, MT, NT, G, true, true>), grid, dim3(64 * g.nw),
                         lds + (size_t)g.a.M * (g.a.K + 8) * sizeof(T), s, g);
      return;
    }
  }
  if constexpr (MT == 1) {
    if (!xvec) {
      hipLaunchKernelGGL((linear_int4_mfma<T, MT, NT, G, false, false>), grid, dim3(64 * g.nw), lds, s, g);
      return;
    }
  }
  hipLaunchKernelGGL((linear_int4_mfma<T, MT, NT, G, true, false>), grid, dim3(64 * g.nw), lds, s, g);
}

template <typename T, int MT, int NT>
void launch_int4_g(const L4Args& g, bool xvec, hipStream_t s) {
  // (64 rows' sums for groups of 32 fit the registers for one tile of columns)
  if (g.a.group == 32) launch_int4<T, MT, MT == 4 ? 1 : NT, 32>(g, xvec, s);
  else if (g.a.group == 64) launch_int4<T, MT, NT, 64>(g, xvec, s);
  else launch_int4<T, MT, NT, 128>(g, xvec, s);
}

}  // namespace

int64_t int4_bytes(int64_t N, int64_t K) { return (N + 15) / 16 * ((K + 127) / 128) * 1024; }

static unsigned grid_for(int64_t n) {
  const int64_t b = (n + 255) / 256;
  return (unsigned)(b < 1 ? 1 : b > 65536 ? 65536 : b);
}

void quantize_int4(DType dt, const void* w, int64_t sn, int64_t sk, int64_t N, int64_t K, int64_t group,
                   uint8_t* packed, void* scales, hipStream_t s) {
  const int64_t steps = (K + 127) / 128, words = int4_bytes(N, K) / 4, n_s = (K + group - 1) / group * N;
  AGPU_FLOAT_SWITCH(dt, {
    hipLaunchKernelGGL((int4_scales_kernel<T>), dim3(grid_for(n_s)), dim3(256), 0, s, (const T*)w, sn, sk, N, K, group,
                       (T*)scales, n_s);
    hipLaunchKernelGGL((quantize_int4_kernel<T>), dim3(grid_for(words)), dim3(256), 0, s, (const T*)w, sn, sk, N, K,
                       group, (const T*)scales, (uint32_t*)packed, words, steps);
  });
  check_launch("quantize_int4");
}

void dequantize_int4(DType dt, const uint8_t* packed, const void* scales, int64_t N, int64_t K, int64_t group,
                     void* out, int64_t ld, hipStream_t s) {
  const int64_t steps = (K + 127) / 128, runs = (N + 15) / 16 * steps * 64;
  const bool vec = ((uintptr_t)out & 15) == 0 && ld * (int64_t)dtype_size(dt) % 16 == 0;
  AGPU_FLOAT_SWITCH(dt, {
    if (vec) hipLaunchKernelGGL((dequantize_int4_kernel<T, true>), dim3(grid_for(runs)), dim3(256), 0, s,
                                (const uint4*)packed, (const T*)scales, N, K, group, (T*)out, ld, runs, steps);
    else hipLaunchKernelGGL((dequantize_int4_kernel<T, false>), dim3(grid_for(runs)), dim3(256), 0, s,
                            (const uint4*)packed, (const T*)scales, N, K, group, (T*)out, ld, runs, steps);
  });
  check_launch("dequantize_int4");
}

void pad_rows(DType dt, const void* x, int64_t sm, int64_t M, int64_t K, void* out, int64_t ld, hipStream_t s) {
  if (M == 0) return;
  if (M > 0x7fffffffLL) fail("pad_rows: too many rows");
  AGPU_FLOAT_SWITCH(dt, hipLaunchKernelGGL((pad_rows_kernel<T>), dim3((unsigned)M), dim3(256), 0, s, (const T*)x, sm, K,
                                           (T*)out, ld));
  check_launch("pad_rows");
}

static bool int4_rows_aligned(const LinearInt4& a) {
  return a.K % 8 == 0 && ((uintptr_t)a.x & 15) == 0 && (a.M == 1 || a.x_sm * (int64_t)dtype_size(a.dt) % 16 == 0);
}

bool linear_int4_ln_ok(const LinearInt4& a) {
  return a.dt != DType::F32 && a.M >= 1 && a.M <= 16 && a.K <= kLnK && a.M * a.K <= kLnX && int4_rows_aligned(a) &&
         ((uintptr_t)a.ln_gamma & 15) == 0 && ((uintptr_t)a.ln_beta & 15) == 0;
}

void linear_int4(const LinearInt4& a, hipStream_t s) {
  if (a.M == 0) return;
  if (a.ln_gamma && !linear_int4_ln_ok(a)) fail("linear_int4: these rows cannot be normalised in the product");
  if (a.K > 0x7fffff00LL || (a.N + 15) / 16 > 0x7fffffffLL)
    fail("linear_int4: too many rows or columns");
  constexpr int64_t kMost = 65535 * 64;  // rows of a grid
  if (a.M > kMost) {
    const int64_t es = (int64_t)dtype_size(a.dt);
    for (int64_t m = 0; m < a.M; m += kMost) {
      LinearInt4 part = a;
      part.M = a.M - m < kMost ? a.M - m : kMost;
      part.x = (const char*)a.x + m * a.x_sm * es;
      part.out = (char*)a.out + m * a.N * es;
      if (a.residual) part.residual = (const char*)a.residual + m * a.N * es;
      linear_int4(part, s);
    }
    return;
  }
  L4Args g;
  g.a = a;
  g.steps = (a.K + 127) / 128;
  const bool xvec = int4_rows_aligned(a);
  if (!xvec && a.M > 1) fail("linear_int4: rows are not aligned");
  // 16, 32 or 64 rows a block; two tiles of columns from 320 tiles on, and
  // about 4096 waves in all (measured above)
  const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
  const int64_t tiles = (a.N + 15) / 16;
  const bool wide = mt > 1 || tiles >= 320;
  const int64_t rows = (a.M + 16 * mt - 1) / (16 * mt);
  const int64_t blocks = (tiles + wide) / (1 + wide) * rows, most = mt == 1 ? 16 : 8;
  int64_t nw = 4096 / blocks;
  nw = nw < 2 ? 2 : nw > most ? most : nw;
  g.nw = (int)(g.steps < nw ? g.steps : nw);
  AGPU_FLOAT_SWITCH(a.dt, {
    if (mt == 1 && !wide) launch_int4_g<T, 1, 1>(g, xvec, s);
    else if (mt == 1) launch_int4_g<T, 1, 2>(g, xvec, s);
    else if (mt == 2) launch_int4_g<T, 2, 2>(g, xvec, s);
    else launch_int4_g<T, 4, 2>(g, xvec, s);
  });
  check_launch("linear_int4");
}

}  // namespace k
}  // namespace agpu
