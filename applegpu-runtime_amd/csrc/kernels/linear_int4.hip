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

template <typename T>
__global__ void __launch_bounds__(256) dequantize_int4_kernel(const uint32_t* __restrict__ packed,
                                                              const T* __restrict__ scales, int64_t N, int64_t K,
                                                              int64_t group, T* __restrict__ out, int64_t ld,
                                                              int64_t words, int64_t steps) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
    // words of a row of W in a row, so that the stores are contiguous
    const int64_t wpr = steps * 16, n = i / wpr, kw = i % wpr, k0 = kw * 8;
    if (k0 >= K) continue;
    const int64_t step = kw >> 4;
    const int run = (int)(n & 15) + 16 * (int)((kw >> 2) & 3), word = (int)(kw & 3);
    const uint32_t v = packed[(((n >> 4) * steps + step) * 64 + run) * 4 + word];
    const float s = to_f(scales[k0 / group * N + n]);
    for (int e = 0; e < 8; ++e)
      if (k0 + e < K) out[n * ld + k0 + e] = from_f<T>((float)((int)((v >> (4 * nibble_of(e))) & 15) - 8) * s);
  }
}

struct L4Args {
  LinearInt4 a;
  int64_t steps;
};

__device__ __forceinline__ float act_of(float v, int act) {
  if (act == kActRelu) return v > 0.f ? v : (v != v ? v : 0.f);
  if (act == kActGelu) return gelu_tanh(v);
  if (act == kActGeluExact) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
  return v;
}

// One wave per 16 columns of the output and row of x: lane l sums the codes
// of its run (row l % 16 of the tile) against x.
template <typename T>
__global__ void __launch_bounds__(64) linear_int4_row(L4Args g) {
  const LinearInt4& a = g.a;
  const int lane = threadIdx.x;
  const int64_t tile = blockIdx.y, m = blockIdx.x, n = tile * 16 + (lane & 15);
  const T* x = (const T*)a.x + m * a.x_sm;
  const T* sc = (const T*)a.scales;
  float acc = 0.f;
  for (int64_t st = 0; st < g.steps; ++st) {
    const uint4 w = *(const uint4*)(a.packed + ((tile * g.steps + st) * 64 + lane) * 16);
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    const int64_t k0 = st * 128 + (lane >> 4) * 32;
    if (k0 >= a.K || n >= a.N) continue;
    float part = 0.f;
    for (int i = 0; i < 4; ++i)
      for (int e = 0; e < 8; ++e) {
        const int64_t k = k0 + i * 8 + e;
        if (k < a.K) part += to_f(x[k]) * (float)((int)((ws[i] >> (4 * nibble_of(e))) & 15) - 8);
      }
    acc += part * to_f(sc[k0 / a.group * a.N + n]);
  }
  acc += __shfl_xor(acc, 16, 64);
  acc += __shfl_xor(acc, 32, 64);
  if (lane < 16 && n < a.N) {
    if (a.bias) acc += to_f(((const T*)a.bias)[n]);
    ((T*)a.out)[m * a.N + n] = from_f<T>(act_of(acc, a.act));
  }
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
  const int64_t steps = (K + 127) / 128, words = N * steps * 16;
  AGPU_FLOAT_SWITCH(dt, hipLaunchKernelGGL((dequantize_int4_kernel<T>), dim3(grid_for(words)), dim3(256), 0, s,
                                           (const uint32_t*)packed, (const T*)scales, N, K, group, (T*)out, ld, words,
                                           steps));
  check_launch("dequantize_int4");
}

void linear_int4(const LinearInt4& a, hipStream_t s) {
  if (a.M == 0) return;
  L4Args g;
  g.a = a;
  g.steps = (a.K + 127) / 128;
  if (a.M > 0x7fffffffLL || a.N > 65535 * 16) fail("linear_int4: too many rows or columns");
  const dim3 grid((unsigned)a.M, (unsigned)((a.N + 15) / 16));
  AGPU_FLOAT_SWITCH(a.dt, hipLaunchKernelGGL((linear_int4_row<T>), grid, dim3(64), 0, s, g));
  check_launch("linear_int4");
}

}  // namespace k
}  // namespace agpu
