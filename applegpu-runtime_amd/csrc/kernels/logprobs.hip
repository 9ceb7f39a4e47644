// Log probabilities of given tokens, with the entropy of each row's
// distribution and its most likely alternatives, and the gradient of the
// first two.  For a row z of V logits with m = max z, e_j = exp(z_j - m):
//   lse = m + log sum e       lp = z_t - lse      H = log sum e - sum e_j (z_j - m) / sum e
//   dz_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H)
// Sums are kept in fp32.  The elements at the maximum count one each: they
// are counted apart from the others, so that log sum e = log1p(..) keeps its
// digits where one token has nearly all of the probability.
// A row of -inf only has no distribution: lse and lp are -inf, H 0, and its
// gradient is 0.
#include "device.hpp"

namespace agpu {
namespace k {
using namespace dev;

namespace {

struct LpArgs {
  TokenLogprobs a;
};

// Unsigned integers in the order of the floats, -0 as 0, NaN above all.
__device__ __forceinline__ uint32_t order_of(float z) {
  if (z != z) return 0xffffffffu;
  const uint32_t u = __float_as_uint(z + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// A logit and its index as one number: larger logits first, then lower indices.
__device__ __forceinline__ uint64_t key_of(float z, uint32_t j) {
  return ((uint64_t)order_of(z) << 32) | (0xffffffffu - j);
}

__device__ __forceinline__ uint64_t wave_kmax(uint64_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), m, 64) << 32) |
                       (uint32_t)__shfl_xor((int)(uint32_t)v, m, 64);
    v = o > v ? o : v;
  }
  return v;
}

template <int NW>
__device__ __forceinline__ uint64_t block_kmax(uint64_t v, uint64_t* sh) {
  v = wave_kmax(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t r = sh[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) r = sh[i] > r ? sh[i] : r;
  return r;
}

template <int NW>
__device__ __forceinline__ float block_add(float v, float* sh) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) r += sh[i];
  return r;
}

__device__ __forceinline__ int64_t token_at(const TokenLogprobs& a, int64_t r) {
  return a.idx_dt == DType::I64 ? ((const int64_t*)a.tokens)[r] : (int64_t)((const int32_t*)a.tokens)[r];
}

// One block per row: a pass for the maximum, one for the sums, one for each
// alternative.
template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_row(LpArgs g) {
  const TokenLogprobs& a = g.a;
  __shared__ uint64_t shk[4];
  __shared__ float shf[4];
  const int64_t r = blockIdx.x;
  const T* z = (const T*)a.z + r * a.ld;
  const int tid = threadIdx.x;
  uint64_t best = 0;
  for (int64_t j = tid; j < a.V; j += 256) {
    const uint64_t k = key_of(to_f(z[j]), (uint32_t)j);
    best = k > best ? k : best;
  }
  best = block_kmax<4>(best, shk);
  const float m = to_f(z[0xffffffffu - (uint32_t)best]);
  float ones = 0.f, rest = 0.f, dot = 0.f;
  for (int64_t j = tid; j < a.V; j += 256) {
    const float d = to_f(z[j]) - m, e = expf(d);
    ones += d == 0.f ? 1.f : 0.f;
    rest += d == 0.f ? 0.f : e;
    dot += e == 0.f ? 0.f : e * d;
  }
  ones = block_add<4>(ones, shf);
  rest = block_add<4>(rest, shf);
  dot = block_add<4>(dot, shf);
  const bool none = m == -INFINITY;
  const float logl = none ? 0.f : log1pf((ones - 1.f) + rest), lse = none ? m : m + logl;
  if (tid == 0) {
    const int64_t t = token_at(a, r);
    a.lp[r] = t < 0 || t >= a.V ? 0.f : none ? m : (to_f(z[t]) - m) - logl;
    a.entropy[r] = none ? 0.f : logl - dot / (ones + rest);
    a.lse[r] = lse;
  }
  for (int i = 0; i < a.top_k; ++i) {
    if (i > 0) {
      uint64_t next = 0;
      for (int64_t j = tid; j < a.V; j += 256) {
        const uint64_t k = key_of(to_f(z[j]), (uint32_t)j);
        if (k < best && k > next) next = k;
      }
      best = block_kmax<4>(next, shk);
    }
    if (tid == 0) {
      const uint32_t j = 0xffffffffu - (uint32_t)best;
      a.top_ids[r * a.top_k + i] = (int32_t)j;
      a.top_lp[r * a.top_k + i] = none ? m : (to_f(z[j]) - m) - logl;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_grad(LpArgs g, const float* __restrict__ g_lp,
                                                           const float* __restrict__ g_h, T* __restrict__ dz) {
  const TokenLogprobs& a = g.a;
  const int64_t r = blockIdx.x, t = token_at(a, r);
  const T* z = (const T*)a.z + r * a.ld;
  const float lse = a.lse[r];
  const float gl = t >= 0 && t < a.V ? g_lp[r] : 0.f, gh = g_h ? g_h[r] : 0.f, H = g_h ? a.entropy[r] : 0.f;
  for (int64_t j = (int64_t)blockIdx.y * 256 + threadIdx.x; j < a.V; j += (int64_t)gridDim.y * 256) {
    float v = 0.f;
    if (lse != -INFINITY) {
      const float lp = to_f(z[j]) - lse, p = expf(lp);
      v = (j == t ? gl : 0.f) - p * gl;
      if (p != 0.f) v -= gh * p * (lp + H);
    }
    dz[r * a.V + j] = from_f<T>(v);
  }
}

}  // namespace

size_t token_logprobs_ws_bytes(const TokenLogprobs&) { return 0; }

void token_logprobs(const TokenLogprobs& a, void* ws, hipStream_t s) {
  (void)ws;
  if (a.R == 0) return;
  if (a.R > 0x7fffffffLL) fail("token_logprobs: too many rows");
  LpArgs g{a};
  AGPU_FLOAT_SWITCH(a.dt, hipLaunchKernelGGL((token_logprobs_row<T>), dim3((unsigned)a.R), dim3(256), 0, s, g));
  check_launch("token_logprobs");
}

void token_logprobs_backward(const TokenLogprobs& a, const float* g_lp, const float* g_H, void* dz, hipStream_t s) {
  if (a.R == 0) return;
  LpArgs g{a};
  int64_t by = (a.V + 2047) / 2048;
  if (by > 65535) by = 65535;
  if (a.R > 0x7fffffffLL) fail("token_logprobs_backward: too many rows");
  AGPU_FLOAT_SWITCH(a.dt, hipLaunchKernelGGL((token_logprobs_grad<T>), dim3((unsigned)a.R, (unsigned)by), dim3(256), 0,
                                             s, g, g_lp, g_H, (T*)dz));
  check_launch("token_logprobs_backward");
}

}  // namespace k
}  // namespace agpu
