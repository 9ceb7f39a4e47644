// Append to and read of a K/V cache held in 8 bits: codes int8 [B, H, Tmax, D]
// and one fp32 scale per (sequence, head, block of 16 .. 128 rows).
//
// An append of rows x at row p of a block that begins at row lo:
//   s  = max(lo < p ? s_old : 0, max |x| / 127)
//   c  = clamp(rint(x / s), -127, 127)              for the new rows
//   c' = rint(c_old * (s_old / s))                  for rows lo .. p - 1, if s > s_old
// so that a block written at once is rounded once, and one that grows row by
// row keeps its rows to half a step for each time that its scale grew (about
// ln(block) times for rows of one distribution).  What the block holds from
// row p on is dropped by the append: rows past the written ones are neither
// read nor written.
//
// Magnitudes are compared as their bit patterns (the order of non-negative
// floats), in which infinities and NaN are the largest: a block that is given
// one gets it as its scale, with codes 0, and reads as NaN.
//
// One wave per (sequence, head, touched block); all traffic is the new rows,
// their codes and, for the first block, the codes before them.
#include "device.hpp"

namespace agpu {
namespace k {
using namespace dev;

namespace {

struct KvArgs8 {
  KvInt8 a;
  int lg_block, lg_cpr;  // log2 of the block and of the 8-code chunks of a row
  int64_t nbt, waves;    // blocks an append touches at most; B * H * nbt
};

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, m, 64);
    v = o > v ? o : v;
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void load_row8(const T* p, float (&x)[8]) {
  uint4 raw[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = ((const uint4*)p)[i];
  T e[8];
  __builtin_memcpy(e, raw, sizeof(e));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f(e[i]);
}

// code of x for scale s (0 where the scale says nothing: 0, infinite or NaN)
__device__ __forceinline__ int code_of(float x, float s, bool ok) {
  const float r = ok ? rintf(x / s) : 0.f;
  return (int)fminf(fmaxf(r, -127.f), 127.f);
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

template <typename T>
__global__ void __launch_bounds__(256) kv_write_int8_kernel(KvArgs8 g) {
  const KvInt8& a = g.a;
  const int lane = threadIdx.x & 63, j = blockIdx.y;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (wave >= g.waves) return;
  const int64_t nb = wave % g.nbt, bh = wave / g.nbt, h = bh % a.H, b = bh / a.H;
  const int64_t p = (int64_t)a.pos[b] + a.pos_off;
  const int64_t first = p > 0 ? p : 0;  // first row written
  int64_t end = p + a.T;
  if (end > a.Tmax) end = a.Tmax;
  const int64_t n = (first >> g.lg_block) + nb, lo = n << g.lg_block;
  const int64_t r0 = lo > first ? lo : first;
  const int64_t r1 = lo + a.block < end ? lo + a.block : end;
  if (r0 >= r1) return;
  const Int8Cache& c = a.c[j];
  int8_t* codes = c.codes + b * c.cs[0] + h * c.cs[1];
  float* scale = c.scales + b * c.ss[0] + h * c.ss[1] + n * c.ss[2];
  const T* x = (const T*)a.x[j] + b * a.xs[j][0] + h * a.xs[j][1];
  const int cpr = 1 << g.lg_cpr;
  const int chunks = (int)(r1 - r0) << g.lg_cpr;

  uint32_t top = 0;
  for (int i = lane; i < chunks; i += 64) {
    float v[8];
    load_row8(x + (r0 + (i >> g.lg_cpr) - p) * a.xs[j][2] + (i & (cpr - 1)) * 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t m = __float_as_uint(v[e]) & 0x7fffffffu;
      top = m > top ? m : top;
    }
  }
  uint32_t s_bits = __float_as_uint(__uint_as_float(wave_umax(top)) / 127.f) & 0x7fffffffu;
  const uint32_t was = r0 > lo ? __float_as_uint(*scale) & 0x7fffffffu : 0u;
  if (was > s_bits) s_bits = was;
  const float s = __uint_as_float(s_bits);
  const bool ok = s > 0.f && s < INFINITY;

  if (s_bits != was) {  // rows before the append, if any, take the grown scale
    const int held = (int)(r0 - lo) << g.lg_cpr;
    const float rate = ok ? __uint_as_float(was) / s : 0.f;
    for (int i = lane; i < held; i += 64) {
      int8_t* q = codes + (lo + (i >> g.lg_cpr)) * c.cs[2] + (i & (cpr - 1)) * 8;
      const uint2 w = *(const uint2*)q;
      int8_t o[8];
      __builtin_memcpy(o, &w, 8);
      int cc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) cc[e] = (int)rintf((float)o[e] * rate);
      store_codes(q, cc);
    }
  }
  for (int i = lane; i < chunks; i += 64) {
    const int64_t r = r0 + (i >> g.lg_cpr);
    const int d = (i & (cpr - 1)) * 8;
    float v[8];
    load_row8(x + (r - p) * a.xs[j][2] + d, v);
    int cc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) cc[e] = code_of(v[e], s, ok);
    store_codes(codes + r * c.cs[2] + d, cc);
  }
  if (lane == 0) *scale = s;
}

template <typename T>
__global__ void __launch_bounds__(256) kv_read_int8_kernel(KvArgs8 g, T* y0, T* y1, int64_t n) {
  const KvInt8& a = g.a;
  const int j = blockIdx.y;
  T* y = j ? y1 : y0;
  const Int8Cache& c = a.c[j];
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i >> g.lg_cpr;
    const int d = (int)(i & ((1 << g.lg_cpr) - 1)) * 8;
    const int64_t t = row % a.T, bh = row / a.T, h = bh % a.H, b = bh / a.H;
    const int64_t r = (int64_t)a.pos[b] + t;
    T e[8];
    if (r >= 0 && r < a.Tmax) {
      const uint2 w = *(const uint2*)(c.codes + b * c.cs[0] + h * c.cs[1] + r * c.cs[2] + d);
      const float s = c.scales[b * c.ss[0] + h * c.ss[1] + (r >> g.lg_block) * c.ss[2]];
      int8_t o[8];
      __builtin_memcpy(o, &w, 8);
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = from_f<T>((float)o[k] * s);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = from_f<T>(0.f);
    }
    uint4 raw[sizeof(T) / 2];
    __builtin_memcpy(raw, e, sizeof(e));
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) ((uint4*)(y + row * a.D + d))[k] = raw[k];
  }
}

int lg2(int64_t v) {
  int l = 0;
  while ((1ll << l) < v) ++l;
  return l;
}

KvArgs8 kv_args(const KvInt8& a) {
  KvArgs8 g;
  g.a = a;
  g.lg_block = lg2(a.block);
  g.lg_cpr = lg2(a.D / 8);
  g.nbt = (a.T + a.block - 2) / a.block + 1;
  g.waves = a.B * a.H * g.nbt;
  return g;
}

}  // namespace

bool kv_int8_supported(int64_t D, int64_t block) {
  return (D == 32 || D == 64 || D == 128) && (block == 16 || block == 32 || block == 64 || block == 128);
}

void kv_write_int8(const KvInt8& a, hipStream_t s) {
  if (!kv_int8_supported(a.D, a.block)) fail("kv_write_int8: head dim %lld or block %d not supported", (long long)a.D, a.block);
  if (a.B * a.H * a.T == 0) return;
  const KvArgs8 g = kv_args(a);
  if ((g.waves + 3) / 4 > 0x7fffffffLL) fail("kv_write_int8: too many rows");
  const dim3 grid((unsigned)((g.waves + 3) / 4), 2);
  AGPU_FLOAT_SWITCH(a.dt, hipLaunchKernelGGL((kv_write_int8_kernel<T>), grid, dim3(256), 0, s, g));
  check_launch("kv_write_int8");
}

void kv_read_int8(const KvInt8& a, void* const y[2], hipStream_t s) {
  if (!kv_int8_supported(a.D, a.block)) fail("kv_read_int8: head dim %lld or block %d not supported", (long long)a.D, a.block);
  const int64_t n = a.B * a.H * a.T * (a.D / 8);
  if (n == 0) return;
  const KvArgs8 g = kv_args(a);
  int64_t blocks = (n + 255) / 256;
  if (blocks > 65536) blocks = 65536;
  AGPU_FLOAT_SWITCH(a.dt, hipLaunchKernelGGL((kv_read_int8_kernel<T>), dim3((unsigned)blocks, 2), dim3(256), 0, s, g,
                                             (T*)y[0], (T*)y[1], n));
  check_launch("kv_read_int8");
}

}  // namespace k
}  // namespace agpu
