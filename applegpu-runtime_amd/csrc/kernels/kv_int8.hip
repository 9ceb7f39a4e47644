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
// their codes and, for the first block, the codes before them.  Bound by HBM
// for prompts (8 x 20 x 509 rows of 64 in f16: 31 MB in 11.3 us, 2.8 TB/s, the
// read back 8.5 us, 3.7 TB/s), where a wave's chain of load, maximum, scale and
// codes keeps it from more; by latency for a token (5 us).
#include "kv_int8.hpp"

namespace agpu {
namespace k {
using namespace dev;

namespace {

struct KvArgs8 {
  KvInt8 a;
  int lg_block, lg_cpr;  // log2 of the block and of the 8-code chunks of a row
  uint32_t nbt, waves;   // blocks an append touches at most; B * H * nbt
};

template <typename T, int NC>
__global__ void __launch_bounds__(256) kv_write_int8_kernel(KvArgs8 g) {
  const KvInt8& a = g.a;
  const int lane = threadIdx.x & 63, j = blockIdx.y;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (wave >= g.waves) return;
  const uint32_t bh = wave / g.nbt, nb = wave % g.nbt, h = bh % (uint32_t)a.H, b = bh / (uint32_t)a.H;
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
  const T* x = (const T*)a.x[j] + b * a.xs[j][0] + h * a.xs[j][1] + (r0 - p) * a.xs[j][2];
  kv8::append_rows<T, NC>(x, a.xs[j][2], codes, c.cs[2], scale, lo, r0, r1, g.lg_cpr, lane);
}

// A block per 2048 values of a (sequence, head): 8 a thread.
template <typename T>
__global__ void __launch_bounds__(256) kv_read_int8_kernel(KvArgs8 g, T* y0, T* y1, uint32_t per) {
  const KvInt8& a = g.a;
  const int j = blockIdx.y;
  const uint32_t bh = blockIdx.x / per, h = bh % (uint32_t)a.H, b = bh / (uint32_t)a.H;
  const int64_t i = (int64_t)(blockIdx.x % per) * 256 + threadIdx.x, t = i >> g.lg_cpr;
  if (t >= a.T) return;
  const int d = (int)(i & ((1 << g.lg_cpr) - 1)) * 8;
  const Int8Cache& c = a.c[j];
  const int64_t r = (int64_t)a.pos[b] + t;
  uint2 w{0, 0};
  float s = 0.f;
  if (r >= 0 && r < a.Tmax) {
    w = *(const uint2*)(c.codes + b * c.cs[0] + h * c.cs[1] + r * c.cs[2] + d);
    s = c.scales[b * c.ss[0] + h * c.ss[1] + (r >> g.lg_block) * c.ss[2]];
  }
  int8_t o[8];
  __builtin_memcpy(o, &w, 8);
  T e[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) e[k] = from_f<T>((float)o[k] * s);
  uint4 raw[sizeof(T) / 2];
  __builtin_memcpy(raw, e, sizeof(e));
  T* y = (j ? y1 : y0) + (bh * a.T + t) * a.D + d;
#pragma unroll
  for (int k = 0; k < (int)sizeof(T) / 2; ++k) ((uint4*)y)[k] = raw[k];
}

int lg2(int64_t v) {
  int l = 0;
  while ((1ll << l) < v) ++l;
  return l;
}

// Fails where the grid would not hold `blocks` blocks.
KvArgs8 kv_args(const char* name, const KvInt8& a, int64_t blocks) {
  if (!kv_int8_supported(a.D, a.block)) fail("%s: head dim %lld or block %d not supported", name, (long long)a.D, a.block);
  if (blocks > 0x7fffffffLL / 4) fail("%s: too many rows", name);
  KvArgs8 g;
  g.a = a;
  g.lg_block = lg2(a.block);
  g.lg_cpr = lg2(a.D / 8);
  g.nbt = (uint32_t)((a.T + a.block - 2) / a.block + 1);
  g.waves = (uint32_t)(a.B * a.H * g.nbt);
  return g;
}

}  // namespace

bool kv_int8_supported(int64_t D, int64_t block) {
  return (D == 32 || D == 64 || D == 128) && (block == 16 || block == 32 || block == 64 || block == 128);
}

void kv_write_int8(const KvInt8& a, hipStream_t s) {
  if (a.B * a.H * a.T == 0) return;
  const int64_t waves = a.B * a.H * ((a.T + a.block - 2) / a.block + 1);
  const KvArgs8 g = kv_args("kv_write_int8", a, waves);
  const dim3 grid((unsigned)((waves + 3) / 4), 2);
  // 64-chunk parts of the new rows of a block
  const int64_t parts = ((a.T < a.block ? a.T : a.block) * (a.D / 8) + 63) / 64;
  AGPU_FLOAT_SWITCH(a.dt, {
    if (parts <= 1) hipLaunchKernelGGL((kv_write_int8_kernel<T, 1>), grid, dim3(256), 0, s, g);
    else if (parts <= 2) hipLaunchKernelGGL((kv_write_int8_kernel<T, 2>), grid, dim3(256), 0, s, g);
    else if (parts <= 4) hipLaunchKernelGGL((kv_write_int8_kernel<T, 4>), grid, dim3(256), 0, s, g);
    else if (parts <= 8) hipLaunchKernelGGL((kv_write_int8_kernel<T, 8>), grid, dim3(256), 0, s, g);
    else hipLaunchKernelGGL((kv_write_int8_kernel<T, 0>), grid, dim3(256), 0, s, g);
  });
  check_launch("kv_write_int8");
}

void kv_read_int8(const KvInt8& a, void* const y[2], hipStream_t s) {
  if (a.B * a.H * a.T == 0) return;
  const int64_t per = (a.T * (a.D / 8) + 255) / 256;
  const KvArgs8 g = kv_args("kv_read_int8", a, a.B * a.H * per);
  const dim3 grid((unsigned)(a.B * a.H * per), 2);
  AGPU_FLOAT_SWITCH(a.dt, hipLaunchKernelGGL((kv_read_int8_kernel<T>), grid, dim3(256), 0, s, g, (T*)y[0], (T*)y[1],
                                             (uint32_t)per));
  check_launch("kv_read_int8");
}

}  // namespace k
}  // namespace agpu
