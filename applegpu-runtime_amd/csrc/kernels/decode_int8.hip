// Attention over a K/V cache held in 8 bits (codes int8, one fp32 scale per
// block of rows and head):
//   s_j = scale ks[j / block] sum_d q_d kc[j, d],   j < visible rows
//   o_d = sum_j e^{s_j - m} vs[j / block] vc[j, d] / sum_j e^{s_j - m}
// One pass over the cache with a running maximum and sum (online softmax).
// A row that sees no key gets zeros.
#include "device.hpp"

namespace agpu {
namespace k {
using namespace dev;

namespace {

struct D8Args {
  DecodeInt8 a;
  int lg_block;
};

// One block of 4 waves per query row: D/16 lanes own one key, 16 codes each
// (one 16-byte load).
template <typename T, int D>
__global__ void __launch_bounds__(256) decode_int8_row(D8Args g) {
  constexpr int LPK = D / 16, KPS = 64 / LPK;
  const DecodeInt8& a = g.a;
  __shared__ float sm_acc[4][D], sm_m[4], sm_l[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, grp = lane / LPK, sub = lane % LPK;
  const int64_t row = blockIdx.x, i = row % a.Tq, bh = row / a.Tq, hq = bh % (a.H * a.G), b = bh / (a.H * a.G);
  const int64_t h = hq / a.G;
  int64_t len = a.lens[b];
  len = len < 0 ? 0 : len > a.Tmax ? a.Tmax : len;
  const int64_t vis = len - a.Tq + i + 1;
  const T* q = (const T*)a.q + b * a.q_sb + hq * a.q_sh + i * a.q_st + sub * 16;
  float qf[16], acc[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) { qf[e] = to_f(q[e]) * a.scale * 1.4426950408889634f; acc[e] = 0.f; }
  const int8_t* K = a.k.codes + b * a.k.cs[0] + h * a.k.cs[1] + sub * 16;
  const int8_t* V = a.v.codes + b * a.v.cs[0] + h * a.v.cs[1] + sub * 16;
  const float* ks = a.k.scales + b * a.k.ss[0] + h * a.k.ss[1];
  const float* vs = a.v.scales + b * a.v.ss[0] + h * a.v.ss[1];
  float m = -INFINITY, l = 0.f;
  for (int64_t j = w * KPS + grp; j < vis; j += 4 * KPS) {
    const uint4 kr = *(const uint4*)(K + j * a.k.cs[2]), vr = *(const uint4*)(V + j * a.v.cs[2]);
    int8_t kc[16], vc[16];
    __builtin_memcpy(kc, &kr, 16);
    __builtin_memcpy(vc, &vr, 16);
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) d += qf[e] * (float)kc[e];
#pragma unroll
    for (int x = 1; x < LPK; x <<= 1) d += __shfl_xor(d, x, 64);
    d *= ks[(j >> g.lg_block) * a.k.ss[2]];
    const float M = fmaxf(m, d), f = m == -INFINITY ? 0.f : exp2f(m - M), pe = exp2f(d - M);
    const float pv = pe * vs[(j >> g.lg_block) * a.v.ss[2]];
    l = l * f + pe;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = acc[e] * f + pv * (float)vc[e];
    m = M;
  }
  auto merge = [](float& m1, float& l1, float m2, float l2, float& f1, float& f2) {
    // a NaN maximum wins, so that it reaches the output
    const float M = m1 != m1 ? m1 : m2 != m2 ? m2 : fmaxf(m1, m2);
    f1 = m1 == -INFINITY ? 0.f : exp2f(m1 - M);
    f2 = m2 == -INFINITY ? 0.f : exp2f(m2 - M);
    l1 = l1 * f1 + l2 * f2;
    m1 = M;
  };
#pragma unroll
  for (int x = LPK; x < 64; x <<= 1) {
    const float om = __shfl_xor(m, x, 64), ol = __shfl_xor(l, x, 64);
    float f1, f2;
    merge(m, l, om, ol, f1, f2);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float oa = __shfl_xor(acc[e], x, 64);
      acc[e] = acc[e] * f1 + oa * f2;
    }
  }
  if (grp == 0) {
#pragma unroll
    for (int e = 0; e < 16; ++e) sm_acc[w][sub * 16 + e] = acc[e];
    if (sub == 0) { sm_m[w] = m; sm_l[w] = l; }
  }
  __syncthreads();
  if (tid >= D) return;
  float M = sm_m[0], L = sm_l[0], A = sm_acc[0][tid];
  for (int x = 1; x < 4; ++x) {
    float f1, f2;
    merge(M, L, sm_m[x], sm_l[x], f1, f2);
    A = A * f1 + sm_acc[x][tid] * f2;
  }
  T* o = (T*)a.o + b * a.o_sb + hq * a.o_sh + i * a.o_st;
  o[tid] = from_f<T>(vis > 0 ? A / L : 0.f);
}

}  // namespace

size_t decode_int8_ws_bytes(const DecodeInt8&) { return 0; }

void decode_attention_int8(const DecodeInt8& a, void* ws, hipStream_t s) {
  (void)ws;
  if (!kv_int8_supported(a.D, a.block))
    fail("decode_attention_int8: head dim %lld or block %d not supported", (long long)a.D, a.block);
  const int64_t rows = a.B * a.H * a.G * a.Tq;
  if (rows == 0) return;
  if (rows > 0x7fffffffLL) fail("decode_attention_int8: too many rows");
  D8Args g;
  g.a = a;
  g.lg_block = a.block == 16 ? 4 : a.block == 32 ? 5 : a.block == 64 ? 6 : 7;
  AGPU_FLOAT_SWITCH(a.dt, {
    if (a.D == 32) hipLaunchKernelGGL((decode_int8_row<T, 32>), dim3((unsigned)rows), dim3(256), 0, s, g);
    else if (a.D == 64) hipLaunchKernelGGL((decode_int8_row<T, 64>), dim3((unsigned)rows), dim3(256), 0, s, g);
    else hipLaunchKernelGGL((decode_int8_row<T, 128>), dim3((unsigned)rows), dim3(256), 0, s, g);
  });
  check_launch("decode_attention_int8");
}

}  // namespace k
}  // namespace agpu
