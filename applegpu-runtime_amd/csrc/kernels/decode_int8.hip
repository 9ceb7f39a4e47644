// Attention over a K/V cache held in 8 bits (codes int8, one fp32 scale per
// block of rows and head):
//   s_j = scale ks[j / block] sum_d q_d kc[j, d],   j < visible rows
//   o_d = sum_j e^{s_j - m} vs[j / block] vc[j, d] / sum_j e^{s_j - m}
// One pass over the cache with a running maximum and sum; a row that sees no
// key gets zeros.
//
// Everything GEMM-shaped is on v_mfma_f32_16x16x32_f16 with 16 query rows
// (the query heads of one cache head, and their Tq rows) as columns, so that
// a read of the cache serves them all; with one query row the 15 idle columns
// cost nothing that the loads do not hide.
//  - Scores: S^T = K Q^T.  Lane l owns key l % 16 of a 16-key tile and reads
//    its codes 16 bytes at a time (a wave instruction is 1 KB in a row); the
//    order of d inside the product is free as long as Q has the same.
//  - Codes become f16 without a conversion: byte u = code + 128 under the
//    byte 0x64 is 1024 + u.  For K the 1152 too many are taken off through
//    the accumulator's initial value, -1152 sum_d q_d (fp32 queries: off the
//    f16 itself, since scores must be good to fp32); for V always off the
//    f16, because there the sum over a long context would lose the difference.
//  - Queries are scaled by a power of two per row so that the largest is in
//    [128, 256): any type then fits f16, bf16 exactly; fp32 as hi + lo (2^-22).
//  - Weights: the accumulators of S^T hold, for a query (lane l % 16), keys
//    4 (l / 16) .. + 3 of each tile, which is the layout of the B operand of
//    O^T = V^T P^T for 32 keys: they are exponentiated, scaled by the block's
//    vs and packed in place, with no exchange between lanes.  V^T's operand
//    is read 4 bytes of 8 keys a lane (D = 64) and its bytes interleaved by
//    v_perm, which the conversion needs anyway.
//  - Weights are rounded to f16 (2^-11 relative, against 2^-8 .. 2^-11 of the
//    output's own rounding), hi + lo for fp32 outputs.  The sum of weights and
//    that of weights times vs have a reference each, a power of two that moves
//    only when the query's own weight, or its weight times vs, exceeds it by
//    2^8: the exchange between lanes that this needs is rare, both stay within
//    2^15 of the reference, a weight times vs is in f16's normal range down to
//    2^-21 of the largest, and blocks that a query does not see or gives no
//    weight move nothing of it, whatever their scales.
// Work: waves of a block take 32-key steps in turn; a context is split over
// blocks while these leave CUs idle, and the splits' (O, m, l) are merged.
// Bound by the read of the codes where contexts are long: 4 x 8 heads of 4
// queries over up to 32768 rows of 128, 218 MB in 45.7 us (4.8 TB/s) and 5 for
// the merge; 16 x 20 heads over 8192 rows of 64 70 us, against 131 for a 16-bit
// cache.  Short contexts are bound by one chain of loads, products and
// exponentials: 12 heads over 100 rows 5 us.
#include "kv_int8.hpp"

namespace agpu {
namespace k {
using namespace dev;

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 32;        // keys of a wave's step
constexpr int kFew = 4;  // waves of a block of a split context
// A block keeps its waves' sums in LDS.
size_t lds_bytes(const DecodeInt8& a, int waves) {
  const int64_t R = a.G * a.Tq;
  return (size_t)(R < 16 ? R : 16) * (a.D + 4) * sizeof(float) * waves;
}
constexpr int kSplits = 1024;    // most parts of a context
constexpr float kLift = 7.f;     // log2 of the weight at the reference maximum
constexpr float kSlack = 8.f;    // log2 by which a weight may exceed that
constexpr int kFar = 1000;       // log2 of what is nothing beside anything in fp32

struct D8Args {
  DecodeInt8 a;
  int lg_block, splits, q_tiles;
  int nw;         // waves of a block: 4, 8 or 16
  int64_t chunk;  // keys of a split
  float* part;     // [units][splits][16 (D + 2)]: O, m, l of each query column
};

// 1024 + (code + 128) of the codes in bytes SEL of w ^ 0x80808080, as f16.
__device__ __forceinline__ uint32_t lift(uint32_t u, uint32_t sel) { return __builtin_amdgcn_perm(0x64646464u, u, sel); }
__device__ __forceinline__ uint32_t drop(uint32_t h) {
  const h2 c = {(_Float16)-1152.f, (_Float16)-1152.f};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, h) + c);
}

// 8 codes in two words as an MFMA operand; EXACT: codes, else codes + 1152.
template <bool EXACT>
__device__ __forceinline__ h8 codes8(uint32_t w0, uint32_t w1) {
  w0 ^= 0x80808080u;
  w1 ^= 0x80808080u;
  uint32_t r[4] = {lift(w0, 0x04010400u), lift(w0, 0x04030402u), lift(w1, 0x04010400u), lift(w1, 0x04030402u)};
  if constexpr (EXACT) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = drop(r[i]);
  }
  h8 o;
  __builtin_memcpy(&o, r, 16);
  return o;
}

// A whole number of any size as a power of two for ldexp.
__device__ __forceinline__ int power(float x) { return (int)fminf(fmaxf(x, (float)-kFar), (float)kFar); }
// 2^(m - M) of two such, 0 for no weight.
__device__ __forceinline__ float weight(float m, float M) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M); }
// x = [1/2, 1) 2^exponent(x).
__device__ __forceinline__ int exponent(float x) { return x != 0.f ? __builtin_amdgcn_frexp_expf(x) : -kFar; }

// 8 consecutive query values, raw.
template <typename T>
struct Raw8q {
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

// A wave's codes of one 32-key step.
template <int D>
struct Step {
  static constexpr int KW = D / 16;   // words of a K row that a lane holds (two tiles of them)
  uint32_t k[2][KW];
  static constexpr int VB = D / 16;   // bytes of a V row that a lane holds (8 keys of them)
  uint32_t v[8][VB < 4 ? 1 : VB / 4];
  float ks[2], vs[2];
};

// NEW: the step's own row is appended too.  The block of waves whose part of
// the context holds it leaves its cache block to the end: two waves append to
// K and V there (as kv_write_int8 does), before anything else, while the others
// are at the rows before it, and after a barrier the block's rows are read
// from the cache like any (8 x 20 heads over 640 rows of 64: 7.5 us without,
// 9.9 so, 11.4 with a launch of its own for the append).
template <typename T, int D, int NW, bool NEW>
__global__ void __launch_bounds__(64 * NW) decode_int8_mfma(D8Args g) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int NK = D / 32;     // MFMAs of a score tile
  constexpr int ND = D / 16;     // tiles of the output's D
  constexpr int LD = D + 4;      // padding of a query's row in LDS
  constexpr int64_t kIter = NW * kStep;
  extern __shared__ float sm_o[];  // [NW][rows of the tile][LD]
  __shared__ float sm_m[NW][16], sm_l[NW][16], sm_new[2];
  const DecodeInt8& a = g.a;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q4 = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t unit = blockIdx.x / (uint32_t)g.splits, split = blockIdx.x % (uint32_t)g.splits;
  const uint32_t bh = unit / (uint32_t)g.q_tiles, qt = unit % (uint32_t)g.q_tiles;
  const uint32_t b = bh / (uint32_t)a.H, h = bh % (uint32_t)a.H;
  const int R = (int)(a.G * a.Tq);
  const int64_t j_lo = (int64_t)split * g.chunk;
  const int8_t* K = a.k.codes + b * a.k.cs[0] + h * a.k.cs[1];
  const int8_t* V = a.v.codes + b * a.v.cs[0] + h * a.v.cs[1];
  const float* KS = a.k.scales + b * a.k.ss[0] + h * a.k.ss[1];
  const float* VS = a.v.scales + b * a.v.ss[0] + h * a.v.ss[1];
  // this lane's bytes of a row, and its rows of a step
  const uint32_t k_at = (D == 32 ? 8 : 16) * q4, v_at = (D / 16) * n;
  const uint32_t k_st = (uint32_t)a.k.cs[2], v_st = (uint32_t)a.v.cs[2];
  uint32_t k_off[2], v_off[8];
#pragma unroll
  for (int t = 0; t < 2; ++t) k_off[t] = (16 * t + n) * k_st + k_at;
#pragma unroll
  for (int e = 0; e < 8; ++e) v_off[e] = (16 * (e >> 2) + 4 * q4 + (e & 3)) * v_st + v_at;

  auto load = [&](Step<D>& s, int64_t j0) __attribute__((always_inline)) {
    const int8_t* kb = K + j0 * a.k.cs[2];
    const int8_t* vb = V + j0 * a.v.cs[2];
    // the last step of the cache reads its last row in place of those behind
    const bool inside = j0 + kStep <= a.Tmax;
    const uint32_t last = inside ? 0 : (uint32_t)(a.Tmax - 1 - j0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t off = k_off[t];
      if (!inside) {
        const uint32_t end = last * k_st + k_at;
        off = off < end ? off : end;
      }
      const int8_t* p = kb + off;
      if constexpr (D == 32) {
        const uint2 x = *(const uint2*)p;
        s.k[t][0] = x.x; s.k[t][1] = x.y;
      } else {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const uint4 x = *(const uint4*)(p + 64 * c);
          s.k[t][4 * c] = x.x; s.k[t][4 * c + 1] = x.y; s.k[t][4 * c + 2] = x.z; s.k[t][4 * c + 3] = x.w;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t off = v_off[e];
      if (!inside) {
        const uint32_t end = last * v_st + v_at;
        off = off < end ? off : end;
      }
      const int8_t* p = vb + off;
      if constexpr (D == 32) s.v[e][0] = *(const uint16_t*)p;
      else if constexpr (D == 64) s.v[e][0] = *(const uint32_t*)p;
      else {
        const uint2 x = *(const uint2*)p;
        s.v[e][0] = x.x; s.v[e][1] = x.y;
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t row = j0 + 16 * t, blk = (row < a.Tmax ? row : a.Tmax - 1) >> g.lg_block;
      s.ks[t] = KS[blk * a.k.ss[2]];
      s.vs[t] = VS[blk * a.v.ss[2]];
    }
  };

  // The loads that everything waits for go out first: the query row of this
  // lane, r = (query head of the group, token), and the first step's rows (any
  // row of the cache may be read before the length is known).
  const int Tq = (int)a.Tq, r0 = (int)qt * 16, r = r0 + n < R ? r0 + n : R - 1;
  const int g_q = Tq == 1 ? r : r / Tq, i_q = r - g_q * Tq;
  const T* q = (const T*)a.q + b * a.q_sb + (h * a.G + g_q) * a.q_sh + i_q * a.q_st;
  Raw8q<T> qr[NK];
#pragma unroll
  for (int t = 0; t < NK; ++t) qr[t].load(q + (D == 32 ? 8 * q4 : 64 * (t >> 1) + 16 * q4 + 8 * (t & 1)));
  Step<D> one, two;
  int64_t j0 = j_lo + w * kStep;
  const bool appends = NEW && w >= NW - 2;
  if (!appends && j0 < a.Tmax) load(one, j0);
  const int64_t asked = a.lens[b], len = asked < 0 ? 0 : asked > a.Tmax ? a.Tmax : asked;

  // the tile's rows r0 .. r1, and what they see
  const int r1 = r0 + 15 < R ? r0 + 15 : R - 1;
  const bool one_head = r0 / Tq == r1 / Tq;
  int64_t vis_lo = len - Tq + (one_head ? r0 % Tq : 0) + 1;
  const int64_t vis_hi = len - Tq + (one_head ? r1 % Tq : Tq - 1) + 1;
  int vis = r0 + n < R && len - Tq + i_q + 1 > 0 ? (int)(len - Tq + i_q + 1) : 0;  // (a length fits 32 bits)

  int64_t j_hi = j_lo + g.chunk < vis_hi ? j_lo + g.chunk : vis_hi;

  // the rows of the cache block that the step's row joins, if it is of this part
  int64_t tail = -1;
  if constexpr (NEW) {
    const int64_t at = asked - 1;  // (a length outside 1 .. Tmax names no row)
    if (at >= 0 && at < a.Tmax && at >= j_lo && at < j_lo + g.chunk) {
      tail = (at >> g.lg_block) << g.lg_block;
      j_hi = vis_lo = tail;
      vis = vis < tail ? vis : (int)tail;
    }
    if (appends) {
      if (tail >= 0) {
        const bool v = w == NW - 2;
        const Int8Cache& c = v ? a.v : a.k;
        const T* x = v ? (const T*)a.vn + b * a.vn_sb + h * a.vn_sh : (const T*)a.kn + b * a.kn_sb + h * a.kn_sh;
        const float s = kv8::append_rows<T, 1>(x, 0, c.codes + b * c.cs[0] + h * c.cs[1], c.cs[2],
                                               c.scales + b * c.ss[0] + h * c.ss[1] + (tail >> g.lg_block) * c.ss[2],
                                               tail, len - 1, len, D == 32 ? 2 : D == 64 ? 3 : 4, lane);
        if (lane == 0) sm_new[v] = s;
      }
      if (j0 < j_hi) load(one, j0);
    }
  }

  // queries as MFMA operands: lane (n, q4) holds d = 64 c + 16 q4 + 8 x + e of
  // row n (D = 32: d = 8 q4 + e), scaled to [128, 256) at the row's largest
  h8 qh[NK], ql[F32 ? NK : 1];
  float corr = 0.f, cq;
  {
    float x[NK][8];
    uint32_t top = 0;
#pragma unroll
    for (int t = 0; t < NK; ++t) {
      qr[t].floats(x[t]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t m = __float_as_uint(x[t][e]) & 0x7fffffffu;
        top = m > top ? m : top;
      }
    }
#pragma unroll
    for (int s = 16; s <= 32; s <<= 1) {
      const uint32_t o = (uint32_t)__shfl_xor((int)top, s, 64);
      top = o > top ? o : top;
    }
    // an infinity or NaN makes its row NaN
    int ex = (int)(top >> 23) - 127;
    ex = ex < -100 ? -100 : ex;
    const float up = top >= 0x7f800000u ? NAN : __uint_as_float((uint32_t)(7 - ex + 127) << 23);
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < NK; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = x[t][e] * up;
        qh[t][e] = (_Float16)y;
        if constexpr (F32) ql[t][e] = (_Float16)(y - (float)qh[t][e]);
        else sum += (float)qh[t][e];
      }
    if constexpr (!F32) {
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      corr = -1152.f * sum;
    }
    // log2 domain: score = cq ks acc
    cq = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(ex - 7 + 127) << 23);
  }

  f4 acc[ND];
#pragma unroll
  for (int c = 0; c < ND; ++c) acc[c] = f4{0.f, 0.f, 0.f, 0.f};
  // Of this lane's query, in whole powers of two: m, what its weights in l are
  // relative to, and m - d, what its weights times vs in acc are relative to.
  float m = -INFINITY, l = 0.f;
  int d = kFar;

  auto attend = [&](const Step<D>& cur, int64_t j0) __attribute__((always_inline)) {
    // (a tile that no query sees may be of a block that holds nothing yet)
    float ks[2], vs[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool seen = j0 + 16 * t < j_hi;
      ks[t] = seen ? cur.ks[t] : 0.f;
      vs[t] = seen ? cur.vs[t] : 0.f;
    }
    // scores of keys 16 t + 4 q4 + i for query n
    float s[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f4 x = f4{corr, corr, corr, corr};
#pragma unroll
      for (int c = 0; c < NK; ++c) {
        const h8 kf = codes8<F32>(cur.k[t][2 * c], cur.k[t][2 * c + 1]);
        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[c], x, 0, 0, 0);
        if constexpr (F32) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[c], x, 0, 0, 0);
      }
      // (a scale that is not finite as NaN: a sum of codes of 0 is not always 0
      // with -1152 sum q in it)
      const float f = cq * fmaf(ks[t], 0.f, ks[t]);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * t + i] = x[i] * f;
    }
    if (j0 + kStep > vis_lo) {
      const int left = vis - (int)j0;  // this query's keys from the step's first on
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (16 * (e >> 2) + 4 * q4 + (e & 3) >= left) s[e] = -INFINITY;
    }
    const float t0 = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), t1 = fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7]));
    float top = fmaxf(t0, t1), top_v = fmaxf(t0 + (float)exponent(vs[0]), t1 + (float)exponent(vs[1]));
    if (__any(top > m + kSlack || top_v > m + (kSlack - (float)d))) {
#pragma unroll
      for (int x = 16; x <= 32; x <<= 1) {
        top = fmaxf(top, __shfl_xor(top, x, 64));
        top_v = fmaxf(top_v, __shfl_xor(top_v, x, 64));
      }
      const float mv = m - (float)d;
      const float M = top > m + kSlack ? ceilf(top) : m, Mv = top_v > mv + kSlack ? ceilf(top_v) : mv;
      l = ldexpf(l, power(m - M));
      const float f = ldexpf(1.f, power(mv - Mv));
#pragma unroll
      for (int c = 0; c < ND; ++c) acc[c] *= f;
      m = M;
      d = power(M - Mv);
    }
    const float ref = m == -INFINITY ? 0.f : m - kLift;
    float p[8];
    // (a weight that a factor past 2^126 would save is 0 in fp32)
    float vn[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) vn[t] = __builtin_amdgcn_fmed3f(ldexpf(vs[t], d), -0x1p126f, 0x1p126f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = __builtin_amdgcn_exp2f(s[e] - ref);
      l += p[e];
      p[e] *= vn[e >> 2];
    }
    if (!(fabsf(vs[0]) < INFINITY && fabsf(vs[1]) < INFINITY)) {
      // a hidden key adds nothing, whatever its block's scale is
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = s[e] == -INFINITY ? 0.f : fabsf(vs[e >> 2]) < INFINITY ? p[e] : NAN;
    }
    h8 ph, pl;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ph[e] = (_Float16)p[e];
      if constexpr (F32) pl[e] = (_Float16)(p[e] - (float)ph[e]);
    }
    // V^T operands: byte c of the 8 keys' words, pairs of keys together
#pragma unroll
    for (int wd = 0; wd < (D < 64 ? 1 : D / 64); ++wd) {
      uint32_t f[4][4];
#pragma unroll
      for (int pr = 0; pr < 4; ++pr) {
        const uint32_t x = cur.v[2 * pr][wd] ^ 0x80808080u, y = cur.v[2 * pr + 1][wd] ^ 0x80808080u;
        const uint32_t a01 = __builtin_amdgcn_perm(y, x, 0x05010400u);  // x0 y0 x1 y1
        f[0][pr] = drop(lift(a01, 0x04010400u));
        f[1][pr] = drop(lift(a01, 0x04030402u));
        if constexpr (D >= 64) {
          const uint32_t a23 = __builtin_amdgcn_perm(y, x, 0x07030602u);
          f[2][pr] = drop(lift(a23, 0x04010400u));
          f[3][pr] = drop(lift(a23, 0x04030402u));
        }
      }
#pragma unroll
      for (int c = 0; c < (D < 64 ? 2 : 4); ++c) {
        h8 vf;
        __builtin_memcpy(&vf, f[c], 16);
        f4& o = acc[4 * wd + c];
        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, o, 0, 0, 0);
        if constexpr (F32) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, o, 0, 0, 0);
      }
    }
  };

  while (j0 < j_hi) {
    if (j0 + kIter < j_hi) load(two, j0 + kIter);
    attend(one, j0);
    j0 += kIter;
    if (j0 >= j_hi) break;
    if (j0 + kIter < j_hi) load(one, j0 + kIter);
    attend(two, j0);
    j0 += kIter;
  }

  if constexpr (NEW) {
    if (tail >= 0) {
      __threadfence_block();  // what the two waves stored, for the others
      __syncthreads();
      j_hi = len;
      vis = r0 + n < R ? (int)len : 0;
      for (j0 = tail + w * kStep; j0 < j_hi; j0 += kIter) {
        load(one, j0);
#pragma unroll
        for (int t = 0; t < 2; ++t) {  // (the scales may be in the scalar cache as they were)
          one.ks[t] = sm_new[0];
          one.vs[t] = sm_new[1];
        }
        attend(one, j0);
      }
    }
  }

  // the waves' states meet in LDS; lane (n, q4) holds d = (D/4) q4 + (D/16) i + c
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  // (each as its own weighted mean, which no sum of large values overflows)
  const int rows = r1 - r0 + 1;
  if (n < rows) {
    float* o = sm_o + (w * rows + n) * LD + (D / 4) * q4;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < ND; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[(D / 16) * i + c] = ldexpf(acc[c][i] * inv, -d);
    if (q4 == 0) { sm_m[w][n] = m; sm_l[w][n] = l; }
  }
  __syncthreads();
  for (int idx = tid; idx < rows * D; idx += 64 * NW) {
    const int qr = idx / D, d = idx % D, rr = r0 + qr, iq = rr % Tq;
    float M = sm_m[0][qr];
#pragma unroll
    for (int x = 1; x < NW; ++x) M = fmaxf(M, sm_m[x][qr]);
    float L = 0.f, A = 0.f, f[NW];
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      f[x] = sm_l[x][qr] * weight(sm_m[x][qr], M);
      L += f[x];
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int x = 0; x < NW; ++x) A += sm_o[(x * rows + qr) * LD + d] * (f[x] * inv);
    if (g.splits == 1) {
      T* o = (T*)a.o + b * a.o_sb + (h * a.G + rr / Tq) * a.o_sh + iq * a.o_st;
      o[d] = from_f<T>(len - Tq + iq + 1 > 0 ? A : 0.f);
    } else {
      float* P = g.part + ((int64_t)blockIdx.x * 16 + qr) * (D + 2);
      P[d] = A;
      if (d == 0) { P[D] = M; P[D + 1] = L; }
    }
  }
}

// One block per query row: merges its splits, parts of them by threads of
// their own.
template <typename T, int D>
__global__ void __launch_bounds__(256) decode_int8_merge(D8Args g) {
  constexpr int NP = 256 / D;  // parts
  __shared__ float f_of[kSplits], sum[NP][D], red[4], red_l[4];
  const DecodeInt8& a = g.a;
  const int tid = threadIdx.x, d = tid % D, part = tid / D, Tq = (int)a.Tq, R = (int)(a.G * a.Tq);
  const int64_t row = blockIdx.x, bh = row / R, h = bh % a.H, b = bh / a.H;
  const int rr = (int)(row % R), iq = rr % Tq;
  const float* P = g.part + ((bh * g.q_tiles + rr / 16) * g.splits * 16 + rr % 16) * (D + 2);
  constexpr int64_t st = 16 * (D + 2);
  constexpr int MS = kSplits / 256;
  float m[MS], l[MS], M = -INFINITY, L = 0.f;
#pragma unroll
  for (int i = 0; i < MS; ++i) {
    const int s = tid + 256 * i;
    m[i] = s < g.splits ? P[s * st + D] : -INFINITY;
    l[i] = s < g.splits ? P[s * st + D + 1] : 0.f;
    M = fmaxf(M, m[i]);
  }
  M = wave_max(M);
  if ((tid & 63) == 0) red[tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
#pragma unroll
  for (int i = 0; i < MS; ++i) {
    const float f = l[i] * weight(m[i], M);
    if (tid + 256 * i < g.splits) f_of[tid + 256 * i] = f;
    L += f;
  }
  L = wave_sum(L);
  if ((tid & 63) == 0) red_l[tid >> 6] = L;
  __syncthreads();
  L = (red_l[0] + red_l[1]) + (red_l[2] + red_l[3]);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  float A = 0.f;
#pragma unroll 4
  for (int s = part; s < g.splits; s += NP) A += P[s * st + d] * (f_of[s] * inv);
  sum[part][d] = A;
  __syncthreads();
  if (part) return;
#pragma unroll
  for (int i = 1; i < NP; ++i) A += sum[i][d];
  int64_t len = a.lens[b];
  len = len < 0 ? 0 : len > a.Tmax ? a.Tmax : len;
  T* o = (T*)a.o + b * a.o_sb + (h * a.G + rr / Tq) * a.o_sh + iq * a.o_st;
  o[d] = from_f<T>(len - Tq + iq + 1 > 0 ? A : 0.f);
}

D8Args plan(const DecodeInt8& a) {
  D8Args g;
  g.a = a;
  g.lg_block = a.block == 16 ? 4 : a.block == 32 ? 5 : a.block == 64 ? 6 : 7;
  g.q_tiles = (int)((a.G * a.Tq + 15) / 16);
  // A context to a block, with the waves that fill the CUs; or split over blocks
  // of 4 waves and merged by a second launch, which costs about as much as three
  // steps of a wave, where that saves more steps than that.  16 waves to a block
  // where few contexts are long, 8 where they are short or many, or where 16
  // would spill more than a few registers (D = 64 in fp32, or with an append:
  // 160 heads, 4096 rows 32 us).  f16, D = 64, us:
  //   heads, rows     16 waves   8 waves   split
  //   12, 600             8.6       7.2      8.5
  //   12, 1536           11.5      10.9      9.0
  //   64, 1536           11.4      11.1     11.2
  //   160, 640            9.2       7.6     12.4
  //   160, 2048          14.4      14.3     18.0
  //   160, 8192          33.7      39.8     37.4
  // (Merged by a unit's last block in the same launch: 20 heads, 8192 rows of 64
  // 14.5 us against 13.4; 32 heads of 4 queries, 32768 rows of 128 60 against
  // 55: the blocks' wait for their stores and the count cost more than the
  // launch.)
  const int64_t units = a.B * a.H * g.q_tiles;
  const bool few = units <= 256 && a.D != 128, brief = few && a.Tmax <= 2048;
  const bool fits = a.D == 32 || (a.dt != DType::F32 && !a.kn);
  g.nw = few && !brief && fits ? 16 : units <= 512 ? 8 : 4;
  while (g.nw > kFew && (lds_bytes(a, g.nw) > (60 << 10) || a.Tmax <= g.nw / 2 * kStep)) g.nw /= 2;
  const int64_t iters = (a.Tmax + g.nw * kStep - 1) / (g.nw * kStep);
  // steps of a wave for the merge, and for a row of a unit with all CUs filled
  const double merge = brief ? 3.7 : 3.0, per = (brief ? 2.3 : a.D == 128 ? 2.0 : 1.0) / 1e5;
  g.splits = 1;
  g.chunk = a.Tmax;
  g.part = nullptr;
  if (units > 0 && units < kSplits && (double)iters > merge + per * (double)a.Tmax * (double)units) {
    g.nw = kFew;
    const int64_t iter = kFew * kStep, most = (a.Tmax + iter - 1) / iter;
    int64_t want = (kSplits + units - 1) / units;  // four blocks a CU
    if (want > most) want = most;
    g.chunk = ((a.Tmax + want - 1) / want + iter - 1) / iter * iter;
    g.splits = (int)((a.Tmax + g.chunk - 1) / g.chunk);
  }
  return g;
}

template <typename T, int D, int NW>
void launch_nw(const D8Args& g, hipStream_t s) {
  constexpr bool kAppends = NW < 16 || D == 32;
  const dim3 grid((unsigned)(g.a.B * g.a.H * g.q_tiles * g.splits));
  if (!g.a.kn) hipLaunchKernelGGL((decode_int8_mfma<T, D, NW, false>), grid, dim3(64 * NW), lds_bytes(g.a, NW), s, g);
  else if constexpr (kAppends)
    hipLaunchKernelGGL((decode_int8_mfma<T, D, NW, true>), grid, dim3(64 * NW), lds_bytes(g.a, NW), s, g);
  else fail("decode_attention_int8: no append in blocks of %d waves", NW);
}

template <typename T, int D>
void launch(const D8Args& g, hipStream_t s) {
  constexpr bool kWide = D == 32 || (D == 64 && sizeof(T) == 2);
  if (g.nw == kFew) launch_nw<T, D, kFew>(g, s);
  else if (g.nw == 8) launch_nw<T, D, 8>(g, s);
  else if constexpr (kWide) launch_nw<T, D, 16>(g, s);
  else fail("decode_attention_int8: no blocks of %d waves", g.nw);
  if (g.splits > 1)
    hipLaunchKernelGGL((decode_int8_merge<T, D>), dim3((unsigned)(g.a.B * g.a.H * g.a.G * g.a.Tq)), dim3(256), 0, s, g);
}

}  // namespace

bool decode_int8_appends(const DecodeInt8& a) { return a.Tq == 1 && a.G <= 16; }

size_t decode_int8_ws_bytes(const DecodeInt8& a) {
  const D8Args g = plan(a);
  if (g.splits <= 1) return 0;
  return (size_t)(a.B * a.H * g.q_tiles) * g.splits * 16 * (a.D + 2) * sizeof(float);
}

void decode_attention_int8(const DecodeInt8& a, void* ws, hipStream_t s) {
  if (!kv_int8_supported(a.D, a.block))
    fail("decode_attention_int8: head dim %lld or block %d not supported", (long long)a.D, a.block);
  if (a.B * a.H * a.G * a.Tq == 0) return;
  D8Args g = plan(a);
  if (a.G * a.Tq > 0x7fffffffLL / 2 || a.B * a.H * a.G * a.Tq > 0x7fffffffLL || a.B * a.H * g.q_tiles * g.splits > 0x7fffffffLL)
    fail("decode_attention_int8: too many query rows");
  if (a.kn && (!a.vn || !decode_int8_appends(a))) fail("decode_attention_int8: cannot append in this launch");
  if (g.splits > 1 && !ws) fail("decode_attention_int8: workspace missing");
  g.part = (float*)ws;
  AGPU_FLOAT_SWITCH(a.dt, {
    if (a.D == 32) launch<T, 32>(g, s);
    else if (a.D == 64) launch<T, 64>(g, s);
    else launch<T, 128>(g, s);
  });
  check_launch("decode_attention_int8");
}

}  // namespace k
}  // namespace agpu
