// Linear layers with weights in 4 bits over many 16-bit rows: y = act(x W^T +
// bias) + residual, the codes in linear_int4.hip's tiles.
//
// One block of 4 wavefronts owns BM = 32 TM rows x 128 columns over the whole
// K, in stages of 64 k, a wavefront all the rows x 32 columns:
//  - x goes global -> LDS by 16-byte copies without registers, a row's 16-byte
//    chunks exchanged so that a fragment read covers all banks (8 rows x 128
//    bytes a copy instruction).
//  - The codes go the same way, a wavefront's own 1 KB a stage: 16 bytes, one
//    row's 32 codes of one scale, to the lane that multiplies them.  They
//    become values of x's type in registers, code * scale rounded once (half a
//    step of the type, what weights held in it would have lost, and far below
//    the codes' own rounding; unrounded they would take two products each) as
//    dequantize_int4 rounds it, while the MFMAs before run: no value of W
//    passes LDS or memory, and each is made once a block.
//  - A ring of S stages: a wavefront waits for its copies of the next stage
//    alone, by their number.
//  - Lane l of the 32x32x16 product's W side holds row l % 32 and 8 of the 32
//    codes that begin at column 32 (l / 32); x is read in the same order of k.
//  - The epilogue goes through LDS, 16 bytes a lane, in loops that stay rolled
//    and for one activation: its instructions come from memory once a launch
//    and compute unit.  (Unrolled, with all activations: 37 us at 1111 x 1280 x
//    3840.)
//
// f16, 1111 x 1280 x 3840, group 128: 22.9 us (477 TFLOP/s), against 33 for
// values written out and multiplied and 21.5 for a library's product of values.
// One block on a compute unit takes 0.5 (TM = 2) to 0.8 us (TM = 5) a stage, of
// which its MFMAs are 0.1 to 0.3: four wavefronts that wait for LDS reads and
// make 2 x 16 values of W a lane (in f16 four instructions a pair, in bf16
// seven) do not fill it, two or three blocks do.  (Eight, half of them for
// half of each stage's k: 85 us for 95 at 300 x 8192 x 8192, but 25.2 for 24.2
// here and 74 for 62 at 4096 rows.)
#include "gemm_kernels.hpp"

namespace agpu {
namespace k {
using namespace dev;

namespace {

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr int kPastEnd = 0x7ffffff0;  // past the end of every resource: zeros

__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)(bytes < kPastEnd ? bytes : kPastEnd),
                                           0x00020000);
}
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t src, void* l, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (lds_ptr)l, 16, voff, soff, 0, 0);
}

// 16 + (code + 8) of nibbles I and I + 4 of a word, in the type's mantissa
template <typename T> struct Codes;
template <> struct Codes<half_t> {
  typedef f16x8 vec;
  template <int I> static __device__ __forceinline__ uint32_t pair(uint32_t w, float, h2 s) {
    const uint32_t v = I == 0 ? w << 6 : I == 1 ? w << 2 : w >> (4 * I - 6);
    const uint32_t u = (v & 0x03c003c0u) | 0x4c004c00u;
    h2 h;
    __builtin_memcpy(&h, &u, 4);
    h = (h - (h2){(_Float16)24.f, (_Float16)24.f}) * s;  // the difference is exact
    uint32_t r;
    __builtin_memcpy(&r, &h, 4);
    return r;
  }
  static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct Codes<bf16_t> {
  typedef bf16x8 vec;
  template <int I> static __device__ __forceinline__ uint32_t pair(uint32_t w, float s, h2) {
    const uint32_t v = I == 0 ? w << 3 : w >> (4 * I - 3);
    const uint32_t u = (v & 0x00780078u) | 0x41804180u;
    // both products are exact in fp32 (5 and 8 bits), and so is their sum
    const float lo = fmaf(__uint_as_float(u << 16), s, -24.f * s);
    const float hi = fmaf(__uint_as_float(u & 0xffff0000u), s, -24.f * s);
    const __bf16 o[2] = {(__bf16)lo, (__bf16)hi};
    uint32_t r;
    __builtin_memcpy(&r, o, 4);
    return r;
  }
  static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

struct L4RArgs {
  GArgs p;  // A = x, bias, res, C, act; tiles_m, tiles_n
  const uint8_t* packed;
  const void* scales;
  int steps, groups, group_log2;
};

template <int ACT>
__device__ __forceinline__ float act_of(float v) {
  if constexpr (ACT == kActRelu) return fmaxf(v, 0.f);  // (0 for NaN, as relu gives elsewhere)
  else if constexpr (ACT == kActGelu) return gelu_tanh(v);
  else if constexpr (ACT == kActGeluExact) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
  else return v;
}

// A barrier of the block that waits for nothing else (a fence would wait for
// every copy under way); what has to be there was waited for before it.
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T, int TM, int S, int ACT>
__global__ void __launch_bounds__(256) linear_int4_rows(L4RArgs g) {
  constexpr int BM = 32 * TM, BN = 128, BK = 64;
  constexpr int AE = BM * BK, CE = AE + 4 * 512, STAGE = CE + 4 * 128;  // elements: x, codes, scales of a stage
  typedef typename Codes<T>::vec V8;
  const GArgs& p = g.p;
  // (an array for each place of the ring: a read then waits for the copies into
  // its own place alone)
  __shared__ __attribute__((aligned(16))) T ring0[STAGE], ring1[STAGE], ring2[S > 2 ? STAGE : 8], ring3[S > 3 ? STAGE : 8];
  auto place = [&](int u) __attribute__((always_inline)) { return u == 0 ? ring0 : u == 1 ? ring1 : u == 2 ? ring2 : ring3; };
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l31 = lane & 31, hi = lane >> 5;
  int tmi, tni;
  tile_coords(p, tmi, tni);
  const int64_t m0 = (int64_t)tmi * BM, n0 = (int64_t)tni * BN;
  const int K = (int)p.K, nk = (K + BK - 1) / BK;
  auto swz = [](int r) { return (r / 2) & 7; };  // chunk c of row r sits at chunk c ^ swz(r)

  const __amdgpu_buffer_rsrc_t sa =
      resource((const T*)p.A + m0 * p.a_sm, ((p.M - m0 - 1) * p.a_sm + p.K) * (int64_t)sizeof(T));
  const int lr = lane / 8;
  int off[TM];
#pragma unroll
  for (int q = 0; q < TM; ++q) {
    const int r = (w * TM + q) * 8 + lr;
    off[q] = (int)((r * p.a_sm + ((lane % 8) ^ swz(r)) * 8) * (int64_t)sizeof(T));
  }
  // the lane's run of codes: tiles of 16 rows, [K / 128][4][16 rows][16 bytes]
  const int64_t tiles = (p.N + 15) / 16, tile = n0 / 16 + 2 * w + l31 / 16;
  const __amdgpu_buffer_rsrc_t sw = resource(g.packed + n0 / 16 * g.steps * 1024, (tiles - n0 / 16) * g.steps * 1024);
  const int woff = (int)(((tile < tiles ? tile : tiles - 1) - n0 / 16) * g.steps * 1024) + (hi * 16 + (l31 & 15)) * 16;
  // the lane's scale is half of 4 aligned bytes
  const int odd = (int)((uintptr_t)g.scales & 2), N = (int)p.N;
  const __amdgpu_buffer_rsrc_t ss = resource((const char*)g.scales - odd, ((int64_t)g.groups * N * 2 + odd + 3) & ~3LL);
  const int n = (int)(n0 + 32 * w + l31 < p.N ? n0 + 32 * w + l31 : p.N - 1);
  auto scale_at = [&](int st) __attribute__((always_inline)) {
    const int gr = (st * BK + 32 * hi) >> g.group_log2;
    return ((gr < g.groups ? gr : g.groups - 1) * N + n) * 2 + odd;
  };

  // stage st (past the last: zeros) into place u of the ring: TM + 2 loads
  auto issue = [&](int u, int st) __attribute__((always_inline)) {
    T* d = place(u);
    const int k = st * (BK * (int)sizeof(T));
    const int left = (K - st * BK) / 8;  // chunks (K is a multiple of 8)
#pragma unroll
    for (int q = 0; q < TM; ++q) {
      const int r = (w * TM + q) * 8 + lr;
      copy16(sa, d + (w * TM + q) * 512, ((lane % 8) ^ swz(r)) < left ? off[q] + k : kPastEnd, 0);
    }
    copy16(sw, d + AE + w * 512, woff, st * 512);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(ss, (lds_ptr)(d + CE + w * 128), 4, scale_at(st) & ~3, 0, 0, 0);
  };

  V8 fa[2][TM], fb[2];
  auto read = [&](int set, int u, int kk) __attribute__((always_inline)) {
    const T* a = place(u);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int r = i * 32 + l31;
      fa[set][i] = *(const V8*)(a + r * BK + (((4 * hi + kk) ^ swz(r)) * 8));
    }
  };
  uint4 codes;
  float sf;
  auto read_codes = [&](int u, int st) __attribute__((always_inline)) {
    const T* d = place(u);
    codes = *(const uint4*)(d + AE + w * 512 + lane * 8);
    sf = to_f(d[CE + w * 128 + lane * 2 + ((scale_at(st) >> 1) & 1)]);
  };
  auto make = [&](int set, uint32_t v) __attribute__((always_inline)) {
    const h2 sh = {(_Float16)sf, (_Float16)sf};
    const uint32_t r[4] = {Codes<T>::template pair<0>(v, sf, sh), Codes<T>::template pair<1>(v, sf, sh),
                           Codes<T>::template pair<2>(v, sf, sh), Codes<T>::template pair<3>(v, sf, sh)};
    __builtin_memcpy(&fb[set], r, 16);
  };
  f32x16 acc[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
  auto mul = [&](int set) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[i] = Codes<T>::mfma(fb[set], fa[set][i], acc[i]);
  };

  // waits until no more than the youngest S - 2 stages are under way (in
  // order), and for this wavefront's LDS reads
  constexpr int kLeft = (S - 2) * (TM + 2), kStage = (kLeft & 15) | (kLeft >> 4) << 14 | 0x0070;
  static_assert(kLeft < 64, "the counter of loads");
#pragma unroll
  for (int u = 0; u + 1 < S; ++u) issue(u, u);
  __builtin_amdgcn_s_waitcnt(kStage);
  __syncthreads();
  read_codes(0, 0);
  read(0, 0, 0);
  make(0, codes.x);
  for (int s0 = 0; s0 < nk; s0 += S) {
#pragma unroll
    for (int u = 0; u < S; ++u) {
      const int st = s0 + u;
      if (st >= nk) break;
      issue((u + S - 1) % S, st + S - 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < 3; ++kk) {
        read((kk + 1) & 1, u, kk + 1);
        __builtin_amdgcn_sched_barrier(0);
        make((kk + 1) & 1, kk == 0 ? codes.y : kk == 1 ? codes.z : codes.w);
        mul(kk & 1);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x2, 24 / TM, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      // this wavefront holds the rest of stage st in registers, and its copies
      // of stage st + 1 have landed; after the barrier so for every wavefront
      __builtin_amdgcn_s_waitcnt(kStage);
      barrier();
      __builtin_amdgcn_sched_barrier(0);
      read_codes((u + 1) % S, st + 1);
      read(0, (u + 1) % S, 0);
      __builtin_amdgcn_sched_barrier(0);
      mul(1);
      make(0, codes.x);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070);  // the copies past the last stage too
  __syncthreads();

  // lane l, register e of a 32 x 32 tile: row l % 32, column 8 (e / 4) + 4 (l
  // / 32) + e % 4.  Through this wavefront's own part of LDS, 32 rows x 32
  // columns of fp32 at a time, so that bias, residual and output move as 16
  // bytes a lane.
  constexpr int CP = 36;
  static_assert(2 * 32 * CP * 4 <= STAGE * (int)sizeof(T), "epilogue staging");
  float* ct = (float*)(w < 2 ? ring0 : ring1) + w % 2 * 32 * CP;
  const T* bias = (const T*)p.bias;
  const T* R = (const T*)p.res;
  T* C = (T*)p.C;
  struct V { T e[8]; };
  const int64_t col = n0 + w * 32 + (lane % 4) * 8;
  const bool full = col + 8 <= p.N;
  // (without the empty asm the compiler gives both branches one access of 2
  // bytes and splits the 16 for it)
  auto load8 = [&](V& v, const T* from) __attribute__((always_inline)) {
    if (full) {
      __builtin_memcpy(&v, from, 16);
      asm volatile("" ::: "memory");
    } else {
      for (int e = 0; e < 8; ++e) v.e[e] = col + e < p.N ? from[e] : (T)0.f;
    }
  };
  float bs[8] = {};
  if (bias) {
    V b;
    load8(b, bias + col);
#pragma unroll
    for (int e = 0; e < 8; ++e) bs[e] = to_f(b.e[e]);
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int h = 0; h < 4; ++h)
      *(float4*)(ct + l31 * CP + 8 * h + 4 * hi) =
          make_float4(acc[i][4 * h], acc[i][4 * h + 1], acc[i][4 * h + 2], acc[i][4 * h + 3]);
    // (the wavefront's own writes and reads: in order, no barrier.  Rolled
    // loops: the instructions of unrolled ones come from memory once a launch
    // and compute unit)
#pragma unroll 1
    for (int it = 0; it < 2; ++it) {
      const int r = it * 16 + lane / 4;
      const int64_t row = m0 + i * 32 + r;
      float v[8];
      *(float4*)v = *(const float4*)(ct + r * CP + (lane % 4) * 8);
      *(float4*)(v + 4) = *(const float4*)(ct + r * CP + (lane % 4) * 8 + 4);
      if (row >= p.M) continue;
      T* out = C + row * p.c_sm + col;
      const T* res = R + row * p.r_sm + col;
      V x, o;
      if (R) {
        load8(x, res);
      } else {
        x = V{};
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) o.e[e] = from_f<T>(act_of<ACT>(v[e] + bs[e]) + to_f(x.e[e]));
      if (full) {
        __builtin_memcpy(out, &o, 16);
        asm volatile("" ::: "memory");
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < p.N) out[e] = o.e[e];
      }
    }
  }
}

template <typename T, int TM, int S>
void launch(L4RArgs& g, hipStream_t s) {
  g.p.tiles_m = (int)((g.p.M + 32 * TM - 1) / (32 * TM));
  g.p.tiles_n = (int)((g.p.N + 127) / 128);
  const dim3 grid((unsigned)(g.p.tiles_m * g.p.tiles_n));
#define AGPU_I4R(ACT) hipLaunchKernelGGL((linear_int4_rows<T, TM, S, ACT>), grid, dim3(256), 0, s, g)
  switch (g.p.act) {
    case kActNone: AGPU_I4R(kActNone); break;
    case kActRelu: AGPU_I4R(kActRelu); break;
    case kActGelu: AGPU_I4R(kActGelu); break;
    default: AGPU_I4R(kActGeluExact);
  }
#undef AGPU_I4R
}

template <typename T>
void launch_tm(L4RArgs& g, int tm, hipStream_t s) {
  if (tm == 2) launch<T, 2, 3>(g, s);
  else if (tm == 3) launch<T, 3, 3>(g, s);
  else if (tm == 4) launch<T, 4, 3>(g, s);
  else launch<T, 5, 2>(g, s);
}

int64_t row_tiles(int64_t M, int64_t N, int tm) { return (M + 32 * tm - 1) / (32 * tm) * ((N + 127) / 128); }

// A stage's time on the compute unit with the most blocks grows as blocks x (2
// TM + 3).  f16, us with TM = 2 / 3 / 4 / 5 (the rule's choice in brackets):
//   512 x 1280 x 3840    [14.6]  16.3   17.4   20.1
//   1111 x 1280 x 3840   27.0    24.1   25.8  [23.0]
//   2000 x 5120 x 1280   56.7   [51.6]  53.8   62.3
//   300 x 8192 x 8192    115    [93.8]  95.5   104   (bf16)
//   4096 x 1280 x 3840   71.9    65.1  [62.2]  64.8
int pick_tm(int64_t M, int64_t N, int cus, int64_t* cost) {
  int best = 0;
  for (int tm = 2; tm <= 5; ++tm) {
    const int64_t c = (row_tiles(M, N, tm) + cus - 1) / cus * (2 * tm + 3);
    if (best && c >= *cost) continue;
    best = tm;
    *cost = c;
  }
  return best;
}

}  // namespace

// The rows of a block lie within the 2 GiB that a buffer resource spans, and so
// do its codes and all scales (K after the rows are padded to whole vectors).
static bool rows_fit(const LinearInt4& a) {
  const int64_t K = (a.K + 7) / 8 * 8;
  return K < (1 << 21) && (K + a.group - 1) / a.group * a.N < (1 << 30) && row_tiles(a.M, a.N, 2) < (1LL << 31);
}

// Which kernels a product of these sizes takes, by what they measured (us):
// few rows straight from the codes (few), these tiles (rows), or the weights
// made values in memory for the framework's GEMM (values).
//   M x K x N              few    rows   values
//   128 x 1280 x 3840      10.7   13.1
//   192 x 1280 x 3840      18.3   13.4
//   256 x 1280 x 1280      9.7    13.0
//   320 x 1280 x 3840             14.0   27.5
//   32 x 768 x 50257       22.2   13.0
//   64 x 8192 x 8192       39.3   74.5          (bf16)
//   256 x 8192 x 8192      112    81.6          (bf16)
//   640 x 8192 x 1024             58.9   44.8
//   3000 x 8192 x 8192            409    430
//   16000 x 1280 x 5120           248    232
//   1500 x 8192 x 8192            243    237    (bf16)
//   4000 x 8192 x 8192            605    474    (bf16)
// The few-row kernel takes 4 us + K / 233 for each round of 256 blocks of 32
// (16: groups of 32) columns x 64 rows (K / 333 for 32 rows), the tiles 4 us +
// K (2.4 + cost) / 1430.  fp32 rows stay there however many they are: three
// products a code keep the 24 bits of x, where values in memory and the split
// fp32 GEMM (two bf16 parts an operand, infinities NaN) are 1.0 to 2.2 times as
// fast (1111 x 1280 x 3840 136 against 91 us, 4096 x 8192 x 8192 4.4 against
// 2.0 ms) and the native fp32 GEMM is slower (236 us, 4.5 ms).
Int4Way linear_int4_way(const LinearInt4& a, int cus) {
  if (a.M <= 16 || a.dt == DType::F32) return Int4Way::Few;
  const int64_t columns = a.group == 32 && a.M > 32 ? 16 : 32, rows = a.M > 32 ? 64 : 32;
  const int64_t blocks = (a.N + columns - 1) / columns * ((a.M + rows - 1) / rows);
  int64_t cost = 0;
  pick_tm(a.M, a.N, cus, &cost);
  if ((blocks + cus - 1) / cus * (a.M > 32 ? 43 : 30) <= 17 + 7 * cost) return Int4Way::Few;
  // (a GEMM splits a long K over the chip where there are few tiles, and has
  // larger tiles where there are many rows)
  const bool few_tiles = row_tiles(a.M, a.N, 2) < cus / 2 && a.K > 4096;
  if (few_tiles || a.M > (a.dt == DType::F16 ? 4096 : 2048) || !rows_fit(a)) return Int4Way::Values;
  return Int4Way::Rows;
}

void linear_int4_rows(const LinearInt4& a, int cus, hipStream_t s) {
  if (a.M == 0) return;
  if (a.dt == DType::F32 || a.ln_gamma || a.K % 8 || a.x_sm % 8 || ((uintptr_t)a.x & 15) || a.x_sm < a.K ||
      a.x_sm >= (1 << 21) || !rows_fit(a))
    fail("linear_int4: these rows do not fit the tiles");
  L4RArgs g{};
  g.p.A = a.x; g.p.a_sm = a.x_sm;
  g.p.M = a.M; g.p.N = a.N; g.p.K = a.K;
  g.p.bias = a.bias;
  g.p.res = a.residual; g.p.r_sm = a.N;
  g.p.C = a.out; g.p.c_sm = a.N;
  g.p.act = a.act;
  g.packed = a.packed;
  g.scales = a.scales;
  g.steps = (int)((a.K + 127) / 128);
  g.groups = (int)((a.K + a.group - 1) / a.group);
  g.group_log2 = a.group == 32 ? 5 : a.group == 64 ? 6 : 7;
  int64_t cost = 0;
  const int tm = pick_tm(a.M, a.N, cus, &cost);
  if (a.dt == DType::F16) launch_tm<half_t>(g, tm, s);
  else launch_tm<bf16_t>(g, tm, s);
  check_launch("linear_int4_rows");
}

}  // namespace k
}  // namespace agpu
