// Products of 16-bit operands for kernels with epilogues of their own:
// acc[m][n] = sum over k of A(m, k) B(n, k), fp32 accumulation on
// v_mfma_f32_32x32x16, with each operand in memory either as rows (k
// contiguous) or as columns (row k holds every m), and either as plain values
// or as two planes, the high and the low half of an fp32 value.
//
//  - A block owns a BM x BN tile in stages of 64 16-bit values per row of an
//    operand: 64 k of plain values, 32 k of both planes.  In memory the planes
//    alternate every 32 values, [.. / 32][high, low][32], so that a stage of a
//    row is one run of 128 bytes either way.
//  - Global -> LDS by buffer loads to LDS, 16 bytes a lane, two stages in LDS;
//    the fragments of the next step are read while the matrix instructions of
//    the current one run.
//  - Rows: 8 rows x 128 bytes a wave instruction, the row's 16-byte chunks
//    exchanged by chunk ^ (row / 2) % 8: the 16 lanes of a fragment read's
//    phase cover all 64 banks.  Columns: whole runs of a k row, its 64-byte
//    groups exchanged by k % 4; a fragment is two transposing reads
//    (ds_read_b64_tr_b16: 16 lanes give the addresses of 4 k x 16 m values,
//    each gets 4 k of its own m), whose 4 rows lie in different banks.
//  - Two planes: high * high + high * low + low * high, three matrix
//    instructions on what is in registers already, where the three products
//    one after another would read each plane twice.  With fp16 planes of
//    values scaled to at most 2^15 the halves hold 22 bits, and what is left
//    out (low * low) is below 2^-22 of a product.
#pragma once

#include "device.hpp"

namespace agpu {
namespace k {
namespace t16 {
using namespace dev;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_void;

template <typename T> struct Mfma;
template <> struct Mfma<half_t> {
  typedef _Float16 vec __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 run(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mfma<bf16_t> {
  typedef __bf16 vec __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 run(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// 16-bit values: rows (or, as columns, k rows) `ld` apart, 16-byte aligned, ld
// a multiple of 8 (two planes: of 64, zeros behind the values); matrices of a
// batch `batch` apart.
struct Operand {
  const void* p = nullptr;
  int64_t ld = 0, batch = 0;
};
struct Args {
  Operand a, b;
  int64_t M = 0, N = 0, K = 0;
  int tiles_m = 0, tiles_n = 0, tiles = 0;  // tiles: those that are computed
  int splits = 1, batches = 1;
  int stages = 0, per_split = 0;
  int group = 8;  // tile rows that share their columns' loads
};

// An offset behind the end of every resource: what is copied from there is
// zeros.
constexpr int kBehind = 0x7ffffff0;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* p, int64_t bytes) {
  bytes = bytes < 0 ? 0 : bytes < kBehind ? bytes : kBehind;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t src, void* l, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (lds_void)l, 16, voff, soff, 0, 0);
}

// One operand's part of a block: B rows (m) of it, L windows of 1 KB a
// wavefront and stage.
template <typename T, int B, int L, int PL, bool COLS>
struct Stream {
  static constexpr int KS = 64 / PL;       // k of a stage
  static constexpr int CPR = B * PL / 8;   // columns: 16-byte chunks of a k row
  const T* base;
  int64_t ld, k_rows, width;
  int off[L], first, lane;
  __amdgpu_buffer_rsrc_t rows;

  static __device__ __forceinline__ int swz(int r) {
    if (COLS) return CPR >= 16 ? 4 * (r & 3) : CPR == 8 ? 4 * ((r >> 1) & 1) : 0;
    return (r >> 1) & 7;
  }
  __device__ __forceinline__ void init(const Operand& o, int64_t b, int64_t m0, int64_t M, int64_t K, int w, int ln) {
    lane = ln;
    first = w * L;
    ld = o.ld;
    base = (const T*)o.p + b * o.batch + (COLS ? m0 * PL : m0 * ld);
    k_rows = K;
    // values of a row from base on (rows: with the zeros up to a whole chunk,
    // or a whole group of planes)
    width = COLS ? ld - m0 * PL : PL == 1 ? (K + 7) / 8 * 8 : (K + 31) / 32 * 64;
    if (!COLS) rows = resource(base, ((M - m0 - 1) * ld + width) * (int64_t)sizeof(T));
#pragma unroll
    for (int q = 0; q < L; ++q) {
      const int i = (first + q) * 64 + lane;
      const int r = COLS ? i / CPR : i / 8, c = COLS ? i % CPR : i % 8;
      off[q] = (int)(r * ld * (int64_t)sizeof(T)) + (c ^ swz(r)) * 16;
    }
  }
  __device__ __forceinline__ void issue(T* to, int st) const {
    if constexpr (COLS) {
      const __amdgpu_buffer_rsrc_t src = resource(
          base + (int64_t)st * KS * ld, ((k_rows - (int64_t)st * KS - 1) * ld + width) * (int64_t)sizeof(T));
#pragma unroll
      for (int q = 0; q < L; ++q) copy16(src, to + (first + q) * 512, off[q], 0);
    } else {
      const int left = (int)((width - (int64_t)st * 64) / 8);  // chunks of the row from here on
      if (left < 8) {
#pragma unroll
        for (int q = 0; q < L; ++q) {
          const int r = (first + q) * 8 + lane / 8;
          copy16(rows, to + (first + q) * 512, (lane % 8 ^ swz(r)) < left ? off[q] + st * 128 : kBehind, 0);
        }
        return;
      }
#pragma unroll
      for (int q = 0; q < L; ++q) copy16(rows, to + (first + q) * 512, off[q], st * 128);
    }
  }
  // The fragment of 32-row block `blk`, step kk of 16 k, plane `pl`: lane l
  // holds row l % 32, k 8 (l / 32) .. + 7.
  static __device__ __forceinline__ typename Mfma<T>::vec read(const T* from, int blk, int kk, int pl, int lane) {
    typename Mfma<T>::vec v;
    if constexpr (COLS) {
      const int i = lane & 15, k = kk * 16 + 8 * (lane >> 5) + (i >> 2);
      const int col = (blk * PL + pl) * 32 + (lane & 16) + 4 * (i & 3);
      const T* at = from + k * (B * PL) + (((col >> 3) ^ swz(i >> 2)) << 3) + (col & 4);
      union {
        i16x4 h[2];
        typename Mfma<T>::vec v;
      } u;
      typedef __attribute__((address_space(3))) i16x4* lds4;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at);
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 4 * B * PL));
      v = u.v;
    } else {
      const int r = blk * 32 + (lane & 31), c = pl * 4 + 2 * kk + (lane >> 5);
      v = *(const typename Mfma<T>::vec*)(from + r * 64 + ((c ^ swz(r)) << 3));
    }
    return v;
  }
};

// Where a block stands.
struct Place {
  int64_t m0, n0;
  int tm, tn, split, batch;
  int wave, wm, wn, lane;
};

template <typename T_, int TM_, int TN_, int WM_, int WN_, int PL_, bool AC_, bool BC_, bool SYM_ = false>
struct Tile {
  typedef T_ T;
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, PL = PL_;
  static constexpr bool SYM = SYM_;  // tiles on and below the diagonal only
  static constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN;
  static constexpr int KS = 64 / PL, KK = KS / 16;
  static constexpr int AW = BM / 8, BW = BN / 8, STAGE = (AW + BW) * 512;
  static constexpr int CP = 32 * TN + 4;  // floats of a staged row of the epilogue
  static_assert(AW % NW == 0 && BW % NW == 0, "tile shape");
  static_assert(NW * 32 * CP * 4 <= 2 * STAGE * 2, "epilogue staging");
  typedef Stream<T, BM, AW / NW, PL, AC_> SA;
  typedef Stream<T, BN, BW / NW, PL, BC_> SB;
  typedef typename Mfma<T>::vec V8;
  typedef f32x16 Acc[TM][TN];

  // Blocks in an order that keeps neighbours on one XCD (its blocks are every
  // eighth), groups of `group` tile rows column by column.
  static __device__ __forceinline__ Place place(const Args& p) {
    Place c;
    c.lane = threadIdx.x & 63;
    c.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    c.wm = c.wave / WN;
    c.wn = c.wave % WN;
    const int nb = gridDim.x, x = blockIdx.x & 7, each = nb >> 3, more = nb & 7;
    const int id = x * each + (x < more ? x : more) + (blockIdx.x >> 3);
    const int t = id % p.tiles, rest = id / p.tiles;
    c.split = rest % p.splits;
    c.batch = rest / p.splits;
    if constexpr (SYM) {
      // tile t of the triangle, row by row
      int r = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
      while (r * (r + 1) / 2 > t) --r;
      while ((r + 1) * (r + 2) / 2 <= t) ++r;
      c.tm = r;
      c.tn = t - r * (r + 1) / 2;
    } else {
      const int per = p.group * p.tiles_n, g = t / per, first = g * p.group;
      const int size = p.tiles_m - first < p.group ? p.tiles_m - first : p.group;
      c.tm = first + (t % per) % size;
      c.tn = (t % per) / size;
    }
    c.m0 = (int64_t)c.tm * BM;
    c.n0 = (int64_t)c.tn * BN;
    return c;
  }

  static __device__ __forceinline__ void product(const Args& p, const Place& c, T* lds, Acc& acc) {
    SA a;
    SB b;
    a.init(p.a, c.batch, c.m0, p.M, p.K, c.wave, c.lane);
    b.init(p.b, c.batch, c.n0, p.N, p.K, c.wave, c.lane);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const int s0 = c.split * p.per_split;
    const int left = p.stages - s0, nk = left < p.per_split ? left : p.per_split;
    if (nk <= 0) return;
    auto issue = [&](int st) __attribute__((always_inline)) {
      T* to = lds + (st & 1) * STAGE;
      a.issue(to, s0 + st);
      b.issue(to + AW * 512, s0 + st);
    };
    V8 fa[2][TM], fb[2][TN];
    auto read = [&](int set, int st, int kk) __attribute__((always_inline)) {
      const T* from = lds + (st & 1) * STAGE;
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[set][j] = SB::read(from + AW * 512, c.wn * TN + j, kk, 0, c.lane);
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[set][i] = SA::read(from, c.wm * TM + i, kk, 0, c.lane);
    };
    auto mul = [&](const V8 (&x)[TM], const V8 (&y)[TN]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = Mfma<T>::run(y[j], x[i], acc[i][j]);
    };
    // waits for this wavefront's copies, for those and its LDS reads, for its
    // LDS reads alone
    constexpr int kCopies = 0x0f70, kBoth = 0x0070, kReads = 0xc07f;
    issue(0);
    __builtin_amdgcn_s_waitcnt(kCopies);
    __syncthreads();
    if (nk > 1) issue(1);
    read(0, 0, 0);
    if constexpr (PL == 1) {
      for (int st = 0; st < nk; ++st) {
        // what was read before the last matrix instructions is there; the
        // compiler, which joins two ways into the loop here, would wait for
        // the next reads too
        __builtin_amdgcn_s_waitcnt(kReads);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk + 1 < KK; ++kk) {
          read((kk + 1) & 1, st, kk + 1);
          __builtin_amdgcn_sched_barrier(0);
          mul(fa[kk & 1], fb[kk & 1]);
          __builtin_amdgcn_sched_barrier(0);
        }
        // this wavefront holds the rest of stage st in registers, and its
        // copies of stage st + 1 have landed; after the barrier every
        // wavefront's have
        __builtin_amdgcn_s_waitcnt(kBoth);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        if (st + 2 < nk) issue(st + 2);
        if (st + 1 < nk) read(0, st + 1, 0);
        __builtin_amdgcn_sched_barrier(0);
        mul(fa[(KK - 1) & 1], fb[(KK - 1) & 1]);
      }
    } else {
      static_assert(KK == 2 || PL == 1, "two steps of 16 k in a stage of planes");
      V8 la[TM], lb[TN];
      auto read_low = [&](int st, int kk) __attribute__((always_inline)) {
        const T* from = lds + (st & 1) * STAGE;
#pragma unroll
        for (int j = 0; j < TN; ++j) lb[j] = SB::read(from + AW * 512, c.wn * TN + j, kk, 1, c.lane);
#pragma unroll
        for (int i = 0; i < TM; ++i) la[i] = SA::read(from, c.wm * TM + i, kk, 1, c.lane);
      };
      for (int st = 0; st < nk; ++st) {
        __builtin_amdgcn_s_waitcnt(kReads);
        __builtin_amdgcn_sched_barrier(0);
        read_low(st, 0);
        __builtin_amdgcn_sched_barrier(0);
        mul(fa[0], fb[0]);
        __builtin_amdgcn_sched_barrier(0);
        read(1, st, 1);
        __builtin_amdgcn_sched_barrier(0);
        mul(fa[0], lb);
        mul(la, fb[0]);
        __builtin_amdgcn_sched_barrier(0);
        read_low(st, 1);
        __builtin_amdgcn_sched_barrier(0);
        mul(fa[1], fb[1]);
        __builtin_amdgcn_s_waitcnt(kBoth);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        if (st + 2 < nk) issue(st + 2);
        if (st + 1 < nk) read(0, st + 1, 0);
        __builtin_amdgcn_sched_barrier(0);
        mul(fa[1], lb);
        mul(la, fb[1]);
      }
    }
  }

  // The accumulators hold C transposed: lane l, register e of a 32 x 32 tile
  // is row l % 32, column 8 (e / 4) + 4 (l / 32) + e % 4.
  static __device__ __forceinline__ int row_of(const Place& c, int i) { return (c.wm * TM + i) * 32 + (c.lane & 31); }
  static __device__ __forceinline__ int col_of(const Place& c, int j, int e) {
    return (c.wn * TN + j) * 32 + 8 * (e >> 2) + 4 * (c.lane >> 5) + (e & 3);
  }

  // Through this wavefront's own part of LDS, 32 rows at a time: fr(row,
  // column, v) for 8 columns of each row and, where `with` is true, fc(row,
  // column, v) for 8 rows of each column (row, column: of the product).  The
  // loops stay rolled: unrolled, their instructions come from memory once a
  // launch and compute unit.
  template <bool COLUMNS, class FR, class FC>
  static __device__ __forceinline__ void runs(const Place& c, T* lds, const Acc& acc, bool with, FR fr, FC fc) {
    float* ct = (float*)lds + c.wave * 32 * CP;
    constexpr int CN = 32 * TN, LPR = CN / 8, RPI = 64 / LPR;
    const int l31 = c.lane & 31, hi = c.lane >> 5;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(float4*)(ct + l31 * CP + 32 * j + 8 * g + 4 * hi) =
              make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
      const int64_t rows = c.m0 + (c.wm * TM + i) * 32, cols = c.n0 + c.wn * CN;
#pragma unroll 1
      for (int it = 0; it < 32 / RPI; ++it) {
        const int r = it * RPI + c.lane / LPR, q = (c.lane % LPR) * 8;
        float v[8];
        *(float4*)v = *(const float4*)(ct + r * CP + q);
        *(float4*)(v + 4) = *(const float4*)(ct + r * CP + q + 4);
        fr(rows + r, cols + q, v);
      }
      if constexpr (COLUMNS) {
        if (with) {
#pragma unroll 1
          for (int it = 0; it < CN / 16; ++it) {
            const int q = it * 16 + (c.lane >> 2), r = (c.lane & 3) * 8;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = ct[(r + e) * CP + q];
            fc(rows + r, cols + q, v);
          }
        }
      }
    }
  }
};

// Wavefronts a SIMD that the registers have to leave room for.
constexpr int waves_for(int nw) { return nw >= 8 ? nw / 4 : 2; }

template <class TL, class Epi>
__global__ void __launch_bounds__(64 * TL::NW, waves_for(TL::NW)) tile_kernel(Args p, Epi e) {
  __shared__ __attribute__((aligned(16))) typename TL::T lds[2 * TL::STAGE];
  const Place c = TL::place(p);
  typename TL::Acc acc;
  TL::product(p, c, lds, acc);
  __syncthreads();
  e.template store<TL>(p, c, lds, acc);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Launches a product: sizes, operands, splits and batches are set in p.
template <class TL, class Epi>
void launch(Args p, const Epi& e, hipStream_t s, const char* what) {
  p.tiles_m = (int)ceil_div(p.M, TL::BM);
  p.tiles_n = (int)ceil_div(p.N, TL::BN);
  const int64_t tiles = TL::SYM ? (int64_t)p.tiles_m * (p.tiles_m + 1) / 2 : (int64_t)p.tiles_m * p.tiles_n;
  p.stages = (int)ceil_div(p.K, TL::KS);
  p.per_split = (int)ceil_div(p.stages, p.splits);
  const int64_t blocks = tiles * p.splits * p.batches;
  // (a tile's rows lie within the 2 GiB that a buffer resource spans)
  if (blocks < 1 || blocks >= (1LL << 31) || p.a.ld >= (1 << 21) || p.b.ld >= (1 << 21))
    fail("%s: a product of %lld x %lld x %lld in %d parts is too large", what, (long long)p.M, (long long)p.N,
         (long long)p.K, p.splits);
  p.tiles = (int)tiles;
  hipLaunchKernelGGL((tile_kernel<TL, Epi>), dim3((unsigned)blocks), dim3(64 * TL::NW), 0, s, p, e);
  check_launch(what);
}

// 8 values of a row as plain 16-bit values or as planes, at an 8-aligned
// column.
template <typename T, int PL>
__device__ __forceinline__ void put_planes(T* row, int64_t col, const float (&v)[8]) {
  struct alignas(16) V { T e[8]; } h, l;
  T* at = PL == 1 ? row + col : row + (col >> 5) * 64 + (col & 31);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    h.e[e] = from_f<T>(v[e]);
    if constexpr (PL == 2) {
      const float hf = to_f(h.e[e]);
      // an infinity has no low half (inf - inf)
      l.e[e] = from_f<T>(fabsf(hf) < INFINITY ? v[e] - hf : 0.f);
    }
  }
  *(V*)at = h;
  if constexpr (PL == 2) *(V*)(at + 32) = l;
}
template <typename T, int PL>
__device__ __forceinline__ void get_planes(const T* row, int64_t col, float (&v)[8]) {
  struct alignas(16) V { T e[8]; };
  const T* at = PL == 1 ? row + col : row + (col >> 5) * 64 + (col & 31);
  const V h = *(const V*)at;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = to_f(h.e[e]);
  if constexpr (PL == 2) {
    const V l = *(const V*)(at + 32);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += to_f(l.e[e]);
  }
}

}  // namespace t16
}  // namespace k
}  // namespace agpu
