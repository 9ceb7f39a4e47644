// Products of 16-bit operands for kernels with epilogues of their own:
// acc[m][n] = sum over k of A(m, k) B(n, k), fp32 accumulation on
// v_mfma_f32_32x32x16, with each operand in memory either as rows (k
// contiguous) or as columns (row k holds every m), and either as plain values
// or as two planes, the high and the low half of an fp32 value.  A matrix that
// one product reads as rows and another as columns can lie in panels of 128
// bytes of every row, one panel after the other: both then read long runs.
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

#include <algorithm>

#include "device.hpp"
#include "extent.hpp"

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
  int tiles_m = 0, tiles_n = 0, tiles = 0;  // tiles: those that are computed of a matrix
  int first = 0, some = 0;  // of all matrices' tiles, the launch's first and number (0: all)
  int splits = 1, batches = 1;
  int stages = 0, per_split = 0;
  const float2* b_power = nullptr;  // what fp32 rows of b are multiplied by before they are split (.x)
  // Products of planes whose epilogue allows it (kFull): where *full is not 0,
  // the fp32 operands themselves instead, laid out as the layouts say, ld and
  // panels counted in fp32 values.
  const int* full = nullptr;
  const float *fa = nullptr, *fb = nullptr;
  int64_t lda = 0, ldb = 0;
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

typedef __attribute__((address_space(3))) i16x4* lds_i16x4;
// 16 lanes' 4 rows x 16 values of 16 bits, each lane its column.  `restrict`
// gives the read an alias scope: without one the compiler takes it to depend
// on every copy to LDS under way and waits for all of them first (2.4 instead
// of 1.6 us a stage); what it does depend on is waited for by hand, once a
// stage.
__device__ __forceinline__ i16x4 read_transposed(const __attribute__((address_space(3))) i16x4* __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)p);
}

// How an operand lies in memory.
enum Layout {
  kRows,       // k contiguous, rows ld apart
  kCols,       // k rows of every m, ld apart
  kRaw,        // rows of fp32 values, split into planes in registers
  kPanelRows,  // panels of 64 values of each row, ld apart; k along the panels
  kPanelCols,  // the same, m along the panels and k down them
};

// One operand's part of a block: B rows (m) of it, L windows of 1 KB a
// wavefront and stage.  kRaw: rows of fp32 values, in the place of their planes
// (32 a stage; K and ld multiples of 4, ld and offsets in 16-bit units all the
// same).
template <typename T, int B, int L, int PL, Layout LAY>
struct Stream {
  static constexpr bool COLS = LAY == kCols || LAY == kPanelCols, PANEL = LAY == kPanelRows || LAY == kPanelCols;
  static constexpr int KS = 64 / PL;                 // k of a stage
  static constexpr int CPR = COLS ? B * PL / 8 : 8;  // 16-byte chunks of a k row, or of a row's stage
  const T* base;
  int64_t ld, k_rows, width;
  int64_t from, cols;  // kCols: the block's first column, all columns
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
    k_rows = K;
    if constexpr (PANEL) {
      // whole panels a block: of its columns as many as the matrix has, of its
      // rows each panel's from base on
      static_assert(!COLS || B * PL % 64 == 0, "a block of panels");
      base = (const T*)o.p + (COLS ? m0 * PL / 64 * ld : m0 * 64);
      const int64_t panels = ((M - m0) * PL + 63) / 64;
      width = !COLS ? (M - m0) * 64 : panels < B * PL / 64 ? panels * ld : B * PL / 64 * ld;
    } else {
      base = (const T*)o.p + b * o.batch + (COLS ? m0 * PL : m0 * ld);
      from = m0;
      cols = M;
      // values of a row, with the zeros up to a whole chunk or a whole group of
      // planes
      width = LAY == kRaw ? K * 2 : row_values(K, PL);
      if (!COLS) rows = resource(base, ((M - m0 - 1) * ld + width) * (int64_t)sizeof(T));
    }
#pragma unroll
    for (int q = 0; q < L; ++q) {
      const int i = (first + q) * 64 + lane, r = i / CPR, c = (i % CPR) ^ swz(r);
      if constexpr (LAY == kPanelCols) off[q] = (int)((c / 8) * ld * (int64_t)sizeof(T)) + r * 128 + c % 8 * 16;
      else off[q] = (int)(r * (PANEL ? 64 : ld) * (int64_t)sizeof(T)) + c * 16;
    }
  }
  __device__ __forceinline__ void issue(T* to, int st) const {
    if constexpr (LAY == kPanelCols) {
      // rows behind the last would be the next panel's first
      const int64_t left = k_rows - (int64_t)st * KS, from = (int64_t)st * KS * 64;
      const __amdgpu_buffer_rsrc_t src = resource(base + from, (width - from) * (int64_t)sizeof(T));
#pragma unroll
      for (int q = 0; q < L; ++q)
        copy16(src, to + (first + q) * 512, ((first + q) * 64 + lane) / CPR < left ? off[q] : kBehind, 0);
    } else if constexpr (LAY == kPanelRows) {
      const __amdgpu_buffer_rsrc_t src = resource(base + (int64_t)st * ld, width * (int64_t)sizeof(T));
#pragma unroll
      for (int q = 0; q < L; ++q) copy16(src, to + (first + q) * 512, off[q], 0);
    } else if constexpr (COLS) {
      const __amdgpu_buffer_rsrc_t src =
          resource(base + (int64_t)st * KS * ld,
                   extent_of_columns(k_rows - (int64_t)st * KS, cols, from, ld, PL) * (int64_t)sizeof(T));
#pragma unroll
      for (int q = 0; q < L; ++q) copy16(src, to + (first + q) * 512, off[q], 0);
    } else {
      const int left = (int)((width - (int64_t)st * 64) / 8);  // chunks of the row from here on
      if (left < CPR) {
#pragma unroll
        for (int q = 0; q < L; ++q) {
          const int i = (first + q) * 64 + lane;
          copy16(rows, to + (first + q) * 512, (i % CPR ^ swz(i / CPR)) < left ? off[q] + st * 128 : kBehind, 0);
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
      u.h[0] = read_transposed((lds_i16x4)at);
      u.h[1] = read_transposed((lds_i16x4)(at + 4 * B * PL));
      v = u.v;
    } else {
      const int r = blk * 32 + (lane & 31), c = pl * 4 + 2 * kk + (lane >> 5);
      v = *(const typename Mfma<T>::vec*)(from + r * 64 + ((c ^ swz(r)) << 3));
    }
    return v;
  }
};

// 8 fp32 values of a row of a RAW stage (step kk of 16 k), and their planes.
struct Raw8 { float e[8]; };
__device__ __forceinline__ Raw8 read_raw(const half_t* from, int blk, int kk, int lane) {
  const int r = blk * 32 + (lane & 31), c = 4 * kk + 2 * (lane >> 5), x = (r >> 1) & 7;
  Raw8 v;
  *(float4*)v.e = *(const float4*)(from + r * 64 + ((c ^ x) << 3));
  *(float4*)(v.e + 4) = *(const float4*)(from + r * 64 + (((c + 1) ^ x) << 3));
  return v;
}
__device__ __forceinline__ void split_raw(const Raw8& v, float power, Mfma<half_t>::vec& h, Mfma<half_t>::vec& l) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    h[e] = (_Float16)(v.e[e] * power);
    l[e] = (_Float16)fmaf(v.e[e], power, -(float)h[e]);
  }
}

// Where a block stands.
struct Place {
  int64_t m0, n0;
  int tm, tn, split, batch;
  int index;  // of the launch's tiles
  int wave, wm, wn, lane;
};

template <typename T_, int TM_, int TN_, int WM_, int WN_, int PL_, Layout AL_, Layout BL_, bool SYM_ = false>
struct Tile {
  typedef T_ T;
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, PL = PL_;
  static constexpr bool SYM = SYM_;  // tiles on and below the diagonal only
  static constexpr bool RAW = BL_ == kRaw;
  static constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN;
  static constexpr int KS = 64 / PL, KK = KS / 16;
  static constexpr int AW = BM / 8, BW = BN / 8, STAGE = (AW + BW) * 512;  // 16-bit values
  static constexpr int LDS = 2 * STAGE;
  static_assert(AW % NW == 0 && BW % NW == 0, "tile shape");
  // the epilogue stages 32 rows of every wavefront in the operands' place
  static_assert(NW * 32 * 32 * TN * 4 <= LDS * 2, "epilogue staging");
  typedef Stream<T, BM, AW / NW, PL, AL_> SA;
  typedef Stream<T, BN, BW / NW, PL, BL_> SB;
  static_assert(!RAW || PL == 2, "fp32 rows of a product of planes");
  typedef typename Mfma<T>::vec V8;
  typedef f32x16 Acc[TM][TN];

  // Blocks in an order that keeps neighbours on one XCD (its blocks are every
  // eighth), groups of `group` tile rows column by column.
  static __device__ __forceinline__ Place place(const Args& p, int block, int blocks) {
    const int x = block & 7, each = blocks >> 3, more = blocks & 7;
    const int id = x * each + (x < more ? x : more) + (block >> 3);
    Place c = place_of(p, id % p.some);
    c.split = id / p.some;
    return c;
  }
  // The launch's tile `index`, not split.
  static __device__ __forceinline__ Place place_of(const Args& p, int index) {
    Place c;
    c.lane = threadIdx.x & 63;
    c.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    c.wm = c.wave / WN;
    c.wn = c.wave % WN;
    c.index = index;
    const int t = (p.first + index) % p.tiles;
    c.split = 0;
    c.batch = (p.first + index) / p.tiles;
    if constexpr (SYM) {
      // tile t of the triangle, row by row
      int r = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
      while (r * (r + 1) / 2 > t) --r;
      while ((r + 1) * (r + 2) / 2 <= t) ++r;
      c.tm = r;
      c.tn = t - r * (r + 1) / 2;
    } else {
      constexpr int kGroup = 8;  // tile rows that share their columns' loads
      const int per = kGroup * p.tiles_n, g = t / per, first = g * kGroup;
      const int size = p.tiles_m - first < kGroup ? p.tiles_m - first : kGroup;
      c.tm = first + (t % per) % size;
      c.tn = (t % per) / size;
    }
    c.m0 = (int64_t)c.tm * BM;
    c.n0 = (int64_t)c.tn * BN;
    return c;
  }

  // The product of a block's tile.  Behind it every wavefront has read all it
  // reads from LDS.
  static __device__ __forceinline__ void product(const Args& p, const Place& c, T* lds, Acc& acc) {
    SA a;
    SB b;
    a.init(p.a, c.batch, c.m0, p.M, p.K, c.wave, c.lane);
    b.init(p.b, c.batch, c.n0, p.N, p.K, c.wave, c.lane);
    const int s0 = c.split * p.per_split;
    const int nk = p.stages - s0 < p.per_split ? p.stages - s0 : p.per_split;
    auto issue = [&](int st) __attribute__((always_inline)) {
      T* to = lds + (st & 1) * STAGE;
      a.issue(to, s0 + st);
      b.issue(to + AW * 512, s0 + st);
    };
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    V8 fa[2][TM], fb[2][TN];
    Raw8 raw[2][TN];
    const float power = RAW ? p.b_power->x : 1.f;
    auto read = [&](int set, int st, int kk) __attribute__((always_inline)) {
      const T* from = lds + (st & 1) * STAGE;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        if constexpr (RAW) raw[set][j] = read_raw((const half_t*)from + AW * 512, c.wn * TN + j, kk, c.lane);
        else fb[set][j] = SB::read(from + AW * 512, c.wn * TN + j, kk, 0, c.lane);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[set][i] = SA::read(from, c.wm * TM + i, kk, 0, c.lane);
    };
    auto mul = [&](const V8 (&x)[TM], const V8 (&y)[TN]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = Mfma<T>::run(y[j], x[i], acc[i][j]);
    };
    // this wavefront's copies of stage st + 1 have landed, and it holds in
    // registers what it reads of stage st; behind the barrier so does every
    // wavefront, and stage st + 2 takes stage st's place.  (Four stages in LDS
    // were no faster where a compute unit has one block, stages of 32 k 10 %
    // slower.)
    auto next = [&](int st) __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(0x0070);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      if (st + 2 < nk) issue(st + 2);
    };
    constexpr int kReads = 0xc07f;  // waits for LDS reads alone
    if (nk > 0) issue(0);
    next(-1);
    if (nk > 0) read(0, 0, 0);
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
        next(st);
        if (st + 1 < nk) read(0, st + 1, 0);
        __builtin_amdgcn_sched_barrier(0);
        mul(fa[(KK - 1) & 1], fb[(KK - 1) & 1]);
      }
    } else {
      static_assert(KK == 2 || PL == 1, "two steps of 16 k in a stage of planes");
      V8 la[TM], lb[TN];
      auto read_low = [&](int st, int kk) __attribute__((always_inline)) {
        const T* from = lds + (st & 1) * STAGE;
        if constexpr (!RAW) {
#pragma unroll
          for (int j = 0; j < TN; ++j) lb[j] = SB::read(from + AW * 512, c.wn * TN + j, kk, 1, c.lane);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) la[i] = SA::read(from, c.wm * TM + i, kk, 1, c.lane);
      };
      auto split = [&](int set) __attribute__((always_inline)) {
        if constexpr (RAW) {
#pragma unroll
          for (int j = 0; j < TN; ++j) split_raw(raw[set][j], power, fb[set][j], lb[j]);
        }
      };
      for (int st = 0; st < nk; ++st) {
        __builtin_amdgcn_s_waitcnt(kReads);
        __builtin_amdgcn_sched_barrier(0);
        read_low(st, 0);
        split(0);
        __builtin_amdgcn_sched_barrier(0);
        mul(fa[0], fb[0]);
        __builtin_amdgcn_sched_barrier(0);
        read(1, st, 1);
        __builtin_amdgcn_sched_barrier(0);
        mul(fa[0], lb);
        mul(la, fb[0]);
        __builtin_amdgcn_sched_barrier(0);
        read_low(st, 1);
        split(1);
        __builtin_amdgcn_sched_barrier(0);
        mul(fa[1], fb[1]);
        next(st);
        if (st + 1 < nk) read(0, st + 1, 0);
        __builtin_amdgcn_sched_barrier(0);
        mul(fa[1], lb);
        mul(la, fb[1]);
      }
    }
  }

  // 4 fp32 values k .. k + 3 of an operand's row m, zeros from `end` on.
  template <Layout LAY>
  static __device__ __forceinline__ void fetch(const float* p, int64_t ld, int64_t m, int64_t k, int64_t end,
                                               float (&v)[4]) {
    if constexpr (LAY == kCols || LAY == kPanelCols) {
      const float* at = LAY == kCols ? p + k * ld + m : p + (m >> 5) * ld + k * 32 + (m & 31);
      const int64_t apart = LAY == kCols ? ld : 32;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = k + q < end ? at[q * apart] : 0.f;
    } else {
      const float* at = LAY == kPanelRows ? p + (k >> 5) * ld + m * 32 + (k & 31) : p + m * ld + k;
      if (k + 4 <= end) __builtin_memcpy(v, at, 16);  // (at any alignment)
      else
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = k + q < end ? at[q] : 0.f;
    }
  }
  // The same product of the fp32 operands themselves (p.full), whatever their
  // sizes: v_mfma_f32_32x32x2, whose lanes take 4 k of 8 in turn, straight from
  // memory, the next 8 k under way meanwhile (1023 x 50257 x 768: 1730 us without,
  // 962 with; planes 313).
  static __device__ __forceinline__ void product_full(const Args& p, const Place& c, Acc& acc) {
    const int64_t k0 = (int64_t)c.split * p.per_split * KS, past = k0 + (int64_t)p.per_split * KS;
    const int64_t end = past < p.K ? past : p.K;
    const int hi = c.lane >> 5;
    int64_t am[TM], bn[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t m = c.m0 + (c.wm * TM + i) * 32 + (c.lane & 31);
      am[i] = m < p.M ? m : p.M - 1;  // (rows behind the last are not stored)
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int64_t n = c.n0 + (c.wn * TN + j) * 32 + (c.lane & 31);
      bn[j] = n < p.N ? n : p.N - 1;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    float a[2][TM][4], b[2][TN][4];
    auto read = [&](int set, int64_t k) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < TM; ++i) fetch<AL_>(p.fa, p.lda, am[i], k + 4 * hi, end, a[set][i]);
#pragma unroll
      for (int j = 0; j < TN; ++j) fetch<BL_>(p.fb, p.ldb, bn[j], k + 4 * hi, end, b[set][j]);
    };
    auto mul = [&](int set) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(b[set][j][q], a[set][i][q], acc[i][j], 0, 0, 0);
    };
    // (zeros from the end on)
    read(0, k0);
#pragma unroll 1
    for (int64_t k = k0; k < end; k += 16) {
      read(1, k + 8);
      mul(0);
      read(0, k + 16);
      mul(1);
    }
  }

  // The accumulators hold C transposed: lane l, register e of a 32 x 32 tile
  // is row l % 32, column 8 (e / 4) + 4 (l / 32) + e % 4.
  static __device__ __forceinline__ int row_of(const Place& c, int i) { return (c.wm * TM + i) * 32 + (c.lane & 31); }
  static __device__ __forceinline__ int col_of(const Place& c, int j, int e) {
    return (c.wn * TN + j) * 32 + 8 * (e >> 2) + 4 * (c.lane >> 5) + (e & 3);
  }

  // 4 columns of a row at a time, as the accumulators hold them: f(i, j, g, v)
  // for row row_of(c, i), columns col_of(c, j, 4 g) of the tile.
  template <class F>
  static __device__ __forceinline__ void fours(Acc& acc, F f) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float v[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
          f(i, j, g, v);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][4 * g + e] = v[e];
        }
      // f's loads of one i at a time: all of them do not fit the registers
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // The same places in a matrix of E: a buffer resource from the tile's first
  // element on, so that a lane's places are one offset and constants.  Rows
  // behind the matrix read zeros and are not written; columns are the caller's
  // to check.
  template <typename E, int PLANES = 1>
  struct Places {
    __amdgpu_buffer_rsrc_t at;
    int lane_at, per_i;
    __device__ __forceinline__ Places(const Place& c, const E* base, int64_t ld, int64_t rows) {
      at = resource(base + c.m0 * ld + c.n0 * PLANES, ((rows - c.m0) * ld - c.n0 * PLANES) * (int64_t)sizeof(E));
      lane_at = (int)((row_of(c, 0) * ld + c.wn * TN * 32 * PLANES + 4 * (c.lane >> 5)) * (int64_t)sizeof(E));
      per_i = (int)(32 * ld * (int64_t)sizeof(E));
    }
    static constexpr int off(int j, int g, int plane) {
      return ((32 * j) * PLANES + 32 * plane + 8 * g) * (int)sizeof(E);
    }
    __device__ __forceinline__ void load(int i, int j, int g, float (&v)[4], int plane = 0) const {
      const int o = lane_at + off(j, g, plane);
      if constexpr (sizeof(E) == 4) {
        const auto r = __builtin_amdgcn_raw_buffer_load_b128(at, o, i * per_i, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_bit_cast(float, (uint32_t)r[e]);
      } else {
        const auto r = __builtin_amdgcn_raw_buffer_load_b64(at, o, i * per_i, 0);
        typedef E E4 __attribute__((ext_vector_type(4)));
        const E4 x = __builtin_bit_cast(E4, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)x[e];
      }
    }
  };

  // Through this wavefront's own part of LDS, 32 rows at a time: fr(row, column,
  // v) for 8 columns of each row and, where `with` is true, fc(row, column, v)
  // for 8 rows of each column (row, column: of the product).  A row's 16-byte chunks are exchanged so that 16 rows at
  // one chunk cover all banks.  The loops stay rolled: unrolled, their
  // instructions come from memory once a launch and compute unit.
  template <bool COLUMNS, class FR, class FC>
  static __device__ __forceinline__ void runs(const Place& c, T* lds, const Acc& acc, bool with, FR fr, FC fc) {
    constexpr int CN = 32 * TN, LPR = CN / 8, RPI = 64 / LPR;
    float* ct = (float*)lds + c.wave * 32 * CN;
    const int l31 = c.lane & 31, hi = c.lane >> 5;
    auto at = [&](int r, int chunk) { return r * CN + ((TN == 1 ? chunk ^ ((r >> 1) & 7) : chunk ^ (r & 15)) << 2); };
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(float4*)(ct + at(l31, 8 * j + 2 * g + hi)) =
              make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
      const int64_t rows = c.m0 + (c.wm * TM + i) * 32, cols = c.n0 + c.wn * CN;
#pragma unroll 1
      for (int it = 0; it < 32 / RPI; ++it) {
        const int r = it * RPI + c.lane / LPR, q = c.lane % LPR;
        float v[8];
        *(float4*)v = *(const float4*)(ct + at(r, 2 * q));
        *(float4*)(v + 4) = *(const float4*)(ct + at(r, 2 * q + 1));
        fr(rows + r, cols + 8 * q, v);
      }
      if constexpr (COLUMNS) {
        if (with) {
#pragma unroll 1
          for (int it = 0; it < CN / 16; ++it) {
            const int q = it * 16 + (c.lane >> 2), r = (c.lane & 3) * 8;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = ct[at(r + e, q >> 2) + (q & 3)];
            fc(rows + r, cols + q, v);
          }
        }
      }
    }
  }
};

// Wavefronts a SIMD that the registers have to leave room for.
constexpr int waves_for(int nw) { return nw >= 8 ? nw / 4 : 2; }

// An epilogue's `form` works on the accumulators, its `store` through LDS.
// (Blocks that take several tiles and copy the next one's first stage meanwhile
// gained 2 % at 25 tiles a compute unit and spilled registers.)
template <class TL, class Epi>
__device__ __forceinline__ void tile_block(const Args& p, const Epi& e, typename TL::T* lds, int block, int blocks) {
  const Place c = TL::place(p, block, blocks);
  typename TL::Acc acc;
  bool full = false;
  if constexpr (TL::PL == 2 && Epi::kFull) full = *p.full != 0;
  if (full) TL::product_full(p, c, acc);
  else TL::product(p, c, lds, acc);
  e.template form<TL>(p, c, acc);
  e.template store<TL>(p, c, lds, acc);
}

template <class TL, class Epi>
__global__ void __launch_bounds__(64 * TL::NW, waves_for(TL::NW)) tile_kernel(Args p, Epi e) {
  __shared__ __attribute__((aligned(16))) typename TL::T lds[TL::LDS];
  tile_block<TL>(p, e, lds, blockIdx.x, gridDim.x);
}

// Two products that do not depend on one another, the first one's blocks
// first: the last blocks of both fill one round of compute units.
template <class TL1, class E1, class TL2, class E2>
__global__ void __launch_bounds__(64 * TL1::NW, waves_for(TL1::NW)) tile_pair_kernel(Args p1, E1 e1, Args p2, E2 e2) {
  static_assert(TL1::NW == TL2::NW, "wavefronts of a block");
  constexpr int n = TL1::LDS > TL2::LDS ? TL1::LDS : TL2::LDS;
  __shared__ __attribute__((aligned(16))) typename TL1::T lds[n];
  const int first = p1.some * p1.splits;
  if ((int)blockIdx.x < first) tile_block<TL1>(p1, e1, lds, blockIdx.x, first);
  else tile_block<TL2>(p2, e2, lds, blockIdx.x - first, gridDim.x - first);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The blocks of a product: sizes, operands, splits and batches are set in p.
template <class TL>
int64_t blocks_of(Args& p, const char* what) {
  p.tiles_m = (int)ceil_div(p.M, TL::BM);
  p.tiles_n = (int)ceil_div(p.N, TL::BN);
  const int64_t tiles = TL::SYM ? (int64_t)p.tiles_m * (p.tiles_m + 1) / 2 : (int64_t)p.tiles_m * p.tiles_n;
  p.stages = (int)ceil_div(p.K, TL::KS);
  p.per_split = (int)ceil_div(p.stages, p.splits);
  const int64_t some = p.some ? p.some : tiles * p.batches, blocks = some * p.splits;
  // (a tile's rows, or its panels, lie within the 2 GiB that a buffer resource
  // spans)
  if (blocks < 1 || blocks >= (1LL << 30) || p.a.ld >= (TL::SA::PANEL ? 1 << 27 : 1 << 21) || p.b.ld >= (1 << 21))
    fail("%s: a product of %lld x %lld x %lld in %d parts is too large", what, (long long)p.M, (long long)p.N,
         (long long)p.K, p.splits);
  p.tiles = (int)tiles;
  p.some = (int)some;
  return blocks;
}

template <class TL, class Epi>
void launch(Args p, const Epi& e, hipStream_t s, const char* what) {
  const int64_t blocks = blocks_of<TL>(p, what);
  hipLaunchKernelGGL((tile_kernel<TL, Epi>), dim3((unsigned)blocks), dim3(64 * TL::NW), 0, s, p, e);
  check_launch(what);
}
template <class TL1, class TL2, class E1, class E2>
void launch_pair(Args p1, const E1& e1, Args p2, const E2& e2, hipStream_t s, const char* what) {
  const int64_t blocks = blocks_of<TL1>(p1, what) + blocks_of<TL2>(p2, what);
  hipLaunchKernelGGL((tile_pair_kernel<TL1, E1, TL2, E2>), dim3((unsigned)blocks), dim3(64 * TL1::NW), 0, s, p1, e1, p2,
                     e2);
  check_launch(what);
}

// A product whose last tiles, fewer than fill the chip, are split over k: the
// tiles from p.some on in `splits` parts, which join_kernel sums in order.
template <class TL, class Epi>
__global__ void __launch_bounds__(64 * TL::NW, waves_for(TL::NW)) tail_kernel(Args p, Epi e, int splits, float* part) {
  __shared__ __attribute__((aligned(16))) typename TL::T lds[TL::LDS];
  const bool tail = (int)blockIdx.x >= p.some;
  const int whole = p.some;
  if (tail) {
    p.first = whole;
    p.some = (int)(gridDim.x - whole) / splits;
    p.splits = splits;
    p.per_split = (p.stages + splits - 1) / splits;
  }
  const Place c = TL::place(p, blockIdx.x - (tail ? whole : 0), tail ? gridDim.x - whole : whole);
  typename TL::Acc acc;
  TL::product(p, c, lds, acc);
  if (!tail) {
    e.template form<TL>(p, c, acc);
    e.template store<TL>(p, c, lds, acc);
    return;
  }
  float* to = part + ((int64_t)c.index * splits + c.split) * (TL::BM * TL::BN);
  Place at = c;
  at.m0 = at.n0 = 0;
  TL::template runs<false>(
      at, lds, acc, false,
      [&](int64_t row, int64_t col, float (&v)[8]) {
        float4* o = (float4*)(to + row * TL::BN + col);
        o[0] = *(const float4*)v;
        o[1] = *(const float4*)(v + 4);
      },
      [](int64_t, int64_t, float (&)[8]) {});
}
// The tiles of BIG that were split, from p.first on, in blocks of JT's shape.
template <class BIG, class JT, class Epi>
__global__ void __launch_bounds__(64 * JT::NW) join_kernel(Args p, Epi e, int splits, const float* part) {
  __shared__ __attribute__((aligned(16))) typename JT::T lds[JT::LDS];
  constexpr int ACROSS = BIG::BN / JT::BN, EACH = BIG::BM / JT::BM * ACROSS;
  const int tile = blockIdx.x / EACH, m = blockIdx.x % EACH / ACROSS * JT::BM, n = blockIdx.x % ACROSS * JT::BN;
  const Place big = BIG::place_of(p, tile);
  Place c = JT::place_of(p, tile);
  c.tm = big.tm;
  c.tn = big.tn;
  c.batch = big.batch;
  c.m0 = big.m0 + m;
  c.n0 = big.n0 + n;
  if (c.m0 >= p.M || c.n0 >= p.N) return;
  constexpr int64_t kTile = BIG::BM * BIG::BN;
  const float* from = part + (int64_t)tile * splits * kTile + m * BIG::BN + n;
  typename JT::Acc acc = {};
  for (int s = 0; s < splits; ++s, from += kTile)
    JT::fours(acc, [&](int i, int j, int g, float (&v)[4]) {
      const float4 q = *(const float4*)(from + JT::row_of(c, i) * BIG::BN + JT::col_of(c, j, 4 * g));
      v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
    });
  e.template form<JT>(p, c, acc);
  e.template store<JT>(p, c, lds, acc);
}
// The first `whole` tiles as they are, those behind them split and joined; part
// holds (tiles - whole) * splits tiles.
template <class TL, class JT, class Epi>
void launch_tail(Args p, const Epi& e, int64_t whole, int splits, float* part, hipStream_t s, const char* what) {
  const int64_t all = blocks_of<TL>(p, what), rest = all - whole, blocks = whole + rest * splits;
  constexpr int EACH = TL::BM / JT::BM * (TL::BN / JT::BN);
  if (rest < 0 || blocks >= (1LL << 30) || rest * EACH >= (1LL << 30))
    fail("%s: %lld tiles in %d parts", what, (long long)rest, splits);
  p.some = (int)whole;
  hipLaunchKernelGGL((tail_kernel<TL, Epi>), dim3((unsigned)blocks), dim3(64 * TL::NW), 0, s, p, e, splits, part);
  check_launch(what);
  if (rest == 0) return;
  p.first = (int)whole;
  p.some = (int)rest;
  hipLaunchKernelGGL((join_kernel<TL, JT, Epi>), dim3((unsigned)(rest * EACH)), dim3(64 * JT::NW), 0, s, p, e, splits,
                     part);
  check_launch(what);
}

// Stores past the L2, for what this launch does not read again: kept there,
// 128 KB a block push out the operands of the next tiles (8191 x 50257 x 768
// with a 16-bit result: 690 us, so 600), and what a launch leaves there is
// written back behind its last block (twelve 768 x 768 x 768 with their mirror
// images: 11.8 us, so 10.6).
template <typename V>
__device__ __forceinline__ void put_past(void* to, const V& v) {
  typedef uint32_t w __attribute__((ext_vector_type(sizeof(V) / 4), aligned(2)));
  __builtin_nontemporal_store(__builtin_bit_cast(w, v), (w*)to);
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
    if constexpr (PL == 2) l.e[e] = from_f<T>(v[e] - to_f(h.e[e]));  // (an infinity's is NaN)
  }
  put_past(at, h);
  if constexpr (PL == 2) put_past(at + 32, l);
}

}  // namespace t16
}  // namespace k
}  // namespace agpu
