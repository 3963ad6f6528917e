// The matrix products behind the gated feed-forward block:
//
//   C[m, n] = sum over k of A[m, k] B[n, k]
//
// on 16-bit matrix instructions.  An operand lies in memory either with k along its rows or as
// the transpose, with k down the columns; LDS reads that transpose blocks of 4 x 16 elements
// give the matrix instruction the same registers from either, so nothing is ever laid out anew.
// 16-bit elements go from memory straight to LDS.  Floats come by way of registers, where each is cut
// into three bfloat16 parts a = a0 + a1 + a2 (24 bits in all), and six of the nine products of
// parts are taken: a0 b0, a0 b1, a1 b0, a1 b1, a0 b2, a2 b0.  What is left out is below 2^-21 of
// |a||b|, and bfloat16 has the exponents of float, so no scaling is needed.
#ifndef SSC_GATED_GEMM_H_
#define SSC_GATED_GEMM_H_

#include <type_traits>

#include "elem.h"

namespace ssc {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <typename T> struct Frag;
template <> struct Frag<f16> { typedef f16x8 type; };
template <> struct Frag<bf16> { typedef bf16x8 type; };

// What is done with the product.
enum Epilogue {
  kGated,    // rows of B are w_gate and w_up: y = act(a + b_gate) * (b + b_up), optionally a and b kept
  kStore,    // C rounded to the output type
  kPartial,  // C as float into the slice blockIdx.z of a workspace
};

// An operand: `rows` rows (m or n) along k.
//   k along its rows:  p[row * ld + k], with a second array (kGated) for every other run of rows
//   k down its columns: p[k * ld + row], and from k = `second` on q[(k - second) * ld + row];
//                       each array has `deep` values of k, the rest count as zero
struct Operand {
  const void *p, *q;
  int64_t rows, ld;
  int32_t deep, second;
};

struct GemmArgs {
  Operand a, b;
  int64_t m, n;           // of the results; kGated: n counts the hidden columns
  int32_t k;              // 16 bits with k along rows: a multiple of 8
  int32_t kslice;         // values of k in a slice (kPartial), a multiple of the tile's
  int32_t tiles_m, tiles_n;
  // kStore, kPartial: rows from `second` on are those of out2; out and out2 have `each` rows
  void *out, *out2;
  int64_t second, each, ldo;
  void *kept;             // kGated: a and b for the backward pass (Kept), or NULL
  const void *bias_a, *bias_b;
  int32_t act;
  int32_t wide;           // rows and pointers of the outputs allow stores of 16 bytes
};

// A tile of BM x BN of C for a workgroup of WM x WN waves.
template <typename T_, int PARTS_, int BM_, int BN_, int BK_, int WM_, int WN_> struct Tile {
  typedef T_ T;
  static constexpr int PARTS = PARTS_, BM = BM_, BN = BN_, BK = BK_, WM = WM_, WN = WN_;
  static constexpr int kWaves = WM * WN, kThreads = kWaves * 64;
  static constexpr int kABytes = BM * BK * 2, kBBytes = BN * BK * 2;
  static constexpr int kStage = (kABytes + kBBytes) * PARTS;
  static constexpr int kMi = BM / WM / 16, kNi = BN / WN / 16;
  // the epilogue turns a wave's results in LDS, some rows at a time
  static constexpr int kPitch = kNi * 16 + 4;
  static constexpr int kTurnBlocks = kNi > 4 ? 2 : 4, kTurnRows = kTurnBlocks * 16;
  static constexpr int kTurn = kWaves * kTurnRows * kPitch * 4;
  static constexpr int kLds = 2 * kStage > kTurn ? 2 * kStage : kTurn;
  static_assert((BK == 64 || BK == 32) && kMi % kTurnBlocks == 0 && kNi % 2 == 0 && kLds <= 160 * 1024, "tile");
};

// Workgroups go to the 8 dies in turn; each die gets a run of tiles that are neighbours, in
// strips of 4 tiles along m, so that its level-2 cache serves their common rows.
__device__ __forceinline__ void tile_of(const GemmArgs &g, int &tm, int &tn) {
  const int total = g.tiles_m * g.tiles_n, id = blockIdx.x;
  const int die = id & 7, each = total >> 3, more = total & 7;
  const int at = die * each + (die < more ? die : more) + (id >> 3);
  const int strip = at / (4 * g.tiles_n), first = strip * 4;
  const int wide = g.tiles_m - first < 4 ? g.tiles_m - first : 4;
  const int in = at - strip * 4 * g.tiles_n;
  tm = first + in % wide;
  tn = in / wide;
}

typedef __attribute__((address_space(3))) void *lds_ptr;
typedef __attribute__((address_space(3))) s16x4 *lds_s16x4;
typedef decltype(__builtin_amdgcn_make_buffer_rsrc((void *)0, (short)0, 0, 0)) rsrc_t;

// One operand's tile: R rows x BK values of k, loaded by W waves straight into LDS, and read back
// as the 16 x 32 blocks of the matrix instruction (lane: row lane & 15, k = 8 (lane >> 4) ...).
//
// k along rows: a tile's row is BK elements; chunk c (16 bytes) of row r lies at chunk
// c ^ swizzle(r), so that the 16 rows which are read at the same c fall on all banks evenly.
template <int R, int BK, int W, bool TR> struct Side {
  static constexpr int kChunks = BK / 8, kRows = 64 / kChunks;  // rows that a load of a wave covers
  static constexpr int kLoads = R / (kRows * W);
  static_assert(kLoads * kRows * W == R, "tile");
  rsrc_t rs[kLoads];
  int off, kc;

  static __device__ __forceinline__ int swizzle(int r) { return BK == 64 ? (r & 7) : ((r >> 1) & 3); }

  // A resource for every load of a wave: it spans the few rows of that load, so offsets stay small
  // however long the rows are, and rows behind the matrix read as zero.  HALF > 0: runs of HALF
  // rows come from p and q in turn.
  template <int HALF>
  __device__ __forceinline__ void init(const Operand &o, int64_t r0, int, int w, int lane) {
    const int srow = lane / kChunks;
    kc = ((lane % kChunks) ^ swizzle(srow)) * 8;  // (a load begins at a multiple of 8 rows)
    off = (int)((srow * o.ld + kc) * 2);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int first = (i * W + w) * kRows;
      const bool other = HALF > 0 && first % (2 * HALF) >= HALF;
      const int64_t row = r0 + (HALF > 0 ? first / (2 * HALF) * HALF + first % HALF : first);
      const int64_t rows = o.rows - row < kRows ? o.rows - row : kRows;
      rs[i] = __builtin_amdgcn_make_buffer_rsrc(
          (void *)((const char *)(other ? o.q : o.p) + (rows > 0 ? row : 0) * o.ld * 2), 0,
          rows > 0 ? (int)(rows * o.ld * 2) : 0, 0x00020000);
    }
  }
  __device__ __forceinline__ void load(const Operand &, int k0, int k_end, int w, char *to) {
    // (what lies behind the slice counts as zero; the whole offset is the lane's, which is the one
    // that the resource's size is held against)
    const int o = k0 + kc < k_end ? off + k0 * 2 : 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs[i], (lds_ptr)(to + (i * W + w) * 1024), 16, o, 0, 0, 0);
  }
  template <typename F>
  static __device__ __forceinline__ F block(const char *tile, int row0, int kk, int lane) {
    const int r = lane & 15, c = (kk * 4 + (lane >> 4)) ^ swizzle(r);
    return *reinterpret_cast<const F *>(tile + (row0 + r) * (BK * 2) + (c << 4));
  }
};

// k down columns: the tile's rows are those of memory, R elements for each k; an LDS read takes 4
// elements of one k from each of 16 lanes and hands every lane the 4 values of k of one column, so
// two reads make a block's 8.  The lanes of a read touch 4 neighbouring k (of 16 k in all) at 32
// neighbouring bytes: chunk c of row k lies at c ^ swizzle(k), which spreads them over the banks.
template <int R, int BK, int W> struct Side<R, BK, W, true> {
  static constexpr int kChunks = R / 8, kRows = 64 / kChunks;  // k that a load of a wave covers
  static constexpr int kLoads = BK / (kRows * W);
  static_assert(kLoads * kRows * W == BK && kChunks >= 8, "tile");
  const char *cur, *next;  // where the next step's first value of k lies; the second array
  int64_t left;            // values of k that cur's array has left
  int k, off[kLoads], row, rest;  // row: bytes of a row, rest: of the last one

  static __device__ __forceinline__ int swizzle(int k) {
    return R >= 128 ? ((k & 3) | (k >> 1 & 4)) << 1 : (k & 3) << 1;
  }

  template <int HALF>
  __device__ __forceinline__ void init(const Operand &o, int64_t r0, int k_begin, int w, int lane) {
    const bool other = k_begin >= o.second;
    k = k_begin;
    left = o.deep - (other ? k_begin - o.second : k_begin);
    next = (const char *)o.q + r0 * 2;
    cur = (other ? next : (const char *)o.p + r0 * 2) + (o.deep - left) * o.ld * 2;
    row = (int)o.ld * 2;
    rest = (int)(o.ld - r0) * 2;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int kr = (i * W + w) * kRows + lane / kChunks;
      const int c = ((lane % kChunks) ^ swizzle(kr)) * 8;
      // (columns behind the matrix count as zero)
      off[i] = r0 + c < o.rows ? kr * row + c * 2 : 0x7FFFFFFF;
    }
  }
  // The next BK values of k.
  __device__ __forceinline__ void load(const Operand &o, int, int, int w, char *to) {
    const int there = left < BK ? (int)left : BK;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void *)cur, 0,
                                                      there > 0 ? (there - 1) * row + rest : 0, 0x00020000);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(to + (i * W + w) * 1024), 16, off[i], 0, 0, 0);
    k += BK;
    const bool turn = k == o.second;
    cur = turn ? next : cur + (int64_t)BK * row;
    left = turn ? (int64_t)o.deep : left - BK;
  }
  template <typename F>
  static __device__ __forceinline__ F block(const char *tile, int row0, int kk, int lane) {
    const int q = lane >> 4, l = lane & 15;
    s16x4 v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = kk * 32 + q * 8 + h * 4 + (l >> 2);
      const int col = row0 + (l & 3) * 4;
      v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(
          tile + k * (R * 2) + (((col >> 3) ^ swizzle(k)) << 4) + (col & 4) * 2));
    }
    return __builtin_bit_cast(F, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// The same for floats, 8 of them to a thread at a time: fetched into registers one step before they
// are cut into parts and stored to LDS, so that the way from memory is covered by a whole step.
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void cut_into_parts(const f32x4 (&v)[2], char *to, int stride) {
  uint32_t p[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // (pairs: one instruction rounds two floats)
    const f32x2 x = {v[i / 2][i % 2 * 2], v[i / 2][i % 2 * 2 + 1]};
    // the first part is cut off, which no finite number overflows at, the others are rounded
    f32x2 r;
#pragma unroll
    for (int e = 0; e < 2; ++e) r[e] = x[e] - __uint_as_float(__float_as_uint(x[e]) & 0xFFFF0000u);
    p[0][i] = __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x07060302);
    p[1][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
    r[0] -= __uint_as_float(p[1][i] << 16);
    r[1] -= __uint_as_float(p[1][i] & 0xFFFF0000u);
    p[2][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
  }
#pragma unroll
  for (int k = 0; k < 3; ++k)
    *reinterpret_cast<uint4 *>(to + k * stride) = make_uint4(p[k][0], p[k][1], p[k][2], p[k][3]);
}

template <int R, int BK, int W, bool TR> struct FloatSide : Side<R, BK, W, false> {
  static constexpr int kAcross = BK / 8, kRows = 64 / kAcross;  // rows that a wave's load covers
  static constexpr int kLoads = R / (kRows * W);
  static_assert(kLoads * kRows * W == R, "tile");
  rsrc_t rs[kLoads];
  f32x4 v[kLoads][2];
  int off, kc, to;

  template <int HALF>
  __device__ __forceinline__ void init(const Operand &o, int64_t r0, int, int w, int lane) {
    const int srow = lane / kAcross;
    kc = lane % kAcross * 8;
    off = (int)((srow * o.ld + kc) * 4);
    to = (w * kRows + srow) * (BK * 2) + (((kc >> 3) ^ Side<R, BK, W, false>::swizzle(srow)) << 4);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int first = (i * W + w) * kRows;
      const bool other = HALF > 0 && first % (2 * HALF) >= HALF;
      const int64_t row = r0 + (HALF > 0 ? first / (2 * HALF) * HALF + first % HALF : first);
      const int64_t rows = o.rows - row < kRows ? o.rows - row : kRows;
      rs[i] = __builtin_amdgcn_make_buffer_rsrc(
          (void *)((const char *)(other ? o.q : o.p) + (rows > 0 ? row : 0) * o.ld * 4), 0,
          rows > 0 ? (int)(rows * o.ld * 4) : 0, 0x00020000);
    }
  }
  __device__ __forceinline__ void fetch(const Operand &, int k0) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        v[i][h] = __builtin_bit_cast(
            f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs[i], off + k0 * 4 + h * 16, 0, 0));
  }
  // Zeros for what lies behind the end: behind a row's end lies the next row.
  __device__ __forceinline__ void end(int k0, int k_end) {
    const int left = k_end - k0 - kc;  // values of this thread that exist
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e / 4][e % 4] = e < left ? v[i][e / 4][e % 4] : 0.f;
  }
  __device__ __forceinline__ void store(char *tile, int stride) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) cut_into_parts(v[i], tile + i * (W * kRows * BK * 2) + to, stride);
  }
};

template <int R, int BK, int W> struct FloatSide<R, BK, W, true> : Side<R, BK, W, true> {
  typedef Side<R, BK, W, true> Base;  // (where it stands in memory, and the blocks' layout)
  using Base::cur;
  using Base::k;
  using Base::left;
  using Base::next;
  using Base::rest;
  using Base::row;
  static constexpr int kAcross = R / 8, kLoads = BK * kAcross / (W * 64);
  static_assert(kLoads * W * 64 == BK * kAcross, "tile");
  f32x4 v[kLoads][2];
  int at[kLoads], to[kLoads];

  template <int HALF>
  __device__ __forceinline__ void init(const Operand &o, int64_t r0, int k_begin, int w, int lane) {
    const bool other = k_begin >= o.second;
    k = k_begin;
    left = o.deep - (other ? k_begin - o.second : k_begin);
    next = (const char *)o.q + r0 * 4;
    cur = (other ? next : (const char *)o.p + r0 * 4) + (o.deep - left) * o.ld * 4;
    row = (int)o.ld * 4;
    rest = (int)(o.ld - r0) * 4;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int id = (i * W + w) * 64 + lane, kr = id / kAcross, c = id % kAcross;
      at[i] = kr * row + c * 32;
      to[i] = kr * (R * 2) + ((c ^ Base::swizzle(kr)) << 4);
    }
  }
  // (behind the last column lies the next row: columns of results that are not stored)
  __device__ __forceinline__ void fetch(const Operand &o, int) {
    const int there = left < BK ? (int)left : BK;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void *)cur, 0,
                                                      there > 0 ? (there - 1) * row + rest : 0, 0x00020000);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        v[i][h] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at[i] + h * 16, 0, 0));
    k += BK;
    const bool turn = k == o.second;
    cur = turn ? next : cur + (int64_t)BK * row;
    left = turn ? (int64_t)o.deep : left - BK;
  }
  __device__ __forceinline__ void end(int, int) {}  // (the resource ends there)
  __device__ __forceinline__ void store(char *tile, int stride) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) cut_into_parts(v[i], tile + to[i], stride);
  }
};

template <typename C> struct Blocks {
  typedef typename Frag<typename C::T>::type F;
  F a[C::PARTS][C::kMi], b[C::PARTS][C::kNi];
};

// The blocks of 32 values of k that a wave multiplies next.  (`stage` is not written while it is
// read: without __restrict__ every read would wait for the loads to the other stage.)
template <typename C, typename SA, typename SB>
__device__ __forceinline__ void read_blocks(const char *__restrict__ stage, int kk, int wm, int wn,
                                            Blocks<C> &x) {
  typedef typename Blocks<C>::F F;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int p = 0; p < C::PARTS; ++p) {
    const char *sa = stage + p * C::kABytes, *sb = stage + C::PARTS * C::kABytes + p * C::kBBytes;
#pragma unroll
    for (int j = 0; j < C::kNi; ++j)
      x.b[p][j] = SB::template block<F>(sb, wn * (C::kNi * 16) + j * 16, kk, lane);
#pragma unroll
    for (int i = 0; i < C::kMi; ++i)
      x.a[p][i] = SA::template block<F>(sa, wm * (C::kMi * 16) + i * 16, kk, lane);
  }
}

template <typename C>
__device__ __forceinline__ void multiply(const Blocks<C> &x, f32x4 (&acc)[C::kNi][C::kMi]) {
#pragma unroll
  for (int i = 0; i < C::kMi; ++i)
#pragma unroll
    for (int j = 0; j < C::kNi; ++j) {
      if constexpr (C::PARTS == 3) {
        acc[j][i] = mfma16(x.b[2][j], x.a[0][i], acc[j][i]);
        acc[j][i] = mfma16(x.b[0][j], x.a[2][i], acc[j][i]);
        acc[j][i] = mfma16(x.b[1][j], x.a[1][i], acc[j][i]);
        acc[j][i] = mfma16(x.b[1][j], x.a[0][i], acc[j][i]);
        acc[j][i] = mfma16(x.b[0][j], x.a[1][i], acc[j][i]);
      }
      acc[j][i] = mfma16(x.b[0][j], x.a[0][i], acc[j][i]);
    }
}

// One LDS read behind every few matrix instructions, so that both units are busy all the time.
template <int READS, int MULS> __device__ __forceinline__ void interleave() {
  constexpr int kEach = MULS / READS > 0 ? MULS / READS : 1;
#pragma unroll
  for (int i = 0; i < READS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x8, kEach, 0);  // matrix instructions
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);    // an LDS read
  }
  __builtin_amdgcn_sched_group_barrier(0x8, MULS, 0);
}

// 8 neighbouring results of a row, of which `left` exist.  ONCE: past the caches.
template <bool ONCE, typename O>
__device__ __forceinline__ void store_row(O *p, const float *v, int64_t left, bool wide) {
  if (wide && left >= 8) {
    constexpr int V = 16 / sizeof(O);
#pragma unroll
    for (int i = 0; i < 8; i += V) {
      if constexpr (ONCE) store_floats_once<O, V>(p + i, v + i);
      else store_floats<O, V>(p + i, v + i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (O)v[i];
  }
}

// What a training step keeps of the projections a (which 0) and b (1): [m, n] each, 16-bit ones
// with 8 more bits of the rounding's remainder.  The backward pass rounds da and db to 16 bits
// once, as an operand of its products has to be; with a and b rounded as well the gradients would be
// off by three such roundings instead of two.
//
// The remainder is the difference of the floats' bits, value minus rounded value, a whole number of
// units in the last place that is right across powers of two as well; its top 8 bits are kept.
// All of it is integer arithmetic, 5 instructions a value (a remainder scaled as a float took 15).
template <typename O> struct Kept {
  static constexpr bool kMore = sizeof(O) == 2;
  static constexpr int kHalf = __is_same(O, f16) ? 12 : 15;  // the largest remainder is 2^kHalf
  static constexpr int kShift = kHalf - 7;
  O *p;
  int8_t *q;
  int64_t count;
  __host__ __device__ Kept(const void *base, int64_t m, int64_t n)
      : p(static_cast<O *>(const_cast<void *>(base))), count((m * n + 15) / 16 * 16) {
    q = reinterpret_cast<int8_t *>(p + 2 * count);
  }
  static size_t bytes(int64_t m, int64_t n) {
    return (size_t)((m * n + 15) / 16 * 16) * 2 * (sizeof(O) + (kMore ? 1 : 0));
  }
  // The remainder in its top 8 bits (-128 .. 127).
  static __device__ __forceinline__ int more(float v) {
    const int d = __float_as_int(v) - __float_as_int((float)(O)v);
    const int most = (1 << kHalf) - (1 << (kShift - 1)) - 1;
    int lo = ((d < most ? d : most) + (1 << (kShift - 1))) >> kShift;
    // (half precision ends before float does: of what rounds to an infinity or a denormal number
    // nothing more is kept)
    if constexpr (__is_same(O, f16)) lo = (uint32_t)(d + (1 << kHalf)) <= (2u << kHalf) ? lo : 0;
    return lo;
  }
  static __device__ __forceinline__ float value(O hi, int lo) {
    return __int_as_float(__float_as_int((float)hi) + lo * (1 << kShift));
  }
  template <bool ONCE>
  __device__ __forceinline__ void put(int which, int64_t at, const float *v, int64_t left, bool wide) const {
    store_row<ONCE>(p + which * count + at, v, left, wide);
    if constexpr (kMore) {
      int8_t *to = q + which * count + at;
      if (wide && left >= 8) {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i / 4] |= ((uint32_t)more(v[i]) & 255u) << (i % 4 * 8);
        const uint64_t both = (uint64_t)w[0] | (uint64_t)w[1] << 32;
        if constexpr (ONCE) __builtin_nontemporal_store(both, reinterpret_cast<uint64_t *>(to));
        else *reinterpret_cast<uint64_t *>(to) = both;
      } else {
        for (int i = 0; i < 8; ++i)
          if (i < left) to[i] = (int8_t)more(v[i]);
      }
    }
  }
  // 8 values; ALIGNED: all of them exist and lie at 8 elements.
  template <bool ALIGNED>
  __device__ __forceinline__ void get(int which, int64_t at, int64_t left, float *v) const {
    const O *from = p + which * count + at;
    if constexpr (!kMore) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        if (ALIGNED) load_floats_once<O, 4>(from + i, v + i);
        else
          for (int e = i; e < i + 4; ++e) v[e] = e < left ? (float)from[e] : 0.f;
      }
    } else {
      const int8_t *more = q + which * count + at;
      if constexpr (ALIGNED) {
        const auto hi = __builtin_nontemporal_load(reinterpret_cast<const typename Pack<O, 8>::type *>(from));
        const uint64_t lo = __builtin_nontemporal_load(reinterpret_cast<const uint64_t *>(more));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = value(hi[i], (int8_t)(lo >> (i * 8)));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? value(from[i], more[i]) : 0.f;
      }
    }
  }
};

__device__ __forceinline__ void load_turned(const float *p, float *v) {
  *reinterpret_cast<f32x4 *>(v) = *reinterpret_cast<const f32x4 *>(p);
  *reinterpret_cast<f32x4 *>(v + 4) = *reinterpret_cast<const f32x4 *>(p + 4);
}

// TA, TB: whether A and B have k down their columns.  O: type of the outputs.
template <typename C, bool TA, bool TB, int EPI, typename O>
__global__ void __launch_bounds__(C::kThreads) gemm_kernel(const GemmArgs g) {
#ifdef __HIP_DEVICE_COMPILE__  // (loads to LDS are no builtins of the host's compiler)
  __shared__ __align__(1024) char lds[C::kLds];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = w / C::WN, wn = w % C::WN;
  int tm, tn;
  tile_of(g, tm, tn);
  const int64_t m0 = (int64_t)tm * C::BM;
  // kGated: a tile holds BN / 2 columns of each projection, a wave's columns half of one and
  // half of the other
  constexpr int kCols = EPI == kGated ? C::BN / 2 : C::BN;
  constexpr int kHalf = C::kNi * 8;
  const int64_t n0 = (int64_t)tn * kCols;
  constexpr bool kFloat = C::PARTS == 3;
  typedef std::conditional_t<kFloat, FloatSide<C::BM, C::BK, C::kWaves, TA>, Side<C::BM, C::BK, C::kWaves, TA>> SA;
  typedef std::conditional_t<kFloat, FloatSide<C::BN, C::BK, C::kWaves, TB>, Side<C::BN, C::BK, C::kWaves, TB>> SB;
  SA sa;
  SB sb;
  const int k_begin = EPI == kPartial ? (int)blockIdx.z * g.kslice : 0;
  const int k_end = EPI == kPartial && k_begin + g.kslice < g.k ? k_begin + g.kslice : g.k;
  sa.template init<0>(g.a, m0, k_begin, w, lane);
  sb.template init<EPI == kGated ? kHalf : 0>(g.b, n0, k_begin, w, lane);

  f32x4 acc[C::kNi][C::kMi];
#pragma unroll
  for (int j = 0; j < C::kNi; ++j)
#pragma unroll
    for (int i = 0; i < C::kMi; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  if constexpr (!kFloat) {
    // Two stages in LDS and two sets of blocks in registers: while one set is multiplied the
    // next one is read, and a stage is loaded while the other one is read.
    // The loads of the step that begins at k0: called for one step after the other.
    auto issue = [&](int k0, int s) {
      char *st = lds + s * C::kStage;
      sa.load(g.a, k0, k_end, w, st);
      sb.load(g.b, k0, k_end, w, st + C::kABytes);
    };
    constexpr int kUnits = C::BK / 32;
    static_assert(kUnits == 2, "the sets change places once a stage");
    constexpr int kReads = C::kMi * (TA ? 2 : 1) + C::kNi * (TB ? 2 : 1), kMuls = C::kMi * C::kNi;
    Blocks<C> x0, x1;
    issue(k_begin, 0);
    __syncthreads();
    issue(k_begin + C::BK, 1);
    read_blocks<C, SA, SB>(lds, 0, wm, wn, x0);
    int s = 0;
    for (int k0 = k_begin; k0 < k_end; k0 += C::BK, s ^= 1) {
      read_blocks<C, SA, SB>(lds + s * C::kStage, 1, wm, wn, x1);
      multiply<C>(x0, acc);
      interleave<kReads, kMuls>();
      __syncthreads();  // stage s is read, the other one is there
      if (k0 + 2 * C::BK < k_end) issue(k0 + 2 * C::BK, s);
      // (behind the last step these are blocks that nobody multiplies)
      read_blocks<C, SA, SB>(lds + (s ^ 1) * C::kStage, 0, wm, wn, x0);
      multiply<C>(x1, acc);
      interleave<kReads, kMuls>();
    }
  } else {
    // Two stages in LDS: while one is multiplied the next step's floats are cut into the other one,
    // and those of the step behind it are under way.
    auto fetch = [&](int k0) {
      sa.fetch(g.a, k0);
      sb.fetch(g.b, k0);
    };
    // (a branch of its own, so that all but the last step is one run of instructions)
    auto end = [&](int k0) {
      if (k0 + C::BK <= k_end) return;
      sa.end(k0, k_end);
      sb.end(k0, k_end);
    };
    auto store = [&](int s) {
      sa.store(lds + s * C::kStage, C::kABytes);
      sb.store(lds + s * C::kStage + 3 * C::kABytes, C::kBBytes);
    };
    fetch(k_begin);
    end(k_begin);
    store(0);
    fetch(k_begin + C::BK);
    int s = 0;
    for (int k0 = k_begin; k0 < k_end; k0 += C::BK, s ^= 1) {
      __syncthreads();
      end(k0 + C::BK);
      Blocks<C> x;
      read_blocks<C, SA, SB>(lds + s * C::kStage, 0, wm, wn, x);
      store(s ^ 1);  // (behind the last step these are zeros)
      fetch(k0 + 2 * C::BK);
      multiply<C>(x, acc);
    }
  }
  __syncthreads();

  // A lane holds 4 neighbouring columns of row (lane & 15) in every block of 16 x 16.  Turned in
  // LDS, a lane gets 8 neighbouring columns of a row: stores of 16 bytes.
  // Where a wave's columns of a row fill whole lines of 128 bytes, the results go past the caches,
  // which keep the operands instead: 1085 -> 1045 us for 16384 x 2048 -> 8192 in bfloat16 with the
  // projections kept (with half lines it is 1160).
  constexpr bool kOnce = EPI == kGated && kHalf * sizeof(O) >= 128;
  float *turn = reinterpret_cast<float *>(lds) + w * (C::kTurnRows * C::kPitch);
  constexpr int kAcross = (EPI == kGated ? kHalf : C::kNi * 16) / 8;  // lanes of a row
  const int64_t col = n0 + wn * (kAcross * 8) + lane % kAcross * 8;
  const int64_t left = g.n - col;
  float bias_a[8], bias_b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    bias_a[e] = bias_b[e] = 0.f;
    if (EPI == kGated && e < left) {
      if (g.bias_a != nullptr) bias_a[e] = (float)static_cast<const O *>(g.bias_a)[col + e];
      if (g.bias_b != nullptr) bias_b[e] = (float)static_cast<const O *>(g.bias_b)[col + e];
    }
  }
  const bool wide = g.wide != 0;
#pragma unroll
  for (int h = 0; h < C::kMi / C::kTurnBlocks; ++h) {
#pragma unroll
    for (int i = 0; i < C::kTurnBlocks; ++i)
#pragma unroll
      for (int j = 0; j < C::kNi; ++j)
        *reinterpret_cast<f32x4 *>(turn + (i * 16 + (lane & 15)) * C::kPitch + j * 16 +
                                   (lane >> 4) * 4) = acc[j][h * C::kTurnBlocks + i];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (left > 0) {
#pragma unroll 1
      for (int r = lane / kAcross; r < C::kTurnRows; r += 64 / kAcross) {
        const int64_t row = m0 + wm * (C::kMi * 16) + h * C::kTurnRows + r;
        if (row >= g.m) break;
        const float *from = turn + r * C::kPitch + lane % kAcross * 8;
        float a[8];
        load_turned(from, a);
        if constexpr (EPI == kGated) {
          float b[8], f[8];
          load_turned(from + kHalf, b);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            a[e] += bias_a[e];
            b[e] += bias_b[e];
          }
          if (g.kept != nullptr) {
            const Kept<O> kept(g.kept, g.m, g.n);
            kept.template put<kOnce>(0, row * g.n + col, a, left, wide);
            kept.template put<kOnce>(1, row * g.n + col, b, left, wide);
          }
          activate<8>(g.act, a, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= b[e];
          store_row<kOnce>(static_cast<O *>(g.out) + row * g.ldo + col, f, left, wide);
        } else {
          const bool other = row >= g.second;
          const int64_t r2 = other ? row - g.second : row;
          if (r2 >= g.each) continue;
          O *y;  // (a slice's rows: those of out and of out2, one behind the other)
          if (EPI == kPartial) y = static_cast<O *>(g.out) + ((blockIdx.z * (g.second < g.m ? 2 : 1) + (other ? 1 : 0)) * g.each + r2) * g.ldo;
          else y = static_cast<O *>(other ? g.out2 : g.out) + r2 * g.ldo;
          store_row<false>(y + col, a, left, wide);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
#endif
}

}  // namespace ssc

#endif
