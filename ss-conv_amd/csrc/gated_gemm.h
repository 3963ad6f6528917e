// The matrix product behind the gated feed-forward block:
//
//   C[m, n] = sum over k of A[m, k] B[n, k]
//
// on 16-bit matrix instructions, both operands with k running along memory.  float operands come
// as three bfloat16 parts a = a0 + a1 + a2 (each the rounding of what the parts before it leave:
// 24 bits in all), laid one behind another in a row, and six of the nine products of parts are
// taken: a0 b0, a0 b1, a1 b0, a1 b1, a0 b2, a2 b0.  What is left out is below 2^-24 of |a||b|,
// and bfloat16 has the exponents of float, so no scaling is needed.
#ifndef SSC_GATED_GEMM_H_
#define SSC_GATED_GEMM_H_

#include "elem.h"

namespace ssc {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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
  kGated,    // rows of B are w_gate and w_up: y = act(a + b_gate) * (b + b_up), optionally a and b
  kStore,    // C rounded to the output type
  kPartial,  // C as float into the slice blockIdx.z of a workspace
};

struct GemmArgs {
  const void *a;          // [m, lda] 16-bit elements
  const void *b, *b2;     // [n, ldb]; kGated: w_gate and w_up, [n / 2, ldb] each
  int64_t m, n;           // kGated: n counts the hidden columns
  int64_t lda, ldb;       // elements of a row (all parts)
  int32_t k;              // elements along k of one part, a multiple of 8
  int32_t kslice;         // elements along k of a slice (kPartial), a multiple of the tile's
  int32_t tiles_m, tiles_n;
  void *out, *out2;       // kStore: rows from `split` on go to out2
  int64_t split;
  int64_t ldo;
  void *pre_a, *pre_b;    // kGated: a and b [m, n], or NULL
  const void *bias_a, *bias_b;
  int32_t act;
  int32_t wide;           // rows and pointers of the outputs allow stores of 16 bytes
};

// A tile of BM x BN of C for a workgroup of WM x WN waves.
template <typename T_, int PARTS_, int BM_, int BN_, int BK_, int WM_, int WN_> struct Tile {
  typedef T_ T;
  static constexpr int PARTS = PARTS_, BM = BM_, BN = BN_, BK = BK_, WM = WM_, WN = WN_;
  static constexpr int kWaves = WM * WN, kThreads = kWaves * 64;
  static constexpr int kChunks = BK / 8;                     // 16-byte chunks of a row
  static constexpr int kRowsAtOnce = 64 / kChunks;           // rows one load of a wave covers
  static constexpr int kABytes = BM * BK * 2, kBBytes = BN * BK * 2;
  static constexpr int kStage = (kABytes + kBBytes) * PARTS;
  static constexpr int kMi = BM / WM / 16, kNi = BN / WN / 16;
  // the epilogue turns a wave's results in LDS, 64 rows at a time
  static constexpr int kPitch = kNi * 16 + 4;
  static constexpr int kTurn = kWaves * 64 * kPitch * 4;
  static constexpr int kLds = 2 * kStage > kTurn ? 2 * kStage : kTurn;
  static constexpr int kALoads = BM / (kRowsAtOnce * kWaves), kBLoads = BN / (kRowsAtOnce * kWaves);
  static_assert(kALoads * kRowsAtOnce * kWaves == BM && kBLoads * kRowsAtOnce * kWaves == BN, "tile");
  static_assert((BK == 64 || BK == 32) && kMi % 4 == 0 && kNi % 2 == 0, "tile");
};

// The 16-byte chunk c of row r lies at chunk c ^ swizzle(r) of the row's place in LDS: the 16
// rows that a matrix operand's lanes read at the same c then fall on all banks evenly.
template <int BK> __device__ __forceinline__ int swizzle(int r) {
  return BK == 64 ? (r & 7) : ((r >> 1) & 3);
}

// Workgroups go to the 8 dies in turn; each die gets a run of tiles that are neighbours, in
// strips of 8 tiles along m, so that its level-2 cache serves their common rows.
__device__ __forceinline__ void tile_of(const GemmArgs &g, int &tm, int &tn) {
  const int total = g.tiles_m * g.tiles_n, id = blockIdx.x;
  const int die = id & 7, each = total >> 3, more = total & 7;
  const int at = die * each + (die < more ? die : more) + (id >> 3);
  const int strip = at / (8 * g.tiles_n), first = strip * 8;
  const int wide = g.tiles_m - first < 8 ? g.tiles_m - first : 8;
  const int in = at - strip * 8 * g.tiles_n;
  tm = first + in % wide;
  tn = in / wide;
}

typedef __attribute__((address_space(3))) void *lds_ptr;
typedef decltype(__builtin_amdgcn_make_buffer_rsrc((void *)0, (short)0, 0, 0)) rsrc_t;

template <typename C>
__device__ __forceinline__ void gemm_compute(const char *__restrict__ stage, int wm, int wn,
                                             f32x4 (&acc)[C::kNi][C::kMi]) {
  typedef typename Frag<typename C::T>::type F;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  constexpr int kRow = C::BK * 2;
#pragma unroll
  for (int kk = 0; kk < C::BK / 32; ++kk) {
    F a[C::PARTS][C::kMi], b[C::PARTS][C::kNi];
#pragma unroll
    for (int p = 0; p < C::PARTS; ++p) {
      const char *sa = stage + p * C::kABytes, *sb = stage + C::PARTS * C::kABytes + p * C::kBBytes;
#pragma unroll
      for (int j = 0; j < C::kNi; ++j) {
        const int row = wn * (C::kNi * 16) + j * 16 + r;
        b[p][j] = *reinterpret_cast<const F *>(sb + row * kRow + (((kk * 4 + q) ^ swizzle<C::BK>(r)) << 4));
      }
#pragma unroll
      for (int i = 0; i < C::kMi; ++i) {
        const int row = wm * (C::kMi * 16) + i * 16 + r;
        a[p][i] = *reinterpret_cast<const F *>(sa + row * kRow + (((kk * 4 + q) ^ swizzle<C::BK>(r)) << 4));
      }
    }
#pragma unroll
    for (int i = 0; i < C::kMi; ++i)
#pragma unroll
      for (int j = 0; j < C::kNi; ++j) {
        if constexpr (C::PARTS == 3) {
          acc[j][i] = mfma16(b[2][j], a[0][i], acc[j][i]);
          acc[j][i] = mfma16(b[0][j], a[2][i], acc[j][i]);
          acc[j][i] = mfma16(b[1][j], a[1][i], acc[j][i]);
          acc[j][i] = mfma16(b[1][j], a[0][i], acc[j][i]);
          acc[j][i] = mfma16(b[0][j], a[1][i], acc[j][i]);
        }
        acc[j][i] = mfma16(b[0][j], a[0][i], acc[j][i]);
      }
  }
}

// 8 neighbouring results of a row, of which `left` exist.
template <typename O>
__device__ __forceinline__ void store_row(O *p, const float *v, int64_t left, bool wide) {
  if (wide && left >= 8) {
    if constexpr (sizeof(O) == 4) {
      store_floats<O, 4>(p, v);
      store_floats<O, 4>(p + 4, v + 4);
    } else {
      store_floats<O, 8>(p, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (O)v[i];
  }
}

__device__ __forceinline__ void load_turned(const float *p, float *v) {
  *reinterpret_cast<f32x4 *>(v) = *reinterpret_cast<const f32x4 *>(p);
  *reinterpret_cast<f32x4 *>(v + 4) = *reinterpret_cast<const f32x4 *>(p + 4);
}

// O: type of the outputs.
template <typename C, int EPI, typename O>
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

  // A resource for every load of a wave: it spans the few rows of that load, so offsets stay
  // small however long the rows are, and rows behind the matrix read as zero.
  const int srow = lane / C::kChunks;                       // row of a load of the wave
  const int kc = ((lane % C::kChunks) ^ swizzle<C::BK>(srow)) * 8;  // (a load begins at a multiple of 8 rows)
  const int va = (int)((srow * g.lda + kc) * 2), vb = (int)((srow * g.ldb + kc) * 2);
  rsrc_t rsa[C::kALoads], rsb[C::kBLoads];
#pragma unroll
  for (int i = 0; i < C::kALoads; ++i) {
    const int64_t row = m0 + (i * C::kWaves + w) * C::kRowsAtOnce;
    const int64_t rows = g.m - row < C::kRowsAtOnce ? g.m - row : C::kRowsAtOnce;
    rsa[i] = __builtin_amdgcn_make_buffer_rsrc(
        (void *)((const char *)g.a + (rows > 0 ? row : 0) * g.lda * 2), 0,
        rows > 0 ? (int)(rows * g.lda * 2) : 0, 0x00020000);
  }
#pragma unroll
  for (int i = 0; i < C::kBLoads; ++i) {
    const int first = (i * C::kWaves + w) * C::kRowsAtOnce;
    const bool up = EPI == kGated && first % (2 * kHalf) >= kHalf;
    const int64_t row = n0 + (EPI == kGated ? first / (2 * kHalf) * kHalf + first % kHalf : first);
    const int64_t rows = g.n - row < C::kRowsAtOnce ? g.n - row : C::kRowsAtOnce;
    rsb[i] = __builtin_amdgcn_make_buffer_rsrc(
        (void *)((const char *)(up ? g.b2 : g.b) + (rows > 0 ? row : 0) * g.ldb * 2), 0,
        rows > 0 ? (int)(rows * g.ldb * 2) : 0, 0x00020000);
  }
  const int k_begin = EPI == kPartial ? (int)blockIdx.z * g.kslice : 0;
  const int k_end = EPI == kPartial && k_begin + g.kslice < g.k ? k_begin + g.kslice : g.k;

  auto issue = [&](int k0, int s) {
    char *st = lds + s * C::kStage;
    const bool in = k0 + kc < k_end;  // (what lies behind the slice counts as zero)
    const int oa = in ? va : 0x7FFFFFFF, ob = in ? vb : 0x7FFFFFFF;
#pragma unroll
    for (int p = 0; p < C::PARTS; ++p) {
      const int at = (k0 + p * g.k) * 2;
#pragma unroll
      for (int i = 0; i < C::kALoads; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsa[i], (lds_ptr)(st + p * C::kABytes + (i * C::kWaves + w) * 1024), 16, oa, at, 0, 0);
#pragma unroll
      for (int i = 0; i < C::kBLoads; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsb[i],
            (lds_ptr)(st + C::PARTS * C::kABytes + p * C::kBBytes + (i * C::kWaves + w) * 1024), 16,
            ob, at, 0, 0);
    }
  };

  f32x4 acc[C::kNi][C::kMi];
#pragma unroll
  for (int j = 0; j < C::kNi; ++j)
#pragma unroll
    for (int i = 0; i < C::kMi; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Two stages: while one is multiplied, the other one's loads are under way.
  issue(k_begin, 0);
  int s = 0;
  for (int k0 = k_begin; k0 < k_end; k0 += C::BK, s ^= 1) {
    __syncthreads();
    if (k0 + C::BK < k_end) issue(k0 + C::BK, s ^ 1);
    gemm_compute<C>(lds + s * C::kStage, wm, wn, acc);
  }
  __syncthreads();

  // A lane holds 4 neighbouring columns of row (lane & 15) in every block of 16 x 16.  Turned in
  // LDS, a lane gets 8 neighbouring columns of a row: stores of 16 bytes.
  float *turn = reinterpret_cast<float *>(lds) + w * (64 * C::kPitch);
  const bool wide = g.wide != 0;
#pragma unroll
  for (int h = 0; h < C::kMi / 4; ++h) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < C::kNi; ++j)
        *reinterpret_cast<f32x4 *>(turn + (i * 16 + (lane & 15)) * C::kPitch + j * 16 +
                                   (lane >> 4) * 4) = acc[j][h * 4 + i];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    constexpr int kAcross = (EPI == kGated ? kHalf : C::kNi * 16) / 8;  // lanes of a row
    const int64_t col = n0 + wn * (kAcross * 8) + lane % kAcross * 8;
    const int64_t left = g.n - col;
    if (left > 0) {
#pragma unroll 1
      for (int r = lane / kAcross; r < 64; r += 64 / kAcross) {
        const int64_t row = m0 + wm * (C::kMi * 16) + h * 64 + r;
        if (row >= g.m) break;
        const float *from = turn + r * C::kPitch + lane % kAcross * 8;
        float a[8];
        load_turned(from, a);
        if constexpr (EPI == kGated) {
          float b[8], f[8];
          load_turned(from + kHalf, b);
          if (g.bias_a != nullptr)
            for (int e = 0; e < 8 && e < left; ++e) a[e] += (float)static_cast<const O *>(g.bias_a)[col + e];
          if (g.bias_b != nullptr)
            for (int e = 0; e < 8 && e < left; ++e) b[e] += (float)static_cast<const O *>(g.bias_b)[col + e];
          if (g.pre_a != nullptr) {
            store_row<O>(static_cast<O *>(g.pre_a) + row * g.ldo + col, a, left, wide);
            store_row<O>(static_cast<O *>(g.pre_b) + row * g.ldo + col, b, left, wide);
          }
          activate<8>(g.act, a, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= b[e];
          store_row<O>(static_cast<O *>(g.out) + row * g.ldo + col, f, left, wide);
        } else {
          O *y;
          if (EPI == kPartial) y = static_cast<O *>(g.out) + ((int64_t)blockIdx.z * g.m + row) * g.ldo;
          else if (row >= g.split) y = static_cast<O *>(g.out2) + (row - g.split) * g.ldo;
          else y = static_cast<O *>(g.out) + row * g.ldo;
          store_row<O>(y + col, a, left, wide);
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
