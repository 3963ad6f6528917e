// Gated feed-forward block: y = act(x w_gate^T + b_gate) * (x w_up^T + b_up), and its gradients.
//
// With a = x w_gate^T + b_gate, b = x w_up^T + b_up:
//   db = dy act(a), da = dy b act'(a)
//   dx = da w_gate + db w_up, dw_gate = da^T x, dw_up = db^T x, db_gate, db_up = column sums.
//
// Forward: one launch of the matrix kernel (gated_gemm.h) whose tiles hold the same columns of
// both projections, so activation and product happen in registers and neither projection goes
// through memory (a training step keeps a and b, in 24 or 32 bits, for the backward pass); for few
// rows a kernel that streams the weights from memory into the matrix instructions.  Backward: one
// pass makes da and db, side by side, then one product gives dx (k runs over both projections'
// columns) and one gives both weight gradients (k runs over the rows, cut into slices where there
// are few tiles; slices are added in order).
//
// Many rows: bound by the matrix instructions, at the clock that the power limit leaves (1.75 to
// 1.95 GHz here): 16384 rows of 2048 -> 8192 in bfloat16, forward with a and b kept 960 to 1080 us
// (1020 to 1150 TFLOP/s), da and db 320 us (4.9 TB/s), dx 880 us (1250 TFLOP/s), weight gradients
// 820 us (1340), where torch's library products of these shapes reach 1390 and 1200.  Few rows: bound
// by the weights' bytes.  Floats: six matrix instructions for one, 57304 rows of 128 -> 512 forward
// 182 us (bound by storing a, b and y), da and db 113, dx 98, weight gradients 96 + 7.
#include "gated_gemm.h"

namespace ssc {
namespace {

// ---- operands of the matrix kernel ----------------------------------------------------------
// 8 neighbouring elements of an array of the kernels' own.
template <typename T> __device__ __forceinline__ void put_eight(T *to, const float *v) {
  constexpr int V = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8; i += V) store_floats<T, V>(to + i, v + i);
}

// src [rows, cols] -> dst [rows][padded], of three matrices in one launch: for rows of 16-bit elements
// that are no multiple of 16 bytes.
template <typename T> struct PackArgs {
  const T *src[3];
  T *dst[3];
  int64_t end[3];  // chunks of 8 columns up to and with this matrix
  int64_t cols, padded;
};
template <typename T>
__global__ void __launch_bounds__(256) pack_rows_kernel(const PackArgs<T> p) {
  const int64_t chunks = p.padded / 8;
  int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= p.end[2]) return;
  const int which = at < p.end[0] ? 0 : at < p.end[1] ? 1 : 2;
  if (which > 0) at -= p.end[which - 1];
  const int64_t r = at / chunks, c = (at - r * chunks) * 8;
  const T *src = p.src[which] + r * p.cols + c;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = c + i < p.cols ? (float)src[i] : 0.f;
  put_eight<T>(p.dst[which] + r * p.padded + c, v);
}

// da and db, rounded to T: g [m][2 hp], da at 0 .., db at hp .., zeros behind h; and the column sums
// of every `rows` rows, sums [tiles of rows][2 h] (NULL: not wanted).  8 neighbouring columns of a row
// to a thread; ALIGNED: rows begin at 16 bytes.  HBM-bound; its inputs are read for the last time and
// need no place in the caches (16384 x 8192 in bfloat16 380 -> 320 us).
constexpr int kGradAcross = 32;  // threads side by side
// Rows of a workgroup: 64, or 16 where that leaves too few workgroups.
int grad_rows(int64_t m, int64_t hp) {
  return ceil_div(m, 64) * ceil_div(hp, kGradAcross * 8) >= 512 ? 64 : 16;
}
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256)
    gated_grad_kernel(const T *__restrict__ dy, const void *__restrict__ ab, int64_t m, int64_t h, int act,
                      int64_t hp, int rows, T *__restrict__ g, float *__restrict__ sums) {
  const Kept<T> kept(ab, m, h);
  constexpr int kDown = 256 / kGradAcross;
  __shared__ float lds[kDown][kGradAcross * 8 + 1];
  const int cx = threadIdx.x % kGradAcross, row = threadIdx.x / kGradAcross;
  const int64_t c = ((int64_t)blockIdx.y * kGradAcross + cx) * 8, r0 = (int64_t)blockIdx.x * rows;
  float sa[8], sb[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sa[i] = sb[i] = 0.f;
  if (c < hp) {
#pragma unroll 2
    for (int64_t r = r0 + row; r < r0 + rows; r += kDown) {
      if (r >= m) break;
      float yv[8], av[8], bv[8], f[8], d[8];
      const int64_t at = r * h + c;
      if (ALIGNED && c < h) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += V) load_floats_once<T, V>(dy + at + i, yv + i);
        kept.template get<true>(0, at, 8, av);
        kept.template get<true>(1, at, 8, bv);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) yv[i] = c + i < h ? (float)dy[at + i] : 0.f;
        kept.template get<false>(0, at, h - c, av);
        kept.template get<false>(1, at, h - c, bv);
      }
      activate_slope<8>(act, av, f, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        av[i] = yv[i] * bv[i] * d[i];
        bv[i] = yv[i] * f[i];
        sa[i] += av[i];
        sb[i] += bv[i];
      }
      put_eight<T>(g + r * 2 * hp + c, av);
      put_eight<T>(g + r * 2 * hp + hp + c, bv);
    }
  }
  if (sums == nullptr) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) lds[row][cx * 8 + i] = which == 0 ? sa[i] : sb[i];
    __syncthreads();
    const int64_t col = (int64_t)blockIdx.y * kGradAcross * 8 + threadIdx.x;
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < kDown; ++r) s += lds[r][threadIdx.x];
    if (col < h) sums[(int64_t)blockIdx.x * 2 * h + which * h + col] = s;
  }
}

// Column sums of the row tiles, added in order: 16 columns of a workgroup, 16 runs of tiles.
template <typename T>
__global__ void __launch_bounds__(256)
    bias_grad_kernel(const float *__restrict__ sums, int64_t tiles, int64_t h, T *__restrict__ db_gate,
                     T *__restrict__ db_up) {
  __shared__ float t[16][16];
  const int x = threadIdx.x & 15, run = threadIdx.x >> 4;
  const int64_t c = (int64_t)blockIdx.x * 16 + x;
  float s = 0.f;
  if (c < 2 * h) {
#pragma unroll 8
    for (int64_t r = run; r < tiles; r += 16) s += sums[r * 2 * h + c];
  }
  t[run][x] = s;
  __syncthreads();
  if (run == 0 && c < 2 * h) {
#pragma unroll
    for (int r = 1; r < 16; ++r) s += t[r][x];
    if (c < h) {
      if (db_gate) db_gate[c] = (T)s;
    } else if (db_up) {
      db_up[c - h] = (T)s;
    }
  }
}

// Slices of a product added in order, rounded once: 4 neighbouring results of a thread where their
// number allows it (V = 4), several slices' loads under way at a time.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    add_slices_kernel(const float *__restrict__ part, int slices, int64_t count, int64_t split,
                      T *__restrict__ out, T *__restrict__ out2) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (i >= count) return;
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.f;
#pragma unroll 8
  for (int z = 0; z < slices; ++z) {
    float v[V];
    load_floats_once<float, V>(part + z * count + i, v);
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] += v[e];
  }
  store_floats<T, V>(i < split ? out + i : out2 + (i - split), s);
}

// ---- few rows -------------------------------------------------------------------------------
// 16 hidden columns of both projections, 16 MT rows; the waves of the workgroup take the steps along
// k in turn and are added up in LDS.  Bound by the weights' bytes up to some 32 rows (one row through
// 4096 -> 8192 in bfloat16: 27 us, 5.0 TB/s; 32 rows 34 us), by the matrix units' waiting for them
// beyond: a lane reads 32 neighbouring bytes of a row of the weights at a step, and rows (16 lanes)
// and steps are independent, so many loads are in flight.  k is dealt to the lanes as the weights
// lie in memory, not in the matrix instruction's own order: a sum does not mind as long as x is
// dealt alike.  Float elements go to float matrix instructions as they are, at 1/16 of the rate of
// 16-bit ones, so what is multiplied shall not wait for what is loaded: a step ahead 4096 -> 8192 one
// row 63 -> 54 us, 16 rows 72 -> 57, 20 rows 81 -> 77 (but 64 rows, at half the waves by their registers,
// 131 -> 140; 16-bit elements gain nothing by it).
template <typename T> struct FewStep;  // one step: 64 elements along k (16 bits), 32 (float)
template <> struct FewStep<f16> { static constexpr int kLane = 16; };
template <> struct FewStep<bf16> { static constexpr int kLane = 16; };
template <> struct FewStep<float> { static constexpr int kLane = 8; };

// kLane elements from p, of which `left` exist (the rest count as zero).
template <typename T, bool ALIGNED>
__device__ __forceinline__ void few_load(const T *p, int64_t left, T *v) {
  constexpr int L = FewStep<T>::kLane, V = 16 / sizeof(T);
  if constexpr (ALIGNED) {
#pragma unroll
    for (int i = 0; i < L; i += V) {
      typename Pack<T, V>::type c = {};
      if (i < left) c = *reinterpret_cast<const typename Pack<T, V>::type *>(p + i);
#pragma unroll
      for (int e = 0; e < V; ++e) v[i + e] = c[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < L; ++i) v[i] = i < left ? p[i] : (T)0.f;
  }
}

__device__ __forceinline__ void few_mul(const float *w, const float *x, f32x4 &acc) {
#pragma unroll
  for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i], x[i], acc, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ void few_mul(const T *w, const T *x, f32x4 &acc) {
  typedef typename Frag<T>::type F;
#pragma unroll
  for (int i = 0; i < 16; i += 8) {
    F wf, xf;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      wf[e] = w[i + e];
      xf[e] = x[i + e];
    }
    acc = mfma16(wf, xf, acc);
  }
}

template <typename T, int MT, bool ALIGNED>
__global__ void __launch_bounds__(512) few_rows_kernel(const GemmArgs g) {
  constexpr int L = FewStep<T>::kLane, W = 8;
  __shared__ f32x4 lds[W][2 * MT][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t col = n0 + r < g.n ? n0 + r : g.n - 1, m0 = (int64_t)blockIdx.y * 16 * MT;
  const T *wg = static_cast<const T *>(g.b.p) + col * g.b.ld, *wu = static_cast<const T *>(g.b.q) + col * g.b.ld;
  const T *x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    x[t] = static_cast<const T *>(g.a.p) + (m0 + t * 16 + r < g.m ? m0 + t * 16 + r : g.m - 1) * g.a.ld;
  f32x4 acc[2 * MT];
#pragma unroll
  for (int t = 0; t < 2 * MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // A step's elements, `left` of each row's existing; floats in up to 32 rows are loaded one step ahead.
  struct Step {
    T gate[L], up[L], x[MT][L];
  };
  auto load = [&](Step &s, int k1, int64_t left) {
    const int k = k1 + q * L;
    few_load<T, ALIGNED>(wg + k, left - q * L, s.gate);
    few_load<T, ALIGNED>(wu + k, left - q * L, s.up);
#pragma unroll
    for (int t = 0; t < MT; ++t) few_load<T, ALIGNED>(x[t] + k, left - q * L, s.x[t]);
  };
  auto mul = [&](const Step &s) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      few_mul(s.gate, s.x[t], acc[2 * t]);
      few_mul(s.up, s.x[t], acc[2 * t + 1]);
    }
  };
  constexpr int kStep = 4 * L, kNext = W * kStep;
  constexpr bool kAhead = sizeof(T) == 4 && MT <= 2;
  int k0 = w * kStep;
  if constexpr (kAhead) {
    Step s0, s1;
    if (k0 + kStep <= g.k) load(s0, k0, kStep);
    while (k0 + kStep <= g.k) {
      if (k0 + kNext + kStep <= g.k) load(s1, k0 + kNext, kStep);
      mul(s0);
      k0 += kNext;
      if (k0 + kStep > g.k) break;
      if (k0 + kNext + kStep <= g.k) load(s0, k0 + kNext, kStep);
      mul(s1);
      k0 += kNext;
    }
  } else {
#pragma unroll 2
    for (; k0 + kStep <= g.k; k0 += kNext) {
      Step s;
      load(s, k0, kStep);
      mul(s);
    }
  }
  if (k0 < g.k) {
    Step s;
    load(s, k0, g.k - k0);
    mul(s);
  }
#pragma unroll
  for (int t = 0; t < 2 * MT; ++t) lds[w][t][lane] = acc[t];
  __syncthreads();
  if (w >= MT) return;
  f32x4 sa = lds[0][2 * w][lane], sb = lds[0][2 * w + 1][lane];
#pragma unroll
  for (int v = 1; v < W; ++v) {
    sa += lds[v][2 * w][lane];
    sb += lds[v][2 * w + 1][lane];
  }
  const int64_t row = m0 + w * 16 + r, c0 = n0 + q * 4;
  if (row >= g.m) return;
  float a[4], b[4], f[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool in = c0 + e < g.n;
    a[e] = sa[e] + (g.bias_a && in ? (float)static_cast<const T *>(g.bias_a)[c0 + e] : 0.f);
    b[e] = sb[e] + (g.bias_b && in ? (float)static_cast<const T *>(g.bias_b)[c0 + e] : 0.f);
  }
  activate<4>(g.act, a, f);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c0 + e < g.n) {
      const int64_t at = row * g.ldo + c0 + e;
      static_cast<T *>(g.out)[at] = (T)(f[e] * b[e]);
      if (g.kept) {
        const Kept<T> kept(g.kept, g.m, g.n);
        kept.template put<false>(0, at, a + e, 1, false);
        kept.template put<false>(1, at, b + e, 1, false);
      }
    }
}

// ---- host -----------------------------------------------------------------------------------
int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }
bool at16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Tiles: large ones reuse more of what they read, small ones fill the chip where there are few, and
// several of them share a CU, so that one's results are stored while another one multiplies.
template <typename T> struct Tiles {
  typedef Tile<T, 1, 256, 256, 64, 4, 2> Large;
  typedef Tile<T, 1, 128, 128, 64, 2, 2> Middle;
  typedef Tile<T, 1, 64, 128, 64, 1, 4> Small;
};
template <> struct Tiles<float> {
  typedef Tile<bf16, 3, 256, 128, 32, 4, 2> Large;
  typedef Tile<bf16, 3, 64, 128, 32, 1, 4> Middle, Small;
};
constexpr int kCUs = 256;

template <typename C> int64_t tiles_of(int64_t m, int64_t n) {
  return ceil_div(m, C::BM) * ceil_div(n, C::BN);
}

struct Shape {
  int64_t m, n, k;
};

// Slices along k of a product with too few tiles to fill the chip, as many workgroups in all as fit on
// it at a time; at least 8 steps each, or the launch that adds them up costs more than they save.
template <typename C> int slices_of(const Shape &s) {
  const int64_t tiles = tiles_of<C>(s.m, s.n), steps = ceil_div(s.k, C::BK);
  int64_t z = tiles >= kCUs * 3 / 4 ? 1 : (C::kLds > 80 * 1024 ? 1 : 2) * kCUs / tiles;
  if (z > steps / 8) z = steps / 8;
  if (z < 1) z = 1;
  return (int)ceil_div(steps, ceil_div(steps, z));
}
// 2: large tiles, 1: middle ones, 0: small ones (float: large or small).
//
// Forward: large tiles where they fill the chip, unless both projections are kept and k is short:
// storing takes longer than multiplying then, and a CU holds only one large tile.  25600 rows ->
// 1024, kept, bfloat16, large against middle tiles: k = 128 73 and 66 us, 256 82 and 81, 512 105 and
// 110; 25437 -> 808, k = 128, float16 118 and 61.  Floats, large against small: 25600 -> 1024 kept,
// k = 64 133 and 135, 128 156 and 164; 4096 -> 4096 kept, k = 64 101 and 68, 256 143 and 145.
template <typename T> int forward_size(const Shape &s, bool kept) {
  const bool stores = kept && s.k <= (sizeof(T) == 4 ? 64 : 384);
  if (tiles_of<typename Tiles<T>::Large>(s.m, s.n) >= kCUs && !stores) return 2;
  return tiles_of<typename Tiles<T>::Middle>(s.m, s.n) >= kCUs ? 1 : 0;
}
// The products of the backward pass are sliced where tiles are few, so they fill the chip with any
// of them; the tile's reuse counts for more the longer the product takes (times with the pass that
// makes da and db).  bfloat16, large, middle, small: 25600 x 2048 (k) x 2048 293, 363, 377 us; 25600 x
// 1024 (k) x 2048 207, 203, 283; 16384 x 512 (k) x 2048 101, 74, 78; 1024 x 2048 (k) x 2048 49, 45, 38.
// Floats, large and small: 57304 x 1024 (k) x 128 203 and 226; 16384 x 512 (k) x 256 60 and 53; 1024 x
// 2048 (k) x 1024 47 and 46; 300 x 8192 (k) x 2048 99 and 92.
template <typename T> int product_size(const Shape &s) {
  const double work = (double)s.m * s.n * s.k;
  if (tiles_of<typename Tiles<T>::Large>(s.m, s.n) >= kCUs * 3 / 4) return 2;
  if (work >= (sizeof(T) == 4 ? 5.5e9 : 8e10)) return 2;
  return tiles_of<typename Tiles<T>::Middle>(s.m, s.n) >= kCUs || work >= 1.2e10 ? 1 : 0;
}
template <typename T> int slices_for(const Shape &s) {
  const int z = product_size<T>(s);
  return z == 2 ? slices_of<typename Tiles<T>::Large>(s)
                : z == 1 ? slices_of<typename Tiles<T>::Middle>(s) : slices_of<typename Tiles<T>::Small>(s);
}

template <typename C, bool TA, bool TB, int EPI, typename O>
int launch(GemmArgs g, int64_t n_tile, int slices, hipStream_t s) {
  g.tiles_m = (int32_t)ceil_div(g.m, C::BM);
  g.tiles_n = (int32_t)ceil_div(n_tile, C::BN);
  SSC_CHECK((int64_t)g.tiles_m * g.tiles_n <= 0x7FFFFFFF, SSC_EINVAL, "too many tiles");
  g.kslice = (int32_t)(ceil_div(ceil_div(g.k, C::BK), slices) * C::BK);
  hipLaunchKernelGGL((gemm_kernel<C, TA, TB, EPI, O>), dim3(g.tiles_m * g.tiles_n, 1, slices), dim3(C::kThreads),
                     0, s, g);
  SSC_LAUNCH_CHECK("gated feed-forward product");
  return SSC_OK;
}

// A product whose result goes to out and out2 (rows from `second` on), in slices where that pays.
template <typename T, bool TA, bool TB>
int product(GemmArgs g, float *part, hipStream_t s) {
  const Shape shape = {g.m, g.n, g.k};
  const int size = product_size<T>(shape), slices = slices_for<T>(shape);
  typedef Tiles<T> S;
  if (slices == 1) {
    g.wide = (g.ldo * sizeof(T)) % 16 == 0 && at16(g.out) && at16(g.out2);
    return size == 2 ? launch<typename S::Large, TA, TB, kStore, T>(g, g.n, 1, s)
                     : size == 1 ? launch<typename S::Middle, TA, TB, kStore, T>(g, g.n, 1, s)
                                 : launch<typename S::Small, TA, TB, kStore, T>(g, g.n, 1, s);
  }
  GemmArgs p = g;
  p.out = part;
  p.wide = g.ldo % 4 == 0;
  const int rc = size == 2 ? launch<typename S::Large, TA, TB, kPartial, float>(p, g.n, slices, s)
                           : size == 1 ? launch<typename S::Middle, TA, TB, kPartial, float>(p, g.n, slices, s)
                                       : launch<typename S::Small, TA, TB, kPartial, float>(p, g.n, slices, s);
  if (rc != SSC_OK) return rc;
  const int64_t split = g.each * g.n, count = g.second < g.m ? 2 * split : split;
  const bool wide = split % 4 == 0 && at16(g.out) && at16(g.out2);
  const dim3 grid((uint32_t)ceil_div(count, 256 * (wide ? 4 : 1)));
  T *out = static_cast<T *>(g.out), *out2 = static_cast<T *>(g.out2);
  if (wide) hipLaunchKernelGGL((add_slices_kernel<T, 4>), grid, dim3(256), 0, s, part, slices, count, split, out, out2);
  else hipLaunchKernelGGL((add_slices_kernel<T, 1>), grid, dim3(256), 0, s, part, slices, count, split, out, out2);
  SSC_LAUNCH_CHECK("add_slices_kernel");
  return SSC_OK;
}

// Whether the matrix kernel reads the user's rows as they are (16-bit ones begin at 16 bytes then).
template <typename T> bool reads_plain(int64_t k) { return sizeof(T) == 4 || k % 8 == 0; }

struct Problem {
  int64_t m, k, h;
};

// Whether the few-rows kernel is taken: for 16 bits up to 64 rows, or a workgroup to a CU; for
// floats, which it takes as they are where tiles want them in parts, up to two to a CU.  It
// against tiles, us: bfloat16, 1024 -> 1024, 256 rows 9.5 and 10.5, 384 rows 14.8 and 10.7; 2048 ->
// 4096, 64 rows 16 and 22, 96 rows 24 and 22; floats, 2048 -> 4096, 128 rows 56 and 65, 192 rows 85
// and 68; 1000 -> 2728, 256 rows 46 and 38; 128 -> 512, 512 rows 5.6 and 8.3.
template <typename T> bool takes_few(const Problem &p) {
  const int64_t groups = ceil_div(p.h, 16) * ceil_div(p.m, 64);
  return sizeof(T) == 4 ? groups <= 2 * kCUs : p.m <= 64 || groups <= kCUs;
}

// x and the weights as the matrix kernel reads them: as they are, or laid out anew in ws.
template <typename T> struct Rows {
  Operand x, wg, wu;
  int32_t k;  // columns
  static size_t bytes(const Problem &p) {
    if (reads_plain<T>(p.k)) return 0;
    const size_t row = up8(p.k) * sizeof(T);
    return align_up(p.m * row) + 2 * align_up(p.h * row);
  }
  int make(const Problem &p, const void *x0, const void *wg0, const void *wu0, Carver &c, hipStream_t s) {
    const bool plain = reads_plain<T>(p.k);
    k = (int32_t)(plain ? p.k : up8(p.k));
    if (plain) {
      x.p = x0;
      wg.p = wg0;
      wu.p = wu0;
    } else {
      T *xp = c.take<T>(p.m * k), *gp = c.take<T>(p.h * k), *up = c.take<T>(p.h * k);
      PackArgs<T> a;
      a.src[0] = static_cast<const T *>(x0);
      a.src[1] = static_cast<const T *>(wg0);
      a.src[2] = static_cast<const T *>(wu0);
      a.dst[0] = xp;
      a.dst[1] = gp;
      a.dst[2] = up;
      a.end[0] = p.m * (k / 8);
      a.end[1] = a.end[0] + p.h * (k / 8);
      a.end[2] = a.end[1] + p.h * (k / 8);
      a.cols = p.k;
      a.padded = k;
      hipLaunchKernelGGL(pack_rows_kernel<T>, dim3((uint32_t)ceil_div(a.end[2], 256)), dim3(256), 0, s, a);
      SSC_LAUNCH_CHECK("pack_rows_kernel");
      x.p = xp;
      wg.p = gp;
      wu.p = up;
    }
    x.ld = wg.ld = wu.ld = k;
    x.second = wg.second = wu.second = 0x7FFFFFFF;
    return SSC_OK;
  }
};

template <typename T> size_t forward_bytes(const Problem &p) {
  return takes_few<T>(p) ? 256 : 256 + Rows<T>::bytes(p);
}

// Rows in as few blocks of at most 64 as there are, of 16 MT rows each, no more than they need: 48 rows
// in a block of 48 rather than 64 2048 -> 4096 floats 35 -> 29 us, bfloat16 16.1 -> 15.0.
template <typename T, bool ALIGNED> void few_rows(const GemmArgs &g, hipStream_t s) {
  const int64_t mt = ceil_div(ceil_div(g.m, ceil_div(g.m, 64)), 16);
  const dim3 grid((uint32_t)ceil_div(g.n, 16), (uint32_t)ceil_div(g.m, 16 * mt));
  if (mt == 1) hipLaunchKernelGGL((few_rows_kernel<T, 1, ALIGNED>), grid, dim3(512), 0, s, g);
  else if (mt == 2) hipLaunchKernelGGL((few_rows_kernel<T, 2, ALIGNED>), grid, dim3(512), 0, s, g);
  else if (mt == 3) hipLaunchKernelGGL((few_rows_kernel<T, 3, ALIGNED>), grid, dim3(512), 0, s, g);
  else hipLaunchKernelGGL((few_rows_kernel<T, 4, ALIGNED>), grid, dim3(512), 0, s, g);
}

template <typename T>
int forward(const Problem &p, const void *x, const void *wg, const void *wu, const void *bg,
            const void *bu, int act, void *y, void *kept, void *ws, hipStream_t s) {
  GemmArgs g = {};
  g.m = p.m;
  g.n = p.h;
  g.bias_a = bg;
  g.bias_b = bu;
  g.act = act;
  g.out = y;
  g.kept = kept;
  g.ldo = p.h;
  if (takes_few<T>(p)) {
    g.a.p = x;
    g.b.p = wg;
    g.b.q = wu;
    g.k = (int32_t)p.k;
    g.a.ld = g.b.ld = p.k;
    const bool aligned = (p.k * sizeof(T)) % 16 == 0 && at16(x) && at16(wg) && at16(wu);
    if (aligned) few_rows<T, true>(g, s);
    else few_rows<T, false>(g, s);
    SSC_LAUNCH_CHECK("few_rows_kernel");
    return SSC_OK;
  }
  Carver c(ws);
  Rows<T> rows = {};
  const int rc = rows.make(p, x, wg, wu, c, s);
  if (rc != SSC_OK) return rc;
  g.k = rows.k;
  g.a = rows.x;
  g.a.rows = p.m;
  g.b = rows.wg;
  g.b.q = rows.wu.p;
  g.b.rows = p.h;
  g.wide = (p.h * sizeof(T)) % 16 == 0 && at16(y);
  const int size = forward_size<T>({p.m, 2 * p.h, g.k}, kept != nullptr);
  typedef Tiles<T> S;
  return size == 2 ? launch<typename S::Large, false, false, kGated, T>(g, 2 * p.h, 1, s)
                   : size == 1 ? launch<typename S::Middle, false, false, kGated, T>(g, 2 * p.h, 1, s)
                               : launch<typename S::Small, false, false, kGated, T>(g, 2 * p.h, 1, s);
}

template <typename T> struct Backward {
  int64_t hp;  // columns of da and of db in g: a multiple of every tile's k
  int rows;    // of a workgroup of the pass that makes g
  T *g;
  float *sums, *part;
  size_t used;
  Backward(const Problem &p, void *ws) {
    hp = ceil_div(p.h, 64) * 64;
    Carver c(ws);
    g = c.take<T>(p.m * 2 * hp);
    rows = grad_rows(p.m, hp);
    sums = c.take<float>(ceil_div(p.m, rows) * 2 * p.h);
    // the slices of the two products, one after the other
    const int zx = slices_for<T>(dx_shape(p)), zw = slices_for<T>(dw_shape(p));
    const int64_t px = zx > 1 ? zx * p.m * p.k : 0, pw = zw > 1 ? zw * 2 * p.h * p.k : 0;
    part = c.take<float>(px > pw ? px : pw);
    used = c.used;
  }
  Shape dx_shape(const Problem &p) const { return {p.m, p.k, 2 * hp}; }
  Shape dw_shape(const Problem &p) const { return {2 * hp, p.k, p.m}; }
  static size_t bytes(const Problem &p) { return Backward(p, nullptr).used + Rows<T>::bytes(p); }
};

template <typename T>
int backward(const Problem &p, const void *x, const void *wg, const void *wu, int act, const void *kept,
             const void *dy, void *dx, void *dwg, void *dwu, void *dbg, void *dbu,
             void *ws, hipStream_t s) {
  const Backward<T> w(p, ws);
  const bool biases = dbg != nullptr || dbu != nullptr;
  const dim3 tiles((uint32_t)ceil_div(p.m, w.rows), (uint32_t)ceil_div(w.hp, kGradAcross * 8));
  const bool aligned = (p.h % 8) == 0 && at16(dy);
#define SSC_GRAD(ALIGNED)                                                                              \
  hipLaunchKernelGGL((gated_grad_kernel<T, ALIGNED>), tiles, dim3(256), 0, s, static_cast<const T *>(dy), \
                     kept, p.m, p.h, act, w.hp, w.rows, w.g, \
                     biases ? w.sums : nullptr)
  if (aligned) SSC_GRAD(true);
  else SSC_GRAD(false);
#undef SSC_GRAD
  SSC_LAUNCH_CHECK("gated_grad_kernel");
  if (biases) {
    hipLaunchKernelGGL(bias_grad_kernel<T>, dim3((uint32_t)ceil_div(2 * p.h, 16)), dim3(256), 0, s, w.sums,
                       ceil_div(p.m, w.rows), p.h, static_cast<T *>(dbg), static_cast<T *>(dbu));
    SSC_LAUNCH_CHECK("bias_grad_kernel");
  }
  if (dx == nullptr && dwg == nullptr) return SSC_OK;
  Carver c(static_cast<char *>(ws) + w.used);
  Rows<T> rows = {};
  int rc = rows.make(p, x, wg, wu, c, s);
  if (rc != SSC_OK) return rc;
  Operand grad = {};
  grad.p = w.g;
  grad.ld = 2 * w.hp;
  grad.second = 0x7FFFFFFF;
  GemmArgs g = {};
  g.n = p.k;
  g.ldo = p.k;
  if (dx) {
    g.a = grad;
    g.a.rows = p.m;
    g.b = rows.wg;
    g.b.q = rows.wu.p;
    g.b.rows = rows.k;
    g.b.second = (int32_t)w.hp;
    g.b.deep = (int32_t)p.h;
    g.m = p.m;
    g.k = (int32_t)(2 * w.hp);
    g.out = dx;
    g.second = g.each = p.m;
    rc = product<T, false, true>(g, w.part, s);
    if (rc != SSC_OK) return rc;
  }
  if (dwg) {
    g.a = grad;
    g.a.rows = 2 * w.hp;
    g.a.deep = (int32_t)p.m;
    g.b = rows.x;
    g.b.rows = rows.k;
    g.b.deep = (int32_t)p.m;
    g.m = 2 * w.hp;
    g.k = (int32_t)p.m;
    g.out = dwg;
    g.out2 = dwu;
    g.second = w.hp;
    g.each = p.h;
    rc = product<T, true, true>(g, w.part, s);
  }
  return rc;
}

// What 32-bit offsets inside a few rows allow.
constexpr int64_t kMostAlong = 1 << 24;

int check(int32_t dtype, int64_t m, int64_t k, int64_t h, int32_t act, const void *x, const void *wg,
          const void *wu) {
  SSC_CHECK(dtype_ok(dtype), SSC_EINVAL, "element type %d", dtype);
  SSC_CHECK(m >= 0 && k >= 1 && h >= 1, SSC_EINVAL, "%lld rows, widths %lld and %lld", (long long)m,
            (long long)k, (long long)h);
  SSC_CHECK(m <= kMostAlong && k <= kMostAlong / 8 && h <= kMostAlong / 8, SSC_EINVAL,
            "%lld rows, widths %lld and %lld: at most %lld and %lld", (long long)m, (long long)k,
            (long long)h, (long long)kMostAlong, (long long)(kMostAlong / 8));
  SSC_CHECK(pointwise_act_ok(act), SSC_EINVAL, "activation %d", act);
  SSC_CHECK(m == 0 || (x && wg && wu), SSC_EINVAL, "NULL pointer");
  SSC_CHECK(m == 0 || dtype == SSC_F32 || k % 8 != 0 || (at16(x) && at16(wg) && at16(wu)), SSC_EINVAL,
            "x and the weights begin at 16 bytes where their rows are multiples of 16 bytes");
  return SSC_OK;
}

}  // namespace
}  // namespace ssc

using namespace ssc;

extern "C" size_t ssc_gated_fwd_workspace_bytes(int32_t dtype, int64_t m, int64_t k, int64_t h) {
  if (m <= 0 || k <= 0 || h <= 0) return 256;  // (the calls refuse all but no rows)
  const Problem p = {m, k, h};
  return dtype == SSC_F32 ? forward_bytes<float>(p) : forward_bytes<f16>(p);
}

extern "C" size_t ssc_gated_kept_bytes(int32_t dtype, int64_t m, int64_t h) {
  if (m <= 0 || h <= 0) return 16;
  const size_t bytes = dtype == SSC_F32 ? Kept<float>::bytes(m, h) : Kept<f16>::bytes(m, h);
  return bytes;
}

extern "C" int ssc_gated_fwd(int32_t dtype, const void *x, int64_t m, int64_t k, const void *w_gate,
                             const void *w_up, int64_t h, const void *b_gate, const void *b_up,
                             int32_t act, void *y, void *kept, void *ws, size_t ws_bytes,
                             ssc_stream_t stream) {
  const int rc = check(dtype, m, k, h, act, x, w_gate, w_up);
  if (rc != SSC_OK) return rc;
  if (m == 0) return SSC_OK;
  SSC_CHECK(y, SSC_EINVAL, "NULL pointer");
  SSC_CHECK(at16(kept), SSC_EINVAL, "what is kept begins at 16 bytes");
  SSC_CHECK(ws != nullptr && ws_bytes >= ssc_gated_fwd_workspace_bytes(dtype, m, k, h), SSC_EWORKSPACE,
            "workspace of %zu bytes, %zu are needed", ws_bytes,
            ssc_gated_fwd_workspace_bytes(dtype, m, k, h));
  const Problem p = {m, k, h};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == SSC_F32) return forward<float>(p, x, w_gate, w_up, b_gate, b_up, act, y, kept, ws, s);
  if (dtype == SSC_F16) return forward<f16>(p, x, w_gate, w_up, b_gate, b_up, act, y, kept, ws, s);
  return forward<bf16>(p, x, w_gate, w_up, b_gate, b_up, act, y, kept, ws, s);
}

extern "C" size_t ssc_gated_bwd_workspace_bytes(int32_t dtype, int64_t m, int64_t k, int64_t h) {
  if (m <= 0 || k <= 0 || h <= 0) return 256;
  const Problem p = {m, k, h};
  return dtype == SSC_F32 ? Backward<float>::bytes(p) : Backward<f16>::bytes(p);
}

extern "C" int ssc_gated_bwd(int32_t dtype, const void *x, int64_t m, int64_t k, const void *w_gate,
                             const void *w_up, int64_t h, int32_t act, const void *kept, const void *dy,
                             void *dx, void *dw_gate, void *dw_up, void *db_gate, void *db_up, void *ws,
                             size_t ws_bytes, ssc_stream_t stream) {
  const int rc = check(dtype, m, k, h, act, x, w_gate, w_up);
  if (rc != SSC_OK) return rc;
  if (m == 0) return SSC_OK;
  SSC_CHECK(kept && dy && (dw_gate == nullptr) == (dw_up == nullptr), SSC_EINVAL,
            "NULL pointer");
  SSC_CHECK(at16(kept), SSC_EINVAL, "what is kept begins at 16 bytes");
  SSC_CHECK(ws != nullptr && ws_bytes >= ssc_gated_bwd_workspace_bytes(dtype, m, k, h), SSC_EWORKSPACE,
            "workspace of %zu bytes, %zu are needed", ws_bytes,
            ssc_gated_bwd_workspace_bytes(dtype, m, k, h));
  const Problem p = {m, k, h};
  hipStream_t s = static_cast<hipStream_t>(stream);
#define SSC_GATED_BWD(T) \
  backward<T>(p, x, w_gate, w_up, act, kept, dy, dx, dw_gate, dw_up, db_gate, db_up, ws, s)
  return dtype == SSC_F32 ? SSC_GATED_BWD(float) : dtype == SSC_F16 ? SSC_GATED_BWD(f16) : SSC_GATED_BWD(bf16);
#undef SSC_GATED_BWD
}
