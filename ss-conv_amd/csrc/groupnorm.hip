// Group norm with an activation over rows [n, c], channels last, rows grouped by cloud.
//
// Cloud b, group g (c / groups neighbouring channels), m = rows(b) * c / groups values:
//   mean, var = E[(x - mean)^2], rstd = 1 / sqrt(var + eps), h = (x - mean) rstd,
//   z = weight h + bias, y = f(z)
// and with dz = dy f'(z)
//   dbias = sum dz, dweight = sum dz h, S1 = sum over the group of weight dz, S2 = of weight dz h
//   dx = rstd (weight dz - (S1 + h S2) / m).
//
// HBM-bound: x has to be read before the first y can be written, so a pass takes the sums and
// another one applies them.  Rows are cut into chunks of equal length whatever the clouds are; a
// chunk that spans a boundary holds one piece of each cloud, and the partial result of cloud b's
// piece in chunk k goes to slot k + b: along the rows each next piece moves k or b by at least
// one, so no two pieces share a slot and no table of pieces is needed.
//
// The second pass takes the chunks from the last one on, reads its inputs for the last time and
// writes past the caches: what the first pass read last is then still in the 256 MB of the last
// cache level.  600153 x 128 floats, forward and backward: 519 us with both passes in order, 492 with
// the second one reversed, 436 with writes and last reads past the caches as well, 428 with half as
// many chunks (an x of 307 MB moves 2.46 GB, 476 us at the 5.16 TB/s of a large copy, if no cache
// helps).
//
// The variance comes from deviations, not from E[x^2] - mean^2: a thread sums x - x0 and
// (x - x0)^2 with its own first value x0 of the channel, which leaves numbers of the spread's
// size, and partial results (count, mean, sum of squared deviations) are joined by
// M = M1 + M2 + (mean2 - mean1)^2 n1 n2 / (n1 + n2).  Every order is fixed: results are
// reproducible.
#include "elem.h"

namespace ssc {
namespace {

constexpr int kThreads = 256;
// Chunks of rows: four workgroups for each of 256 CUs.  More of them pay for finding their cloud and for
// adding up too often: forward and backward with 2048, 1024 and 512 chunks 50001 x 200 float16 76, 67
// and 70 us, 100000 x 64 bfloat16 69, 61 and 57, 600153 x 128 floats 437, 432 and 451.
constexpr int kChunksMost = 1024;

struct Norm {
  const void *x, *dy;
  void *out;                 // y or dx
  const int32_t *offsets;    // [clouds + 1]
  const void *weight, *bias;  // [c] or NULL
  float *mean, *rstd;        // [clouds, groups]
  float2 *partial;           // [chunks + clouds, c]
  float2 *sums;              // [clouds, c]: sum dz, sum dz h
  float2 *group;             // [clouds, groups]: S1 / m, S2 / m
  void *dweight, *dbias;     // [c] or NULL
  int64_t n;
  int32_t c, clouds, groups, per, wtype, act, rows;  // rows: of a chunk
  int32_t chunks;
  int32_t first;             // a launch with a workgroup to a cloud's group: the first one's number
  float eps;
};

// Rows of cloud b: they begin at 0 and end at n whatever the first and last offset say, and
// never lie outside the rows.
__device__ __forceinline__ int64_t cloud_begin(const Norm &a, int b) {
  if (b <= 0) return 0;
  if (b >= a.clouds) return a.n;
  const int64_t o = a.offsets[b];
  return o < 0 ? 0 : o > a.n ? a.n : o;
}

// The first cloud that ends behind row r.
__device__ __forceinline__ int cloud_of(const Norm &a, int64_t r) {
  int lo = 0, hi = a.clouds - 1;  // the answer is in lo .. hi
  while (hi - lo > 63) {
    const int mid = (lo + hi) >> 1;
    if (cloud_begin(a, mid + 1) > r) hi = mid;
    else lo = mid + 1;
  }
  const int i = lo + (int)(threadIdx.x & 63);
  const int below = __popcll(__ballot(i < hi && cloud_begin(a, i + 1) <= r));
  return __builtin_amdgcn_readfirstlane(lo + below);
}

// How the threads of a workgroup lie on rows and channels: `tx` threads of V channels side by
// side, `ty` rows at a time, column tile blockIdx.y.
template <int V> struct Lay {
  int tx, ty, cx, row;
  int64_t ch;
  bool in;
  __device__ Lay(const Norm &a) {
    const int cv = a.c / V;
    tx = cv < kThreads ? cv : kThreads;
    ty = kThreads / tx;
    row = (int)threadIdx.x / tx;
    cx = (int)threadIdx.x - row * tx;
    ch = ((int64_t)blockIdx.y * tx + cx) * V;
    in = row < ty && ch < a.c;
  }
};

// Rows of a thread whose loads are in flight together (four: 3 % slower, by their registers).
constexpr int kUnroll = 2;

// Elements as they lie in memory: half the registers of their floats while they are on their way.
template <typename T, int V> struct Raw {
  typename Pack<T, V>::type v;
  __device__ __forceinline__ void floats(float *out) const {
    if constexpr (V == 1) {
      out[0] = (float)v;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = (float)v[i];
    }
  }
};

// The rows of a thread in s .. e - 1, kUnroll of them at a time.
template <typename T, int V> struct Walk {
  int64_t from, step;  // element of the next row; elements from one row of the thread to its next
  int left;            // rows that are left of the thread's (a chunk's are fewer than 2^31)
  __device__ __forceinline__ Walk(const Norm &a, const Lay<V> &lay, int64_t s, int64_t e)
      : from((s + lay.row) * a.c), step((int64_t)lay.ty * a.c) {
    const int rows = (int)(e - s) - lay.row;
    left = rows > 0 ? (int)((uint32_t)(rows + lay.ty - 1) / (uint32_t)lay.ty) : 0;
  }
  __device__ __forceinline__ bool in(int u) const { return u < left; }
  __device__ __forceinline__ int64_t at(int u) const { return from + u * step; }
  __device__ __forceinline__ void next() {
    from += kUnroll * step;
    left -= kUnroll;
  }
  // ONCE: what is not read again need not push other lines out of the caches.
  template <bool ONCE> __device__ __forceinline__ void load(const T *p, Raw<T, V> *out) const {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (in(u)) {
        const auto *q = reinterpret_cast<const typename Pack<T, V>::type *>(p + at(u));
        if constexpr (ONCE && V > 1) out[u].v = __builtin_nontemporal_load(q);
        else out[u].v = *q;
      }
  }
};

// ---- statistics ---------------------------------------------------------------------------
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_stats_kernel(const Norm a) {
  __shared__ float2 lds[kThreads * V];
  __shared__ float counts[kThreads];
  const Lay<V> lay(a);
  const int64_t r0 = (int64_t)blockIdx.x * a.rows;
  const int64_t r1 = r0 + a.rows < a.n ? r0 + a.rows : a.n;
  const T *x = static_cast<const T *>(a.x) + lay.ch;
  for (int b = cloud_of(a, r0); b < a.clouds; ++b) {
    const int64_t cb = cloud_begin(a, b), ce = cloud_begin(a, b + 1);
    if (cb >= r1) break;
    const int64_t s = cb > r0 ? cb : r0, e = ce < r1 ? ce : r1;
    if (s >= e) continue;
    float first[V], s1[V], s2[V], count = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) first[i] = s1[i] = s2[i] = 0.f;
    if (lay.in && s + lay.row < e) {
      load_floats<T, V>(x + (s + lay.row) * a.c, first);
      Walk<T, V> walk(a, lay, s, e);
      for (; walk.left > 0; walk.next()) {
        Raw<T, V> v[kUnroll];
        walk.template load<false>(x, v);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (walk.in(u)) {
            float f[V];
            v[u].floats(f);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float d = f[i] - first[i];
              s1[i] += d;
              s2[i] += d * d;
            }
            count += 1.f;
          }
      }
    }
    const float inv = count > 0.f ? 1.f / count : 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = s1[i] * inv;
      // (squares that pass float stay infinite, as the variance is then, and NaN stays NaN)
      const float dev = s2[i] < __builtin_inff() ? fmaxf(s2[i] - s1[i] * d, 0.f) : s2[i];
      lds[threadIdx.x * V + i] = make_float2(first[i] + d, dev);
    }
    counts[threadIdx.x] = count;
    __syncthreads();
    int half = 1;
    while (half * 2 < lay.ty) half *= 2;
    for (; half > 0 && lay.ty > 1; half >>= 1) {
      if (lay.row < half && lay.row + half < lay.ty) {
        const int o = threadIdx.x + half * lay.tx;
        const float n1 = counts[threadIdx.x], n2 = counts[o];
        if (n2 > 0.f) {  // (rows are dealt in order: n1 >= n2)
          const float w2 = n2 / (n1 + n2), w = n1 * w2;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float2 p = lds[threadIdx.x * V + i], q = lds[o * V + i];
            const float d = q.x - p.x;
            lds[threadIdx.x * V + i] = make_float2(p.x + d * w2, p.y + q.y + d * d * w);
          }
        }
      }
      __syncthreads();
      if (lay.row < half && lay.row + half < lay.ty && lay.cx < lay.tx)
        counts[threadIdx.x] += counts[threadIdx.x + half * lay.tx];
      __syncthreads();
    }
    if (lay.in && lay.row == 0) {
      float2 *p = a.partial + ((int64_t)blockIdx.x + b) * a.c + lay.ch;
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = lds[threadIdx.x * V + i];
    }
    __syncthreads();
  }
}

// Sum over the workgroup, the same in every thread.
template <typename S>
__device__ __forceinline__ S block_sum(S v, S *lds) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  S t = 0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) t += lds[w];
  return t;
}

// How the threads of a workgroup that adds up pieces lie on the `per` channels of a group and on the
// pieces: channels side by side (in turns of `tx`), `ty` pieces at a time.
struct GroupLay {
  int tx, ty, row, cx;
  __device__ GroupLay(const Norm &a) {
    const int threads = (int)blockDim.x;
    tx = a.per < threads ? a.per : threads;
    ty = threads / tx;
    row = (int)threadIdx.x / tx;
    cx = (int)threadIdx.x - row * tx;
  }
};

// mean and rstd of a group of a cloud, from the channels'
// means and squared deviations in the pieces of the cloud.  Sums over at most a few thousand
// numbers, in double: their cost does not show.
__global__ void __launch_bounds__(1024) norm_finish_kernel(const Norm a) {
  __shared__ double lds[3][16];
  const int id = a.first + (int)blockIdx.x, b = id / a.groups, g = id - b * a.groups;
  const int64_t s = cloud_begin(a, b), e = cloud_begin(a, b + 1);
  if (s >= e) {
    if (threadIdx.x == 0) {
      a.mean[id] = 0.f;
      a.rstd[id] = 0.f;
    }
    return;
  }
  const int k0 = (int)(s / a.rows), pieces = (int)((e - 1) / a.rows) - k0 + 1;
  const float2 *p = a.partial + ((int64_t)k0 + b) * a.c + (int64_t)g * a.per;
  const double shift = p[0].x;
  double sums[3] = {0, 0, 0};  // rows, of means, of squared deviations
  const GroupLay lay(a);
  if (lay.row < lay.ty)
    for (int c = lay.cx; c < a.per; c += lay.tx) {
#pragma unroll 4
      for (int k = lay.row; k < pieces; k += lay.ty) {
        const float2 v = p[(int64_t)k * a.c + c];
        const int64_t kb = ((int64_t)k0 + k) * a.rows, ke = kb + a.rows;
        const double rows = (double)(int)((ke < e ? ke : e) - (kb > s ? kb : s));
        const double d = (double)v.x - shift;
        sums[0] += rows;
        sums[1] += rows * d;
        sums[2] += (double)v.y + rows * d * d;
      }
    }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sums[i] += __shfl_xor(sums[i], d, 64);
    if ((threadIdx.x & 63) == 0) lds[i][threadIdx.x >> 6] = sums[i];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      sums[i] = 0;
      for (int w = 0; w < (int)(blockDim.x >> 6); ++w) sums[i] += lds[i][w];
    }
    const double d = sums[1] / sums[0], var = sums[2] / sums[0] - d * d;
    a.mean[id] = (float)(shift + d);
    a.rstd[id] = (float)(1.0 / sqrt((var < 0 ? 0 : var) + (double)a.eps));
  }
}

// ---- y --------------------------------------------------------------------------------------
// Elements of the groups of cloud b that the channels ch .. of a thread lie in: one load where they
// are one group's.
template <int V, typename E>
__device__ __forceinline__ void of_groups(const Norm &a, const E *p, int b, int64_t ch, E *out) {
  const uint32_t per = (uint32_t)a.per, g0 = (uint32_t)ch / per;
  p += (int64_t)b * a.groups + g0;
  if (per % V == 0) {
    const E e = *p;
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = e;
    return;
  }
  uint32_t at = (uint32_t)ch - g0 * per, g = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    out[i] = p[g];
    if (++at == per) {
      at = 0;
      ++g;
    }
  }
}
// V neighbouring elements of a parameter, `none` without one.
template <int V>
__device__ __forceinline__ void of_channels(const void *p, int64_t ch, int type, float none, float *out) {
  const size_t bytes = type == SSC_F32 ? 4 : 2;
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = none;
  } else if (V > 1 && (reinterpret_cast<uintptr_t>(p) & ((V * bytes < 16 ? V * bytes : 16) - 1)) == 0) {
    // (ch is a multiple of V)
    if (type == SSC_F32) {
#pragma unroll
      for (int i = 0; i < V; i += 4)
        load_floats<float, V < 4 ? V : 4>(static_cast<const float *>(p) + ch + i, out + i);
    } else if (type == SSC_F16) {
      load_floats<f16, V>(static_cast<const f16 *>(p) + ch, out);
    } else {
      load_floats<bf16, V>(static_cast<const bf16 *>(p) + ch, out);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = load_any(p, ch + i, type);
  }
}
template <int V>
__device__ __forceinline__ void channel_params(const Norm &a, int64_t ch, float *w, float *bias) {
  of_channels<V>(a.weight, ch, a.wtype, 1.f, w);
  of_channels<V>(a.bias, ch, a.wtype, 0.f, bias);
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_apply_kernel(const Norm a) {
  const Lay<V> lay(a);
  if (!lay.in) return;
  const int64_t r0 = (int64_t)(gridDim.x - 1 - blockIdx.x) * a.rows;
  const int64_t r1 = r0 + a.rows < a.n ? r0 + a.rows : a.n;
  const T *x = static_cast<const T *>(a.x) + lay.ch;
  T *y = static_cast<T *>(a.out) + lay.ch;
  float w[V], bias[V];
  channel_params<V>(a, lay.ch, w, bias);
  for (int b = cloud_of(a, r0); b < a.clouds; ++b) {
    const int64_t cb = cloud_begin(a, b), ce = cloud_begin(a, b + 1);
    if (cb >= r1) break;
    const int64_t s = cb > r0 ? cb : r0, e = ce < r1 ? ce : r1;
    if (s >= e) continue;
    float mean[V], rstd[V];
    of_groups<V>(a, a.mean, b, lay.ch, mean);
    of_groups<V>(a, a.rstd, b, lay.ch, rstd);
#pragma unroll
    for (int i = 0; i < V; ++i) rstd[i] *= w[i];
    Walk<T, V> walk(a, lay, s, e);
    for (; walk.left > 0; walk.next()) {
      Raw<T, V> v[kUnroll];
      walk.template load<true>(x, v);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (walk.in(u)) {
          float z[V], f[V];
          v[u].floats(z);
#pragma unroll
          for (int i = 0; i < V; ++i) z[i] = (z[i] - mean[i]) * rstd[i] + bias[i];
          activate<V>(a.act, z, f);
          store_floats_once<T, V>(y + walk.at(u), f);
        }
    }
  }
}

// ---- backward -------------------------------------------------------------------------------
// h and dz of one row's V channels.
template <int V>
__device__ __forceinline__ void row_terms(int act, const float *x, const float *dy,
                                          const float *mean, const float *rstd, const float *w,
                                          const float *bias, float *h, float *dz) {
  float z[V], f[V], d[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    h[i] = (x[i] - mean[i]) * rstd[i];
    z[i] = h[i] * w[i] + bias[i];
  }
  activate_slope<V>(act, z, f, d);
#pragma unroll
  for (int i = 0; i < V; ++i) dz[i] = dy[i] * d[i];
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_sums_kernel(const Norm a) {
  __shared__ float2 lds[kThreads * V];
  const Lay<V> lay(a);
  const int64_t r0 = (int64_t)blockIdx.x * a.rows;
  const int64_t r1 = r0 + a.rows < a.n ? r0 + a.rows : a.n;
  const T *x = static_cast<const T *>(a.x) + lay.ch;
  const T *dy = static_cast<const T *>(a.dy) + lay.ch;
  float w[V], bias[V];
  if (lay.in) channel_params<V>(a, lay.ch, w, bias);
  for (int b = cloud_of(a, r0); b < a.clouds; ++b) {
    const int64_t cb = cloud_begin(a, b), ce = cloud_begin(a, b + 1);
    if (cb >= r1) break;
    const int64_t s = cb > r0 ? cb : r0, e = ce < r1 ? ce : r1;
    if (s >= e) continue;
    float s1[V], s2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
    if (lay.in) {
      float mean[V], rstd[V];
      of_groups<V>(a, a.mean, b, lay.ch, mean);
      of_groups<V>(a, a.rstd, b, lay.ch, rstd);
      Walk<T, V> walk(a, lay, s, e);
      for (; walk.left > 0; walk.next()) {
        Raw<T, V> v[kUnroll], g[kUnroll];
        walk.template load<false>(x, v);
        walk.template load<false>(dy, g);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (walk.in(u)) {
            float xv[V], gv[V], h[V], dz[V];
            v[u].floats(xv);
            g[u].floats(gv);
            row_terms<V>(a.act, xv, gv, mean, rstd, w, bias, h, dz);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              s1[i] += dz[i];
              s2[i] += dz[i] * h[i];
            }
          }
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) lds[threadIdx.x * V + i] = make_float2(s1[i], s2[i]);
    __syncthreads();
    int half = 1;
    while (half * 2 < lay.ty) half *= 2;
    for (; half > 0 && lay.ty > 1; half >>= 1) {
      if (lay.row < half && lay.row + half < lay.ty) {
        const int o = threadIdx.x + half * lay.tx;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 p = lds[threadIdx.x * V + i], q = lds[o * V + i];
          lds[threadIdx.x * V + i] = make_float2(p.x + q.x, p.y + q.y);
        }
      }
      __syncthreads();
    }
    if (lay.in && lay.row == 0) {
      float2 *p = a.partial + ((int64_t)blockIdx.x + b) * a.c + lay.ch;
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = lds[threadIdx.x * V + i];
    }
    __syncthreads();
  }
}

// A group of a cloud: the pieces' sums added up, channel by
// channel, and S1 / m, S2 / m of the group.
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const Norm a) {
  __shared__ float2 lds[1024];
  __shared__ float total[16];
  const int id = a.first + (int)blockIdx.x, b = id / a.groups, g = id - b * a.groups;
  const int64_t s = cloud_begin(a, b), e = cloud_begin(a, b + 1);
  const int k0 = (int)(s / a.rows), pieces = s < e ? (int)((e - 1) / a.rows) - k0 + 1 : 0;
  const float2 *p = a.partial + ((int64_t)k0 + b) * a.c + (int64_t)g * a.per;
  const GroupLay lay(a);
  float t1 = 0.f, t2 = 0.f;
  for (int c0 = 0; c0 < a.per; c0 += lay.tx) {  // (one turn unless a group has over 1024 channels)
    const int c = c0 + lay.cx;
    const bool in = lay.row < lay.ty && c < a.per;
    float s1 = 0.f, s2 = 0.f;
    if (in) {
#pragma unroll 4
      for (int k = lay.row; k < pieces; k += lay.ty) {
        const float2 v = p[(int64_t)k * a.c + c];
        s1 += v.x;
        s2 += v.y;
      }
    }
    __syncthreads();
    lds[threadIdx.x] = make_float2(s1, s2);
    __syncthreads();
    int half = 1;
    while (half * 2 < lay.ty) half *= 2;
    for (; half > 0 && lay.ty > 1; half >>= 1) {
      if (lay.row < half && lay.row + half < lay.ty) {
        const float2 v = lds[threadIdx.x], o = lds[threadIdx.x + half * lay.tx];
        lds[threadIdx.x] = make_float2(v.x + o.x, v.y + o.y);
      }
      __syncthreads();
    }
    if (in && lay.row == 0) {
      const int64_t ch = (int64_t)g * a.per + c;
      const float2 v = lds[threadIdx.x];
      a.sums[(int64_t)b * a.c + ch] = v;
      const float w = a.weight ? load_any(a.weight, ch, a.wtype) : 1.f;
      t1 += w * v.x;
      t2 += w * v.y;
    }
  }
  t1 = block_sum(t1, total);
  t2 = block_sum(t2, total);
  if (threadIdx.x == 0) {
    const float inv = s < e ? 1.f / ((float)(e - s) * (float)a.per) : 0.f;
    a.group[id] = make_float2(t1 * inv, t2 * inv);
  }
}

// dweight and dbias of 16 channels, from the clouds' sums.
__device__ __forceinline__ void param_grads(const Norm &a, int block) {
  __shared__ float2 lds[kThreads];
  const int cx = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int64_t ch = (int64_t)block * 16 + cx;
  float s1 = 0.f, s2 = 0.f;
  if (ch < a.c)
    for (int b = row; b < a.clouds; b += kThreads / 16) {
      const float2 v = a.sums[(int64_t)b * a.c + ch];
      s1 += v.x;
      s2 += v.y;
    }
  lds[threadIdx.x] = make_float2(s1, s2);
  __syncthreads();
  if (row == 0 && ch < a.c) {
    for (int y = 1; y < kThreads / 16; ++y) {
      s1 += lds[y * 16 + cx].x;
      s2 += lds[y * 16 + cx].y;
    }
    if (a.dbias) store_any(a.dbias, ch, a.wtype, s1);
    if (a.dweight) store_any(a.dweight, ch, a.wtype, s2);
  }
}

__global__ void __launch_bounds__(kThreads) norm_params_kernel(const Norm a) {
  param_grads(a, blockIdx.x);
}

// The parameters' gradients need no launch of their own: the workgroups in front of the chunks'
// make them (50001 x 200 float16, forward and backward: 2 us of 67 less).
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_dx_kernel(const Norm a) {
  const int before = (int)gridDim.x - a.chunks;
  if ((int)blockIdx.x < before) {
    if (blockIdx.y == 0) param_grads(a, blockIdx.x);
    return;
  }
  const Lay<V> lay(a);
  if (!lay.in) return;
  const int64_t r0 = (int64_t)(gridDim.x - 1 - blockIdx.x) * a.rows;
  const int64_t r1 = r0 + a.rows < a.n ? r0 + a.rows : a.n;
  const T *x = static_cast<const T *>(a.x) + lay.ch;
  const T *dy = static_cast<const T *>(a.dy) + lay.ch;
  T *dx = static_cast<T *>(a.out) + lay.ch;
  float w[V], bias[V];
  channel_params<V>(a, lay.ch, w, bias);
  for (int b = cloud_of(a, r0); b < a.clouds; ++b) {
    const int64_t cb = cloud_begin(a, b), ce = cloud_begin(a, b + 1);
    if (cb >= r1) break;
    const int64_t s = cb > r0 ? cb : r0, e = ce < r1 ? ce : r1;
    if (s >= e) continue;
    float mean[V], rstd[V];
    float2 m[V];
    of_groups<V>(a, a.mean, b, lay.ch, mean);
    of_groups<V>(a, a.rstd, b, lay.ch, rstd);
    of_groups<V>(a, a.group, b, lay.ch, m);
    Walk<T, V> walk(a, lay, s, e);
    for (; walk.left > 0; walk.next()) {
      Raw<T, V> v[kUnroll], g[kUnroll];
      walk.template load<true>(x, v);
      walk.template load<true>(dy, g);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (walk.in(u)) {
          float xv[V], gv[V], h[V], dz[V];
          v[u].floats(xv);
          g[u].floats(gv);
          row_terms<V>(a.act, xv, gv, mean, rstd, w, bias, h, dz);
#pragma unroll
          for (int i = 0; i < V; ++i) xv[i] = rstd[i] * (w[i] * dz[i] - (m[i].x + h[i] * m[i].y));
          store_floats_once<T, V>(dx + walk.at(u), xv);
        }
    }
  }
}

// ---- few rows -------------------------------------------------------------------------------
// A workgroup to a cloud's group, all passes in one launch: the rows of a group lie in the caches
// after the first pass.  Threads: `per` channels side by side, kFewThreads / per rows at a time.
constexpr int kFewThreads = 512;
// The form pays up to some 8192 values of a group: 2100 rows in 2 clouds, 4 channels in a group
// (4200 values), forward and backward 8 and 11 us against 15 and 17 of the passes over chunks; 1024
// rows of 8 channels 9 and 13 against 12 and 14; 1024 rows of 16 channels 14 and 20 against 12 and
// 14.  How many rows a cloud has is not known here: the mean is taken, and a limit for all rows, so
// that a batch whose rows are nearly all one cloud's stays near (32768 values of one group: 23 and
// 34 us against 12 and 14).
constexpr int64_t kFewMean = 8192, kFewMost = 32768;

struct FewLay {
  int ty, row, cx;
  bool in;
  __device__ FewLay(const Norm &a) {
    ty = kFewThreads / a.per;
    row = (int)threadIdx.x / a.per;
    cx = (int)threadIdx.x - row * a.per;
    in = row < ty;
  }
};

template <typename T>
__global__ void __launch_bounds__(kFewThreads) norm_few_kernel(const Norm a) {
  __shared__ float lds[kFewThreads / 64];
  const int id = a.first + (int)blockIdx.x, b = id / a.groups, g = id - b * a.groups;
  const FewLay lay(a);
  const int64_t s = cloud_begin(a, b), e = cloud_begin(a, b + 1);
  const int64_t ch = (int64_t)g * a.per + lay.cx;
  const T *x = static_cast<const T *>(a.x) + ch;
  T *y = static_cast<T *>(a.out) + ch;
  if (s >= e) {
    if (threadIdx.x == 0) a.mean[id] = a.rstd[id] = 0.f;
    return;
  }
  const float inv = 1.f / ((float)(e - s) * (float)a.per);
  const int64_t r0 = lay.in ? s + lay.row : e;
  // the deviations from the group's first value are of the spread's size
  const float first = (float)static_cast<const T *>(a.x)[s * a.c + (int64_t)g * a.per];
  float sum = 0.f;
#pragma unroll 4
  for (int64_t r = r0; r < e; r += lay.ty) sum += (float)x[r * a.c] - first;
  const float mean = first + block_sum(sum, lds) * inv;
  float dev = 0.f;
#pragma unroll 4
  for (int64_t r = r0; r < e; r += lay.ty) {
    const float d = (float)x[r * a.c] - mean;
    dev += d * d;
  }
  const float rstd = 1.f / sqrtf(block_sum(dev, lds) * inv + a.eps);
  if (threadIdx.x == 0) {
    a.mean[id] = mean;
    a.rstd[id] = rstd;
  }
  if (!lay.in) return;
  float w, bias;
  channel_params<1>(a, ch, &w, &bias);
  w *= rstd;
#pragma unroll 4
  for (int64_t r = r0; r < e; r += lay.ty) {
    float z = ((float)x[r * a.c] - mean) * w + bias, f;
    activate<1>(a.act, &z, &f);
    y[r * a.c] = (T)f;
  }
}

template <typename T>
__global__ void __launch_bounds__(kFewThreads) norm_few_backward_kernel(const Norm a) {
  __shared__ float2 lds[kFewThreads];
  __shared__ float total[kFewThreads / 64];
  const int id = a.first + (int)blockIdx.x, b = id / a.groups, g = id - b * a.groups;
  const FewLay lay(a);
  const int64_t s = cloud_begin(a, b), e = cloud_begin(a, b + 1);
  const int64_t ch = (int64_t)g * a.per + lay.cx;
  const T *x = static_cast<const T *>(a.x) + ch, *dy = static_cast<const T *>(a.dy) + ch;
  const float mean = a.mean[id], rstd = a.rstd[id];
  const int64_t r0 = lay.in ? s + lay.row : e;
  float w = 0.f, bias = 0.f, s1 = 0.f, s2 = 0.f;
  if (lay.in) channel_params<1>(a, ch, &w, &bias);
#pragma unroll 4
  for (int64_t r = r0; r < e; r += lay.ty) {
    const float xv = (float)x[r * a.c], gv = (float)dy[r * a.c];
    float h, dz;
    row_terms<1>(a.act, &xv, &gv, &mean, &rstd, &w, &bias, &h, &dz);
    s1 += dz;
    s2 += dz * h;
  }
  lds[threadIdx.x] = make_float2(s1, s2);
  __syncthreads();
  float t1 = 0.f, t2 = 0.f;
  if (lay.row == 0) {
    for (int k = 1; k < lay.ty; ++k) {
      s1 += lds[k * a.per + lay.cx].x;
      s2 += lds[k * a.per + lay.cx].y;
    }
    a.sums[(int64_t)b * a.c + ch] = make_float2(s1, s2);
    t1 = w * s1;
    t2 = w * s2;
  }
  if (a.out == nullptr || s >= e) return;
  const float inv = 1.f / ((float)(e - s) * (float)a.per);
  const float m1 = block_sum(t1, total) * inv, m2 = block_sum(t2, total) * inv;
  T *dx = static_cast<T *>(a.out) + ch;
#pragma unroll 4
  for (int64_t r = r0; r < e; r += lay.ty) {
    const float xv = (float)x[r * a.c], gv = (float)dy[r * a.c];
    float h, dz;
    row_terms<1>(a.act, &xv, &gv, &mean, &rstd, &w, &bias, &h, &dz);
    dx[r * a.c] = (T)(rstd * (w * dz - (m1 + h * m2)));
  }
}

// ---- host -----------------------------------------------------------------------------------
// Rows of a chunk: enough that at most kChunksMost chunks are left, that the partial results stay
// small beside the rows, and that every thread of a workgroup has some (8 channels to a thread).
int64_t chunk_rows(int64_t n, int c) {
  const int64_t r = ceil_div(n, kChunksMost), across = ceil_div(c, 8);
  const int64_t least = across < kThreads / 16 ? 2 * kThreads / across : 32;
  return r < least ? least : r;
}

bool same_alignment(const void *a, const void *b, const void *c, size_t to) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) |
           reinterpret_cast<uintptr_t>(c)) & (to - 1)) == 0;
}

dim3 chunk_grid(const Norm &a, int v, int before) {
  const int cv = a.c / v;
  const int tx = cv < kThreads ? cv : kThreads;
  return dim3((uint32_t)(a.chunks + before), (uint32_t)ceil_div(cv, tx));
}

// Threads of a workgroup that adds up the pieces of one group.
int finish_threads(const Norm &a) {
  const int64_t items = (int64_t)(a.chunks / a.clouds + 1) * a.per;
  return items > 2048 ? 1024 : items > 256 ? 256 : 64;
}

bool few(const Norm &a) {
  return a.per <= kFewThreads && a.n * a.per <= kFewMost && a.n * a.per <= kFewMean * a.clouds;
}

// Channels of a thread: 16 bytes of a row where rows and pointers allow it, 8 bytes, or one.
template <typename T> int width(const Norm &a) {
  constexpr int V = 16 / sizeof(T);
  if (a.c % V == 0 && same_alignment(a.x, a.dy, a.out, 16)) return V;
  return V == 8 && a.c % 4 == 0 && same_alignment(a.x, a.dy, a.out, 8) ? 4 : 1;
}
// (BEFORE: workgroups in front of the chunks')
#define SSC_NORM_LAUNCH(KERNEL, V, BEFORE) \
  hipLaunchKernelGGL((KERNEL<T, V>), chunk_grid(a, V, BEFORE), dim3(kThreads), 0, s, a)
#define SSC_NORM_WIDTHS(KERNEL, BEFORE)                                         \
  if (v == 16 / (int)sizeof(T)) SSC_NORM_LAUNCH(KERNEL, 16 / sizeof(T), BEFORE); \
  else if (v == 4) SSC_NORM_LAUNCH(KERNEL, 4, BEFORE);                           \
  else SSC_NORM_LAUNCH(KERNEL, 1, BEFORE)

// A workgroup to a cloud's group, in launches of at most 2^21 of them: a grid has fewer than 2^32
// threads.
constexpr int kGroupsMost = 1 << 21;
template <typename K> void launch_groups(K kernel, Norm a, int threads, hipStream_t s) {
  const int64_t all = (int64_t)a.clouds * a.groups;
  for (int64_t at = 0; at < all; at += kGroupsMost) {
    a.first = (int32_t)at;
    const int64_t now = all - at < kGroupsMost ? all - at : kGroupsMost;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)now), dim3(threads), 0, s, a);
  }
}

template <typename T> int forward(const Norm &a, hipStream_t s) {
  if (few(a)) {
    launch_groups(norm_few_kernel<T>, a, kFewThreads, s);
    SSC_LAUNCH_CHECK("group norm, forward");
    return SSC_OK;
  }
  const int v = width<T>(a);
  SSC_NORM_WIDTHS(norm_stats_kernel, 0);
  launch_groups(norm_finish_kernel, a, finish_threads(a), s);
  SSC_NORM_WIDTHS(norm_apply_kernel, 0);
  SSC_LAUNCH_CHECK("group norm, forward");
  return SSC_OK;
}

template <typename T> int backward(const Norm &a, hipStream_t s) {
  int params = a.dweight || a.dbias ? (int)ceil_div(a.c, 16) : 0;  // workgroups that make their gradients
  if (few(a)) {
    launch_groups(norm_few_backward_kernel<T>, a, kFewThreads, s);
  } else {
    const int v = width<T>(a);
    SSC_NORM_WIDTHS(norm_sums_kernel, 0);
    launch_groups(norm_reduce_kernel, a, finish_threads(a), s);
    if (a.out) {
      SSC_NORM_WIDTHS(norm_dx_kernel, params);
      params = 0;
    }
  }
  if (params > 0) hipLaunchKernelGGL(norm_params_kernel, dim3(params), dim3(kThreads), 0, s, a);
  SSC_LAUNCH_CHECK("group norm, backward");
  return SSC_OK;
}
#undef SSC_NORM_WIDTHS
#undef SSC_NORM_LAUNCH

size_t workspace(int64_t n, int32_t c, int32_t clouds, int32_t groups) {
  if (n <= 0 || c <= 0 || clouds <= 0 || groups <= 0) return 256;  // (the calls refuse all but no rows)
  const int64_t chunks = ceil_div(n, chunk_rows(n, c));
  return align_up((size_t)(chunks + clouds) * c * sizeof(float2)) +
         align_up((size_t)clouds * c * sizeof(float2)) +
         align_up((size_t)clouds * groups * sizeof(float2));
}

int check(int32_t dtype, int64_t n, int32_t c, const int32_t *offsets, int32_t clouds,
          int32_t groups, int32_t wtype, int32_t act, const void *ws, size_t ws_bytes) {
  SSC_CHECK(dtype_ok(dtype), SSC_EINVAL, "element type %d", dtype);
  SSC_CHECK(dtype_ok(wtype), SSC_EINVAL, "element type %d of the parameters", wtype);
  SSC_CHECK(n >= 0 && c >= 1 && groups >= 1 && c % groups == 0, SSC_EINVAL,
            "%lld rows of %d channels cannot be cut into %d groups", (long long)n, c, groups);
  SSC_CHECK(n <= 0x7FFFFFFF, SSC_EINVAL, "offsets of rows are int32: %lld rows", (long long)n);
  SSC_CHECK(clouds >= (n > 0 ? 1 : 0) && (int64_t)clouds * groups <= 0x7FFFFFFF, SSC_EINVAL,
            "%d clouds of %d groups", clouds, groups);
  SSC_CHECK(pointwise_act_ok(act), SSC_EINVAL, "activation %d", act);
  SSC_CHECK(n == 0 || offsets != nullptr, SSC_EINVAL, "offsets is NULL");
  SSC_CHECK(n == 0 || (ws != nullptr && ws_bytes >= workspace(n, c, clouds, groups)), SSC_EWORKSPACE,
            "workspace of %zu bytes, %zu are needed", ws_bytes, workspace(n, c, clouds, groups));
  return SSC_OK;
}

Norm carve(int64_t n, int32_t c, int32_t clouds, int32_t groups, void *ws) {
  Norm a = {};
  a.n = n;
  a.c = c;
  a.clouds = clouds;
  a.groups = groups;
  a.per = c / groups;
  a.rows = (int32_t)chunk_rows(n, c);
  a.chunks = (int32_t)ceil_div(n, a.rows);
  Carver w(ws);
  a.partial = w.take<float2>((size_t)(a.chunks + clouds) * c);
  a.sums = w.take<float2>((size_t)clouds * c);
  a.group = w.take<float2>((size_t)clouds * groups);
  return a;
}

}  // namespace
}  // namespace ssc

using namespace ssc;

extern "C" size_t ssc_groupnorm_workspace_bytes(int64_t n, int32_t c, int32_t clouds,
                                                int32_t groups) {
  return workspace(n, c, clouds, groups);
}

extern "C" int ssc_groupnorm_fwd(int32_t dtype, const void *x, int64_t n, int32_t c,
                                 const int32_t *offsets, int32_t clouds, int32_t groups,
                                 int32_t wtype, const void *weight, const void *bias, float eps,
                                 int32_t act, void *y, float *mean, float *rstd, void *ws,
                                 size_t ws_bytes, ssc_stream_t stream) {
  const int rc = check(dtype, n, c, offsets, clouds, groups, wtype, act, ws, ws_bytes);
  if (rc != SSC_OK) return rc;
  SSC_CHECK(eps >= 0.f, SSC_EINVAL, "eps is not negative");
  if (n == 0) return SSC_OK;
  SSC_CHECK(x && y && mean && rstd, SSC_EINVAL, "NULL pointer");
  Norm a = carve(n, c, clouds, groups, ws);
  a.x = x;
  a.out = y;
  a.offsets = offsets;
  a.weight = weight;
  a.bias = bias;
  a.wtype = wtype;
  a.act = act;
  a.eps = eps;
  a.mean = mean;
  a.rstd = rstd;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == SSC_F32 ? forward<float>(a, s) : dtype == SSC_F16 ? forward<f16>(a, s) : forward<bf16>(a, s);
}

extern "C" int ssc_groupnorm_bwd(int32_t dtype, const void *x, const void *dy, int64_t n, int32_t c,
                                 const int32_t *offsets, int32_t clouds, int32_t groups,
                                 int32_t wtype, const void *weight, const void *bias, int32_t act,
                                 const float *mean, const float *rstd, void *dx, void *dweight,
                                 void *dbias, void *ws, size_t ws_bytes, ssc_stream_t stream) {
  const int rc = check(dtype, n, c, offsets, clouds, groups, wtype, act, ws, ws_bytes);
  if (rc != SSC_OK) return rc;
  if (n == 0) return SSC_OK;
  SSC_CHECK(x && dy && mean && rstd, SSC_EINVAL, "NULL pointer");
  Norm a = carve(n, c, clouds, groups, ws);
  a.x = x;
  a.dy = dy;
  a.out = dx;
  a.offsets = offsets;
  a.weight = weight;
  a.bias = bias;
  a.wtype = wtype;
  a.act = act;
  a.mean = const_cast<float *>(mean);
  a.rstd = const_cast<float *>(rstd);
  a.dweight = dweight;
  a.dbias = dbias;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == SSC_F32 ? backward<float>(a, s) : dtype == SSC_F16 ? backward<f16>(a, s) : backward<bf16>(a, s);
}
