// AdamW over many tensors at once, moments in 32 bits or in 8.
//
//   m <- b1 m + (1 - b1) g          v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Every element is read and written once: 28 bytes for a float parameter with 32-bit moments,
// 16 with 8-bit ones.  HBM-bound for large sets, bound by launches for small ones, so the
// table of tensors travels in the kernel arguments (no copy to the device, no launch per
// tensor) and a workgroup finds its tensor in it with one vector load.
//
// 8-bit moments: 256 neighbouring elements of a tensor share a float scale q.
//   m = q c |c|, c in -127 .. 127, q = max |m| / 127^2
//   sqrt(v) = q c^2, c in 0 .. 255, q = max sqrt(v) / 255^2
// The code is linear in the root of the magnitude: its steps are 1/64 of a value near the
// block's largest and grow to the value itself 1/16000 below it, where a linear code would
// have given zeros from 1/254 on.  The step divides by sqrt(v), so a v that is not zero never
// gets the code zero: it is rounded up to the smallest one, which makes the step shorter,
// never longer.  The codes follow from sums, products, divisions and square roots that are
// each rounded once, in one stated order (no fused multiply-add), so they are the same on any
// machine.  A block with a value that is no finite number has the scale NaN, and all of it
// comes back as NaN.
#include <float.h>
#include <math.h>

#include "elem.h"

namespace ssc {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 4;                          // elements of a thread at a time
constexpr int kTurns = 2;                        // such turns of a workgroup
constexpr int kChunk = kThreads * kPer * kTurns;  // elements of a workgroup
constexpr int kBlock = SSC_ADAMW_BLOCK;          // elements that share a scale: a wave's turn
static_assert(kBlock == 64 * kPer, "a wave's turn is one block of a tensor");

struct Entry32 {
  void *p;
  const void *g;
  float *m, *v;
  int64_t n;
};
struct Entry8 {
  void *p;
  const void *g;
  int8_t *m;
  uint8_t *v;
  float *mq, *vq;
  int64_t n;
};
struct Consts {
  float b1, omb1, b2, omb2, eps, decay, step, root;
};
// kernel arguments of at most 4 KiB
template <typename E, int N> struct Table {
  E e[N];
  int32_t first[N];   // first workgroup of every tensor
  uint8_t kind[N];    // element type of the parameter, + 4: every pointer aligned for kPer
  Consts k;
  int32_t count;
};
constexpr int64_t kBlocksMost = (int64_t(1) << 32) / kThreads - 1;  // a grid has fewer than 2^32 threads
constexpr int kMost32 = 88, kMost8 = 64;
static_assert(sizeof(Table<Entry32, kMost32>) <= 4096 && sizeof(Table<Entry8, kMost8>) <= 4096,
              "kernel arguments");

// The tensor of this workgroup: the last one that begins at or before it.
template <int N>
__device__ __forceinline__ int tensor_of(const int32_t (&first)[N], int count) {
  const int lane = threadIdx.x & 63;
  int below = 0;
#pragma unroll
  for (int i = 0; i < N; i += 64) {
    const int at = i + lane;
    const bool in = at < count && first[at < N ? at : N - 1] <= (int)blockIdx.x;
    below += __popcll(__ballot(in));
  }
  return __builtin_amdgcn_readfirstlane(below - 1);
}

// (the quotient by a reciprocal that is right to a unit in the last place: the parameter's own
// rounding hides it)
__device__ __forceinline__ void update(const Consts &k, float g, float &p, float &m, float &v,
                                       float &root) {
#pragma clang fp contract(off)
  m = k.b1 * m + k.omb1 * g;
  v = k.b2 * v + k.omb2 * (g * g);
  root = sqrtf(v);
  p = p * k.decay - (m * __builtin_amdgcn_rcpf(root * k.root + k.eps)) * k.step;
}

template <typename T, bool WIDE>
__device__ __forceinline__ void step32(const Entry32 &e, const Consts &k, int64_t base) {
  constexpr int V = WIDE ? kPer : 1;
  T *p = static_cast<T *>(e.p);
  const T *g = static_cast<const T *>(e.g);
#pragma unroll
  for (int turn = 0; turn < kChunk / (kThreads * V); ++turn) {
    const int64_t i = base + ((int64_t)turn * kThreads + threadIdx.x) * V;
    if (i + V <= e.n) {
      float pv[V], gv[V], mv[V], vv[V], root;
      load_floats<T, V>(p + i, pv);
      load_floats<T, V>(g + i, gv);
      load_floats<float, V>(e.m + i, mv);
      load_floats<float, V>(e.v + i, vv);
#pragma unroll
      for (int j = 0; j < V; ++j) update(k, gv[j], pv[j], mv[j], vv[j], root);
      store_floats<T, V>(p + i, pv);
      store_floats<float, V>(e.m + i, mv);
      store_floats<float, V>(e.v + i, vv);
    } else {
      for (int64_t j = i; j < e.n; ++j) {  // fewer than V elements at a tensor's end
        float pv = (float)p[j], mv = e.m[j], vv = e.v[j], root;
        update(k, (float)g[j], pv, mv, vv, root);
        p[j] = (T)pv;
        e.m[j] = mv;
        e.v[j] = vv;
      }
    }
  }
}

__global__ void __launch_bounds__(kThreads) adamw32_kernel(const Table<Entry32, kMost32> t) {
  const int i = tensor_of(t.first, t.count);
  const Entry32 &e = t.e[i];
  const int64_t base = (int64_t)((int)blockIdx.x - t.first[i]) * kChunk;
  switch (t.kind[i]) {
    case SSC_F32: step32<float, false>(e, t.k, base); break;
    case SSC_F16: step32<f16, false>(e, t.k, base); break;
    case SSC_BF16: step32<bf16, false>(e, t.k, base); break;
    case SSC_F32 + 4: step32<float, true>(e, t.k, base); break;
    case SSC_F16 + 4: step32<f16, true>(e, t.k, base); break;
    default: step32<bf16, true>(e, t.k, base); break;
  }
}

// Non-negative floats order as their bits do, infinity above every number and NaN above
// infinity, so a maximum of bits keeps them where a maximum of floats would drop a NaN.  Within
// rows of 16 lanes and then from row to row in the vector unit, without the trips to LDS that a
// shuffle takes; lane 63 ends with the maximum of all.
template <int CTRL> __device__ __forceinline__ uint32_t max_with(uint32_t x) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
  return x > o ? x : o;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max_with<0xB1>(x);   // quad_perm 1 0 3 2
  x = max_with<0x4E>(x);   // quad_perm 2 3 0 1
  x = max_with<0x141>(x);  // row_half_mirror
  x = max_with<0x140>(x);  // row_mirror
  x = max_with<0x142>(x);  // row_bcast:15
  x = max_with<0x143>(x);  // row_bcast:31
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

__device__ __forceinline__ float scale_of(uint32_t top, float per_step) {
  if (top >= 0x7F800000u) return __builtin_nanf("");
  return fmaxf(__uint_as_float(top) * per_step, FLT_MIN);
}

// floor(sqrt(x / q) + 1/2), quotient and root rounded once each.  The quick way, with inv = 1 / q
// and the hardware's root, is off by less than 4 units of 2^-24 relative, 7e-5 of a code at 255:
// where it does not lie that near a boundary between two codes both give the same one (all but 3
// in 10000 values).
__device__ __forceinline__ float code_of(float x, float q, float inv) {
#pragma clang fp contract(off)
  const float t = __builtin_amdgcn_sqrtf(x * inv) + 0.5f;
  float c = floorf(t);
  if (fabsf(t - c - 0.5f) > 0.5f - 1.5e-4f) c = floorf(sqrtf(x / q) + 0.5f);
  return c;
}

__device__ __forceinline__ float m_value(int c, float q) { return (float)(c * (c < 0 ? -c : c)) * q; }
__device__ __forceinline__ float v_value(int c, float q) {
  const float u = (float)(c * c) * q;
  return u * u;
}

template <typename T, bool WIDE>
__device__ __forceinline__ void step8(const Entry8 &e, const Consts &k, int64_t base) {
  T *p = static_cast<T *>(e.p);
  const T *g = static_cast<const T *>(e.g);
#pragma unroll
  for (int turn = 0; turn < kTurns; ++turn) {
    const int64_t i = base + ((int64_t)turn * kThreads + threadIdx.x) * kPer;
    const int64_t b = i / kBlock;  // the same for a wave
    if (b * kBlock >= e.n) return;
    const float mq = e.mq[b], vq = e.vq[b];
    float pv[kPer], gv[kPer], mv[kPer], vv[kPer], root[kPer];
    const bool whole = WIDE && i + kPer <= e.n;
    if (whole) {
      load_floats<T, kPer>(p + i, pv);
      load_floats<T, kPer>(g + i, gv);
      const uint32_t mc = *reinterpret_cast<const uint32_t *>(e.m + i);
      const uint32_t vc = *reinterpret_cast<const uint32_t *>(e.v + i);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        mv[j] = m_value((int)(int8_t)(mc >> (8 * j)), mq);
        vv[j] = v_value((int)(uint8_t)(vc >> (8 * j)), vq);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const bool in = i + j < e.n;
        pv[j] = in ? (float)p[i + j] : 0.f;
        gv[j] = in ? (float)g[i + j] : 0.f;
        mv[j] = in ? m_value(e.m[i + j], mq) : 0.f;
        vv[j] = in ? v_value(e.v[i + j], vq) : 0.f;
      }
    }
    uint32_t mtop = 0, vtop = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      update(k, gv[j], pv[j], mv[j], vv[j], root[j]);
      const uint32_t a = __float_as_uint(mv[j]) & 0x7FFFFFFFu;
      // (the bits of -0 and of a negative NaN without their sign)
      const uint32_t c = __float_as_uint(root[j]) & 0x7FFFFFFFu;
      mtop = a > mtop ? a : mtop;  // (what lies behind a tensor's end is 0)
      vtop = c > vtop ? c : vtop;
    }
    mtop = wave_max(mtop);
    vtop = wave_max(vtop);
    const float mn = scale_of(mtop, 1.f / (127.f * 127.f)), vn = scale_of(vtop, 1.f / (255.f * 255.f));
    // (scales are normal numbers below 2^115, so their reciprocals are normal too)
    const float mi = __builtin_amdgcn_rcpf(mn), vi = __builtin_amdgcn_rcpf(vn);
    int mc[kPer], vc[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const float a = fminf(code_of(fabsf(mv[j]), mn, mi), 127.f);
      const float c = fminf(code_of(root[j], vn, vi), 255.f);
      // (a NaN scale: the codes are 0)
      const int ai = mn == mn ? (int)a : 0;
      mc[j] = mv[j] < 0.f ? -ai : ai;
      vc[j] = vn == vn ? (int)fmaxf(c, root[j] > 0.f ? 1.f : 0.f) : 0;
    }
    if (whole) {
      uint32_t a = 0, c = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        a |= ((uint32_t)mc[j] & 255u) << (8 * j);
        c |= (uint32_t)vc[j] << (8 * j);
      }
      store_floats<T, kPer>(p + i, pv);
      *reinterpret_cast<uint32_t *>(e.m + i) = a;
      *reinterpret_cast<uint32_t *>(e.v + i) = c;
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (i + j < e.n) {
          p[i + j] = (T)pv[j];
          e.m[i + j] = (int8_t)mc[j];
          e.v[i + j] = (uint8_t)vc[j];
        }
    }
    if ((threadIdx.x & 63) == 0) {
      e.mq[b] = mn;
      e.vq[b] = vn;
    }
  }
}

__global__ void __launch_bounds__(kThreads) adamw8_kernel(const Table<Entry8, kMost8> t) {
  const int i = tensor_of(t.first, t.count);
  const Entry8 &e = t.e[i];
  const int64_t base = (int64_t)((int)blockIdx.x - t.first[i]) * kChunk;
  switch (t.kind[i]) {
    case SSC_F32: step8<float, false>(e, t.k, base); break;
    case SSC_F16: step8<f16, false>(e, t.k, base); break;
    case SSC_BF16: step8<bf16, false>(e, t.k, base); break;
    case SSC_F32 + 4: step8<float, true>(e, t.k, base); break;
    case SSC_F16 + 4: step8<f16, true>(e, t.k, base); break;
    default: step8<bf16, true>(e, t.k, base); break;
  }
}

// The values that 8-bit moments stand for: p and g of an entry are the float arrays they go to
// (either may be NULL).
__global__ void __launch_bounds__(kThreads) adamw_values_kernel(const Table<Entry8, kMost8> t) {
  const int i = tensor_of(t.first, t.count);
  const Entry8 &e = t.e[i];
  const int64_t base = (int64_t)((int)blockIdx.x - t.first[i]) * kChunk;
  float *mo = static_cast<float *>(e.p), *vo = static_cast<float *>(const_cast<void *>(e.g));
#pragma unroll
  for (int turn = 0; turn < kTurns; ++turn) {
    const int64_t at = base + ((int64_t)turn * kThreads + threadIdx.x) * kPer;
    if (at >= e.n) return;
    const float mq = mo ? e.mq[at / kBlock] : 0.f, vq = vo ? e.vq[at / kBlock] : 0.f;
    if (t.kind[i] >= 4 && at + kPer <= e.n) {
      float mv[kPer], vv[kPer];
      const uint32_t mc = mo ? *reinterpret_cast<const uint32_t *>(e.m + at) : 0;
      const uint32_t vc = vo ? *reinterpret_cast<const uint32_t *>(e.v + at) : 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        mv[j] = m_value((int)(int8_t)(mc >> (8 * j)), mq);
        vv[j] = v_value((int)(uint8_t)(vc >> (8 * j)), vq);
      }
      if (mo) store_floats_once<float, kPer>(mo + at, mv);
      if (vo) store_floats_once<float, kPer>(vo + at, vv);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (at + j < e.n) {
          if (mo) mo[at + j] = m_value(e.m[at + j], mq);
          if (vo) vo[at + j] = v_value(e.v[at + j], vq);
        }
    }
  }
}

bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

void put(Entry32 &e, const ssc_adamw_tensor &t) {
  e = {t.param, t.grad, static_cast<float *>(t.exp_avg), static_cast<float *>(t.exp_avg_sq), t.numel};
}
void put(Entry8 &e, const ssc_adamw_tensor &t) {
  e = {t.param, t.grad, static_cast<int8_t *>(t.exp_avg), static_cast<uint8_t *>(t.exp_avg_sq),
       t.exp_avg_scale, t.exp_avg_sq_scale, t.numel};
}

// One launch for every N tensors that are not empty (or as many as a grid has room for).
template <typename E, int N, typename K>
int launch_all(K kernel, const ssc_adamw_tensor *tensors, int32_t n, size_t moment_align,
               const Consts &k, const char *name, hipStream_t s) {
  Table<E, N> t;
  t.k = k;
  t.count = 0;
  int64_t blocks = 0;
  for (int32_t i = 0; i <= n; ++i) {
    const int64_t more = i < n ? ceil_div(tensors[i].numel, kChunk) : 0;
    if (t.count > 0 && (i == n || t.count == N || blocks + more > kBlocksMost)) {
      hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(kThreads), 0, s, t);
      SSC_LAUNCH_CHECK(name);
      t.count = 0;
      blocks = 0;
    }
    if (more == 0) continue;
    const ssc_adamw_tensor &a = tensors[i];
    const size_t pa = (size_t)kPer * dtype_bytes((int)a.dtype);
    const bool wide = aligned(a.param, pa) && aligned(a.grad, pa) &&
                      aligned(a.exp_avg, moment_align) && aligned(a.exp_avg_sq, moment_align);
    put(t.e[t.count], a);
    t.first[t.count] = (int32_t)blocks;
    t.kind[t.count] = (uint8_t)(a.dtype + (wide ? 4 : 0));
    ++t.count;
    blocks += more;
  }
  return SSC_OK;
}

}  // namespace
}  // namespace ssc

using namespace ssc;

extern "C" int ssc_adamw_step(const ssc_adamw_tensor *tensors, int32_t n_tensors,
                              int32_t state_bits, double lr, double beta1, double beta2, double eps,
                              double weight_decay, int64_t step, ssc_stream_t stream) {
  SSC_CHECK(state_bits == 32 || state_bits == 8, SSC_EINVAL, "moments have 32 bits or 8, not %d",
            state_bits);
  SSC_CHECK(n_tensors >= 0 && (n_tensors == 0 || tensors != nullptr), SSC_EINVAL,
            "bad table of tensors");
  SSC_CHECK(step >= 1, SSC_EINVAL, "the step is counted from 1");
  // (written so that a NaN fails)
  SSC_CHECK(lr >= 0 && weight_decay >= 0 && eps >= 0, SSC_EINVAL,
            "lr, eps and weight_decay are not negative");
  SSC_CHECK(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, SSC_EINVAL, "betas are in [0, 1)");
  for (int32_t i = 0; i < n_tensors; ++i) {
    const ssc_adamw_tensor &t = tensors[i];
    SSC_CHECK(t.numel >= 0 && ceil_div(t.numel, kChunk) <= kBlocksMost, SSC_EINVAL,
              "tensor %d: bad number of elements", i);
    SSC_CHECK(t.dtype >= 0 && dtype_ok((int)t.dtype), SSC_EINVAL,
              "tensor %d: element type %lld", i, (long long)t.dtype);
    SSC_CHECK(t.numel == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq &&
                               (state_bits == 32 || (t.exp_avg_scale && t.exp_avg_sq_scale))),
              SSC_EINVAL, "tensor %d: NULL pointer", i);
  }
  Consts k;
  k.b1 = (float)beta1;
  k.omb1 = (float)(1.0 - beta1);
  k.b2 = (float)beta2;
  k.omb2 = (float)(1.0 - beta2);
  k.eps = (float)eps;
  k.decay = (float)(1.0 - lr * weight_decay);
  k.step = (float)(lr / (1.0 - pow(beta1, (double)step)));
  k.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (state_bits == 32)
    return launch_all<Entry32, kMost32>(adamw32_kernel, tensors, n_tensors, 16, k, "adamw32_kernel", s);
  return launch_all<Entry8, kMost8>(adamw8_kernel, tensors, n_tensors, 4, k, "adamw8_kernel", s);
}

extern "C" int ssc_adamw_values(const ssc_adamw_tensor *tensors, int32_t n_tensors,
                                ssc_stream_t stream) {
  SSC_CHECK(n_tensors >= 0 && (n_tensors == 0 || tensors != nullptr), SSC_EINVAL,
            "bad table of tensors");
  for (int32_t i = 0; i < n_tensors; ++i) {
    const ssc_adamw_tensor &t = tensors[i];
    SSC_CHECK(t.numel >= 0 && ceil_div(t.numel, kChunk) <= kBlocksMost, SSC_EINVAL,
              "tensor %d: bad number of elements", i);
    SSC_CHECK(t.dtype == SSC_F32, SSC_EINVAL, "tensor %d: values are floats", i);
    SSC_CHECK(t.numel == 0 || ((!t.param || (t.exp_avg && t.exp_avg_scale)) &&
                               (!t.grad || (t.exp_avg_sq && t.exp_avg_sq_scale))),
              SSC_EINVAL, "tensor %d: NULL pointer", i);
  }
  return launch_all<Entry8, kMost8>(adamw_values_kernel, tensors, n_tensors, 4, Consts(),
                                    "adamw_values_kernel", static_cast<hipStream_t>(stream));
}
