// Elements of float, half and bfloat16 arrays as floats, and the activation functions of the
// pointwise operators with their derivatives.
#ifndef SSC_ELEM_H_
#define SSC_ELEM_H_

#include "ssc_common.h"

namespace ssc {

typedef _Float16 f16;
typedef __bf16 bf16;

template <typename T> struct ElemCode;
template <> struct ElemCode<float> { static constexpr int value = SSC_F32; };
template <> struct ElemCode<f16> { static constexpr int value = SSC_F16; };
template <> struct ElemCode<bf16> { static constexpr int value = SSC_BF16; };

static inline bool dtype_ok(int d) { return d == SSC_F32 || d == SSC_F16 || d == SSC_BF16; }
static inline int dtype_bytes(int d) { return d == SSC_F32 ? 4 : 2; }
// The activations of the pointwise operators (the convolution's epilogue and the batch norm
// know the first four).
static inline bool pointwise_act_ok(int a) { return a >= SSC_ACT_NONE && a <= SSC_ACT_GELU; }

// V elements as one load or store (V * sizeof(T) <= 16, p aligned to it).
template <typename T, int V> struct Pack {
  typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T> struct Pack<T, 1> { typedef T type; };

template <typename T, int V>
__device__ __forceinline__ void load_floats(const T *p, float *out) {
  if constexpr (V == 1) {
    out[0] = (float)p[0];
  } else {
    const auto v = *reinterpret_cast<const typename Pack<T, V>::type *>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)v[i];
  }
}

// The same for data that is not read again: it need not push other lines out of the caches.
template <typename T, int V>
__device__ __forceinline__ void load_floats_once(const T *p, float *out) {
  if constexpr (V == 1) {
    out[0] = (float)p[0];
  } else {
    const auto v = __builtin_nontemporal_load(
        reinterpret_cast<const typename Pack<T, V>::type *>(p));
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)v[i];
  }
}

// Rounded to nearest even, once.
template <typename T, int V>
__device__ __forceinline__ void store_floats(T *p, const float *in) {
  if constexpr (V == 1) {
    p[0] = (T)in[0];
  } else {
    typename Pack<T, V>::type v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)in[i];
    *reinterpret_cast<typename Pack<T, V>::type *>(p) = v;
  }
}

// The same for results that are not read again soon: they need not push other lines out of the
// caches.
template <typename T, int V>
__device__ __forceinline__ void store_floats_once(T *p, const float *in) {
  if constexpr (V == 1) {
    p[0] = (T)in[0];
  } else {
    typename Pack<T, V>::type v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)in[i];
    __builtin_nontemporal_store(v, reinterpret_cast<typename Pack<T, V>::type *>(p));
  }
}

// Element i of an array whose type is known at run time only (parameter vectors).
__device__ __forceinline__ float load_any(const void *p, int64_t i, int dtype) {
  if (dtype == SSC_F32) return static_cast<const float *>(p)[i];
  if (dtype == SSC_F16) return (float)static_cast<const f16 *>(p)[i];
  return (float)static_cast<const bf16 *>(p)[i];
}
__device__ __forceinline__ void store_any(void *p, int64_t i, int dtype, float v) {
  if (dtype == SSC_F32) static_cast<float *>(p)[i] = v;
  else if (dtype == SSC_F16) static_cast<f16 *>(p)[i] = (f16)v;
  else static_cast<bf16 *>(p)[i] = (bf16)v;
}

__device__ __forceinline__ float sigmoid_of(float z) {
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}

// The normal distribution function c of z, and e = exp(-z^2 / 2), by formula 7.1.26 of Abramowitz
// and Stegun, Handbook of Mathematical Functions: erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2), t = 1 / (1 +
// p x), off by at most 1.5e-7.  One exponential and one reciprocal serve value and slope, where the
// library's erf and another exponential take three times the instructions (norm of 300000 x 256
// bfloat16 with gelu, the writing pass 102 -> 75 us, the backward pass' sums 170 -> 132), and below
// zero nothing cancels.
__device__ __forceinline__ float normal_cdf(float z, float &e) {
  const float x = fabsf(z) * 0.70710678f;
  const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * x);
  e = __expf(-x * x);
  float p = 1.061405429f;
  p = p * t - 1.453152027f;
  p = p * t + 1.421413741f;
  p = p * t - 0.284496736f;
  p = p * t + 0.254829592f;
  const float tail = 0.5f * p * t * e;
  return z < 0.f ? tail : 1.f - tail;
}

// f(z) of V values; `kind` is the same for a whole launch, so the branch is uniform.
template <int V>
__device__ __forceinline__ void activate(int kind, const float *z, float *f) {
  switch (kind) {
    case SSC_ACT_RELU:
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = z[i] < 0.f ? 0.f : z[i];  // (NaN stays NaN)
      break;
    case SSC_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = sigmoid_of(z[i]);
      break;
    case SSC_ACT_TANH:
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = tanhf(z[i]);
      break;
    case SSC_ACT_SILU:
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = z[i] * sigmoid_of(z[i]);
      break;
    case SSC_ACT_GELU:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float e;
        f[i] = z[i] * normal_cdf(z[i], e);
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = z[i];
  }
}

// f(z) and f'(z).
template <int V>
__device__ __forceinline__ void activate_slope(int kind, const float *z, float *f, float *d) {
  switch (kind) {
    case SSC_ACT_RELU:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f[i] = z[i] < 0.f ? 0.f : z[i];
        d[i] = z[i] > 0.f ? 1.f : 0.f;
      }
      break;
    case SSC_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f[i] = sigmoid_of(z[i]);
        d[i] = f[i] * (1.f - f[i]);
      }
      break;
    case SSC_ACT_TANH:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f[i] = tanhf(z[i]);
        d[i] = 1.f - f[i] * f[i];
      }
      break;
    case SSC_ACT_SILU:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float s = sigmoid_of(z[i]);
        f[i] = z[i] * s;
        d[i] = s * (1.f + z[i] * (1.f - s));
      }
      break;
    case SSC_ACT_GELU:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float e;
        const float c = normal_cdf(z[i], e);
        f[i] = z[i] * c;
        d[i] = c + z[i] * e * 0.39894228f;
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f[i] = z[i];
        d[i] = 1.f;
      }
  }
}

}  // namespace ssc

#endif
