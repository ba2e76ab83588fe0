// Activations of the gated feed-forward block and their derivatives, in FP32.
//
//   SILU       x p,  p = 1 / (1 + e^-x)                    derivative p (1 + x (1 - p))
//   GELU       x Phi(x),  Phi(x) = erfc(-x / sqrt 2) / 2   derivative Phi(x) + x e^(-x^2/2) / sqrt(2 pi)
//   GELU_TANH  x s,  s = 1 / (1 + e^-2z), z = sqrt(2/pi) (x + 0.044715 x^3)
//                                                          derivative s + x s (1 - s) 2 dz/dx
//   RELU       max(x, 0)                                   derivative 1 for x > 0, else 0
//   SIGMOID    p                                           derivative p (1 - p)
//
// A NaN stays one.  The logistic function is formed from t = e^-|x|, which never overflows, as 1 / (1 + t) or t / (1 + t),
// so that it and its complement are both accurate relative to their own size.  The reciprocal is the 2-ulp one (the
// denominators lie in [1, 2]), the exponential is CUDA's expf.
#pragma once
#include <cuda_runtime.h>

#include "../../include/dragon_cu32.h"

namespace dragon {

// p = 1 / (1 + e^-x) and q = 1 - p
__device__ __forceinline__ void sigmoid_pq(float x, float* p, float* q) {
  const float t = expf(-fabsf(x));
  const float r = __fdividef(1.0f, 1.0f + t), tr = t * r;
  *p = x < 0.0f ? tr : r;
  *q = x < 0.0f ? r : tr;
}
__device__ __forceinline__ float sigmoid_f(float x) {
  float p, q;
  sigmoid_pq(x, &p, &q);
  return p;
}
// 2z of GELU_TANH; the cube stays finite, s has long reached 0 or 1 at 100
__device__ __forceinline__ float gelu_tanh_2z(float x, float* slope) {
  const float c = fminf(fmaxf(x, -100.0f), 100.0f);
  const float cc = c * c;
  *slope = 1.5957691216057308f * fmaf(0.134145f, cc, 1.0f);
  return 1.5957691216057308f * fmaf(0.044715f * cc, c, c);
}

template <int ACT>
__device__ __forceinline__ float act_value(float x) {
  if (ACT == CU32_ACT_SILU) return x * sigmoid_f(x);
  if (ACT == CU32_ACT_GELU) return 0.5f * x * erfcf(-0.70710678118654752f * x);
  if (ACT == CU32_ACT_GELU_TANH) {
    float slope;
    return x * sigmoid_f(gelu_tanh_2z(x, &slope));
  }
  if (ACT == CU32_ACT_RELU) return x < 0.0f ? 0.0f : x;
  return sigmoid_f(x);
}

// act(x) and act'(x)
template <int ACT>
__device__ __forceinline__ void act_both(float x, float* a, float* d) {
  if (ACT == CU32_ACT_SILU) {
    float p, q;
    sigmoid_pq(x, &p, &q);
    *a = x * p;
    *d = p * fmaf(x, q, 1.0f);
  } else if (ACT == CU32_ACT_GELU) {
    const float phi = 0.5f * erfcf(-0.70710678118654752f * x);
    *a = x * phi;
    *d = fmaf(x * 0.3989422804014327f, expf(-0.5f * x * x), phi);
  } else if (ACT == CU32_ACT_GELU_TANH) {
    float slope, s, q;
    sigmoid_pq(gelu_tanh_2z(x, &slope), &s, &q);
    *a = x * s;
    *d = fmaf(x * s * q, slope, s);
  } else if (ACT == CU32_ACT_RELU) {
    *a = x < 0.0f ? 0.0f : x;
    *d = x > 0.0f ? 1.0f : (x <= 0.0f ? 0.0f : x);
  } else {
    float p, q;
    sigmoid_pq(x, &p, &q);
    *a = p;
    *d = p * q;
  }
}

// v[j] = act(v[j]) * v[HW + j] for j < HW (the switch is uniform: one case runs)
template <int HW, int ACT, int W>
__device__ __forceinline__ void gated_forward_as(float (&v)[W]) {
#pragma unroll
  for (int j = 0; j < HW; ++j) v[j] = act_value<ACT>(v[j]) * v[HW + j];
}
template <int HW, int W>
__device__ __forceinline__ void gated_forward(int act, float (&v)[W]) {
  switch (act) {
    case CU32_ACT_SILU: gated_forward_as<HW, CU32_ACT_SILU>(v); break;
    case CU32_ACT_GELU: gated_forward_as<HW, CU32_ACT_GELU>(v); break;
    case CU32_ACT_GELU_TANH: gated_forward_as<HW, CU32_ACT_GELU_TANH>(v); break;
    case CU32_ACT_RELU: gated_forward_as<HW, CU32_ACT_RELU>(v); break;
    default: gated_forward_as<HW, CU32_ACT_SIGMOID>(v); break;
  }
}

// dg = d u act'(g), du = d act(g)
template <int ACT>
__device__ __forceinline__ void gated_backward1(float d, float g, float u, float* dg, float* du) {
  float a, e;
  act_both<ACT>(g, &a, &e);
  *dg = d * u * e;
  *du = d * a;
}
template <int ACT>
__device__ __forceinline__ void gated_backward4_as(float4 d, float4 g, float4 u, float4* dg, float4* du) {
  gated_backward1<ACT>(d.x, g.x, u.x, &dg->x, &du->x);
  gated_backward1<ACT>(d.y, g.y, u.y, &dg->y, &du->y);
  gated_backward1<ACT>(d.z, g.z, u.z, &dg->z, &du->z);
  gated_backward1<ACT>(d.w, g.w, u.w, &dg->w, &du->w);
}
__device__ __forceinline__ void gated_backward4(int act, float4 d, float4 g, float4 u, float4* dg, float4* du) {
  switch (act) {
    case CU32_ACT_SILU: gated_backward4_as<CU32_ACT_SILU>(d, g, u, dg, du); break;
    case CU32_ACT_GELU: gated_backward4_as<CU32_ACT_GELU>(d, g, u, dg, du); break;
    case CU32_ACT_GELU_TANH: gated_backward4_as<CU32_ACT_GELU_TANH>(d, g, u, dg, du); break;
    case CU32_ACT_RELU: gated_backward4_as<CU32_ACT_RELU>(d, g, u, dg, du); break;
    default: gated_backward4_as<CU32_ACT_SIGMOID>(d, g, u, dg, du); break;
  }
}

}  // namespace dragon
