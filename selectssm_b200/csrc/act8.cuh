// The activations and their derivatives for pairs of values, in packed fp32
// (add, mul and fma of two values are one instruction each).  Every pass of the
// block operators is near the limit of instructions issued, and this form takes
// about two thirds of the unpacked one's.
//
// With s(t) = 1 / (1 + e^-t):  silu(x) = x s(x), and gelu in its tanh form is
// x s(2 z), z = sqrt(2/pi) (x + 0.044715 x^3), because (1 + tanh z) / 2 = s(2 z).
#pragma once

#include "common.cuh"

namespace ssm {

// 1 / (1 + 2^t); 2^t overflowing to infinity gives 0
__device__ __forceinline__ float2 inv1p_ex2(float2 t) {
  const float2 d = fadd2(make_float2(ex2(t.x), ex2(t.y)), dup2(1.f));
  return make_float2(rcp(d.x), rcp(d.y));
}
// -2 z log2(e) as x (c1 + c3 x^2)
constexpr float kGelu1 = -2.f * kGeluC * kLog2e, kGelu3 = kGelu1 * 0.044715f;

// relu: NaN stays NaN (fmaxf would return the 0)
__device__ __forceinline__ float relu1(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
  return y;
}

template <int ACT>
__device__ __forceinline__ float2 act2(float2 x) {
  if constexpr (ACT == 1) return fmul2(x, inv1p_ex2(fmul2(x, dup2(-kLog2e))));
  if constexpr (ACT == 2) return fmul2(x, inv1p_ex2(fmul2(x, ffma2(fmul2(x, x), dup2(kGelu3), dup2(kGelu1)))));
  if constexpr (ACT == 3) return make_float2(relu1(x.x), relu1(x.y));
  return x;
}

template <int ACT>
__device__ __forceinline__ float2 slope2(float2 x) {
  if constexpr (ACT == 1) {  // s + x s (1 - s)
    const float2 s = inv1p_ex2(fmul2(x, dup2(-kLog2e)));
    return ffma2(fmul2(x, s), fsub2(dup2(1.f), s), s);
  }
  if constexpr (ACT == 2) {  // s + x s (1 - s) 2 z'
    const float2 q = fmul2(x, x);
    const float2 s = inv1p_ex2(fmul2(x, ffma2(q, dup2(kGelu3), dup2(kGelu1))));
    const float2 dz = ffma2(q, dup2(6.f * kGeluC * 0.044715f), dup2(2.f * kGeluC));
    return ffma2(fmul2(fmul2(x, s), fsub2(dup2(1.f), s)), dz, s);
  }
  if constexpr (ACT == 3) return make_float2(x.x <= 0.f ? 0.f : 1.f, x.y <= 0.f ? 0.f : 1.f);  // 1 at NaN, as PyTorch's
  return dup2(1.f);
}

// v = act(v)
template <int ACT>
__device__ __forceinline__ void act8(float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 y = act2<ACT>(make_float2(v[i], v[i + 1]));
    v[i] = y.x;
    v[i + 1] = y.y;
  }
}
// d = d act'(u)
template <int ACT>
__device__ __forceinline__ void slope8(float (&d)[8], const float (&u)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 y = fmul2(make_float2(d[i], d[i + 1]), slope2<ACT>(make_float2(u[i], u[i + 1])));
    d[i] = y.x;
    d[i + 1] = y.y;
  }
}
__device__ __forceinline__ void add8(float (&v)[8], const float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 y = fadd2(make_float2(v[i], v[i + 1]), make_float2(b[i], b[i + 1]));
    v[i] = y.x;
    v[i + 1] = y.y;
  }
}
__device__ __forceinline__ void scale8(float (&v)[8], float f) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 y = fmul2(make_float2(v[i], v[i + 1]), dup2(f));
    v[i] = y.x;
    v[i + 1] = y.y;
  }
}

}  // namespace ssm
