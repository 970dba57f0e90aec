// The dense layer's forward for a few rows (single tokens while generating).
//
// y has rows * fout sums of fin products each: the weights are read once and
// everything else is small, so the pass is bound by how many of their bytes are
// in flight at once.  A CTA takes CT columns and a part of fin, a lane V
// columns of every row of x, summed in registers.  One row takes V = 8 (one
// 16-byte load of bf16 a lane, and lanes that share columns join by shuffles);
// more rows take V = 2, where a warp's lanes share one row of the kernel, so
// that x is read from shared memory by broadcast, four rows at a time, and no
// shuffles are needed (16 rows of 1024 x 512 in fp32: 19 us with V = 8).  Warps
// and the cluster's CTAs join their sums in a fixed order, the cluster through
// its shared memory.  Arithmetic is fp32 throughout.
//
// 1 x 768 x 1536 in bf16: 6.7 us, 12 rows of 1024 x 512 in fp32: 9.4 us; the 2.4 and
// 2.1 MB of weights are 0.4 us of HBM's time, the rest a launch, a round trip to
// memory and the cluster's join.
#pragma once

#include "dense_mma.cuh"

namespace ssm {

constexpr int kFewRows = 16;     // most rows
constexpr int kFewMaxFin = 16384;  // its part of x, 16 rows in fp32, fits shared memory
constexpr int kFewThreads = 256;

// V consecutive values as they lie in memory
template <typename T, int V> struct RawV;
template <typename T> struct RawV<T, 8> : Raw8<T> {};
template <> struct RawV<float, 2> {
  float2 r;
  __device__ __forceinline__ void load(const float* p) { r = __ldcs(reinterpret_cast<const float2*>(p)); }
  __device__ __forceinline__ void get(float (&v)[2]) const { v[0] = r.x; v[1] = r.y; }
};
template <> struct RawV<__nv_bfloat16, 2> {
  uint32_t r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = __ldcs(reinterpret_cast<const unsigned*>(p)); }
  __device__ __forceinline__ void get(float (&v)[2]) const {
    v[0] = __uint_as_float(r << 16);
    v[1] = __uint_as_float(r & 0xffff0000u);
  }
};

// R: rows held (1, 4 or 16), CT: columns of a CTA, V: columns of a lane
template <typename T, int R, int CT, int V>
__global__ void __launch_bounds__(kFewThreads)
    dense_few_kernel(const T* x, int64_t x_stride, const T* kernel, const __grid_constant__ DenseEpi e, int parts,
                     bool vec) {
  constexpr int kLanes = CT / V, kRows = kFewThreads / kLanes, kWarps = kFewThreads / 32;
  constexpr int kAtOnce = V == 8 ? 4 : 8;  // rows of the kernel a thread loads before it uses them
  extern __shared__ __align__(16) float xs[];  // [k][R] of this part
  __shared__ __align__(16) float sums[kWarps][R * CT];
  const int part = parts > 1 ? (int)cluster_rank() : 0, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int K = (int)e.K, k0 = (int)((int64_t)K * part / parts), k1 = (int)((int64_t)K * (part + 1) / parts);
  const int n0 = blockIdx.x / parts * CT, n = n0 + (threadIdx.x % kLanes) * V;
  const bool in = n < e.N;
  const int first = k0 + threadIdx.x / kLanes;

  RawV<T, V> w[kAtOnce];
  const auto ask = [&](int k) {
    if (vec && in)
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
        if (k + i * kRows < k1) w[i].load(kernel + (int64_t)(k + i * kRows) * e.N + n);
  };
  ask(first);
  for (int i = threadIdx.x; i < (k1 - k0) * R; i += kFewThreads) {
    const int r = i / (k1 - k0), k = i - r * (k1 - k0);
    xs[k * R + r] = r < e.M ? Cvt<T>::to_f(x[r * x_stride + k0 + k]) : 0.f;
  }
  __syncthreads();
  float acc[R][V] = {};
  for (int k = first; k < k1; k += kAtOnce * kRows) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int kk = k + i * kRows;
      if (kk >= k1 || !in) break;
      float v[V];
      if (vec) {
        w[i].get(v);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = n + j < e.N ? Cvt<T>::to_f(kernel[(int64_t)kk * e.N + n + j]) : 0.f;
      }
      float xr[R];
      if constexpr (R % 4 == 0) {
#pragma unroll
        for (int r = 0; r < R; r += 4) {
          const float4 q = *reinterpret_cast<const float4*>(xs + (kk - k0) * R + r);
          xr[r] = q.x; xr[r + 1] = q.y; xr[r + 2] = q.z; xr[r + 3] = q.w;
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) xr[r] = xs[(kk - k0) * R + r];
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[r][j] = fmaf(xr[r], v[j], acc[r][j]);
    }
    ask(k + kAtOnce * kRows);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int o = kLanes; o < 32; o <<= 1) acc[r][j] += __shfl_xor_sync(0xffffffffu, acc[r][j], o);
      if (lane < kLanes) sums[warp][r * CT + lane * V + j] = acc[r][j];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < R * CT; i += kFewThreads) {
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < kWarps; ++q) s += sums[q][i];
    sums[0][i] = s;  // only this thread reads or writes element i of any warp's
  }
  __syncthreads();
  if (parts > 1) cluster_barrier();
  // one block of eight columns of a row a thread, dealt out over the parts
  const EpiConst c(e);
  for (int i = threadIdx.x * parts + part; i < R * CT / 8; i += kFewThreads * parts) {
    const int64_t m = i / (CT / 8);
    const int col = i % (CT / 8) * 8;
    if (m >= e.M || n0 + col >= e.N) continue;
    float v[1][8] = {}, bias[8];
    for (int q = 0; q < parts; ++q) {
      const float* at = &sums[0][i / (CT / 8) * CT + col];
      float4 lo, hi;
      if (parts > 1) {
        uint32_t there;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_u32(at)), "r"(q));
        asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(lo.x), "=f"(lo.y), "=f"(lo.z), "=f"(lo.w)
                     : "r"(there) : "memory");
        asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(hi.x), "=f"(hi.y), "=f"(hi.z), "=f"(hi.w)
                     : "r"(there + 16) : "memory");
      } else {
        lo = *reinterpret_cast<const float4*>(at);
        hi = *reinterpret_cast<const float4*>(at + 4);
      }
      const float t[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      add8(v[0], t);
    }
    dense_bias8(e, c, n0 + col, bias);
    dense_epilogue<T, 1>(
        e, c, m, n0 + col, bias, v,
        [&](float (&res)[1][8]) {
          get8<T>(e.residual, m * e.res_stride + n0 + col, e.N - n0 - col, c.vec_res, res[0]);
        },
        [&](void* base, const float (&u)[1][8]) { dense_put<T, 1>(e, c, base, m, 1, n0 + col, u); });
  }
  __syncwarp();
  if (parts > 1) cluster_barrier();  // the others read this CTA's sums
}

}  // namespace ssm
