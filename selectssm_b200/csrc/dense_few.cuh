// The dense layer's forward for a few rows (single tokens while generating).
//
// y has rows * fout sums of fin products each: the weights are read once and
// everything else is small, so the pass is bound by how many of their bytes are
// in flight at once.  A CTA takes 64 (or 32) columns and a part of fin: eight
// neighbouring lanes (four) read one row's 128 bytes of bf16, each lane keeps
// eight columns of every row of x in registers, and the lanes, warps and the
// cluster's CTAs that share columns join their sums in a fixed order, the
// cluster through its shared memory.  Arithmetic is fp32 throughout.
#pragma once

#include "dense_mma.cuh"

namespace ssm {

constexpr int kFewRows = 16;     // most rows
constexpr int kFewMaxFin = 16384;  // its part of x, 16 rows in fp32, fits shared memory
constexpr int kFewThreads = 256;
constexpr int kFewAtOnce = 4;    // rows of the kernel a thread loads before it uses them

// R: rows held (1, 4 or 16), CT: columns of a CTA
template <typename T, int R, int CT>
__global__ void __launch_bounds__(kFewThreads)
    dense_few_kernel(const T* x, int64_t x_stride, const T* kernel, const __grid_constant__ DenseEpi e, int parts,
                     bool vec) {
  constexpr int kLanes = CT / 8, kRows = kFewThreads / kLanes, kWarps = kFewThreads / 32;
  extern __shared__ float sm[];
  float* xs = sm;                                       // [k][R] of this part
  __shared__ __align__(16) float sums[kWarps][R * CT];
  const int part = parts > 1 ? (int)cluster_rank() : 0, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int K = (int)e.K, k0 = (int)((int64_t)K * part / parts), k1 = (int)((int64_t)K * (part + 1) / parts);
  const int n0 = blockIdx.x / parts * CT, n = n0 + (threadIdx.x % kLanes) * 8, cnt = min(8, e.N - n);
  const int first = k0 + threadIdx.x / kLanes;

  Raw8<T> w[kFewAtOnce];
  const auto ask = [&](int k) {
    if (vec && cnt > 0)
#pragma unroll
      for (int i = 0; i < kFewAtOnce; ++i)
        if (k + i * kRows < k1) w[i].load(kernel + (int64_t)(k + i * kRows) * e.N + n);
  };
  ask(first);
  for (int i = threadIdx.x; i < (k1 - k0) * R; i += kFewThreads) {
    const int r = i / (k1 - k0), k = i - r * (k1 - k0);
    xs[k * R + r] = r < e.M ? Cvt<T>::to_f(x[r * x_stride + k0 + k]) : 0.f;
  }
  __syncthreads();
  float acc[R][8] = {};
  for (int k = first; k < k1; k += kFewAtOnce * kRows) {
#pragma unroll
    for (int i = 0; i < kFewAtOnce; ++i) {
      const int kk = k + i * kRows;
      if (kk >= k1 || cnt <= 0) break;
      float v[8];
      if (vec) w[i].get(v);
      else get8<T>(kernel, (int64_t)kk * e.N + n, cnt, false, v);
      const float* xr = xs + (kk - k0) * R;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float xv = xr[r];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[r][j] = fmaf(xv, v[j], acc[r][j]);
      }
    }
    ask(k + kFewAtOnce * kRows);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int o = kLanes; o < 32; o <<= 1) acc[r][j] += __shfl_xor_sync(0xffffffffu, acc[r][j], o);
      if (lane < kLanes) sums[warp][r * CT + lane * 8 + j] = acc[r][j];
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
  for (int i = threadIdx.x * parts + part; i < R * kLanes; i += kFewThreads * parts) {
    const int64_t m[1] = {i / kLanes};
    const int col = i % kLanes * 8;
    if (m[0] >= e.M || n0 + col >= e.N) continue;
    float v[1][8] = {}, bias[8], res[1][8] = {};
    for (int q = 0; q < parts; ++q) {
      const float* at = &sums[0][i / kLanes * CT + col];
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
      v[0][0] += lo.x; v[0][1] += lo.y; v[0][2] += lo.z; v[0][3] += lo.w;
      v[0][4] += hi.x; v[0][5] += hi.y; v[0][6] += hi.z; v[0][7] += hi.w;
    }
    dense_bias8(e, c, n0 + col, bias);
    if (e.residual) get8<T>(e.residual, m[0] * e.res_stride + n0 + col, e.N - n0 - col, c.vec_res, res[0]);
    dense_epilogue<T, 1>(e, c, m, n0 + col, bias, res, v);
  }
  __syncwarp();
  if (parts > 1) cluster_barrier();  // the others read this CTA's sums
}

}  // namespace ssm
