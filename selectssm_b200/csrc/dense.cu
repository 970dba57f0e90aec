// The dense layer with its epilogue (src/selectssm/selectssm.py:355-362):
//
//   pre = x W + bias,  u = keep * f * pre,  y = residual + act(u)
//   dpre = keep * f * dy * act'(u),  dx = dpre W^T,  dW = x^T dpre,  dbias = sum over rows of dpre
//
// keep and f are dropout's (philox.cuh), recomputed in both directions.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "philox.cuh"
#include "vec8.cuh"
#include "../../include/selectssm_b200.h"

namespace ssm {

int launch_error(const char* where, cudaError_t e);  // scan.cu
int bind_device(const void* ptr);                      // scan.cu

struct Epilogue {
  const void* bias;
  int32_t bias_dtype;
  const void* residual;
  int64_t res_stride;
  void* pre;
  DropRng rng;
  int32_t act;
  int32_t per_row;  // dropout blocks in a row
};

// C = A B with A (M, K) and B (K, N) at any strides; one 64 x 64 tile per CTA,
// 4 x 4 values per thread, fp32 FMA.
constexpr int kTile = 64, kDepth = 16;

template <typename T, typename TO, bool EPI>
__global__ void __launch_bounds__(256) dense_simt_kernel(const T* A, const T* B, TO* C, int64_t M, int64_t N, int64_t K,
                                                         int64_t sam, int64_t sak, int64_t sbk, int64_t sbn,
                                                         const Epilogue e) {
  __shared__ float as[kDepth][kTile + 4], bs[kDepth][kTile + 4];
  const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kTile;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += kDepth) {
#pragma unroll
    for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
      const int ak = sak == 1 ? i % kDepth : i / kTile, am = sak == 1 ? i / kDepth : i % kTile;
      as[ak][am] = m0 + am < M && k0 + ak < K ? Cvt<T>::to_f(A[(m0 + am) * sam + (k0 + ak) * sak]) : 0.f;
      const int bk = sbk == 1 ? i % kDepth : i / kTile, bn = sbk == 1 ? i / kDepth : i % kTile;
      bs[bk][bn] = n0 + bn < N && k0 + bk < K ? Cvt<T>::to_f(B[(k0 + bk) * sbk + (n0 + bn) * sbn]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = as[k][ty * 4 + i];
        b[i] = bs[k][tx * 4 + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
  PhiloxKey key = {};
  float f = 1.f;
  if (EPI && e.rng.drop) {
    key = philox_key(e.rng);
    f = keep_factor(e.rng.drop);
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    if (m >= M) break;
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx * 4 + j;
      if (n >= N) break;
      float v = acc[i][j];
      if (EPI) {
        if (e.bias)
          v += e.bias_dtype == SSM_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(e.bias)[n])
                                        : static_cast<const float*>(e.bias)[n];
        if (e.pre) static_cast<T*>(e.pre)[m * N + n] = Cvt<T>::from_f(v);
        if (e.rng.drop) {
          const uint32_t bits = keep_bits8(m * e.per_row + n / 8, key, e.rng.drop);
          v = bits >> (n & 7) & 1 ? v * f : 0.f;
        }
        v = act_f(v, e.act);
        if (e.residual) v += Cvt<T>::to_f(static_cast<const T*>(e.residual)[m * e.res_stride + n]);
      }
      C[m * N + n] = Cvt<TO>::from_f(v);
    }
  }
}

// dpre, rounded to the operand type of the two products that follow, and the
// column sums of its unrounded values over a run of rows.
constexpr int kDpreCols = 32, kDpreLanes = 8;
template <typename T>
__global__ void __launch_bounds__(kDpreCols* kDpreLanes)
    dense_dpre_kernel(const T* dy, int64_t dy_stride, const T* pre, T* dpre, float* part, int64_t M, int N,
                      int64_t run, int act, DropRng rng, int per_row) {
  __shared__ float red[kDpreLanes][kDpreCols];
  const int n = blockIdx.x * kDpreCols + threadIdx.x % kDpreCols, lane = threadIdx.x / kDpreCols;
  const int64_t m0 = (int64_t)blockIdx.y * run, m1 = m0 + run < M ? m0 + run : M;
  PhiloxKey key = {};
  float f = 1.f;
  if (rng.drop) {
    key = philox_key(rng);
    f = keep_factor(rng.drop);
  }
  float sum = 0.f;
  if (n < N)
    for (int64_t m = m0 + lane; m < m1; m += kDpreLanes) {
      float d = Cvt<T>::to_f(dy[m * dy_stride + n]);
      bool keep = true;
      if (rng.drop) keep = keep_bits8(m * per_row + n / 8, key, rng.drop) >> (n & 7) & 1;
      if (act != SSM_ACT_NONE) d *= act_grad_f(keep ? Cvt<T>::to_f(pre[m * N + n]) * f : 0.f, act);
      d = keep ? d * f : 0.f;
      sum += d;
      dpre[m * N + n] = Cvt<T>::from_f(d);
    }
  red[lane][threadIdx.x % kDpreCols] = sum;
  __syncthreads();
  if (lane == 0 && n < N) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kDpreLanes; ++i) s += red[i][threadIdx.x];
    part[(int64_t)blockIdx.y * N + n] = s;
  }
}

__global__ void dense_dbias_kernel(const float* part, int parts, int N, void* dbias, int dtype) {
  const int n = blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= N) return;
  float s = 0.f;
  for (int i = 0; i < parts; ++i) s += part[(int64_t)i * N + n];
  if (dtype == SSM_BF16) static_cast<__nv_bfloat16*>(dbias)[n] = __float2bfloat16_rn(s);
  else static_cast<float*>(dbias)[n] = s;
}

static bool known(int dtype) { return dtype == SSM_F32 || dtype == SSM_BF16; }

static int check_dense(const ssm_dense_params_t* p) {
  if (!p) return SSM_ERR_NULL;
  if (p->rows < 0 || p->rows > 0x7fffffff || p->fin < 1 || p->fout < 1 || p->fin > (1 << 24) || p->fout > (1 << 24) ||
      p->drop < 0 || p->drop > 65536 || p->act < SSM_ACT_NONE || p->act > SSM_ACT_RELU)
    return SSM_ERR_SHAPE;
  if ((p->x_stride && p->x_stride < p->fin) || (p->res_stride && p->res_stride < p->fout) ||
      (p->dy_stride && p->dy_stride < p->fout))
    return SSM_ERR_SHAPE;
  if (!known(p->dtype) || !known(p->bias_dtype) || !known(p->dkernel_dtype)) return SSM_ERR_DTYPE;
  return SSM_OK;
}

static size_t round256(size_t v) { return (v + 255) / 256 * 256; }
static size_t elem_bytes(int dtype) { return dtype == SSM_BF16 ? 2 : 4; }
static DropRng drop_rng(const ssm_dense_params_t* p) { return {p->seed, p->offset, p->rng, (uint32_t)p->drop}; }

// rows of dpre that one CTA sums for dbias
static int64_t dpre_run(const ssm_dense_params_t* p) {
  const int64_t tiles = (p->fout + kDpreCols - 1) / kDpreCols, want = (8 * 148 + tiles - 1) / tiles;
  const int64_t run = (p->rows + want - 1) / want;
  return run < 32 ? 32 : run;
}

static int launched(const char* where, unsigned n) {
  note_launches(n);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SSM_OK : launch_error(where, e);
}

template <typename T>
static int dense_fwd(const ssm_dense_params_t* p, cudaStream_t s) {
  Epilogue e;
  e.bias = p->bias;
  e.bias_dtype = p->bias_dtype;
  e.residual = p->residual;
  e.res_stride = p->res_stride ? p->res_stride : p->fout;
  e.pre = p->pre;
  e.rng = drop_rng(p);
  e.act = p->act;
  e.per_row = (p->fout + 7) / 8;
  const dim3 grid((p->fout + kTile - 1) / kTile, (unsigned)((p->rows + kTile - 1) / kTile));
  if (grid.y > 65535) return SSM_ERR_SHAPE;
  dense_simt_kernel<T, T, true><<<grid, 256, 0, s>>>(
      static_cast<const T*>(p->x), static_cast<const T*>(p->kernel), static_cast<T*>(p->y), p->rows, p->fout, p->fin,
      p->x_stride ? p->x_stride : p->fin, 1, p->fout, 1, e);
  return launched("launch dense kernel", 1);
}

template <typename T>
static int dense_bwd(const ssm_dense_params_t* p, cudaStream_t s) {
  const int64_t M = p->rows, run = dpre_run(p);
  const int N = p->fout, K = p->fin, parts = (int)((M + run - 1) / run);
  char* w = static_cast<char*>(p->workspace);
  T* dpre = reinterpret_cast<T*>(w);
  float* part = reinterpret_cast<float*>(w + round256((size_t)M * N * sizeof(T)));
  dense_dpre_kernel<T><<<dim3((N + kDpreCols - 1) / kDpreCols, parts), kDpreCols * kDpreLanes, 0, s>>>(
      static_cast<const T*>(p->dy), p->dy_stride ? p->dy_stride : N, static_cast<const T*>(p->pre), dpre, part, M, N, run,
      p->act, drop_rng(p), (N + 7) / 8);
  int st = launched("launch dense dpre kernel", 1);
  if (st) return st;
  if (p->dbias) {
    dense_dbias_kernel<<<(N + 127) / 128, 128, 0, s>>>(part, parts, N, p->dbias, p->bias_dtype);
    st = launched("launch dense dbias kernel", 1);
    if (st) return st;
  }
  const Epilogue none = {};
  const int64_t xs = p->x_stride ? p->x_stride : K;
  if (p->dx) {
    const dim3 grid((K + kTile - 1) / kTile, (unsigned)((M + kTile - 1) / kTile));
    dense_simt_kernel<T, T, false><<<grid, 256, 0, s>>>(dpre, static_cast<const T*>(p->kernel), static_cast<T*>(p->dx), M,
                                                        K, N, N, 1, 1, N, none);
    st = launched("launch dense dx kernel", 1);
    if (st) return st;
  }
  if (p->dkernel) {
    const dim3 grid((N + kTile - 1) / kTile, (K + kTile - 1) / kTile);
    if (p->dkernel_dtype == SSM_BF16)
      dense_simt_kernel<T, __nv_bfloat16, false><<<grid, 256, 0, s>>>(
          static_cast<const T*>(p->x), dpre, static_cast<__nv_bfloat16*>(p->dkernel), K, N, M, 1, xs, N, 1, none);
    else
      dense_simt_kernel<T, float, false><<<grid, 256, 0, s>>>(static_cast<const T*>(p->x), dpre,
                                                              static_cast<float*>(p->dkernel), K, N, M, 1, xs, N, 1, none);
    st = launched("launch dense dkernel kernel", 1);
    if (st) return st;
  }
  return SSM_OK;
}

}  // namespace ssm

using namespace ssm;

extern "C" {

size_t ssm_dense_fwd_workspace_bytes(const ssm_dense_params_t* p) { return check_dense(p) ? 0 : 0; }

size_t ssm_dense_bwd_workspace_bytes(const ssm_dense_params_t* p) {
  if (check_dense(p) || p->rows == 0) return 0;
  const int64_t run = dpre_run(p), parts = (p->rows + run - 1) / run;
  return round256((size_t)p->rows * p->fout * elem_bytes(p->dtype)) + round256((size_t)parts * p->fout * sizeof(float));
}

int ssm_dense_act_fwd(const ssm_dense_params_t* p, ssm_stream_t stream) {
  int st = check_dense(p);
  if (st) return st;
  if (p->rows == 0) return SSM_OK;
  if (!p->x || !p->kernel || !p->y) return SSM_ERR_NULL;
  if (p->workspace_bytes < ssm_dense_fwd_workspace_bytes(p)) return SSM_ERR_WORKSPACE;
  st = bind_device(p->x);
  if (st) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return p->dtype == SSM_BF16 ? dense_fwd<__nv_bfloat16>(p, s) : dense_fwd<float>(p, s);
}

int ssm_dense_act_bwd(const ssm_dense_params_t* p, ssm_stream_t stream) {
  int st = check_dense(p);
  if (st) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (p->rows == 0) {
    const size_t bytes[2] = {(size_t)p->fin * p->fout * elem_bytes(p->dkernel_dtype),
                             (size_t)p->fout * elem_bytes(p->bias_dtype)};
    void* dst[2] = {p->dkernel, p->dbias};
    for (int i = 0; i < 2; ++i) {
      if (!dst[i]) continue;
      st = bind_device(dst[i]);
      if (st) return st;
      const cudaError_t e = cudaMemsetAsync(dst[i], 0, bytes[i], s);
      if (e != cudaSuccess) return launch_error("cudaMemsetAsync(dense gradients)", e);
    }
    return SSM_OK;
  }
  if (!p->dy || (p->act != SSM_ACT_NONE && !p->pre) || (p->dx && !p->kernel) || (p->dkernel && !p->x))
    return SSM_ERR_NULL;
  if (!p->workspace || p->workspace_bytes < ssm_dense_bwd_workspace_bytes(p)) return SSM_ERR_WORKSPACE;
  st = bind_device(p->dy);
  if (st) return st;
  return p->dtype == SSM_BF16 ? dense_bwd<__nv_bfloat16>(p, s) : dense_bwd<float>(p, s);
}

}  // extern "C"
