// Dropout with an activation and a residual (src/selectssm/selectssm.py:355-362:
// h = act(dropout(mlp(x))), x = skip + dropout(mlp_proj(h))):
//
//   u = keep * x * f,  f = 65536 / (65536 - drop)
//   y = residual + act(u)                 dx = keep * f * dy * act'(u)
//
// keep comes from philox.cuh and is recomputed in the backward, so neither pass
// moves a mask: the forward reads x (and the residual) and writes y, the
// backward reads dy (and x, when act' needs it) and writes dx.
//
// One thread owns the eight columns of one counter.  Where rows are multiples
// of eight columns and 16-byte aligned they are moved with 16-byte accesses;
// otherwise a warp owns 32 such blocks, each lane draws its own block's bits,
// and the elements are moved one by one with neighbouring lanes on neighbouring
// addresses, taking address and bits from the block's lane by shuffle.
//
// Measured, 65536 x 768 bf16 with silu, cold: forward 45 us (201 MB, 4.5 TB/s),
// backward 53 us (302 MB, 5.7 TB/s).  131072 x 768: 84 and 100 us.
// Issue is what bounds both (65% of cycles: the generator, the selects on 16-bit
// draws, the activation), not HBM (38 and 55% of its peak).

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "act8.cuh"
#include "common.cuh"
#include "philox.cuh"
#include "vec8.cuh"
#include "../../include/selectssm_b200.h"

namespace ssm {

int launch_error(const char* where, cudaError_t e);  // scan.cu
int bind_device(const void* ptr);                      // scan.cu

constexpr int kDropThreads = 128;

struct DropArgs {
  int64_t blocks, rows;   // blocks of eight columns, all rows
  int32_t dim, per_row;   // columns, blocks in a row
  int64_t a_stride, b_stride;
  const void* a;          // forward x, backward dy
  const void* b;          // forward residual or null, backward x (null without an activation)
  void* out;              // dense
  DropRng rng;
};

// Eight elements of a block.  Forward: a = x, b = residual.  Backward: a = dy,
// b = x.  The mask enters by selection only, so that what a dropped place holds
// (NaN and infinities among it) has no effect; every activation here maps 0 to 0.
template <bool BWD, int ACT, bool HAS_B, typename KEEP>
__device__ __forceinline__ void drop_block(float (&a)[8], float (&b)[8], float f, KEEP keep) {
  scale8(a, f);
  if (BWD) {
    if (ACT) {
      scale8(b, f);
      slope8<ACT>(a, b);
    }
    keep(a);
  } else {
    keep(a);
    act8<ACT>(a);
    if (HAS_B)
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] += b[i];
  }
}

template <typename T, bool BWD, int ACT, bool HAS_B, int UNROLL>
__global__ void __launch_bounds__(kDropThreads) dropout_vec_kernel(const DropArgs p) {
  const PhiloxKey key = philox_key(p.rng);
  const float f = keep_factor(p.rng.drop);
  const T* A = static_cast<const T*>(p.a);
  const T* B = static_cast<const T*>(p.b);
  T* out = static_cast<T*>(p.out);
  // A CTA's blocks are an aligned run of a power of two, so their counters
  // share the upper word, and with it the two of the generator's products that
  // depend on no other part of the counter.
  static_assert((kDropThreads * UNROLL & (kDropThreads * UNROLL - 1)) == 0);
  const int64_t run = (int64_t)blockIdx.x * (kDropThreads * UNROLL);
  const int64_t first = run + threadIdx.x;
  const uint32_t upper = (uint32_t)(run >> 32);
  const bool dense = p.a_stride == p.dim && (!HAS_B || p.b_stride == p.dim);
  Raw8<T> a[UNROLL], b[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int64_t blk = first + u * kDropThreads;
    if (blk < p.blocks) {
      int64_t ao = blk * 8, bo = ao;
      if (!dense) {
        const int64_t row = blk / p.per_row;
        const int64_t col = (blk - row * p.per_row) * 8;
        ao = row * p.a_stride + col;
        bo = row * p.b_stride + col;
      }
      a[u].load(A + ao);
      if (HAS_B) b[u].load(B + bo);
    }
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int64_t blk = first + u * kDropThreads;
    if (blk >= p.blocks) break;
    float x[8], r[8];
    a[u].get(x);
    if (HAS_B) b[u].get(r);
    drop_block<BWD, ACT, HAS_B>(x, r, f, [&](float (&v)[8]) {
      if (p.rng.drop) keep8(philox4x32_10((uint32_t)blk, upper, key), p.rng.drop, v);
    });
    store8(out + blk * 8, x);
  }
}

template <typename T, bool BWD, int ACT, bool HAS_B>
__global__ void __launch_bounds__(kDropThreads) dropout_any_kernel(const DropArgs p) {
  const PhiloxKey key = philox_key(p.rng);
  const float f = keep_factor(p.rng.drop);
  const T* A = static_cast<const T*>(p.a);
  const T* B = static_cast<const T*>(p.b);
  T* out = static_cast<T*>(p.out);
  const int lane = threadIdx.x & 31;
  const int64_t blk = (int64_t)blockIdx.x * kDropThreads + threadIdx.x;
  int64_t row = 0;
  int col = 0, cnt = 0;
  uint32_t m = 0;
  if (blk < p.blocks) {
    row = blk / p.per_row;
    col = (int)(blk - row * p.per_row) * 8;
    cnt = min(8, p.dim - col);
    if (p.rng.drop) for_kept8(philox4x32_10(blk, key), p.rng.drop, [&](int i, bool keep) { m |= (uint32_t)keep << i; });
    else m = 0xff;
  }
  float a[8], b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int src = 4 * j + (lane >> 3), i = lane & 7;
    const int64_t r = __shfl_sync(0xffffffffu, row, src);
    const int c = __shfl_sync(0xffffffffu, col, src) + i;
    const bool ok = i < __shfl_sync(0xffffffffu, cnt, src);
    a[j] = ok ? Cvt<T>::to_f(A[r * p.a_stride + c]) : 0.f;
    b[j] = HAS_B && ok ? Cvt<T>::to_f(B[r * p.b_stride + c]) : 0.f;
  }
  uint32_t kept = 0;  // bit j: this lane's element of blocks 4 j ..
#pragma unroll
  for (int j = 0; j < 8; ++j)
    kept |= (__shfl_sync(0xffffffffu, m, 4 * j + (lane >> 3)) >> (lane & 7) & 1) << j;
  drop_block<BWD, ACT, HAS_B>(a, b, f, [&](float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = kept >> j & 1 ? v[j] : 0.f;
  });
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int src = 4 * j + (lane >> 3), i = lane & 7;
    const int64_t r = __shfl_sync(0xffffffffu, row, src);
    const int c = __shfl_sync(0xffffffffu, col, src) + i;
    if (i < __shfl_sync(0xffffffffu, cnt, src)) out[r * p.dim + c] = Cvt<T>::from_f(a[j]);
  }
}

template <typename T, bool BWD, int ACT, bool HAS_B>
static int launch_drop(const DropArgs& p, cudaStream_t s) {
  const bool vec = p.dim % 8 == 0 && aligned16(p.a) && aligned16(p.out) && (!HAS_B || aligned16(p.b)) &&
                   p.a_stride * sizeof(T) % 16 == 0 && (!HAS_B || p.b_stride * sizeof(T) % 16 == 0);
  constexpr int kUnroll = sizeof(T) == 2 ? 4 : 2;  // 64 bytes of each input in flight a thread
  const int64_t per = vec ? kDropThreads * kUnroll : kDropThreads;
  const int64_t grid = (p.blocks + per - 1) / per;
  if (grid > 0x7fffffff) return SSM_ERR_SHAPE;
  if (vec)
    dropout_vec_kernel<T, BWD, ACT, HAS_B, kUnroll><<<(unsigned)grid, kDropThreads, 0, s>>>(p);
  else
    dropout_any_kernel<T, BWD, ACT, HAS_B><<<(unsigned)grid, kDropThreads, 0, s>>>(p);
  note_launches(1);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SSM_OK : launch_error("launch dropout kernel", e);
}

template <typename T, bool BWD, int ACT>
static int launch_drop_b(const DropArgs& p, cudaStream_t s) {
  if constexpr (BWD) return launch_drop<T, BWD, ACT, ACT != 0>(p, s);
  else return p.b ? launch_drop<T, BWD, ACT, true>(p, s) : launch_drop<T, BWD, ACT, false>(p, s);
}

template <typename T, bool BWD>
static int launch_drop_act(const DropArgs& p, int act, cudaStream_t s) {
  switch (act) {
    case SSM_ACT_SILU: return launch_drop_b<T, BWD, SSM_ACT_SILU>(p, s);
    case SSM_ACT_GELU: return launch_drop_b<T, BWD, SSM_ACT_GELU>(p, s);
    case SSM_ACT_RELU: return launch_drop_b<T, BWD, SSM_ACT_RELU>(p, s);
    default: return launch_drop_b<T, BWD, SSM_ACT_NONE>(p, s);
  }
}

static int check_drop(const ssm_dropout_params_t* p) {
  if (!p) return SSM_ERR_NULL;
  if (p->rows < 0 || p->dim < 1 || p->dim > 0x7ffffff0 || p->drop < 0 || p->drop > 65536 || p->act < SSM_ACT_NONE ||
      p->act > SSM_ACT_RELU)
    return SSM_ERR_SHAPE;
  if ((p->x_stride && p->x_stride < p->dim) || (p->res_stride && p->res_stride < p->dim) ||
      (p->dy_stride && p->dy_stride < p->dim))
    return SSM_ERR_SHAPE;
  if (p->dtype != SSM_F32 && p->dtype != SSM_BF16) return SSM_ERR_DTYPE;
  if (!all_aligned(p->dtype == SSM_BF16 ? 2 : 4, {p->x, p->residual, p->y, p->dy, p->dx}) ||
      !all_aligned(sizeof(uint64_t), {p->rng}))
    return SSM_ERR_ALIGN;
  return SSM_OK;
}

static DropArgs drop_args(const ssm_dropout_params_t* p, bool bwd) {
  DropArgs a;
  a.rows = p->rows;
  a.dim = p->dim;
  a.per_row = (p->dim + 7) / 8;
  a.blocks = p->rows * a.per_row;
  const int64_t xs = p->x_stride ? p->x_stride : p->dim;
  a.a = bwd ? p->dy : p->x;
  a.a_stride = bwd ? (p->dy_stride ? p->dy_stride : p->dim) : xs;
  a.b = bwd ? p->x : p->residual;
  a.b_stride = bwd ? xs : (p->res_stride ? p->res_stride : p->dim);
  a.out = bwd ? p->dx : p->y;
  a.rng = {p->seed, p->offset, p->rng, (uint32_t)p->drop};
  return a;
}

}  // namespace ssm

using namespace ssm;

extern "C" {

int ssm_dropout_act_fwd(const ssm_dropout_params_t* p, ssm_stream_t stream) {
  int st = check_drop(p);
  if (st) return st;
  if (p->rows == 0) return SSM_OK;
  if (!p->x || !p->y) return SSM_ERR_NULL;
  st = bind_device(p->y);
  if (st) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const DropArgs a = drop_args(p, false);
  return p->dtype == SSM_BF16 ? launch_drop_act<__nv_bfloat16, false>(a, p->act, s)
                              : launch_drop_act<float, false>(a, p->act, s);
}

int ssm_dropout_act_bwd(const ssm_dropout_params_t* p, ssm_stream_t stream) {
  int st = check_drop(p);
  if (st) return st;
  if (p->rows == 0) return SSM_OK;
  if (!p->dy || !p->dx || (p->act != SSM_ACT_NONE && !p->x)) return SSM_ERR_NULL;
  st = bind_device(p->dx);
  if (st) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const DropArgs a = drop_args(p, true);
  return p->dtype == SSM_BF16 ? launch_drop_act<__nv_bfloat16, true>(a, p->act, s)
                              : launch_drop_act<float, true>(a, p->act, s);
}

}  // extern "C"
