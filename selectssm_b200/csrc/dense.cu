// The dense layer with its epilogue (src/selectssm/selectssm.py:355-362):
//
//   pre = x W + bias,  u = keep * f * pre,  y = residual + act(u)
//   dpre = keep * f * dy * act'(u),  dx = dpre W^T,  dW = x^T dpre,  dbias = sum over rows of dpre
//
// keep and f are dropout's (philox.cuh), recomputed in both directions.  The
// three products run on the tensor cores (dense_mma.cuh) over bf16 planes: a
// bf16 operand whose rows TMA can address is read where it lies; an fp32 one is
// split into three planes, and rows TMA cannot address (a stride or start that
// is not a multiple of 16 bytes) are copied to padded ones, by one pass over it.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense_few.cuh"
#include "dense_mma.cuh"
#include "../../include/selectssm_b200.h"

namespace ssm {

int launch_error(const char* where, cudaError_t e);  // scan.cu
int bind_device(const void* ptr);                      // scan.cu

// ---------------------------------------------------------------- operands
// Splits v into bf16 values that sum to it exactly: each takes the leading 8
// bits of what is left.  A value that would round to infinity is cut instead.
__device__ __forceinline__ void split3(float v, float (&h)[3]) {
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    float r = __bfloat162float(__float2bfloat16_rn(v));
    if (isinf(r) && !isinf(v)) r = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
    h[p] = r;
    v = isinf(v) ? 0.f : v - r;
  }
}

template <int PLANES>
__device__ __forceinline__ void store_planes(__nv_bfloat16* dst, int64_t plane, const float (&v)[8]) {
  if (PLANES == 1) {
    store8(dst, v);
  } else {
    // Pairs are converted together and need no second conversion to be stored;
    // values that would round to infinity, and infinities, take the long way.
    float rest[8];
    bool large = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      rest[i] = v[i];
      large |= fabsf(v[i]) > __uint_as_float(0x7f7f0000u);  // the largest bf16 value
    }
    if (!large) {
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(rest[2 * i], rest[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&b);
          const float2 left = fsub2(make_float2(rest[2 * i], rest[2 * i + 1]),
                                    make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)));
          rest[2 * i] = left.x;
          rest[2 * i + 1] = left.y;
        }
        *reinterpret_cast<uint4*>(dst + p * plane) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      return;
    }
    float h[8][3], t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) split3(v[i], h[i]);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = h[i][p];
      store8(dst + p * plane, t);
    }
  }
}

// What has to be ready before the products, in one launch (a small call's time is
// its launches'): up to two operands as planes, and dbias from its runs' sums.
// (300 x 500) @ (500 x 400), fp32, forward and backward: 150 us of the host's time,
// 163 with a launch for each.  16384 x 768 twice in fp32: 36 us for 252 MB, 7 TB/s.
struct Pack {  // (rows, cols) at row stride `stride` to planes of row length ld, a multiple of 8; zeros beyond cols
  const void* src;
  __nv_bfloat16* dst;
  int64_t stride, rows;
  int cols, ld;
  bool vec;
};
struct Ready {
  Pack pack[2];
  int64_t blocks[2];  // CTAs of each, 0 where it is read in place
  const float* sums;  // (parts, n)
  int parts, n;
  void* dbias;
  bool dbias_bf16;
  int64_t all() const { return blocks[0] + blocks[1] + (dbias ? (n + 7) / 8 : 0); }
};

template <typename T, int PLANES>
__global__ void __launch_bounds__(256) dense_ready_kernel(const __grid_constant__ Ready g) {
  int64_t blk = blockIdx.x;
  if (blk < g.blocks[0] + g.blocks[1]) {  // eight columns a thread
    const Pack& o = g.pack[blk >= g.blocks[0]];
    if (blk >= g.blocks[0]) blk -= g.blocks[0];
    const int per = o.ld / 8;
    const int64_t i = blk * 256 + threadIdx.x;
    if (i >= o.rows * per) return;
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 8;
    float v[8];
    get8<T>(static_cast<const T*>(o.src), r * o.stride + c, o.cols - c, o.vec && c + 8 <= o.cols, v);
    store_planes<PLANES>(o.dst + r * o.ld + c, o.rows * o.ld, v);
    return;
  }
  blk -= g.blocks[0] + g.blocks[1];
  __shared__ float red[32][9];  // eight columns a CTA, 32 threads a column, in a fixed order
  const int col = threadIdx.x & 7, lane = threadIdx.x >> 3, n = (int)blk * 8 + col;
  float s = 0.f;
  if (n < g.n)
#pragma unroll 4
    for (int i = lane; i < g.parts; i += 32) s += g.sums[(int64_t)i * g.n + n];
  red[lane][col] = s;
  __syncthreads();
  if (lane == 0 && n < g.n) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += red[i][col];
    if (g.dbias_bf16) static_cast<__nv_bfloat16*>(g.dbias)[n] = __float2bfloat16_rn(t);
    else static_cast<float*>(g.dbias)[n] = t;
  }
}

template <typename T>
constexpr int kDpreRows = sizeof(T) == 2 ? 4 : 2;
constexpr int kDpreCtas = 3;  // on an SM

// dpre as planes for the two products that follow, and the column sums of its
// unrounded values over a run of rows.  In bf16 it is one plane, as `pre` was kept in
// bf16: the operands' own precision, for half and a quarter of the bytes of fp32 and of
// three planes.  It costs accuracy that 32-bit arithmetic with bf16 results would have:
// dx and dW of 32768 x 768 -> 1536, silu, 0.0024 off 64-bit ones (norms), 0.0017 there.  A thread keeps eight columns (one
// dropout counter each row) and takes ROWS rows at a time, whose loads it issues
// together: a loop that loads, computes and stores row by row ran at half the
// rate.  32768 x 1536 bf16, silu, dropout, dbias: 62 us for 302 MB, 4.9 TB/s; issue (54%
// of cycles) and latency at 80 registers, where HBM alone would take 46.
template <typename T, int PLANES, bool WRITE, int ACT>
__global__ void __launch_bounds__(256, kDpreCtas)
    dense_dpre_kernel(const T* dy, int64_t dy_stride, const T* pre, __nv_bfloat16* dpre, int ld, float* part, int64_t M,
                      int N, int64_t run, int cb, DropRng rng, bool vec) {
  constexpr int ROWS = kDpreRows<T>;
  extern __shared__ float red[];
  const int per_row = (N + 7) / 8, rl = 256 / cb;
  const int lane = threadIdx.x / cb, blk = blockIdx.x * cb + threadIdx.x % cb, n = blk * 8;
  const int64_t m0 = (int64_t)blockIdx.y * run, m1 = min(m0 + run, M);
  PhiloxKey key = {};
  float f = 1.f;
  if (rng.drop) {
    key = philox_key(rng);
    f = keep_factor(rng.drop);
  }
  float sum[8] = {};
  if (lane < rl && blk < per_row) {
    const int cnt = min(8, N - n);
    const T* pd = dy + (m0 + lane) * dy_stride + n;
    const T* pp = ACT ? pre + (m0 + lane) * N + n : nullptr;
    __nv_bfloat16* po = dpre + (m0 + lane) * ld + n;
    int64_t counter = (m0 + lane) * per_row + blk;
    int left = m1 > m0 + lane ? (int)((m1 - m0 - lane + rl - 1) / rl) : 0;  // rows of this thread
    for (; left > 0; left -= ROWS) {
      Raw8<T> rd[ROWS], ru[ROWS];
      if (vec) {
#pragma unroll
        for (int q = 0; q < ROWS; ++q)
          if (q < left) {
            rd[q].load(pd + q * rl * dy_stride);
            if (ACT) ru[q].load(pp + (int64_t)q * rl * N);
          }
      }
#pragma unroll
      for (int q = 0; q < ROWS; ++q) {
        if (q >= left) break;
        float d[8], u[8];
        if (vec) {
          rd[q].get(d);
          if (ACT) ru[q].get(u);
        } else {
          get8<T>(pd, q * rl * dy_stride, cnt, false, d);
          if (ACT) get8<T>(pp, (int64_t)q * rl * N, cnt, false, u);
        }
        if (ACT) {
          scale8(u, f);
          slope8<ACT>(d, u);
        }
        if (rng.drop) {
          scale8(d, f);
          keep8(philox4x32_10(counter + q * rl * per_row, key), rng.drop, d);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += d[i];
        if (WRITE) store_planes<PLANES>(po + (int64_t)q * rl * ld, M * ld, d);
      }
      pd += ROWS * rl * dy_stride;
      if (ACT) pp += (int64_t)ROWS * rl * N;
      po += (int64_t)ROWS * rl * ld;
      counter += (int64_t)ROWS * rl * per_row;
    }
  }
  if (!part) return;
  if (lane < rl)
#pragma unroll
    for (int i = 0; i < 8; ++i) red[(lane * cb + threadIdx.x % cb) * 8 + i] = sum[i];
  __syncthreads();
  for (int c = threadIdx.x; c < cb * 8; c += 256) {
    const int col = blockIdx.x * cb * 8 + c;
    if (col >= N) break;
    float s = 0.f;
    for (int i = 0; i < rl; ++i) s += red[i * cb * 8 + c];
    part[(int64_t)blockIdx.y * N + col] = s;
  }
}

// ---------------------------------------------------------------- checks and sizes
static bool known(int dtype) { return dtype == SSM_F32 || dtype == SSM_BF16; }
static size_t elem_bytes(int dtype) { return dtype == SSM_BF16 ? 2 : 4; }

static int check_dense(const ssm_dense_params_t* p) {
  if (!p) return SSM_ERR_NULL;
  if (p->rows < 0 || p->rows > 0x7fffff00 || p->fin < 1 || p->fout < 1 || p->fin > (1 << 24) || p->fout > (1 << 24) ||
      p->drop < 0 || p->drop > 65536 || p->act < SSM_ACT_NONE || p->act > SSM_ACT_RELU)
    return SSM_ERR_SHAPE;
  if ((p->x_stride && p->x_stride < p->fin) || (p->res_stride && p->res_stride < p->fout) ||
      (p->dy_stride && p->dy_stride < p->fout))
    return SSM_ERR_SHAPE;
  if (!known(p->dtype) || !known(p->bias_dtype) || !known(p->dkernel_dtype)) return SSM_ERR_DTYPE;
  if (!all_aligned(elem_bytes(p->dtype), {p->x, p->kernel, p->residual, p->y, p->pre, p->dy, p->dx}) ||
      !all_aligned(elem_bytes(p->bias_dtype), {p->bias, p->dbias}) || !all_aligned(elem_bytes(p->dkernel_dtype), {p->dkernel}) ||
      !all_aligned(sizeof(uint64_t), {p->rng}) || !all_aligned(sizeof(int32_t), {p->status}) ||
      !all_aligned(kWorkspaceAlign, {p->workspace}))
    return SSM_ERR_ALIGN;
  return SSM_OK;
}

static size_t round256(size_t v) { return (v + 255) / 256 * 256; }
static DropRng drop_rng(const ssm_dense_params_t* p) { return {p->seed, p->offset, p->rng, (uint32_t)p->drop}; }
static int pad8(int n) { return (n + 7) / 8 * 8; }
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int planes_of(const ssm_dense_params_t* p) { return p->dtype == SSM_BF16 ? 1 : 3; }
static int64_t stride_or(int64_t s, int64_t dense) { return s ? s : dense; }

static int launched(const char* where, unsigned n) {
  note_launches(n);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SSM_OK : launch_error(where, e);
}

// An operand of a product: (rows, cols), cols contiguous.
struct Operand {
  const void* src;
  int64_t stride, rows;
  int cols;
  bool bf16;
  // read in place: bf16 rows TMA can address (a null pointer counts as aligned)
  bool direct() const { return bf16 && stride % 8 == 0 && aligned16(src); }
  size_t bytes() const { return direct() ? 0 : round256((size_t)rows * pad8(cols) * 2 * (bf16 ? 1 : 3)); }
};

static Operand x_operand(const ssm_dense_params_t* p) {
  return {p->x, stride_or(p->x_stride, p->fin), p->rows, p->fin, p->dtype == SSM_BF16};
}
static Operand kernel_operand(const ssm_dense_params_t* p) {
  return {p->kernel, p->fout, p->fin, p->fout, p->dtype == SSM_BF16};
}

// The planes of an operand: read in place, or packed into `ws` by pack `slot` of `ready`.
static Planes planes(const Operand& o, bool k_major, char* ws, Ready* ready, int slot) {
  if (o.direct()) return {static_cast<const __nv_bfloat16*>(o.src), 0, o.stride, k_major};
  const int ld = pad8(o.cols);
  __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(ws);
  ready->pack[slot] = {o.src, dst, o.stride, o.rows, o.cols, ld, aligned16(o.src) && o.stride % (o.bf16 ? 8 : 4) == 0};
  ready->blocks[slot] = ceil_div(o.rows * (ld / 8), 256);
  return {dst, o.rows * ld, ld, k_major};
}

static int launch_ready(const Ready& g, bool bf16, cudaStream_t s) {
  const int64_t grid = g.all();
  if (grid == 0) return SSM_OK;
  if (grid > 0x7fffffff) return SSM_ERR_SHAPE;
  if (bf16) dense_ready_kernel<__nv_bfloat16, 1><<<(unsigned)grid, 256, 0, s>>>(g);
  else dense_ready_kernel<float, 3><<<(unsigned)grid, 256, 0, s>>>(g);
  return launched("launch dense ready kernel", 1);
}

// ---------------------------------------------------------------- one product
constexpr int kSms = 148;

struct Plan {
  bool pair;
  DenseWork w;
  size_t part_bytes;
};

// Tile (128 x 128 by one CTA, 256 x 256 by a pair) and cuts of the K loop: the
// choice with the least estimated time.  The terms are measured: a 64-deep step
// takes 0.22 us of a single CTA's and 0.36 of a pair's, all six products of three
// planes 1.2 us; an item 3 us around its steps, a pair's 4.5; and joining cut
// products a launch, a share of a round trip for each part, and the parts' way
// through memory.  (bf16, one way against the other: 8192 x 768 x 768 14 us by
// single CTAs and 16 by pairs, 16384 x 768 x 1536 38 and 35, 768 x 1536 of
// K 32768 67 and 59.)
static Plan plan_product(int64_t M, int64_t N, int64_t K, int planes) {
  Plan best = {};
  double least = 0;
  for (int pair = 0; pair < (planes == 3 ? 1 : 2); ++pair) {
    const double step = planes == 3 ? 1.2 : pair ? 0.36 : 0.22, item = pair ? 4.5 : 3;
    DenseWork w;
    w.tiles_m = (int)ceil_div(M, pair ? Tile<true, float>::kM : Tile<false, float>::kM);
    w.tiles_n = (int)ceil_div(N, pair ? Tile<true, float>::kN : Tile<false, float>::kN);
    w.kblocks = (int)ceil_div(K, kBK);
    const int64_t tiles = (int64_t)w.tiles_m * w.tiles_n, teams = pair ? kSms / 2 : kSms;
    for (w.splits = 1; w.splits == 1 || (w.splits * tiles <= 2 * teams && w.splits <= w.kblocks &&
                                         (planes == 3 || w.splits * 4 <= w.kblocks));
         ++w.splits) {
      const double rounds = (double)ceil_div(tiles * w.splits, teams);
      double us = rounds * (ceil_div(w.kblocks, w.splits) * step + item);
      if (w.splits > 1) us += 3.5 + (w.splits < kJoinShared ? 0.35 * w.splits : 2 + 0.09 * w.splits) +
                              w.splits * 2.0 * (double)M * N * 4 / 5e6;
      if (least == 0 || us < least) {
        best.pair = pair;
        best.w = w;
        least = us;
      }
    }
  }
  best.part_bytes = best.w.splits > 1 ? round256((size_t)best.w.splits * M * pad8((int)N) * sizeof(float)) : 0;
  return best;
}

static bool operand_map(CUtensorMap* m, const Planes& o, int64_t rows, int64_t cols, int planes) {
  const uint64_t ld = (uint64_t)o.ld * 2;
  return make_map(m, o.base, true, cols, rows, planes, ld, planes == 3 ? (uint64_t)o.plane * 2 : ld, kBK,
                  o.k_major ? 128 : kBK, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool A_MN, bool B_MN, bool PAIR, int PLANES, typename T>
static int launch_mma(const DenseEpi& e, const Plan& q, const CUtensorMap& ma, const CUtensorMap& mb, int32_t* status,
                      cudaStream_t s) {
  const auto kernel = dense_mma_kernel<A_MN, B_MN, PAIR, PLANES, T>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<PAIR, T>::kBytes);
  if (err != cudaSuccess) return launch_error("cudaFuncSetAttribute(dense)", err);
  const int items = q.w.tiles_m * q.w.tiles_n * q.w.splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(PAIR ? 2 * std::min(items, kSms / 2) : std::min(items, kSms));
  cfg.blockDim = dim3(kMmaThreads);
  cfg.dynamicSmemBytes = Tile<PAIR, T>::kBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2 : 1;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, kernel, ma, mb, e, q.w, status);
  note_launches(1);
  return err == cudaSuccess ? SSM_OK : launch_error("launch dense product kernel", err);
}

// The bounds of a product's waits; `omit` leaves the last item's loads out (the self-test).
struct DenseWait {
  int32_t* status;
  uint32_t spin;
  bool omit;
};

// e.M, e.N, e.K, e.a, e.b and the epilogue are set; `part` holds plan_product's part_bytes.
template <bool A_MN, bool B_MN, typename T>
static int product(DenseEpi e, float* part, const DenseWait& wait, cudaStream_t s) {
  Plan q = plan_product(e.M, e.N, e.K, e.planes);
  int32_t* status = wait.status;
  e.per_row = (e.N + 7) / 8;
  if ((int64_t)q.w.tiles_m * q.w.tiles_n * q.w.splits > 0x7fffffff) return SSM_ERR_SHAPE;
  q.w.loaded = q.w.tiles_m * q.w.tiles_n * q.w.splits - (wait.omit ? 1 : 0);
  q.w.spin = wait.spin;
  CUtensorMap ma, mb;
  if (!operand_map(&ma, e.a, A_MN ? e.K : e.M, A_MN ? e.M : e.K, e.planes) ||
      !operand_map(&mb, e.b, B_MN ? e.K : e.N, B_MN ? e.N : e.K, e.planes))
    return SSM_ERR_LAUNCH;
  DenseEpi first = e;
  if (q.w.splits > 1) {
    first.partial = part;
    first.residual = first.bias = nullptr;
  }
  // only a kernel's gradient has another type than the operands
  constexpr bool kAny = A_MN && B_MN;
  int st = SSM_ERR_DTYPE;
  if constexpr (sizeof(T) == 4 || kAny)
    if (e.planes == 3) st = launch_mma<A_MN, B_MN, false, 3, T>(first, q, ma, mb, status, s);
  if constexpr (sizeof(T) == 2 || kAny)
    if (e.planes == 1)
      st = q.pair ? launch_mma<A_MN, B_MN, true, 1, T>(first, q, ma, mb, status, s)
                  : launch_mma<A_MN, B_MN, false, 1, T>(first, q, ma, mb, status, s);
  if (st || q.w.splits == 1) return st;
  const int64_t chunks = ceil_div(e.M, 32) * ceil_div(e.N, kCW);
  const int64_t grid = q.w.splits >= kJoinShared ? chunks : ceil_div(chunks, kJoinWarps);
  if (grid > 0x7fffffff) return SSM_ERR_SHAPE;
  dense_join_kernel<T><<<(unsigned)grid, 32 * kJoinWarps, 0, s>>>(part, q.w.splits, e);
  return launched("launch dense join kernel", 1);
}

// ---------------------------------------------------------------- forward and backward
static bool few_rows(const ssm_dense_params_t* p) { return p->rows <= kFewRows && p->fin <= kFewMaxFin; }

constexpr size_t kFewPart = 128 * 1024;  // most bytes of x a CTA holds

template <typename T, int R, int CT, int V>
static int launch_few(const ssm_dense_params_t* p, const DenseEpi& e, cudaStream_t s) {
  const int tiles = (int)ceil_div(p->fout, CT);
  // parts of fin: enough CTAs for the SMs, and at least 64 rows of the kernel each
  // (and few enough for x's part to fit: 16384 rows of 16 values need all eight)
  const int64_t useful = std::min<int64_t>({8, ceil_div(kSms, tiles), p->fin / 64});
  const int parts = (int)std::max<int64_t>({1, useful, ceil_div((int64_t)p->fin * R * sizeof(float), kFewPart)});
  const size_t smem = (size_t)ceil_div(p->fin, parts) * R * sizeof(float) + R * sizeof(float);
  const auto kernel = dense_few_kernel<T, R, CT, V>;
  cudaError_t err;
  if (smem > 16 * 1024) {
    // The limit belongs to the kernel, not to this launch: always the same one (a part's, and
    // a row for its rounding up and one behind it), as another thread may be launching too.
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)(kFewPart + 2 * R * sizeof(float)));
    if (err != cudaSuccess) return launch_error("cudaFuncSetAttribute(dense few rows)", err);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts * tiles);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool vec = p->fout % V == 0 && reinterpret_cast<uintptr_t>(p->kernel) % std::min<size_t>(16, V * sizeof(T)) == 0;
  err = cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(p->x), stride_or(p->x_stride, p->fin),
                           static_cast<const T*>(p->kernel), e, parts, vec);
  note_launches(1);
  return err == cudaSuccess ? SSM_OK : launch_error("launch dense few rows kernel", err);
}
template <typename T>
static int dense_few(const ssm_dense_params_t* p, const DenseEpi& e, cudaStream_t s) {
  if (p->rows > 4) return launch_few<T, 16, 64, 2>(p, e, s);
  if (p->rows > 1) return launch_few<T, 4, 64, 2>(p, e, s);
  // 64 columns read 128 bytes of bf16 a row; 32 where that leaves SMs without work
  return ceil_div(p->fout, 64) * 8 >= kSms ? launch_few<T, 1, 64, 8>(p, e, s) : launch_few<T, 1, 32, 8>(p, e, s);
}

static int dense_fwd(const ssm_dense_params_t* p, const DenseWait& wait, cudaStream_t s) {
  char* ws = static_cast<char*>(p->workspace);
  DenseEpi e = {};
  int st = SSM_OK;
  const bool few = few_rows(p);
  if (!few) {
    const Operand x = x_operand(p), w = kernel_operand(p);
    Ready ready = {};
    e.a = planes(x, true, ws, &ready, 0);
    e.b = planes(w, false, ws + x.bytes(), &ready, 1);
    ws += x.bytes() + w.bytes();
    st = launch_ready(ready, p->dtype == SSM_BF16, s);
    if (st) return st;
  }
  e.M = p->rows;
  e.N = p->fout;
  e.K = p->fin;
  e.planes = few ? 0 : planes_of(p);
  e.out = p->y;
  e.bias = p->bias;
  e.bias_bf16 = p->bias_dtype == SSM_BF16;
  e.act = p->act;
  e.residual = p->residual;
  e.res_stride = stride_or(p->res_stride, p->fout);
  e.pre = p->pre;
  e.per_row = (p->fout + 7) / 8;
  e.rng = drop_rng(p);
  if (few) return p->dtype == SSM_BF16 ? dense_few<__nv_bfloat16>(p, e, s) : dense_few<float>(p, e, s);
  float* part = reinterpret_cast<float*>(ws);
  return p->dtype == SSM_BF16 ? product<false, true, __nv_bfloat16>(e, part, wait, s)
                              : product<false, true, float>(e, part, wait, s);
}

// How the dpre pass cuts (rows, fout): cb blocks of eight columns a CTA, `run` rows.
struct DpreGeom {
  int cb, tiles, parts;
  int64_t run;
};
static DpreGeom dpre_geom(const ssm_dense_params_t* p) {
  DpreGeom g;
  const int per_row = (p->fout + 7) / 8;
  g.tiles = (int)ceil_div(per_row, 32);
  g.cb = (int)ceil_div(per_row, g.tiles);
  const int rl = 256 / g.cb;
  // bf16: as many CTAs as the SMs hold at once, with long runs (131072 x 768 120 us, 133 with
  // 256 parts of each column's sum; 32768 x 1536 62 for 67).  fp32, whose rounds are twice as
  // long, is better off with more (32768 x 1536 119 and 112): one round of the rows' loads a
  // CTA, more where that made over 256 parts.
  const int64_t round = (int64_t)rl * (p->dtype == SSM_BF16 ? kDpreRows<__nv_bfloat16> : kDpreRows<float>);
  if (p->dtype == SSM_BF16) g.run = std::max(round, ceil_div(p->rows, std::max(1, kDpreCtas * kSms / g.tiles)));
  else g.run = round * ceil_div(p->rows, 256 * round);
  g.parts = (int)ceil_div(p->rows, g.run);
  return g;
}

// dy serves as dpre itself
static bool dpre_is_dy(const ssm_dense_params_t* p) {
  return p->dtype == SSM_BF16 && p->act == SSM_ACT_NONE && p->drop == 0 && stride_or(p->dy_stride, p->fout) % 8 == 0 &&
         aligned16(p->dy);
}

template <typename T, int PLANES, int ACT>
static int launch_dpre_act(const ssm_dense_params_t* p, __nv_bfloat16* dpre, float* part, cudaStream_t s) {
  const DpreGeom g = dpre_geom(p);
  const dim3 grid(g.tiles, g.parts);
  const size_t smem = (size_t)(256 / g.cb) * g.cb * 8 * sizeof(float);
  const int64_t ds = stride_or(p->dy_stride, p->fout);
  const bool vec = p->fout % 8 == 0 && ds % 8 == 0 && aligned16(p->dy) && aligned16(p->pre);
  const T *dy = static_cast<const T*>(p->dy), *pre = static_cast<const T*>(p->pre);
  if (dpre)
    dense_dpre_kernel<T, PLANES, true, ACT><<<grid, 256, smem, s>>>(dy, ds, pre, dpre, pad8(p->fout), part, p->rows,
                                                                    p->fout, g.run, g.cb, drop_rng(p), vec);
  else
    dense_dpre_kernel<T, PLANES, false, ACT><<<grid, 256, smem, s>>>(dy, ds, pre, dpre, pad8(p->fout), part, p->rows,
                                                                     p->fout, g.run, g.cb, drop_rng(p), vec);
  return launched("launch dense dpre kernel", 1);
}
template <typename T, int PLANES>
static int launch_dpre(const ssm_dense_params_t* p, __nv_bfloat16* dpre, float* part, cudaStream_t s) {
  switch (p->act) {
    case SSM_ACT_SILU: return launch_dpre_act<T, PLANES, SSM_ACT_SILU>(p, dpre, part, s);
    case SSM_ACT_GELU: return launch_dpre_act<T, PLANES, SSM_ACT_GELU>(p, dpre, part, s);
    case SSM_ACT_RELU: return launch_dpre_act<T, PLANES, SSM_ACT_RELU>(p, dpre, part, s);
    default: return launch_dpre_act<T, PLANES, SSM_ACT_NONE>(p, dpre, part, s);
  }
}

struct BwdBytes {
  size_t dpre, sums, x, kernel, part;
  size_t all() const { return dpre + sums + x + kernel + part; }
};
static BwdBytes bwd_bytes(const ssm_dense_params_t* p) {
  const int pl = planes_of(p);
  BwdBytes b;
  b.dpre = round256((size_t)p->rows * pad8(p->fout) * 2 * pl);  // also when dy serves: pointers may be unknown here
  b.sums = round256((size_t)dpre_geom(p).parts * p->fout * sizeof(float));
  b.x = x_operand(p).bytes();
  b.kernel = kernel_operand(p).bytes();
  b.part = std::max(plan_product(p->rows, p->fin, p->fout, pl).part_bytes,
                    plan_product(p->fin, p->fout, p->rows, pl).part_bytes);
  return b;
}

static int dense_bwd(const ssm_dense_params_t* p, const DenseWait& wait, cudaStream_t s) {
  const int pl = planes_of(p), N = p->fout, K = p->fin, ld = pad8(N);
  const BwdBytes bytes = bwd_bytes(p);
  char* ws = static_cast<char*>(p->workspace);
  __nv_bfloat16* dpre = reinterpret_cast<__nv_bfloat16*>(ws);
  float* sums = reinterpret_cast<float*>(ws + bytes.dpre);
  ws += bytes.dpre + bytes.sums;
  const bool same = dpre_is_dy(p);
  int st = SSM_OK;
  if (!same || p->dbias)
    st = pl == 1 ? launch_dpre<__nv_bfloat16, 1>(p, same ? nullptr : dpre, p->dbias ? sums : nullptr, s)
                 : launch_dpre<float, 3>(p, dpre, p->dbias ? sums : nullptr, s);
  if (st) return st;
  Ready ready = {};
  if (p->dbias) {
    ready.sums = sums;
    ready.parts = dpre_geom(p).parts;
    ready.n = N;
    ready.dbias = p->dbias;
    ready.dbias_bf16 = p->bias_dtype == SSM_BF16;
  }
  Planes x = {}, kernel = {};
  if (p->dkernel) x = planes(x_operand(p), false, ws, &ready, 0);
  if (p->dx) kernel = planes(kernel_operand(p), true, ws + bytes.x, &ready, 1);
  st = launch_ready(ready, p->dtype == SSM_BF16, s);
  if (st) return st;
  const Planes d = same ? Planes{static_cast<const __nv_bfloat16*>(p->dy), 0, stride_or(p->dy_stride, N), true}
                        : Planes{dpre, p->rows * ld, ld, true};
  float* part = reinterpret_cast<float*>(ws + bytes.x + bytes.kernel);
  DenseEpi e = {};
  e.planes = pl;
  if (p->dx) {  // (rows, fout) (fin, fout)^T
    e.a = d;
    e.b = kernel;
    e.M = p->rows;
    e.N = K;
    e.K = N;
    e.out = p->dx;
    st = p->dtype == SSM_BF16 ? product<false, false, __nv_bfloat16>(e, part, wait, s)
                              : product<false, false, float>(e, part, wait, s);
    if (st) return st;
  }
  if (p->dkernel) {  // (rows, fin)^T (rows, fout)
    e.a = x;
    e.b = d;
    e.b.k_major = false;
    e.M = K;
    e.N = N;
    e.K = p->rows;
    e.out = p->dkernel;
    st = p->dkernel_dtype == SSM_BF16 ? product<true, true, __nv_bfloat16>(e, part, wait, s)
                                      : product<true, true, float>(e, part, wait, s);
  }
  return st;
}

}  // namespace ssm

using namespace ssm;

static int dense_fwd_call(const ssm_dense_params_t* p, const DenseWait& wait, ssm_stream_t stream) {
  int st = check_dense(p);
  if (st) return st;
  if (p->rows == 0) return SSM_OK;
  if (!p->x || !p->kernel || !p->y) return SSM_ERR_NULL;
  const size_t need = ssm_dense_fwd_workspace_bytes(p);
  if (need && (!p->workspace || p->workspace_bytes < need)) return SSM_ERR_WORKSPACE;
  st = bind_device(p->x);
  if (st) return st;
  return dense_fwd(p, wait, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" {

size_t ssm_dense_fwd_workspace_bytes(const ssm_dense_params_t* p) {
  if (check_dense(p) || p->rows == 0 || few_rows(p)) return 0;
  return x_operand(p).bytes() + kernel_operand(p).bytes() +
         plan_product(p->rows, p->fout, p->fin, planes_of(p)).part_bytes;
}

size_t ssm_dense_bwd_workspace_bytes(const ssm_dense_params_t* p) {
  if (check_dense(p) || p->rows == 0) return 0;
  return bwd_bytes(p).all();
}

int ssm_dense_act_fwd(const ssm_dense_params_t* p, ssm_stream_t stream) {
  return dense_fwd_call(p, {p ? p->status : nullptr, kMmaSpin, false}, stream);
}

int ssm_selftest_dense_timeout(const ssm_dense_params_t* p, uint32_t spin_limit, ssm_stream_t stream) {
  int st = check_dense(p);
  if (st) return st;
  if (!p->status) return SSM_ERR_NULL;
  if (p->rows == 0 || few_rows(p) || spin_limit < 2 || spin_limit > kMmaSpin) return SSM_ERR_SHAPE;
  return dense_fwd_call(p, {p->status, spin_limit, true}, stream);
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
  return dense_bwd(p, {p->status, kMmaSpin, false}, s);
}

}  // extern "C"
