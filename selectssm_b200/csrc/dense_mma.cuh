// C = A B on the tensor cores (tcgen05), with the dense layer's epilogue.
//
// A is (M, K), B is (K, N), each as one bf16 plane or, for fp32 operands, as
// three whose sum is the fp32 value exactly (8 + 8 + 8 significant bits).  The
// product of two such sums is formed from the six plane pairs of weight above
// 2^-24, smallest first, so the accumulator is small while the corrections go
// in and only the last K / 16 steps round at the size of the result.
//
// A persistent CTA walks over items (tile of 128 x BN, part of the K loop).
// Warp 0 moves 64-deep slices of the operands to shared memory by TMA (128-byte
// swizzle), warp 1 issues the products, and warps 4 to 11 read the finished
// accumulator from tensor memory, apply the epilogue and store; two
// accumulators let the epilogue of one tile overlap the products of the next.
#pragma once

#include <cstdint>

#include "common.cuh"
#include "philox.cuh"
#include "vec8.cuh"

namespace ssm {

enum DenseOut { kOutF32 = 0, kOutBF16 = 1, kOutPartial = 2 };

// bf16 planes of an operand, element (row, col) of plane p at
// base[p * plane + row * ld + col]; `cols` is its contiguous axis.
struct Planes {
  const __nv_bfloat16* base;
  int64_t plane, ld;
  bool k_major;  // rows are M (or N) and columns K; otherwise rows are K
  __device__ __forceinline__ float at(int64_t mn, int64_t k) const {
    const __nv_bfloat16* q = base + (k_major ? mn * ld + k : k * ld + mn);
    return __bfloat162float(q[0]) + __bfloat162float(q[plane]) + __bfloat162float(q[2 * plane]);
  }
};

struct DenseEpi {
  int64_t M, K;
  int32_t N;
  int32_t planes;      // 1 or 3
  Planes a, b;
  int32_t out_kind;    // DenseOut
  void* out;           // (M, N) dense, or partials (splits, M, N) fp32
  // the forward's epilogue; all absent for the gradients' products
  const void* bias;
  int32_t bias_bf16;
  int32_t act;
  const void* residual;
  int64_t res_stride;
  void* pre;
  int32_t per_row;
  DropRng rng;
};

template <typename T>
__device__ __forceinline__ void put8(void* base, int64_t off, int cnt, bool vec, const float (&v)[8]) {
  T* p = static_cast<T*>(base) + off;
  if (vec) {
    store8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < cnt) p[i] = Cvt<T>::from_f(v[i]);
  }
}
template <typename T>
__device__ __forceinline__ void get8(const void* base, int64_t off, int cnt, bool vec, float (&v)[8]) {
  const T* p = static_cast<const T*>(base) + off;
  if (vec) {
    load8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < cnt ? Cvt<T>::to_f(p[i]) : 0.f;
  }
}

// What is the same for every element of a launch.
struct EpiConst {
  PhiloxKey key;
  float f;
  bool vec_out, vec_res;
  __device__ __forceinline__ explicit EpiConst(const DenseEpi& e) {
    key = {};
    f = 1.f;
    if (e.rng.drop) {
      key = philox_key(e.rng);
      f = keep_factor(e.rng.drop);
    }
    // rows of a multiple of 8 elements from a 16-byte aligned start
    const auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    vec_out = e.N % 8 == 0 && a16(e.out) && a16(e.pre);
    vec_res = e.residual && e.N % 8 == 0 && e.res_stride % 8 == 0 && a16(e.residual);
  }
};

// bias of columns n .. n+7, zeros where there is none
__device__ __forceinline__ void dense_bias8(const DenseEpi& e, int n, float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    b[i] = 0.f;
    if (e.bias && n + i < e.N)
      b[i] = e.bias_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(e.bias)[n + i])
                         : static_cast<const float*>(e.bias)[n + i];
  }
}

// Columns n .. n+7 (those below N) of row m from the summed products v.
__device__ __forceinline__ void dense_epilogue8(const DenseEpi& e, const EpiConst& c, int64_t m, int n,
                                                const float (&bias)[8], float (&v)[8]) {
  const int cnt = min(8, e.N - n);
  if (e.planes == 3) {
    // An infinite operand has no finite planes besides its first, and infinity
    // times the other operand's planes gives NaN where the product is infinite.
    // Such elements are summed again from the fp32 values.
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < cnt && isnan(v[i])) {
        float s = 0.f;
        for (int64_t k = 0; k < e.K; ++k) s = fmaf(e.a.at(m, k), e.b.at(n + i, k), s);
        v[i] = s;
      }
  }
  const int64_t off = m * e.N + n;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += bias[i];
  if (e.pre) {
    if (e.out_kind == kOutBF16) put8<__nv_bfloat16>(e.pre, off, cnt, c.vec_out, v);
    else put8<float>(e.pre, off, cnt, c.vec_out, v);
  }
  if (e.rng.drop) {
    const uint32_t bits = keep_bits8(m * e.per_row + n / 8, c.key, e.rng.drop);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bits >> i & 1 ? v[i] * c.f : 0.f;
  }
  switch (e.act) {
    case 1:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_f(v[i], 1);
      break;
    case 2:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_f(v[i], 2);
      break;
    case 3:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_f(v[i], 3);
      break;
    default: break;
  }
  if (e.residual) {
    float r[8];
    const int64_t ro = m * e.res_stride + n;
    if (e.out_kind == kOutBF16) get8<__nv_bfloat16>(e.residual, ro, cnt, c.vec_res, r);
    else get8<float>(e.residual, ro, cnt, c.vec_res, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
  }
  if (e.out_kind == kOutBF16) put8<__nv_bfloat16>(e.out, off, cnt, c.vec_out, v);
  else put8<float>(e.out, off, cnt, c.vec_out, v);
}

// ---------------------------------------------------------------- tensor-core pieces
constexpr int kBM = 128, kBK = 64;
constexpr int kMmaThreads = 384;
constexpr int kEpiWarps = 8;
// Polls before a wait gives up; a tile takes microseconds, so this is far above any wait that ends.
constexpr uint32_t kMmaSpin = 1u << 20;

// Shared-memory operand descriptor, 128-byte swizzle.  K-major rows of 128
// bytes: groups of 8 rows are 1024 bytes apart.  MN-major rows (one k each, 64
// values of m or n): groups of 8 k are 1024 bytes apart, the next 64 values of
// m or n 8192 bytes.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  constexpr uint64_t kLead = 8192 >> 4, kStep = 1024 >> 4;
  return (uint64_t)((addr >> 4) & 0x3fff) | kLead << 16 | kStep << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// bf16 x bf16 -> fp32, M rows, N columns
constexpr uint32_t mma_idesc(int m, int n, bool a_mn, bool b_mn) {
  return 1u << 4 | 1u << 7 | 1u << 10 | (a_mn ? 1u : 0u) << 15 | (b_mn ? 1u : 0u) << 16 | (uint32_t)(n >> 3) << 17 |
         (uint32_t)(m >> 4) << 24;
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

struct DenseWork {
  int32_t tiles_m, tiles_n, splits;
  int32_t kblocks;  // ceil(K / 64)
  int32_t steps;    // kblocks * plane pairs
};

template <int BN>
struct MmaSmem {
  static constexpr int kA = kBM * kBK * 2, kB = BN * kBK * 2, kStage = kA + kB;
  static constexpr int kStages = BN == 256 ? 4 : 6;
  static constexpr int kEpi = kEpiWarps * 4096;  // 32 x 32 fp32 for each epilogue warp
  static constexpr int kBytes = kStages * kStage + kEpi + 1024;  // and alignment
};

// plane pairs (of A, of B), smallest products first
__device__ __forceinline__ void plane_pair(int planes, int seg, int& pa, int& pb) {
  if (planes == 1) {
    pa = pb = 0;
    return;
  }
  pa = 0x001012 >> (4 * seg) & 15;  // 2 1 0 1 0 0
  pb = 0x010210 >> (4 * seg) & 15;  // 0 1 2 0 1 0
}

template <bool A_MN, bool B_MN, int BN>
__global__ void __launch_bounds__(kMmaThreads, 1)
    dense_mma_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const __grid_constant__ DenseEpi e, const DenseWork w, int32_t* status) {
  using S = MmaSmem<BN>;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t full[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base;
  __shared__ volatile int dead;
  uint8_t* tiles = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpiWarps);
    }
    dead = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 2) tmem_alloc(&tmem_base, 2 * BN);
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  const uint32_t tmem = tmem_base;
  const int items = w.tiles_m * w.tiles_n * w.splits;

  // Bounded wait; a role that gives up (or sees that another did) stops.
  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < kMmaSpin; ++i) {
      if (mbar_try_wait(bar, parity)) return true;
      if ((i & 63) == 63 && dead) return false;
    }
    dead = 1;
    report(status, kStatusTimeout);
    return false;
  };

  if (warp == 0 && lane == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const int n0 = item % w.tiles_n * BN, rest = item / w.tiles_n;
      const int m0 = rest % w.tiles_m * kBM, split = rest / w.tiles_m;
      const int t0 = (int)((int64_t)w.steps * split / w.splits), t1 = (int)((int64_t)w.steps * (split + 1) / w.splits);
      for (int t = t0; t < t1; ++t) {
        if (!wait(&empty[stage], phase ^ 1)) {
          ok = false;
          break;
        }
        int pa, pb;
        const int seg = t / w.kblocks, k0 = (t - seg * w.kblocks) * kBK;
        plane_pair(e.planes, seg, pa, pb);
        uint8_t* sa = tiles + stage * S::kStage;
        uint8_t* sb = sa + S::kA;
        mbar_arrive_expect_tx(&full[stage], S::kStage);
        if (A_MN) {
#pragma unroll
          for (int j = 0; j < kBM / 64; ++j) tma_load_3d(sa + j * 8192, &map_a, &full[stage], m0 + 64 * j, k0, pa);
        } else {
          tma_load_3d(sa, &map_a, &full[stage], k0, m0, pa);
        }
        if (B_MN) {
#pragma unroll
          for (int j = 0; j < BN / 64; ++j) tma_load_3d(sb + j * 8192, &map_b, &full[stage], n0 + 64 * j, k0, pb);
        } else {
          tma_load_3d(sb, &map_b, &full[stage], k0, n0, pb);
        }
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // Loads still in flight when the products stopped early: wait for the last
    // ones so that none lands after the CTA has gone.
    if (!ok)
      for (int i = 0; i < S::kStages; ++i) {
        mbar_wait_bounded(&full[stage], phase ^ 1, 1u << 16);
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = mma_idesc(kBM, BN, A_MN, B_MN);
    constexpr uint32_t kStepA = (A_MN ? 2048 : 32) >> 4, kStepB = (B_MN ? 2048 : 32) >> 4;
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const int split = item / w.tiles_n / w.tiles_m;
      const int t0 = (int)((int64_t)w.steps * split / w.splits), t1 = (int)((int64_t)w.steps * (split + 1) / w.splits);
      if (!wait(&acc_empty[acc], acc_phase ^ 1)) break;
      tmem_fence_after_sync();
      const uint32_t d = tmem + acc * BN;
      for (int t = t0; t < t1; ++t) {
        if (!wait(&full[stage], phase)) {
          ok = false;
          break;
        }
        tmem_fence_after_sync();
        const uint32_t sa = smem_u32(tiles + stage * S::kStage);
        const uint64_t da = smem_desc(sa), db = smem_desc(sa + S::kA);
#pragma unroll
        for (int k = 0; k < kBK / 16; ++k) mma_f16(d, da + k * kStepA, db + k * kStepB, idesc, t > t0 || k > 0);
        mma_commit(&empty[stage]);
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      mma_commit(&acc_full[acc]);
      if (!ok) mbar_wait_bounded(&acc_full[acc], acc_phase, 1u << 16);  // products still running use the buffers
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  } else if (warp >= 4) {
    const EpiConst c(e);
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    uint4* stage = reinterpret_cast<uint4*>(tiles + S::kStages * S::kStage) + (warp - 4) * 256;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      const int n0 = item % w.tiles_n * BN, rest = item / w.tiles_n;
      const int64_t m0 = (int64_t)(rest % w.tiles_m) * kBM + quarter * 32;
      const int split = rest / w.tiles_m;
      if (!__all_sync(0xffffffffu, wait(&acc_full[acc], acc_phase))) break;
      tmem_fence_after_sync();
      const uint32_t src = tmem + acc * BN + half * (BN / 2) + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int j = 0; j < BN / 2; j += 32) {
        const int n = n0 + half * (BN / 2) + j;
        if (n >= e.N) break;
        // A lane reads 32 columns of its own row of the accumulator; through
        // shared memory (16-byte pieces, swizzled by row) it gets eight
        // columns of four rows, so that four lanes cover 32 columns of a row
        // in global memory and the eight share one dropout counter.
        uint32_t r[2][16];
        tmem_ld16(src + j, r[0]);
        tmem_ld16(src + j + 16, r[1]);
        const int nl = n + (lane & 3) * 8;
        float bias[8];
        dense_bias8(e, nl, bias);
        tmem_wait_ld();
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q)
          stage[lane * 8 + (q ^ (lane & 7))] = make_uint4(r[q >> 2][(q & 3) * 4], r[q >> 2][(q & 3) * 4 + 1],
                                                          r[q >> 2][(q & 3) * 4 + 2], r[q >> 2][(q & 3) * 4 + 3]);
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int row = q * 8 + (lane >> 2);
          const int64_t m = m0 + row;
          const uint4 lo = stage[row * 8 + (((lane & 3) * 2) ^ (row & 7))];
          const uint4 hi = stage[row * 8 + (((lane & 3) * 2 + 1) ^ (row & 7))];
          float v[8] = {__uint_as_float(lo.x), __uint_as_float(lo.y), __uint_as_float(lo.z), __uint_as_float(lo.w),
                        __uint_as_float(hi.x), __uint_as_float(hi.y), __uint_as_float(hi.z), __uint_as_float(hi.w)};
          if (m >= e.M || nl >= e.N) continue;
          if (e.out_kind == kOutPartial)
            put8<float>(e.out, ((int64_t)split * e.M + m) * e.N + nl, min(8, e.N - nl), c.vec_out, v);
          else
            dense_epilogue8(e, c, m, nl, bias, v);
        }
      }
      tmem_fence_before_sync();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
      __syncwarp();
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  }
  __syncwarp();
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  if (warp == 2) tmem_dealloc(tmem, 2 * BN);
}

// The epilogue of a product whose K loop was cut: the parts summed in order.
__global__ void __launch_bounds__(256) dense_join_kernel(const float* part, int splits, const __grid_constant__ DenseEpi e) {
  const EpiConst c(e);
  const int64_t blocks = e.M * ((e.N + 7) / 8), per = (e.N + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= blocks) return;
  const int64_t m = i / per;
  const int n = (int)(i - m * per) * 8, cnt = min(8, e.N - n);
  const bool vec = e.N % 8 == 0;
  float v[8], t[8];
  get8<float>(part, m * e.N + n, cnt, vec, v);
  for (int s = 1; s < splits; ++s) {
    get8<float>(part, ((int64_t)s * e.M + m) * e.N + n, cnt, vec, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += t[k];
  }
  float bias[8];
  dense_bias8(e, n, bias);
  dense_epilogue8(e, c, m, n, bias, v);
}

}  // namespace ssm
