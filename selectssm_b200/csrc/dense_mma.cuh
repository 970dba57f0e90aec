// C = A B on the tensor cores (tcgen05), with the dense layer's epilogue.
//
// A is (M, K), B is (K, N), each as one bf16 plane or, for fp32 operands, as
// three whose sum is the fp32 value exactly (8 + 8 + 8 significant bits).  The
// product of two such sums is formed from the six plane pairs of weight above
// 2^-24: the leading planes' in one accumulator, the other five, 2^-8 of it and
// less, in another.
//
// The tensor core cuts, not rounds, what an addition to an accumulator cannot
// hold, so an error grows with the number of additions.  For fp32 operands the
// leading accumulator therefore starts afresh every 512 of K (32 additions) and
// the other every 4096, and what they held is added in rounded fp32 to a sum that
// stays in tensor memory: a sum of 2042 products is good to 6e-7 so, 2.4e-6 without.
//
// A persistent CTA walks over items (tile of 128 x BN, part of the K loop).
// Warps 0 and 3 move 64-deep slices of A and of B to shared memory by TMA (128-byte
// swizzle), warp 1 issues the products, and warps 4 to 11 read the finished
// accumulator from tensor memory, apply the epilogue and store; two
// accumulators let the epilogue of one tile overlap the products of the next.
//
// Measured in bf16.  131072 x 1536 x 768, residual and dropout: 232 us, 1.33
// PFLOP/s; without the epilogue 197 us, 1.57 PFLOP/s, the rate of a plain library
// product at these sizes (203 us).  Call after call for seconds the power limit holds
// the SM clock at 1.06 GHz and they take 312 and 270 us, the library's 267 at 1.3 GHz.
// 32768 x 768 x 1536, silu, dropout and `pre`: 106 us, where the epilogue's issue is
// the bound (66 us without it), and its two gradients 59 and 55 us, 1.3 and 1.4
// PFLOP/s.  In fp32 8192 x 768 x 1536: 107 us with the planes' pass, 66% of the rate
// of six bf16 products; 2042 x 515 x 1001, forward and both gradients: 24, 25 and 21
// us, bound by the latency of the loads of one round of tiles.
#pragma once

#include <cstdint>

#include "act8.cuh"
#include "common.cuh"
#include "philox.cuh"
#include "vec8.cuh"

namespace ssm {

// bf16 planes of an operand, element (row, col) of plane p at
// base[p * plane + row * ld + col]; `cols` is its contiguous axis.
struct Planes {
  const __nv_bfloat16* base;
  int64_t plane, ld;
  bool k_major;  // rows are M (or N) and columns K; otherwise rows are K
};

struct DenseEpi {
  int64_t M, K;
  int32_t N;
  int32_t planes;      // 1 or 3
  Planes a, b;
  void* out;           // (M, N) dense, of the kernel's type T
  float* partial;      // not null: the sums go here, (splits, M, per_row * 8), and nothing else is done
  // the forward's epilogue; all absent for the gradients' products
  const void* bias;
  int32_t bias_bf16;
  int32_t act;
  const void* residual;
  int64_t res_stride;
  void* pre;
  int32_t per_row;     // blocks of eight columns in a row
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
  bool vec_out, vec_res, vec_bias, low;
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
    low = e.M * e.per_row <= (int64_t)1 << 32;
    vec_bias = e.N % 8 == 0 && a16(e.bias);
    vec_res = e.residual && e.N % 8 == 0 && e.res_stride % 8 == 0 && a16(e.residual);
  }
};

template <int ACT, int R>
__device__ __forceinline__ void act_rows(float (&v)[R][8]) {
#pragma unroll
  for (int q = 0; q < R; ++q) act8<ACT>(v[q]);
}

// bias of columns n .. n+7, zeros where there is none
__device__ __forceinline__ void dense_bias8(const DenseEpi& e, const EpiConst& c, int n, float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = 0.f;
  if (!e.bias || n >= e.N) return;
  if (e.bias_bf16) get8<__nv_bfloat16>(e.bias, n, e.N - n, c.vec_bias, b);
  else get8<float>(e.bias, n, e.N - n, c.vec_bias, b);
}

// What an epilogue does to columns n .. n+7 of R rows (row, row + 32 / R, ...)
// from the summed products v.  Not all of the rows exist, and only get_res and put
// look at that: written stage by stage over all rows, the rows' chains
// (ten dependent rounds of the generator, the activation) overlap.  The
// instructions of this function are what an epilogue costs: issued beside the
// warp that starts the tensor core's products, they delay it one for one.
// get_res() gives the residual's values, put(base, v) stores to `pre` or `out`.
template <typename T, int R, typename RES, typename PUT>
__device__ __forceinline__ void dense_epilogue(const DenseEpi& e, const EpiConst& c, int64_t row, int n,
                                               const float (&bias)[8], float (&v)[R][8], RES get_res, PUT put) {
  constexpr int RS = 32 / R;
  if (e.bias)
#pragma unroll
    for (int q = 0; q < R; ++q) add8(v[q], bias);
  if (e.pre) put(e.pre, v);
  if (e.rng.drop) {
    uint4 w[R];
    const int64_t block = row * e.per_row + n / 8;
    if (c.low) {  // no counter passes 32 bits: the generator's first products are common to all
#pragma unroll
      for (int q = 0; q < R; ++q) w[q] = philox4x32_10((uint32_t)block + (uint32_t)(q * RS * e.per_row), 0u, c.key);
    } else {
#pragma unroll
      for (int q = 0; q < R; ++q) w[q] = philox4x32_10((uint64_t)(block + (int64_t)q * RS * e.per_row), c.key);
    }
#pragma unroll
    for (int q = 0; q < R; ++q) {
      scale8(v[q], c.f);
      keep8(w[q], e.rng.drop, v[q]);
    }
  }
  switch (e.act) {
    case 1: act_rows<1, R>(v); break;
    case 2: act_rows<2, R>(v); break;
    case 3: act_rows<3, R>(v); break;
    default: break;
  }
  if (e.residual) {
    float res[R][8];
    get_res(res);
#pragma unroll
    for (int q = 0; q < R; ++q) add8(v[q], res[q]);
  }
  put(e.out, v);
}
// put of R rows of eight columns by the thread that holds them
template <typename T, int R>
__device__ __forceinline__ void dense_put(const DenseEpi& e, const EpiConst& c, void* base, int64_t row, int left, int n,
                                          const float (&v)[R][8]) {
  T* p = static_cast<T*>(base) + row * e.N + n;
#pragma unroll
  for (int q = 0; q < R; ++q)
    if (q * (32 / R) < left) put8<T>(p, (int64_t)(q * (32 / R)) * e.N, min(8, e.N - n), c.vec_out, v[q]);
}

// A warp's chunk of an epilogue: 32 rows by kCW columns.  kCW / 8 lanes cover a
// row, each with eight columns of kCR rows, kCStep apart.  (16 warps with chunks
// of 16 columns have half the registers each: 131072 x 1536 x 768 with residual
// and dropout 250 us for 242, 32768 x 768 x 1536 with silu and dropout 110 for 115.)
constexpr int kCW = 32, kCLanes = kCW / 8, kCR = kCLanes, kCStep = 32 / kCLanes;

// The chunk in shared memory: 16-byte pieces, swizzled by row so that a lane's
// own row (as the accumulator has it) and the arrangement above both reach it
// without conflicts.
struct Stage {
  uint4* s;
  int lane;
  static constexpr int kPieces = kCW / 4;  // of a row
  __device__ __forceinline__ int row() const { return lane / kCLanes; }
  __device__ __forceinline__ int col() const { return lane % kCLanes * 8; }
  __device__ __forceinline__ uint4& piece(int row, int p) const {
    return s[row * kPieces + (p ^ (kPieces == 8 ? row & 7 : row >> 1 & 3))];
  }
  __device__ __forceinline__ float& at(int row, int c) const { return reinterpret_cast<float*>(&piece(row, c >> 2))[c & 3]; }
  // this lane's two pieces of its first row; kCStep rows below they have the same swizzle
  __device__ __forceinline__ uint4* mine(int half) const { return &piece(row(), lane % kCLanes * 2 + half); }
  __device__ __forceinline__ void get(float (&v)[kCR][8]) const {
    const uint4 *a = mine(0), *b = mine(1);
#pragma unroll
    for (int q = 0; q < kCR; ++q) {
      const uint4 lo = a[q * kCStep * kPieces], hi = b[q * kCStep * kPieces];
      v[q][0] = __uint_as_float(lo.x); v[q][1] = __uint_as_float(lo.y);
      v[q][2] = __uint_as_float(lo.z); v[q][3] = __uint_as_float(lo.w);
      v[q][4] = __uint_as_float(hi.x); v[q][5] = __uint_as_float(hi.y);
      v[q][6] = __uint_as_float(hi.z); v[q][7] = __uint_as_float(hi.w);
    }
  }
  __device__ __forceinline__ void put(const float (&v)[kCR][8]) const {
    uint4 *a = mine(0), *b = mine(1);
#pragma unroll
    for (int q = 0; q < kCR; ++q) {
      a[q * kCStep * kPieces] = make_uint4(__float_as_uint(v[q][0]), __float_as_uint(v[q][1]), __float_as_uint(v[q][2]),
                                           __float_as_uint(v[q][3]));
      b[q * kCStep * kPieces] = make_uint4(__float_as_uint(v[q][4]), __float_as_uint(v[q][5]), __float_as_uint(v[q][6]),
                                           __float_as_uint(v[q][7]));
    }
  }
};

// For rows that start anywhere: a chunk from row m0, column n, with a lane a
// column, so that its accesses lie together, and through shared memory to or
// from the epilogue's arrangement.
static_assert(kCW == 32);
template <typename T>
__device__ __forceinline__ void dense_stage_rows(const DenseEpi& e, const Stage& st, int64_t m0, int n, float (&res)[kCR][8]) {
  __syncwarp();
  if (n + st.lane < e.N) {
    const int rows = (int)min(e.M - m0, (int64_t)32);
    const T* p = static_cast<const T*>(e.residual) + m0 * e.res_stride + n + st.lane;
    for (int r0 = 0; r0 < 32; r0 += 8, p += 8 * e.res_stride)
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (r0 + u < rows) st.at(r0 + u, st.lane) = Cvt<T>::to_f(p[u * e.res_stride]);
  }
  __syncwarp();
  st.get(res);
}
template <typename T>
__device__ __forceinline__ void dense_put_chunk(const DenseEpi& e, const EpiConst& c, const Stage& st, void* base, int64_t m0,
                                                int n, int left, const float (&v)[kCR][8]) {
  if (c.vec_out) {
    dense_put<T, kCR>(e, c, base, m0 + st.row(), left, n + st.col(), v);
    return;
  }
  __syncwarp();
  st.put(v);
  __syncwarp();
  if (n + st.lane < e.N) {
    const int rows = (int)min(e.M - m0, (int64_t)32);
    T* p = static_cast<T*>(base) + m0 * e.N + n + st.lane;
    for (int r0 = 0; r0 < 32; r0 += 8, p += 8 * (int64_t)e.N)
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (r0 + u < rows) p[u * (int64_t)e.N] = Cvt<T>::from_f(st.at(r0 + u, st.lane));
  }
}
// The residual of a chunk by plain loads.
template <typename T>
__device__ __forceinline__ void dense_get_chunk(const DenseEpi& e, const EpiConst& c, const Stage& st, int64_t m0, int n,
                                                int left, float (&res)[kCR][8]) {
  if (!c.vec_res) {
    dense_stage_rows<T>(e, st, m0, n, res);
    return;
  }
  const T* p = static_cast<const T*>(e.residual) + (m0 + st.row()) * e.res_stride + n + st.col();
#pragma unroll
  for (int q = 0; q < kCR; ++q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) res[q][i] = 0.f;
    if (q * kCStep < left) get8<T>(p, q * kCStep * e.res_stride, 8, true, res[q]);
  }
}
// rows of a chunk from m0, counted from this lane's first; 0 beyond the last column
__device__ __forceinline__ int dense_left(const DenseEpi& e, int64_t m0, int n, const Stage& st) {
  return n + st.col() < e.N ? (int)min(e.M - m0 - st.row(), (int64_t)32) : 0;
}

// ---------------------------------------------------------------- tensor-core pieces
constexpr int kBK = 64;  // depth of a step
constexpr int kEpiWarps = 8;
constexpr int kMmaThreads = 32 * (4 + kEpiWarps);
// Polls before a wait gives up; a tile takes microseconds, so this is far above any wait that ends.
constexpr uint32_t kMmaSpin = 1u << 20;
// Polls for what is still under way when one has given up.
constexpr uint32_t kDrainSpin = 1u << 16;

// Shared-memory operand descriptor, 128-byte swizzle.  K-major rows of 128
// bytes: groups of 8 rows are 1024 bytes apart.  MN-major rows (one k each, 64
// values of m or n): groups of 8 k are 1024 bytes apart, the next 64 values of
// m or n 8192 bytes.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  constexpr uint64_t kLead = 8192 >> 4, kStep = 1024 >> 4;
  return (uint64_t)((addr >> 4) & 0x3fff) | kLead << 16 | kStep << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// bf16 x bf16 -> fp32, m rows, n columns
constexpr uint32_t mma_idesc(int m, int n, bool a_mn, bool b_mn) {
  return 1u << 4 | 1u << 7 | 1u << 10 | (a_mn ? 1u : 0u) << 15 | (b_mn ? 1u : 0u) << 16 | (uint32_t)(n >> 3) << 17 |
         (uint32_t)(m >> 4) << 24;
}

// The instructions that differ between a CTA of its own and a pair of CTAs (a
// cluster of two) that share one product: the pair's first CTA issues for both.
template <bool PAIR>
struct Mma {
  // `one`: nonzero in the lane that issues.  The whole warp comes here with the
  // same operands.
  __device__ __forceinline__ static void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate,
                                             uint32_t one) {
    if constexpr (PAIR)
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
          "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
          "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one)
          : "memory");
    else
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
          "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
          "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one)
          : "memory");
  }
  // arrives on `bar` (of a pair's CTAs in `mask`) when the products issued so far are done
  __device__ __forceinline__ static void commit(uint64_t* bar, uint32_t one, uint16_t mask = 3) {
    if constexpr (PAIR)
      asm volatile(
          "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
          "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::
              "r"(smem_u32(bar)),
          "h"(mask), "r"(one)
          : "memory");
    else
      asm volatile(
          "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
          "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
          "r"(one)
          : "memory");
  }
  __device__ __forceinline__ static void alloc(uint32_t* dst, uint32_t ncols) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(ncols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(dst, ncols);
    }
  }
  __device__ __forceinline__ static void dealloc(uint32_t t, uint32_t ncols) {
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(ncols) : "memory");
    else
      tmem_dealloc(t, ncols);
  }
  // a box to this CTA's `dst`, counted on `bar`: an address in the cluster's
  // shared memory, for a pair that of the first CTA's barrier
  __device__ __forceinline__ static void load(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                              uint32_t one) {
    if constexpr (PAIR)
      asm volatile(
          "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
          "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
          " [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(smem_u32(dst)),
          "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar), "r"(one)
          : "memory");
    else
      asm volatile(
          "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
          "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
          " [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(smem_u32(dst)),
          "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar), "r"(one)
          : "memory");
  }
};
__device__ __forceinline__ void expect_bytes(uint64_t* bar, uint32_t bytes, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(smem_u32(bar)),
      "r"(bytes), "r"(one)
      : "memory");
}
// the same shared-memory address in the cluster's CTA 0
__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
// Relaxed: what the waiting side relies on are reads of tensor memory, which
// tcgen05.wait::ld has completed.  A release at the cluster's scope would first wait
// for all the warp's stores to global memory (4% of 32768 x 768 x 1536).
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// nonzero in one lane of the warp
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// A bounded wait as one stretch of code: at most `polls` polls, then `polls`
// becomes 1, so that the waits after one that gave up do not wait.  Nothing
// branches on the outcome, and the code around it stays the same for the warp.
__device__ __forceinline__ void wait_through(uint64_t* bar, uint32_t parity, uint32_t& polls) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, %0;\n\t"
      "POLL_%=:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra DONE_%=;\n\t"
      "sub.u32 n, n, 1;\n\tsetp.ne.u32 q, n, 0;\n\t@q bra POLL_%=;\n\tmov.u32 %0, 1;\n\t"
      "DONE_%=:\n\t}"
      : "+r"(polls)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
}

struct DenseWork {
  int32_t tiles_m, tiles_n, splits;
  int32_t kblocks;  // ceil(K / 64)
  int32_t loaded;   // items whose slices are loaded: all, except in the self-test of a wait that gives up
  uint32_t spin;    // polls before a wait gives up, 2 at least
  // the 64-deep blocks of a split
  __device__ __forceinline__ int block(int split) const { return (int)((int64_t)kblocks * split / splits); }
};

__device__ __forceinline__ bool any_nan(const float (&v)[kCR][8]) {
  bool bad = false;
#pragma unroll
  for (int q = 0; q < kCR; ++q)
#pragma unroll
    for (int i = 0; i < 8; ++i) bad |= isnan(v[q][i]);
  return bad;
}

// A CTA of its own makes a tile of 128 x 128, a pair one of 256 x 256: each CTA
// of it holds 128 rows of A and 128 columns of B and accumulates its 128 rows
// of all 256 columns, so a step moves 32 KB into each SM for twice the products
// that 32 KB give a single CTA.
//
// Three planes take a CTA of its own.  A block's planes are loaded once, one of A
// and one of B a stage, and its six products made from three stages: 16 KB a
// product (32 when each product had its own stage, and its time was L2's).  Tensor
// memory holds two leading accumulators in turn, the other one and the sum.
template <bool PAIR, typename T>
struct Tile {
  static constexpr int kM = PAIR ? 256 : 128, kN = PAIR ? 256 : 128;  // of the item
  static constexpr int kBoxA = 128, kBoxB = 128;                      // rows or columns one CTA loads
  static constexpr int kA = kBoxA * kBK * 2, kB = kBoxB * kBK * 2, kStage = kA + kB;
  static constexpr int kStages = 6;
  static constexpr int kEpi = kEpiWarps * 32 * kCW * 4;  // a chunk of fp32 for each epilogue warp
  static constexpr int kCols = kN / (kEpiWarps / 4);     // columns of an epilogue warp
  static constexpr int kChunks = kCols / kCW;
  // Two chunks of bf16 residual a warp, in the place of the last stage (not for
  // fp32, where an item's products take six times as long).
  static constexpr int kAhead = sizeof(T) == 2 ? 2 : 0;
  static_assert(kEpiWarps * kAhead * 32 * kCW * 2 <= kStage);
  static constexpr int kBytes = kStages * kStage + kEpi + 1024;  // and alignment
};

// An infinite operand has no finite planes besides its first, and infinity times
// the other operand's planes gives NaN where the product is infinite; so do
// products of finite values that pass the type's largest.  A warp that met NaN in
// a sum of three planes comes here after its last item, when nothing waits for it
// any more, finds its chunks that hold NaN as they were stored, and sums them again
// in fp32 from the operands' values: a rank-one step for each k, with a row of A
// and a column of B a lane.  What was not NaN stays.  Where all sums of a chunk have
// become NaN the rest of K changes nothing.  dW of 20011 x 2056 -> 2000, 0.93 ms: 4.6 with
// an infinity in dy, 23 with a row of them, which makes every sum anew.
constexpr int kDeep = 16;  // of K at a time: A's and B's values fill a warp's staged chunk

// 32 rows (or columns) from `mn` by kDeep of K from `k` of one operand's planes, on
// their way; `limit` rows exist, k ends at `end`.  Rows along K: a lane holds its own
// row's.  Rows along mn: four lanes hold a k's 32 values.  Starts are multiples of 8
// values, as are plane and ld, so that 16 bytes are loaded at a time.
struct RepairLoad {
  uint4 r[2][3];
  __device__ __forceinline__ void load(const Planes& o, int lane, int64_t mn, int64_t limit, int64_t k, int64_t end) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t row = o.k_major ? mn + lane : k + lane / 4 + 8 * j, col = o.k_major ? k + 8 * j : mn + lane % 4 * 8;
      const bool in = o.k_major ? row < limit && col < end : row < end && col < limit;
#pragma unroll
      for (int p = 0; p < 3; ++p)
        r[j][p] = in ? *reinterpret_cast<const uint4*>(o.base + p * o.plane + row * o.ld + col) : make_uint4(0, 0, 0, 0);
    }
  }
  // the fp32 values to v[k][mn], zeros where k has ended
  __device__ __forceinline__ void put(float* v, bool k_major, int lane, int64_t k, int64_t end) const {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float t[8], u[8];
      unpack8(r[j][2], t);
#pragma unroll
      for (int p = 1; p >= 0; --p) {
        unpack8(r[j][p], u);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] += u[i];
      }
      if (k_major) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[(8 * j + i) * 32 + lane] = k + 8 * j + i < end ? t[i] : 0.f;
      } else {
        store8(v + (lane / 4 + 8 * j) * 32 + lane % 4 * 8, t);
      }
    }
  }
};

// The sums of a chunk (its first row m of `rows`, column n of `cols`) over k .. end - 1,
// left in its staged form.  A function of its own, and its operands by value: its loop
// has no registers to spare for anything else.
__device__ __noinline__ void dense_sum_again(const Planes pa, const Planes pb, const Stage st, int64_t m, int64_t rows,
                                             int64_t n, int64_t cols, int64_t k, int64_t end) {
  float acc[32] = {};
  float* va = reinterpret_cast<float*>(st.s);  // [kDeep][32] of A, then of B
  float* vb = va + kDeep * 32;
  RepairLoad a, b;
  a.load(pa, st.lane, m, rows, k, end);
  b.load(pb, st.lane, n, cols, k, end);
#pragma unroll 1
  for (; k < end; k += kDeep) {
    __syncwarp();
    a.put(va, pa.k_major, st.lane, k, end);
    b.put(vb, pb.k_major, st.lane, k, end);
    a.load(pa, st.lane, m, rows, k + kDeep, end);
    b.load(pb, st.lane, n, cols, k + kDeep, end);
    __syncwarp();
#pragma unroll 2
    for (int i = 0; i < kDeep; ++i) {
      const float y = vb[i * 32 + st.lane];
#pragma unroll
      for (int r = 0; r < 32; r += 4) {
        const float4 x = *reinterpret_cast<const float4*>(va + i * 32 + r);
        acc[r] = fmaf(x.x, y, acc[r]);
        acc[r + 1] = fmaf(x.y, y, acc[r + 1]);
        acc[r + 2] = fmaf(x.z, y, acc[r + 2]);
        acc[r + 3] = fmaf(x.w, y, acc[r + 3]);
      }
    }
    bool all = true;
#pragma unroll
    for (int r = 0; r < 32; ++r) all &= isnan(acc[r]) || m + r >= rows || n + st.lane >= cols;
    if (__all_sync(0xffffffffu, all)) break;
  }
  __syncwarp();
#pragma unroll
  for (int r = 0; r < 32; ++r) st.at(r, st.lane) = acc[r];
  __syncwarp();
}

template <typename T>
__device__ __noinline__ void dense_repair(const DenseEpi& e, const DenseWork w, const Stage st, int quarter, int col0) {
  using S = Tile<false, T>;
  const EpiConst c(e);
  for (int item = blockIdx.x; item < w.tiles_m * w.tiles_n * w.splits; item += gridDim.x) {
    const int rest = item / w.tiles_n, split = rest / w.tiles_m;
    const int64_t m0 = (int64_t)(rest % w.tiles_m) * S::kM + quarter * 32;
    const int64_t k0 = (int64_t)w.block(split) * kBK, k1 = min((int64_t)w.block(split + 1) * kBK, e.K);
    for (int chunk = 0; chunk < S::kChunks; ++chunk) {
      const int n = item % w.tiles_n * S::kN + col0 + chunk * kCW, nl = n + st.col();
      if (n >= e.N || m0 >= e.M) break;
      const int left = dense_left(e, m0, n, st);
      // f(row, column) of this lane's elements
      const auto each = [&](auto f) {
#pragma unroll
        for (int q = 0; q < kCR; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (q * kCStep < left && nl + i < e.N) f(q, i);
      };
      float* part = e.partial ? e.partial + ((int64_t)split * e.M + m0 + st.row()) * (e.per_row * 8) + nl : nullptr;
      const auto stored = [&](void* base, int q, int i) -> T& {
        return static_cast<T*>(base)[(m0 + st.row() + q * kCStep) * e.N + nl + i];
      };
      bool bad = false;
      each([&](int q, int i) {
        bad |= isnan(part ? part[(int64_t)(q * kCStep * 8) * e.per_row + i] : Cvt<T>::to_f(stored(e.pre ? e.pre : e.out, q, i)));
      });
      if (!__any_sync(0xffffffffu, bad)) continue;
      dense_sum_again(e.a, e.b, st, m0, e.M, n, e.N, k0, k1);
      float v[kCR][8], bias[8];
      st.get(v);
      if (part) {
        each([&](int q, int i) {
          float& p = part[(int64_t)(q * kCStep * 8) * e.per_row + i];
          if (isnan(p)) p = v[q][i];
        });
        continue;
      }
      dense_bias8(e, c, nl, bias);
      dense_epilogue<T, kCR>(
          e, c, m0 + st.row(), nl, bias, v,
          [&](float (&res)[kCR][8]) { dense_get_chunk<T>(e, c, st, m0, n, left, res); },
          [&](void* base, const float (&u)[kCR][8]) {
            each([&](int q, int i) {
              T& p = stored(base, q, i);
              if (isnan(Cvt<T>::to_f(p))) p = Cvt<T>::from_f(u[q][i]);
            });
          });
    }
  }
}

// NaN for a warp's 32 rows by `cols` columns of the items from `item` on, whose products never came.
template <typename T>
__device__ __noinline__ void dense_poison(const DenseEpi& e, const DenseWork w, int lane, int item, int stride, int tile_m,
                                          int row0, int tile_n, int col0, int cols) {
  const float nan = __uint_as_float(0x7fc00000u);
  for (; item < w.tiles_m * w.tiles_n * w.splits; item += stride) {
    const int rest = item / w.tiles_n, split = rest / w.tiles_m;
    const int64_t m0 = (int64_t)(rest % w.tiles_m) * tile_m + row0;
    const int rows = (int)min(e.M - m0, (int64_t)32);
    for (int j = lane; j < cols; j += 32) {
      const int64_t n = (int64_t)(item % w.tiles_n) * tile_n + col0 + j;
      if (n >= e.N) break;
      for (int r = 0; r < rows; ++r) {
        const int64_t at = (m0 + r) * e.N + n;
        if (e.partial) {
          e.partial[((int64_t)split * e.M + m0 + r) * (e.per_row * 8) + n] = nan;
        } else {
          static_cast<T*>(e.out)[at] = Cvt<T>::from_f(nan);
          if (e.pre) static_cast<T*>(e.pre)[at] = Cvt<T>::from_f(nan);
        }
      }
    }
  }
}

constexpr int kCut = 512 / kBK;  // most blocks that the leading accumulator of three planes takes
constexpr int kCutsOfRest = 8;   // cuts that the other one takes
// cuts of a split as even as they go
__device__ __forceinline__ int even_cut(int blocks) {
  const int cuts = (blocks + kCut - 1) / kCut;
  return (blocks + cuts - 1) / cuts;
}

template <bool A_MN, bool B_MN, bool PAIR, int PLANES, typename T>
__global__ void __launch_bounds__(kMmaThreads, 1)
    dense_mma_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const __grid_constant__ DenseEpi e, const DenseWork w, int32_t* status) {
  using S = Tile<PAIR, T>;
  using I = Mma<PAIR>;
  constexpr int BN = S::kN;
  static_assert(PLANES == 1 || (PLANES == 3 && !PAIR && S::kStages % 3 == 0));
  constexpr int kTmem = PLANES == 3 ? 4 * BN : 2 * BN;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t full[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t tmem_base;
  __shared__ volatile int dead;
  uint8_t* tiles = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_rank() : 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], PAIR ? 2 * kEpiWarps : kEpiWarps);
    }
    mbar_init(&drained, 1);
    dead = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  __syncthreads();
  if constexpr (PAIR) cluster_barrier();
  if (warp == 2) I::alloc(&tmem_base, kTmem);
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  const uint32_t tmem = tmem_base;
  const int items = w.tiles_m * w.tiles_n * w.splits;
  const bool ahead = PLANES == 1 && S::kAhead && e.residual && EpiConst(e).vec_res;
  const int stages = ahead ? S::kStages - 1 : S::kStages;
  const int first = PAIR ? blockIdx.x / 2 : blockIdx.x, stride = PAIR ? gridDim.x / 2 : gridDim.x;

  // Bounded wait; a role that gives up (or sees that another did) stops.  Outputs
  // whose products never came are NaN then, and what is under way (loads, products)
  // is waited for before the CTA leaves.
  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < w.spin; ++i) {
      if (mbar_try_wait(bar, parity)) return true;
      if ((i & 63) == 63 && dead) return false;
    }
    dead = 1;
    report(status, kStatusTimeout);
    return false;
  };

  // The warps that load and that issue products walk their loops whole and one
  // lane issues: in a branch of one lane every operand (descriptors, addresses)
  // passes through vector registers, and what stands between two steps' products
  // or loads then takes longer than the queue of products lasts.  (131072 x 1536
  // x 768 without its epilogue: 329 thousand cycles that way, 312 with only the
  // products' warp whole, 264 with all three; the products alone take 256.)
  if (warp == 0 || warp == 3) {
    // Warp 0 loads A, warp 3 loads B.
    const bool of_a = warp == 0;
    const uint32_t one = elect_one();
    int stage = 0;
    uint32_t phase = 0, polls = w.spin;
    for (int item = first; item < w.loaded; item += stride) {
      const int rest = item / w.tiles_n, split = rest / w.tiles_m;
      const int n0 = item % w.tiles_n * BN + (PAIR ? rank * 128 : 0);
      const int m0 = rest % w.tiles_m * S::kM + (PAIR ? rank * 128 : 0);
      const int kb0 = w.block(split), kb1 = w.block(split + 1);
      // three planes in the order 1 0 2, in which their products need them
      int plane = PLANES == 3 ? 1 : 0, kb = kb0;
      for (int t = (kb1 - kb0) * PLANES; t > 0; --t) {
        wait_through(&empty[stage], phase ^ 1, polls);
        if (polls == 1) break;  // what it would overwrite may still be read
        const int k0 = kb * kBK;
        uint8_t* sa = tiles + stage * S::kStage;
        uint8_t* sb = sa + S::kA;
        const uint32_t bar = PAIR ? in_first_cta(&full[stage]) : smem_u32(&full[stage]);
        if (of_a) {
          if (rank == 0) expect_bytes(&full[stage], PAIR ? 2 * S::kStage : S::kStage, one);
          if (A_MN) {
#pragma unroll
            for (int j = 0; j < S::kBoxA / 64; ++j) I::load(sa + j * 8192, &map_a, bar, m0 + 64 * j, k0, plane, one);
          } else {
            I::load(sa, &map_a, bar, k0, m0, plane, one);
          }
        } else if (B_MN) {
#pragma unroll
          for (int j = 0; j < S::kBoxB / 64; ++j) I::load(sb + j * 8192, &map_b, bar, n0 + 64 * j, k0, plane, one);
        } else {
          I::load(sb, &map_b, bar, k0, n0, plane, one);
        }
        if (PLANES == 3) {
          kb += plane == 2;
          plane = plane == 2 ? 1 : plane == 1 ? 0 : 2;
        } else {
          ++kb;
        }
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (polls == 1) break;
    }
    if (polls == 1) {
      dead = 1;
      if (one) report(status, kStatusTimeout);
    }
    // No load may land after the CTA has gone: the last one of each stage is waited
    // for, whoever gave up (otherwise the products have waited for them).
    if (of_a && rank == 0)
      for (int i = 0; i < stages; ++i) {
        mbar_wait_bounded(&full[stage], phase ^ 1, kDrainSpin);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
  } else if (warp == 1 && rank == 0) {
    constexpr uint32_t idesc = mma_idesc(S::kM, BN, A_MN, B_MN);
    constexpr uint32_t kStepA = (A_MN ? 2048 : 32) >> 4, kStepB = (B_MN ? 2048 : 32) >> 4;
    const uint32_t one = elect_one();
    const uint64_t da0 = smem_desc(smem_u32(tiles)), db0 = smem_desc(smem_u32(tiles + S::kA));
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0, polls = w.spin;
    // asked once an item (or cut), of the whole warp: a branch on one lane's count would
    // cost the loop its uniform operands
    const auto gave_up = [&] { return __any_sync(0xffffffffu, polls == 1); };
    // the four products of one plane of A with one of B, from stages sa and sb
    const auto block = [&](uint32_t d, int sa, int sb, bool add) {
      const uint64_t da = da0 + sa * (S::kStage >> 4), db = db0 + sb * (S::kStage >> 4);
#pragma unroll
      for (int k = 0; k < kBK / 16; ++k) I::mma(d, da + k * kStepA, db + k * kStepB, idesc, add || k > 0, one);
    };
    for (int item = first; item < items; item += stride) {
      const int split = item / w.tiles_n / w.tiles_m;
      const int blocks = w.block(split + 1) - w.block(split);
      if constexpr (PLANES == 3) {
        const uint32_t rest = tmem + 2 * BN;
        const int cut = even_cut(blocks);
        for (int b0 = 0; b0 < blocks; b0 += cut) {
          const int b1 = min(b0 + cut, blocks);
          const bool fresh = b0 % (cut * kCutsOfRest) == 0;
          wait_through(&acc_empty[acc], acc_phase ^ 1, polls);
          // the last cut has been taken, the accumulator of the rest with it
          if (fresh && (b0 > 0 || item != first)) wait_through(&acc_empty[acc ^ 1], acc ? acc_phase : acc_phase ^ 1, polls);
          if (gave_up()) break;  // what the products would overwrite may still be read
          tmem_fence_after_sync();
          const uint32_t lead = tmem + acc * BN;
          for (int b = b0; b < b1; ++b) {
            const int s1 = stage, s0 = stage + 1, s2 = stage + 2;  // of planes 1, 0, 2
            wait_through(&full[s1], phase, polls);
            tmem_fence_after_sync();
            block(rest, s1, s1, !fresh || b > b0);
            wait_through(&full[s0], phase, polls);
            tmem_fence_after_sync();
            block(rest, s0, s1, true);
            block(rest, s1, s0, true);
            I::commit(&empty[s1], one);
            block(lead, s0, s0, b > b0);
            wait_through(&full[s2], phase, polls);
            tmem_fence_after_sync();
            block(rest, s0, s2, true);
            block(rest, s2, s0, true);
            I::commit(&empty[s0], one);
            I::commit(&empty[s2], one);
            if ((stage += 3) == S::kStages) {
              stage = 0;
              phase ^= 1;
            }
          }
          if (gave_up()) break;  // these are products of what was never loaded
          I::commit(&acc_full[acc], one);
          if (++acc == 2) {
            acc = 0;
            acc_phase ^= 1;
          }
        }
        if (gave_up()) break;
      } else {
        wait_through(&acc_empty[acc], acc_phase ^ 1, polls);
        if (gave_up()) break;
        tmem_fence_after_sync();
        const uint32_t d = tmem + acc * BN;
        wait_through(&full[stage], phase, polls);
        for (int b = 0; b < blocks; ++b) {
          tmem_fence_after_sync();
          const int used = stage;
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
          block(d, used, used, b > 0);
          I::commit(&empty[used], one);
          if (b + 1 < blocks) wait_through(&full[stage], phase, polls);
        }
        if (gave_up()) break;
        I::commit(&acc_full[acc], one);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
    }
    if (gave_up()) {
      dead = 1;
      if (one) report(status, kStatusTimeout);
      I::commit(&drained, one, 1);  // products still running use the buffers
      mbar_wait_bounded(&drained, 0, kDrainSpin);
    }
  } else if (warp >= 4) {
    const EpiConst c(e);
    const int quarter = warp & 3, col0 = ((warp - 4) >> 2) * S::kCols;
    const Stage st = {reinterpret_cast<uint4*>(tiles + S::kStages * S::kStage) + (warp - 4) * (8 * kCW), lane};
    // The slices that TMA has asked for keep the SM's way from L2 busy: a plain
    // load issued now is answered some 4000 cycles later, as long as a chunk
    // takes.  So the residual is fetched to shared memory two chunks ahead, each
    // lane its own pieces.
    uint4* held = reinterpret_cast<uint4*>(tiles + (S::kStages - 1) * S::kStage) + (warp - 4) * (8 * kCW);
    int f_item = first, f_chunk = 0, slot = 0;  // next to fetch; where it goes and the oldest one is
    const T* f_from = nullptr;                  // this lane's first piece of the item
    int f_left = 0, f_n = 0;
    const auto fetch = [&]() {
      if (!ahead) return;
      if (f_item < items) {
        if (f_chunk == 0) {
          f_n = f_item % w.tiles_n * BN + col0 + st.col();
          const int64_t m = (int64_t)(f_item / w.tiles_n % w.tiles_m) * S::kM + rank * 128 + quarter * 32 + st.row();
          f_from = static_cast<const T*>(e.residual) + m * e.res_stride + f_n;
          f_left = (int)min(e.M - m, (int64_t)32);
        }
        const uint32_t to = smem_u32(held + slot * (4 * kCW) + lane);
#pragma unroll
        for (int q = 0; q < kCR; ++q)
          if (q * kCStep < f_left && f_n < e.N)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + q * 512),
                         "l"(f_from + q * kCStep * e.res_stride)
                         : "memory");
        f_from += kCW;
        f_n += kCW;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      slot ^= 1;
      if (++f_chunk == S::kChunks) {
        f_chunk = 0;
        f_item += stride;
      }
    };
    for (int i = 0; i < S::kAhead; ++i) fetch();
    int acc = 0;
    uint32_t acc_phase = 0;
    bool bad = false, ended = false;
    int item = first;
    for (; item < items; item += stride) {
      const int rest = item / w.tiles_n, split = rest / w.tiles_m;
      const int n0 = item % w.tiles_n * BN + col0;
      const int64_t m0 = (int64_t)(rest % w.tiles_m) * S::kM + rank * 128 + quarter * 32;
      const uint32_t at = tmem + col0 + ((uint32_t)(quarter * 32) << 16);
      // of both, what the products' warp waits for before it uses the accumulator again
      const auto release = [&]() {
        tmem_fence_before_sync();
        if (lane == 0) {
          if constexpr (PAIR) arrive_cluster(in_first_cta(&acc_empty[acc]));
          else mbar_arrive(&acc_empty[acc]);
        }
        __syncwarp();
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      };
      uint32_t src = at + acc * BN;
      if constexpr (PLANES == 3) {
        // each cut is added to the sum and its accumulator given back; what
        // follows reads the sum
        src = at + 3 * BN;
        const int blocks = w.block(split + 1) - w.block(split), cut = even_cut(blocks);
        for (int b0 = 0; b0 < blocks; b0 += cut) {
          if (!__all_sync(0xffffffffu, wait(&acc_full[acc], acc_phase))) {
            ended = true;
            break;
          }
          tmem_fence_after_sync();
          const bool rest = b0 + cut >= blocks || (b0 + cut) % (cut * kCutsOfRest) == 0;
#pragma unroll 1
          for (int j = 0; j < S::kCols; j += 16) {
            uint32_t lead[16], more[16], sum[16];
            tmem_ld16(at + acc * BN + j, lead);
            if (rest) tmem_ld16(at + 2 * BN + j, more);
            if (b0 > 0) tmem_ld16(src + j, sum);
            tmem_wait_ld();
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              v[i] = __uint_as_float(lead[i]);
              if (rest) v[i] += __uint_as_float(more[i]);
              if (b0 > 0) v[i] += __uint_as_float(sum[i]);
            }
            tmem_st16(src + j, v);
          }
          tmem_wait_st();
          release();
        }
        if (ended) break;
      } else {
        if (!__all_sync(0xffffffffu, wait(&acc_full[acc], acc_phase))) {
          ended = true;
          break;
        }
        tmem_fence_after_sync();
      }
#pragma unroll 1
      for (int chunk = 0; chunk < S::kChunks; ++chunk) {
        const int j = chunk * kCW, n = n0 + j;
        if (n >= e.N) {
          fetch();
          continue;
        }
        // A lane reads the columns of its own row of the accumulator; through
        // shared memory it gets eight columns of a few rows, so that
        // neighbouring lanes cover a row's columns in global memory and the
        // eight share one dropout counter.
        uint32_t r[kCW / 16][16];
#pragma unroll
        for (int q = 0; q < kCW / 16; ++q) tmem_ld16(src + j + 16 * q, r[q]);
        const int nl = n + st.col(), left = dense_left(e, m0, n, st);
        float bias[8];
        dense_bias8(e, c, nl, bias);
        tmem_wait_ld();
        __syncwarp();
#pragma unroll
        for (int q = 0; q < kCW / 4; ++q)
          st.piece(lane, q) = make_uint4(r[q >> 2][(q & 3) * 4], r[q >> 2][(q & 3) * 4 + 1], r[q >> 2][(q & 3) * 4 + 2],
                                         r[q >> 2][(q & 3) * 4 + 3]);
        __syncwarp();
        float v[kCR][8];
        st.get(v);
        if (PLANES == 3) bad |= any_nan(v);
        if (e.partial) {
          float* p = e.partial + ((int64_t)split * e.M + m0 + st.row()) * (e.per_row * 8) + nl;
#pragma unroll
          for (int q = 0; q < kCR; ++q)
            if (q * kCStep < left) store8(p + (int64_t)(q * kCStep * 8) * e.per_row, v[q]);
        } else {
          dense_epilogue<T, kCR>(
              e, c, m0 + st.row(), nl, bias, v,
              [&](float (&res)[kCR][8]) {
                if (ahead) {
                  asm volatile("cp.async.wait_group 1;" ::: "memory");
#pragma unroll
                  for (int q = 0; q < kCR; ++q) unpack8(held[slot * (4 * kCW) + q * 32 + lane], res[q]);
                } else {
                  dense_get_chunk<T>(e, c, st, m0, n, left, res);
                }
              },
              [&](void* base, const float (&u)[kCR][8]) { dense_put_chunk<T>(e, c, st, base, m0, n, left, u); });
          fetch();
        }
      }
      if constexpr (PLANES == 1) release();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (ended) dense_poison<T>(e, w, lane, item, stride, S::kM, rank * 128 + quarter * 32, BN, col0, S::kCols);
    if constexpr (PLANES == 3)
      if (__any_sync(0xffffffffu, bad) && !ended) dense_repair<T>(e, w, st, quarter, col0);
  }
  __syncwarp();
  tmem_fence_before_sync();
  __syncthreads();
  if constexpr (PAIR) cluster_barrier();  // the other CTA's products, loads and arrivals reach into this one
  tmem_fence_after_sync();
  if (warp == 2) I::dealloc(tmem, kTmem);
}

// The epilogue of a product whose K loop was cut: the parts summed in order, a
// chunk a warp or, of many parts (then there are few chunks, and one part after
// another is a round trip each), a chunk a CTA and a run of the parts a warp.  768 x 1536 of 4 parts (19 MB, mostly in L2): 6 us.
constexpr int kJoinWarps = 4;
constexpr int kJoinShared = 8;  // parts from which a CTA's warps share a chunk's
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps)
    dense_join_kernel(const float* part, int splits, const __grid_constant__ DenseEpi e) {
  __shared__ uint4 staged[kJoinWarps][8 * kCW];
  const EpiConst c(e);
  const int warp = threadIdx.x >> 5;
  const bool share = splits >= kJoinShared;
  const Stage st = {staged[warp], (int)threadIdx.x & 31};
  const int64_t ld = (int64_t)e.per_row * 8, chunks_n = (e.N + kCW - 1) / kCW;
  const int64_t i = share ? blockIdx.x : (int64_t)blockIdx.x * kJoinWarps + warp;
  const int s0 = share ? splits * warp / kJoinWarps : 0, s1 = share ? splits * (warp + 1) / kJoinWarps : splits;
  const int64_t m0 = i / chunks_n * 32;
  const int n = (int)(i % chunks_n) * kCW, nl = n + st.col();
  if (m0 >= e.M) return;
  const int left = dense_left(e, m0, n, st);
  float v[kCR][8] = {}, bias[8];
  // two parts' loads together: one after another each is a round trip
  for (int s = s0; s < s1; s += 2) {
    float t[2][kCR][8] = {};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float* p = part + ((int64_t)(s + u) * e.M + m0 + st.row()) * ld + nl;
#pragma unroll
      for (int q = 0; q < kCR; ++q)
        if (q * kCStep < left && s + u < s1) load8(p + q * kCStep * ld, t[u][q]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int q = 0; q < kCR; ++q) add8(v[q], t[u][q]);
  }
  if (share) {
    if (warp) st.put(v);
    __syncthreads();
    if (warp) return;
    for (int w = 1; w < kJoinWarps; ++w) {
      float t[kCR][8];
      Stage{staged[w], st.lane}.get(t);
#pragma unroll
      for (int q = 0; q < kCR; ++q) add8(v[q], t[q]);
    }
  }
  dense_bias8(e, c, nl, bias);
  dense_epilogue<T, kCR>(
      e, c, m0 + st.row(), nl, bias, v,
      [&](float (&res)[kCR][8]) { dense_get_chunk<T>(e, c, st, m0, n, left, res); },
      [&](void* base, const float (&u)[kCR][8]) { dense_put_chunk<T>(e, c, st, base, m0, n, left, u); });
}

}  // namespace ssm
