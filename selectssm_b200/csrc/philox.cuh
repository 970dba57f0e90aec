// Counter-based random bits for dropout: Philox4x32-10 (J. Salmon, M. Moraes,
// R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011).
//
// A mask element is a pure function of (seed, offset, row, column), so it is
// never stored: forward, backward and the product's epilogue each recompute it.
// Rows are those of the last axis; the eight columns 8j .. 8j+7 of row r share
// the counter (r * ceil(dim / 8) + j, offset) under the key `seed`, and column
// 8j+i takes the 16 bits number i of its 128 output bits.  An element is kept
// when its 16 bits are at least `drop` (0 .. 65536), so the probability of
// dropping is exactly drop / 65536 and the kept values' factor
// 65536 / (65536 - drop) is its exact inverse.
//
// Sixteen bits a value, not 32: ten rounds are about 45 instructions, which is
// about 6 a value when eight values share them.  HBM at 6555 GB/s leaves a bf16
// pass of one read and one write about 20 instructions a value.
#pragma once

#include <cstdint>

namespace ssm {

struct DropRng {
  uint64_t seed, offset;
  const uint64_t* dev;  // {seed, offset} in device memory, or null: the fields above
  uint32_t drop;        // of 65536
};

struct PhiloxKey {
  uint32_t k0, k1, c2, c3;
};

__device__ __forceinline__ PhiloxKey philox_key(const DropRng& r) {
  const uint64_t seed = r.dev ? r.dev[0] : r.seed, off = r.dev ? r.dev[1] : r.offset;
  return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)off, (uint32_t)(off >> 32)};
}

__device__ __forceinline__ uint4 philox4x32_10(uint32_t c0, uint32_t c1, const PhiloxKey& key) {
  uint32_t c2 = key.c2, c3 = key.c3;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint4 philox4x32_10(uint64_t counter, const PhiloxKey& key) {
  return philox4x32_10((uint32_t)counter, (uint32_t)(counter >> 32), key);
}

// Calls f(i, kept) for the block's eight columns.  A 16-bit draw is at least
// drop (1 .. 65536) exactly when it exceeds drop - 1; with the draw in the upper
// half of a word both compare as they stand, whatever the lower half holds.
template <typename F>
__device__ __forceinline__ void for_kept8(uint4 w, uint32_t drop, F f) {
  const uint32_t over = (drop << 16) - 1u;  // drop 65536: nothing exceeds it
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f(2 * j, v[j] << 16 > over);
    f(2 * j + 1, v[j] > over);
  }
}
// v[i] where column i is kept, else 0
__device__ __forceinline__ void keep8(uint4 w, uint32_t drop, float (&v)[8]) {
  for_kept8(w, drop, [&](int i, bool keep) { v[i] = keep ? v[i] : 0.f; });
}

// Factor of a kept value; 0 when everything is dropped.
__host__ __device__ __forceinline__ float keep_factor(uint32_t drop) {
  return drop >= 65536u ? 0.f : 65536.f / (float)(65536u - drop);
}

}  // namespace ssm
