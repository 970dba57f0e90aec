// Group norm with an activation over channels-last x (batch, seqlen, dim)
// (src/selectssm/selectssm.py:306-313, norm_type "group"; flax.linen.GroupNorm):
// for each batch row and each run of dim / groups channels
//
//   mean, var over (seqlen, the run's channels);  rstd = 1 / sqrt(var + eps)
//   xhat = (x - mean) rstd,  y = act(xhat scale + bias)
// and with du = dy act'(xhat scale + bias), g = du scale, m the mean over the group
//   dx = rstd (g - m(g) - xhat m(g xhat)),  dscale = sum du xhat,  dbias = sum du.
//
// All sums a group needs follow from sums per channel: m(g) is the sum over its
// channels of scale * (sum of du), m(g xhat) of scale * (sum of du xhat).  So a
// thread keeps a fixed run of channels, walks down the sequence, and no
// group's width matters to the inner loops.
//
// Two forms.  Held: a cluster of up to eight CTAs keeps some groups of one batch
// row in its shared memory between the statistics and their use, so each input
// is read once and the call is one kernel (and a small one for dscale and
// dbias).  Split, where a single group is too long for that: one pass for the
// sums per chunk of the sequence, a small kernel that joins them, and a second
// pass over the inputs.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "act8.cuh"
#include "common.cuh"
#include "vec8.cuh"
#include "../../include/selectssm_b200.h"

namespace ssm {

int launch_error(const char* where, cudaError_t e);  // scan.cu
int bind_device(const void* ptr);                      // scan.cu

constexpr int kGnThreads = 256;

// How a pass cuts (batch, seqlen, dim): column tiles of `ct` vectors of V
// channels, `rt` rows at a time, chunks of `chunk` rows.
struct GnGeom {
  int64_t L;
  int32_t B, D, G, cg;
  int32_t nvec, ct, tiles, rt;
  int32_t chunks;
  int64_t chunk;
};

struct GnArgs {
  GnGeom g;
  float eps;
  const void* x;
  const void* dy;
  const float* scale;
  const float* bias;
  float* stats;      // (B, G, 2) mean, rstd
  float2* part;      // (B, chunks, D) per-channel partials: forward (mean, M2), backward (sum du, sum du xhat)
  float2* sums;      // backward: (B, D) the same, summed over the chunks
  float2* means;     // backward: (B, G) m(g), m(g xhat)
  void* out;         // y or dx
  float* dscale;
  float* dbias;
};

template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&v)[V]) {
  if constexpr (V == 8) store8(p, v);
  else *p = Cvt<T>::from_f(v[0]);
}

struct GnPlace {
  int b, chunk, vec, r0;
  bool active;
  int64_t l0, l1;
};
__device__ __forceinline__ GnPlace gn_place(const GnGeom& g, bool reversed) {
  GnPlace q;
  unsigned id = blockIdx.x;  // (batch, chunk)
  if (reversed) id = gridDim.x - 1 - id;
  q.b = id / g.chunks;
  q.chunk = id - q.b * g.chunks;
  q.vec = blockIdx.z * g.ct + threadIdx.x % g.ct;
  q.r0 = threadIdx.x / g.ct;
  q.active = q.r0 < g.rt && q.vec < g.nvec;
  q.l0 = q.chunk * g.chunk;
  q.l1 = min(q.l0 + g.chunk, g.L);
  return q;
}

// Elementwise on V values, two at a time.
template <int V, typename F>
__device__ __forceinline__ void gn_pairs(float (&a)[V], F f) {
  if constexpr (V == 1) {
    a[0] = f(make_float2(a[0], 0.f), 0).x;
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = f(make_float2(a[i], a[i + 1]), i);
      a[i] = r.x;
      a[i + 1] = r.y;
    }
  }
}
template <int V>
__device__ __forceinline__ float2 gn_at(const float (&a)[V], int i) {
  return make_float2(a[i], V == 1 ? 0.f : a[i + (V > 1)]);
}
template <int V>
__device__ __forceinline__ void gn_add(float (&a)[V], const float (&b)[V]) {
  gn_pairs<V>(a, [&](float2 x, int i) { return fadd2(x, gn_at<V>(b, i)); });
}
template <int V>
__device__ __forceinline__ void gn_sub(float (&a)[V], const float (&b)[V]) {
  gn_pairs<V>(a, [&](float2 x, int i) { return fsub2(x, gn_at<V>(b, i)); });
}
template <int V>
__device__ __forceinline__ void gn_mul(float (&a)[V], const float (&b)[V]) {
  gn_pairs<V>(a, [&](float2 x, int i) { return fmul2(x, gn_at<V>(b, i)); });
}
template <int V>  // a += b c
__device__ __forceinline__ void gn_fma(float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  gn_pairs<V>(a, [&](float2 x, int i) { return ffma2(gn_at<V>(b, i), gn_at<V>(c, i), x); });
}
template <int V>  // a = a b + c
__device__ __forceinline__ void gn_muladd(float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  gn_pairs<V>(a, [&](float2 x, int i) { return ffma2(x, gn_at<V>(b, i), gn_at<V>(c, i)); });
}

// du of V elements from d = dy and xh = xhat (d is overwritten)
template <int V, int ACT>
__device__ __forceinline__ void gn_du(float (&d)[V], const float (&xh)[V], const float (&scale)[V], const float (&bias)[V]) {
  if constexpr (ACT != 0) {
    float u[V];
#pragma unroll
    for (int i = 0; i < V; ++i) u[i] = xh[i];
    gn_muladd<V>(u, scale, bias);
    gn_pairs<V>(d, [&](float2 x, int i) { return fmul2(x, slope2<ACT>(gn_at<V>(u, i))); });
  }
}

// ---------------------------------------------------------------- split form
// A thread's walk over its rows of x, and of dy with IN = 2: f(offset, v, d) for
// every row's V values (d only with IN = 2).  Rows on their way wait in a ring of
// the thread's own places in shared memory, `kGnAhead` deep, filled by cp.async:
// 128 bytes a thread in flight at any time, without a register or a scoreboard
// held for them.  (Four rows of loads into registers, then their use, then the
// next four: 3.8 TB/s; asking for each register's next row as it empties: 2.1,
// because a wait for one load waits for younger ones too.)
template <int IN> constexpr int kGnAhead = IN == 1 ? 8 : 4;
template <typename T, int V, int IN>
constexpr size_t kGnRing = V == 1 ? 0 : (size_t)kGnThreads * kGnAhead<IN> * IN * V * sizeof(T);

template <typename T, int V, int IN, typename F>
__device__ __forceinline__ void gn_walk(uint8_t* ring, const T* x, const T* dy, int64_t step, int rows, F f) {
  if constexpr (V == 1) {
    constexpr int R = 8;  // rows loaded together
    for (; rows > 0; rows -= R, x += R * step, dy += IN == 2 ? R * step : 0) {
      T a[R], b[R];
#pragma unroll
      for (int k = 0; k < R; ++k)
        if (k < rows) {
          a[k] = x[k * step];
          if (IN == 2) b[k] = dy[k * step];
        }
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (k >= rows) break;
        float v[1] = {Cvt<T>::to_f(a[k])}, d[1] = {0.f};
        if (IN == 2) d[0] = Cvt<T>::to_f(b[k]);
        f(v, d);
      }
    }
  } else {
    constexpr int S = kGnAhead<IN>, P = sizeof(T) * V / 16;  // 16-byte pieces of a vector
    uint4* mine = reinterpret_cast<uint4*>(ring) + threadIdx.x;
    const auto ask = [&](int row, int slot) {
      if (row < rows)
#pragma unroll
        for (int q = 0; q < P; ++q) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                           smem_u32(mine + ((slot * IN) * P + q) * kGnThreads)),
                       "l"(reinterpret_cast<const uint4*>(x + row * step) + q)
                       : "memory");
          if (IN == 2)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                             smem_u32(mine + ((slot * IN + 1) * P + q) * kGnThreads)),
                         "l"(reinterpret_cast<const uint4*>(dy + row * step) + q)
                         : "memory");
        }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const auto take = [&](int slot, int in, float (&v)[V]) {
      if constexpr (P == 1) {
        unpack8(mine[(slot * IN + in) * kGnThreads], v);
      } else {
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const uint4 r = mine[((slot * IN + in) * P + q) * kGnThreads];
          v[4 * q] = __uint_as_float(r.x); v[4 * q + 1] = __uint_as_float(r.y);
          v[4 * q + 2] = __uint_as_float(r.z); v[4 * q + 3] = __uint_as_float(r.w);
        }
      }
    };
#pragma unroll
    for (int k = 0; k < S; ++k) ask(k, k);
    for (int row = 0, slot = 0; row < rows; ++row) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");  // the oldest row's
      float v[V], d[V];
      take(slot, 0, v);
      if constexpr (IN == 2) take(slot, 1, d);
      f(v, d);
      ask(row + S, slot);
      slot = slot + 1 == S ? 0 : slot + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
}

// Mean and sum of squared deviations per channel of a chunk.  The values are
// summed about the thread's first one of each channel, runs of 64 rows at a time
// whose mean and deviations are merged into the running pair with Chan's update:
// a far-off first value costs digits of one run only, and no large mean is ever
// subtracted from a sum of squares.  2 x 131072 x 256 bf16 (134 MB): 30 us, 4.5 TB/s,
// 36 while L2 still writes another kernel's output back; a bare maximum over the
// same bytes takes 26.  What is left is the start and the end of 1024 CTAs' walks.
template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads, 4) gn_stats_kernel(const GnArgs p) {
  extern __shared__ __align__(16) float sm[];
  const GnGeom& g = p.g;
  const GnPlace q = gn_place(g, false);
  float mean[V], m2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.f;
  float n = 0.f;
  if (q.active) {
    const int64_t step = (int64_t)g.rt * g.D;
    const T* x = static_cast<const T*>(p.x) + ((int64_t)q.b * g.L + q.l0 + q.r0) * g.D + (int64_t)q.vec * V;
    const int rows = (int)((q.l1 - q.l0 - q.r0 + g.rt - 1) / g.rt);
    float ref[V], s[V], ss[V];
    int run = 0;
    const auto close = [&] {
      const float inv = 1.f / (float)run, nn = n + (float)run, w = (float)run / nn;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float off = s[i] * inv, dev = fmaxf(fmaf(-s[i], off, ss[i]), 0.f), delta = ref[i] + off - mean[i];
        mean[i] = fmaf(delta, w, mean[i]);
        m2[i] += fmaf(delta * delta, n * w, dev);
      }
      n = nn;
      run = 0;
    };
    gn_walk<T, V, 1>(reinterpret_cast<uint8_t*>(sm), x, x, step, rows, [&](float (&v)[V], float (&)[V]) {
      if (run == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          ref[i] = v[i];
          s[i] = ss[i] = 0.f;
        }
      }
      gn_sub<V>(v, ref);
      gn_add<V>(s, v);
      gn_fma<V>(ss, v, v);
      if (++run == 64) close();
    });
    if (run) close();
  }
  __syncthreads();  // the rings' memory serves below
  // merge the rt row lanes of each channel in order
  const int width = g.ct * V, mine = (threadIdx.x % g.ct) * V;
  float *smean = sm, *sm2 = sm + g.rt * width, *sn = sm + 2 * g.rt * width;
  if (q.r0 < g.rt) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      smean[q.r0 * width + mine + i] = mean[i];
      sm2[q.r0 * width + mine + i] = m2[i];
    }
    if (threadIdx.x % g.ct == 0) sn[q.r0] = q.active ? n : 0.f;
  }
  __syncthreads();
  const float total = (float)(q.l1 - q.l0);
  for (int c = threadIdx.x; c < width; c += kGnThreads) {
    const int ch = blockIdx.z * width + c;
    if (ch >= g.D) break;
    const float ref = smean[c];
    float s = 0.f;
    for (int r = 1; r < g.rt; ++r) s = fmaf(sn[r], smean[r * width + c] - ref, s);
    const float mu = ref + s / total;
    float d2 = 0.f;
    for (int r = 0; r < g.rt; ++r) {
      const float d = smean[r * width + c] - mu;
      d2 += sm2[r * width + c] + sn[r] * d * d;
    }
    p.part[((int64_t)q.b * g.chunks + q.chunk) * g.D + ch] = make_float2(mu, d2);
  }
}

constexpr int kMergeThreads = 256;  // of the small kernels, a CTA a group
__device__ __forceinline__ float block_sum(float v, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < kMergeThreads / 32; ++w) s += buf[w];
  return s;
}

// Calls f(chunk, channel) for every partial of a group, dealt out over the
// CTA's threads: neighbouring threads take neighbouring channels.
template <typename F>
__device__ __forceinline__ void gn_each_part(const GnGeom& g, F f) {
  if (g.cg <= kMergeThreads) {
    const int at_once = kMergeThreads / g.cg, k = threadIdx.x / g.cg, c = threadIdx.x - k * g.cg;
    if (k < at_once)
#pragma unroll 8
      for (int ck = k; ck < g.chunks; ck += at_once) f(ck, c);
  } else {
    for (int ck = 0; ck < g.chunks; ++ck)
      for (int c = threadIdx.x; c < g.cg; c += kMergeThreads) f(ck, c);
  }
}

// mean and rstd of one group from its chunks' and channels' partials (2 MB of them at
// 2 x 131072 x 256: 6 us, a launch and a round trip to memory)
__global__ void __launch_bounds__(kMergeThreads) gn_merge_kernel(const GnArgs p) {
  __shared__ float buf[kMergeThreads / 32];
  const GnGeom& g = p.g;
  const int grp = blockIdx.x % g.G, b = blockIdx.x / g.G;
  const float2* part = p.part + (int64_t)b * g.chunks * g.D + grp * g.cg;
  const float inv = 1.f / ((float)g.L * (float)g.cg), ref = part[0].x;  // so that equal means merge to themselves
  const auto size = [&](int ck) { return (float)(min((ck + 1) * g.chunk, g.L) - ck * g.chunk); };
  float s = 0.f;
  gn_each_part(g, [&](int ck, int c) { s = fmaf(size(ck) * inv, part[(int64_t)ck * g.D + c].x - ref, s); });
  const float mu = block_sum(s, buf) + ref;
  float d2 = 0.f;
  gn_each_part(g, [&](int ck, int c) {
    const float2 v = part[(int64_t)ck * g.D + c];
    d2 += v.y + size(ck) * (v.x - mu) * (v.x - mu);
  });
  const float var = block_sum(d2, buf) * inv;
  if (threadIdx.x == 0) reinterpret_cast<float2*>(p.stats)[blockIdx.x] = make_float2(mu, rsqrtf(var + p.eps));
}

// A thread's constants: one pair of statistics where its channels share a group
// (ONE), else one a channel.
template <int V, bool ONE>
struct GnStat {
  float a[ONE ? 1 : V], b[ONE ? 1 : V];
  __device__ __forceinline__ void load(const float2* from, int b_, const GnGeom& g, int c0) {
#pragma unroll
    for (int i = 0; i < (ONE ? 1 : V); ++i) {
      const float2 s = from[(int64_t)b_ * g.G + (c0 + i) / g.cg];
      a[i] = s.x;
      b[i] = s.y;
    }
  }
  __device__ __forceinline__ float2 a2(int i) const { return ONE ? dup2(a[0]) : gn_at<ONE ? 1 : V>(a, ONE ? 0 : i); }
  __device__ __forceinline__ float2 b2(int i) const { return ONE ? dup2(b[0]) : gn_at<ONE ? 1 : V>(b, ONE ? 0 : i); }
};
template <int V>
__device__ __forceinline__ void gn_affine(const GnArgs& p, int c0, float (&scale)[V], float (&bias)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    scale[i] = p.scale ? p.scale[c0 + i] : 1.f;
    bias[i] = p.bias ? p.bias[c0 + i] : 0.f;
  }
}

// y.  2 x 131072 x 256 bf16 with silu: 42 us for 268 MB, 6.4 TB/s, the copy's rate; the
// special-function unit (an exponential and a reciprocal a value) is 71% busy.
template <typename T, int V, int ACT, bool ONE>
__global__ void __launch_bounds__(kGnThreads, 4) gn_apply_kernel(const GnArgs p) {
  extern __shared__ __align__(16) uint8_t ring[];
  const GnGeom& g = p.g;
  const GnPlace q = gn_place(g, true);
  if (!q.active) return;
  float scale[V], bias[V];
  gn_affine<V>(p, q.vec * V, scale, bias);
  GnStat<V, ONE> st;
  st.load(reinterpret_cast<const float2*>(p.stats), q.b, g, q.vec * V);
  gn_pairs<V>(scale, [&](float2 x, int i) { return fmul2(x, st.b2(i)); });
  const int64_t base = ((int64_t)q.b * g.L + q.l0 + q.r0) * g.D + (int64_t)q.vec * V, step = (int64_t)g.rt * g.D;
  const T* x = static_cast<const T*>(p.x) + base;
  T* y = static_cast<T*>(p.out) + base;
  gn_walk<T, V, 1>(ring, x, x, step, (int)((q.l1 - q.l0 - q.r0 + g.rt - 1) / g.rt), [&](float (&v)[V], float (&)[V]) {
    gn_pairs<V>(v, [&](float2 t, int i) {
      return act2<ACT>(ffma2(fsub2(t, st.a2(i)), gn_at<V>(scale, i), gn_at<V>(bias, i)));
    });
    store_v<T, V>(y, v);
    y += step;
  });
}

// Sums over a chunk of du and du xhat per channel.  2 x 131072 x 256 bf16 with silu: 66 us
// for 268 MB, 4.1 TB/s: latency at three CTAs an SM (80 registers) and the slope's
// special functions (51% busy) together; HBM is at half its peak.
template <typename T, int V, int ACT, bool ONE>
__global__ void __launch_bounds__(kGnThreads, 3) gn_sums_kernel(const GnArgs p) {
  extern __shared__ __align__(16) float sm[];
  const GnGeom& g = p.g;
  const GnPlace q = gn_place(g, false);
  float s1[V], s2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
  if (q.active) {
    float scale[V], bias[V];
    gn_affine<V>(p, q.vec * V, scale, bias);
    GnStat<V, ONE> st;
    st.load(reinterpret_cast<const float2*>(p.stats), q.b, g, q.vec * V);
    const int64_t base = ((int64_t)q.b * g.L + q.l0 + q.r0) * g.D + (int64_t)q.vec * V, step = (int64_t)g.rt * g.D;
    gn_walk<T, V, 2>(reinterpret_cast<uint8_t*>(sm), static_cast<const T*>(p.x) + base, static_cast<const T*>(p.dy) + base,
                     step, (int)((q.l1 - q.l0 - q.r0 + g.rt - 1) / g.rt), [&](float (&v)[V], float (&d)[V]) {
                       gn_pairs<V>(v, [&](float2 t, int i) { return fmul2(fsub2(t, st.a2(i)), st.b2(i)); });
                       gn_du<V, ACT>(d, v, scale, bias);
                       gn_add<V>(s1, d);
                       gn_fma<V>(s2, d, v);
                     });
  }
  __syncthreads();  // the rings' memory serves below
  const int width = g.ct * V, mine = (threadIdx.x % g.ct) * V;
  float *a1 = sm, *a2 = sm + g.rt * width;
  if (q.r0 < g.rt) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a1[q.r0 * width + mine + i] = s1[i];
      a2[q.r0 * width + mine + i] = s2[i];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += kGnThreads) {
    const int ch = blockIdx.z * width + c;
    if (ch >= g.D) break;
    float t1 = 0.f, t2 = 0.f;
    for (int r = 0; r < g.rt; ++r) {
      t1 += a1[r * width + c];
      t2 += a2[r * width + c];
    }
    p.part[((int64_t)q.b * g.chunks + q.chunk) * g.D + ch] = make_float2(t1, t2);
  }
}

// One group of one batch row: its channels' sums over the chunks (kept for
// dscale and dbias) and the two means that dx needs.
__global__ void __launch_bounds__(kMergeThreads) gn_means_kernel(const GnArgs p) {
  __shared__ float buf[kMergeThreads / 32];
  const GnGeom& g = p.g;
  const int grp = blockIdx.x % g.G, b = blockIdx.x / g.G;
  __shared__ float2 sums[kMergeThreads];
  const float2* part = p.part + (int64_t)b * g.chunks * g.D + grp * g.cg;
  float m1 = 0.f, m2 = 0.f;
  const auto channel = [&](int c, float2 s) {  // a channel's sums over the chunks
    p.sums[(int64_t)b * g.D + grp * g.cg + c] = s;
    const float w = p.scale ? p.scale[grp * g.cg + c] : 1.f;
    m1 = fmaf(w, s.x, m1);
    m2 = fmaf(w, s.y, m2);
  };
  if (g.cg <= kMergeThreads) {
    float2 s = make_float2(0.f, 0.f);
    gn_each_part(g, [&](int ck, int c) { s = fadd2(s, part[(int64_t)ck * g.D + c]); });
    sums[threadIdx.x] = s;  // of channel threadIdx.x % cg
    __syncthreads();
    if ((int)threadIdx.x < g.cg) {
      for (int k = 1; k < kMergeThreads / g.cg; ++k) s = fadd2(s, sums[k * g.cg + threadIdx.x]);
      channel(threadIdx.x, s);
    }
  } else {
    for (int c = threadIdx.x; c < g.cg; c += kMergeThreads) {
      float2 s = make_float2(0.f, 0.f);
      for (int ck = 0; ck < g.chunks; ++ck) s = fadd2(s, part[(int64_t)ck * g.D + c]);
      channel(c, s);
    }
  }
  const float t1 = block_sum(m1, buf), t2 = block_sum(m2, buf);
  const float count = (float)g.L * (float)g.cg;
  if (threadIdx.x == 0) p.means[blockIdx.x] = make_float2(t1 / count, t2 / count);
}

// dx.  2 x 131072 x 256 bf16 with silu: 57 us for 403 MB, 7.0 TB/s (some of it still in
// L2 from the sums' pass): bound by HBM.
template <typename T, int V, int ACT, bool ONE>
__global__ void __launch_bounds__(kGnThreads, 3) gn_dx_kernel(const GnArgs p) {
  extern __shared__ __align__(16) uint8_t ring[];
  const GnGeom& g = p.g;
  const GnPlace q = gn_place(g, true);
  if (!q.active) return;
  float scale[V], bias[V];
  gn_affine<V>(p, q.vec * V, scale, bias);
  GnStat<V, ONE> st, mm;
  st.load(reinterpret_cast<const float2*>(p.stats), q.b, g, q.vec * V);
  mm.load(p.means, q.b, g, q.vec * V);
  const int64_t base = ((int64_t)q.b * g.L + q.l0 + q.r0) * g.D + (int64_t)q.vec * V, step = (int64_t)g.rt * g.D;
  T* dx = static_cast<T*>(p.out) + base;
  gn_walk<T, V, 2>(ring, static_cast<const T*>(p.x) + base, static_cast<const T*>(p.dy) + base, step,
                   (int)((q.l1 - q.l0 - q.r0 + g.rt - 1) / g.rt), [&](float (&v)[V], float (&d)[V]) {
                     gn_pairs<V>(v, [&](float2 t, int i) { return fmul2(fsub2(t, st.a2(i)), st.b2(i)); });
                     gn_du<V, ACT>(d, v, scale, bias);
                     gn_pairs<V>(d, [&](float2 t, int i) {  // rstd (du scale - m1 - xhat m2)
                       const float2 r = fsub2(fmul2(t, gn_at<V>(scale, i)), mm.a2(i));
                       return fmul2(fsub2(r, fmul2(gn_at<V>(v, i), mm.b2(i))), st.b2(i));
                     });
                     store_v<T, V>(dx, d);
                     dx += step;
                   });
}

// dscale and dbias: `rows` partial sums of every channel in a fixed order
__global__ void __launch_bounds__(1024) gn_param_kernel(const float2* sums, int rows, int D, float* dscale, float* dbias) {
  __shared__ float2 red[32][33];
  const int col = threadIdx.x & 31, lane = threadIdx.x >> 5, c = blockIdx.x * 32 + col;
  float2 s = make_float2(0.f, 0.f);
  if (c < D)
    for (int r = lane; r < rows; r += 32) s = fadd2(s, sums[(int64_t)r * D + c]);
  red[lane][col] = s;
  __syncthreads();
  if (lane == 0 && c < D) {
    float2 t = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 32; ++i) t = fadd2(t, red[i][col]);
    if (dbias) dbias[c] = t.x;
    if (dscale) dscale[c] = t.y;
  }
}

// ---------------------------------------------------------------- held form
// A job: `gpj` groups (W channels) of one batch row, `ctas` CTAs with `rows`
// rows each; a cluster takes the same groups of every `turns`-th batch row, so
// that many short rows (a norm per token) need few sums for dscale and dbias.  nv
// vectors of V channels by rt row lanes; each thread keeps `slots` vectors of its
// own in shared memory.
constexpr int kHoldThreads = 256;  // at most
struct GnHold {
  int32_t threads, W, gpj, jobs, ctas, turns, nv, rt, slots;
  int64_t rows;
  size_t smem;
};

template <typename T, int V>
struct GnVec;  // V values as they lie in shared memory
template <> struct GnVec<float, 4> {
  float4 r;
  __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
  __device__ __forceinline__ static void put(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <> struct GnVec<__nv_bfloat16, 8> {
  uint4 r;
  __device__ __forceinline__ void get(float (&v)[8]) const { unpack8(r, v); }
  __device__ __forceinline__ static void put(__nv_bfloat16* p, const float (&v)[8]) { store8(p, v); }
};
template <typename T> struct GnVec<T, 1> {
  T r;
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = Cvt<T>::to_f(r); }
  __device__ __forceinline__ static void put(T* p, const float (&v)[1]) { *p = Cvt<T>::from_f(v[0]); }
};

__device__ __forceinline__ void gn_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void gn_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float2 gn_peer(const float2* p, int cta) {
  uint32_t at;
  float2 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(cta));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}

// SHORT: more batch rows than turns, or rows so short that the sums over a group
// are a thread's work.  (The loop and the other form of the sums cost a call that
// has no need of them up to a fifth of its time, in registers.)
// 64 x 2048 x 768 bf16: 95 us for 403 MB, 4.2 TB/s.  A CTA reads its part, meets its
// cluster, and writes, and what a thread does once (80 registers of constants, two
// sums over the CTA) stands against 26 vectors of its own: the phases of four CTAs
// an SM overlap only in part.  The backward in bf16 with an activation has too few
// registers (88 to 124 bytes spilled).
template <typename T, int V, int ACT, bool BWD, bool SHORT>
__global__ void __launch_bounds__(kHoldThreads, 3) gn_hold_kernel(const GnArgs p, const GnHold h) {
  using Vec = GnVec<T, V>;
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ float parts[kHoldThreads / 32];
  const GnGeom& g = p.g;
  const int threads = blockDim.x, warps = threads >> 5;
  Vec* hx = reinterpret_cast<Vec*>(raw);
  Vec* hd = hx + (BWD ? h.slots * threads : 0);
  float* red = reinterpret_cast<float*>(raw + ((size_t)h.slots * threads * sizeof(Vec) * (BWD ? 2 : 1) + 15) / 16 * 16);
  float2* chan = reinterpret_cast<float2*>(red + threads * (BWD || g.cg % V ? V : 2));  // backward: sums per channel
  float2* acc = chan + (BWD ? h.W : 0);  // backward: those of all the batch rows so far
  float2* own = acc + (BWD ? h.W : 0);   // this CTA's pair of each group
  float2* all = own + h.gpj;            // the job's
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int rank = 0;
  if (h.ctas > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int job = blockIdx.x / h.ctas, turn = job / h.jobs, g0 = job % h.jobs * h.gpj;
  const int ng = min(h.gpj, g.G - g0), width = ng * g.cg, c0 = g0 * g.cg;
  const int cv = tid % h.nv, rl = tid / h.nv;
  const bool active = rl < h.rt && cv * V < width;
  const int64_t l0 = rank * h.rows, l1 = min(l0 + h.rows, g.L);
  const int mine = active && l0 + rl < l1 ? (int)((l1 - l0 - rl + h.rt - 1) / h.rt) : 0;  // vectors of this thread
  const int64_t step = (int64_t)h.rt * g.D;
  const auto fetch = [&](int64_t b) {
    const int64_t base = (b * g.L + l0 + rl) * g.D + c0 + cv * V;
    const T* x = static_cast<const T*>(p.x) + base;
    const T* dy = BWD ? static_cast<const T*>(p.dy) + base : nullptr;
#pragma unroll 4
    for (int i = 0; i < mine; ++i) {
      if constexpr (sizeof(Vec) == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(hx + i * threads + tid)), "l"(x + i * step)
                     : "memory");
        if (BWD)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(hd + i * threads + tid)),
                       "l"(dy + i * step)
                       : "memory");
      } else {
        hx[i * threads + tid].r = x[i * step];
        if (BWD) hd[i * threads + tid].r = dy[i * step];
      }
    }
  };
  fetch(turn);
  int grp[V];  // of the job's groups
#pragma unroll
  for (int j = 0, q = cv * V / g.cg, left = (q + 1) * g.cg - cv * V; j < V; ++j) {
    grp[j] = active ? q : 0;
    if (--left == 0) {
      ++q;
      left = g.cg;
    }
  }
  float scale[V], bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    scale[i] = active && p.scale ? p.scale[c0 + cv * V + i] : 1.f;
    bias[i] = active && p.bias ? p.bias[c0 + cv * V + i] : 0.f;
  }
  const float per_group = 1.f / ((float)g.L * (float)g.cg);
  const int step_c = h.rt <= 8 ? 1 : 32;  // backward: lanes for a channel's sum
  // The job's groups of every h.turns-th batch row, one after another.
  for (int64_t b = turn; SHORT ? b < g.B : b == turn; b += SHORT ? h.turns : g.B) {
    const int64_t base = (b * g.L + l0 + rl) * g.D + c0 + cv * V;
    T* out = static_cast<T*>(p.out) + base;
    if (SHORT && b != turn) fetch(b);
    asm volatile("cp.async.wait_all;" ::: "memory");  // a thread reads only what it fetched itself

    // Per-thread values to sums over each group, in a fixed order, handed to
    // finish(group, sum).  Vectors that lie in one group are summed first.  A
    // group's values lie together, so that as many warps as there are for each
    // group walk over them without a division.
    const bool single = g.cg % V == 0;
    const int unit = single ? V : 1, entries = g.cg / unit * h.rt;
    const int share = max(warps / ng, 1);  // warps for a group
    const auto group_sums = [&](const float (&s)[V], auto finish) {
      if (active) {
        if (single) {
          float t = 0.f;
#pragma unroll
          for (int i = 0; i < V; ++i) t += s[i];
          red[cv * h.rt + rl] = t;
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) red[(cv * V + i) * h.rt + rl] = s[i];
        }
      }
      __syncthreads();
      if (SHORT && entries <= 32) {  // a thread a group
        for (int q = tid; q < ng; q += threads) {
          float t = 0.f;
          for (int i = 0; i < entries; ++i) t += red[q * entries + i];
          finish(q, t);
        }
        __syncthreads();
        return;
      }
      for (int w = warp; w < ng * share; w += warps) {
        const int q = w / share, part = w - q * share;
        const float* from = red + q * entries;
        float t = 0.f;
        for (int i = part * 32 + lane; i < entries; i += 32 * share) t += from[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (lane == 0) {
          if (share == 1) finish(q, t);
          else parts[w] = t;
        }
      }
      __syncthreads();
      if (share > 1) {
        if (tid < ng) {
          float t = 0.f;
          for (int i = 0; i < share; ++i) t += parts[tid * share + i];
          finish(tid, t);
        }
        __syncthreads();
      }
    };

    if constexpr (!BWD) {
      const float n = (float)max(l1 - l0, (int64_t)0) * (float)g.cg;  // this CTA's values of a group
      float s[V] = {}, mean[V], gain[V];
#pragma unroll 4
      for (int i = 0; i < mine; ++i) {
        float v[V];
        hx[i * threads + tid].get(v);
        gn_add<V>(s, v);
      }
      group_sums(s, [&](int q, float t) { own[q].x = n > 0.f ? t / n : 0.f; });
#pragma unroll
      for (int j = 0; j < V; ++j) {
        mean[j] = own[grp[j]].x;
        s[j] = 0.f;
      }
#pragma unroll 4
      for (int i = 0; i < mine; ++i) {
        float v[V];
        hx[i * threads + tid].get(v);
        gn_sub<V>(v, mean);
        gn_fma<V>(s, v, v);
      }
      group_sums(s, [&](int q, float t) { own[q].y = t; });
      // the CTAs' means and squared deviations, merged about the common mean
      if (h.ctas > 1) {
        gn_cluster_arrive();
        gn_cluster_wait();
      }
      // (from the first one's mean, so that equal means merge to themselves); a
      // lane for each CTA
      const auto settle = [&](int q, float mu, float m2) {
        const float2 st = make_float2(mu, rsqrtf(fmaf(m2, per_group, p.eps)));
        all[q] = st;
        if (rank == 0 && p.stats) reinterpret_cast<float2*>(p.stats)[(int64_t)b * g.G + g0 + q] = st;
      };
      if (SHORT && h.ctas == 1)
        for (int q = tid; q < ng; q += threads) settle(q, own[q].x, own[q].y);
      for (int q = warp; (!SHORT || h.ctas > 1) && q < ng; q += warps) {
        float2 each = own[q];
        float cnt = lane ? 0.f : n;
        if (h.ctas > 1) {
          const int r = min(lane, h.ctas - 1);
          each = gn_peer(own + q, r);
          cnt = lane < h.ctas ? (float)((int)max(min((r + 1) * h.rows, g.L) - r * h.rows, (int64_t)0) * g.cg) : 0.f;
        }
        const float ref = __shfl_sync(0xffffffffu, each.x, 0);
        float mu = cnt * (each.x - ref);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) mu += __shfl_xor_sync(0xffffffffu, mu, o, 8);
        mu = fmaf(mu, per_group, ref);
        const float d = each.x - mu;
        float m2 = cnt > 0.f ? fmaf(cnt * d, d, each.y) : 0.f;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, o, 8);
        if (lane == 0) settle(q, mu, m2);
      }
      __syncthreads();
      if (h.ctas > 1) gn_cluster_arrive();
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 st = all[grp[j]];
        mean[j] = st.x;
        gain[j] = scale[j] * st.y;
      }
#pragma unroll 4
      for (int i = 0; i < mine; ++i) {
        float v[V];
        hx[i * threads + tid].get(v);
        gn_sub<V>(v, mean);
        gn_muladd<V>(v, gain, bias);
        gn_pairs<V>(v, [](float2 x, int) { return act2<ACT>(x); });
        Vec::put(out + i * step, v);
      }
    } else {
      float mean[V], rstd[V], s1[V] = {}, s2[V] = {};
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 st = reinterpret_cast<const float2*>(p.stats)[(int64_t)b * g.G + g0 + grp[j]];
        mean[j] = st.x;
        rstd[j] = st.y;
      }
#pragma unroll 4
      for (int i = 0; i < mine; ++i) {
        float xh[V], d[V];
        hx[i * threads + tid].get(xh);
        hd[i * threads + tid].get(d);
        gn_sub<V>(xh, mean);
        gn_mul<V>(xh, rstd);
        gn_du<V, ACT>(d, xh, scale, bias);
        gn_add<V>(s1, d);
        gn_fma<V>(s2, d, xh);
      }
      // sums per channel, for dscale and dbias, and from them the groups' means; a
      // thread a channel where its row lanes are few, a warp where they are many
      const auto channel_sums = [&](const float (&s)[V], auto finish) {
        if (active)
#pragma unroll
          for (int j = 0; j < V; ++j) red[(cv * V + j) * h.rt + rl] = s[j];
        __syncthreads();
        for (int c = step_c == 1 ? tid : warp; c < width; c += step_c == 1 ? threads : warps) {
          float t = 0.f;
          for (int r = step_c == 1 ? 0 : lane; r < h.rt; r += step_c) t += red[c * h.rt + r];
          if (step_c > 1)
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
          if (step_c == 1 || lane == 0) finish(c, t);
        }
        __syncthreads();
      };
      channel_sums(s1, [&](int c, float t) { chan[c].x = t; });
      channel_sums(s2, [&](int c, float t) {
        const float2 v = make_float2(chan[c].x, t);
        acc[c] = !SHORT || b == turn ? v : fadd2(acc[c], v);  // a channel is always the same thread's
        chan[c] = fmul2(v, dup2(p.scale ? p.scale[c0 + c] : 1.f));
      });
      const int lanes = SHORT && g.cg <= 32 && ng > warps ? 1 : 32;  // for a group: a thread where its channels are few
      for (int q = lanes == 1 ? tid : warp; q < ng; q += lanes == 1 ? threads : warps) {
        float t1 = 0.f, t2 = 0.f;
        for (int c = lanes == 1 ? 0 : lane; c < g.cg; c += lanes) {
          t1 += chan[q * g.cg + c].x;
          t2 += chan[q * g.cg + c].y;
        }
        if (lanes > 1)
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            t1 += __shfl_xor_sync(0xffffffffu, t1, o);
            t2 += __shfl_xor_sync(0xffffffffu, t2, o);
          }
        if (lanes == 1 || lane == 0) own[q] = make_float2(t1, t2);
      }
      __syncthreads();
      if (h.ctas > 1) {
        gn_cluster_arrive();
        gn_cluster_wait();
      }
      if (SHORT && h.ctas == 1)
        for (int q = tid; q < ng; q += threads) all[q] = make_float2(own[q].x * per_group, own[q].y * per_group);
      for (int q = warp; (!SHORT || h.ctas > 1) && q < ng; q += warps) {
        float2 t = own[q];
        if (h.ctas > 1) {
          t = lane < h.ctas ? gn_peer(own + q, lane) : make_float2(0.f, 0.f);
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) {
            t.x += __shfl_xor_sync(0xffffffffu, t.x, o, 8);
            t.y += __shfl_xor_sync(0xffffffffu, t.y, o, 8);
          }
        }
        if (lane == 0) all[q] = make_float2(t.x * per_group, t.y * per_group);
      }
      __syncthreads();
      if (h.ctas > 1) gn_cluster_arrive();
      float m1[V], m2[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 m = all[grp[j]];
        m1[j] = m.x;
        m2[j] = -m.y;
      }
#pragma unroll 4
      for (int i = 0; i < mine; ++i) {
        float xh[V], d[V];
        hx[i * threads + tid].get(xh);
        hd[i * threads + tid].get(d);
        gn_sub<V>(xh, mean);
        gn_mul<V>(xh, rstd);
        gn_du<V, ACT>(d, xh, scale, bias);
        gn_mul<V>(d, scale);
        gn_sub<V>(d, m1);
        gn_fma<V>(d, xh, m2);  // m2 holds its negative
        gn_mul<V>(d, rstd);
        Vec::put(out + i * step, d);
      }
    }
    __syncwarp();
    if (h.ctas > 1) gn_cluster_wait();  // the others read this CTA's pairs
  }
  if (BWD)
    for (int c = step_c == 1 ? tid : warp; c < width; c += step_c == 1 ? threads : warps)
      if (step_c == 1 || lane == 0) p.sums[((int64_t)turn * h.ctas + rank) * g.D + c0 + c] = acc[c];
}

static int check_gn(const ssm_group_norm_params_t* p) {
  if (!p) return SSM_ERR_NULL;
  if (p->batch < 0 || p->seqlen < 0 || p->dim < 1 || p->groups < 1 || p->dim % p->groups || p->dim > (1 << 20) ||
      p->batch > 0x7fffffff / p->groups || p->seqlen > (1ll << 40) || p->act < SSM_ACT_NONE || p->act > SSM_ACT_RELU)
    return SSM_ERR_SHAPE;
  if (p->dtype != SSM_F32 && p->dtype != SSM_BF16) return SSM_ERR_DTYPE;
  // x, y, dy and dx of whole vectors a row are accessed by vectors
  if (!all_aligned(p->dim % 8 == 0 ? 16 : p->dtype == SSM_BF16 ? 2 : 4, {p->x, p->y, p->dy, p->dx}) ||
      !all_aligned(sizeof(float), {p->scale, p->bias, p->dscale, p->dbias}) || !all_aligned(sizeof(float2), {p->stats}) ||
      !all_aligned(kWorkspaceAlign, {p->workspace}))
    return SSM_ERR_ALIGN;
  return SSM_OK;
}

static bool gn_vector(const ssm_group_norm_params_t* p) { return p->dim % 8 == 0; }

static GnGeom gn_geom(const ssm_group_norm_params_t* p) {
  GnGeom g;
  g.B = (int)p->batch;
  g.L = p->seqlen;
  g.D = p->dim;
  g.G = p->groups;
  g.cg = p->dim / p->groups;
  const int V = gn_vector(p) ? 8 : 1;
  g.nvec = g.D / V;
  g.tiles = (g.nvec + kGnThreads - 1) / kGnThreads;
  g.ct = (g.nvec + g.tiles - 1) / g.tiles;
  g.rt = kGnThreads / g.ct;
  const int64_t want = 8 * 148;  // CTAs
  const int64_t per_b = (want + (int64_t)g.B * g.tiles - 1) / ((int64_t)g.B * g.tiles);
  int64_t chunk = (g.L + per_b - 1) / per_b;
  const int64_t least = (int64_t)g.rt * 8;
  chunk = chunk < least ? least : (chunk + least - 1) / least * least;
  g.chunk = chunk;
  g.chunks = (int)((g.L + chunk - 1) / chunk);
  return g;
}

// The held form's cut, or false where a group is too long for it.  Jobs are
// sized so that three CTAs share an SM (one's loads overlap another's sums), that
// rows read 64 bytes or more (with 16 a call of 16 x 4096 x 256 bf16 took 39 us
// for 24), and that small calls spread over the SMs.
constexpr size_t kHoldSmem = 74 * 1024;
constexpr int kHoldCtas = 32 * 148;  // at most, where there are that many batch rows
static bool gn_hold(const ssm_group_norm_params_t* p, bool bwd, GnHold* h, int* V) {
  const int es = p->dtype == SSM_BF16 ? 2 : 4, cg = p->dim / p->groups;
  const int wide = 16 / es;
  const bool vec = p->dim % wide == 0 && aligned16(p->x) && aligned16(bwd ? p->dx : p->y) && (!bwd || aligned16(p->dy));
  // the fewest groups that make whole vectors (all of them do) and 64 bytes
  int least = 1;
  *V = vec ? wide : 1;
  while (least < p->groups && (least * cg % *V || least * cg * es < 64)) ++least;
  bool found = false;
  for (int ctas = 1; ctas <= 8; ctas *= 2) {
    if (ctas > 1 && p->seqlen < ctas * 4) break;
    const int64_t rows = (p->seqlen + ctas - 1) / ctas;
    if (rows > 65536) continue;
    GnHold c;
    c.ctas = ctas;
    c.rows = rows;
    // The backward's held form keeps two inputs and runs the activation's slope
    // twice between two barriers of the cluster: with more than two CTAs the
    // split form's extra reads cost less (64 x 2048 x 768 bf16: 199 us for 338),
    // unless the call is small enough that its launches count.
    if (bwd && ctas > 2 && p->batch * p->seqlen * p->dim * es > (8 << 20)) break;
    const auto cut = [&](int gpj) {  // the job of gpj groups; whether it fits
      const size_t bytes = (size_t)rows * gpj * cg * es * (bwd ? 2 : 1);
      c.gpj = gpj;
      c.W = gpj * cg;
      c.jobs = (p->groups + gpj - 1) / gpj;
      c.nv = c.W / *V;
      if (c.nv > kHoldThreads) return false;
      // Half the threads, each with twice the rows, where four CTAs then share an SM
      // and there are several rounds of them: what a thread does once weighs less, and
      // a fourth CTA's loads are under way (64 x 2048 x 768 bf16 forward 95 us for 108,
      // 64 x 1024 x 768 53 for 55; with jobs of 64 KB, three to an SM, 35 for 32).
      const bool many = !bwd && *V > 1 && bytes <= 52 * 1024 && p->batch * c.jobs * ctas >= 8 * 148;
      c.threads = bytes > 4096 && !many ? 256 : 128;
      while (c.threads < c.nv) c.threads *= 2;
      c.rt = c.threads / c.nv;
      c.slots = (int)((rows + c.rt - 1) / c.rt);
      c.smem = ((size_t)c.slots * c.threads * *V * es * (bwd ? 2 : 1) + 15) / 16 * 16 +
               (size_t)c.threads * 4 * (bwd || cg % *V ? *V : 2) + (bwd ? 2 * (size_t)c.W : 0) * sizeof(float2) +
               2 * (size_t)gpj * sizeof(float2);
      c.turns = (int)std::min<int64_t>(p->batch, std::max(1, kHoldCtas / (c.jobs * ctas)));
      return c.smem <= kHoldSmem && (int64_t)c.jobs * c.turns * ctas <= 0x7fffffff;
    };
    if (!cut(least)) continue;
    int gpj = least;
    while (gpj + least <= p->groups && cut(gpj + least)) gpj += least;
    const auto count = [&](int q) { return p->batch * ((p->groups + q - 1) / q) * ctas; };
    while (gpj > least && gpj * cg * es > 128 && count(gpj) < 2 * 148) gpj -= least;
    cut(gpj);
    *h = c;
    found = true;
    if (count(gpj) >= 2 * 148) break;
  }
  return found;
}

static size_t gn_round(size_t v) { return (v + 255) / 256 * 256; }
static size_t gn_stats_bytes(const ssm_group_norm_params_t* p) {  // of statistics that the caller does not keep
  return p->stats ? 0 : gn_round((size_t)p->batch * p->groups * sizeof(float2));
}
static size_t gn_part_bytes(const GnGeom& g) { return gn_round((size_t)g.B * g.chunks * g.D * sizeof(float2)); }
static size_t gn_sums_bytes(const GnGeom& g) { return gn_round((size_t)g.B * g.D * sizeof(float2)); }
static size_t gn_means_bytes(const GnGeom& g) { return gn_round((size_t)g.B * g.G * sizeof(float2)); }

template <typename T, int V, int ACT>
static void gn_fwd_launch(const GnArgs& a, cudaStream_t s) {
  const GnGeom& g = a.g;
  const dim3 grid((unsigned)(g.chunks * g.B), 1, g.tiles);
  constexpr size_t ring = kGnRing<T, V, 1>;
  const size_t smem = std::max(ring, (2 * (size_t)g.rt * g.ct * V + g.rt) * sizeof(float));
  if (ring > 48 * 1024) {
    cudaFuncSetAttribute(gn_stats_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring);
    cudaFuncSetAttribute(gn_apply_kernel<T, V, ACT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring);
    cudaFuncSetAttribute(gn_apply_kernel<T, V, ACT, V == 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring);
  }
  gn_stats_kernel<T, V><<<grid, kGnThreads, smem, s>>>(a);
  gn_merge_kernel<<<g.B * g.G, kMergeThreads, 0, s>>>(a);
  if (g.cg % V == 0) gn_apply_kernel<T, V, ACT, true><<<grid, kGnThreads, ring, s>>>(a);
  else gn_apply_kernel<T, V, ACT, V == 1><<<grid, kGnThreads, ring, s>>>(a);
  note_launches(3);
}

template <typename T, int V, int ACT, bool ONE>
static void gn_bwd_launch_one(const GnArgs& a, cudaStream_t s) {
  const GnGeom& g = a.g;
  const dim3 grid((unsigned)(g.chunks * g.B), 1, g.tiles);
  constexpr size_t ring = kGnRing<T, V, 2>;
  const size_t smem = std::max(ring, 2 * (size_t)g.rt * g.ct * V * sizeof(float));
  if (ring > 48 * 1024) {
    cudaFuncSetAttribute(gn_sums_kernel<T, V, ACT, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring);
    cudaFuncSetAttribute(gn_dx_kernel<T, V, ACT, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring);
  }
  gn_sums_kernel<T, V, ACT, ONE><<<grid, kGnThreads, smem, s>>>(a);
  gn_means_kernel<<<g.B * g.G, kMergeThreads, 0, s>>>(a);
  gn_dx_kernel<T, V, ACT, ONE><<<grid, kGnThreads, ring, s>>>(a);
  gn_param_kernel<<<(g.D + 31) / 32, 1024, 0, s>>>(a.sums, g.B, g.D, a.dscale, a.dbias);
  note_launches(4);
}
template <typename T, int V, int ACT>
static void gn_bwd_launch(const GnArgs& a, cudaStream_t s) {
  if (a.g.cg % V == 0) gn_bwd_launch_one<T, V, ACT, true>(a, s);
  else gn_bwd_launch_one<T, V, ACT, V == 1>(a, s);
}

template <typename T, int V>
static void gn_launch(const GnArgs& a, int act, bool bwd, cudaStream_t s) {
  switch (act) {
    case SSM_ACT_SILU: return bwd ? gn_bwd_launch<T, V, SSM_ACT_SILU>(a, s) : gn_fwd_launch<T, V, SSM_ACT_SILU>(a, s);
    case SSM_ACT_GELU: return bwd ? gn_bwd_launch<T, V, SSM_ACT_GELU>(a, s) : gn_fwd_launch<T, V, SSM_ACT_GELU>(a, s);
    case SSM_ACT_RELU: return bwd ? gn_bwd_launch<T, V, SSM_ACT_RELU>(a, s) : gn_fwd_launch<T, V, SSM_ACT_RELU>(a, s);
    default: return bwd ? gn_bwd_launch<T, V, SSM_ACT_NONE>(a, s) : gn_fwd_launch<T, V, SSM_ACT_NONE>(a, s);
  }
}

template <typename T, int V, int ACT, bool BWD, bool SHORT>
static cudaError_t gn_hold_launch(const GnArgs& a, const GnHold& h, cudaStream_t s) {
  const auto kernel = gn_hold_kernel<T, V, ACT, BWD, SHORT>;
  if (h.smem > 48 * 1024) {  // the kernel's limit, always the same: another thread may be launching it too
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kHoldSmem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(h.turns * h.jobs * h.ctas));
  cfg.blockDim = dim3(h.threads);
  cfg.dynamicSmemBytes = h.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = h.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, h);
  note_launches(1);
  if (BWD && e == cudaSuccess && (a.dscale || a.dbias)) {
    gn_param_kernel<<<(a.g.D + 31) / 32, 1024, 0, s>>>(a.sums, h.turns * h.ctas, a.g.D, a.dscale, a.dbias);
    note_launches(1);
  }
  return e;
}
template <typename T, int V, int ACT, bool BWD>
static cudaError_t gn_hold_length(const GnArgs& a, const GnHold& h, cudaStream_t s) {
  return h.turns < a.g.B || h.rows <= 4 ? gn_hold_launch<T, V, ACT, BWD, true>(a, h, s) : gn_hold_launch<T, V, ACT, BWD, false>(a, h, s);
}
template <typename T, int V, bool BWD>
static cudaError_t gn_hold_act(const GnArgs& a, const GnHold& h, int act, cudaStream_t s) {
  switch (act) {
    case SSM_ACT_SILU: return gn_hold_length<T, V, SSM_ACT_SILU, BWD>(a, h, s);
    case SSM_ACT_GELU: return gn_hold_length<T, V, SSM_ACT_GELU, BWD>(a, h, s);
    case SSM_ACT_RELU: return gn_hold_length<T, V, SSM_ACT_RELU, BWD>(a, h, s);
    default: return gn_hold_length<T, V, SSM_ACT_NONE, BWD>(a, h, s);
  }
}
template <bool BWD>
static cudaError_t gn_hold_run(const ssm_group_norm_params_t* p, const GnArgs& a, const GnHold& h, int V, cudaStream_t s) {
  if (p->dtype == SSM_BF16)
    return V == 1 ? gn_hold_act<__nv_bfloat16, 1, BWD>(a, h, p->act, s) : gn_hold_act<__nv_bfloat16, 8, BWD>(a, h, p->act, s);
  return V == 1 ? gn_hold_act<float, 1, BWD>(a, h, p->act, s) : gn_hold_act<float, 4, BWD>(a, h, p->act, s);
}

static int gn_dispatch(const ssm_group_norm_params_t* p, GnArgs& a, bool bwd, cudaStream_t s) {
  GnHold h;
  int V;
  if (gn_hold(p, bwd, &h, &V)) {
    a.sums = reinterpret_cast<float2*>(p->workspace);
    cudaError_t e = bwd ? gn_hold_run<true>(p, a, h, V, s) : gn_hold_run<false>(p, a, h, V, s);
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? SSM_OK : launch_error("launch group norm kernel", e);
  }
  const bool vec = gn_vector(p);
  if (p->dtype == SSM_BF16) {
    if (vec) gn_launch<__nv_bfloat16, 8>(a, p->act, bwd, s);
    else gn_launch<__nv_bfloat16, 1>(a, p->act, bwd, s);
  } else {
    if (vec) gn_launch<float, 8>(a, p->act, bwd, s);
    else gn_launch<float, 1>(a, p->act, bwd, s);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SSM_OK : launch_error("launch group norm kernel", e);
}

}  // namespace ssm

using namespace ssm;

extern "C" {

size_t ssm_group_norm_fwd_workspace_bytes(const ssm_group_norm_params_t* p) {
  if (check_gn(p) || p->batch == 0 || p->seqlen == 0) return 0;
  GnHold h;
  int V;
  // without the pointers their alignment, which has a say in the form, is unknown
  return p->x && p->y && gn_hold(p, false, &h, &V)
             ? 0
             : gn_part_bytes(gn_geom(p)) + gn_stats_bytes(p);
}

size_t ssm_group_norm_bwd_workspace_bytes(const ssm_group_norm_params_t* p) {
  if (check_gn(p) || p->batch == 0 || p->seqlen == 0) return 0;
  const GnGeom g = gn_geom(p);
  GnHold h;
  int V;
  if (p->x && p->dy && p->dx && gn_hold(p, true, &h, &V))
    return gn_round((size_t)h.turns * h.ctas * g.D * sizeof(float2));
  // without the pointers their alignment, which has a say in the form, is unknown
  const size_t split = gn_part_bytes(g) + gn_sums_bytes(g) + gn_means_bytes(g);
  return std::max(split, gn_round((size_t)std::min<int64_t>(8 * p->batch, kHoldCtas + 8) * g.D * sizeof(float2)));
}

int ssm_group_norm_act_fwd(const ssm_group_norm_params_t* p, ssm_stream_t stream) {
  int st = check_gn(p);
  if (st) return st;
  if (p->batch == 0 || p->seqlen == 0) return SSM_OK;
  if (!p->x || !p->y) return SSM_ERR_NULL;
  const size_t need = ssm_group_norm_fwd_workspace_bytes(p);
  if (need && (!p->workspace || p->workspace_bytes < need)) return SSM_ERR_WORKSPACE;
  st = bind_device(p->x);
  if (st) return st;
  GnArgs a = {};
  a.g = gn_geom(p);
  a.eps = p->eps;
  a.x = p->x;
  a.scale = p->scale;
  a.bias = p->bias;
  a.stats = p->stats;
  a.part = static_cast<float2*>(p->workspace);
  // the split form's second pass reads the statistics; the held one keeps them itself
  if (!a.stats && need) a.stats = reinterpret_cast<float*>(static_cast<char*>(p->workspace) + gn_part_bytes(a.g));
  a.out = p->y;
  return gn_dispatch(p, a, false, reinterpret_cast<cudaStream_t>(stream));
}

int ssm_group_norm_act_bwd(const ssm_group_norm_params_t* p, ssm_stream_t stream) {
  int st = check_gn(p);
  if (st) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (p->batch == 0 || p->seqlen == 0) {
    for (float* d : {p->dscale, p->dbias}) {
      if (!d) continue;
      st = bind_device(d);
      if (st) return st;
      const cudaError_t e = cudaMemsetAsync(d, 0, (size_t)p->dim * sizeof(float), s);
      if (e != cudaSuccess) return launch_error("cudaMemsetAsync(group norm sums)", e);
    }
    return SSM_OK;
  }
  if (!p->x || !p->dy || !p->dx || !p->stats) return SSM_ERR_NULL;
  if (!p->workspace || p->workspace_bytes < ssm_group_norm_bwd_workspace_bytes(p)) return SSM_ERR_WORKSPACE;
  st = bind_device(p->x);
  if (st) return st;
  GnArgs a = {};
  a.g = gn_geom(p);
  a.x = p->x;
  a.dy = p->dy;
  a.scale = p->scale;
  a.bias = p->bias;
  a.stats = p->stats;
  char* w = static_cast<char*>(p->workspace);
  a.part = reinterpret_cast<float2*>(w);
  w += gn_part_bytes(a.g);
  a.sums = reinterpret_cast<float2*>(w);
  w += gn_sums_bytes(a.g);
  a.means = reinterpret_cast<float2*>(w);
  a.out = p->dx;
  a.dscale = p->dscale;
  a.dbias = p->dbias;
  return gn_dispatch(p, a, true, s);
}

}  // extern "C"
