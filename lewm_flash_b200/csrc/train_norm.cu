// Layer norm and adaptive layer norm for training: forward, and a backward pass that also
// reduces the gradients of the weights or of the modulation.
//
// Row r of n values, z = (x - mu) rs, mu = mean(x), rs = 1 / sqrt(mean((x - mu)^2) + eps):
//   y  = z a + b
//   d  = dy a,  dx = rs (d - mean(d) - z mean(d z))
//   da = sum over rows of dy z,  db = sum over rows of dy
// Layer norm: a = weight, b = bias, one (a, b) for all rows. Adaptive layer norm (reference
// lewm/module.py:6-8,96-110: modulate(norm(x), shift, scale)): a = 1 + scale, b = shift, one
// (a, b) per `group` consecutive rows. Both are the same computation over groups of rows that
// share (a, b), with one group for layer norm, so one kernel each way serves both.
//
// Bound: bytes. About 10 (forward) and 16 (backward) instructions per element against 4 to 12
// bytes of HBM traffic. A row therefore stays in registers from its only load to its only
// store (mean and variance are two passes over registers), and sums over rows are kept in
// registers by persistent blocks that own fixed columns, so x and dy are read once.
//
// Layout: a team of TPR threads holds one row, NV vectors of E elements per thread (16-byte
// vectors where every row starts on 16 bytes, else single elements), at most 16 elements a
// thread: the backward then holds 16 gains, 32 sums and the raw row, 128 registers at two
// 256-thread blocks per SM. Rows wider than 16384 take the looping kernels below.
//
// Work is cut into items: a run of rows within one group. An item is a block's (its teams
// interleave the rows and add up through shared memory), or a team's where there are many
// groups of few rows. A group cut into several items writes float32
// partial sums, which k_norm_reduce adds in a fixed order: no atomics, the same bits on every
// run of the same shape.
//
// Types: x, y, dy, dx are float32, bf16 or fp16; weights and modulation are float32 or any of
// these; all arithmetic, statistics and sums are float32, rounded once at the store.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdarg>
#include <cstdio>

#include "lewm_b200.h"
#include "lewm_common.cuh"
#include "lewm_internal.h"

namespace lewm {
namespace {

constexpr int kSms = 148;          // B200
constexpr int kMaxRowRegs = 16384;  // widest row held in registers (1024 threads x 16)

struct NormArgs {
  const void* x;
  const void* dy;
  const void* a;       // weight or scale, or null (a = 1)
  const void* b;       // bias or shift, or null
  void* out;           // y or dx
  float* stats;        // [2][rows]: mu, rs
  void* da;            // [groups][width] in the parameters' type, or null
  void* db;
  float* ws;           // [groups * split][2][width] partial sums when split > 1
  int64_t rows, x_stride, dy_stride, a_stride, b_stride;
  int64_t group;       // rows per (a, b)
  int64_t items;       // groups * split
  int64_t chunk;       // rows per item
  int split;           // items per group
  int width;
  int p_type;
  int one_plus;        // a = 1 + a[]
  int team_items;      // 1: an item per team, 0: per block
  float eps;
};

// ------------------------------------------------------------------ element types
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// E consecutive elements moved as one access.
template <typename T, int E>
struct alignas(sizeof(T) * E) Vec {
  T v[E];
};

// E parameters at element offset `at` as float32, whatever their type.
template <int E>
__device__ __forceinline__ void load_params(const void* p, int type, int64_t at, float* f) {
  if (type == LEWM_TYPE_F32) {
    const float* q = static_cast<const float*>(p) + at;
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = q[e];
  } else if (type == LEWM_TYPE_BF16) {
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p) + at;
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = to_f(q[e]);
  } else {
    const __half* q = static_cast<const __half*>(p) + at;
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = to_f(q[e]);
  }
}
__device__ __forceinline__ void store_param(void* p, int type, int64_t at, float f) {
  if (type == LEWM_TYPE_F32) static_cast<float*>(p)[at] = f;
  else if (type == LEWM_TYPE_BF16) static_cast<__nv_bfloat16*>(p)[at] = from_f<__nv_bfloat16>(f);
  else static_cast<__half*>(p)[at] = from_f<__half>(f);
}

// ------------------------------------------------------------------ team sums
// Sum of `v` over the TPR threads of a team, the same bits in all of them. Teams of more than
// a warp add their warps' sums through `red` (a slot per warp of the block) in warp order;
// every thread of the block must call it. One barrier per call: the caller alternates between
// two `red` buffers, so a buffer is rewritten only after a later barrier.
template <int TPR>
__device__ __forceinline__ float team_sum(float v, float* red) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    const int w0 = warp / (TPR / 32) * (TPR / 32);
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) v += red[w0 + i];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ float2 team_sum2(float2 v, float2* red) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    const int w0 = warp / (TPR / 32) * (TPR / 32);
    v = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) {
      v.x += red[w0 + i].x;
      v.y += red[w0 + i].y;
    }
  }
  return v;
}

// Rows of an item: [r0, r1) within group g.
struct Item {
  int64_t g, r0, r1;
};
__device__ __forceinline__ Item item_rows(const NormArgs& p, int64_t item) {
  Item it{0, 0, 0};
  if (item >= p.items) return it;  // no rows
  it.g = item / p.split;
  const int64_t s = item - it.g * p.split;
  it.r0 = it.g * p.group + s * p.chunk;
  it.r1 = min(it.r0 + p.chunk, (it.g + 1) * p.group);
  return it;
}

constexpr int block_threads(int tpr) { return tpr < 256 ? 256 : tpr; }
constexpr int blocks_per_sm(int tpr, bool backward) { return (backward ? 512 : 1024) / block_threads(tpr); }

// ------------------------------------------------------------------ forward
template <typename T, int E, int NV, int TPR>
__global__ void __launch_bounds__(block_threads(TPR), blocks_per_sm(TPR, false)) k_norm_fwd(const NormArgs p) {
  griddep_wait();  // launched as a programmatic dependent: wait for the kernel before
  constexpr int TEAMS = block_threads(TPR) / TPR;
  using V = Vec<T, E>;
  __shared__ float red[2][32];
  const int team = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  const int nvec = p.width / E;
  const float inv_n = 1.0f / p.width;
  const int64_t step = p.team_items ? 1 : TEAMS;
  const int64_t iters = (p.chunk + step - 1) / step;
  const int64_t per_block = p.team_items ? TEAMS : 1;
  for (int64_t base = blockIdx.x * per_block; base < p.items; base += gridDim.x * per_block) {
    const Item it = item_rows(p, base + (p.team_items ? team : 0));
    float ga[NV * E], gb[NV * E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * TPR;
#pragma unroll
      for (int e = 0; e < E; ++e) ga[i * E + e] = 1.f, gb[i * E + e] = 0.f;
      if (v < nvec && it.r0 < it.r1) {
        if (p.a) load_params<E>(p.a, p.p_type, it.g * p.a_stride + (int64_t)v * E, ga + i * E);
        if (p.b) load_params<E>(p.b, p.p_type, it.g * p.b_stride + (int64_t)v * E, gb + i * E);
        if (p.one_plus) {
#pragma unroll
          for (int e = 0; e < E; ++e) ga[i * E + e] += 1.f;
        }
      }
    }
    for (int64_t k = 0; k < iters; ++k) {
      const int64_t r = it.r0 + (p.team_items ? 0 : team) + k * step;
      const bool live = r < it.r1;
      float f[NV * E];
      V raw[NV];
      const T* xr = static_cast<const T*>(p.x) + r * p.x_stride;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * TPR;
        if (live && v < nvec) raw[i] = *reinterpret_cast<const V*>(xr + (int64_t)v * E);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool in = live && lane + i * TPR < nvec;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          f[i * E + e] = in ? to_f(raw[i].v[e]) : 0.f;
          s += f[i * E + e];
        }
      }
      const float mu = team_sum<TPR>(s, red[0]) * inv_n;
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool in = lane + i * TPR < nvec;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float c = in ? f[i * E + e] - mu : 0.f;
          q = fmaf(c, c, q);
        }
      }
      const float var = team_sum<TPR>(q, red[1]) * inv_n;
      const float rs = 1.0f / sqrtf(var + p.eps);
      if (!live) continue;
      if (p.stats && lane == 0) {
        p.stats[r] = mu;
        p.stats[p.rows + r] = rs;
      }
      T* yr = static_cast<T*>(p.out) + r * p.width;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * TPR;
        if (v >= nvec) continue;
        V o;
#pragma unroll
        for (int e = 0; e < E; ++e)
          o.v[e] = from_f<T>(fmaf((f[i * E + e] - mu) * rs, ga[i * E + e], gb[i * E + e]));
        *reinterpret_cast<V*>(yr + (int64_t)v * E) = o;
      }
    }
  }
}

// Where the sums of column `col` of an item go.
__device__ __forceinline__ void store_sums(const NormArgs& p, int64_t item, int64_t g, int64_t col, float a, float b) {
  if (p.split > 1) {
    float* w = p.ws + item * 2 * p.width + col;
    w[0] = a;
    w[p.width] = b;
  } else {
    if (p.da) store_param(p.da, p.p_type, g * p.width + col, a);
    if (p.db) store_param(p.db, p.p_type, g * p.width + col, b);
  }
}

// ------------------------------------------------------------------ backward
template <typename T, int E, int NV, int TPR>
__global__ void __launch_bounds__(block_threads(TPR), TPR < 1024 ? blocks_per_sm(TPR, true) : 1) k_norm_bwd(const NormArgs p) {
  griddep_wait();  // launched as a programmatic dependent: wait for the kernel before
  constexpr int THREADS = block_threads(TPR), TEAMS = THREADS / TPR;
  using V = Vec<T, E>;
  __shared__ float2 red[2][32];
  __shared__ float2 sums[TEAMS > 1 ? TEAMS : 1][TEAMS > 1 ? TPR * E : 1];
  const int team = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  const int nvec = p.width / E;
  const float inv_n = 1.0f / p.width;
  const int64_t step = p.team_items ? 1 : TEAMS;
  const int64_t iters = (p.chunk + step - 1) / step;
  const int64_t per_block = p.team_items ? TEAMS : 1;
  int flip = 0;
  for (int64_t base = blockIdx.x * per_block; base < p.items; base += gridDim.x * per_block) {
    const int64_t item = base + (p.team_items ? team : 0);
    const Item it = item_rows(p, item);
    float ga[NV * E], sa[NV * E], sb[NV * E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * TPR;
#pragma unroll
      for (int e = 0; e < E; ++e) ga[i * E + e] = 1.f, sa[i * E + e] = 0.f, sb[i * E + e] = 0.f;
      if (p.a && v < nvec && it.r0 < it.r1) {
        load_params<E>(p.a, p.p_type, it.g * p.a_stride + (int64_t)v * E, ga + i * E);
        if (p.one_plus) {
#pragma unroll
          for (int e = 0; e < E; ++e) ga[i * E + e] += 1.f;
        }
      }
    }
    for (int64_t k = 0; k < iters; ++k) {
      const int64_t r = it.r0 + (p.team_items ? 0 : team) + k * step;
      const bool live = r < it.r1;
      V rx[NV], rd[NV];
      const T* xr = static_cast<const T*>(p.x) + r * p.x_stride;
      const T* dr = static_cast<const T*>(p.dy) + r * p.dy_stride;
      float mu = 0.f, rs = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * TPR;
        if (live && v < nvec) {
          rx[i] = *reinterpret_cast<const V*>(xr + (int64_t)v * E);
          rd[i] = *reinterpret_cast<const V*>(dr + (int64_t)v * E);
        }
      }
      if (live) {
        mu = p.stats[r];
        rs = p.stats[p.rows + r];
      }
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!(live && lane + i * TPR < nvec)) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float z = (to_f(rx[i].v[e]) - mu) * rs, g = to_f(rd[i].v[e]), d = g * ga[i * E + e];
          s.x += d;
          s.y = fmaf(d, z, s.y);
          sa[i * E + e] = fmaf(g, z, sa[i * E + e]);
          sb[i * E + e] += g;
        }
      }
      if (!p.out) continue;  // only the parameters' gradients are wanted
      s = team_sum2<TPR>(s, red[flip]);
      flip ^= 1;
      if (!live) continue;
      const float m1 = s.x * inv_n, m2 = s.y * inv_n;
      T* o = static_cast<T*>(p.out) + r * p.width;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * TPR;
        if (v >= nvec) continue;
        V w;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float z = (to_f(rx[i].v[e]) - mu) * rs, d = to_f(rd[i].v[e]) * ga[i * E + e];
          w.v[e] = from_f<T>(rs * (d - m1 - z * m2));
        }
        *reinterpret_cast<V*>(o + (int64_t)v * E) = w;
      }
    }
    if (!p.da && !p.db) continue;
    if (p.team_items || TEAMS == 1) {
      if (it.r0 >= it.r1) continue;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * TPR;
        if (v >= nvec) continue;
#pragma unroll
        for (int e = 0; e < E; ++e)
          store_sums(p, item, it.g, (int64_t)v * E + e, sa[i * E + e], sb[i * E + e]);
      }
    } else {
      // Add the teams' sums in team order, a slab of TPR vectors of columns at a time.
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i * TPR >= nvec) break;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) sums[team][lane * E + e] = make_float2(sa[i * E + e], sb[i * E + e]);
        __syncthreads();
        for (int c = threadIdx.x; c < TPR * E; c += THREADS) {
          float a = 0.f, b = 0.f;
#pragma unroll
          for (int t = 0; t < TEAMS; ++t) a += sums[t][c].x, b += sums[t][c].y;
          const int64_t col = (int64_t)i * TPR * E + c;
          if (col < p.width) store_sums(p, item, it.g, col, a, b);
        }
      }
      __syncthreads();
    }
  }
}

// Sum of the `split` partial sums of each group, in item order within 32 interleaved runs and
// then over the runs: 32 columns x 32 rows per block, grid (column tiles, groups, a or b).
__global__ void __launch_bounds__(1024) k_norm_reduce(const NormArgs p) {
  griddep_wait();
  __shared__ float part[32][33];
  const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.x;
  void* out = blockIdx.z ? p.db : p.da;
  if (!out) return;
  const int64_t groups = p.items / p.split;
  for (int64_t g = blockIdx.y; g < groups; g += gridDim.y) {
    float s = 0.f;
    if (col < p.width) {
      const float* w = p.ws + (g * p.split * 2 + blockIdx.z) * p.width + col;
#pragma unroll 4
      for (int i = threadIdx.y; i < p.split; i += 32) s += w[(int64_t)i * 2 * p.width];
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    // Warp c adds column c's 32 runs.
    float t = warp_sum(part[threadIdx.x][threadIdx.y]);
    const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && c < p.width) store_param(out, p.p_type, g * p.width + c, t);
    __syncthreads();
  }
}

// ------------------------------------------------------------------ rows wider than kMaxRowRegs
// One block per row, the row re-read from L2 for each pass.
template <typename T>
__global__ void __launch_bounds__(1024) k_norm_fwd_wide(const NormArgs p) {
  griddep_wait();
  __shared__ float red[2][32];
  const float inv_n = 1.0f / p.width;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x; c < p.width; c += 1024) s += to_f(x[c]);
    const float mu = team_sum<1024>(s, red[0]) * inv_n;
    for (int c = threadIdx.x; c < p.width; c += 1024) {
      const float d = to_f(x[c]) - mu;
      q = fmaf(d, d, q);
    }
    const float rs = 1.0f / sqrtf(team_sum<1024>(q, red[1]) * inv_n + p.eps);
    if (p.stats && threadIdx.x == 0) {
      p.stats[r] = mu;
      p.stats[p.rows + r] = rs;
    }
    const int64_t g = r / p.group;
    T* y = static_cast<T*>(p.out) + r * p.width;
    for (int c = threadIdx.x; c < p.width; c += 1024) {
      float a = 1.f, b = 0.f;
      if (p.a) load_params<1>(p.a, p.p_type, g * p.a_stride + c, &a);
      if (p.b) load_params<1>(p.b, p.p_type, g * p.b_stride + c, &b);
      if (p.one_plus) a += 1.f;
      y[c] = from_f<T>(fmaf((to_f(x[c]) - mu) * rs, a, b));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) k_norm_dx_wide(const NormArgs p) {
  griddep_wait();
  __shared__ float2 red[2][32];
  const float inv_n = 1.0f / p.width;
  int flip = 0;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
    const T* dy = static_cast<const T*>(p.dy) + r * p.dy_stride;
    const float mu = p.stats[r], rs = p.stats[p.rows + r];
    const int64_t g = r / p.group;
    auto gain = [&](int c) {
      float a = 1.f;
      if (p.a) load_params<1>(p.a, p.p_type, g * p.a_stride + c, &a);
      return p.one_plus ? a + 1.f : a;
    };
    float2 s = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < p.width; c += 1024) {
      const float d = to_f(dy[c]) * gain(c);
      s.x += d;
      s.y = fmaf(d, (to_f(x[c]) - mu) * rs, s.y);
    }
    s = team_sum2<1024>(s, red[flip]);
    flip ^= 1;
    const float m1 = s.x * inv_n, m2 = s.y * inv_n;
    T* o = static_cast<T*>(p.out) + r * p.width;
    for (int c = threadIdx.x; c < p.width; c += 1024) {
      const float z = (to_f(x[c]) - mu) * rs, d = to_f(dy[c]) * gain(c);
      o[c] = from_f<T>(rs * (d - m1 - z * m2));
    }
  }
}

// The sums of dy z and dy: a thread per column, a block per 256 columns and item.
template <typename T>
__global__ void __launch_bounds__(256) k_norm_sums_wide(const NormArgs p) {
  griddep_wait();
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= p.width) return;
  for (int64_t item = blockIdx.y; item < p.items; item += gridDim.y) {
    const Item it = item_rows(p, item);
    if (it.r0 >= it.r1) {
      if (p.split > 1) store_sums(p, item, it.g, col, 0.f, 0.f);
      continue;
    }
    float a = 0.f, b = 0.f;
    for (int64_t r = it.r0; r < it.r1; ++r) {
      const float g = to_f(static_cast<const T*>(p.dy)[r * p.dy_stride + col]);
      const float z = (to_f(static_cast<const T*>(p.x)[r * p.x_stride + col]) - p.stats[r]) * p.stats[p.rows + r];
      a = fmaf(g, z, a);
      b += g;
    }
    store_sums(p, item, it.g, col, a, b);
  }
}

// ------------------------------------------------------------------ host side
// Team size of a row: threads x elements per thread covers the width.
struct Tier {
  int tpr, teams, ept;
};
Tier tier_of(int64_t width) {
  if (width <= 64) return {8, 32, 8};
  if (width <= 256) return {32, 8, 8};
  int tpr = 32;
  while (tpr * 16 < width) tpr *= 2;  // width <= kMaxRowRegs: tpr <= 1024
  return {tpr, block_threads(tpr) / tpr, 16};
}

// Blocks that fill the GPU: 256-thread blocks with up to 128 registers a thread, two per SM
// backward; the lighter forward four.
int64_t full_grid(const Tier& t, bool backward) {
  const int per_sm = backward ? 2 : 4;
  return (int64_t)kSms * std::max(1, per_sm * 256 / block_threads(t.tpr));
}

// How rows are cut into items; the same function sizes the workspace.
void cut_items(NormArgs* p, bool backward) {
  const int64_t groups = p->rows / p->group;
  if (p->width > kMaxRowRegs) {
    // Column blocks x items: split each group until the grid has about 8 blocks per SM.
    const int64_t cols = (p->width + 255) / 256;
    const int64_t want = (int64_t)kSms * 8 / std::max<int64_t>(1, cols * groups);
    p->team_items = 0;
    p->split = (int)std::max<int64_t>(1, std::min<int64_t>(want, p->group));
  } else {
    const Tier t = tier_of(p->width);
    // A team's items where a group has too few rows to keep a block's teams busy and there
    // are groups enough to fill the GPU without splitting them.
    p->team_items = p->group < 2 * t.teams && groups >= 2 * kSms;
    const int64_t want = (full_grid(t, backward) + groups - 1) / groups;
    const int64_t most = (p->group + t.teams - 1) / t.teams;
    p->split = p->team_items ? 1 : (int)std::max<int64_t>(1, std::min(want, most));
  }
  p->chunk = (p->group + p->split - 1) / p->split;
  p->split = (int)((p->group + p->chunk - 1) / p->chunk);  // no empty item
  p->items = groups * p->split;
}

size_t workspace_bytes(const NormArgs& p) {
  return p.split > 1 ? (size_t)p.items * 2 * (size_t)p.width * sizeof(float) : 0;
}

template <typename T, int E, int NV, int TPR>
cudaError_t launch_tier(const NormArgs& p, bool backward, cudaStream_t st) {
  const Tier t{TPR, block_threads(TPR) / TPR, NV * E};
  const int64_t blocks = p.team_items ? (p.items + t.teams - 1) / t.teams : p.items;
  const dim3 grid((unsigned)std::min(blocks, full_grid(t, backward)));
  return backward ? launch_k(k_norm_bwd<T, E, NV, TPR>, grid, dim3(block_threads(TPR)), 0, st, p)
                  : launch_k(k_norm_fwd<T, E, NV, TPR>, grid, dim3(block_threads(TPR)), 0, st, p);
}

template <typename T, int E>
cudaError_t launch_width(const NormArgs& p, bool backward, cudaStream_t st) {
  switch (tier_of(p.width).tpr) {
    case 8: return launch_tier<T, E, 8 / E, 8>(p, backward, st);
    case 32:
      return p.width <= 256 ? launch_tier<T, E, 8 / E, 32>(p, backward, st)
                            : launch_tier<T, E, 16 / E, 32>(p, backward, st);
    case 64: return launch_tier<T, E, 16 / E, 64>(p, backward, st);
    case 128: return launch_tier<T, E, 16 / E, 128>(p, backward, st);
    case 256: return launch_tier<T, E, 16 / E, 256>(p, backward, st);
    case 512: return launch_tier<T, E, 16 / E, 512>(p, backward, st);
    default: return launch_tier<T, E, 16 / E, 1024>(p, backward, st);
  }
}

template <typename T>
cudaError_t launch_wide(const NormArgs& p, bool backward, cudaStream_t st) {
  const dim3 rows_grid((unsigned)std::min<int64_t>(p.rows, 2 * kSms));
  if (!backward) return launch_k(k_norm_fwd_wide<T>, rows_grid, dim3(1024), 0, st, p);
  if (p.out) {
    const cudaError_t e = launch_k(k_norm_dx_wide<T>, rows_grid, dim3(1024), 0, st, p);
    if (e != cudaSuccess) return e;
  }
  if (!p.da && !p.db) return cudaSuccess;
  const dim3 grid((unsigned)((p.width + 255) / 256), (unsigned)std::min<int64_t>(p.items, 65535));
  return launch_k(k_norm_sums_wide<T>, grid, dim3(256), 0, st, p);
}

template <typename T>
cudaError_t launch_type(const NormArgs& p, bool backward, bool vec, cudaStream_t st) {
  if (p.width > kMaxRowRegs) return launch_wide<T>(p, backward, st);
  return vec ? launch_width<T, 16 / sizeof(T)>(p, backward, st) : launch_width<T, 1>(p, backward, st);
}

cudaError_t launch_norm(const NormArgs& p, int x_type, bool backward, cudaStream_t st) {
  const int64_t size = x_type == LEWM_TYPE_F32 ? 4 : 2;
  auto aligned = [&](const void* q, int64_t stride) {
    return !q || ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(stride * size)) & 15) == 0;
  };
  const bool vec = aligned(p.x, p.x_stride) && aligned(p.out, p.width) &&
                   (!backward || aligned(p.dy, p.dy_stride)) && (p.width * size) % 16 == 0;
  cudaError_t e = x_type == LEWM_TYPE_F32    ? launch_type<float>(p, backward, vec, st)
                  : x_type == LEWM_TYPE_BF16 ? launch_type<__nv_bfloat16>(p, backward, vec, st)
                                             : launch_type<__half>(p, backward, vec, st);
  if (e != cudaSuccess || !backward || p.split == 1 || (!p.da && !p.db)) return e;
  const int64_t groups = p.items / p.split;
  const dim3 grid((unsigned)((p.width + 31) / 32), (unsigned)std::min<int64_t>(groups, 65535), 2);
  return launch_k(k_norm_reduce, grid, dim3(32, 32), 0, st, p);
}

lewm_status norm_fail(lewm_status s, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  set_noctx_error(buf);
  return s;
}

bool type_ok(int32_t t) { return t == LEWM_TYPE_F32 || t == LEWM_TYPE_BF16 || t == LEWM_TYPE_F16; }

// Checks a descriptor and fills the arguments that both passes share.
lewm_status norm_args(const lewm_norm_desc* d, NormArgs* p) {
  if (!d) return norm_fail(LEWM_INVALID_ARG, "norm desc is NULL");
  if (d->rows < 0 || d->width <= 0)
    return norm_fail(LEWM_INVALID_ARG, "need rows >= 0 and width >= 1, got %lld x %lld", (long long)d->rows,
                     (long long)d->width);
  if (d->width > (1 << 24))
    return norm_fail(LEWM_UNSUPPORTED_SHAPE, "width %lld exceeds 2^24", (long long)d->width);
  if (!type_ok(d->x_type) || !type_ok(d->p_type))
    return norm_fail(LEWM_INVALID_ARG, "unknown element type %d / %d", d->x_type, d->p_type);
  if (!(d->eps >= 0.f)) return norm_fail(LEWM_INVALID_ARG, "eps must be >= 0");
  if (d->x_stride < 0 || d->a_stride < 0 || d->b_stride < 0)
    return norm_fail(LEWM_INVALID_ARG, "strides must be >= 0");
  if (d->group < 0 || (d->group > 0 && d->rows % d->group))
    return norm_fail(LEWM_INVALID_ARG, "rows %lld are not whole groups of %lld", (long long)d->rows,
                     (long long)d->group);
  *p = NormArgs{};
  p->rows = d->rows;
  p->width = (int)d->width;
  p->x_stride = d->x_stride;
  p->a_stride = d->group ? d->a_stride : 0;
  p->b_stride = d->group ? d->b_stride : 0;
  p->group = d->group ? d->group : std::max<int64_t>(d->rows, 1);
  p->one_plus = d->group > 0;
  p->p_type = d->p_type;
  p->eps = d->eps;
  return LEWM_OK;
}

struct NormDevice {
  int prev = -1;
  cudaError_t err = cudaSuccess;
  explicit NormDevice(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) err = cudaSetDevice(dev);
    else prev = -1;
  }
  ~NormDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

}  // namespace
}  // namespace lewm

using namespace lewm;

extern "C" size_t lewm_norm_workspace(const lewm_norm_desc* desc) {
  NormArgs p;
  if (norm_args(desc, &p) != LEWM_OK || p.rows == 0) return 0;
  cut_items(&p, true);
  return workspace_bytes(p);
}

extern "C" lewm_status lewm_norm_forward(const lewm_norm_desc* desc, const void* x, const void* a, const void* b,
                                         void* y, float* stats, int32_t device, void* stream) {
  NormArgs p;
  const lewm_status s = norm_args(desc, &p);
  if (s != LEWM_OK) return s;
  if (p.rows == 0) return LEWM_OK;
  if (!x || !y) return norm_fail(LEWM_INVALID_ARG, "x and y must be non-NULL");
  if (p.one_plus && (!a || !b)) return norm_fail(LEWM_INVALID_ARG, "scale and shift must be non-NULL");
  NormDevice nd(device);
  if (nd.err != cudaSuccess)
    return norm_fail(LEWM_CUDA_ERROR, "cudaSetDevice(%d): %s", device, cudaGetErrorString(nd.err));
  p.x = x;
  p.a = a;
  p.b = b;
  p.out = y;
  p.stats = stats;
  cut_items(&p, false);
  const cudaError_t e = launch_norm(p, desc->x_type, false, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return norm_fail(LEWM_CUDA_ERROR, "norm forward launch: %s", cudaGetErrorString(e));
  return LEWM_OK;
}

extern "C" lewm_status lewm_norm_backward(const lewm_norm_desc* desc, const void* dy, int64_t dy_stride,
                                          const void* x, const void* a, const float* stats, void* dx, void* da,
                                          void* db, void* workspace, size_t workspace_bytes_given, int32_t device,
                                          void* stream) {
  NormArgs p;
  const lewm_status s = norm_args(desc, &p);
  if (s != LEWM_OK) return s;
  if (!dx && !da && !db) return LEWM_OK;
  if (dy_stride < 0) return norm_fail(LEWM_INVALID_ARG, "dy_stride must be >= 0");
  if (p.rows == 0) {
    if ((da || db) && p.one_plus == 0)
      return norm_fail(LEWM_INVALID_ARG, "no rows: the gradients of weight and bias are zeros the caller sets");
    return LEWM_OK;
  }
  if (!dy || !x || !stats) return norm_fail(LEWM_INVALID_ARG, "dy, x and stats must be non-NULL");
  if (p.one_plus && !a) return norm_fail(LEWM_INVALID_ARG, "scale must be non-NULL");
  cut_items(&p, true);
  if ((da || db) && workspace_bytes_given < workspace_bytes(p))
    return norm_fail(LEWM_INVALID_ARG, "workspace of %zu bytes, needs %zu", workspace_bytes_given, workspace_bytes(p));
  if ((da || db) && p.split > 1 && !workspace) return norm_fail(LEWM_INVALID_ARG, "workspace must be non-NULL");
  NormDevice nd(device);
  if (nd.err != cudaSuccess)
    return norm_fail(LEWM_CUDA_ERROR, "cudaSetDevice(%d): %s", device, cudaGetErrorString(nd.err));
  p.x = x;
  p.dy = dy;
  p.dy_stride = dy_stride;
  p.a = a;
  p.out = dx;
  p.da = da;
  p.db = db;
  p.stats = const_cast<float*>(stats);
  p.ws = static_cast<float*>(workspace);
  const cudaError_t e = launch_norm(p, desc->x_type, true, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return norm_fail(LEWM_CUDA_ERROR, "norm backward launch: %s", cudaGetErrorString(e));
  return LEWM_OK;
}
