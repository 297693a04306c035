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
// thread: the backward then holds 16 gains and 32 sums, 128 registers at two 256-thread blocks
// per SM. Rows of more than 32 KB take the looping kernels below.
//
// Rows arrive through a ring of 2 to 4 stages in shared memory, filled by cp.async one to
// three rows ahead: registers alone kept 32 KB per SM on the way at best and none while a row
// was being reduced, half of HBM's rate (131072 x 2048 bf16: forward 307 us, backward 404).
// With 16-byte vectors each thread copies just what it reads itself, so the ring needs no
// barrier; rows at odd addresses are copied by 16-byte pieces with 4-byte ends and read back
// element by element after a team barrier.
//
// Work is cut into items: a run of rows within one group. An item is a block's (its teams
// interleave the rows and add up through shared memory), or a team's where there are many
// groups of few rows. A group cut into several items writes float32 partial sums, which
// k_norm_reduce adds in a fixed order: no atomics, the same bits on every run of the same
// shape. A modulation row per row of x (group 1) has nothing to sum over: there the modulation
// streams through the ring beside x (k_rowmod_*).
//
// Types: x, y, dy, dx are float32, bf16 or fp16; weights and modulation are float32 or any of
// these; all arithmetic, statistics and sums are float32, rounded once at the store.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "lewm_b200.h"
#include "lewm_common.cuh"
#include "lewm_internal.h"

namespace lewm {
namespace {

constexpr int kSms = 148;          // B200
constexpr int kMaxRowBytes = 32768;  // widest row held by a block: 1024 threads x 16 16-bit elements

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
  int stages;          // of the ring
  int p_vec;           // 1: E parameters load as vectors
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

// E elements of type P at `q` as float32; `vec`: aligned for accesses of min(16, E sizeof(P)) bytes.
template <typename P, int E>
__device__ __forceinline__ void load_as_float(const P* q, bool vec, float* f) {
  if (E > 1 && vec) {
    constexpr int N = E * (int)sizeof(P) > 16 ? 16 / (int)sizeof(P) : E;
#pragma unroll
    for (int k = 0; k < E / N; ++k) {
      const Vec<P, N> v = reinterpret_cast<const Vec<P, N>*>(q)[k];
#pragma unroll
      for (int e = 0; e < N; ++e) f[k * N + e] = to_f(v.v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = to_f(q[e]);
  }
}
template <typename P, int E>
__device__ __forceinline__ void store_from_float(P* q, bool vec, const float* f) {
  if (E > 1 && vec) {
    constexpr int N = E * (int)sizeof(P) > 16 ? 16 / (int)sizeof(P) : E;
#pragma unroll
    for (int k = 0; k < E / N; ++k) {
      Vec<P, N> v;
#pragma unroll
      for (int e = 0; e < N; ++e) v.v[e] = from_f<P>(f[k * N + e]);
      reinterpret_cast<Vec<P, N>*>(q)[k] = v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = from_f<P>(f[e]);
  }
}
// E parameters at element offset `at`, whatever their type.
template <int E>
__device__ __forceinline__ void load_params(const void* p, int type, int64_t at, bool vec, float* f) {
  if (type == LEWM_TYPE_F32) load_as_float<float, E>(static_cast<const float*>(p) + at, vec, f);
  else if (type == LEWM_TYPE_BF16) load_as_float<__nv_bfloat16, E>(static_cast<const __nv_bfloat16*>(p) + at, vec, f);
  else load_as_float<__half, E>(static_cast<const __half*>(p) + at, vec, f);
}
template <int E>
__device__ __forceinline__ void store_params(void* p, int type, int64_t at, bool vec, const float* f) {
  if (type == LEWM_TYPE_F32) store_from_float<float, E>(static_cast<float*>(p) + at, vec, f);
  else if (type == LEWM_TYPE_BF16) store_from_float<__nv_bfloat16, E>(static_cast<__nv_bfloat16*>(p) + at, vec, f);
  else store_from_float<__half, E>(static_cast<__half*>(p) + at, vec, f);
}

// ------------------------------------------------------------------ ring of rows
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Wait until at most stages - 2 groups of this thread are on their way.
__device__ __forceinline__ void cp_wait(int stages) {
  if (stages == 2) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (stages == 3) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 2;" ::: "memory");
}
template <int TPR>
__device__ __forceinline__ void team_barrier() {
  if constexpr (TPR > 32) __syncthreads();
  else __syncwarp();
}

constexpr int block_threads(int tpr) { return tpr < 256 ? 256 : tpr; }

// One stage of the ring for one tensor of element type P: a row of each team of the block.
//   E > 1: vector i of a thread lies at [piece][i][thread] in 16-byte (or 8-byte) pieces; only
//          that thread copies and reads it.
//   E = 1: a team's row lies in its slot at its address modulo 16; any thread copies any part.
template <typename P, int E, int NV, int TPR>
struct Stage {
  static constexpr int THREADS = block_threads(TPR), TEAMS = THREADS / TPR;
  static constexpr int VB = E * (int)sizeof(P);           // bytes of a vector
  [[maybe_unused]] static constexpr int PB = VB > 16 ? 16 : VB;  // of a piece
  static constexpr int SLOT = NV * TPR * (int)sizeof(P) + 32;  // E = 1
  static constexpr int BYTES = E > 1 ? NV * VB * THREADS : TEAMS * SLOT;

  // Starts the copy of a row. [lo, hi) is the whole tensor: a 4-byte end piece of a row of 16-bit
  // elements may take a neighbouring element along, but nothing outside the tensor.
  static __device__ __forceinline__ void fetch(char* buf, const P* row, int width, bool live, const P* lo,
                                               const P* hi) {
    const int team = threadIdx.x / TPR, lane = threadIdx.x % TPR;
    if (!live) return;
    if constexpr (E > 1) {
      const int nvec = width / E;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * TPR;
        if (v >= nvec) continue;
#pragma unroll
        for (int k = 0; k < VB / PB; ++k) {
          const uint32_t dst = smem_u32(buf + ((k * NV + i) * THREADS + threadIdx.x) * PB);
          const char* src = reinterpret_cast<const char*>(row + (int64_t)v * E) + k * PB;
          if constexpr (PB == 16) cp_async16(dst, src);
          else cp_async8(dst, src);
        }
      }
    } else {
      const uintptr_t s = reinterpret_cast<uintptr_t>(row), e = s + (uintptr_t)width * sizeof(P);
      char* slot = buf + team * SLOT;
      const uintptr_t origin = s & ~(uintptr_t)15;  // lies at slot[0]
      const uintptr_t a0 = (s + 15) & ~(uintptr_t)15, last = e & ~(uintptr_t)15, a1 = last > a0 ? last : a0;
      for (uintptr_t a = a0 + 16 * lane; a < a1; a += 16 * TPR)
        cp_async16(smem_u32(slot + (a - origin)), reinterpret_cast<const void*>(a));
      if (lane < 8) {  // up to four 4-byte words before a0 and after a1
        const uintptr_t w = lane < 4 ? (s & ~(uintptr_t)3) + 4 * lane : a1 + 4 * (lane - 4);
        if (w < (lane < 4 ? (a0 < e ? a0 : e) : e)) {
          if (w >= reinterpret_cast<uintptr_t>(lo) && w + 4 <= reinterpret_cast<uintptr_t>(hi)) {
            cp_async4(smem_u32(slot + (w - origin)), reinterpret_cast<const void*>(w));
          } else {
            for (uintptr_t q = w; q < w + 4; q += sizeof(P))
              if (q >= s && q < e) *reinterpret_cast<P*>(slot + (q - origin)) = *reinterpret_cast<const P*>(q);
          }
        }
      }
    }
  }

  // This thread's values of a row, 0 outside it.
  static __device__ __forceinline__ void read(const char* buf, const P* row, int width, bool live, float* f) {
    const int team = threadIdx.x / TPR, lane = threadIdx.x % TPR;
    if constexpr (E > 1) {
      const int nvec = width / E;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool in = live && lane + i * TPR < nvec;
#pragma unroll
        for (int k = 0; k < VB / PB; ++k) {
          constexpr int N = PB / (int)sizeof(P);
          if (in) {
            const Vec<P, N> v =
                *reinterpret_cast<const Vec<P, N>*>(buf + ((k * NV + i) * THREADS + threadIdx.x) * PB);
#pragma unroll
            for (int e = 0; e < N; ++e) f[i * E + k * N + e] = to_f(v.v[e]);
          } else {
#pragma unroll
            for (int e = 0; e < N; ++e) f[i * E + k * N + e] = 0.f;
          }
        }
      }
    } else {
      const P* q = reinterpret_cast<const P*>(buf + team * SLOT + (reinterpret_cast<uintptr_t>(row) & 15));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = lane + i * TPR;
        f[i] = live && c < width ? to_f(q[c]) : 0.f;
      }
    }
  }
};

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
  it.g = p.split == 1 ? item : item / p.split;
  const int64_t s = item - it.g * p.split;
  it.r0 = it.g * p.group + s * p.chunk;
  it.r1 = min(it.r0 + p.chunk, (it.g + 1) * p.group);
  return it;
}

// Blocks per SM that the registers are limited for: 80 a thread forward, 128 backward.
constexpr int blocks_per_sm(int tpr, bool backward) { return (backward ? 512 : 768) / block_threads(tpr); }
constexpr int bound_blocks(int tpr, bool backward) {
  return blocks_per_sm(tpr, backward) > 0 ? blocks_per_sm(tpr, backward) : 1;
}

// ------------------------------------------------------------------ forward
// mu and rs of a row from the team's values (0 outside the row), which become x - mu.
template <int N, int TPR>
__device__ __forceinline__ float2 row_stats(float* f, const bool* in, float inv_n, float eps, float (*red)[32]) {
  float s = 0.f, q = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) s += f[k];
  const float mu = team_sum<TPR>(s, red[0]) * inv_n;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    f[k] = in[k] ? f[k] - mu : 0.f;
    q = fmaf(f[k], f[k], q);
  }
  const float var = team_sum<TPR>(q, red[1]) * inv_n;
  return make_float2(mu, 1.0f / sqrtf(var + eps));
}

template <typename T, int E, int NV, int TPR>
__global__ void __launch_bounds__(block_threads(TPR), bound_blocks(TPR, false)) k_norm_fwd(const NormArgs p) {
  griddep_wait();  // launched as a programmatic dependent: wait for the kernel before
  using St = Stage<T, E, NV, TPR>;
  constexpr int TEAMS = St::TEAMS, N = NV * E;
  extern __shared__ __align__(16) char ring[];
  __shared__ float red[2][32];
  const int team = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  const int nvec = p.width / E;
  const float inv_n = 1.0f / p.width;
  const T* x = static_cast<const T*>(p.x);
  const T* x_end = x + (p.rows - 1) * p.x_stride + p.width;
  bool in[N];
#pragma unroll
  for (int k = 0; k < N; ++k) in[k] = lane + k / E * TPR < nvec;
  const int64_t step = p.team_items ? 1 : TEAMS;
  const int64_t iters = (p.chunk + step - 1) / step;
  const int64_t per_block = p.team_items ? TEAMS : 1;
  for (int64_t base = blockIdx.x * per_block; base < p.items; base += gridDim.x * per_block) {
    const Item it = item_rows(p, base + (p.team_items ? team : 0));
    const int64_t first = it.r0 + (p.team_items ? 0 : team);
    auto fetch = [&](int64_t k, int slot) {
      const int64_t r = first + k * step;
      St::fetch(ring + slot * St::BYTES, x + r * p.x_stride, p.width, k < iters && r < it.r1, x, x_end);
      cp_commit();
    };
    for (int k = 0; k < p.stages - 1; ++k) fetch(k, k);
    float ga[N], gb[N];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * TPR;
#pragma unroll
      for (int e = 0; e < E; ++e) ga[i * E + e] = 1.f, gb[i * E + e] = 0.f;
      if (v < nvec && it.r0 < it.r1) {
        if (p.a) load_params<E>(p.a, p.p_type, it.g * p.a_stride + (int64_t)v * E, p.p_vec, ga + i * E);
        if (p.b) load_params<E>(p.b, p.p_type, it.g * p.b_stride + (int64_t)v * E, p.p_vec, gb + i * E);
        if (p.one_plus) {
#pragma unroll
          for (int e = 0; e < E; ++e) ga[i * E + e] += 1.f;
        }
      }
    }
    int slot = 0;
    for (int64_t k = 0; k < iters; ++k) {
      const int64_t r = first + k * step;
      const bool live = r < it.r1;
      cp_wait(p.stages);
      if constexpr (E == 1) team_barrier<TPR>();
      fetch(k + p.stages - 1, slot == 0 ? p.stages - 1 : slot - 1);
      float f[N];
      St::read(ring + slot * St::BYTES, x + r * p.x_stride, p.width, live, f);
      if (++slot == p.stages) slot = 0;
      const float2 ms = row_stats<N, TPR>(f, in, inv_n, p.eps, red);
      if (!live) continue;
      if (p.stats && lane == 0) {
        p.stats[r] = ms.x;
        p.stats[p.rows + r] = ms.y;
      }
      T* y = static_cast<T*>(p.out) + r * p.width;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * TPR;
        if (v >= nvec) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) f[i * E + e] = fmaf(f[i * E + e] * ms.y, ga[i * E + e], gb[i * E + e]);
        store_from_float<T, E>(y + (int64_t)v * E, true, f + i * E);
      }
    }
    if constexpr (E == 1) team_barrier<TPR>();  // the ring is refilled for the next item
  }
}

// A modulation row per row of x: rows in a grid stride, scale and shift in the ring beside x.
template <typename T, typename P, int E, int NV, int TPR>
__global__ void __launch_bounds__(block_threads(TPR), bound_blocks(TPR, false)) k_rowmod_fwd(const NormArgs p) {
  griddep_wait();
  using St = Stage<T, E, NV, TPR>;
  using Sp = Stage<P, E, NV, TPR>;
  constexpr int TEAMS = St::TEAMS, N = NV * E, BYTES = St::BYTES + 2 * Sp::BYTES;
  extern __shared__ __align__(16) char ring[];
  __shared__ float red[2][32];
  const int team = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  const int nvec = p.width / E;
  const float inv_n = 1.0f / p.width;
  const T* x = static_cast<const T*>(p.x);
  const P* a = static_cast<const P*>(p.a);
  const P* b = static_cast<const P*>(p.b);
  const T* x_end = x + (p.rows - 1) * p.x_stride + p.width;
  const P* a_end = a + (p.rows - 1) * p.a_stride + p.width;
  const P* b_end = b + (p.rows - 1) * p.b_stride + p.width;
  bool in[N];
#pragma unroll
  for (int k = 0; k < N; ++k) in[k] = lane + k / E * TPR < nvec;
  const int64_t first = (int64_t)blockIdx.x * TEAMS + team, step = (int64_t)gridDim.x * TEAMS;
  const int64_t iters = (p.rows - (int64_t)blockIdx.x * TEAMS + step - 1) / step;
  auto fetch = [&](int64_t k, int slot) {
    const int64_t r = first + k * step;
    const bool live = r < p.rows;
    char* buf = ring + slot * BYTES;
    St::fetch(buf, x + r * p.x_stride, p.width, live, x, x_end);
    Sp::fetch(buf + St::BYTES, a + r * p.a_stride, p.width, live, a, a_end);
    Sp::fetch(buf + St::BYTES + Sp::BYTES, b + r * p.b_stride, p.width, live, b, b_end);
    cp_commit();
  };
  for (int k = 0; k < p.stages - 1; ++k) fetch(k, k);
  int slot = 0;
  for (int64_t k = 0; k < iters; ++k) {
    const int64_t r = first + k * step;
    const bool live = r < p.rows;
    cp_wait(p.stages);
    if constexpr (E == 1) team_barrier<TPR>();
    fetch(k + p.stages - 1, slot == 0 ? p.stages - 1 : slot - 1);
    const char* buf = ring + slot * BYTES;
    float f[N];
    St::read(buf, x + r * p.x_stride, p.width, live, f);
    const float2 ms = row_stats<N, TPR>(f, in, inv_n, p.eps, red);
    float ga[N], gb[N];
    Sp::read(buf + St::BYTES, a + r * p.a_stride, p.width, live, ga);
    Sp::read(buf + St::BYTES + Sp::BYTES, b + r * p.b_stride, p.width, live, gb);
    if (++slot == p.stages) slot = 0;
    if (!live) continue;
    if (p.stats && lane == 0) {
      p.stats[r] = ms.x;
      p.stats[p.rows + r] = ms.y;
    }
    T* y = static_cast<T*>(p.out) + r * p.width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * TPR;
      if (v >= nvec) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) f[i * E + e] = fmaf(f[i * E + e] * ms.y, 1.f + ga[i * E + e], gb[i * E + e]);
      store_from_float<T, E>(y + (int64_t)v * E, true, f + i * E);
    }
  }
}

// ------------------------------------------------------------------ backward
// Where the sums of E columns from `col` on of an item go. Partial sums are float4-aligned where
// E > 1 (the width is then a multiple of 4).
template <int E>
__device__ __forceinline__ void store_sums(const NormArgs& p, int64_t item, int64_t g, int64_t col, bool vec,
                                           const float* a, const float* b) {
  if (p.split > 1) {
    float* w = p.ws + item * 2 * p.width + col;
    store_from_float<float, E>(w, true, a);
    store_from_float<float, E>(w + p.width, true, b);
  } else {
    if (p.da) store_params<E>(p.da, p.p_type, g * p.width + col, vec, a);
    if (p.db) store_params<E>(p.db, p.p_type, g * p.width + col, vec, b);
  }
}

template <typename T, int E, int NV, int TPR>
__global__ void __launch_bounds__(block_threads(TPR), bound_blocks(TPR, true)) k_norm_bwd(const NormArgs p) {
  griddep_wait();  // launched as a programmatic dependent: wait for the kernel before
  using St = Stage<T, E, NV, TPR>;
  constexpr int THREADS = St::THREADS, TEAMS = St::TEAMS, N = NV * E, BYTES = 2 * St::BYTES;
  extern __shared__ __align__(16) char ring[];
  __shared__ float2 red[2][32];
  // The teams' sums of a slab of columns; the ring (two stages at least) is idle then.
  float2* sums = reinterpret_cast<float2*>(ring);
  static_assert(TEAMS == 1 || TEAMS * TPR * E * (int)sizeof(float2) <= 2 * BYTES, "sums fit the ring");
  const int team = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  const int nvec = p.width / E;
  const float inv_n = 1.0f / p.width;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  const T* x_end = x + (p.rows - 1) * p.x_stride + p.width;
  const T* dy_end = dy + (p.rows - 1) * p.dy_stride + p.width;
  const int64_t step = p.team_items ? 1 : TEAMS;
  const int64_t iters = (p.chunk + step - 1) / step;
  const int64_t per_block = p.team_items ? TEAMS : 1;
  int flip = 0;
  for (int64_t base = blockIdx.x * per_block; base < p.items; base += gridDim.x * per_block) {
    const int64_t item = base + (p.team_items ? team : 0);
    const Item it = item_rows(p, item);
    const int64_t first = it.r0 + (p.team_items ? 0 : team);
    auto fetch = [&](int64_t k, int slot) {
      const int64_t r = first + k * step;
      const bool live = k < iters && r < it.r1;
      char* buf = ring + slot * BYTES;
      St::fetch(buf, x + r * p.x_stride, p.width, live, x, x_end);
      St::fetch(buf + St::BYTES, dy + r * p.dy_stride, p.width, live, dy, dy_end);
      cp_commit();
    };
    for (int k = 0; k < p.stages - 1; ++k) fetch(k, k);
    float ga[N], sa[N], sb[N];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * TPR;
#pragma unroll
      for (int e = 0; e < E; ++e) ga[i * E + e] = 1.f, sa[i * E + e] = 0.f, sb[i * E + e] = 0.f;
      if (p.a && v < nvec && it.r0 < it.r1) {
        load_params<E>(p.a, p.p_type, it.g * p.a_stride + (int64_t)v * E, p.p_vec, ga + i * E);
        if (p.one_plus) {
#pragma unroll
          for (int e = 0; e < E; ++e) ga[i * E + e] += 1.f;
        }
      }
    }
    // Statistics of the first row; each row loads the next one's.
    float mu = 0.f, rs = 0.f;
    if (first < it.r1) mu = p.stats[first], rs = p.stats[p.rows + first];
    int slot = 0;
    for (int64_t k = 0; k < iters; ++k) {
      const int64_t r = first + k * step;
      const bool live = r < it.r1;
      cp_wait(p.stages);
      if constexpr (E == 1) team_barrier<TPR>();
      fetch(k + p.stages - 1, slot == 0 ? p.stages - 1 : slot - 1);
      float mu_next = 0.f, rs_next = 0.f;
      if (r + step < it.r1) mu_next = p.stats[r + step], rs_next = p.stats[p.rows + r + step];
      const char* buf = ring + slot * BYTES;
      if (++slot == p.stages) slot = 0;
      float z[N], g[N];
      St::read(buf, x + r * p.x_stride, p.width, live, z);
      St::read(buf + St::BYTES, dy + r * p.dy_stride, p.width, live, g);
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        // Values outside the row are 0 and leave every sum as it is, but for a row whose
        // statistics are not finite: 0 times infinity would reach the other columns' sums.
        if (!(live && lane + i * TPR < nvec)) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int c = i * E + e;
          z[c] = (z[c] - mu) * rs;
          sa[c] = fmaf(g[c], z[c], sa[c]);
          sb[c] += g[c];
          g[c] *= ga[c];
          s.x += g[c];
          s.y = fmaf(g[c], z[c], s.y);
        }
      }
      if (p.out) {
        s = team_sum2<TPR>(s, red[flip]);
        flip ^= 1;
        const float m1 = s.x * inv_n, m2 = s.y * inv_n;
        T* o = static_cast<T*>(p.out) + r * p.width;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int v = lane + i * TPR;
          if (!live || v >= nvec) continue;
#pragma unroll
          for (int e = 0; e < E; ++e) g[i * E + e] = rs * (g[i * E + e] - m1 - z[i * E + e] * m2);
          store_from_float<T, E>(o + (int64_t)v * E, true, g + i * E);
        }
      }
      mu = mu_next;
      rs = rs_next;
    }
    if constexpr (E == 1) team_barrier<TPR>();  // the ring is refilled for the next item
    if (!p.da && !p.db) continue;
    if (p.team_items || TEAMS == 1) {
      if (it.r0 >= it.r1) continue;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * TPR;
        if (v < nvec) store_sums<E>(p, item, it.g, (int64_t)v * E, p.p_vec, sa + i * E, sb + i * E);
      }
    } else {
      // Add the teams' sums in team order, a slab of TPR vectors of columns at a time.
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i * TPR >= nvec) break;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) sums[team * TPR * E + lane * E + e] = make_float2(sa[i * E + e], sb[i * E + e]);
        __syncthreads();
        for (int c = threadIdx.x; c < TPR * E; c += THREADS) {
          float a = 0.f, b = 0.f;
#pragma unroll
          for (int t = 0; t < TEAMS; ++t) a += sums[t * TPR * E + c].x, b += sums[t * TPR * E + c].y;
          const int64_t col = (int64_t)i * TPR * E + c;
          if (col < p.width) store_sums<1>(p, item, it.g, col, false, &a, &b);
        }
      }
      __syncthreads();
    }
  }
}

// A modulation row per row of x: d scale = dy z and d shift = dy row by row, nothing to sum up.
template <typename T, typename P, int E, int NV, int TPR>
__global__ void __launch_bounds__(block_threads(TPR), bound_blocks(TPR, false)) k_rowmod_bwd(const NormArgs p) {
  griddep_wait();
  using St = Stage<T, E, NV, TPR>;
  using Sp = Stage<P, E, NV, TPR>;
  constexpr int TEAMS = St::TEAMS, N = NV * E, BYTES = 2 * St::BYTES + Sp::BYTES;
  extern __shared__ __align__(16) char ring[];
  __shared__ float2 red[2][32];
  const int team = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  const int nvec = p.width / E;
  const float inv_n = 1.0f / p.width;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  const P* a = static_cast<const P*>(p.a);
  const T* x_end = x + (p.rows - 1) * p.x_stride + p.width;
  const T* dy_end = dy + (p.rows - 1) * p.dy_stride + p.width;
  const P* a_end = a + (p.rows - 1) * p.a_stride + p.width;
  const int64_t first = (int64_t)blockIdx.x * TEAMS + team, step = (int64_t)gridDim.x * TEAMS;
  const int64_t iters = (p.rows - (int64_t)blockIdx.x * TEAMS + step - 1) / step;
  int flip = 0;
  auto fetch = [&](int64_t k, int slot) {
    const int64_t r = first + k * step;
    const bool live = r < p.rows;
    char* buf = ring + slot * BYTES;
    St::fetch(buf, x + r * p.x_stride, p.width, live, x, x_end);
    St::fetch(buf + St::BYTES, dy + r * p.dy_stride, p.width, live, dy, dy_end);
    Sp::fetch(buf + 2 * St::BYTES, a + r * p.a_stride, p.width, live, a, a_end);
    cp_commit();
  };
  for (int k = 0; k < p.stages - 1; ++k) fetch(k, k);
  float mu = 0.f, rs = 0.f;
  if (first < p.rows) mu = p.stats[first], rs = p.stats[p.rows + first];
  int slot = 0;
  for (int64_t k = 0; k < iters; ++k) {
    const int64_t r = first + k * step;
    const bool live = r < p.rows;
    cp_wait(p.stages);
    if constexpr (E == 1) team_barrier<TPR>();
    fetch(k + p.stages - 1, slot == 0 ? p.stages - 1 : slot - 1);
    float mu_next = 0.f, rs_next = 0.f;
    if (r + step < p.rows) mu_next = p.stats[r + step], rs_next = p.stats[p.rows + r + step];
    const char* buf = ring + slot * BYTES;
    if (++slot == p.stages) slot = 0;
    float z[N], g[N], ga[N];
    St::read(buf, x + r * p.x_stride, p.width, live, z);
    St::read(buf + St::BYTES, dy + r * p.dy_stride, p.width, live, g);
    Sp::read(buf + 2 * St::BYTES, a + r * p.a_stride, p.width, live, ga);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * TPR;
      if (!live || v >= nvec) continue;
      if (p.db) store_from_float<P, E>(static_cast<P*>(p.db) + r * p.width + (int64_t)v * E, true, g + i * E);
      float dz[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = i * E + e;
        z[c] = (z[c] - mu) * rs;
        dz[e] = g[c] * z[c];
        g[c] *= 1.f + ga[c];
        s.x += g[c];
        s.y = fmaf(g[c], z[c], s.y);
      }
      if (p.da) store_from_float<P, E>(static_cast<P*>(p.da) + r * p.width + (int64_t)v * E, true, dz);
    }
    if (p.out) {
      s = team_sum2<TPR>(s, red[flip]);
      flip ^= 1;
      const float m1 = s.x * inv_n, m2 = s.y * inv_n;
      T* o = static_cast<T*>(p.out) + r * p.width;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * TPR;
        if (!live || v >= nvec) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) g[i * E + e] = rs * (g[i * E + e] - m1 - z[i * E + e] * m2);
        store_from_float<T, E>(o + (int64_t)v * E, true, g + i * E);
      }
    }
    mu = mu_next;
    rs = rs_next;
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
    if (threadIdx.x == 0 && c < p.width) store_params<1>(out, p.p_type, g * p.width + c, false, &t);
    __syncthreads();
  }
}

// ------------------------------------------------------------------ rows of more than kMaxRowBytes
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
      if (p.a) load_params<1>(p.a, p.p_type, g * p.a_stride + c, false, &a);
      if (p.b) load_params<1>(p.b, p.p_type, g * p.b_stride + c, false, &b);
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
      if (p.a) load_params<1>(p.a, p.p_type, g * p.a_stride + c, false, &a);
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
    float a = 0.f, b = 0.f;
    for (int64_t r = it.r0; r < it.r1; ++r) {
      const float g = to_f(static_cast<const T*>(p.dy)[r * p.dy_stride + col]);
      const float z = (to_f(static_cast<const T*>(p.x)[r * p.x_stride + col]) - p.stats[r]) * p.stats[p.rows + r];
      a = fmaf(g, z, a);
      b += g;
    }
    store_sums<1>(p, item, it.g, col, false, &a, &b);
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
  while (tpr * 16 < width) tpr *= 2;  // rows of at most kMaxRowBytes: tpr <= 1024
  return {tpr, block_threads(tpr) / tpr, 16};
}
int64_t type_size(int type) { return type == LEWM_TYPE_F32 ? 4 : 2; }
bool is_wide(const NormArgs& p, int x_type) { return p.width * type_size(x_type) > kMaxRowBytes; }

int64_t full_grid(int tpr, bool backward) { return (int64_t)kSms * bound_blocks(tpr, backward); }

// How rows are cut into items; the same function sizes the workspace.
void cut_items(NormArgs* p, int x_type, bool backward) {
  const int64_t groups = p->rows / p->group;
  if (is_wide(*p, x_type)) {
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
    const int64_t want = (full_grid(t.tpr, backward) + groups - 1) / groups;
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

// Stages of `bytes` each that fit `blocks` blocks per SM, 4 at most; 0 where not even two fit one
// block.
constexpr int kSmemPerSm = 227 * 1024, kSmemReserved = 2 * 1024;  // the latter: static and the system's, per block
int ring_stages(int bytes, int blocks) {
  for (; blocks >= 1; blocks = blocks / 2) {
    const int n = (kSmemPerSm / blocks - kSmemReserved) / bytes;
    if (n >= 3 || (blocks == 1 && n >= 2)) return std::min(n, 4);
  }
  return 0;
}

// Launches a kernel with a ring, raising its limit of dynamic shared memory (once per device).
template <typename K>
cudaError_t launch_ring(K kern, bool* raised, int64_t grid, int threads, int smem, const NormArgs& p,
                        cudaStream_t st) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !raised[dev]) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerSm - kSmemReserved);
    if (e != cudaSuccess) return e;
    if (dev < 64) raised[dev] = true;
  }
  return launch_k(kern, dim3((unsigned)grid), dim3(threads), smem, st, p);
}

template <typename T, int E, int NV, int TPR>
cudaError_t launch_items(NormArgs p, bool backward, cudaStream_t st) {
  using St = Stage<T, E, NV, TPR>;
  static bool raised[2][64];  // only ever set to true: calls from several threads may repeat the attribute
  const int bytes = (backward ? 2 : 1) * St::BYTES;
  p.stages = ring_stages(bytes, bound_blocks(TPR, backward));
  const int64_t blocks = p.team_items ? (p.items + St::TEAMS - 1) / St::TEAMS : p.items;
  const int64_t grid = std::min(blocks, full_grid(TPR, backward));
  return backward ? launch_ring(k_norm_bwd<T, E, NV, TPR>, raised[1], grid, St::THREADS, bytes * p.stages, p, st)
                  : launch_ring(k_norm_fwd<T, E, NV, TPR>, raised[0], grid, St::THREADS, bytes * p.stages, p, st);
}

// group 1: the modulation in the ring, if two stages of it fit.
template <typename T, typename P, int E, int NV, int TPR>
cudaError_t launch_rowmod(NormArgs p, bool backward, cudaStream_t st) {
  using St = Stage<T, E, NV, TPR>;
  using Sp = Stage<P, E, NV, TPR>;
  static bool raised[2][64];
  const int bytes = backward ? 2 * St::BYTES + Sp::BYTES : St::BYTES + 2 * Sp::BYTES;
  p.stages = ring_stages(bytes, bound_blocks(TPR, false));
  if (p.stages == 0) return launch_items<T, E, NV, TPR>(p, backward, st);
  const int64_t grid = std::min((p.rows + St::TEAMS - 1) / St::TEAMS, full_grid(TPR, false));
  return backward ? launch_ring(k_rowmod_bwd<T, P, E, NV, TPR>, raised[1], grid, St::THREADS, bytes * p.stages, p, st)
                  : launch_ring(k_rowmod_fwd<T, P, E, NV, TPR>, raised[0], grid, St::THREADS, bytes * p.stages, p, st);
}

template <typename T, int E, int NV, int TPR>
cudaError_t launch_tier(const NormArgs& p, bool backward, cudaStream_t st) {
  if (p.group > 1 || !p.one_plus) return launch_items<T, E, NV, TPR>(p, backward, st);
  if (p.p_type == LEWM_TYPE_F32) return launch_rowmod<T, float, E, NV, TPR>(p, backward, st);
  constexpr bool any = std::is_same<T, float>::value;
  if constexpr (any || std::is_same<T, __nv_bfloat16>::value)
    if (p.p_type == LEWM_TYPE_BF16) return launch_rowmod<T, __nv_bfloat16, E, NV, TPR>(p, backward, st);
  if constexpr (any || std::is_same<T, __half>::value)
    if (p.p_type == LEWM_TYPE_F16) return launch_rowmod<T, __half, E, NV, TPR>(p, backward, st);
  return launch_items<T, E, NV, TPR>(p, backward, st);  // bf16 beside fp16
}

template <typename T, int E>
cudaError_t launch_width(const NormArgs& p, bool backward, cudaStream_t st) {
  constexpr int E8 = E, V8 = 8 / E, V16 = 16 / E;
  switch (tier_of(p.width).tpr) {
    case 8: return launch_tier<T, E8, V8, 8>(p, backward, st);
    case 32:
      return p.width <= 256 ? launch_tier<T, E8, V8, 32>(p, backward, st) : launch_tier<T, E8, V16, 32>(p, backward, st);
    case 64: return launch_tier<T, E, V16, 64>(p, backward, st);
    case 128: return launch_tier<T, E, V16, 128>(p, backward, st);
    case 256: return launch_tier<T, E, V16, 256>(p, backward, st);
    case 512: return launch_tier<T, E, V16, 512>(p, backward, st);
    default:
      if constexpr (sizeof(T) == 2) return launch_tier<T, E, V16, 1024>(p, backward, st);
      return cudaErrorInvalidValue;  // float32 rows this wide are more than kMaxRowBytes
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
cudaError_t launch_type(const NormArgs& p, bool wide, bool backward, bool vec, cudaStream_t st) {
  if (wide) return launch_wide<T>(p, backward, st);
  return vec ? launch_width<T, 16 / sizeof(T)>(p, backward, st) : launch_width<T, 1>(p, backward, st);
}

cudaError_t launch_norm(NormArgs p, int x_type, bool backward, cudaStream_t st) {
  const int64_t size = type_size(x_type), vec_elems = 16 / size;
  auto aligned = [](const void* q, int64_t stride_bytes, int64_t to) {
    return !q || ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)stride_bytes) & (uintptr_t)(to - 1)) == 0;
  };
  bool vec = aligned(p.x, p.x_stride * size, 16) && aligned(p.out, p.width * size, 16) &&
             (!backward || aligned(p.dy, p.dy_stride * size, 16)) && (p.width * size) % 16 == 0;
  // A vector's parameters as 16-byte (8-byte: 16-bit ones beside float32 rows) accesses.
  const int64_t ps = type_size(p.p_type), to = std::min<int64_t>(16, vec_elems * ps);
  p.p_vec = aligned(p.a, p.a_stride * ps, to) && aligned(p.b, p.b_stride * ps, to) &&
            aligned(p.da, p.width * ps, to) && aligned(p.db, p.width * ps, to) && (p.width * ps) % to == 0;
  if (p.one_plus && p.group == 1) vec = vec && p.p_vec;  // the ring moves both the same way
  const bool wide = is_wide(p, x_type);
  cudaError_t e = x_type == LEWM_TYPE_F32    ? launch_type<float>(p, wide, backward, vec, st)
                  : x_type == LEWM_TYPE_BF16 ? launch_type<__nv_bfloat16>(p, wide, backward, vec, st)
                                             : launch_type<__half>(p, wide, backward, vec, st);
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
  cut_items(&p, desc->x_type, true);
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
  cut_items(&p, desc->x_type, false);
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
  cut_items(&p, desc->x_type, true);
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
