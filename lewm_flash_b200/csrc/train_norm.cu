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
// Arithmetic on packed pairs of float32 (add, mul and fma .f32x2): 16-bit rows are bound by
// instructions otherwise (131072 x 2048 bf16: forward 220 us, backward 317).
//
// Types: x, y, dy, dx are float32, bf16 or fp16; weights and modulation are float32 or any of
// these; all arithmetic, statistics and sums are float32, rounded once at the store.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "lewm_b200.h"
#include "lewm_common.cuh"
#include "lewm_internal.h"
#include "train_elem.cuh"

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
  int split;           // items per group
  int loop_min, loop_rem;  // a loop that starts `o` rows into its rows has loop_min + (o < loop_rem) rounds
  int width;
  int p_type;
  int one_plus;        // a = 1 + a[]
  int team_items;      // 1: an item per team, 0: per block
  int stages;          // of the ring
  int p_vec;           // 1: E parameters load as vectors
  float eps;
};

// ------------------------------------------------------------------ parameters
// E elements of type P at `q` as pairs (E > 1), in accesses of min(16, E sizeof(P)) bytes if the
// address allows it (`vec`).
template <typename P, int E>
__device__ __forceinline__ void load_pairs(const P* q, bool vec, F2* f) {
  constexpr int N = E * (int)sizeof(P) > 16 ? 16 / (int)sizeof(P) : E;
#pragma unroll
  for (int k = 0; k < E / N; ++k) {
    Vec<P, N> v;
    if (vec) {
      v = reinterpret_cast<const Vec<P, N>*>(q)[k];
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v.v[e] = q[k * N + e];
    }
#pragma unroll
    for (int e = 0; e < N; e += 2) f[(k * N + e) / 2] = unpack(v.v + e);
  }
}
template <typename P, int E>
__device__ __forceinline__ void store_pairs(P* q, bool vec, const F2* f) {
  constexpr int N = E * (int)sizeof(P) > 16 ? 16 / (int)sizeof(P) : E;
#pragma unroll
  for (int k = 0; k < E / N; ++k) {
    Vec<P, N> v;
#pragma unroll
    for (int e = 0; e < N; e += 2) pack(v.v + e, f[(k * N + e) / 2]);
    if (vec) {
      reinterpret_cast<Vec<P, N>*>(q)[k] = v;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) q[k * N + e] = v.v[e];
    }
  }
}
// One parameter, whatever the type.
__device__ __forceinline__ float load_param(const void* p, int type, int64_t at) {
  if (type == LEWM_TYPE_F32) return static_cast<const float*>(p)[at];
  if (type == LEWM_TYPE_BF16) return to_f(static_cast<const __nv_bfloat16*>(p)[at]);
  return to_f(static_cast<const __half*>(p)[at]);
}
__device__ __forceinline__ void store_param(void* p, int type, int64_t at, float f) {
  if (type == LEWM_TYPE_F32) static_cast<float*>(p)[at] = f;
  else if (type == LEWM_TYPE_BF16) static_cast<__nv_bfloat16*>(p)[at] = from_f<__nv_bfloat16>(f);
  else static_cast<__half*>(p)[at] = from_f<__half>(f);
}

// ------------------------------------------------------------------ teams
constexpr int block_threads(int tpr) { return tpr < 256 ? 256 : tpr; }

// What a thread holds of a row. N values as N / 2 pairs: vector i of the team's vectors lane +
// i TPR, whose E values are pairs i E / 2 on (E > 1); or single values lane + i TPR, two of
// consecutive i in a pair (E = 1).
template <int E_, int NV_, int TPR_>
struct Team {
  static constexpr int E = E_, NV = NV_, TPR = TPR_, N = E * NV, H = N / 2;
  static constexpr int THREADS = block_threads(TPR), TEAMS = THREADS / TPR;
  // Vectors that lie inside every row of the tier: its narrowest row fills more than half of a
  // team (a quarter in the tier of 65 to 256).
  static constexpr int SURE = TPR == 8 ? 0 : N == 8 ? NV / 4 : NV / 2;

  static __device__ __forceinline__ int team() { return threadIdx.x / TPR; }
  static __device__ __forceinline__ int lane() { return threadIdx.x % TPR; }
  // Barrier of the threads that share a row.
  static __device__ __forceinline__ void barrier() {
    if constexpr (TPR > 32) named_bar(1 + team(), TPR);
    else __syncwarp();
  }
  // Sum over the team, the same bits in all of its threads. Teams of more than a warp add their
  // warps' sums through `red` (a slot per warp of the block) in warp order; the caller alternates
  // between two `red` buffers, so that one is rewritten only after a later barrier.
  static __device__ __forceinline__ float sum(float v, float* red) {
    constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (TPR > 32) {
      const int warp = threadIdx.x >> 5, w0 = team() * (TPR / 32);
      if ((threadIdx.x & 31) == 0) red[warp] = v;
      barrier();
      v = 0.f;
#pragma unroll
      for (int i = 0; i < TPR / 32; ++i) v += red[w0 + i];
    }
    return v;
  }
  static __device__ __forceinline__ float2 sum2(float2 v, float2* red) {
    constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if constexpr (TPR > 32) {
      const int warp = threadIdx.x >> 5, w0 = team() * (TPR / 32);
      if ((threadIdx.x & 31) == 0) red[warp] = v;
      barrier();
      v = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < TPR / 32; ++i) {
        v.x += red[w0 + i].x;
        v.y += red[w0 + i].y;
      }
    }
    return v;
  }

  // This thread's parameters of a row of `width` at element offset `at`, `outside` beyond it.
  static __device__ __forceinline__ void load_params(const void* p, int type, int64_t at, int width, bool vec, F2* f) {
    if constexpr (E > 1) {
      const int nvec = width / E;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane() + i * TPR;
        if (v >= nvec) continue;
        F2* o = f + i * (E / 2);
        const int64_t c = at + (int64_t)v * E;
        if (type == LEWM_TYPE_F32) load_pairs<float, E>(static_cast<const float*>(p) + c, vec, o);
        else if (type == LEWM_TYPE_BF16) load_pairs<__nv_bfloat16, E>(static_cast<const __nv_bfloat16*>(p) + c, vec, o);
        else load_pairs<__half, E>(static_cast<const __half*>(p) + c, vec, o);
      }
    } else {
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const int c = lane() + 2 * i * TPR;
        float2 v = split(f[i]);
        if (c < width) v.x = load_param(p, type, at + c);
        if (c + TPR < width) v.y = load_param(p, type, at + c + TPR);
        f[i] = f2(v.x, v.y);
      }
    }
  }
  // Stores a row of `width` values of type P at `row`.
  template <typename P>
  static __device__ __forceinline__ void store_row(P* row, int width, const F2* f) {
    if constexpr (E > 1) {
      const int nvec = width / E;
      P* q = row + lane() * E;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i < SURE || lane() + i * TPR < nvec) store_pairs<P, E>(q + i * TPR * E, true, f + i * (E / 2));
    } else {
      P* q = row + lane();
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float2 v = split(f[i]);
        if (2 * i < SURE || lane() + 2 * i * TPR < width) q[2 * i * TPR] = from_f<P>(v.x);
        if (2 * i + 1 < SURE || lane() + (2 * i + 1) * TPR < width) q[(2 * i + 1) * TPR] = from_f<P>(v.y);
      }
    }
  }
  static __device__ __forceinline__ void store_params(void* p, int type, int64_t at, int width, bool vec,
                                                      const F2* f) {
    if constexpr (E > 1) {
      const int nvec = width / E;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane() + i * TPR;
        if (v >= nvec) continue;
        const F2* o = f + i * (E / 2);
        const int64_t c = at + (int64_t)v * E;
        if (type == LEWM_TYPE_F32) store_pairs<float, E>(static_cast<float*>(p) + c, vec, o);
        else if (type == LEWM_TYPE_BF16) store_pairs<__nv_bfloat16, E>(static_cast<__nv_bfloat16*>(p) + c, vec, o);
        else store_pairs<__half, E>(static_cast<__half*>(p) + c, vec, o);
      }
    } else {
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const int c = lane() + 2 * i * TPR;
        const float2 v = split(f[i]);
        if (c < width) store_param(p, type, at + c, v.x);
        if (c + TPR < width) store_param(p, type, at + c + TPR, v.y);
      }
    }
  }
};

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

// One stage of the ring for one tensor of element type P: a row of each team of the block.
//   E > 1: vector i of a thread lies at [piece][i][thread] in 16-byte (or 8-byte) pieces; only
//          that thread copies and reads it.
//   E = 1: a team's row lies in its slot at its address modulo 16; any thread copies any part.
template <typename P, typename Tm>
struct Stage {
  static constexpr int E = Tm::E, NV = Tm::NV, TPR = Tm::TPR, THREADS = Tm::THREADS;
  static constexpr int VB = E * (int)sizeof(P);                  // bytes of a vector
  [[maybe_unused]] static constexpr int PB = VB > 16 ? 16 : VB;  // of a piece
  [[maybe_unused]] static constexpr int SLOT = NV * TPR * (int)sizeof(P) + 32;  // E = 1
  static constexpr int BYTES = E > 1 ? NV * VB * THREADS : Tm::TEAMS * SLOT;

  // Starts the copy of a row to the stage at `buf`. [lo, hi) is the whole tensor: a 4-byte end
  // piece of a row of 16-bit elements may take a neighbouring element along, but nothing outside
  // the tensor.
  static __device__ __forceinline__ void fetch(uint32_t buf, const P* row, int width, const P* lo, const P* hi) {
    const int lane = Tm::lane();
    if constexpr (E > 1) {
      const int nvec = width / E;
      const char* src = reinterpret_cast<const char*>(row) + lane * VB;
      const uint32_t dst = buf + threadIdx.x * PB;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i < Tm::SURE || lane + i * TPR < nvec) {
#pragma unroll
          for (int k = 0; k < VB / PB; ++k) {
            if constexpr (PB == 16) cp_async16(dst + (k * NV + i) * THREADS * PB, src + i * TPR * VB + k * PB);
            else cp_async8(dst + (k * NV + i) * THREADS * PB, src + i * TPR * VB + k * PB);
          }
        }
      }
    } else {
      // Byte offsets from the row's start, which lies `mis` bytes behind the slot's: 16-byte pieces
      // [a0, a1), up to four 4-byte words before and after them.
      const int mis = (int)(reinterpret_cast<uintptr_t>(row) & 15), bytes = width * (int)sizeof(P);
      const int a0 = (16 - mis) & 15, a1 = max(a0, ((mis + bytes) & ~15) - mis);
      const uint32_t slot = buf + Tm::team() * SLOT + mis;
      const char* src = reinterpret_cast<const char*>(row);
      constexpr int PIECES = (NV * (int)sizeof(P) + 15) / 16;  // of a thread at most
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        const int a = a0 + 16 * (lane + k * TPR);
        if (a < a1) cp_async16(slot + a, src + a);
      }
      if (lane < 8) {
        const int w = lane < 4 ? -(mis & 3) + 4 * lane : a1 + 4 * (lane - 4);
        if (w < (lane < 4 ? min(a0, bytes) : bytes)) {
          if (src + w >= reinterpret_cast<const char*>(lo) && src + w + 4 <= reinterpret_cast<const char*>(hi)) {
            cp_async4(slot + w, src + w);
          } else {
            for (int q = w; q < w + 4; q += (int)sizeof(P))
              if (q >= 0 && q < bytes)
                *reinterpret_cast<P*>(__cvta_shared_to_generic(slot + q)) = *reinterpret_cast<const P*>(src + q);
          }
        }
      }
    }
  }

  // This thread's values of a row, 0 beyond it. `row` gives the address modulo 16.
  static __device__ __forceinline__ void read(const char* buf, const P* row, int width, F2* f) {
    const int lane = Tm::lane();
    if constexpr (E > 1) {
      const int nvec = width / E;
      constexpr int K = PB / (int)sizeof(P);
      const char* src = buf + threadIdx.x * PB;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int k = 0; k < VB / PB; ++k) {
          F2* o = f + (i * E + k * K) / 2;
          if (i < Tm::SURE || lane + i * TPR < nvec) {
            const Vec<P, K> v = *reinterpret_cast<const Vec<P, K>*>(src + (k * NV + i) * THREADS * PB);
#pragma unroll
            for (int e = 0; e < K; e += 2) o[e / 2] = unpack(v.v + e);
          } else {
#pragma unroll
            for (int e = 0; e < K; e += 2) o[e / 2] = f2(0.f);
          }
        }
      }
    } else {
      const P* q = reinterpret_cast<const P*>(buf + Tm::team() * SLOT + (reinterpret_cast<uintptr_t>(row) & 15)) + lane;
#pragma unroll
      for (int i = 0; i < Tm::H; ++i) {
        const float x = 2 * i < Tm::SURE || lane + 2 * i * TPR < width ? to_f(q[2 * i * TPR]) : 0.f;
        const float y = 2 * i + 1 < Tm::SURE || lane + (2 * i + 1) * TPR < width ? to_f(q[(2 * i + 1) * TPR]) : 0.f;
        f[i] = f2(x, y);
      }
    }
  }
};

// Rows of an item for one team: first, first + step, ... below end, in group g. The items of a
// group take its rows in turn, a block's worth at a time, so that the blocks sweep x in one
// front: with a contiguous run of rows for each block DRAM gave less (73881 x 1536 float32
// backward: 4.3 against 6.4 TB/s).
struct Item {
  int64_t g, first, step;
  int rows, iters;  // of this team; of the whole block's loop
};
template <int TEAMS>
__device__ __forceinline__ Item item_rows(const NormArgs& p, int64_t base, int team) {
  Item it{0, 0, 1, 0, p.loop_min};
  if (p.team_items) {
    it.g = base + team;
    it.rows = it.g < p.items ? p.loop_min : 0;
    it.first = it.g * p.group;
  } else {
    int s = 0;
    if (p.split == p.items) s = (int)base;  // one group
    else if (p.split == 1) it.g = base;
    else if (p.items <= UINT_MAX) {
      it.g = (uint32_t)base / (uint32_t)p.split;
      s = (int)((uint32_t)base - (uint32_t)it.g * (uint32_t)p.split);
    } else {
      it.g = base / p.split;
      s = (int)(base - it.g * p.split);
    }
    const int64_t o = (int64_t)s * TEAMS;
    it.step = (int64_t)p.split * TEAMS;
    it.first = it.g * p.group + o + team;
    it.iters = p.loop_min + (o < p.loop_rem);
    it.rows = p.loop_min + (o + team < p.loop_rem);
  }
  return it;
}

// A tensor's rows from the loop's first one on, advanced by pointer.
template <typename P>
struct Walk {
  const P *at, *lo, *hi;
  int64_t step;
  __device__ __forceinline__ Walk(const void* base, int64_t rows, int64_t stride, int width, int64_t first,
                                  int64_t step_rows)
      : at(static_cast<const P*>(base) + first * stride),
        lo(static_cast<const P*>(base)),
        hi(static_cast<const P*>(base) + (rows - 1) * stride + width),
        step(step_rows * stride) {}
};

// Blocks per SM that the registers are limited for: 80 a thread forward (128 with 32 values), 128 in
// the backward that keeps sums. More, smaller blocks were slower on short rows (16448 x 192 bf16 forward, 3, 4 and 5
// blocks: 6.8, 6.9, 7.2 us): every block loads the parameters anew. The backward of a modulation
// row per row has neither and takes 4 there (57600 x 192 bf16, 2, 3 and 4 blocks: 26.2, 22.9,
// 21.6 us).
template <typename Tm>
constexpr int bound_blocks(bool backward, bool rowmod = false) {
  if (rowmod && backward && Tm::N == 8) return 4;
  const int n = (backward || Tm::N == 32 ? 512 : 768) / Tm::THREADS;
  return n > 0 ? n : 1;
}

// What multiplies z in group g, and what is added: weight or 1 + scale, bias or shift.
template <typename Tm>
__device__ __forceinline__ void load_gain(const NormArgs& p, int64_t g, F2* a) {
#pragma unroll
  for (int k = 0; k < Tm::H; ++k) a[k] = f2(p.one_plus ? 0.f : 1.f);
  if (p.a) Tm::load_params(p.a, p.p_type, g * p.a_stride, p.width, p.p_vec, a);
  if (p.one_plus) {
#pragma unroll
    for (int k = 0; k < Tm::H; ++k) a[k] = a[k] + f2(1.f);
  }
}
template <typename Tm>
__device__ __forceinline__ void load_offset(const NormArgs& p, int64_t g, F2* b) {
#pragma unroll
  for (int k = 0; k < Tm::H; ++k) b[k] = f2(0.f);
  if (p.b) Tm::load_params(p.b, p.p_type, g * p.b_stride, p.width, p.p_vec, b);
}

// ------------------------------------------------------------------ forward
// x - mu in place of the team's values x (0 beyond the row), mu and rs.
template <typename Tm>
__device__ __forceinline__ float2 row_stats(F2* f, int width, float inv_n, float eps, float (*red)[32]) {
  constexpr int E = Tm::E, TPR = Tm::TPR;
  F2 s = f2(0.f), q = f2(0.f);
#pragma unroll
  for (int k = 0; k < Tm::H; ++k) s = s + f[k];
  const float mu = Tm::sum(both(s), red[0]) * inv_n;
  const F2 nm = f2(-mu);
#pragma unroll
  for (int k = 0; k < Tm::H; ++k) {
    f[k] = f[k] + nm;
    if constexpr (E > 1) {
      const int i = k / (E / 2);
      if (i < Tm::SURE || Tm::lane() + i * TPR < width / E) q = fma2(f[k], f[k], q);
    } else {
      const int i = 2 * k;
      if (i + 1 < Tm::SURE) {
        q = fma2(f[k], f[k], q);
      } else {
        const float2 v = split(f[k]);
        const F2 c = f2(Tm::lane() + i * TPR < width ? v.x : 0.f, Tm::lane() + (i + 1) * TPR < width ? v.y : 0.f);
        q = fma2(c, c, q);
      }
    }
  }
  const float var = Tm::sum(both(q), red[1]) * inv_n;
  return make_float2(mu, 1.0f / sqrtf(var + eps));
}

template <typename T, typename Tm>
__global__ void __launch_bounds__(Tm::THREADS, bound_blocks<Tm>(false)) k_norm_fwd(const NormArgs p) {
  griddep_wait();  // launched as a programmatic dependent: wait for the kernel before
  using St = Stage<T, Tm>;
  constexpr int H = Tm::H;
  extern __shared__ __align__(16) char ring[];
  __shared__ float red[2][32];
  const float inv_n = 1.0f / p.width;
  const uint32_t ring0 = smem_u32(ring), ring_end = ring0 + p.stages * St::BYTES;
  const int64_t per_block = p.team_items ? Tm::TEAMS : 1;
  for (int64_t base = blockIdx.x * per_block; base < p.items; base += gridDim.x * per_block) {
    const Item it = item_rows<Tm::TEAMS>(p, base, Tm::team());
    Walk<T> x(p.x, p.rows, p.x_stride, p.width, it.first, it.step);
    const T* x_now = x.at;  // the row being computed; x.at is the one being fetched
    int left = it.rows, ahead = left;
    uint32_t in = ring0, out = ring0;
    auto fetch = [&]() {
      if (ahead > 0) St::fetch(in, x.at, p.width, x.lo, x.hi);
      --ahead;
      x.at += x.step;
      in = in + St::BYTES == ring_end ? ring0 : in + St::BYTES;
      cp_commit();
    };
    for (int k = 0; k < p.stages - 1; ++k) fetch();
    F2 ga[H], gb[H];
    if (left > 0) {
      load_gain<Tm>(p, it.g, ga);
      load_offset<Tm>(p, it.g, gb);
    }
    int64_t r = it.first;
    T* y = static_cast<T*>(p.out) + r * p.width;
    for (int k = 0; k < it.iters; ++k) {
      cp_wait(p.stages);
      if constexpr (Tm::E == 1) Tm::barrier();
      fetch();
      F2 f[H];
      if (left > 0) {
        St::read(ring + (out - ring0), x_now, p.width, f);
      } else {
#pragma unroll
        for (int h = 0; h < H; ++h) f[h] = f2(0.f);
      }
      out = out + St::BYTES == ring_end ? ring0 : out + St::BYTES;
      const float2 ms = row_stats<Tm>(f, p.width, inv_n, p.eps, red);
      if (left > 0) {
        if (p.stats && Tm::lane() == 0) {
          p.stats[r] = ms.x;
          p.stats[p.rows + r] = ms.y;
        }
        const F2 rs = f2(ms.y);
#pragma unroll
        for (int h = 0; h < H; ++h) f[h] = fma2(f[h] * rs, ga[h], gb[h]);
        Tm::store_row(y, p.width, f);
      }
      --left;
      r += it.step;
      y += it.step * p.width;
      x_now += x.step;
    }
    if constexpr (Tm::E == 1) Tm::barrier();  // the ring is refilled for the next item
  }
}

// A modulation row per row of x: rows in a grid stride, scale and shift in the ring beside x.
template <typename T, typename P, typename Tm>
__global__ void __launch_bounds__(Tm::THREADS, bound_blocks<Tm>(false)) k_rowmod_fwd(const NormArgs p) {
  griddep_wait();
  using St = Stage<T, Tm>;
  using Sp = Stage<P, Tm>;
  constexpr int H = Tm::H, BYTES = St::BYTES + 2 * Sp::BYTES;
  extern __shared__ __align__(16) char ring[];
  __shared__ float red[2][32];
  const float inv_n = 1.0f / p.width;
  const uint32_t ring0 = smem_u32(ring), ring_end = ring0 + p.stages * BYTES;
  const int64_t first = (int64_t)blockIdx.x * Tm::TEAMS + Tm::team(), step = (int64_t)gridDim.x * Tm::TEAMS;
  const int iters = p.loop_min + ((int64_t)blockIdx.x * Tm::TEAMS < p.loop_rem);
  Walk<T> x(p.x, p.rows, p.x_stride, p.width, first, step);
  Walk<P> a(p.a, p.rows, p.a_stride, p.width, first, step), b(p.b, p.rows, p.b_stride, p.width, first, step);
  const T* x_now = x.at;
  const P *a_now = a.at, *b_now = b.at;
  int left = p.loop_min + (first < p.loop_rem), ahead = left;
  uint32_t in = ring0, out = ring0;
  auto fetch = [&]() {
    if (ahead > 0) {
      St::fetch(in, x.at, p.width, x.lo, x.hi);
      Sp::fetch(in + St::BYTES, a.at, p.width, a.lo, a.hi);
      Sp::fetch(in + St::BYTES + Sp::BYTES, b.at, p.width, b.lo, b.hi);
    }
    --ahead;
    x.at += x.step, a.at += a.step, b.at += b.step;
    in = in + BYTES == ring_end ? ring0 : in + BYTES;
    cp_commit();
  };
  for (int k = 0; k < p.stages - 1; ++k) fetch();
  int64_t r = first;
  T* y = static_cast<T*>(p.out) + r * p.width;
  for (int k = 0; k < iters; ++k) {
    cp_wait(p.stages);
    if constexpr (Tm::E == 1) Tm::barrier();
    fetch();
    const char* buf = ring + (out - ring0);
    out = out + BYTES == ring_end ? ring0 : out + BYTES;
    F2 f[H];
    if (left > 0) {
      St::read(buf, x_now, p.width, f);
    } else {
#pragma unroll
      for (int h = 0; h < H; ++h) f[h] = f2(0.f);
    }
    const float2 ms = row_stats<Tm>(f, p.width, inv_n, p.eps, red);
    if (left > 0) {
      if (p.stats && Tm::lane() == 0) {
        p.stats[r] = ms.x;
        p.stats[p.rows + r] = ms.y;
      }
      F2 ga[H], gb[H];
      Sp::read(buf + St::BYTES, a_now, p.width, ga);
      Sp::read(buf + St::BYTES + Sp::BYTES, b_now, p.width, gb);
      const F2 rs = f2(ms.y), one = f2(1.f);
#pragma unroll
      for (int h = 0; h < H; ++h) f[h] = fma2(f[h] * rs, ga[h] + one, gb[h]);
      Tm::store_row(y, p.width, f);
    }
    --left;
    r += step;
    y += step * p.width;
    x_now += x.step, a_now += a.step, b_now += b.step;
  }
}

// ------------------------------------------------------------------ backward
// dx of a row from z, d and the row's sums.
template <typename T, typename Tm>
__device__ __forceinline__ void store_dx(T* dx, int width, const F2* z, F2* d, float2 s, float inv_n, float rs) {
  const F2 m1 = f2(-s.x * inv_n), m2 = f2(-s.y * inv_n), r = f2(rs);
#pragma unroll
  for (int h = 0; h < Tm::H; ++h) d[h] = fma2(z[h], m2, d[h] + m1) * r;
  Tm::store_row(dx, width, d);
}

template <typename T, typename Tm>
__global__ void __launch_bounds__(Tm::THREADS, bound_blocks<Tm>(true)) k_norm_bwd(const NormArgs p) {
  griddep_wait();  // launched as a programmatic dependent: wait for the kernel before
  // The whole grid is resident by now, so the reduction's blocks take no slot from it; they
  // wait for its end with their launch behind them.
  if (p.split > 1) griddep_launch();
  using St = Stage<T, Tm>;
  constexpr int THREADS = Tm::THREADS, TEAMS = Tm::TEAMS, TPR = Tm::TPR, E = Tm::E, H = Tm::H, BYTES = 2 * St::BYTES;
  extern __shared__ __align__(16) char ring[];
  __shared__ float2 red[2][32];
  // The teams' sums of a slab of columns; the ring (two stages at least) is idle then.
  float2* sums = reinterpret_cast<float2*>(ring);
  constexpr int SLAB = TPR * (E > 1 ? E : 2);  // columns added up at a time
  static_assert(TEAMS == 1 || TEAMS * SLAB * (int)sizeof(float2) <= 2 * BYTES, "sums fit the ring");
  const float inv_n = 1.0f / p.width;
  const uint32_t ring0 = smem_u32(ring), ring_end = ring0 + p.stages * BYTES;
  const int64_t per_block = p.team_items ? TEAMS : 1;
  int flip = 0;
  for (int64_t base = blockIdx.x * per_block; base < p.items; base += gridDim.x * per_block) {
    const Item it = item_rows<TEAMS>(p, base, Tm::team());
    Walk<T> x(p.x, p.rows, p.x_stride, p.width, it.first, it.step);
    Walk<T> dy(p.dy, p.rows, p.dy_stride, p.width, it.first, it.step);
    const T *x_now = x.at, *dy_now = dy.at;
    int left = it.rows, ahead = left;
    const bool any = left > 0;
    uint32_t in = ring0, out = ring0;
    auto fetch = [&]() {
      if (ahead > 0) {
        St::fetch(in, x.at, p.width, x.lo, x.hi);
        St::fetch(in + St::BYTES, dy.at, p.width, dy.lo, dy.hi);
      }
      --ahead;
      x.at += x.step, dy.at += dy.step;
      in = in + BYTES == ring_end ? ring0 : in + BYTES;
      cp_commit();
    };
    for (int k = 0; k < p.stages - 1; ++k) fetch();
    F2 ga[H], sa[H], sb[H];
#pragma unroll
    for (int k = 0; k < H; ++k) sa[k] = sb[k] = f2(0.f);
    if (any) load_gain<Tm>(p, it.g, ga);
    // Statistics of the first row; each row loads the next one's.
    const float* stat = p.stats + it.first;
    float mu = 0.f, rs = 0.f;
    if (any) mu = stat[0], rs = stat[p.rows];
    T* dx = static_cast<T*>(p.out) + it.first * p.width;
    for (int k = 0; k < it.iters; ++k) {
      cp_wait(p.stages);
      if constexpr (E == 1) Tm::barrier();
      fetch();
      stat += it.step;
      float mu_next = 0.f, rs_next = 0.f;
      if (left > 1) mu_next = stat[0], rs_next = stat[p.rows];
      const char* buf = ring + (out - ring0);
      out = out + BYTES == ring_end ? ring0 : out + BYTES;
      F2 z[H], d[H];
      float2 s = make_float2(0.f, 0.f);
      if (left > 0) {
        St::read(buf, x_now, p.width, z);
        St::read(buf + St::BYTES, dy_now, p.width, d);
        const F2 nm = f2(-mu), r = f2(rs);
        F2 s1 = f2(0.f), s2 = f2(0.f);
        // Beyond the row dy is 0 and adds nothing.
#pragma unroll
        for (int h = 0; h < H; ++h) {
          z[h] = (z[h] + nm) * r;
          sa[h] = fma2(d[h], z[h], sa[h]);
          sb[h] = sb[h] + d[h];
          d[h] = d[h] * ga[h];
          s1 = s1 + d[h];
          s2 = fma2(d[h], z[h], s2);
        }
        s = make_float2(both(s1), both(s2));
      }
      if (p.out) {
        s = Tm::sum2(s, red[flip]);
        flip ^= 1;
        if (left > 0) store_dx<T, Tm>(dx, p.width, z, d, s, inv_n, rs);
      }
      --left;
      mu = mu_next;
      rs = rs_next;
      dx += it.step * p.width;
      x_now += x.step, dy_now += dy.step;
    }
    if constexpr (E == 1) Tm::barrier();  // the ring is refilled for the next item
    if (!p.da && !p.db) continue;
    if (p.team_items || TEAMS == 1) {
      if (!any) continue;
      if (p.split > 1) {  // rows of partial sums are 16-byte aligned where E > 1
        float* w = p.ws + base * 2 * p.width;
        Tm::store_params(w, LEWM_TYPE_F32, 0, p.width, true, sa);
        Tm::store_params(w, LEWM_TYPE_F32, p.width, p.width, true, sb);
      } else {
        if (p.da) Tm::store_params(p.da, p.p_type, it.g * p.width, p.width, p.p_vec, sa);
        if (p.db) Tm::store_params(p.db, p.p_type, it.g * p.width, p.width, p.p_vec, sb);
      }
    } else {
      // Add the teams' sums in team order, a slab of columns at a time.
      constexpr int PAIRS = E > 1 ? E / 2 : 1;
#pragma unroll
      for (int i = 0; i < H / PAIRS; ++i) {
        if (i * SLAB >= p.width) break;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
          const float2 a = split(sa[i * PAIRS + k]), b = split(sb[i * PAIRS + k]);
          const int c = E > 1 ? Tm::lane() * E + 2 * k : Tm::lane(), next = E > 1 ? c + 1 : c + TPR;
          sums[Tm::team() * SLAB + c] = make_float2(a.x, b.x);
          sums[Tm::team() * SLAB + next] = make_float2(a.y, b.y);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < SLAB; c += THREADS) {
          const int64_t col = (int64_t)i * SLAB + c;
          if (col >= p.width) continue;
          float a = 0.f, b = 0.f;
#pragma unroll
          for (int t = 0; t < TEAMS; ++t) a += sums[t * SLAB + c].x, b += sums[t * SLAB + c].y;
          if (p.split > 1) {
            float* w = p.ws + base * 2 * p.width + col;
            w[0] = a;
            w[p.width] = b;
          } else {
            if (p.da) store_param(p.da, p.p_type, it.g * p.width + col, a);
            if (p.db) store_param(p.db, p.p_type, it.g * p.width + col, b);
          }
        }
      }
      __syncthreads();
    }
  }
}

// A modulation row per row of x: d scale = dy z and d shift = dy row by row, nothing to sum up.
template <typename T, typename P, typename Tm>
__global__ void __launch_bounds__(Tm::THREADS, bound_blocks<Tm>(true, true)) k_rowmod_bwd(const NormArgs p) {
  griddep_wait();
  using St = Stage<T, Tm>;
  using Sp = Stage<P, Tm>;
  constexpr int H = Tm::H, BYTES = 2 * St::BYTES + Sp::BYTES;
  extern __shared__ __align__(16) char ring[];
  __shared__ float2 red[2][32];
  const float inv_n = 1.0f / p.width;
  const uint32_t ring0 = smem_u32(ring), ring_end = ring0 + p.stages * BYTES;
  const int64_t first = (int64_t)blockIdx.x * Tm::TEAMS + Tm::team(), step = (int64_t)gridDim.x * Tm::TEAMS;
  const int iters = p.loop_min + ((int64_t)blockIdx.x * Tm::TEAMS < p.loop_rem);
  Walk<T> x(p.x, p.rows, p.x_stride, p.width, first, step), dy(p.dy, p.rows, p.dy_stride, p.width, first, step);
  Walk<P> a(p.a, p.rows, p.a_stride, p.width, first, step);
  const T *x_now = x.at, *dy_now = dy.at;
  const P* a_now = a.at;
  int left = p.loop_min + (first < p.loop_rem), ahead = left;
  uint32_t in = ring0, out = ring0;
  auto fetch = [&]() {
    if (ahead > 0) {
      St::fetch(in, x.at, p.width, x.lo, x.hi);
      St::fetch(in + St::BYTES, dy.at, p.width, dy.lo, dy.hi);
      Sp::fetch(in + 2 * St::BYTES, a.at, p.width, a.lo, a.hi);
    }
    --ahead;
    x.at += x.step, dy.at += dy.step, a.at += a.step;
    in = in + BYTES == ring_end ? ring0 : in + BYTES;
    cp_commit();
  };
  for (int k = 0; k < p.stages - 1; ++k) fetch();
  const float* stat = p.stats + first;
  float mu = 0.f, rs = 0.f;
  if (left > 0) mu = stat[0], rs = stat[p.rows];
  int64_t at = first * p.width;
  int flip = 0;
  for (int k = 0; k < iters; ++k) {
    cp_wait(p.stages);
    if constexpr (Tm::E == 1) Tm::barrier();
    fetch();
    stat += step;
    float mu_next = 0.f, rs_next = 0.f;
    if (left > 1) mu_next = stat[0], rs_next = stat[p.rows];
    const char* buf = ring + (out - ring0);
    out = out + BYTES == ring_end ? ring0 : out + BYTES;
    F2 z[H], d[H];
    float2 s = make_float2(0.f, 0.f);
    if (left > 0) {
      F2 t[H];
      St::read(buf, x_now, p.width, z);
      St::read(buf + St::BYTES, dy_now, p.width, d);
      if (p.db) Tm::store_row(static_cast<P*>(p.db) + at, p.width, d);
      const F2 nm = f2(-mu), r = f2(rs), one = f2(1.f);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        z[h] = (z[h] + nm) * r;
        t[h] = d[h] * z[h];
      }
      if (p.da) Tm::store_row(static_cast<P*>(p.da) + at, p.width, t);
      Sp::read(buf + 2 * St::BYTES, a_now, p.width, t);
      F2 s1 = f2(0.f), s2 = f2(0.f);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        d[h] = d[h] * (t[h] + one);
        s1 = s1 + d[h];
        s2 = fma2(d[h], z[h], s2);
      }
      s = make_float2(both(s1), both(s2));
    }
    if (p.out) {
      s = Tm::sum2(s, red[flip]);
      flip ^= 1;
      if (left > 0) store_dx<T, Tm>(static_cast<T*>(p.out) + at, p.width, z, d, s, inv_n, rs);
    }
    --left;
    mu = mu_next;
    rs = rs_next;
    at += step * p.width;
    x_now += x.step, dy_now += dy.step, a_now += a.step;
  }
}

// Sum of the `split` partial sums of each group in a fixed order. R = 32: 32 interleaved runs of
// items by 8 vectors of VW columns in a block, all of a run's loads started together, then the
// runs through shared memory. R = 1, for few items: a thread adds a vector's partials by itself.
// Grid (column tiles, groups, a or b).
template <int R, int VW>
__global__ void __launch_bounds__(256) k_norm_reduce(const NormArgs p) {
  griddep_wait();
  constexpr int LANES = 256 / R, COLS = LANES * VW;
  using V = Vec<float, VW>;
  __shared__ V part[R][LANES];
  const int cx = threadIdx.x % LANES, run = threadIdx.x / LANES;
  const int64_t col = (int64_t)blockIdx.x * COLS + cx * VW;
  void* out = blockIdx.z ? p.db : p.da;
  if (!out) return;
  const int64_t groups = p.items / p.split, stride = 2 * (int64_t)p.width;
  for (int64_t g = blockIdx.y; g < groups; g += gridDim.y) {
    V s;
#pragma unroll
    for (int e = 0; e < VW; ++e) s.v[e] = 0.f;
    if (col < p.width) {
      const float* w = p.ws + (g * p.split * 2 + blockIdx.z) * p.width + col;
      for (int i = run; i < p.split; i += 8 * R) {
        V v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i + k * R < p.split) v[k] = *reinterpret_cast<const V*>(w + (i + k * R) * stride);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i + k * R < p.split) {
#pragma unroll
            for (int e = 0; e < VW; ++e) s.v[e] += v[k].v[e];
          }
      }
    }
    if constexpr (R > 1) {
      part[run][cx] = s;
      __syncthreads();
#pragma unroll
      for (int half = R / 2; half > 0; half >>= 1) {
        if (run < half) {
#pragma unroll
          for (int e = 0; e < VW; ++e) part[run][cx].v[e] += part[run + half][cx].v[e];
        }
        if (half * LANES > 32) __syncthreads();
        else __syncwarp();
      }
      s = part[0][cx];
    }
    if (run == 0 && col < p.width) {
#pragma unroll
      for (int e = 0; e < VW; ++e) store_param(out, p.p_type, g * p.width + col + e, s.v[e]);
    }
    if (R > 1) __syncthreads();
  }
}

// ------------------------------------------------------------------ rows of more than kMaxRowBytes
// One block per row, the row re-read from L2 for each pass.
using Wide = Team<1, 2, 1024>;
template <typename T>
__global__ void __launch_bounds__(1024) k_norm_fwd_wide(const NormArgs p) {
  griddep_wait();
  __shared__ float red[2][32];
  const float inv_n = 1.0f / p.width;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x; c < p.width; c += 1024) s += to_f(x[c]);
    const float mu = Wide::sum(s, red[0]) * inv_n;
    for (int c = threadIdx.x; c < p.width; c += 1024) {
      const float d = to_f(x[c]) - mu;
      q = fmaf(d, d, q);
    }
    const float rs = 1.0f / sqrtf(Wide::sum(q, red[1]) * inv_n + p.eps);
    if (p.stats && threadIdx.x == 0) {
      p.stats[r] = mu;
      p.stats[p.rows + r] = rs;
    }
    const int64_t g = r / p.group;
    T* y = static_cast<T*>(p.out) + r * p.width;
    for (int c = threadIdx.x; c < p.width; c += 1024) {
      float a = 1.f, b = 0.f;
      if (p.a) a = load_param(p.a, p.p_type, g * p.a_stride + c);
      if (p.b) b = load_param(p.b, p.p_type, g * p.b_stride + c);
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
      if (p.a) a = load_param(p.a, p.p_type, g * p.a_stride + c);
      return p.one_plus ? a + 1.f : a;
    };
    float2 s = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < p.width; c += 1024) {
      const float d = to_f(dy[c]) * gain(c);
      s.x += d;
      s.y = fmaf(d, (to_f(x[c]) - mu) * rs, s.y);
    }
    s = Wide::sum2(s, red[flip]);
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
    const Item it = item_rows<1>(p, item, 0);
    float a = 0.f, b = 0.f;
    int64_t r = it.first;
    for (int k = 0; k < it.rows; ++k, r += it.step) {
      const float g = to_f(static_cast<const T*>(p.dy)[r * p.dy_stride + col]);
      const float z = (to_f(static_cast<const T*>(p.x)[r * p.x_stride + col]) - p.stats[r]) * p.stats[p.rows + r];
      a = fmaf(g, z, a);
      b += g;
    }
    if (p.split > 1) {
      float* w = p.ws + item * 2 * p.width + col;
      w[0] = a;
      w[p.width] = b;
    } else {
      if (p.da) store_param(p.da, p.p_type, it.g * p.width + col, a);
      if (p.db) store_param(p.db, p.p_type, it.g * p.width + col, b);
    }
  }
}

// ------------------------------------------------------------------ host side
// Team of a row: threads x elements per thread covers the width.
struct Tier {
  int tpr, ept;
  int teams() const { return block_threads(tpr) / tpr; }
};
Tier tier_of(int64_t width, bool backward) {
  if (width <= 64) return {8, 8};
  if (width <= 256) return {32, 8};
  // The forward keeps no sums: 32 values a thread leave two blocks per SM where 16 leave one.
  if (!backward && width > 4096 && width <= 8192) return {256, 32};
  int tpr = 32;
  while (tpr * 16 < width) tpr *= 2;  // rows of at most kMaxRowBytes: tpr <= 1024
  return {tpr, 16};
}
int64_t type_size(int type) { return type == LEWM_TYPE_F32 ? 4 : 2; }
bool is_wide(const NormArgs& p, int x_type) { return p.width * type_size(x_type) > kMaxRowBytes; }

// Blocks that fill the GPU once.
int64_t full_grid(const Tier& t, bool backward) {
  return (int64_t)kSms * (t.ept == 32      ? bound_blocks<Team<1, 32, 256>>(backward)
                          : t.tpr <= 256   ? bound_blocks<Team<1, 16, 256>>(backward)
                          : t.tpr == 512   ? bound_blocks<Team<1, 16, 512>>(backward)
                                           : bound_blocks<Team<1, 16, 1024>>(backward));
}
// Rounds of loops over `rows` rows in steps of `step`. (No tensor that fits a GPU makes 2^31 rounds: a
// step is a row for groups of a few, else a block's teams times the blocks that share the rows.)
void set_loop(NormArgs* p, int64_t rows, int64_t step) {
  p->loop_min = (int)std::min<int64_t>(rows / step, INT_MAX - 1);
  p->loop_rem = (int)(rows % step);
}

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
    const Tier t = tier_of(p->width, backward);
    // A team's items where a group has too few rows to keep a block's teams busy and there
    // are groups enough to fill the GPU without splitting them.
    p->team_items = p->group < 2 * t.teams() && groups >= 2 * kSms;
    const int64_t want = full_grid(t, backward) / groups;  // one wave of blocks
    const int64_t most = (p->group + t.teams() - 1) / t.teams();
    p->split = p->team_items ? 1 : (int)std::max<int64_t>(1, std::min(want, most));
  }
  p->items = groups * p->split;
  set_loop(p, p->group, p->team_items ? 1 : (int64_t)p->split * (is_wide(*p, x_type) ? 1 : tier_of(p->width, backward).teams()));
}

size_t workspace_bytes(const NormArgs& p) {
  return p.split > 1 ? (size_t)p.items * 2 * (size_t)p.width * sizeof(float) : 0;
}

// Stages of `bytes` each for `blocks` blocks per SM (fewer if they do not fit): 2 to 4, as many as
// keep `ahead` bytes per SM on their way; 0 where not even two fit one block. More than needed is
// slower: rows fetched far ahead compete with the stores in DRAM. 48 KB do where a pass writes as
// much as it reads (73881 x 1536 float32 forward with 2, 3 and 4 stages of 48 KB per SM: 142, 170
// and 172 us; 131072 x 2048 bf16 with 24 KB stages: 184, 174, 183), 96 KB in the backward (float32
// with 64 KB stages: 209, 203, 203; bf16 with 32 KB: 276, 258, 260).
constexpr int kSmemPerSm = 227 * 1024, kSmemReserved = 2 * 1024;  // the latter: static and the system's, per block
constexpr int kAhead = 48 * 1024, kAheadBackward = 96 * 1024;
int ring_stages(int bytes, int blocks, int ahead) {
  for (; blocks >= 1; blocks = blocks / 2) {
    const int fit = (kSmemPerSm / blocks - kSmemReserved) / bytes;
    const int want = std::min(4, 1 + (ahead + bytes * blocks - 1) / (bytes * blocks));
    if (fit >= std::min(want, 3) || (blocks == 1 && fit >= 2)) return std::min(fit, std::max(want, 2));
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

// The passes that use a tier (tier_of).
template <typename Tm>
constexpr bool has_backward = Tm::N != 32;
template <typename Tm>
constexpr bool has_forward = !(Tm::N == 16 && Tm::TPR == 512);

template <typename T, typename Tm>
cudaError_t launch_items(NormArgs p, bool backward, cudaStream_t st) {
  static bool raised[2][64];  // only ever set to true: calls from several threads may repeat the attribute
  const int bytes = (backward ? 2 : 1) * Stage<T, Tm>::BYTES;
  p.stages = ring_stages(bytes, bound_blocks<Tm>(backward), backward ? kAheadBackward : kAhead);
  const int64_t blocks = p.team_items ? (p.items + Tm::TEAMS - 1) / Tm::TEAMS : p.items;
  const int64_t grid = std::min(blocks, (int64_t)kSms * bound_blocks<Tm>(backward));
  if constexpr (has_backward<Tm>)
    if (backward) return launch_ring(k_norm_bwd<T, Tm>, raised[1], grid, Tm::THREADS, bytes * p.stages, p, st);
  if constexpr (has_forward<Tm>)
    if (!backward) return launch_ring(k_norm_fwd<T, Tm>, raised[0], grid, Tm::THREADS, bytes * p.stages, p, st);
  return cudaErrorInvalidValue;  // not a tier of this pass
}

// group 1: the modulation in the ring, if two stages of it fit.
template <typename T, typename P, typename Tm>
cudaError_t launch_rowmod(NormArgs p, bool backward, cudaStream_t st) {
  static bool raised[2][64];
  const int x_bytes = Stage<T, Tm>::BYTES, p_bytes = Stage<P, Tm>::BYTES;
  const int bytes = backward ? 2 * x_bytes + p_bytes : x_bytes + 2 * p_bytes;
  p.stages = ring_stages(bytes, bound_blocks<Tm>(backward, true), kAhead);
  if (p.stages == 0) return launch_items<T, Tm>(p, backward, st);
  const int64_t grid = std::min((p.rows + Tm::TEAMS - 1) / Tm::TEAMS, (int64_t)kSms * bound_blocks<Tm>(backward, true));
  set_loop(&p, p.rows, grid * Tm::TEAMS);
  if constexpr (has_backward<Tm>)
    if (backward) return launch_ring(k_rowmod_bwd<T, P, Tm>, raised[1], grid, Tm::THREADS, bytes * p.stages, p, st);
  if constexpr (has_forward<Tm>)
    if (!backward) return launch_ring(k_rowmod_fwd<T, P, Tm>, raised[0], grid, Tm::THREADS, bytes * p.stages, p, st);
  return cudaErrorInvalidValue;  // not a tier of this pass
}

template <typename T, int E, int NV, int TPR>
cudaError_t launch_tier(const NormArgs& p, bool backward, cudaStream_t st) {
  using Tm = Team<E, NV, TPR>;
  if (p.group > 1 || !p.one_plus) return launch_items<T, Tm>(p, backward, st);
  if (p.p_type == LEWM_TYPE_F32) return launch_rowmod<T, float, Tm>(p, backward, st);
  constexpr bool any = std::is_same<T, float>::value;
  if constexpr (any || std::is_same<T, __nv_bfloat16>::value)
    if (p.p_type == LEWM_TYPE_BF16) return launch_rowmod<T, __nv_bfloat16, Tm>(p, backward, st);
  if constexpr (any || std::is_same<T, __half>::value)
    if (p.p_type == LEWM_TYPE_F16) return launch_rowmod<T, __half, Tm>(p, backward, st);
  return launch_items<T, Tm>(p, backward, st);  // bf16 beside fp16
}

template <typename T, int E>
cudaError_t launch_width(const NormArgs& p, bool backward, cudaStream_t st) {
  constexpr int V8 = 8 / E, V16 = 16 / E, V32 = 32 / E;
  const Tier t = tier_of(p.width, backward);
  if (t.ept == 8) return t.tpr == 8 ? launch_tier<T, E, V8, 8>(p, backward, st) : launch_tier<T, E, V8, 32>(p, backward, st);
  if (t.ept == 32) return launch_tier<T, E, V32, 256>(p, false, st);
  switch (t.tpr) {
    case 32: return launch_tier<T, E, V16, 32>(p, backward, st);
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
  const unsigned gy = (unsigned)std::min<int64_t>(groups, 65535);
  const int vw = p.width % 4 == 0 ? 4 : 1, cols = (p.split <= 16 ? 256 : 8) * vw;
  const dim3 grid((p.width + cols - 1) / cols, gy, 2);
  if (p.split <= 16)
    return vw == 4 ? launch_k(k_norm_reduce<1, 4>, grid, dim3(256), 0, st, p)
                   : launch_k(k_norm_reduce<1, 1>, grid, dim3(256), 0, st, p);
  return vw == 4 ? launch_k(k_norm_reduce<32, 4>, grid, dim3(256), 0, st, p)
                 : launch_k(k_norm_reduce<32, 1>, grid, dim3(256), 0, st, p);
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
