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
// Bound: bytes, 4 to 12 per element and pass. Many rows run at 91 to 102% of the rate of a plain copy
// (131072 x 2048 bf16: forward 168 us, backward 261; 73881 x 1536 float32, groups of 8209 rows: 140 and
// 206), at odd addresses at about 55%: there a row costs 1.5 times the instructions (16384 x 2047 bf16:
// 36 and 51 us). A row therefore stays in registers from its only load to its only
// store (mean and variance are two passes over registers, row_stats), and sums over rows are kept in
// registers by persistent blocks that own fixed columns, so x and dy are read once.
//
// Layout: a team of TPR threads holds one row, NV vectors of E elements per thread (vectors of 16, 8
// or 4 bytes, whatever every row starts on, or single 16-bit elements). In the backward that is at
// most 16 elements a thread: it then holds 16 gains and 32 sums, 128 registers at two 256-thread
// blocks per SM. Rows of more than 32 KB, and of more than 8192 values in the backward that keeps
// sums, take the looping kernels below.
//
// Rows arrive through a ring of 2 to 4 stages in shared memory, filled by cp.async one to
// three rows ahead: registers alone kept 32 KB per SM on the way at best and none while a row
// was being reduced, half of HBM's rate (131072 x 2048 bf16: forward 307 us, backward 404).
// With vectors each thread copies just what it reads itself, so the ring needs no barrier; rows
// of odd 16-bit addresses (odd float32 widths, and rows off 16 bytes with a modulation row each) are copied
// by 16-byte pieces with 4-byte ends and read back element by element after a team barrier.
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
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "lewm_b200.h"
#include "lewm_common.cuh"
#include "lewm_internal.h"
#include "train_elem.cuh"
#include "train_norm.h"

namespace lewm {
namespace {

// ------------------------------------------------------------------ parameters
// E values as elements of type P at `q` (E > 1), in accesses of min(16, E sizeof(P)) bytes if the
// address allows it (`vec`).
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

// Passes: an item's rows share their parameters, or each row has its own modulation row.
enum Pass { FWD, BWD, ROW_FWD, ROW_BWD };
constexpr bool is_backward(Pass p) { return p == BWD || p == ROW_BWD; }

// Team of a row: threads x values a thread cover the width.
struct Tier {
  int tpr, n;
  constexpr int teams() const { return block_threads(tpr) / tpr; }
};
// Many narrow rows take small teams of many values (`dense`), so several rows to a warp: a row costs a
// thread some hundred instructions beside those of its values, and a team of 32 spends them 32
// times (57600 x 192 bf16 with a modulation row per row: forward 19.0 us in teams of 32, 15.9 in teams
// of 8; 16448 x 192 forward 6.9 and 5.8). Fewer rows than fill the GPU that way keep teams of 32, whose
// threads have less to do one after the other (900 x 192 float32 forward 3.1 us, 4.8 in teams of 8), and
// so do rows at odd addresses, whose single-element accesses are then 64 bytes wide.
constexpr bool dense_rows(int64_t rows, bool vec) { return vec && rows >= 32 * kSms; }
//
// Wider rows take teams of a power of 2 with 16 values a thread, or
//   24 in the forward of 16-bit rows, where half the team covers them: fewer idle lanes (49152 x 2720
//      bf16 129 us with 16, 88 with 24; float32 rows, which are bound by DRAM, mostly lose: 73881 x 1536 from
//      140 to 156);
//   24 or 32 in the forward of more than 4096: two blocks per SM instead of one (16384 x 8192 bf16: 120
//      and 85 us);
//   12 in the backward where they cover the row (32768 x 1301 bf16 86 and 76 us).
constexpr Tier tier_of(int64_t width, Pass pass, bool dense, int size) {
  if (width <= 64) return {8, 8};
  if (!dense) {
    if (width <= 256) return {32, 8};
  } else {
    if (width <= 128) return {8, 16};
    if (width <= 192 && pass != BWD) return {8, 24};
    if (width <= 256) return {16, 16};
    if (width <= 384 && pass != BWD) return {16, 24};
  }
  int tpr = 32;
  while (tpr * 16 < width) tpr *= 2;  // rows of at most kMaxRowBytes: tpr <= 1024
  if (!is_backward(pass) && tpr >= 512) return {tpr / 2, width <= tpr * 12 ? 24 : 32};
  if (pass == FWD && size == 2 && tpr > 32 && width <= tpr * 12) return {tpr / 2, 24};
  if (pass == BWD && tpr > 32 && width <= tpr * 12) return {tpr, 12};
  return {tpr, 16};
}
// The narrowest row of a tier, 0 for one that the pass does not use. (The tiers that dense rows and
// others share have the same narrowest row, or the lower one.)
constexpr int64_t min_width_of(int tpr, int n, Pass pass, bool dense, int size) {
  const int64_t edges[] = {64,      128,  192,      256,  384,      512,  32 * 24,  1024,
                           64 * 24, 2048, 128 * 24, 4096, 256 * 24, 8192, 512 * 24, 16384};
  int64_t before = 0;
  for (int64_t e : edges) {
    const Tier t = tier_of(e, pass, dense, size);
    if (t.tpr == tpr && t.n == n) return before + 1;
    before = e;
  }
  return 0;
}
constexpr int64_t min_width(int tpr, int n, Pass pass, bool vec, int size) {
  const int64_t a = min_width_of(tpr, n, pass, false, size), b = vec ? min_width_of(tpr, n, pass, true, size) : 0;
  return a == 0 ? b : b == 0 || a < b ? a : b;
}

template <int E_, int NV_, int TPR_, int64_t MIN_WIDTH>
struct Team {
  static constexpr int E = E_, NV = NV_, TPR = TPR_, N = E * NV, H = N / 2;
  static constexpr int THREADS = block_threads(TPR), TEAMS = THREADS / TPR;
  // Vectors that lie inside every row of the tier.
  static constexpr int SURE = (int)(MIN_WIDTH / (TPR * E));

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
  // The sum over a team of more than 8 warps and what its last addition lost: exact where the sums of
  // 8 warps are.
  static __device__ __forceinline__ float2 sum_and_rest(float v, float* red) {
    constexpr int WARPS = TPR / 32;
    static_assert(WARPS > 8 && WARPS <= 16, "two runs of warps");
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warp = threadIdx.x >> 5, w0 = team() * WARPS;
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    barrier();
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a += red[w0 + i];
      if (8 + i < WARPS) b += red[w0 + 8 + i];
    }
    // The rounding error of a + b (Knuth's TwoSum).
    const float s = a + b, t = s - a;
    return make_float2(s, (a - (s - t)) + (b - t));
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

  // This thread's parameters of a row of `width`, 0 beyond it. All loads before the first conversion:
  // one after the other they cost a block several us.
  template <typename P>
  static __device__ __forceinline__ void load_typed(const P* q, int width, bool vec, F2* f) {
    if constexpr (E > 1) {
      constexpr int K = E * (int)sizeof(P) > 16 ? 16 / (int)sizeof(P) : E, PIECES = E / K;
      const int nvec = width / E;
      Vec<P, K> raw[NV][PIECES] = {};
      q += lane() * E;
      if (vec) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int k = 0; k < PIECES; ++k)
            if (i < SURE || lane() + i * TPR < nvec) raw[i][k] = reinterpret_cast<const Vec<P, K>*>(q + i * TPR * E)[k];
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (i < SURE || lane() + i * TPR < nvec) raw[i][e / K].v[e % K] = q[i * TPR * E + e];
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
#pragma unroll
          for (int e = 0; e < K; e += 2) f[(i * E + k * K + e) / 2] = unpack(raw[i][k].v + e);
    } else {
      P raw[N] = {};
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < SURE || lane() + i * TPR < width) raw[i] = q[lane() + i * TPR];
#pragma unroll
      for (int i = 0; i < H; ++i) f[i] = f2(to_f(raw[2 * i]), to_f(raw[2 * i + 1]));
    }
  }
  static __device__ __forceinline__ void load_params(const void* p, int type, int64_t at, int width, bool vec, F2* f) {
    if (type == LEWM_TYPE_F32) load_typed(static_cast<const float*>(p) + at, width, vec, f);
    else if (type == LEWM_TYPE_BF16) load_typed(static_cast<const __nv_bfloat16*>(p) + at, width, vec, f);
    else load_typed(static_cast<const __half*>(p) + at, width, vec, f);
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
//   E > 1: vector i of a thread lies at [piece][i][thread] in pieces of 16 bytes (8 or 4 where the
//          vector is that small); only that thread copies and reads it.
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
            else if constexpr (PB == 8) cp_async8(dst + (k * NV + i) * THREADS * PB, src + i * TPR * VB + k * PB);
            else cp_async4(dst + (k * NV + i) * THREADS * PB, src + i * TPR * VB + k * PB);
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

// Blocks per SM that the registers are limited for: 80 a thread forward (128 with 24 or 32 values), 128
// in the backward that keeps sums. More, smaller blocks were slower on short rows: every block
// loads the parameters anew. The backward of a modulation row per row has neither and takes 4
// with 8 values (57600 x 192 bf16 in teams of 32, 2, 3 and 4 blocks: 26.2, 22.9, 21.6 us).
constexpr int bound_blocks(int tpr, int n, Pass pass) {
  const int threads = pass == ROW_BWD && n == 8 ? 1024 : is_backward(pass) || n >= 24 ? 512 : 768;
  return threads >= block_threads(tpr) ? threads / block_threads(tpr) : 1;
}
template <typename Tm, Pass PASS>
constexpr int kBound = bound_blocks(Tm::TPR, Tm::N, PASS);

// What multiplies z in group g, and what is added: weight or 1 + scale, bias or shift.
template <typename Tm>
__device__ __forceinline__ void load_gain(const NormArgs& p, int64_t g, F2* a) {
  if (p.a) {
    Tm::load_params(p.a, p.p_type, g * p.a_stride, p.width, p.p_vec, a);
  } else {
#pragma unroll
    for (int k = 0; k < Tm::H; ++k) a[k] = f2(1.f);
  }
  if (p.one_plus) {
#pragma unroll
    for (int k = 0; k < Tm::H; ++k) a[k] = a[k] + f2(1.f);
  }
}
template <typename Tm>
__device__ __forceinline__ void load_offset(const NormArgs& p, int64_t g, F2* b) {
  if (p.b) {
    Tm::load_params(p.b, p.p_type, g * p.b_stride, p.width, p.p_vec, b);
  } else {
#pragma unroll
    for (int k = 0; k < Tm::H; ++k) b[k] = f2(0.f);
  }
}

// ------------------------------------------------------------------ forward
// The variance from the sums q of c^2 and s of c, and d = s / n: mean(c^2) - d^2. q of infinity stays.
__device__ __forceinline__ float variance(float q, float s, float d, float inv_n) {
  return (q <= FLT_MAX ? fmaxf(fmaf(-s, d, q), 0.f) : q) * inv_n;
}

// x - mean in place of the team's values x (0 beyond the row), mean and rs. An error of the mean comes out up
// to 1 / sqrt(eps) times as large, so that of float32 rows, whose sum is rounded, is taken in two steps:
// c = x - mu with the rounded mean mu, then what is left, d = mean(c), comes off too (and off the variance,
// mean(c^2) - d^2). In one step a constant row (padding) of 1234.567 gave z of 0.1 instead of 0. The sum of a
// constant row c of 16-bit values is exact, but for fp16 (11 bits) beyond 8192 of them: the last addition's
// error is kept there. n c / n is c then, and z of a constant row 0. One step and two: 73881 x 1536 float32
// 140 and 141 us, 57600 x 192 16.4 and 16.5, 32768 x 2720 120 and 121; 16384 x 16384 fp16 without and with
// the error 193 and 193.
template <typename T, typename Tm>
__device__ __forceinline__ float2 row_stats(F2* f, int width, float inv_n, float eps, float2 (*red)[32]) {
  constexpr int E = Tm::E, TPR = Tm::TPR;
  constexpr bool TWO_STEPS = sizeof(T) == 4;
  constexpr bool REST = std::is_same<T, __half>::value && TPR * Tm::N > 8192;
  F2 s = f2(0.f), q = f2(0.f);
#pragma unroll
  for (int k = 0; k < Tm::H; ++k) s = s + f[k];
  float* const red0 = reinterpret_cast<float*>(red[0]);
  float mu;
  if constexpr (TWO_STEPS) {
    mu = Tm::sum(both(s), red0) * inv_n;
  } else if constexpr (REST) {
    const float2 sum = Tm::sum_and_rest(both(s), red0);
    mu = sum.x / (float)width;
    mu = fmaf(fmaf(-mu, (float)width, sum.x) + sum.y, inv_n, mu);
  } else {
    mu = Tm::sum(both(s), red0) / (float)width;
  }
  const F2 nm = f2(-mu);
  s = f2(0.f);
#pragma unroll
  for (int k = 0; k < Tm::H; ++k) {
    f[k] = f[k] + nm;
    if constexpr (E > 1) {
      const int i = k / (E / 2);
      if (i < Tm::SURE || Tm::lane() + i * TPR < width / E) {
        q = fma2(f[k], f[k], q);
        if constexpr (TWO_STEPS) s = s + f[k];
      }
    } else {
      const int i = 2 * k;
      F2 c = f[k];
      if (i + 1 >= Tm::SURE) {
        const float2 v = split(c);
        c = f2(Tm::lane() + i * TPR < width ? v.x : 0.f, Tm::lane() + (i + 1) * TPR < width ? v.y : 0.f);
      }
      q = fma2(c, c, q);
      if constexpr (TWO_STEPS) s = s + c;
    }
  }
  float var;
  if constexpr (TWO_STEPS) {
    const float2 qs = Tm::sum2(make_float2(both(q), both(s)), red[1]);
    const float d = qs.y / (float)width;
    var = variance(qs.x, qs.y, d, inv_n);
    mu += d;
    const F2 nd = f2(-d);
#pragma unroll
    for (int k = 0; k < Tm::H; ++k) f[k] = f[k] + nd;
  } else {
    var = Tm::sum(both(q), reinterpret_cast<float*>(red[1])) * inv_n;
  }
  return make_float2(mu, 1.0f / sqrtf(var + eps));
}

template <typename T, typename Tm>
__global__ void __launch_bounds__(Tm::THREADS, kBound<Tm, FWD>) k_norm_fwd(const NormArgs p) {
  griddep_wait();  // launched as a programmatic dependent: wait for the kernel before
  using St = Stage<T, Tm>;
  constexpr int H = Tm::H;
  extern __shared__ __align__(16) char ring[];
  __shared__ float2 red[2][32];
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
      const float2 ms = row_stats<T, Tm>(f, p.width, inv_n, p.eps, red);
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
__global__ void __launch_bounds__(Tm::THREADS, kBound<Tm, ROW_FWD>) k_rowmod_fwd(const NormArgs p) {
  griddep_wait();
  using St = Stage<T, Tm>;
  using Sp = Stage<P, Tm>;
  constexpr int H = Tm::H, BYTES = St::BYTES + 2 * Sp::BYTES;
  extern __shared__ __align__(16) char ring[];
  __shared__ float2 red[2][32];
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
    const float2 ms = row_stats<T, Tm>(f, p.width, inv_n, p.eps, red);
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
__global__ void __launch_bounds__(Tm::THREADS, kBound<Tm, BWD>) k_norm_bwd(const NormArgs p) {
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
__global__ void __launch_bounds__(Tm::THREADS, kBound<Tm, ROW_BWD>) k_rowmod_bwd(const NormArgs p) {
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

// ------------------------------------------------------------------ rows too wide for a block (is_wide)
// A block per row, the row re-read (from L2) for each pass, in vectors of E elements.
// Threads of a block, 2048 on an SM: 256, 512 and 1024 took 35, 33 and 39 us forward (1000 x 20000 bf16; the
// mean's second step adds 2 to each) and 414, 424 and 530 us backward (16384 x 10000 bf16).
constexpr int kWideThreads = 512;
using Wide = Team<1, 2, kWideThreads, 0>;

// E elements of T at `q` as float32.
template <typename T, int E>
__device__ __forceinline__ void load_f(const T* q, float* f) {
  const Vec<T, E> v = *reinterpret_cast<const Vec<T, E>*>(q);
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = to_f(v.v[e]);
}
template <typename T, int E>
__device__ __forceinline__ void store_f(T* q, const float* f) {
  Vec<T, E> v;
#pragma unroll
  for (int e = 0; e < E; ++e) v.v[e] = from_f<T>(f[e]);
  *reinterpret_cast<Vec<T, E>*>(q) = v;
}
// E parameters at element offset `at`, `otherwise` where there are none.
template <int E>
__device__ __forceinline__ void load_params_f(const void* p, int type, int64_t at, bool vec, float otherwise,
                                              float* f) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = otherwise;
  } else if (E > 1 && vec && type == LEWM_TYPE_F32) {
#pragma unroll
    for (int e = 0; e < E; e += 4) load_f<float, E < 4 ? E : 4>(static_cast<const float*>(p) + at + e, f + e);
  } else if (E > 1 && vec && type == LEWM_TYPE_BF16) {
    load_f<__nv_bfloat16, E>(static_cast<const __nv_bfloat16*>(p) + at, f);
  } else if (E > 1 && vec) {
    load_f<__half, E>(static_cast<const __half*>(p) + at, f);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = load_param(p, type, at + e);
  }
}

template <typename T, int E>
__global__ void __launch_bounds__(kWideThreads, 2048 / kWideThreads) k_norm_fwd_wide(const NormArgs p) {
  griddep_wait();
  __shared__ float2 red[2][32];
  const float inv_n = 1.0f / p.width;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
    float s = 0.f, q = 0.f, f[E];
#pragma unroll 4
    for (int c = threadIdx.x * E; c < p.width; c += kWideThreads * E) {
      load_f<T, E>(x + c, f);
#pragma unroll
      for (int e = 0; e < E; ++e) s += f[e];
    }
    const float mu = Wide::sum(s, reinterpret_cast<float*>(red[0])) * inv_n;
    s = 0.f;
#pragma unroll 4
    for (int c = threadIdx.x * E; c < p.width; c += kWideThreads * E) {
      load_f<T, E>(x + c, f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float c = f[e] - mu;
        q = fmaf(c, c, q);
        s += c;
      }
    }
    // The mean in two steps, as row_stats takes it.
    const float2 qs = Wide::sum2(make_float2(q, s), red[1]);
    const float d = qs.y / (float)p.width;
    const float rs = 1.0f / sqrtf(variance(qs.x, qs.y, d, inv_n) + p.eps);
    if (p.stats && threadIdx.x == 0) {
      p.stats[r] = mu + d;
      p.stats[p.rows + r] = rs;
    }
    const int64_t g = r / p.group;
    T* y = static_cast<T*>(p.out) + r * p.width;
    const float plus = p.one_plus ? 1.f : 0.f;
#pragma unroll 2
    for (int c = threadIdx.x * E; c < p.width; c += kWideThreads * E) {
      float a[E], b[E];
      load_f<T, E>(x + c, f);
      load_params_f<E>(p.a, p.p_type, g * p.a_stride + c, p.p_vec, 1.f, a);
      load_params_f<E>(p.b, p.p_type, g * p.b_stride + c, p.p_vec, 0.f, b);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = fmaf((f[e] - mu - d) * rs, a[e] + plus, b[e]);
      store_f<T, E>(y + c, f);
    }
  }
}

template <typename T, int E>
__global__ void __launch_bounds__(kWideThreads, 2048 / kWideThreads) k_norm_dx_wide(const NormArgs p) {
  griddep_wait();
  __shared__ float2 red[2][32];
  const float inv_n = 1.0f / p.width, plus = p.one_plus ? 1.f : 0.f;
  int flip = 0;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
    const T* dy = static_cast<const T*>(p.dy) + r * p.dy_stride;
    const float mu = p.stats[r], rs = p.stats[p.rows + r];
    const int64_t g = r / p.group;
    float2 s = make_float2(0.f, 0.f);
    float z[E], d[E], a[E];
    auto load = [&](int c) {
      load_f<T, E>(x + c, z);
      load_f<T, E>(dy + c, d);
      load_params_f<E>(p.a, p.p_type, g * p.a_stride + c, p.p_vec, 1.f, a);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        z[e] = (z[e] - mu) * rs;
        d[e] *= a[e] + plus;
      }
    };
#pragma unroll 2
    for (int c = threadIdx.x * E; c < p.width; c += kWideThreads * E) {
      load(c);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s.x += d[e];
        s.y = fmaf(d[e], z[e], s.y);
      }
    }
    s = Wide::sum2(s, red[flip]);
    flip ^= 1;
    const float m1 = s.x * inv_n, m2 = s.y * inv_n;
    T* o = static_cast<T*>(p.out) + r * p.width;
#pragma unroll 2
    for (int c = threadIdx.x * E; c < p.width; c += kWideThreads * E) {
      load(c);
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = rs * (d[e] - m1 - z[e] * m2);
      store_f<T, E>(o + c, d);
    }
  }
}

// The sums of dy z and dy: a thread per E columns, a block per 256 threads and item.
template <typename T, int E>
__global__ void __launch_bounds__(256) k_norm_sums_wide(const NormArgs p) {
  griddep_wait();
  const int64_t col = ((int64_t)blockIdx.x * 256 + threadIdx.x) * E;
  if (col >= p.width) return;
  for (int64_t item = blockIdx.y; item < p.items; item += gridDim.y) {
    const Item it = item_rows<1>(p, item, 0);
    float a[E], b[E];
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] = b[e] = 0.f;
    int64_t r = it.first;
#pragma unroll 4
    for (int k = 0; k < it.rows; ++k, r += it.step) {
      float x[E], g[E];
      load_f<T, E>(static_cast<const T*>(p.x) + r * p.x_stride + col, x);
      load_f<T, E>(static_cast<const T*>(p.dy) + r * p.dy_stride + col, g);
      const float mu = p.stats[r], rs = p.stats[p.rows + r];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        a[e] = fmaf(g[e], (x[e] - mu) * rs, a[e]);
        b[e] += g[e];
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (p.split > 1) {
        float* w = p.ws + item * 2 * p.width + col + e;
        w[0] = a[e];
        w[p.width] = b[e];
      } else {
        if (p.da) store_param(p.da, p.p_type, it.g * p.width + col + e, a[e]);
        if (p.db) store_param(p.db, p.p_type, it.g * p.width + col + e, b[e]);
      }
    }
  }
}

// ------------------------------------------------------------------ host side
inline int64_t type_size(int type) { return type == LEWM_TYPE_F32 ? 4 : 2; }
// Rows for the looping kernels: too wide for a block's ring, or for its registers in the backward that
// keeps sums (16384 x 10000 bf16: 555 us with 64 registers a thread and the rest spilled, 424 there).
constexpr int64_t kMaxSumWidth = 8192;
inline bool is_wide(const NormArgs& p, int x_type, bool backward) {
  return p.width * type_size(x_type) > kMaxRowBytes || (backward && p.width > kMaxSumWidth);
}

// Rounds of loops over `rows` rows in steps of `step`. (No tensor that fits a GPU makes 2^31 rounds: a
// step is a row for groups of a few, else a block's teams times the blocks that share the rows.)
inline void set_loop(NormArgs* p, int64_t rows, int64_t step) {
  p->loop_min = (int)std::min<int64_t>(rows / step, INT_MAX - 1);
  p->loop_rem = (int)(rows % step);
}

// Stages of `bytes` each for `blocks` blocks per SM (fewer if they do not fit): 2 to 4, as many as
// keep `ahead` bytes per SM on their way; 0 where not even two fit one block. More than needed is
// slower: rows fetched far ahead compete with the stores in DRAM. 48 KB do where a pass writes as
// much as it reads (73881 x 1536 float32 forward with 2, 3 and 4 stages of 48 KB per SM: 142, 170
// and 172 us; 131072 x 2048 bf16 with 24 KB stages: 184, 174, 183), 96 KB in the backward (float32
// with 64 KB stages: 209, 203, 203; bf16 with 32 KB: 276, 258, 260).
constexpr int kSmemPerSm = 227 * 1024, kSmemReserved = 2 * 1024;  // the latter: static and the system's, per block
constexpr int kAhead = 48 * 1024, kAheadBackward = 96 * 1024;
inline int ring_stages(int bytes, int blocks, int ahead) {
  for (; blocks >= 1; blocks = blocks / 2) {
    const int fit = (kSmemPerSm / blocks - kSmemReserved) / bytes;
    const int want = std::min(4, 1 + (ahead + bytes * blocks - 1) / (bytes * blocks));
    if (fit >= std::min(want, 3) || (blocks == 1 && fit >= 2)) return std::min(fit, std::max(want, 2));
  }
  return 0;
}

// Launches a kernel with a ring, raising its limit of dynamic shared memory (once per device).
template <typename K>
cudaError_t launch_ring(K kern, std::atomic<bool>* raised, int64_t grid, int threads, int smem, const NormArgs& p,
                        cudaStream_t st) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !raised[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerSm - kSmemReserved);
    if (e != cudaSuccess) return e;
    if (dev < 64) raised[dev].store(true, std::memory_order_release);
  }
  return launch_k(kern, dim3((unsigned)grid), dim3(threads), smem, st, p);
}

// One pass of a tier, if the pass uses it: sets *e and returns true.
template <typename T, typename P, int E, Pass PASS, int TPR, int N>
bool launch_tier(const Tier& t, NormArgs p, cudaStream_t st, cudaError_t* e) {
  constexpr int64_t MIN = min_width(TPR, N, PASS, E * sizeof(T) == 16, sizeof(T));
  if constexpr (MIN > 0 && N % E == 0 && MIN * (int)sizeof(T) <= kMaxRowBytes &&
                !(PASS == BWD && MIN > kMaxSumWidth)) {
    if (t.tpr != TPR || t.n != N) return false;
    using Tm = Team<E, N / E, TPR, MIN>;
    static std::atomic<bool> raised[64];
    constexpr int x_bytes = Stage<T, Tm>::BYTES, p_bytes = Stage<P, Tm>::BYTES;
    constexpr int bytes = PASS == FWD       ? x_bytes
                          : PASS == BWD     ? 2 * x_bytes
                          : PASS == ROW_FWD ? x_bytes + 2 * p_bytes
                                            : 2 * x_bytes + p_bytes;
    p.stages = ring_stages(bytes, kBound<Tm, PASS>, PASS == BWD ? kAheadBackward : kAhead);
    if (p.stages == 0) return false;  // modulation too wide for the ring
    const int64_t full = (int64_t)kSms * kBound<Tm, PASS>;
    if constexpr (PASS == FWD || PASS == BWD) {
      const int64_t blocks = p.team_items ? (p.items + Tm::TEAMS - 1) / Tm::TEAMS : p.items;
      const int64_t grid = std::min(blocks, full);
      if constexpr (PASS == FWD) *e = launch_ring(k_norm_fwd<T, Tm>, raised, grid, Tm::THREADS, bytes * p.stages, p, st);
      else *e = launch_ring(k_norm_bwd<T, Tm>, raised, grid, Tm::THREADS, bytes * p.stages, p, st);
    } else {
      const int64_t grid = std::min((p.rows + Tm::TEAMS - 1) / Tm::TEAMS, full);
      set_loop(&p, p.rows, grid * Tm::TEAMS);
      if constexpr (PASS == ROW_FWD)
        *e = launch_ring(k_rowmod_fwd<T, P, Tm>, raised, grid, Tm::THREADS, bytes * p.stages, p, st);
      else *e = launch_ring(k_rowmod_bwd<T, P, Tm>, raised, grid, Tm::THREADS, bytes * p.stages, p, st);
    }
    return true;
  }
  return false;
}

template <typename T, typename P, int E, Pass PASS>
bool launch_pass(const NormArgs& p, cudaStream_t st, cudaError_t* e) {
  const Tier t = tier_of(p.width, PASS, dense_rows(p.rows, E * sizeof(T) == 16), sizeof(T));
  return launch_tier<T, P, E, PASS, 8, 8>(t, p, st, e) || launch_tier<T, P, E, PASS, 8, 16>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 8, 24>(t, p, st, e) || launch_tier<T, P, E, PASS, 16, 16>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 16, 24>(t, p, st, e) || launch_tier<T, P, E, PASS, 32, 8>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 32, 16>(t, p, st, e) || launch_tier<T, P, E, PASS, 64, 16>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 128, 16>(t, p, st, e) || launch_tier<T, P, E, PASS, 256, 16>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 512, 16>(t, p, st, e) || launch_tier<T, P, E, PASS, 1024, 16>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 32, 24>(t, p, st, e) || launch_tier<T, P, E, PASS, 64, 24>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 128, 24>(t, p, st, e) || launch_tier<T, P, E, PASS, 256, 24>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 512, 24>(t, p, st, e) || launch_tier<T, P, E, PASS, 256, 32>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 512, 32>(t, p, st, e) || launch_tier<T, P, E, PASS, 64, 12>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 128, 12>(t, p, st, e) || launch_tier<T, P, E, PASS, 256, 12>(t, p, st, e) ||
         launch_tier<T, P, E, PASS, 512, 12>(t, p, st, e);
}
template <typename T, typename P, int E>
bool launch_rows_mod(const NormArgs& p, bool backward, cudaStream_t st, cudaError_t* e) {
  return backward ? launch_pass<T, P, E, ROW_BWD>(p, st, e) : launch_pass<T, P, E, ROW_FWD>(p, st, e);
}

template <typename T, int E>
cudaError_t launch_items(const NormArgs& p, bool backward, cudaStream_t st) {
  cudaError_t e = cudaErrorInvalidValue;
  if (backward) launch_pass<T, T, E, BWD>(p, st, &e);
  else launch_pass<T, T, E, FWD>(p, st, &e);
  return e;
}

// A modulation row per row of x: the modulation in the ring, if two stages of it fit (false: no). bf16
// beside fp16 goes without.
template <typename T, int E>
bool launch_modulated(const NormArgs& p, bool backward, cudaStream_t st, cudaError_t* e) {
  constexpr bool any = std::is_same<T, float>::value;
  if (p.p_type == LEWM_TYPE_F32) return launch_rows_mod<T, float, E>(p, backward, st, e);
  if constexpr (any || std::is_same<T, __nv_bfloat16>::value)
    if (p.p_type == LEWM_TYPE_BF16) return launch_rows_mod<T, __nv_bfloat16, E>(p, backward, st, e);
  if constexpr (any || std::is_same<T, __half>::value)
    if (p.p_type == LEWM_TYPE_F16) return launch_rows_mod<T, __half, E>(p, backward, st, e);
  return false;
}

template <typename T, int E>
cudaError_t launch_wide(const NormArgs& p, bool backward, cudaStream_t st) {
  const dim3 rows_grid((unsigned)std::min<int64_t>(p.rows, kSms * (2048 / kWideThreads)));
  if (!backward) return launch_k(k_norm_fwd_wide<T, E>, rows_grid, dim3(kWideThreads), 0, st, p);
  if (p.out) {
    const cudaError_t e = launch_k(k_norm_dx_wide<T, E>, rows_grid, dim3(kWideThreads), 0, st, p);
    if (e != cudaSuccess) return e;
  }
  if (!p.da && !p.db) return cudaSuccess;
  const dim3 grid((unsigned)((p.width + 256 * E - 1) / (256 * E)), (unsigned)std::min<int64_t>(p.items, 65535));
  return launch_k(k_norm_sums_wide<T, E>, grid, dim3(256), 0, st, p);
}

}  // namespace

template <typename T>
cudaError_t launch_norm_rows(const NormArgs& p, bool wide, bool backward, int vec, cudaStream_t st) {
  constexpr int E16 = 16 / sizeof(T), E8 = 8 / sizeof(T);
  if (p.one_plus && p.group == 1 && p.width * (int)sizeof(T) <= kMaxRowBytes) {
    cudaError_t e = cudaSuccess;
    const bool done = vec == 16 ? launch_modulated<T, E16>(p, backward, st, &e)
                                : launch_modulated<T, 1>(p, backward, st, &e);
    if (done) return e;
  }
  if (wide) return vec == 16 ? launch_wide<T, E16>(p, backward, st) : launch_wide<T, 1>(p, backward, st);
  // 12 values are no whole 16-byte vectors of 16-bit elements.
  const bool halves = backward && tier_of(p.width, BWD, dense_rows(p.rows, vec == 16), sizeof(T)).n % E16 != 0;
  if (vec == 16 && !halves) return launch_items<T, E16>(p, backward, st);
  if (vec == 16) return launch_items<T, E8>(p, backward, st);
  if (vec == 8) return launch_items<T, E8>(p, backward, st);
  if constexpr (sizeof(T) == 2)
    if (vec == 4) return launch_items<T, 2>(p, backward, st);
  return launch_items<T, 1>(p, backward, st);
}

}  // namespace lewm
