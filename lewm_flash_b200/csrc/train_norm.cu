// Layer norm and adaptive layer norm: how rows are cut into work, the reduction of partial sums, and
// the C ABI. The kernels: train_norm.cuh.
#include <algorithm>
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "train_norm.cuh"

namespace lewm {

extern template cudaError_t launch_norm_rows<float>(const NormArgs&, bool, bool, int, cudaStream_t);
extern template cudaError_t launch_norm_rows<__nv_bfloat16>(const NormArgs&, bool, bool, int, cudaStream_t);
extern template cudaError_t launch_norm_rows<__half>(const NormArgs&, bool, bool, int, cudaStream_t);

namespace {

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
      constexpr int B = 12;  // loads in flight
      for (int i = run; i < p.split; i += B * R) {
        V v[B];
#pragma unroll
        for (int k = 0; k < B; ++k)
          if (i + k * R < p.split) v[k] = *reinterpret_cast<const V*>(w + (i + k * R) * stride);
#pragma unroll
        for (int k = 0; k < B; ++k)
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

// Items per group: the fewest that come within 5% of the least rounds of rows that one of `full`
// resident blocks goes through, where an item costs about four rounds beside its rows (its loads from
// cold) and a backward's second launch eight. 340 groups of 139 rows on 296 blocks run in 2 waves of 139
// rounds undivided, 3 of 70 in halves.
int64_t best_split(int64_t groups, int64_t group, int64_t teams, int64_t full, bool backward) {
  const int64_t most = (group + teams - 1) / teams;
  auto cost = [&](int64_t split) {
    const int64_t waves = (groups * split + full - 1) / full, rounds = (group + split * teams - 1) / (split * teams);
    return waves * (rounds + 4) + (backward && split > 1 ? 8 : 0);
  };
  auto clamp = [&](int64_t split) { return std::max<int64_t>(1, std::min(split, most)); };
  int64_t best = 1;
  for (int64_t waves = 1; waves <= 8; ++waves) {
    const int64_t split = clamp(waves * full / groups);
    if (cost(split) < cost(best)) best = split;
  }
  for (int64_t waves = 1; waves <= 8; ++waves) {
    const int64_t split = clamp(waves * full / groups);
    if (split < best && cost(split) * 100 <= cost(best) * 105) best = split;
  }
  return best;
}

// Whether a team takes whole groups rather than a block (`split` items each): by the rounds of rows that
// each way goes through, where an item of the block's costs about four rounds beside its rows, six in the
// backward (it adds up its teams), and a team's four. A round of teams on rows far apart is dearer, by 6/5
// with 16-bit rows and 5/3 with float32, measured over widths of 64 to 1024, groups of 3 to 60 rows and 300
// to 19000 groups: 4700 groups of 3 x 192 bf16 forward and backward 37 and 57 us by blocks, 5.5 and 8.4 by
// teams; 28 x 128: 30 and 63, 20 and 25; 2400 of 60 x 640: 80 and 129, 102 and 131.
bool teams_pay(int64_t groups, int64_t group, int64_t teams, int64_t full, int64_t split, int size, bool backward) {
  if (group > 64) return false;
  const int64_t by_team = (groups + full * teams - 1) / (full * teams) * (group + 4);
  const int64_t by_block = (groups * split + full - 1) / full *
                               ((group + split * teams - 1) / (split * teams) + (backward ? 6 : 4)) +
                           (backward && split > 1 ? 8 : 0);
  return size == 2 ? by_team * 6 < by_block * 5 : by_team * 5 < by_block * 3;
}

// How rows are cut into items; the same function sizes the workspace.
void cut_items(NormArgs* p, int x_type, bool backward, int vec) {
  const int64_t groups = p->rows / p->group;
  int64_t teams = 1;
  p->team_items = 0;
  if (is_wide(*p, x_type, backward)) {
    // Column blocks x items: split each group until the grid has about 4 blocks per SM.
    const int64_t cols = (p->width + 2047) / 2048;
    const int64_t want = (int64_t)kSms * 4 / std::max<int64_t>(1, cols * groups);
    p->split = (int)std::max<int64_t>(1, std::min<int64_t>(want, p->group));
  } else {
    const Pass pass = backward ? BWD : FWD;
    const Tier t = tier_of(p->width, pass, dense_rows(p->rows, vec == 16), (int)type_size(x_type));
    teams = t.teams();
    const int64_t full = (int64_t)kSms * bound_blocks(t.tpr, t.n, pass);
    const int64_t split = best_split(groups, p->group, teams, full, backward);
    p->team_items = teams_pay(groups, p->group, teams, full, split, (int)type_size(x_type), backward);
    p->split = p->team_items ? 1 : (int)split;
  }
  p->items = groups * p->split;
  set_loop(p, p->group, p->team_items ? 1 : p->split * teams);
}

size_t workspace_bytes(const NormArgs& p) {
  return p.split > 1 ? (size_t)p.items * 2 * (size_t)p.width * sizeof(float) : 0;
}

// Bytes of the vectors that rows move in: 16, 8, 4 or an element's. Sets p_vec.
int vector_bytes(NormArgs* q, int x_type, bool backward) {
  NormArgs& p = *q;
  const int64_t size = type_size(x_type), ps = type_size(p.p_type);
  auto aligned = [](const void* q, int64_t stride_bytes, int64_t to) {
    return !q || ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)stride_bytes) & (uintptr_t)(to - 1)) == 0;
  };
  for (int vec = 16; vec > size; vec /= 2) {
    if (!aligned(p.x, p.x_stride * size, vec) || !aligned(p.out, p.width * size, vec) || (p.width * size) % vec ||
        (backward && !aligned(p.dy, p.dy_stride * size, vec)))
      continue;
    // A vector's parameters as accesses of up to 16 bytes.
    const int64_t to = std::min<int64_t>(16, vec / size * ps);
    p.p_vec = aligned(p.a, p.a_stride * ps, to) && aligned(p.b, p.b_stride * ps, to) &&
              aligned(p.da, p.width * ps, to) && aligned(p.db, p.width * ps, to) && (p.width * ps) % to == 0;
    if (p.one_plus && p.group == 1 && !p.p_vec) break;  // the ring moves both the same way
    return vec;
  }
  p.p_vec = 0;
  return (int)size;
}

cudaError_t launch_norm(const NormArgs& p, int x_type, bool backward, int vec, cudaStream_t st) {
  const bool wide = is_wide(p, x_type, backward);
  cudaError_t e = x_type == LEWM_TYPE_F32    ? launch_norm_rows<float>(p, wide, backward, vec, st)
                  : x_type == LEWM_TYPE_BF16 ? launch_norm_rows<__nv_bfloat16>(p, wide, backward, vec, st)
                                             : launch_norm_rows<__half>(p, wide, backward, vec, st);
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

// Whether pointers lie on whole elements (of 4-byte floats for statistics).
bool on_elements(int type, std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if (reinterpret_cast<uintptr_t>(q) % (uintptr_t)type_size(type)) return false;
  return true;
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
  cut_items(&p, desc->x_type, true, 16);
  const size_t bytes = workspace_bytes(p);
  cut_items(&p, desc->x_type, true, 1);
  return std::max(bytes, workspace_bytes(p));  // whichever way the tensors lie
}

extern "C" lewm_status lewm_norm_forward(const lewm_norm_desc* desc, const void* x, const void* a, const void* b,
                                         void* y, float* stats, int32_t device, void* stream) {
  NormArgs p;
  const lewm_status s = norm_args(desc, &p);
  if (s != LEWM_OK) return s;
  if (p.rows == 0) return LEWM_OK;
  if (!x || !y) return norm_fail(LEWM_INVALID_ARG, "x and y must be non-NULL");
  if (p.one_plus && (!a || !b)) return norm_fail(LEWM_INVALID_ARG, "scale and shift must be non-NULL");
  if (!on_elements(desc->x_type, {x, y}) || !on_elements(desc->p_type, {a, b}) || !on_elements(LEWM_TYPE_F32, {stats}))
    return norm_fail(LEWM_INVALID_ARG, "a pointer is not aligned to its element type");
  NormDevice nd(device);
  if (nd.err != cudaSuccess)
    return norm_fail(LEWM_CUDA_ERROR, "cudaSetDevice(%d): %s", device, cudaGetErrorString(nd.err));
  p.x = x;
  p.a = a;
  p.b = b;
  p.out = y;
  p.stats = stats;
  const int vec = vector_bytes(&p, desc->x_type, false);
  cut_items(&p, desc->x_type, false, vec);
  const cudaError_t e = launch_norm(p, desc->x_type, false, vec, static_cast<cudaStream_t>(stream));
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
  if (!on_elements(desc->x_type, {dy, x, dx}) || !on_elements(desc->p_type, {a, da, db}) ||
      !on_elements(LEWM_TYPE_F32, {stats}))
    return norm_fail(LEWM_INVALID_ARG, "a pointer is not aligned to its element type");
  p.x = x;
  p.dy = dy;
  p.dy_stride = dy_stride;
  p.a = a;
  p.out = dx;
  p.da = da;
  p.db = db;
  p.stats = const_cast<float*>(stats);
  p.ws = static_cast<float*>(workspace);
  const int vec = vector_bytes(&p, desc->x_type, true);
  cut_items(&p, desc->x_type, true, vec);
  if ((da || db) && workspace_bytes_given < workspace_bytes(p))
    return norm_fail(LEWM_INVALID_ARG, "workspace of %zu bytes, needs %zu", workspace_bytes_given, workspace_bytes(p));
  if ((da || db) && p.split > 1 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16))
    return norm_fail(LEWM_INVALID_ARG, "workspace must be non-NULL and 16-byte aligned");
  NormDevice nd(device);
  if (nd.err != cudaSuccess)
    return norm_fail(LEWM_CUDA_ERROR, "cudaSetDevice(%d): %s", device, cudaGetErrorString(nd.err));
  const cudaError_t e = launch_norm(p, desc->x_type, true, vec, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return norm_fail(LEWM_CUDA_ERROR, "norm backward launch: %s", cudaGetErrorString(e));
  return LEWM_OK;
}
