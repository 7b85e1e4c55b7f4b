// Distillation from a teacher's top logits. A row has V student logits s and K teacher entries (id_k, t_k); entries whose id lies outside
// [0, V) are absent. With p = softmax(t / T) over the present entries and q = softmax(s / T) over the vocabulary
//
//   loss = T^2 sum_k p_k (log p_k - log q_id_k),     d loss / d s_v = T (q_v - sum over the entries of v of p_k)
//
// A row without a present entry (or whose present entries are all -inf) has loss and gradient 0, whatever its logits hold.
//
// What bounds it is memory: the logits are read once (and the gradient written once); an element takes one exponential in a pass
// over the logits, two where loss and gradient are made together. In that case a row stays in registers between the sum of its exponentials and the
// gradient: 512 threads of eight 16-byte pieces hold 32768 bf16 logits; of longer rows a cluster of up to eight CTAs takes a share each, and the
// shares' (maximum, sum) meet through distributed shared memory. Rows too long for that too are read again.
//
// Maxima and sums are fp32, per thread first, then in a fixed order: results do not depend on the schedule. Entries of the same id add up.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common/bounds.cuh"
#include "common/host_util.h"
#include "common/sm100.cuh"

RA_BOUNDS_TRANSLATION_UNIT()

namespace ra {
namespace distill {

namespace cg = cooperative_groups;

constexpr int MAX_THREADS = 512;
constexpr int HELD = 8;        // 16-byte pieces of a row a thread holds
constexpr int MAX_SHARES = 8;  // CTAs of a cluster
constexpr int MAX_K = 2048;

struct Params {
  const void* logits;   // (rows, V), distance ld
  void* grad;           // (rows, V), distance ldg
  long long ld, ldg;
  const void* ids;      // (rows, K) 32 or 64 bits
  const void* teacher;  // (rows, K) bf16 or fp32
  long long ld_ids, ld_t;
  int ids64, teacher_f32;
  int V, K, shares;
  float per_t;          // log2(e) / T
  float t;              // T
  float* loss;          // (rows)
  float2* stats;        // (rows): largest logit * log2(e) / T, 1 / sum of exponentials, 0 for a row without entries
  float grad_scale;     // of T (q - p)
  const float* dloss;   // backward: gradient of the rows' losses, distance dloss_s (0: one number), times *per_row if that is not null
  int dloss_s;
  const float* per_row;
};

template <typename T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
  static constexpr int PER = 8;
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __uint_as_float(w[e] << 16);
      f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <> struct Elem<float> {
  static constexpr int PER = 4;
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// A row cut into 16-byte pieces of its address range: piece j holds elements j * PER - phase .. + PER - 1 of it, as far as they are of the row.
template <typename T>
struct Row {
  static constexpr int PER = Elem<T>::PER;
  const T* base;
  int V, phase, pieces;
  __device__ __forceinline__ Row(const T* b, int v)
      : base(b), V(v), phase(static_cast<int>((reinterpret_cast<uintptr_t>(b) & 15) / sizeof(T))), pieces((v + phase + PER - 1) / PER) {}
  __device__ __forceinline__ int first(int j) const { return j * PER - phase; }
  __device__ __forceinline__ bool whole(int j) const { return first(j) >= 0 && first(j) + PER <= V; }
  __device__ __forceinline__ uint4 load(int j) const {  // -inf beyond the row's ends
    if (whole(j)) return *reinterpret_cast<const uint4*>(base + first(j));
    float f[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int i = first(j) + e;
      f[e] = i >= 0 && i < V ? Elem<T>::get(base + i) : -INFINITY;
    }
    return Elem<T>::pack(f);
  }
};

template <typename T>
__device__ __forceinline__ void store_piece(T* out, bool same_phase, const Row<T>& row, int j, const float* f) {
  constexpr int PER = Elem<T>::PER;
  if (same_phase && row.whole(j)) {
    if (RA_IN_BOUNDS(row.first(j), PER, row.V, kTagDistill)) *reinterpret_cast<uint4*>(out + row.first(j)) = Elem<T>::pack(f);
    return;
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = row.first(j) + e;
    if (i >= 0 && i < row.V) Elem<T>::put(out + i, f[e]);
  }
}

__device__ __forceinline__ float2 join(float2 a, float2 b) {  // (maximum, sum of exponentials), log2 domain
  const float m = fmaxf(a.x, b.x), mu = m == -INFINITY ? 0.f : m;
  return make_float2(m, a.y * exp2_approx(a.x - mu) + b.y * exp2_approx(b.x - mu));
}
__device__ __forceinline__ float2 join_warp(float2 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
  return v;
}

// The entries of a row in shared memory: K ids (-1: absent), their weights p and the student's logits there. Called by one warp; returns (in every lane)
// the largest present teacher logit (log2 domain) and the sum of the exponentials, 0 where nothing is present.
struct Entries {
  int* id;
  float* p;
  float* s;
};
__device__ __forceinline__ Entries entries_in(uint8_t* smem, int K) {
  const int n = (K + 3) / 4 * 4;
  return Entries{reinterpret_cast<int*>(smem), reinterpret_cast<float*>(smem) + n, reinterpret_cast<float*>(smem) + 2 * n};
}
template <typename T>
__device__ __forceinline__ float2 gather_entries(const Params& p, long long r, const T* logits, Entries en, int lane) {
  float2 all = make_float2(-INFINITY, 0.f);
  const int padded = (p.K + 3) / 4 * 4;
  for (int k = lane; k < padded; k += 32) {
    long long id = -1;
    float t = -INFINITY, s = 0.f;
    if (k < p.K) {
      id = p.ids64 ? static_cast<const long long*>(p.ids)[r * p.ld_ids + k] : static_cast<const int*>(p.ids)[r * p.ld_ids + k];
      if (id < 0 || id >= p.V) id = -1;
      if (id >= 0) {
        t = (p.teacher_f32 ? static_cast<const float*>(p.teacher)[r * p.ld_t + k]
                           : __bfloat162float(static_cast<const __nv_bfloat16*>(p.teacher)[r * p.ld_t + k])) * p.per_t;
        s = Elem<T>::get(logits + id);
      }
    }
    en.id[k] = static_cast<int>(id);
    en.p[k] = t;
    en.s[k] = s;
    all = join(all, make_float2(t, id >= 0 ? (t == t ? 1.f : t) : 0.f));
  }
  all = join_warp(all);
  __syncwarp();
  const float inv = all.y > 0.f ? 1.f / all.y : (all.y == all.y ? 0.f : all.y);
  const float mu = all.x == -INFINITY ? 0.f : all.x;
  for (int k = lane; k < padded; k += 32) en.p[k] = en.id[k] >= 0 ? exp2_approx(en.p[k] - mu) * inv : 0.f;
  __syncwarp();
  return all;
}

// sum of p over the entries of entry k's id
__device__ __forceinline__ float weight_of(const Entries& en, int K, int id) {
  float w = 0.f;
  const int4* ids = reinterpret_cast<const int4*>(en.id);
  const float4* ps = reinterpret_cast<const float4*>(en.p);
  for (int j = 0; j < (K + 3) / 4; ++j) {
    const int4 i4 = ids[j];
    const float4 p4 = ps[j];
    w += (i4.x == id ? p4.x : 0.f) + (i4.y == id ? p4.y : 0.f) + (i4.z == id ? p4.z : 0.f) + (i4.w == id ? p4.w : 0.f);
  }
  return w;
}

// Loss and stats of a row, with GRAD also its gradient. grid (rows * shares), clusters of `shares`.
template <typename T, bool GRAD, bool HOLD>
__global__ void __launch_bounds__(MAX_THREADS) distill_row_kernel(const Params p) {
  constexpr int PER = Elem<T>::PER;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 red[MAX_THREADS / 32];
  __shared__ float2 mine, teacher;
  const long long r = blockIdx.x / p.shares;
  const int share = blockIdx.x - static_cast<int>(r) * p.shares;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const T* logits = static_cast<const T*>(p.logits) + r * p.ld;
  const Row<T> row(logits, p.V);
  const int per = (row.pieces + p.shares - 1) / p.shares;
  const int j0 = share * per, j1 = min(row.pieces, j0 + per);
  const Entries en = entries_in(smem, p.K);

  uint4 held[HOLD ? HELD : 1];
  if (HOLD) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const int j = j0 + static_cast<int>(threadIdx.x) + i * static_cast<int>(blockDim.x);
      if (j < j1) held[i] = row.load(j);
    }
  }
  if (warp == 0) {
    const float2 t = gather_entries(p, r, logits, en, lane);
    if (lane == 0) teacher = t;
  }
  // ---- largest logit and sum of exponentials
  float2 own = make_float2(-INFINITY, 0.f);
  auto add = [&](const uint4* u, int n) {  // n pieces at most HELD
    float m = own.x;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      if (i >= n) break;
      float f[PER];
      Elem<T>::unpack(u[i], f);
#pragma unroll
      for (int e = 0; e < PER; ++e) m = fmaxf(m, f[e] * p.per_t);
    }
    const float mu = m == -INFINITY ? 0.f : m;
    float s = own.y * exp2_approx(own.x - mu);
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      if (i >= n) break;
      float f[PER];
      Elem<T>::unpack(u[i], f);
#pragma unroll
      for (int e = 0; e < PER; ++e) s += exp2_approx(fmaf(f[e], p.per_t, -mu));
    }
    own = make_float2(m, s);
  };
  const int first = j0 + static_cast<int>(threadIdx.x), step = static_cast<int>(blockDim.x);
  const int count = first < j1 ? (j1 - first + step - 1) / step : 0;  // pieces of this thread
  if (HOLD) {
    add(held, count);
  } else {
    for (int i = 0; i < count; i += HELD) {
      uint4 u[HELD];
      const int n = min(HELD, count - i);
#pragma unroll
      for (int e = 0; e < HELD; ++e)
        if (e < n) u[e] = row.load(first + (i + e) * step);
      add(u, n);
    }
  }
  own = join_warp(own);
  if (lane == 0) red[warp] = own;
  __syncthreads();
  float2 all = red[0];
  for (int w = 1; w < warps; ++w) all = join(all, red[w]);
  if (p.shares > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x == 0) mine = all;
    cluster.sync();
    all = *cluster.map_shared_rank(&mine, 0);
    for (int c = 1; c < p.shares; ++c) all = join(all, *cluster.map_shared_rank(&mine, c));
  }
  const bool there = teacher.y != 0.f;
  const float inv = there ? 1.f / all.y : 0.f;
  // ---- loss
  if (share == 0 && warp == 0) {
    float sum = 0.f;
    for (int k = lane; k < p.K; k += 32) {
      const float w = en.p[k];
      // log2 p less log2 q; an entry of weight 0 has no part in it
      if (w != 0.f) sum += w * ((log2f(w) + log2f(all.y)) - fmaf(en.s[k], p.per_t, -all.x));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      p.loss[r] = there ? p.t * p.t * 0.6931471805599453f * sum : 0.f;
      if (p.stats) p.stats[r] = make_float2(all.x, inv);
    }
  }
  if (GRAD) {
    T* grad = static_cast<T*>(p.grad) + r * p.ldg;
    const bool same = ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(logits)) & 15) == 0;
    const float scale = p.grad_scale * p.t, mul = scale * inv;
    auto write = [&](const uint4& u, int j) {
      float f[PER];
      Elem<T>::unpack(u, f);
#pragma unroll
      for (int e = 0; e < PER; ++e) f[e] = there ? exp2_approx(fmaf(f[e], p.per_t, -all.x)) * mul : 0.f;
      store_piece<T>(grad, same, row, j, f);
    };
    if (HOLD) {
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (i < count) write(held[i], first + i * step);
    } else {
      for (int i = 0; i < count; ++i) write(row.load(first + i * step), first + i * step);
    }
    __syncthreads();
    // the entries of this share, over what was written there
    if (there) {
      for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
        const int id = en.id[k], j = (id + row.phase) / PER;
        if (id < 0 || j < j0 || j >= j1) continue;
        Elem<T>::put(grad + id, (exp2_approx(fmaf(en.s[k], p.per_t, -all.x)) * inv - weight_of(en, p.K, id)) * scale);
      }
    }
  }
  if (p.shares > 1) cg::this_cluster().sync();  // nobody leaves while its sums are being read
}

// Gradient of the logits from that of the losses: grid (rows, shares).
template <typename T>
__global__ void __launch_bounds__(MAX_THREADS) distill_bwd_kernel(const Params p) {
  constexpr int PER = Elem<T>::PER;
  extern __shared__ __align__(16) uint8_t smem[];
  const long long r = blockIdx.x;
  const T* logits = static_cast<const T*>(p.logits) + r * p.ld;
  T* grad = static_cast<T*>(p.grad) + r * p.ldg;
  const Row<T> row(logits, p.V);
  const bool same = ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(logits)) & 15) == 0;
  const int per = (row.pieces + p.shares - 1) / p.shares;
  const int j0 = static_cast<int>(blockIdx.y) * per, j1 = min(row.pieces, j0 + per);
  const Entries en = entries_in(smem, p.K);
  const float2 st = p.stats[r];
  const bool there = st.y != 0.f;
  const float scale = p.dloss[r * p.dloss_s] * (p.per_row ? *p.per_row : 1.f) * p.t, mul = scale * st.y;
  if (threadIdx.x < 32 && there) gather_entries(p, r, logits, en, threadIdx.x);
  const int step = blockDim.x;
  int j = j0 + static_cast<int>(threadIdx.x);
  auto write = [&](const uint4& u, int at) {
    float f[PER];
    Elem<T>::unpack(u, f);
#pragma unroll
    for (int e = 0; e < PER; ++e) f[e] = there ? exp2_approx(fmaf(f[e], p.per_t, -st.x)) * mul : 0.f;
    store_piece<T>(grad, same, row, at, f);
  };
  for (; j + 3 * step < j1; j += 4 * step) {
    uint4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = row.load(j + i * step);
#pragma unroll
    for (int i = 0; i < 4; ++i) write(u[i], j + i * step);
  }
  for (; j < j1; j += step) write(row.load(j), j);
  __syncthreads();
  if (!there) return;
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    const int id = en.id[k], at = (id + row.phase) / PER;
    if (id < 0 || at < j0 || at >= j1) continue;
    Elem<T>::put(grad + id, (exp2_approx(fmaf(en.s[k], p.per_t, -st.x)) * st.y - weight_of(en, p.K, id)) * scale);
  }
}

// total = sum of the losses, or with `mean` their mean over the rows that have entries; per_row = what a row's loss was multiplied by. One CTA.
__global__ void __launch_bounds__(1024) distill_reduce_kernel(const float* __restrict__ loss, const float2* __restrict__ stats, long long rows, int mean,
                                                              float* __restrict__ total, float* __restrict__ per_row) {
  __shared__ double red[32];
  __shared__ int cnt[32];
  double s = 0.0;
  int n = 0;
  for (long long i = threadIdx.x; i < rows; i += 1024) {
    s += loss[i];
    n += stats[i].y != 0.f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = s;
    cnt[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) {
      s += red[w];
      n += cnt[w];
    }
    const double per = mean ? 1.0 / (n > 0 ? n : 1) : 1.0;
    *total = static_cast<float>(s * per);
    *per_row = static_cast<float>(per);
  }
}

}  // namespace distill
}  // namespace ra

struct RaDistillArgs {
  const void* logits; long long ld;
  void* grad; long long ldg;             // null: the loss alone
  const void* ids; long long ld_ids;
  const void* teacher; long long ld_t;
  int f32, ids64, teacher_f32;           // types: of the logits and the gradient, ids, teacher
  long long rows;
  int V, K;
  float temperature, grad_scale;
  float* loss;
  void* stats;                           // (rows, 2) fp32, or null; the backward reads it
  const float* dloss; int dloss_s; const float* per_row;  // backward
  void* stream;
};

namespace {
int to_params(const RaDistillArgs* a, ra::distill::Params& p) {
  using namespace ra;
  const int size = a->f32 ? 4 : 2;
  if (a->rows < 1 || a->V < 1 || a->V > (1 << 30) || a->K < 1 || a->K > distill::MAX_K || !(a->temperature > 0.f) || !a->logits || !a->ids || !a->teacher ||
      (reinterpret_cast<uintptr_t>(a->logits) % size) || (reinterpret_cast<uintptr_t>(a->grad) % size)) {
    set_error("distill: bad shape (1 to 2048 teacher entries, a positive temperature)");
    return kHostBadArg;
  }
  p = distill::Params{a->logits, a->grad, a->ld, a->ldg, a->ids, a->teacher, a->ld_ids, a->ld_t, a->ids64, a->teacher_f32, a->V, a->K, 1,
                      1.4426950408889634f / a->temperature, a->temperature, a->loss, static_cast<float2*>(a->stats), a->grad_scale, a->dloss,
                      a->dloss_s, a->per_row};
  return kHostOk;
}
size_t entry_bytes(int K) { return static_cast<size_t>((K + 3) / 4 * 4) * 12; }
}  // namespace

// Loss (and stats, and with `grad` the gradient times grad_scale, which may overwrite the logits) of every row.
extern "C" int ra_distill(const RaDistillArgs* a) {
  using namespace ra;
  using namespace ra::distill;
  Params p;
  if (int rc = to_params(a, p)) return rc;
  if (!a->loss) {
    set_error("distill: no room for the losses");
    return kHostBadArg;
  }
  const int per16 = a->f32 ? 4 : 8;
  const int pieces = (a->V + 2 * per16 - 2) / per16;  // at most, whatever the row's alignment
  constexpr int held = HELD * MAX_THREADS;
  // as few CTAs a row as hold it; more where there are too few rows for the SMs and enough of a row to share
  while (p.shares < MAX_SHARES && (pieces > p.shares * held || (a->rows * p.shares < sm_count() && pieces >= p.shares * 2 * 1024))) p.shares *= 2;
  const int share = (pieces + p.shares - 1) / p.shares;
  const bool hold = share <= held;
  int threads = ((hold ? (share + HELD - 1) / HELD : MAX_THREADS) + 31) / 32 * 32;
  if (threads < 64) threads = 64;
  if (a->rows * p.shares > 0x7fffffffll) {
    set_error("distill: too many rows");
    return kHostTooLarge;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a->rows * p.shares));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = entry_bytes(a->K);
  cfg.stream = static_cast<cudaStream_t>(a->stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.shares;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.shares > 1 ? 1 : 0;
  auto kern = a->f32 ? (a->grad ? (hold ? distill_row_kernel<float, true, true> : distill_row_kernel<float, true, false>)
                                : (hold ? distill_row_kernel<float, false, true> : distill_row_kernel<float, false, false>))
                     : (a->grad ? (hold ? distill_row_kernel<__nv_bfloat16, true, true> : distill_row_kernel<__nv_bfloat16, true, false>)
                                : (hold ? distill_row_kernel<__nv_bfloat16, false, true> : distill_row_kernel<__nv_bfloat16, false, false>));
  cudaLaunchKernelEx(&cfg, kern, p);
  return check_launch("distill_row_kernel");
}

// grad <- the gradient of every row's logits, from `dloss` and the stats that ra_distill left.
extern "C" int ra_distill_bwd(const RaDistillArgs* a) {
  using namespace ra;
  using namespace ra::distill;
  Params p;
  if (int rc = to_params(a, p)) return rc;
  if (!a->grad || !a->stats || !a->dloss || a->rows > 0x7fffffffll || a->grad == a->logits) {
    set_error("distill_bwd: no gradient, stats or room for the result");
    return kHostBadArg;
  }
  const int per16 = a->f32 ? 4 : 8;
  const int pieces = (a->V + 2 * per16 - 2) / per16;
  int threads = (pieces / 4 + 31) / 32 * 32;
  threads = threads < 64 ? 64 : (threads > MAX_THREADS ? MAX_THREADS : threads);
  while (p.shares < 64 && (pieces > p.shares * threads * 16 || (a->rows * p.shares < 2 * sm_count() && pieces > p.shares * threads * 4))) p.shares *= 2;
  auto kern = a->f32 ? distill_bwd_kernel<float> : distill_bwd_kernel<__nv_bfloat16>;
  kern<<<dim3(static_cast<unsigned>(a->rows), p.shares), threads, entry_bytes(a->K), static_cast<cudaStream_t>(a->stream)>>>(p);
  return check_launch("distill_bwd_kernel");
}

// total <- the losses' sum, or with `mean` their mean over the rows that have entries; per_row <- what a row's loss was multiplied by.
extern "C" int ra_distill_reduce(const float* loss, const void* stats, long long rows, int mean, float* total, float* per_row, void* stream) {
  ra::distill::distill_reduce_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(loss, static_cast<const float2*>(stats), rows, mean, total,
                                                                                          per_row);
  return ra::check_launch("distill_reduce_kernel");
}

RA_PACKED(ra_distill_reduce)
