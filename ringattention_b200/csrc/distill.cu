// Distillation from a teacher's top logits. A row has V student logits s and K teacher entries (id_k, t_k); entries whose id lies outside
// [0, V) are absent. With p = softmax(t / T) over the present entries and q = softmax(s / T) over the vocabulary
//
//   loss = T^2 sum_k p_k (log p_k - log q_id_k),     d loss / d s_v = T (q_v - sum over the entries of v of p_k)
//
// A row without a present entry (or whose present entries are all -inf) has loss and gradient 0, whatever its logits hold.
//
// One kernel, a CTA for each row: the sum of the row's exponentials, and the gradient, which reads the row again (it is in the L2 by then) and takes
// each exponential once more; the backward of the loss alone is the second half. What bounds it is memory (the logits in, the gradient
// out), with the exponentials next: 4096 rows of 32000 in bf16 in 47 us for the sums among launches of its kind (5.5 TB/s; 55 us alone), 88 to 97 us with
// the gradient (6.0 to 5.4), of which the exponentials alone would take 29 and 58. The sums are furthest from memory's rate: nothing of a row is in
// flight at the barrier behind the last one's end (8192 rows of 10000: 35 us, 4.7 TB/s). What that takes:
//  - CTAs of 256 threads, four on an SM, each in a phase of its own: one that waits for its row or its barrier leaves the SM to the others. Persistent
//    CTAs that bring in the next row meanwhile (cp.async or bulk copies, the row's exponentials kept in registers, clusters for long rows) were all
//    slower, 71 to 80 us and 103 to 120: their warps are in the same phase, waiting or all taking exponentials.
//  - eight 16-byte loads of a thread in flight, without a branch between them: pieces behind the row's end are -inf, the pieces that its two ends cut are
//    two threads' work, apart.
//  - few instructions an element: the maximum on packed pairs, products and sums two at a time.
// A warp of its own has the teacher's entries: a chain of loads (ids, then the logits there) beside the sums, the loss and the search for repeated ids
// beside the gradient, and their gradients over the row's while that is in the L2. (The first warp with all of that: 108 us; a kernel of its own
// behind all rows: 15 us more.)
//
// Maxima and sums are fp32, per thread first, then in a fixed order: results do not depend on the schedule. Entries of the same id add up.
//
// At a high temperature p and q are nearly the same where the entries make up much of the vocabulary: the loss is T^2 times a sum of p log(p / q) that is of
// the order of 1 / T^2, so the 2^-22 or so that each logarithm is off by in 32 bits come out as T^2 2^-22 (0.02 at T = 300, all of the loss at
// 10^4), and likewise T (q - p). Such rows, of fewer logits than twice the entries, have a kernel in 64 bits from T = 4 on (distill_wide_kernel). With
// more logits than that q has half of its weight or more elsewhere once T is beyond the spread of the logits, and nothing cancels.
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

constexpr int MAX_THREADS = 512;
constexpr int HELD = 8;  // 16-byte pieces of a row that a thread asks for at a time
constexpr int MAX_K = 1024;

struct Params {
  const void* logits;   // (rows, V), distance ld
  void* grad;           // (rows, V), distance ldg
  long long ld, ldg;
  const void* ids;      // (rows, K) 32 or 64 bits
  const void* teacher;  // (rows, K) bf16 or fp32
  long long ld_ids, ld_t;
  int ids64, teacher_f32;
  int V, K;
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

// A row cut into 16-byte pieces of its address range: `first` elements before the whole ones, `pieces` of these, `last` behind them.
template <typename T>
struct Row {
  const T* base;
  int first, pieces, last;
  __device__ __forceinline__ Row(const T* b, int V) : base(b) {
    constexpr int PER = Elem<T>::PER;
    const int phase = static_cast<int>((reinterpret_cast<uintptr_t>(b) & 15) / sizeof(T));
    first = min(V, (PER - phase) % PER);
    pieces = (V - first) / PER;
    last = V - first - pieces * PER;
  }
  __device__ __forceinline__ const uint4* body() const { return reinterpret_cast<const uint4*>(base + first); }
  // an element of one of the two ends, -1: none. The threads of the first and the last warp have one each, if any.
  __device__ __forceinline__ int end_of(int tid, int threads) const {
    if (tid < first) return tid;
    const int k = tid - (threads - 32);
    return k >= 0 && k < last ? first + pieces * Elem<T>::PER + k : -1;
  }
};
template <typename T>
__device__ __forceinline__ uint4 no_piece() {
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}
__device__ __forceinline__ float largest(float m, const uint4& u, float) {
  return max3(max3(m, __uint_as_float(u.x), __uint_as_float(u.y)), __uint_as_float(u.z), __uint_as_float(u.w));
}
__device__ __forceinline__ float largest(float m, const uint4& u, __nv_bfloat16) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  const __nv_bfloat162 x = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return max3(m, __low2float(x), __high2float(x));
}

__device__ __forceinline__ float2 join(float2 a, float2 b) {  // (maximum, sum of exponentials), log2 domain
  const float m = fmaxf(a.x, b.x), mu = m == -INFINITY ? 0.f : m;
  return make_float2(m, a.y * exp2_approx(a.x - mu) + b.y * exp2_approx(b.x - mu));
}
// over the lanes of a warp, with one exponential a lane (joined pair by pair on the way it would be ten)
__device__ __forceinline__ float2 join_warp(float2 v) {
  float m = v.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = v.y * exp2_approx(v.x - (m == -INFINITY ? 0.f : m));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return make_float2(m, s);
}

// The entries of a row in shared memory: K ids (-1: absent), their weights p, the weights w of all entries of the same id, the student's
// logits there.
struct Entries {
  int* there;        // whether there are any (as far as they weigh something)
  int* id;
  float* p;
  float* w;
  float* s;
  uint32_t* again;   // a bit for each entry whose id another entry has too
  int* table;        // of ids, to find those
};
__host__ __device__ __forceinline__ int entry_words(int K) { return (K + 3) / 4 * 4; }
__host__ __device__ __forceinline__ int table_words(int K) {
  int n = 64;
  while (n < 2 * K) n *= 2;
  return n;
}
__host__ __device__ __forceinline__ int bit_words(int K) { return (K + 127) / 128 * 4; }
__host__ __device__ __forceinline__ size_t entry_smem(int K) {
  return 4 * (4 + 4 * static_cast<size_t>(entry_words(K)) + bit_words(K) + table_words(K));
}
__device__ __forceinline__ Entries entries_in(uint8_t* smem, int K) {
  const int n = entry_words(K);
  int* at = reinterpret_cast<int*>(smem);
  float* f = reinterpret_cast<float*>(at + 4 + n);
  return Entries{at, at + 4, f, f + n, f + 2 * n, reinterpret_cast<uint32_t*>(f + 3 * n), reinterpret_cast<int*>(f + 3 * n) + bit_words(K)};
}

// Three steps of a warp each, so that the first one's loads are under way beside the row's, and the last one's search beside the gradient's stores.
// 1: ids, teacher's logits (in p) and student's logits. Four entries a lane are asked for at a time. Returns the lane's largest t.
template <typename T>
__device__ __forceinline__ float fetch_entries(const Params& p, long long r, const T* logits, const Entries& en, int lane) {
  const int padded = entry_words(p.K);
  float most = -INFINITY;
  for (int k0 = 0; k0 < padded; k0 += 128) {
    long long id[4];
    float t[4], s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + u * 32 + lane;
      id[u] = -1;
      t[u] = -INFINITY;
      if (k < p.K) {
        id[u] = p.ids64 ? static_cast<const long long*>(p.ids)[r * p.ld_ids + k] : static_cast<const int*>(p.ids)[r * p.ld_ids + k];
        t[u] = p.teacher_f32 ? static_cast<const float*>(p.teacher)[r * p.ld_t + k]
                             : __bfloat162float(static_cast<const __nv_bfloat16*>(p.teacher)[r * p.ld_t + k]);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (id[u] < 0 || id[u] >= p.V) {
        id[u] = -1;
        t[u] = -INFINITY;
      }
      s[u] = id[u] >= 0 ? Elem<T>::get(logits + id[u]) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + u * 32 + lane;
      if (k < padded) {
        en.id[k] = static_cast<int>(id[u]);
        en.p[k] = t[u];
        en.s[k] = s[u];
      }
      most = fmaxf(most, t[u]);
    }
  }
  return most;
}
// 2: the weights, and whether there are any. (Differences of logits are taken ahead of the product with 1 / T: a rounded t / T is off by as much as two
// entries may differ by where T is low.)
__device__ __forceinline__ void weigh_entries(int K, const Entries& en, float most, float per_t, int lane) {
  const int padded = entry_words(K);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  const float mu = most == -INFINITY ? 0.f : most;
  float sum = 0.f;
  for (int k = lane; k < padded; k += 32) {
    const float e = en.id[k] >= 0 ? exp2_approx((en.p[k] - mu) * per_t) : 0.f;
    en.p[k] = e;
    sum += e;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  for (int k = lane; k < padded; k += 32) en.p[k] = en.w[k] = en.p[k] * inv;
  if (lane == 0) *en.there = sum != 0.f;  // (NaN: there are)
}
// 3: w of ids that are there more than once.
__device__ __forceinline__ void join_entries(int K, const Entries& en, int lane) {
  const int padded = entry_words(K), slots = table_words(K);
  for (int k = lane; k < slots; k += 32) en.table[k] = -1;
  __syncwarp();
  bool some_again = false;
  for (int k0 = 0; k0 < padded; k0 += 32) {
    const int k = k0 + lane, v = k < padded ? en.id[k] : -1;
    bool again = false;
    if (v >= 0) {
      for (unsigned at = static_cast<unsigned>(v) * 2654435761u >> 12;; ++at) {  // the table is at most half full: ends
        const int was = atomicCAS(&en.table[at & (slots - 1)], -1, v);
        again = was == v;
        if (was == -1 || was == v) break;
      }
    }
    const uint32_t bits = __ballot_sync(0xffffffffu, again);
    if (lane == 0) en.again[k0 >> 5] = bits;
    some_again |= bits != 0u;
  }
  __syncwarp();
  if (!some_again) return;
  // once for each such id: the sum over its entries, in a fixed order
  for (int word = 0; word < (K + 31) / 32; ++word) {
    while (const uint32_t left = en.again[word]) {
      const int id = en.id[word * 32 + __ffs(static_cast<int>(left)) - 1];
      float w = 0.f;
      for (int k = lane; k < padded; k += 32) w += en.id[k] == id ? en.p[k] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
      __syncwarp();
      for (int k0 = 0; k0 < padded; k0 += 32) {
        const int k = k0 + lane;
        const bool mine = k < padded && en.id[k] == id;
        if (mine) en.w[k] = w;
        const uint32_t bits = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) en.again[k0 >> 5] &= ~bits;
      }
      __syncwarp();
    }
  }
}

// SUM: makes the row's stats (otherwise they are given) and its loss; GRAD: its gradient, which may overwrite the logits.
template <typename T, bool SUM, bool GRAD>
__global__ void __launch_bounds__(MAX_THREADS + 32, 2) distill_kernel(const Params p) {
  constexpr int PER = Elem<T>::PER;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 red[MAX_THREADS / 32];
  const long long r = blockIdx.x;
  const int tid = threadIdx.x, threads = blockDim.x - 32, warp = tid >> 5, lane = tid & 31;  // threads: those of the row
  const bool for_row = tid < threads;
  const T* logits = static_cast<const T*>(p.logits) + r * p.ld;
  const Row<T> row(logits, p.V);
  const uint4* body = row.body();
  const Entries en = entries_in(smem, p.K);
  const int end = for_row ? row.end_of(tid, threads) : -1;
  float2 st = SUM ? make_float2(-INFINITY, 0.f) : p.stats[r];
  if (!for_row) {
    if (SUM || st.y != 0.f) {
      const float most = fetch_entries(p, r, logits, en, lane);
      __syncwarp();
      weigh_entries(p.K, en, most, p.per_t, lane);
    }
  } else if constexpr (SUM) {
    if (end >= 0) {  // (every exponential is taken against a rounded product, this one too: 1 only where nothing was rounded)
      const float s = Elem<T>::get(logits + end), m = s * p.per_t;
      st = make_float2(m, exp2_approx(fmaf(s, p.per_t, -m)));
    }
    if (!(st.x > -INFINITY)) st.y = st.x == st.x ? 0.f : st.x;  // (-inf: nothing; NaN stays)
    for (int j = tid; j < row.pieces; j += HELD * threads) {
      uint4 u[HELD];
#pragma unroll
      for (int k = 0; k < HELD; ++k) u[k] = j + k * threads < row.pieces ? body[j + k * threads] : no_piece<T>();
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < HELD; ++k) m = largest(m, u[k], T());
      m = fmaxf(st.x, m * p.per_t);
      const float mu = m == -INFINITY ? 0.f : m;
      uint64_t sum = f2_pack(st.y * exp2_approx(st.x - mu), 0.f);
      const uint64_t c2 = f2_pack(p.per_t, p.per_t), r2 = f2_pack(-mu, -mu);
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        float f[PER];
        Elem<T>::unpack(u[k], f);
#pragma unroll
        for (int e = 0; e < PER; e += 2) {
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(f[e], f[e + 1]), c2, r2), x0, x1);
          sum = f2_add(sum, f2_pack(exp2_approx(x0), exp2_approx(x1)));
        }
      }
      float s0, s1;
      f2_unpack(sum, s0, s1);
      st = make_float2(m, s0 + s1);
    }
    st = join_warp(st);
    if (lane == 0) red[warp] = st;
  }
  if (SUM) __syncthreads();  // (the backward's gradient never overwrites the logits)
  const bool there = SUM ? *en.there != 0 : st.y != 0.f;
  float z = 0.f;
  if constexpr (SUM) {
    st = join_warp(lane < threads / 32 ? red[lane] : make_float2(-INFINITY, 0.f));
    z = st.y;
    st.y = 1.f / z;
  }
  T* grad = GRAD ? static_cast<T*>(p.grad) + r * p.ldg : nullptr;
  const float scale = (SUM ? p.grad_scale : p.dloss[r * p.dloss_s] * (p.per_row ? *p.per_row : 1.f)) * p.t, mul = scale * st.y;
  if (GRAD && for_row) {
    const uint64_t c2 = f2_pack(p.per_t, p.per_t), r2 = f2_pack(-st.x, -st.x), m2 = f2_pack(mul, mul);
    const bool same = ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(logits)) & 15) == 0;
    if (end >= 0) Elem<T>::put(grad + end, there ? exp2_approx(fmaf(Elem<T>::get(logits + end), p.per_t, -st.x)) * mul : 0.f);
    uint4* to = reinterpret_cast<uint4*>(grad + row.first);
    if (there && same) {
      for (int j = tid; j < row.pieces; j += HELD * threads) {
        uint4 u[HELD];
#pragma unroll
        for (int k = 0; k < HELD; ++k) u[k] = j + k * threads < row.pieces ? __ldcs(body + j + k * threads) : no_piece<T>();
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
          float f[PER];
          Elem<T>::unpack(u[k], f);
#pragma unroll
          for (int e = 0; e < PER; e += 2) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(f[e], f[e + 1]), c2, r2), x0, x1);
            f2_unpack(f2_mul(f2_pack(exp2_approx(x0), exp2_approx(x1)), m2), f[e], f[e + 1]);
          }
          if (j + k * threads < row.pieces && RA_IN_BOUNDS((j + k * threads) * PER, PER, p.V, kTagDistill)) __stcs(to + j + k * threads, Elem<T>::pack(f));
        }
      }
    } else if (there) {  // into memory that starts elsewhere within 16 bytes
      for (int i = row.first + tid; i < row.first + row.pieces * PER; i += threads)
        Elem<T>::put(grad + i, exp2_approx(fmaf(Elem<T>::get(logits + i), p.per_t, -st.x)) * mul);
    } else {
      for (int i = row.first + tid; i < row.first + row.pieces * PER; i += threads) Elem<T>::put(grad + i, 0.f);
    }
  }
  if (!for_row) {
    if (GRAD && there) join_entries(p.K, en, lane);
    if (SUM) {
      float sum = 0.f;
      const float log_z = log2f(z);
      for (int k = lane; k < p.K; k += 32) {
        const float w = en.p[k];
        // log2 p less log2 q; an entry of weight 0 has no part in it
        if (w != 0.f) sum += w * ((log2f(w) + log_z) - fmaf(en.s[k], p.per_t, -st.x));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) {
        p.loss[r] = there ? p.t * p.t * 0.6931471805599453f * sum : 0.f;
        if (p.stats) p.stats[r] = make_float2(st.x, there ? st.y : 0.f);
      }
    }
  }
  if (GRAD) {
    __syncthreads();
    if (!for_row && there) {  // the entries, over what was written there
      __syncwarp();
      for (int k = lane; k < p.K; k += 32) {
        const int id = en.id[k];
        if (id >= 0 && RA_IN_BOUNDS(id, 1, p.V, kTagDistill))
          Elem<T>::put(grad + id, (exp2_approx(fmaf(en.s[k], p.per_t, -st.x)) * st.y - en.w[k]) * scale);
      }
    }
  }
}

// The same in 64 bits for rows of fewer than 2 K logits. A CTA for each row. Bound by the exponentials in 64 bits, two a logit and one an entry; us in
// 32 / 64 bits, 8192 rows of 512 logits and 300 entries in bf16: loss 37 / 86, loss and gradient 55 / 104, gradient 51 / 92; 8192 rows of 2000 and 1024:
// 127 / 199, 246 / 270, 232 / 244; 512 rows of 1000 and 512 in fp32: 14 / 16, 25 / 18, 23 / 18. Up to T = 4 a loss in 32 bits is off by 2^-17 at most.
constexpr int WIDE_THREADS = 128;
constexpr float WIDE_FROM = 4.f;  // temperature

__device__ __forceinline__ double sum_block(double v, double* red) {  // in a fixed order; the value in every thread
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < WIDE_THREADS / 32; ++w) v += red[w];
  return v;
}
__device__ __forceinline__ float most_block(float v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WIDE_THREADS / 32; ++w) v = fmaxf(v, static_cast<float>(red[w]));
  return v;
}

template <typename T, bool SUM>
__global__ void __launch_bounds__(WIDE_THREADS) distill_wide_kernel(const Params p) {
  __shared__ double weight[MAX_K];     // of an entry
  __shared__ double target[2 * MAX_K]; // of a logit: the weights of its entries
  __shared__ int id[MAX_K], first[2 * MAX_K];  // -1: absent; the first entry of a logit
  __shared__ unsigned char again[2 * MAX_K];   // the logit has more entries than one
  __shared__ double red[WIDE_THREADS / 32];
  const long long r = blockIdx.x;
  const int tid = threadIdx.x;
  const T* logits = static_cast<const T*>(p.logits) + r * p.ld;
  const double per_t = 1.0 / p.t;
  auto teacher = [&](int k) {
    return p.teacher_f32 ? static_cast<const float*>(p.teacher)[r * p.ld_t + k]
                         : __bfloat162float(static_cast<const __nv_bfloat16*>(p.teacher)[r * p.ld_t + k]);
  };
  float m = -INFINITY, mt = -INFINITY;
  for (int v = tid; v < p.V; v += WIDE_THREADS) {
    target[v] = 0.0;
    first[v] = MAX_K;
    again[v] = 0;
    m = fmaxf(m, Elem<T>::get(logits + v));
  }
  __syncthreads();
  for (int k = tid; k < p.K; k += WIDE_THREADS) {
    const long long at = p.ids64 ? static_cast<const long long*>(p.ids)[r * p.ld_ids + k] : static_cast<const int*>(p.ids)[r * p.ld_ids + k];
    const bool in = at >= 0 && at < p.V;
    id[k] = in ? static_cast<int>(at) : -1;
    if (in) {
      atomicMin(&first[at], k);
      mt = fmaxf(mt, teacher(k));
    }
  }
  m = most_block(m, red);
  mt = most_block(mt, red);
  if (m == -INFINITY) m = 0.f;
  if (mt == -INFINITY) mt = 0.f;
  double z = 0.0, w = 0.0;
  for (int v = tid; v < p.V; v += WIDE_THREADS) z += exp((static_cast<double>(Elem<T>::get(logits + v)) - m) * per_t);
  for (int k = tid; k < p.K; k += WIDE_THREADS) {
    const double e = id[k] >= 0 ? exp((static_cast<double>(teacher(k)) - mt) * per_t) : 0.0;
    weight[k] = e;
    w += e;
    if (id[k] >= 0 && first[id[k]] != k) again[id[k]] = 1;
  }
  z = sum_block(z, red);
  w = sum_block(w, red);
  const bool there = w != 0.0;  // (NaN: there are)
  const double log_w = log(w), log_z = log(z);
  double sum = 0.0;
  for (int k = tid; k < p.K; k += WIDE_THREADS) {
    const int v = id[k];
    if (v < 0) continue;
    const double pk = there ? weight[k] / w : 0.0;
    weight[k] = pk;
    if (!again[v]) target[v] = pk;
    if (SUM && pk != 0.0)
      sum += pk * (((static_cast<double>(teacher(k)) - mt) * per_t - log_w) - ((static_cast<double>(Elem<T>::get(logits + v)) - m) * per_t - log_z));
  }
  if (SUM) {
    sum = sum_block(sum, red);
    if (tid == 0) {
      p.loss[r] = there ? static_cast<float>(sum * p.t * p.t) : 0.f;
      if (p.stats) p.stats[r] = make_float2(m * p.per_t, there ? static_cast<float>(1.0 / z) : 0.f);
    }
  }
  if (!p.grad) return;
  __syncthreads();  // the weights are there, and the entries' logits are read: the gradient may overwrite them
  T* grad = static_cast<T*>(p.grad) + r * p.ldg;
  const double scale = static_cast<double>(SUM ? p.grad_scale : p.dloss[r * p.dloss_s] * (p.per_row ? *p.per_row : 1.f)) * p.t;
  for (int v = tid; v < p.V; v += WIDE_THREADS) {
    double t = target[v];
    if (again[v])
      for (int k = 0; k < p.K; ++k) t += id[k] == v ? weight[k] : 0.0;
    const double q = exp((static_cast<double>(Elem<T>::get(logits + v)) - m) * per_t) / z;
    if (RA_IN_BOUNDS(v, 1, p.V, kTagDistill)) Elem<T>::put(grad + v, there ? static_cast<float>((q - t) * scale) : 0.f);
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
template <bool SUM, bool GRAD>
int launch_distill(const RaDistillArgs* a) {
  using namespace ra;
  using namespace ra::distill;
  const int size = a->f32 ? 4 : 2;
  if (a->rows < 1 || a->rows > 0x7fffffffll || a->V < 1 || a->V > (1 << 30) || a->K < 1 || a->K > MAX_K || !(a->temperature > 0.f) || !a->logits || !a->ids ||
      !a->teacher || (reinterpret_cast<uintptr_t>(a->logits) % size) || (reinterpret_cast<uintptr_t>(a->grad) % size)) {
    set_error("distill: bad shape (1 to 1024 teacher entries, a positive temperature)");
    return kHostBadArg;
  }
  const Params p{a->logits, a->grad, a->ld, a->ldg, a->ids, a->teacher, a->ld_ids, a->ld_t, a->ids64, a->teacher_f32, a->V, a->K,
                 1.4426950408889634f / a->temperature, a->temperature, a->loss, static_cast<float2*>(a->stats), a->grad_scale, a->dloss, a->dloss_s,
                 a->per_row};
  if (a->V < 2 * a->K && a->temperature > WIDE_FROM) {
    auto wide = a->f32 ? distill_wide_kernel<float, SUM> : distill_wide_kernel<__nv_bfloat16, SUM>;
    wide<<<static_cast<unsigned>(a->rows), WIDE_THREADS, 0, static_cast<cudaStream_t>(a->stream)>>>(p);
    return check_launch("distill_wide_kernel");
  }
  // Eight pieces a thread, up to 256 threads (four CTAs an SM): us for 4096 rows of 32000 in bf16, loss / both, up to 192 threads 51 / 99, 256 47 / 94,
  // 512 60 / 114. 512 where the rows that are being worked on would outgrow the L2 before they are read again: 2048 rows of 64000 with 256 / 512
  // threads 49 / 55 for the loss, 107 / 108 for both (102 / 93 on another machine), 1024 rows of 128000 49 / 51 and 123 / 108. (The loss alone loses 4 to
  // 11 % by it, and so has the same bits with and without the gradient.)
  const long long bytes = static_cast<long long>(a->V) * size;
  long long threads = ((bytes / 16 + HELD - 1) / HELD + 31) / 32 * 32;
  const long long most = SUM && bytes > 96 * 1024 ? MAX_THREADS : 256;
  threads = threads < 64 ? 64 : (threads > most ? most : threads);
  const int smem = static_cast<int>(entry_smem(a->K));
  static_assert(4 * (4 + 4 * MAX_K + MAX_K / 32 + 2 * MAX_K) + 256 <= 48 * 1024, "a row's entries");
  auto kern = a->f32 ? distill_kernel<float, SUM, GRAD> : distill_kernel<__nv_bfloat16, SUM, GRAD>;
  kern<<<static_cast<unsigned>(a->rows), static_cast<unsigned>(threads + 32), smem, static_cast<cudaStream_t>(a->stream)>>>(p);
  return check_launch("distill_kernel");
}
}  // namespace

// Loss (and stats, and with `grad` the gradient times grad_scale, which may overwrite the logits) of every row.
extern "C" int ra_distill(const RaDistillArgs* a) {
  if (!a->loss) {
    ra::set_error("distill: no room for the losses");
    return ra::kHostBadArg;
  }
  return a->grad ? launch_distill<true, true>(a) : launch_distill<true, false>(a);
}

// grad <- the gradient of every row's logits, from `dloss` and the stats that ra_distill left.
extern "C" int ra_distill_bwd(const RaDistillArgs* a) {
  if (!a->grad || !a->stats || !a->dloss || a->grad == a->logits) {
    ra::set_error("distill_bwd: no gradient, stats or room for the result");
    return ra::kHostBadArg;
  }
  return launch_distill<false, true>(a);
}

// total <- the losses' sum, or with `mean` their mean over the rows that have entries; per_row <- what a row's loss was multiplied by.
extern "C" int ra_distill_reduce(const float* loss, const void* stats, long long rows, int mean, float* total, float* per_row, void* stream) {
  ra::distill::distill_reduce_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(loss, static_cast<const float2*>(stats), rows, mean, total,
                                                                                          per_row);
  return ra::check_launch("distill_reduce_kernel");
}

RA_PACKED(ra_distill_reduce)
