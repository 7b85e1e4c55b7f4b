// RMS norm of each head's query and key and their rotation by position, in one pass, forward and backward.
//
//   n = x r,  r = 1 / sqrt(mean(x^2) + eps);   y = R(pos) (g n)        (R turns the pairs (i, i + D/2) by pos * theta^(-2i/D))
//   backward: u = R(pos)^T dy;  w = g u;  dx = r (w - n mean(w n));  dg = sum over rows of u n
//
// r is made again in the backward from x, which has to be read anyway: nothing is saved between the passes but the inputs. Both passes are
// bound by memory (forward: x in, y out; backward: x and dy in, dx out; about 8 and 20 operations an element).
//
// A row (one head of one token) is taken by D / 16 lanes: each has eight elements of the first half and their partners of the second, so that
// the rotation needs no exchange and the sums log2(D / 16) shuffles. A warp takes the query heads or the key heads of one token, of several at
// once where the heads do not fill it: it makes their sines and cosines once, a lane keeps those of its elements in registers for all heads, and
// rows come through a ring of asynchronous copies into shared memory. Warps do not wait for one another.
//
// Measured, 16384 tokens of 32 and 8 heads: D 128 bf16 forward / backward 58 / 84 us, 5.7 / 6.0 TB/s, fp32 112 / 163 us, 6.0 / 6.2 TB/s; D 64
// (32 and 32 heads) bf16 40 / 64 us. What brought it there, forward / backward at D 128 in bf16: CTAs that share a table of sines, with barriers, 96 /
// 153; a table for each warp, read again for each row and prefetched rows in registers, 65 / 107 (bound by instructions and by shared memory, whose
// reads of eight floats in a row met in the banks: 87 % busy); tables in registers for all heads of a token and addresses stepped instead of made
// again, 58 / 84.
//
// Angles: pos * theta^(-2i/D) / 2 pi in 64 bits, less the whole turns, then the fp32 sine and cosine of the rest: an fp32 angle is off by 0.03
// at position 10^6. The frequencies are made on the host in 64 bits and come as launch parameters (1 KB).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common/bounds.cuh"
#include "common/host_util.h"
#include "common/mma_sync.cuh"
#include "common/sm100.cuh"

RA_BOUNDS_TRANSLATION_UNIT()

namespace ra {
namespace qk {

constexpr int THREADS = 128, WARPS = THREADS / 32;
constexpr int MAX_HALF = 128;  // of a head
// CTAs an SM, and stages of a lane's rows, one less of them under way: what registers (91 a thread forward, 128 backward without spills) and 60 to 80 KB
// in flight an SM (bf16 forward 60, fp32 forward 80, both backwards 64) ask for. 16384 tokens of 32 and 8 heads of 128 in bf16, forward: 58.4 us as
// here, 59.3 with 6 CTAs and 3 stages, 66.1 with 8 and 2 (64 registers); backward: 84.4 as here, 94.4 with 3 CTAs and 4 stages, 111 with 5 and 3 (spills).
template <bool BWD, bool F32> struct Cut {
  static constexpr int RESIDENT = BWD ? 4 : 5;
  static constexpr int STAGES = BWD ? (F32 ? 2 : 3) : (F32 ? 3 : 4);
  static constexpr int PIECES = (BWD ? 4 : 2) * (F32 ? 2 : 1);  // of 16 bytes, of x (and dy), that a lane has of a row
};

// one of the two tensors
struct Side {
  const void* x;       // (B, S, n, D), element strides
  long long x_sb, x_ss, x_sh;
  const void* dy;      // backward
  long long dy_sb, dy_ss, dy_sh;
  void* y;             // forward: y, backward: dx
  long long y_sb, y_ss, y_sh;
  const void* gain;    // (D)
  int n;               // heads
};

struct Params {
  Side side[2];        // queries, keys
  int B, S;
  unsigned tokens;
  int together[2];     // log2 of the heads that a warp takes at once, of queries and keys: all its groups of lanes, or as many as divide the heads
  int ctas[2];         // CTAs of each: first the queries', then the keys'
  int gain_f32;
  // positions: token s of batch row b at pos[b * pos_sb + s * pos_ss] (32 or 64 bits), or, without pos, at off0 + s, from `half` on at
  // off1 + (s - half)
  const void* pos;
  int pos64;
  long long pos_sb, pos_ss;
  int off0, off1, half;
  float eps;
  float* part;         // backward: (parts, D) sums of the gains' gradients, a row for each CTA
  int parts;
  double freq[MAX_HALF];  // turns per position
};

// A lane's eight elements of a half row as four pairs in 32 bits. `from`: its place in a stage, whose pieces lie 32 x 16 bytes apart; `next`: from the
// first run of four to the second in 32 bits.
template <typename T> struct Eight;
template <> struct Eight<__nv_bfloat16> {
  static __device__ __forceinline__ void get(const uint4* from, uint64_t* f) {
    const uint4 u = *from;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = f2_pack_u(w[e] << 16, w[e] & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, int, const uint64_t* f) {
    uint32_t v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float lo, hi;
      f2_unpack(f[e], lo, hi);
      v[e] = pack_bf16x2(lo, hi);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
  }
};
template <> struct Eight<float> {
  static __device__ __forceinline__ void get(const uint4* from, uint64_t* f) {
    const uint4 a = from[0], b = from[32];
    f[0] = f2_pack_u(a.x, a.y);
    f[1] = f2_pack_u(a.z, a.w);
    f[2] = f2_pack_u(b.x, b.y);
    f[3] = f2_pack_u(b.z, b.w);
  }
  static __device__ __forceinline__ void store(float* p, int next, const uint64_t* f) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) f2_unpack(f[e], v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + next) = make_float4(v[4], v[5], v[6], v[7]);
  }
};

template <int LANES>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Of a half row a lane has eight elements in two runs of four: in bf16 behind one another (16 bytes), in 32 bits a quarter row apart (so that each
// run's 16 bytes lie beside those of the next lane). In shared memory, in 32 bits, all runs lie like the latter.
template <typename T, int D>
__device__ __forceinline__ int spread(int f) { return sizeof(T) == 4 ? f : ((f >> 2) & 1) * (D / 4) + (f >> 3) * 4 + (f & 3); }
template <typename T, int D>
__device__ __forceinline__ int run(int l, int i) { return sizeof(T) == 4 ? i * (D / 4) + l * 4 : l * 8 + i * 4; }

// cosines and sines of the tokens t0 .. t0 + n - 1, by one warp: turn[token][cos D / 2 | sin D / 2]
template <typename T, int D>
__device__ __forceinline__ void fill_turns(const Params& p, unsigned t0, int n, float* turn, int lane) {
  for (int i = lane; i < n * (D / 2); i += 32) {
    const unsigned t = t0 + i / (D / 2);
    if (t >= p.tokens) break;
    const unsigned b = t / static_cast<unsigned>(p.S), s = t - b * p.S;
    long long pos;
    if (p.pos) {
      const long long at = b * p.pos_sb + s * p.pos_ss;
      pos = p.pos64 ? static_cast<const long long*>(p.pos)[at] : static_cast<const int*>(p.pos)[at];
    } else {
      pos = static_cast<int>(s) < p.half ? p.off0 + static_cast<int>(s) : p.off1 + (static_cast<int>(s) - p.half);
    }
    const int f = i % (D / 2);
    double turns = static_cast<double>(pos) * p.freq[f];
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.f * static_cast<float>(turns), &sn, &cs);
    float* to = turn + (i / (D / 2)) * D + spread<T, D>(f);
    to[0] = cs;
    to[D / 2] = sn;
  }
}

template <int D>
__device__ __forceinline__ void load_pairs(const float* p, uint64_t* v) {  // a lane's eight floats of a half row as pairs
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 f = *reinterpret_cast<const float4*>(p + i * (D / 4));
    v[2 * i] = f2_pack(f.x, f.y);
    v[2 * i + 1] = f2_pack(f.z, f.w);
  }
}

// BWD keeps the sums for the gain of its columns in registers: one row of partial sums a CTA, which dgain_kernel adds up in a fixed order. (A
// CTA that takes both sides needs twice the registers for them.)
template <typename T, int D, bool BWD>
__global__ void __launch_bounds__(THREADS, (Cut<BWD, sizeof(T) == 4>::RESIDENT)) qk_norm_rope_kernel(const Params p) {
  using C = Cut<BWD, sizeof(T) == 4>;
  constexpr int LANES = D / 16, GROUPS = 32 / LANES, ST = C::STAGES, PIECES = C::PIECES, PER = 16 / sizeof(T), TENSOR = PIECES / (BWD ? 2 : 1);
  __shared__ __align__(16) uint4 ring[WARPS][ST][PIECES][32];
  __shared__ __align__(16) float turns[WARPS][GROUPS * D];
  static_assert(sizeof(ring) >= WARPS * D * sizeof(float), "the ring becomes the place of the warps' sums");
  const int which = static_cast<int>(blockIdx.x) >= p.ctas[0];
  const int cta = static_cast<int>(blockIdx.x) - (which ? p.ctas[0] : 0);
  const Side& s = p.side[which];
  const int together = p.together[which], at_once = GROUPS >> together, steps = s.n >> together;  // heads (log2) and tokens at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / LANES, l = lane % LANES;
  const int my_token = group >> together, my_head = group & ((1 << together) - 1);
  const unsigned units = (p.tokens + at_once - 1) / at_once, stride = static_cast<unsigned>(p.ctas[which]) * WARPS;
  uint64_t g0[4], g1[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int f = run<T, D>(l, e >> 1) + (e & 1) * 2;
    if (p.gain_f32) {
      const float* g = static_cast<const float*>(s.gain);
      g0[e] = f2_pack(g[f], g[f + 1]);
      g1[e] = f2_pack(g[D / 2 + f], g[D / 2 + f + 1]);
    } else {
      const __nv_bfloat16* g = static_cast<const __nv_bfloat16*>(s.gain);
      g0[e] = f2_pack(__bfloat162float(g[f]), __bfloat162float(g[f + 1]));
      g1[e] = f2_pack(__bfloat162float(g[D / 2 + f]), __bfloat162float(g[D / 2 + f + 1]));
    }
  }
  // this lane's first row of a unit of tokens, in a tensor of these strides; whether there is one
  auto row = [&](unsigned unit, long long sb, long long ss, long long sh) {
    const unsigned t = unit * at_once + my_token, b = t / static_cast<unsigned>(p.S);
    return b * sb + (t - b * p.S) * ss + my_head * sh + run<T, D>(l, 0);
  };
  auto there = [&](unsigned unit) { return unit * at_once + my_token < p.tokens; };

  // What is fetched runs ahead of what is computed. A lane fetches what it alone reads, so its own count of copies under way is all that it waits for.
  unsigned unit = static_cast<unsigned>(cta) * WARPS + warp, ahead = unit;
  int ahead_step = 0;
  const T *x = nullptr, *dy = nullptr;
  auto fetch_next = [&](int slot) {
    if (ahead < units) {
      if (ahead_step == 0) {
        x = static_cast<const T*>(s.x) + row(ahead, s.x_sb, s.x_ss, s.x_sh);
        if (BWD) dy = static_cast<const T*>(s.dy) + row(ahead, s.dy_sb, s.dy_ss, s.dy_sh);
      }
      if (there(ahead)) {
        uint4* to = &ring[warp][slot][0][lane];
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {  // x, then dy; of each the first half's, then the second's
          const int j = i % TENSOR, in_half = j % (8 / PER);
          cp_async16(to + i * 32, (i < TENSOR ? x : dy) + (j / (8 / PER)) * (D / 2) + in_half * (D / 4), 16);
        }
      }
      x += s.x_sh << together;
      if (BWD) dy += s.dy_sh << together;
      if (++ahead_step == steps) {
        ahead_step = 0;
        ahead += stride;
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) fetch_next(i);
  uint64_t sum[BWD ? 8 : 1];
#pragma unroll
  for (int e = 0; e < (BWD ? 8 : 1); ++e) sum[e] = f2_pack(0.f, 0.f);
  int slot = 0;
  for (; unit < units; unit += stride) {
    __syncwarp();
    fill_turns<T, D>(p, unit * at_once, at_once, turns[warp], lane);
    __syncwarp();
    const bool in = there(unit);
    uint64_t cs[4], sn[4];
    {
      const float* tn = turns[warp] + (in ? my_token * D : 0) + l * 4;
      load_pairs<D>(tn, cs);
      load_pairs<D>(tn + D / 2, sn);
    }
    T* y = static_cast<T*>(s.y) + row(unit, s.y_sb, s.y_ss, s.y_sh);
    for (int step = 0; step < steps; ++step, y += s.y_sh << together) {
      uint64_t a[4], c[4], da[4], dc[4];
      fetch_next(slot == 0 ? ST - 1 : slot - 1);  // the place that the last step has read
      cp_async_wait<ST - 1>();
      if (in) {
        const uint4* from = &ring[warp][slot][0][lane];
        Eight<T>::get(from, a);
        Eight<T>::get(from + TENSOR / 2 * 32, c);
        if (BWD) {
          Eight<T>::get(from + TENSOR * 32, da);
          Eight<T>::get(from + TENSOR / 2 * 3 * 32, dc);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = c[e] = da[e] = dc[e] = f2_pack(0.f, 0.f);
      }
      slot = slot + 1 == ST ? 0 : slot + 1;
      uint64_t ss2 = f2_mul(a[0], a[0]);
#pragma unroll
      for (int e = 1; e < 4; ++e) ss2 = f2_fma(a[e], a[e], ss2);
#pragma unroll
      for (int e = 0; e < 4; ++e) ss2 = f2_fma(c[e], c[e], ss2);
      float ss, ss_hi;
      f2_unpack(ss2, ss, ss_hi);
      const float rstd = rsqrtf(sum_lanes<LANES>(ss + ss_hi) * (1.f / D) + p.eps);
      const uint64_t r2 = f2_pack(rstd, rstd);
      if constexpr (BWD) {
        uint64_t dot2 = f2_pack(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = f2_mul(a[e], r2);
          c[e] = f2_mul(c[e], r2);
          const uint64_t u0 = f2_fma(da[e], cs[e], f2_mul(dc[e], sn[e])), u1 = f2_sub(f2_mul(dc[e], cs[e]), f2_mul(da[e], sn[e]));
          if (in) {
            sum[e] = f2_fma(u0, a[e], sum[e]);
            sum[BWD ? 4 + e : 0] = f2_fma(u1, c[e], sum[BWD ? 4 + e : 0]);
          }
          da[e] = f2_mul(u0, g0[e]);
          dc[e] = f2_mul(u1, g1[e]);
          dot2 = f2_fma(dc[e], c[e], f2_fma(da[e], a[e], dot2));
        }
        float dot, dot_hi;
        f2_unpack(dot2, dot, dot_hi);
        dot = sum_lanes<LANES>(dot + dot_hi) * (-1.f / D);
        const uint64_t d2 = f2_pack(dot, dot);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = f2_mul(r2, f2_fma(a[e], d2, da[e]));
          c[e] = f2_mul(r2, f2_fma(c[e], d2, dc[e]));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t m = f2_mul(f2_mul(a[e], r2), g0[e]), k = f2_mul(f2_mul(c[e], r2), g1[e]);
          a[e] = f2_sub(f2_mul(m, cs[e]), f2_mul(k, sn[e]));
          c[e] = f2_fma(k, cs[e], f2_mul(m, sn[e]));
        }
      }
      if (in && RA_IN_BOUNDS((step << together) + my_head, 1, s.n, kTagQkNorm)) {
        Eight<T>::store(y, D / 4, a);
        Eight<T>::store(y + D / 2, D / 4, c);
      }
    }
  }
  if constexpr (BWD) {
    cp_async_wait<0>();
    __syncthreads();  // all rows are read: the ring becomes [warp][D]
    float* const red = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v[2];
      f2_unpack(sum[e], v[0], v[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 16; o >= LANES; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        if (lane < LANES) red[warp * D + (e >> 2) * (D / 2) + run<T, D>(l, (e >> 1) & 1) + (e & 1) * 2 + i] = v[i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += THREADS) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += red[w * D + i];
      p.part[static_cast<long long>(blockIdx.x) * D + i] = v;
    }
  }
}

// dgain (2, D) in the gains' type <- the sums over the partial rows of each side. A CTA takes eight columns, as 128 groups of eight threads.
__global__ void __launch_bounds__(1024) dgain_kernel(const float* __restrict__ part, int ctas0, int ctas1, int D, void* dgain, int f32) {
  __shared__ float red[128][9];
  const int c = threadIdx.x & 7, g = threadIdx.x >> 3, col = blockIdx.x * 8 + c, which = blockIdx.y;
  const float* from = part + (which ? static_cast<long long>(ctas0) * D : 0) + col;
  const int n = which ? ctas1 : ctas0;
  float v = 0.f;
  for (int i = g; i < n; i += 128) v += from[static_cast<long long>(i) * D];
  red[g][c] = v;
  __syncthreads();
  for (int k = 64; k > 0; k >>= 1) {
    if (g < k) red[g][c] += red[g + k][c];
    __syncthreads();
  }
  if (g == 0) {
    if (f32) static_cast<float*>(dgain)[which * D + col] = red[0][c];
    else static_cast<__nv_bfloat16*>(dgain)[which * D + col] = __float2bfloat16(red[0][c]);
  }
}

}  // namespace qk
}  // namespace ra

// One of queries and keys: (B, S, heads, D) views with element strides, the innermost contiguous, everything on 16 bytes.
struct RaQkSide {
  const void* x; long long x_sb, x_ss, x_sh;
  const void* dy; long long dy_sb, dy_ss, dy_sh;  // backward
  void* y; long long y_sb, y_ss, y_sh;            // forward: the result, backward: dx
  const void* gain;
  int heads;
};

struct RaQkNormArgs {
  RaQkSide q; RaQkSide k;
  int B, S, D;
  int f32, gain_f32;       // types: of the activations and of the gains, 1: fp32, 0: bf16
  const void* pos; int pos64; long long pos_sb, pos_ss;
  int off0, off1, half;
  float eps;
  double theta;
  float* part; int parts;  // backward: parts * D floats, parts as ra_qk_norm_parts says; dgain (2, D) in the gains' type
  void* dgain;
  void* stream;
};

namespace {
bool ready(const void* t, long long sb, long long ss, long long sh, int per16) {
  return t && !(reinterpret_cast<uintptr_t>(t) & 15) && !(sb % per16) && !(ss % per16) && !(sh % per16);
}
int to_params(const RaQkNormArgs* a, bool backward, ra::qk::Params& p) {
  using namespace ra;
  const int per16 = a->f32 ? 4 : 8;
  if (a->B < 1 || a->S < 1 || a->q.heads < 1 || a->k.heads < 1 || (a->D != 64 && a->D != 128 && a->D != 256) || !(a->theta > 0.0) ||
      !(a->eps >= 0.f) || a->half < 0) {
    set_error("qk_norm_rope: head_dim must be 64, 128 or 256, theta positive, eps not negative");
    return kHostBadArg;
  }
  const RaQkSide* side[2] = {&a->q, &a->k};
  for (int i = 0; i < 2; ++i) {
    const RaQkSide& s = *side[i];
    if (!ready(s.x, s.x_sb, s.x_ss, s.x_sh, per16) || !ready(s.y, s.y_sb, s.y_ss, s.y_sh, per16) ||
        (backward && !ready(s.dy, s.dy_sb, s.dy_ss, s.dy_sh, per16)) || !s.gain) {
      set_error("qk_norm_rope: rows must start on 16 bytes");
      return kHostBadArg;
    }
    p.side[i] = qk::Side{s.x, s.x_sb, s.x_ss, s.x_sh, s.dy, s.dy_sb, s.dy_ss, s.dy_sh, s.y, s.y_sb, s.y_ss, s.y_sh, s.gain, s.heads};
  }
  p.B = a->B;
  p.S = a->S;
  const long long tokens = static_cast<long long>(a->B) * a->S;
  if (tokens > 0x7fffffffll) {
    set_error("qk_norm_rope: too many tokens");
    return kHostTooLarge;
  }
  p.tokens = static_cast<unsigned>(tokens);
  p.gain_f32 = a->gain_f32;
  p.pos = a->pos;
  p.pos64 = a->pos64;
  p.pos_sb = a->pos_sb;
  p.pos_ss = a->pos_ss;
  p.off0 = a->off0;
  p.off1 = a->off1;
  p.half = a->half;
  p.eps = a->eps;
  p.part = a->part;
  p.parts = a->parts;
  for (int i = 0; i < a->D / 2; ++i) p.freq[i] = pow(a->theta, -2.0 * i / a->D) / 6.283185307179586476925;
  return kHostOk;
}
}  // namespace

namespace {
// Heads at once and CTAs of both sides: `resident` CTAs an SM, shared by queries and keys as their work is. (The sines and cosines of a token take a
// warp as long as two steps. Shared as the rows are, one key head beside 32 query heads took 16384 tokens 235 us instead of 59.)
void cut_up(ra::qk::Params& p, int D, int resident) {
  using namespace ra;
  const int groups = 32 / (D / 16), all = p.side[0].n + p.side[1].n + 4 * groups;
  const long long room = static_cast<long long>(resident) * sm_count();
  for (int i = 0; i < 2; ++i) {
    const int n = p.side[i].n;
    int together = 0;
    while ((2 << together) <= groups && n % (2 << together) == 0) ++together;
    const long long at_once = groups >> together;
    const long long ctas = ((static_cast<long long>(p.tokens) + at_once - 1) / at_once + qk::WARPS - 1) / qk::WARPS;
    long long most = room * (n + 2 * groups) / all;
    if (most < 1) most = 1;
    p.together[i] = together;
    p.ctas[i] = static_cast<int>(ctas < most ? ctas : most);
  }
}
template <typename T, int D, bool BWD>
int launch(ra::qk::Params& p, cudaStream_t s) {
  using namespace ra::qk;
  cut_up(p, D, Cut<BWD, sizeof(T) == 4>::RESIDENT);
  if (BWD && p.parts < p.ctas[0] + p.ctas[1]) {
    ra::set_error("qk_norm_rope_bwd: no room for the gains' gradients");
    return ra::kHostBadArg;
  }
  qk_norm_rope_kernel<T, D, BWD><<<p.ctas[0] + p.ctas[1], THREADS, 0, s>>>(p);
  return ra::check_launch(BWD ? "qk_norm_rope_bwd" : "qk_norm_rope");
}
template <bool BWD>
int launch(ra::qk::Params& p, const RaQkNormArgs* a) {
  using bf16 = __nv_bfloat16;
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  switch (a->D) {
    case 64: return a->f32 ? launch<float, 64, BWD>(p, s) : launch<bf16, 64, BWD>(p, s);
    case 128: return a->f32 ? launch<float, 128, BWD>(p, s) : launch<bf16, 128, BWD>(p, s);
    default: return a->f32 ? launch<float, 256, BWD>(p, s) : launch<bf16, 256, BWD>(p, s);
  }
}
}  // namespace

extern "C" int ra_qk_norm_rope(const RaQkNormArgs* a) {
  ra::qk::Params p;
  if (int rc = to_params(a, false, p)) return rc;
  return launch<false>(p, a);
}

// Rows of partial sums that the backward may write (each D floats).
extern "C" int ra_qk_norm_parts() { return ra::qk::Cut<true, false>::RESIDENT * ra::sm_count() + 2; }

extern "C" int ra_qk_norm_rope_bwd(const RaQkNormArgs* a) {
  using namespace ra;
  using namespace ra::qk;
  Params p;
  if (int rc = to_params(a, true, p)) return rc;
  if (!a->part || !a->dgain) {
    set_error("qk_norm_rope_bwd: no room for the gains' gradients");
    return kHostBadArg;
  }
  if (int rc = launch<true>(p, a)) return rc;
  dgain_kernel<<<dim3(a->D / 8, 2), 1024, 0, static_cast<cudaStream_t>(a->stream)>>>(a->part, p.ctas[0], p.ctas[1], a->D, a->dgain, a->gain_f32);
  return check_launch("dgain");
}
