// RMS norm of each head's query and key and their rotation by position, in one pass, forward and backward.
//
//   n = x r,  r = 1 / sqrt(mean(x^2) + eps);   y = R(pos) (g n)        (R turns the pairs (i, i + D/2) by pos * theta^(-2i/D))
//   backward: u = R(pos)^T dy;  w = g u;  dx = r (w - n mean(w n));  dg = sum over rows of u n
//
// r is made again in the backward from x, which has to be read anyway: nothing is saved between the passes but the inputs. Both passes are
// bound by memory (forward: x in, y out; backward: x and dy in, dx out; about 8 and 20 operations an element).
//
// A row (one head of one token) is taken by D / 16 lanes: each has eight elements of the first half and their partners of the second, two
// 16-byte loads in bf16, so that the rotation needs no exchange and the sums log2(D / 16) shuffles. A CTA takes `tile` tokens and all of their
// heads, or a share of the heads where there are few tokens (decoding); the sines and cosines of its tokens are made once, in
// shared memory, by one thread for each angle.
//
// Angles: pos * theta^(-2i/D) / 2 pi in 64 bits, less the whole turns, then the fp32 sine and cosine of the rest: an fp32 angle is off by 0.03
// at position 10^6. The frequencies are made on the host in 64 bits and come as launch parameters (1 KB).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common/bounds.cuh"
#include "common/host_util.h"

RA_BOUNDS_TRANSLATION_UNIT()

namespace ra {
namespace qk {

constexpr int THREADS = 256;
constexpr int MAX_HALF = 128;  // of a head

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
  long long tokens;
  int tile;            // tokens a CTA takes at a time
  int gain_f32;
  // positions: token s of batch row b at pos[b * pos_sb + s * pos_ss] (32 or 64 bits), or, without pos, at off0 + s, from `half` on at
  // off1 + (s - half)
  const void* pos;
  int pos64;
  long long pos_sb, pos_ss;
  int off0, off1, half;
  float eps;
  float* part;         // backward: (gridDim.x, 2, D) sums of the gains' gradients
  double freq[MAX_HALF];  // turns per position
};

template <typename T> struct Eight;  // eight elements of a row
template <> struct Eight<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float* f) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __uint_as_float(w[e] << 16);
      f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* f) {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
    *reinterpret_cast<uint4*>(p) = v;
  }
};
template <> struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float* f) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  }
};

template <int LANES>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float gain_at(const Params& p, const Side& s, int i) {
  return p.gain_f32 ? static_cast<const float*>(s.gain)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(s.gain)[i]);
}

// cosines and sines of the tokens t0 .. t0 + tile - 1, and the gains
template <int D>
__device__ __forceinline__ void fill_tables(const Params& p, long long t0, float2* turn) {
  for (int i = threadIdx.x; i < p.tile * (D / 2); i += THREADS) {
    const long long t = t0 + i / (D / 2);
    if (t >= p.tokens) break;
    const int b = static_cast<int>(t / p.S), s = static_cast<int>(t - static_cast<long long>(b) * p.S);
    long long pos;
    if (p.pos) {
      const long long at = b * p.pos_sb + s * p.pos_ss;
      pos = p.pos64 ? static_cast<const long long*>(p.pos)[at] : static_cast<const int*>(p.pos)[at];
    } else {
      pos = s < p.half ? p.off0 + s : p.off1 + (s - p.half);
    }
    double turns = static_cast<double>(pos) * p.freq[i % (D / 2)];
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.f * static_cast<float>(turns), &sn, &cs);
    turn[i] = make_float2(cs, sn);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS) qk_norm_rope_fwd_kernel(const Params p) {
  constexpr int LANES = D / 16, GROUPS = THREADS / LANES;
  extern __shared__ float2 turn[];      // [tile][D / 2]
  __shared__ float gain[2][D];
  const long long t0 = static_cast<long long>(blockIdx.x) * p.tile;
  fill_tables<D>(p, t0, turn);
  for (int i = threadIdx.x; i < 2 * D; i += THREADS) gain[i / D][i % D] = gain_at(p, p.side[i / D], i % D);
  __syncthreads();
  const int group = threadIdx.x / LANES, l = threadIdx.x % LANES;
  const int heads = p.side[0].n + p.side[1].n;
  // rows of the tile, token by token; gridDim.y CTAs share them. The lanes of a warp stay together for the shuffles.
  const int rows = p.tile * heads, step = GROUPS * gridDim.y;
  for (int r0 = blockIdx.y * GROUPS; r0 < rows; r0 += step) {
    const int r = r0 + group;
    const int tt = r / heads;
    int h = r - tt * heads;
    const long long t = t0 + tt;
    const bool in = r < rows && t < p.tokens;
    const int which = h >= p.side[0].n;
    const Side& s = p.side[which];
    h -= which ? p.side[0].n : 0;
    const int b = static_cast<int>(t / p.S);
    const long long at = t - static_cast<long long>(b) * p.S;
    float a[8], c[8];
    if (in) {
      const T* x = static_cast<const T*>(s.x) + b * s.x_sb + at * s.x_ss + h * s.x_sh + l * 8;
      Eight<T> u, v;
      u.load(x);
      v.load(x + D / 2);
      u.get(a);
      v.get(c);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = c[e] = 0.f;
    }
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + c[e] * c[e];
    ss = sum_lanes<LANES>(ss);
    if (!in || !RA_IN_BOUNDS(h, 1, s.n, kTagQkNorm)) continue;
    const float rstd = rsqrtf(ss * (1.f / D) + p.eps);
    const float2* tn = turn + tt * (D / 2) + l * 8;
    const float* g = gain[which] + l * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float m = a[e] * rstd * g[e], k = c[e] * rstd * g[e + D / 2];
      a[e] = m * tn[e].x - k * tn[e].y;
      c[e] = k * tn[e].x + m * tn[e].y;
    }
    T* y = static_cast<T*>(s.y) + b * s.y_sb + at * s.y_ss + h * s.y_sh + l * 8;
    Eight<T>::store(y, a);
    Eight<T>::store(y + D / 2, c);
  }
}

// A CTA walks its tiles of tokens with stride gridDim.x and keeps the sums for the gains of its columns in registers, first for the queries,
// then for the keys; one row of partial sums a CTA, which dgain_kernel adds up in a fixed order.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS) qk_norm_rope_bwd_kernel(const Params p) {
  constexpr int LANES = D / 16, GROUPS = THREADS / LANES, WARPS = THREADS / 32;
  extern __shared__ float2 turn[];
  __shared__ float gain[2][D];
  __shared__ float red[WARPS][D];
  for (int i = threadIdx.x; i < 2 * D; i += THREADS) gain[i / D][i % D] = gain_at(p, p.side[i / D], i % D);
  const int group = threadIdx.x / LANES, l = threadIdx.x % LANES;
  float sum[2][16];
#pragma unroll
  for (int e = 0; e < 32; ++e) sum[e / 16][e % 16] = 0.f;
  for (long long t0 = static_cast<long long>(blockIdx.x) * p.tile; t0 < p.tokens; t0 += static_cast<long long>(gridDim.x) * p.tile) {
    __syncthreads();
    fill_tables<D>(p, t0, turn);
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const Side& s = p.side[which];
      const int rows = p.tile * s.n;
      for (int r0 = 0; r0 < rows; r0 += GROUPS) {
        const int r = r0 + group;
        const int tt = r / s.n, h = r - tt * s.n;
        const long long t = t0 + tt;
        const bool in = r < rows && t < p.tokens;
        const int b = static_cast<int>(t / p.S);
        const long long at = t - static_cast<long long>(b) * p.S;
        float a[8], c[8], da[8], dc[8];
        if (in) {
          const T* x = static_cast<const T*>(s.x) + b * s.x_sb + at * s.x_ss + h * s.x_sh + l * 8;
          const T* dy = static_cast<const T*>(s.dy) + b * s.dy_sb + at * s.dy_ss + h * s.dy_sh + l * 8;
          Eight<T> u, v, du, dv;
          u.load(x);
          v.load(x + D / 2);
          du.load(dy);
          dv.load(dy + D / 2);
          u.get(a);
          v.get(c);
          du.get(da);
          dv.get(dc);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = c[e] = da[e] = dc[e] = 0.f;
        }
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + c[e] * c[e];
        const float rstd = rsqrtf(sum_lanes<LANES>(ss) * (1.f / D) + p.eps);
        const float2* tn = turn + (in ? tt * (D / 2) : 0) + l * 8;
        const float* g = gain[which] + l * 8;
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[e] *= rstd;
          c[e] *= rstd;
          const float u0 = da[e] * tn[e].x + dc[e] * tn[e].y, u1 = dc[e] * tn[e].x - da[e] * tn[e].y;
          if (in) {
            sum[which][e] += u0 * a[e];
            sum[which][8 + e] += u1 * c[e];
          }
          da[e] = u0 * g[e];
          dc[e] = u1 * g[e + D / 2];
          dot += da[e] * a[e] + dc[e] * c[e];
        }
        dot = sum_lanes<LANES>(dot) * (1.f / D);
        if (!in || !RA_IN_BOUNDS(h, 1, s.n, kTagQkNorm)) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[e] = rstd * (da[e] - a[e] * dot);
          c[e] = rstd * (dc[e] - c[e] * dot);
        }
        T* y = static_cast<T*>(s.y) + b * s.y_sb + at * s.y_ss + h * s.y_sh + l * 8;
        Eight<T>::store(y, a);
        Eight<T>::store(y + D / 2, c);
      }
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float v = sum[which][e];
#pragma unroll
      for (int o = 16; o >= LANES; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane < LANES) red[warp][(e >> 3) * (D / 2) + l * 8 + (e & 7)] = v;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += THREADS) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += red[w][i];
      p.part[(static_cast<long long>(blockIdx.x) * 2 + which) * D + i] = v;
    }
  }
}

// dgain (2, D) in the gains' type <- the sum over the `parts` partial rows (2 D floats). A CTA takes eight columns, as 128 groups of eight threads.
__global__ void __launch_bounds__(1024) dgain_kernel(const float* __restrict__ part, int parts, int width, void* dgain, int f32) {
  __shared__ float red[128][9];
  const int c = threadIdx.x & 7, g = threadIdx.x >> 3, col = blockIdx.x * 8 + c;
  float v = 0.f;
  for (int i = g; i < parts; i += 128) v += part[static_cast<long long>(i) * width + col];
  red[g][c] = v;
  __syncthreads();
  for (int n = 64; n > 0; n >>= 1) {
    if (g < n) red[g][c] += red[g + n][c];
    __syncthreads();
  }
  if (g == 0) {
    if (f32) static_cast<float*>(dgain)[col] = red[0][c];
    else static_cast<__nv_bfloat16*>(dgain)[col] = __float2bfloat16(red[0][c]);
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
  float* part; int parts;  // backward: parts * 2 * D floats, parts as ra_qk_norm_parts says; dgain (2, D) in the gains' type
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
  p.tokens = static_cast<long long>(a->B) * a->S;
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
  for (int i = 0; i < a->D / 2; ++i) p.freq[i] = pow(a->theta, -2.0 * i / a->D) / 6.283185307179586476925;
  return kHostOk;
}
}  // namespace

extern "C" int ra_qk_norm_rope(const RaQkNormArgs* a) {
  using namespace ra;
  using namespace ra::qk;
  Params p;
  if (int rc = to_params(a, false, p)) return rc;
  const int heads = a->q.heads + a->k.heads, groups = THREADS / (a->D / 16);
  p.tile = 1;
  while (p.tile < 8 && p.tile * heads < 4 * groups && p.tokens / p.tile >= 8ll * sm_count()) p.tile *= 2;
  const long long gx = (p.tokens + p.tile - 1) / p.tile;
  long long gy = 1;
  while (gx * gy < sm_count() && gy * groups < heads * p.tile) ++gy;
  if (gx > 0x7fffffffll) {
    set_error("qk_norm_rope: too many tokens");
    return kHostTooLarge;
  }
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  const size_t smem = static_cast<size_t>(p.tile) * a->D / 2 * sizeof(float2);
  auto kern = a->D == 64 ? (a->f32 ? qk_norm_rope_fwd_kernel<float, 64> : qk_norm_rope_fwd_kernel<__nv_bfloat16, 64>)
            : a->D == 128 ? (a->f32 ? qk_norm_rope_fwd_kernel<float, 128> : qk_norm_rope_fwd_kernel<__nv_bfloat16, 128>)
                          : (a->f32 ? qk_norm_rope_fwd_kernel<float, 256> : qk_norm_rope_fwd_kernel<__nv_bfloat16, 256>);
  kern<<<grid, THREADS, smem, static_cast<cudaStream_t>(a->stream)>>>(p);
  return check_launch("qk_norm_rope_fwd");
}

// Rows of partial sums that the backward of `tokens` tokens writes (each 2 D floats).
extern "C" int ra_qk_norm_parts(long long tokens) {
  const long long most = 4ll * ra::sm_count();
  return static_cast<int>(tokens < most ? (tokens < 1 ? 1 : tokens) : most);
}

extern "C" int ra_qk_norm_rope_bwd(const RaQkNormArgs* a) {
  using namespace ra;
  using namespace ra::qk;
  Params p;
  if (int rc = to_params(a, true, p)) return rc;
  if (!a->part || !a->dgain || a->parts != ra_qk_norm_parts(p.tokens)) {
    set_error("qk_norm_rope_bwd: no room for the gains' gradients");
    return kHostBadArg;
  }
  const int heads = a->q.heads + a->k.heads, groups = THREADS / (a->D / 16);
  p.tile = 1;
  while (p.tile < 8 && p.tile * heads < 4 * groups && p.tokens / p.tile >= 4ll * sm_count()) p.tile *= 2;
  const size_t smem = static_cast<size_t>(p.tile) * a->D / 2 * sizeof(float2);
  auto kern = a->D == 64 ? (a->f32 ? qk_norm_rope_bwd_kernel<float, 64> : qk_norm_rope_bwd_kernel<__nv_bfloat16, 64>)
            : a->D == 128 ? (a->f32 ? qk_norm_rope_bwd_kernel<float, 128> : qk_norm_rope_bwd_kernel<__nv_bfloat16, 128>)
                          : (a->f32 ? qk_norm_rope_bwd_kernel<float, 256> : qk_norm_rope_bwd_kernel<__nv_bfloat16, 256>);
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  kern<<<static_cast<unsigned>(a->parts), THREADS, smem, s>>>(p);
  if (int rc = check_launch("qk_norm_rope_bwd")) return rc;
  dgain_kernel<<<2 * a->D / 8, 1024, 0, s>>>(a->part, a->parts, 2 * a->D, a->dgain, a->gain_f32);
  return check_launch("dgain");
}
