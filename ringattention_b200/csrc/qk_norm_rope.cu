// RMS norm of each head's query and key and their rotation by position, in one pass, forward and backward.
//
//   n = x r,  r = 1 / sqrt(mean(x^2) + eps);   y = R(pos) (g n)        (R turns the pairs (i, i + D/2) by pos * theta^(-2i/D))
//   backward: u = R(pos)^T dy;  w = g u;  dx = r (w - n mean(w n));  dg = sum over rows of u n
//
// r is made again in the backward from x, which has to be read anyway: nothing is saved between the passes but the inputs. Both passes are
// bound by memory (forward: x in, y out; backward: x and dy in, dx out; about 8 and 20 operations an element).
//
// A row (one head of one token) is taken by D / 16 lanes: each has eight elements of the first half and their partners of the second, two
// 16-byte loads in bf16, so that the rotation needs no exchange and the sums log2(D / 16) shuffles. A warp takes the query heads or the key
// heads of a few tokens: it makes their sines and cosines once, in shared memory of its own, and walks the rows, with the loads of the next
// ones under way. Warps do not wait for one another (CTAs that share the table, with barriers: 16384 tokens of 32 and 8 heads of 128 forward / backward 96 / 153 us instead of 65 / 107).
//
// Angles: pos * theta^(-2i/D) / 2 pi in 64 bits, less the whole turns, then the fp32 sine and cosine of the rest: an fp32 angle is off by 0.03
// at position 10^6. The frequencies are made on the host in 64 bits and come as launch parameters (1 KB).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common/bounds.cuh"
#include "common/host_util.h"
#include "common/sm100.cuh"

RA_BOUNDS_TRANSLATION_UNIT()

namespace ra {
namespace qk {

constexpr int THREADS = 128;
constexpr int MAX_HALF = 128;  // of a head
constexpr int resident(bool bwd, bool f32) { return bwd ? (f32 ? 4 : 5) : 8; }  // CTAs an SM

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
  int tile[2];         // tokens a warp takes at a time, of queries and keys
  int ctas[2];         // CTAs of each: first the queries', then the keys'
  int gain_f32;
  // positions: token s of batch row b at pos[b * pos_sb + s * pos_ss] (32 or 64 bits), or, without pos, at off0 + s, from `half` on at
  // off1 + (s - half)
  const void* pos;
  int pos64;
  long long pos_sb, pos_ss;
  int off0, off1, half;
  float eps;
  float* part;         // backward: (gridDim.x, D) sums of the gains' gradients
  double freq[MAX_HALF];  // turns per position
};

template <typename T> struct Eight;  // eight elements of a row; in 32 bits as four pairs
template <> struct Eight<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(uint64_t* f) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = f2_pack_u(w[e] << 16, w[e] & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const uint64_t* f) {
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
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void get(uint64_t* f) const {
    f[0] = f2_pack(a.x, a.y);
    f[1] = f2_pack(a.z, a.w);
    f[2] = f2_pack(b.x, b.y);
    f[3] = f2_pack(b.z, b.w);
  }
  static __device__ __forceinline__ void store(float* p, const uint64_t* f) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) f2_unpack(f[e], v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
};

template <int LANES>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// cosines and sines of the tokens t0 .. t0 + n - 1, by one warp: turn[token][cos D / 2 | sin D / 2]
template <int D>
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
    float* to = turn + (i / (D / 2)) * D + f;
    to[0] = cs;
    to[D / 2] = sn;
  }
}

__device__ __forceinline__ void load_pairs(const float* p, uint64_t* v) {  // eight floats as pairs
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 f = reinterpret_cast<const float4*>(p)[i];
    v[2 * i] = f2_pack(f.x, f.y);
    v[2 * i + 1] = f2_pack(f.z, f.w);
  }
}

// BWD keeps the sums for the gain of its columns in registers: one row of partial sums a CTA, which dgain_kernel adds up in a fixed order. (A
// CTA that takes both sides needs twice the registers for them.)
template <typename T, int D, bool BWD>
__global__ void __launch_bounds__(THREADS, resident(BWD, sizeof(T) == 4)) qk_norm_rope_kernel(const Params p) {
  constexpr int LANES = D / 16, GROUPS = 32 / LANES, WARPS = THREADS / 32;
  extern __shared__ __align__(16) float turns[];  // [warp][tile][D]
  __shared__ __align__(16) float gain[D];
  __shared__ float red[BWD ? WARPS : 1][D];
  const int which = static_cast<int>(blockIdx.x) >= p.ctas[0];
  const int cta = static_cast<int>(blockIdx.x) - (which ? p.ctas[0] : 0);
  const Side& s = p.side[which];
  const int tile = p.tile[which], rows = tile * s.n;
  const int per_tile = (rows + GROUPS - 1) / GROUPS;  // steps
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / LANES, l = lane % LANES;
  float* const turn = turns + warp * p.tile[p.tile[1] > p.tile[0]] * D;
  for (int i = threadIdx.x; i < D; i += THREADS)
    gain[i] = p.gain_f32 ? static_cast<const float*>(s.gain)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(s.gain)[i]);
  __syncthreads();
  const unsigned tiles = (p.tokens + tile - 1) / tile, stride = static_cast<unsigned>(p.ctas[which]) * WARPS;
  const int tokens_step = GROUPS / s.n, heads_step = GROUPS - tokens_step * s.n;  // what a step adds to a row's token and head
  const int tt0 = group / s.n, h0 = group - tt0 * s.n;

  // the row of this lane: its tile's first token as batch row and place, token and head in the tile
  struct Place {
    unsigned t, b, at;
    int tt, h;
  };
  auto start = [&](unsigned t) {
    Place w;
    w.t = t * tile;
    w.b = w.t / static_cast<unsigned>(p.S);
    w.at = w.t - w.b * p.S;
    w.tt = tt0;
    w.h = h0;
    return w;
  };
  auto next_step = [&](Place& w) {
    w.tt += tokens_step;
    w.h += heads_step;
    if (w.h >= s.n) {
      w.h -= s.n;
      ++w.tt;
    }
  };
  auto inside = [&](const Place& w) { return w.tt < tile && w.t + w.tt < p.tokens; };
  // (a tile that reaches over the end of a batch row)
  auto offset = [&](const Place& w, long long sb, long long ss, long long sh) {
    unsigned b = w.b, at = w.at + w.tt;
    if (at >= static_cast<unsigned>(p.S)) {
      const unsigned over = at / static_cast<unsigned>(p.S);
      b += over;
      at -= over * p.S;
    }
    return b * sb + at * ss + w.h * sh + l * 8;
  };
  Eight<T> x[2], dy[BWD ? 2 : 1];
  auto load = [&](const Place& w) {
    if (!inside(w)) return;
    const T* from = static_cast<const T*>(s.x) + offset(w, s.x_sb, s.x_ss, s.x_sh);
    x[0].load(from);
    x[1].load(from + D / 2);
    if (BWD) {
      const T* d = static_cast<const T*>(s.dy) + offset(w, s.dy_sb, s.dy_ss, s.dy_sh);
      dy[0].load(d);
      dy[BWD ? 1 : 0].load(d + D / 2);
    }
  };
  uint64_t sum[BWD ? 8 : 1];
#pragma unroll
  for (int e = 0; e < (BWD ? 8 : 1); ++e) sum[e] = f2_pack(0.f, 0.f);

  unsigned t = static_cast<unsigned>(cta) * WARPS + warp;
  Place next = start(t);
  if (t < tiles) load(next);
  for (; t < tiles; t += stride) {
    __syncwarp();
    fill_turns<D>(p, t * tile, tile, turn, lane);
    __syncwarp();
    for (int step = 0; step < per_tile; ++step) {
      const Place w = next;
      const bool in = inside(w);
      uint64_t a[4], c[4], da[4], dc[4];
      if (in) {
        x[0].get(a);
        x[1].get(c);
        if (BWD) {
          dy[0].get(da);
          dy[BWD ? 1 : 0].get(dc);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = c[e] = da[e] = dc[e] = f2_pack(0.f, 0.f);
      }
      if (step + 1 < per_tile) {
        next_step(next);
        load(next);
      } else if (t + stride < tiles) {
        next = start(t + stride);
        load(next);
      }
      uint64_t ss2 = f2_pack(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) ss2 = f2_fma(c[e], c[e], f2_fma(a[e], a[e], ss2));
      float ss, ss_hi;
      f2_unpack(ss2, ss, ss_hi);
      const float rstd = rsqrtf(sum_lanes<LANES>(ss + ss_hi) * (1.f / D) + p.eps);
      const uint64_t r2 = f2_pack(rstd, rstd);
      uint64_t cs[4], sn[4];
      const float* tn = turn + (in ? w.tt * D : 0) + l * 8;
      load_pairs(tn, cs);
      load_pairs(tn + D / 2, sn);
      if constexpr (BWD) {
        uint64_t dot2 = f2_pack(0.f, 0.f), g0[4], g1[4];
        load_pairs(gain + l * 8, g0);
        load_pairs(gain + D / 2 + l * 8, g1);
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
        uint64_t g0[4], g1[4];
        load_pairs(gain + l * 8, g0);
        load_pairs(gain + D / 2 + l * 8, g1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t m = f2_mul(f2_mul(a[e], r2), g0[e]), k = f2_mul(f2_mul(c[e], r2), g1[e]);
          a[e] = f2_sub(f2_mul(m, cs[e]), f2_mul(k, sn[e]));
          c[e] = f2_fma(k, cs[e], f2_mul(m, sn[e]));
        }
      }
      if (in && RA_IN_BOUNDS(w.h, 1, s.n, kTagQkNorm)) {
        T* y = static_cast<T*>(s.y) + offset(w, s.y_sb, s.y_ss, s.y_sh);
        Eight<T>::store(y, a);
        Eight<T>::store(y + D / 2, c);
      }
    }
  }
  if constexpr (BWD) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v[2];
      f2_unpack(sum[e], v[0], v[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 16; o >= LANES; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        if (lane < LANES) red[warp][(e >> 2) * (D / 2) + l * 8 + (e & 3) * 2 + i] = v[i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += THREADS) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += red[w][i];
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
  for (int i = 0; i < a->D / 2; ++i) p.freq[i] = pow(a->theta, -2.0 * i / a->D) / 6.283185307179586476925;
  return kHostOk;
}
}  // namespace

namespace {
// Tiles and CTAs of both sides: tiles of eight steps of rows or so, at most eight tokens, fewer where that leaves warps without work; `resident` CTAs an
// SM, shared by queries and keys as their work is. (The sines and cosines of a token take a warp as long as two steps. Shared as the rows
// are, one key head beside 32 query heads took 16384 tokens 235 us instead of 59.)
void cut_up(ra::qk::Params& p, int D, int resident) {
  using namespace ra;
  constexpr int WARPS = qk::THREADS / 32;
  const int groups = 32 / (D / 16), all = p.side[0].n + p.side[1].n + 4 * groups;
  const long long room = static_cast<long long>(resident) * sm_count();
  for (int i = 0; i < 2; ++i) {
    const int n = p.side[i].n;
    int tile = 1;
    while (tile < 8 && 2 * tile * D <= 1024 && tile * n < 8 * groups && static_cast<long long>(p.tokens) * all >= 2 * tile * room * WARPS * (n + 2 * groups)) tile *= 2;
    const long long ctas = ((static_cast<long long>(p.tokens) + tile - 1) / tile + WARPS - 1) / WARPS;
    long long most = room * (n + 2 * groups) / all;
    if (most < 1) most = 1;
    p.tile[i] = tile;
    p.ctas[i] = static_cast<int>(ctas < most ? ctas : most);
  }
}
size_t turn_bytes(const ra::qk::Params& p, int D) {
  return static_cast<size_t>(p.tile[0] > p.tile[1] ? p.tile[0] : p.tile[1]) * D * sizeof(float) * (ra::qk::THREADS / 32);
}
}  // namespace

extern "C" int ra_qk_norm_rope(const RaQkNormArgs* a) {
  using namespace ra;
  using namespace ra::qk;
  Params p;
  if (int rc = to_params(a, false, p)) return rc;
  cut_up(p, a->D, resident(false, a->f32));
  auto kern = a->D == 64 ? (a->f32 ? qk_norm_rope_kernel<float, 64, false> : qk_norm_rope_kernel<__nv_bfloat16, 64, false>)
            : a->D == 128 ? (a->f32 ? qk_norm_rope_kernel<float, 128, false> : qk_norm_rope_kernel<__nv_bfloat16, 128, false>)
                          : (a->f32 ? qk_norm_rope_kernel<float, 256, false> : qk_norm_rope_kernel<__nv_bfloat16, 256, false>);
  kern<<<p.ctas[0] + p.ctas[1], THREADS, turn_bytes(p, a->D), static_cast<cudaStream_t>(a->stream)>>>(p);
  return check_launch("qk_norm_rope");
}

// Rows of partial sums that the backward may write (each D floats).
extern "C" int ra_qk_norm_parts() { return ra::qk::resident(true, false) * ra::sm_count() + 2; }

extern "C" int ra_qk_norm_rope_bwd(const RaQkNormArgs* a) {
  using namespace ra;
  using namespace ra::qk;
  Params p;
  if (int rc = to_params(a, true, p)) return rc;
  cut_up(p, a->D, resident(true, a->f32));
  if (!a->part || !a->dgain || a->parts < p.ctas[0] + p.ctas[1]) {
    set_error("qk_norm_rope_bwd: no room for the gains' gradients");
    return kHostBadArg;
  }
  auto kern = a->D == 64 ? (a->f32 ? qk_norm_rope_kernel<float, 64, true> : qk_norm_rope_kernel<__nv_bfloat16, 64, true>)
            : a->D == 128 ? (a->f32 ? qk_norm_rope_kernel<float, 128, true> : qk_norm_rope_kernel<__nv_bfloat16, 128, true>)
                          : (a->f32 ? qk_norm_rope_kernel<float, 256, true> : qk_norm_rope_kernel<__nv_bfloat16, 256, true>);
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  kern<<<p.ctas[0] + p.ctas[1], THREADS, turn_bytes(p, a->D), s>>>(p);
  if (int rc = check_launch("qk_norm_rope_bwd")) return rc;
  dgain_kernel<<<dim3(a->D / 8, 2), 1024, 0, s>>>(a->part, p.ctas[0], p.ctas[1], a->D, a->dgain, a->gain_f32);
  return check_launch("dgain");
}
