// Launchers of the flash-attention backward (attn_bwd_kernel.cuh) and its preparation.
#include "attn_bwd_kernel.cuh"

RA_BOUNDS_TRANSLATION_UNIT()

namespace ra {
namespace attn {

// Eight consecutive bf16 as floats; ALIGNED: the address is a multiple of 16 bytes (else of 4).
template <bool ALIGNED>
__device__ __forceinline__ void load8(const __nv_bfloat16* src, float* f) {
  uint4 u;
  if (ALIGNED) {
    u = *reinterpret_cast<const uint4*>(src);
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(src);
    u = make_uint4(w[0], w[1], w[2], w[3]);
  }
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 t = __bfloat1622float2(h[e]);
    f[2 * e] = t.x;
    f[2 * e + 1] = t.y;
  }
}

// delta[b,h,q] = sum_d dO*O ; lse2 = -lse*log2(e) (-inf where lse is -inf); padded rows get
// (-inf, 0) so that exp2(s*c + lse2) is 0 for them. With dq_acc the fp32 rows that dQ is reduced into are zeroed too.
// A CTA takes 64 (q, h) rows, up to eight heads of consecutive queries, so that its reads of o and d_o and its zeros
// are contiguous in a (B, S, H, D) tensor; D/8 lanes a row, all of a thread's loads issued before the first is used; the
// results turn in shared memory so that they leave as runs along q. It is bound by memory: one warp a row, rows a whole
// (H, D) line apart and 8 bytes a lane moved 2 TB/s (33 us at B1 S4096 H32 D128, beside 10 us for a fill kernel); this takes 29 us for both.
constexpr int PREP_ROWS = 64;
// LO: o_lo, with o's strides, holds what rounding took from o. Where one key has nearly all of a row's weight, dP - delta is the
// small difference of two numbers as large as dO O, and the 2^-9 that rounding takes from O can be as much as 1 % of it.
template <int D, bool ALIGNED, bool LO>
__global__ void __launch_bounds__(256) attn_bwd_prep_kernel(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ o_lo,
                                     long long o_sb, long long o_ss,
                                     long long o_sh, const __nv_bfloat16* __restrict__ d_o,
                                     long long do_sb, long long do_ss, long long do_sh,
                                     const float* __restrict__ lse, float* __restrict__ lse2,
                                     float* __restrict__ delta, float* __restrict__ dq_acc, int B, int H, int Sq,
                                     int Sq_pad, int heads_log2) {
  constexpr int LPR = D / 8, GROUPS = 256 / LPR, PER = PREP_ROWS / GROUPS;
  __shared__ float sum[PREP_ROWS];
  const int heads = 1 << heads_log2, qs = PREP_ROWS >> heads_log2, nq = Sq_pad / qs;
  const int b = static_cast<int>(blockIdx.x) / nq, q0 = (static_cast<int>(blockIdx.x) - b * nq) * qs, h0 = blockIdx.y * heads;
  const int grp = threadIdx.x / LPR, dl = (threadIdx.x % LPR) * 8;
  float fo[PER][8], fg[PER][8];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int r = grp + u * GROUPS, h = h0 + (r & (heads - 1)), q = q0 + (r >> heads_log2);
    if (h < H && q < Sq) {
      load8<ALIGNED>(o + b * o_sb + static_cast<long long>(q) * o_ss + h * o_sh + dl, fo[u]);
      if (LO) {
        float lo[8];
        load8<ALIGNED>(o_lo + b * o_sb + static_cast<long long>(q) * o_ss + h * o_sh + dl, lo);
#pragma unroll
        for (int e = 0; e < 8; ++e) fo[u][e] += lo[e];
      }
      load8<ALIGNED>(d_o + b * do_sb + static_cast<long long>(q) * do_ss + h * do_sh + dl, fg[u]);
      const long long at = ((static_cast<long long>(b) * Sq + q) * H + h) * D + dl;
      if (dq_acc && RA_IN_BOUNDS(at, 8, static_cast<long long>(B) * Sq * H * D, kTagAttnBwdPrep)) {
        *reinterpret_cast<float4*>(dq_acc + at) = make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(dq_acc + at + 4) = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) fo[u][e] = fg[u][e] = 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    float acc = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc += fo[u][e] * fg[u][e];
#pragma unroll
    for (int i = LPR / 2; i > 0; i >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, i);
    if (dl == 0) sum[grp + u * GROUPS] = acc;
  }
  __syncthreads();
  if (threadIdx.x < PREP_ROWS) {
    const int hl = static_cast<int>(threadIdx.x) / qs, ql = static_cast<int>(threadIdx.x) - hl * qs;
    const int h = h0 + hl, q = q0 + ql;
    const long long bh = static_cast<long long>(b) * H + h, at = bh * Sq_pad + q;
    if (h < H && RA_IN_BOUNDS(at, 1, static_cast<long long>(B) * H * Sq_pad, kTagAttnBwdPrep)) {
      const float l = q < Sq ? lse[bh * Sq + q] : -INFINITY;
      lse2[at] = l == -INFINITY ? -INFINITY : -l * kLog2e;
      delta[at] = sum[(ql << heads_log2) + hl];
    }
  }
}

}  // namespace attn
}  // namespace ra

namespace {
int make_bshd_map_bwd(CUtensorMap* m, const void* base, int B, int S, int H, int D, long long sb,
                      long long ss, long long sh) {
  uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(H), static_cast<uint64_t>(S),
                      static_cast<uint64_t>(B)};
  uint64_t str[3] = {static_cast<uint64_t>(sh) * 2, static_cast<uint64_t>(ss) * 2,
                     static_cast<uint64_t>(sb) * 2};
  uint32_t box[4] = {64, 1, 128, 1};
  return ra::make_tmap_bf16_sw128(m, base, 4, dims, str, box);
}
}  // namespace


extern "C" int ra_attn_bwd(const RaAttnBwdArgs* a) {
  using namespace ra;
  using namespace ra::attn;
  if (a->D != 128 && a->D != 64) {
    set_error("ra_attn_bwd: head_dim must be 64 or 128");
    return kHostBadArg;
  }
  if (a->B <= 0 || a->H <= 0 || a->Sq <= 0 || a->Sk <= 0 || (a->Sq_pad % 128) || a->Sq_pad < a->Sq ||
      (a->q_half < a->Sq && a->q_half % 128) || (a->k_half < a->Sk && a->k_half % 128) ||
      (a->copy_bytes % 16)) {
    set_error("ra_attn_bwd: bad shape");
    return kHostBadArg;
  }
  CUtensorMap tq, tk, tv, tdo;
  int rc;
  if ((rc = make_bshd_map_bwd(&tq, a->q, a->B, a->Sq, a->H, a->D, a->q_sb, a->q_ss, a->q_sh))) return rc;
  if ((rc = make_bshd_map_bwd(&tk, a->k, a->B, a->Sk, a->H, a->D, a->k_sb, a->k_ss, a->k_sh))) return rc;
  if ((rc = make_bshd_map_bwd(&tv, a->v, a->B, a->Sk, a->H, a->D, a->v_sb, a->v_ss, a->v_sh))) return rc;
  if ((rc = make_bshd_map_bwd(&tdo, a->d_o, a->B, a->Sq, a->H, a->D, a->do_sb, a->do_ss, a->do_sh)))
    return rc;
  CUtensorMap tdq;
  {
    if (reinterpret_cast<uintptr_t>(a->dq_acc) & 15) {
      set_error("ra_attn_bwd: dq_acc must be 16-byte aligned");
      return kHostBadArg;
    }
    uint64_t dims[4] = {static_cast<uint64_t>(a->D), static_cast<uint64_t>(a->H),
                        static_cast<uint64_t>(a->Sq), static_cast<uint64_t>(a->B)};
    uint64_t str[3] = {static_cast<uint64_t>(a->D) * 4, static_cast<uint64_t>(a->H) * a->D * 4,
                       static_cast<uint64_t>(a->Sq) * a->H * a->D * 4};
    uint32_t box[4] = {32, 1, 128, 1};
    if ((rc = make_tmap_f32_sw128(&tdq, a->dq_acc, 4, dims, str, box))) return rc;
  }
  BwdParams p;
  p.B = a->B;
  p.H = a->H;
  p.mask.Sq = a->Sq;
  p.mask.Sk = a->Sk;
  p.mask.cbs = a->causal_block_size;
  p.mask.qmap = PosMap{a->q_off0, a->q_off1, a->q_half};
  p.mask.kmap = PosMap{a->k_off0, a->k_off1, a->k_half};
  p.mask.seg_q = a->seg_q;
  p.mask.seg_k = a->seg_k;
  p.mask.seg_q_mm = a->seg_q_mm;
  p.mask.seg_k_mm = a->seg_k_mm;
  p.mask.bias = a->bias;
  p.mask.bias_stride_b = a->bias_sb;
  p.mask.bias_stride_h = a->bias_sh;
  p.mask.seed_lo = static_cast<unsigned int>(a->seed & 0xffffffffull);
  p.mask.seed_hi = static_cast<unsigned int>(a->seed >> 32);
  p.mask.drop_threshold = a->drop_threshold;
  p.mask.keep = a->keep;
  p.mask.keep_sb = a->keep_sb;
  p.mask.keep_sh = a->keep_sh;
  p.mask.keep_sr = a->keep_sr;
  p.mask.keep_tiles = a->keep_tiles;
  p.mask.keep_tiles_sb = a->keep_tiles_sb;
  p.mask.keep_tiles_sh = a->keep_tiles_sh;
  p.scale = a->softmax_scale;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.lse2 = a->lse2;
  p.delta = a->delta;
  p.Sq_pad = a->Sq_pad;
  p.dq_acc = a->dq_acc;
  p.dk = a->dk;
  p.dv = a->dv;
  p.dkv_sb = a->dkv_sb;
  p.dkv_ss = a->dkv_ss;
  p.dkv_sh = a->dkv_sh;
  p.dkv_mode = a->dkv_mode;
  p.copy_src = reinterpret_cast<const uint4*>(a->copy_src);
  p.copy_dst = reinterpret_cast<uint4*>(a->copy_dst);
  p.copy_n16 = a->copy_bytes / 16;
  p.copy_ctas = (a->copy_src && a->copy_bytes > 0) ? a->copy_ctas : 0;
  p.status = a->status;
  p.trace = a->trace;
  if (!(a->logit_cap >= 0.f) || a->logit_cap > 1e30f) {
    set_error("ra_attn_bwd: the cap must be positive and finite");
    return kHostBadArg;
  }
  p.shape = ShapeParams{tanh_params(a->softmax_scale, a->logit_cap), a->logit_cap * kLog2e, a->causal_block_size != 1 || a->prefix || a->q_from, a->slopes,
                        a->prefix, a->q_from, a->q_lo, a->q_hi};
  const int shape = (a->logit_cap > 0.f ? kShapeOn | kShapeCap : 0) | (a->slopes ? kShapeOn | kShapeSlopes : 0) | (a->prefix ? kShapeOn : 0);
  const int nkt = (a->Sk + 127) / 128;
  // a head's Q, dO and the fp32 dQ that is reduced into in L2: 8 bytes an element
  p.order = TileOrder{nkt, a->B * a->H,
                      a->causal_block_size ? head_groups(nkt, a->B * a->H, 8ll * a->Sq * a->D, sm_count()) : a->B * a->H};
  const long long grid = static_cast<long long>(nkt) * a->H * a->B + p.copy_ctas;
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  if (a->D == 128) {
    const BwdKernel kern = shape ? bwd_kernel_shaped(128, shape) : attn_bwd_kernel<128, 0>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdSmem<128>::TOTAL) !=
        cudaSuccess) {
      set_error("attn_bwd: smem attribute");
      return kHostLaunchFail;
    }
    kern<<<static_cast<unsigned>(grid), BWD_THREADS, BwdSmem<128>::TOTAL, s>>>(tq, tk, tv, tdo, tdq, p);
  } else {
    const BwdKernel kern = shape ? bwd_kernel_shaped(64, shape) : attn_bwd_kernel<64, 0>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdSmem<64>::TOTAL) !=
        cudaSuccess) {
      set_error("attn_bwd: smem attribute");
      return kHostLaunchFail;
    }
    kern<<<static_cast<unsigned>(grid), BWD_THREADS, BwdSmem<64>::TOTAL, s>>>(tq, tk, tv, tdo, tdq, p);
  }
  return check_launch("attn_bwd_kernel");
}

// Touch every kernel of this file on the current device so that its code is resident before a caller that
// can no longer afford implicit device allocations launches it (CUDA loads kernels lazily by default).
extern "C" int ra_attn_bwd_load_kernels(void) {
  using namespace ra;
  using namespace ra::attn;
  cudaFuncAttributes fa;
  if (cudaFuncGetAttributes(&fa, attn_bwd_kernel<128, 0>) != cudaSuccess ||
      cudaFuncGetAttributes(&fa, attn_bwd_kernel<64, 0>) != cudaSuccess ||
      cudaFuncGetAttributes(&fa, attn_bwd_prep_kernel<128, true, false>) != cudaSuccess ||
      cudaFuncGetAttributes(&fa, attn_bwd_prep_kernel<64, true, false>) != cudaSuccess ||
      cudaFuncGetAttributes(&fa, attn_bwd_prep_kernel<128, false, false>) != cudaSuccess ||
      cudaFuncGetAttributes(&fa, attn_bwd_prep_kernel<64, false, false>) != cudaSuccess) {
    set_error("ra_attn_bwd_load_kernels: cudaFuncGetAttributes failed");
    cudaGetLastError();
    return kHostLaunchFail;
  }
  return kHostOk;
}

// Backward preprocessing: delta and scaled lse into (B, H, Sq_pad) buffers, and, unless null, zeros into dq_acc (B, Sq, H, D)
// contiguous. o / d_o are (B, Sq, H, D) bf16 views with element strides.
extern "C" int ra_attn_bwd_prep_lo(const void* o, const void* o_lo, long long o_sb, long long o_ss, long long o_sh,
                                   const void* d_o, long long do_sb, long long do_ss, long long do_sh,
                                   const float* lse, float* lse2, float* delta, float* dq_acc, int B, int H, int Sq,
                                   int Sq_pad, int D, void* stream) {
  using namespace ra;
  using namespace ra::attn;
  if ((D != 128 && D != 64) || B < 1 || H < 1 || Sq < 1 || Sq_pad < Sq || Sq_pad % 128 ||
      (reinterpret_cast<uintptr_t>(dq_acc) & 15)) {
    set_error("ra_attn_bwd_prep: head_dim must be 64 or 128, Sq_pad a multiple of 128, dq_acc 16-byte aligned");
    return kHostBadArg;
  }
  const bool aligned = !((o_sb | o_ss | o_sh | do_sb | do_ss | do_sh) & 7) &&
                       !((reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(o_lo) | reinterpret_cast<uintptr_t>(d_o)) & 15);
  const int heads_log2 = H >= 5 ? 3 : (H >= 3 ? 2 : H - 1);
  const dim3 grid(static_cast<unsigned>(static_cast<long long>(B) * (Sq_pad / (PREP_ROWS >> heads_log2))),
                  static_cast<unsigned>((H + (1 << heads_log2) - 1) >> heads_log2));
  auto kern = D == 128 ? (aligned ? attn_bwd_prep_kernel<128, true, false> : attn_bwd_prep_kernel<128, false, false>)
                       : (aligned ? attn_bwd_prep_kernel<64, true, false> : attn_bwd_prep_kernel<64, false, false>);
  if (o_lo)
    kern = D == 128 ? (aligned ? attn_bwd_prep_kernel<128, true, true> : attn_bwd_prep_kernel<128, false, true>)
                    : (aligned ? attn_bwd_prep_kernel<64, true, true> : attn_bwd_prep_kernel<64, false, true>);
  kern<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(o), static_cast<const __nv_bfloat16*>(o_lo), o_sb, o_ss, o_sh, static_cast<const __nv_bfloat16*>(d_o), do_sb, do_ss, do_sh,
      lse, lse2, delta, dq_acc, B, H, Sq, Sq_pad, heads_log2);
  return check_launch("attn_bwd_prep_kernel");
}

extern "C" int ra_attn_bwd_prep(const void* o, long long o_sb, long long o_ss, long long o_sh,
                                const void* d_o, long long do_sb, long long do_ss, long long do_sh,
                                const float* lse, float* lse2, float* delta, float* dq_acc, int B, int H, int Sq,
                                int Sq_pad, int D, void* stream) {
  return ra_attn_bwd_prep_lo(o, nullptr, o_sb, o_ss, o_sh, d_o, do_sb, do_ss, do_sh, lse, lse2, delta, dq_acc, B, H, Sq, Sq_pad, D, stream);
}

RA_PACKED(ra_attn_bwd_prep)
RA_PACKED(ra_attn_bwd_prep_lo)
