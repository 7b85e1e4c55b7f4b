// Launchers of the flash-attention forward (attn_fwd_kernel.cuh): a ring step, two-part queries and keys, a window over a ring cache; how a
// launch is cut up, and the merge of one that is split over the keys.
#include "attn_fwd_kernel.cuh"

RA_BOUNDS_TRANSLATION_UNIT()

namespace ra {
namespace attn {

// Puts the partial results of a launch split over the keys together: o (splits, B, Sq, H, D) and lse (splits, B, H, Sq) fp32 ->
// out (bf16 or fp32 view) and lse_out (B, H, Sq). A warp per row. Every split's row is read and multiplied, by a weight of 0 where the
// split sees no key (lse = -inf) or its keys weigh nothing beside the others': NaN and infinities then come out as they do of a launch that is
// not split, where a probability of 0 meets them in the product with V. lse is NaN where a split's sum is.
// `out_lo`: as in FwdParams.
template <int D>
__global__ void __launch_bounds__(256) attn_merge_kernel(const float* __restrict__ o, const float* __restrict__ lse, int splits,
                                                         int B, int H, int Sq, void* out, int out_fp32, long long o_sb,
                                                         long long o_ss, long long o_sh, float* __restrict__ lse_out,
                                                         __nv_bfloat16* out_lo) {
  constexpr int PER = D / 32;
  const long long rows = static_cast<long long>(B) * Sq * H;
  const long long row = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int h = static_cast<int>(row % H), q = static_cast<int>(row / H % Sq), b = static_cast<int>(row / H / Sq);
  const long long at = (static_cast<long long>(b) * H + h) * Sq + q;
  float mx = -INFINITY;
  for (int s = 0; s < splits; ++s) mx = fmaxf(mx, lse[s * rows + at]);  // (of the numbers among them)
  float acc[PER], sum = 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float l = lse[s * rows + at];
    const float w = l == -INFINITY ? 0.f : expf(l - mx);
    const float* src = o + (s * rows + row) * D + lane * PER;
    sum += w;
#pragma unroll
    for (int e = 0; e < PER; e += 2) {
      const float2 v = *reinterpret_cast<const float2*>(src + e);
      acc[e] += w * v.x;
      acc[e + 1] += w * v.y;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (lane == 0 && RA_IN_BOUNDS(at, 1, rows, kTagAttnFwdLse)) lse_out[at] = sum > 0.f ? mx + logf(sum) : -INFINITY;
  const long long off = b * o_sb + static_cast<long long>(q) * o_ss + h * o_sh + lane * PER;
#pragma unroll
  for (int e = 0; e < PER; e += 2) {
    if (out_fp32) {
      *reinterpret_cast<float2*>(static_cast<float*>(out) + off + e) = make_float2(acc[e] * inv, acc[e + 1] * inv);
    } else {
      const uint32_t hi = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
      *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(out) + off + e) = hi;
      if (out_lo)
        *reinterpret_cast<uint32_t*>(out_lo + off + e) =
            pack_bf16x2(acc[e] * inv - __uint_as_float(hi << 16), acc[e + 1] * inv - __uint_as_float(hi & 0xffff0000u));
    }
  }
}

// How a launch is cut up: two query tiles a CTA ("pairs"), one (HALVES), or one and its keys over several CTAs. The estimate is the time of
// the launch in hundredths of a step of pairs (two 128 x 128 tiles; 1.8 us at D 128, 1.6 at D 64): a CTA takes its steps and a
// fixed cost (start-up, first loads, epilogue), and the CTAs, longest first, go to whichever SM is free: the SMs are busy for the average load at
// least, and the k-th CTA of an SM is no shorter than the longest that starts behind k - 1 full rounds. Segment ids and bitmaps are not
// looked at: the causal rule alone gives the lengths.
// The constants are fitted to 110 launches of both head dims timed in every form on B200 (256 to 32768 query rows, 2 to 32 heads, causal or not, up to
// 65536 keys): the choice takes 0.2 % longer than the fastest form on average, 6 % at worst (three of them more than 3 %). A step of HALVES
// loads K and V for one query tile only and takes as long as one of pairs all the same; its CTAs end later (the two groups' results
// are put together). us, pairs / HALVES / keys over 2 / over 4 CTAs, D 128, * the choice:
//   32 heads x 512, not causal 17.2 / 13.6* / 35.0 / -       32 x 4096, not causal 277* / 283 / - / -     32 x 4096, causal 153* / 182 / - / -
//   4 x 4096, causal 68.5 / 41.4* / 48.1 / 68.0              16 x 2048, not causal 40.7* / 49.9 / 92 / 126 16 x 500 on 16384 keys 245 / 136 / 85* / 99
//   32 x 1000 on 16384 keys 249* / 275 / 327 / 343           32 x 128 on 4096 keys 62 / 41 / 32 / 25*     2 x 12318, causal 187 / 106* / 120 / 149
// With constants of an earlier kernel (a step of HALVES 15 % longer, its CTA 1.4 steps shorter) the last of them went to keys over two CTAs, and the
// choice took 0.7 % longer than the fastest on average, 14 % at worst.
// Launches with shaped scores go by the same rule: they were not timed in every form. Their steps take 1.2 to 1.6 times as long beside the same fixed
// costs, and a prefix makes rows longer than the causal rule says, so their choice may be further from the fastest.
struct FwdShape {
  bool halves;
  int splits;
};
inline FwdShape fwd_shape(int B, int H, int Sq, int Sk, int D, int cbs, long long q_off, long long k_off, bool one_run, bool may_split) {
  const int step = D == 128 ? 99 : 102, cta = D == 128 ? 630 : 635, cta_pair = D == 128 ? 565 : 590;  // of HALVES, HALVES, pairs
  constexpr int step_pair = 100, merge = 425;  // merge: partial results out and in again, one more launch
  const int nk = (Sk + 127) / 128, nq = (Sq + 127) / 128, sms = sm_count();
  const long long bh = static_cast<long long>(B) * H;
  FwdShape best{false, 1};
  if (nq > 1024 || bh * nq > 64ll * sms) return best;  // plenty of work per SM: two query tiles share the loads of K and V
  auto tiles = [&](int i) -> long long {  // visible kv tiles of query tile i; no fewer than of the tile before
    const long long v = cbs && one_run ? (q_off + i * 128ll + 127 - k_off) / 128 + 1 : nk;
    return v < 0 ? 0 : (v > nk ? nk : v);
  };
  // `each` CTAs of each of n lengths, cost(0) the longest
  auto makespan = [&](int n, long long each, auto cost) -> long long {
    long long sum = 0;
    for (int i = 0; i < n; ++i) sum += cost(i);
    long long t = sum * each / sms;
    for (long long k = 1, at = 0; at < n * each; ++k, at += sms) {
      const long long c = k * cost(static_cast<int>(at / each));
      if (c > t) t = c;
    }
    return t;
  };
  long long t_best = makespan((nq + 1) / 2, bh, [&](int i) {
    const int later = 2 * ((nq + 1) / 2 - 1 - i) + 1;  // second tile of the i-th pair from the end
    return tiles(later < nq ? later : nq - 1) * step_pair + cta_pair;
  });
  long long all = 0;
  for (int i = 0; i < nq; ++i) all += tiles(i);
  for (int s = 1; s <= (may_split ? 32 : 1) && s <= nk; ++s) {
    const long long extra = s > 1 ? merge : 0;
    // more CTAs only add to the average load: no larger s is worth a look
    if (((all * step / 2 + static_cast<long long>(s) * nq * cta) * bh / sms + extra) * 100 >= t_best * 97) break;
    const long long t = extra + makespan(nq, bh * s, [&](int i) { return (tiles(nq - 1 - i) + 2 * s - 1) / (2 * s) * step + cta; });
    if (t * 100 < t_best * 97) {
      t_best = t;
      best = FwdShape{true, s};
    }
  }
  return best;
}

}  // namespace attn
}  // namespace ra

namespace {
// (B, S, H, D) bf16 view with element strides -> 4-D map (d, h, s, b), box 64 x 1 x 128 x 1.
int make_bshd_map(CUtensorMap* m, const void* base, int B, int S, int H, int D, long long sb,
                  long long ss, long long sh) {
  uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(H), static_cast<uint64_t>(S),
                      static_cast<uint64_t>(B)};
  uint64_t str[3] = {static_cast<uint64_t>(sh) * 2, static_cast<uint64_t>(ss) * 2,
                     static_cast<uint64_t>(sb) * 2};
  uint32_t box[4] = {64, 1, 128, 1};
  return ra::make_tmap_bf16_sw128(m, base, 4, dims, str, box);
}
}  // namespace

struct RaAttnFwdArgs {
  const void* q; const void* k; const void* v;
  long long q_sb, q_ss, q_sh;   // element strides of (B, Sq, H, D) views; D contiguous
  long long k_sb, k_ss, k_sh;
  long long v_sb, v_ss, v_sh;
  void* out; long long o_sb, o_ss, o_sh; int out_fp32;
  float* lse_out;
  const float* o_prev; const float* lse_prev;
  int B, H, Sq, Sk, D;
  float softmax_scale;          // 1/sqrt(D)
  int causal_block_size;
  int q_off0, q_off1, q_half;
  int k_off0, k_off1, k_half;
  const int* seg_q; const int* seg_k; const int* seg_q_mm; const int* seg_k_mm;
  const float* bias; long long bias_sb, bias_sh;
  unsigned long long seed; unsigned int drop_threshold;
  const unsigned int* keep; long long keep_sb, keep_sh, keep_sr;  // boolean mask bitmap by query row, or null
  const unsigned char* keep_tiles; long long keep_tiles_sb, keep_tiles_sh;  // kinds of its tiles, or null
  const void* copy_src; void* copy_dst; long long copy_bytes; int copy_ctas;
  int* status;
  void* stream;
  // splits > 1 (as ra_attn_fwd_splits says, or any number up to 32): the keys are split over that many CTAs per query tile; ws
  // holds splits * B * Sq * H * (D + 1) floats. Without o_prev and a copy job.
  int splits;
  float* ws;
  // shaped scores: cap (0: none), slopes (H), prefix (B) and the queries' first positions q_from (B) with their range (see ShapeParams), the last
  // three or null; out_lo: the rounding errors of a bf16 `out`, with its strides, or null
  float logit_cap;
  const float* slopes; const int* prefix; const int* q_from;
  int q_lo, q_hi;
  void* out_lo;
};

namespace {
int shape_bits(const RaAttnFwdArgs* a) {
  using namespace ra::attn;
  return (a->logit_cap > 0.f ? kShapeOn | kShapeCap : 0) | (a->slopes ? kShapeOn | kShapeSlopes : 0) | (a->prefix ? kShapeOn : 0);
}
ra::attn::FwdShape shape_of(const RaAttnFwdArgs* a, bool may_split) {
  const bool one_run = a->q_half >= a->Sq && a->k_half >= a->Sk;
  return ra::attn::fwd_shape(a->B, a->H, a->Sq, a->Sk, a->D, a->causal_block_size, a->q_off0, a->k_off0, one_run, may_split);
}
}  // namespace

// Over how many CTAs per query tile ra_attn_fwd would like to split the keys of this launch (1: not at all).
extern "C" int ra_attn_fwd_splits(const RaAttnFwdArgs* a) {
  if (a->B <= 0 || a->H <= 0 || a->Sq <= 0 || a->Sk <= 0) return 1;
  if (a->o_prev || a->copy_src || (a->Sk + 127) / 128 > 32 * ra::attn::VIS_WORDS) return 1;
  return shape_of(a, true).splits;
}

extern "C" int ra_attn_fwd(const RaAttnFwdArgs* a) {
  using namespace ra;
  using namespace ra::attn;
  if (a->D != 128 && a->D != 64) {
    set_error("ra_attn_fwd: head_dim must be 64 or 128");
    return kHostBadArg;
  }
  if (a->B <= 0 || a->H <= 0 || a->Sq <= 0 || a->Sk <= 0 || (a->q_half < a->Sq && a->q_half % 128) ||
      (a->k_half < a->Sk && a->k_half % 128) || (a->copy_bytes % 16)) {
    set_error("ra_attn_fwd: bad shape");
    return kHostBadArg;
  }
  const int splits = a->splits > 1 ? a->splits : 1;
  if (splits > 1 && (splits > 32 || !a->ws || (reinterpret_cast<uintptr_t>(a->ws) & 15) || a->o_prev || a->copy_src ||
                     !a->lse_out || (a->Sk + 127) / 128 > 32 * VIS_WORDS)) {
    set_error("ra_attn_fwd: a launch split over the keys takes a workspace, at most 32 splits, no carry and no copy job");
    return kHostBadArg;
  }
  if (!(a->logit_cap >= 0.f) || a->logit_cap > 1e30f || (a->out_lo && (a->out_fp32 || (reinterpret_cast<uintptr_t>(a->out_lo) & 15)))) {
    set_error("ra_attn_fwd: the cap must be positive and finite; rounding errors are those of a bf16 output");
    return kHostBadArg;
  }
  CUtensorMap tq, tk, tv;
  int rc;
  if ((rc = make_bshd_map(&tq, a->q, a->B, a->Sq, a->H, a->D, a->q_sb, a->q_ss, a->q_sh))) return rc;
  if ((rc = make_bshd_map(&tk, a->k, a->B, a->Sk, a->H, a->D, a->k_sb, a->k_ss, a->k_sh))) return rc;
  if ((rc = make_bshd_map(&tv, a->v, a->B, a->Sk, a->H, a->D, a->v_sb, a->v_ss, a->v_sh))) return rc;
  FwdParams p;
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
  if (a->keep && ((a->keep_sr % 4) || (a->keep_sb % 4) || (a->keep_sh % 4) || (reinterpret_cast<uintptr_t>(a->keep) & 15))) {
    set_error("ra_attn_fwd: mask bitmap rows must be 16-byte aligned");
    return kHostBadArg;
  }
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.out = a->out;
  p.out_fp32 = a->out_fp32;
  p.o_stride_b = a->o_sb;
  p.o_stride_s = a->o_ss;
  p.o_stride_h = a->o_sh;
  p.lse_out = a->lse_out;
  p.o_prev = a->o_prev;
  p.lse_prev = a->lse_prev;
  p.copy_src = reinterpret_cast<const uint4*>(a->copy_src);
  p.copy_dst = reinterpret_cast<uint4*>(a->copy_dst);
  p.copy_n16 = a->copy_bytes / 16;
  p.copy_ctas = (a->copy_src && a->copy_bytes > 0) ? a->copy_ctas : 0;
  p.status = a->status;
  p.dv = a->D;
  p.sink = nullptr;
  p.gate = nullptr;
  p.gate_ld = 0;
  p.window = p.kv_share = p.k_row0 = p.k_rows = 0;
  const float cap_log2 = a->logit_cap * kLog2e;
  const int shape = shape_bits(a);
  p.shape = ShapeParams{tanh_params(a->softmax_scale, a->logit_cap), cap_log2, a->causal_block_size != 1 || a->prefix || a->q_from, a->slopes, a->prefix,
                        a->q_from, a->q_lo, a->q_hi};
  p.out_lo = static_cast<__nv_bfloat16*>(a->out_lo);
  // A cap bounds the scores from both sides. With caps up to 80 (log2) a reference of at least cap - 90 keeps the exponentials below 2^90 and the
  // largest of a row above 2^-70: sums and products with V stay in the range of fp32 and bf16. A bias or a penalty could take all of
  // a row's keys further down. The bound from below is hardly ever met: a reference that is one of the row's own scores makes the weights near it
  // exact in bf16, one that is the same for all rows cost 5 % more error in dQ (0.00253 of its norm instead of 0.00245, 1 x 4096 tokens, 32 heads of 128).
  p.fixed_ref = a->logit_cap > 0.f && cap_log2 <= 80.f && !a->bias && !a->slopes;
  p.least_ref = cap_log2 - 90.f;
  const bool halves = splits > 1 || shape_of(a, false).halves;
  const int n_q = halves ? (a->Sq + 127) / 128 : (a->Sq + 255) / 256;
  p.order = TileOrder{n_q, a->B * a->H,
                      a->causal_block_size ? head_groups(n_q, a->B * a->H, 4ll * a->Sk * a->D, sm_count()) : a->B * a->H};
  p.splits = splits;
  p.split_l = static_cast<long long>(a->B) * a->H * a->Sq;
  p.split_o = p.split_l * a->D;
  if (splits > 1) {
    p.out = a->ws;
    p.out_fp32 = 1;
    p.o_stride_h = a->D;
    p.o_stride_s = static_cast<long long>(a->H) * a->D;
    p.o_stride_b = p.o_stride_s * a->Sq;
    p.lse_out = a->ws + splits * p.split_o;
  }
  const long long grid = static_cast<long long>(n_q) * a->H * a->B * splits + p.copy_ctas;
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  if (splits > 1) p.out_lo = nullptr;
  if (shape) {
    if (!launch_fwd_shaped) {
      set_error("ra_attn_fwd: this library was built without attn_fwd_shaped_sm100");
      return kHostBadArg;
    }
    rc = launch_fwd_shaped(tq, tk, tv, p, a->D, halves, shape, grid, s);
  } else if (a->out_lo) {
    set_error("ra_attn_fwd: rounding errors come with shaped scores only");
    return kHostBadArg;
  } else if (halves)
    rc = a->D == 128 ? launch_fwd<2, 0, 128, false, true>(tq, tk, tv, tq, tk, p, grid, s)
                     : launch_fwd<1, 0, 64, false, true>(tq, tk, tv, tq, tk, p, grid, s);
  else
    rc = a->D == 128 ? launch_fwd<2, 0, 128>(tq, tk, tv, tq, tk, p, grid, s)
                     : launch_fwd<1, 0, 64>(tq, tk, tv, tq, tk, p, grid, s);
  if (rc || splits == 1) return rc;
  const unsigned blocks = static_cast<unsigned>((p.split_l + 7) / 8);
  auto merge = a->D == 128 ? attn_merge_kernel<128> : attn_merge_kernel<64>;
  merge<<<blocks, 256, 0, s>>>(static_cast<const float*>(p.out), p.lse_out, splits, a->B, a->H, a->Sq, a->out, a->out_fp32, a->o_sb,
                               a->o_ss, a->o_sh, a->lse_out, static_cast<__nv_bfloat16*>(a->out_lo));
  return check_launch("attn_merge_kernel");
}

// Causal attention with two-part queries and keys: score = (q1 . k1 + q2 . k2) * scale, where k2 is shared by all heads.
// q (B, Sq, H, d1 + d2) with q1 first, k1 (B, Sk, H, d1), k2 (B, Sk, d2), v (B, Sk, H, dv), out (B, Sq, H, dv); bf16, element
// strides, innermost contiguous; query i sits at position q_pos0 + i, key j at j. d1 <= 128, d2 <= 64, dv <= 128, all
// multiples of 8. `sink` (H) fp32 and `gate` (B * Sq, gate_ld) bf16 are optional (see FwdParams).
struct RaAttnTwoPartArgs {
  const void* q; long long q_sb, q_ss, q_sh;
  const void* k1; long long k1_sb, k1_ss, k1_sh;
  const void* k2; long long k2_sb, k2_ss;
  const void* v; long long v_sb, v_ss, v_sh;
  void* out; long long o_sb, o_ss, o_sh;
  const float* sink;
  const void* gate; long long gate_ld;
  int B, H, Sq, Sk, d1, d2, dv;
  float scale;
  int q_pos0;
  int* status;
  void* stream;
};

extern "C" int ra_attn_two_part(const RaAttnTwoPartArgs* a) {
  using namespace ra;
  using namespace ra::attn;
  const long long odd = (a->q_sb | a->q_ss | a->q_sh | a->k1_sb | a->k1_ss | a->k1_sh | a->k2_sb | a->k2_ss | a->v_sb |
                         a->v_ss | a->v_sh | a->o_sb | a->o_ss | a->o_sh) & 7;
  if (a->B < 1 || a->H < 1 || a->Sq < 1 || a->Sk < 1 || a->q_pos0 < 0 || a->d1 < 8 || a->d1 > 128 || a->d1 % 8 ||
      a->d2 < 8 || a->d2 > 64 || a->d2 % 8 || a->dv < 8 || a->dv > 128 || a->dv % 8 || odd ||
      ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k1) | reinterpret_cast<uintptr_t>(a->k2) |
        reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->out)) & 15)) {
    set_error("ra_attn_two_part: bad shape or alignment");
    return kHostBadArg;
  }
  CUtensorMap tq, tk, tv, tq2, tk2;
  int rc;
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a->q);
  if ((rc = make_bshd_map(&tq, q, a->B, a->Sq, a->H, a->d1, a->q_sb, a->q_ss, a->q_sh))) return rc;
  if ((rc = make_bshd_map(&tq2, q + a->d1, a->B, a->Sq, a->H, a->d2, a->q_sb, a->q_ss, a->q_sh))) return rc;
  if ((rc = make_bshd_map(&tk, a->k1, a->B, a->Sk, a->H, a->d1, a->k1_sb, a->k1_ss, a->k1_sh))) return rc;
  if ((rc = make_bshd_map(&tk2, a->k2, a->B, a->Sk, 1, a->d2, a->k2_sb, a->k2_ss, a->k2_ss))) return rc;
  if ((rc = make_bshd_map(&tv, a->v, a->B, a->Sk, a->H, a->dv, a->v_sb, a->v_ss, a->v_sh))) return rc;
  FwdParams p = {};
  p.B = a->B;
  p.H = a->H;
  p.mask.Sq = a->Sq;
  p.mask.Sk = a->Sk;
  p.mask.cbs = 1;
  p.mask.qmap = PosMap{a->q_pos0, 0, 1 << 30};
  p.mask.kmap = PosMap{0, 0, 1 << 30};
  p.scale_log2 = a->scale * kLog2e;
  p.out = a->out;
  p.o_stride_b = a->o_sb;
  p.o_stride_s = a->o_ss;
  p.o_stride_h = a->o_sh;
  p.status = a->status;
  p.dv = a->dv;
  p.sink = a->sink;
  p.gate = static_cast<const __nv_bfloat16*>(a->gate);
  p.gate_ld = a->gate_ld;
  const int n_qp = (a->Sq + 255) / 256;
  p.order = TileOrder{n_qp, a->B * a->H, a->B * a->H};
  const long long grid = static_cast<long long>(n_qp) * a->H * a->B;
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  if (a->d1 > 64)
    return a->dv > 64 ? launch_fwd<2, 1, 128>(tq, tk, tv, tq2, tk2, p, grid, s)
                      : launch_fwd<2, 1, 64>(tq, tk, tv, tq2, tk2, p, grid, s);
  return a->dv > 64 ? launch_fwd<1, 1, 128>(tq, tk, tv, tq2, tk2, p, grid, s)
                    : launch_fwd<1, 1, 64>(tq, tk, tv, tq2, tk2, p, grid, s);
}

// Causal attention over the last `window` keys with grouped heads, a sink per head and keys and values in a ring: query i sits
// at position q_pos0 + i and sees the keys at distances 0 .. window - 1; position j lies in row j % k_rows, k_rows a multiple
// of 128. Head h reads key/value head h / (H / G). q (B, Sq, H, dk), k (B, k_rows, G, dk), v (B, k_rows, G, dv), out (B, Sq,
// H, dv): bf16, element strides, innermost contiguous; dk and dv multiples of 8 up to 128. `sink` (H) fp32.
struct RaAttnWindowArgs {
  const void* q; long long q_sb, q_ss, q_sh;
  const void* k; long long k_sb, k_ss, k_sh;
  const void* v; long long v_sb, v_ss, v_sh;
  void* out; long long o_sb, o_ss, o_sh;
  const float* sink;
  int B, H, G, Sq, dk, dv, window, k_rows;
  float scale;
  long long q_pos0;
  int* status;
  void* stream;
};

extern "C" int ra_attn_window(const RaAttnWindowArgs* a) {
  using namespace ra;
  using namespace ra::attn;
  const long long odd = (a->q_sb | a->q_ss | a->q_sh | a->k_sb | a->k_ss | a->k_sh | a->v_sb | a->v_ss | a->v_sh | a->o_sb |
                         a->o_ss | a->o_sh) & 7;
  if (a->B < 1 || a->G < 1 || a->H < 1 || a->H % a->G || a->Sq < 1 || a->q_pos0 < 0 || a->window < 1 || a->dk < 8 ||
      a->dk > 128 || a->dk % 8 || a->dv < 8 || a->dv > 128 || a->dv % 8 || a->k_rows < 128 || a->k_rows % 128 || odd ||
      ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
        reinterpret_cast<uintptr_t>(a->out)) & 15)) {
    set_error("ra_attn_window: bad shape or alignment");
    return kHostBadArg;
  }
  // the first tile with a visible key; everything below counts keys from there
  const long long lo = a->q_pos0 - a->window + 1, base = lo > 0 ? lo / 128 * 128 : 0;
  const long long n_keys = a->q_pos0 + a->Sq - base;
  if (n_keys > a->k_rows || n_keys > (1 << 30)) {
    set_error("ra_attn_window: the ring does not hold the window of this step");
    return kHostBadArg;
  }
  CUtensorMap tq, tk, tv;
  int rc;
  if ((rc = make_bshd_map(&tq, a->q, a->B, a->Sq, a->H, a->dk, a->q_sb, a->q_ss, a->q_sh))) return rc;
  if ((rc = make_bshd_map(&tk, a->k, a->B, a->k_rows, a->G, a->dk, a->k_sb, a->k_ss, a->k_sh))) return rc;
  if ((rc = make_bshd_map(&tv, a->v, a->B, a->k_rows, a->G, a->dv, a->v_sb, a->v_ss, a->v_sh))) return rc;
  FwdParams p = {};
  p.B = a->B;
  p.H = a->H;
  p.mask.Sq = a->Sq;
  p.mask.Sk = static_cast<int>(n_keys);
  p.mask.cbs = 1;
  p.mask.qmap = PosMap{static_cast<int>(a->q_pos0 - base), 0, 1 << 30};
  p.mask.kmap = PosMap{0, 0, 1 << 30};
  p.scale_log2 = a->scale * kLog2e;
  p.out = a->out;
  p.o_stride_b = a->o_sb;
  p.o_stride_s = a->o_ss;
  p.o_stride_h = a->o_sh;
  p.status = a->status;
  p.dv = a->dv;
  p.sink = a->sink;
  p.window = a->window;
  p.kv_share = a->H / a->G;
  p.k_row0 = static_cast<int>(base % a->k_rows);
  p.k_rows = a->k_rows;
  const int n_qp = (a->Sq + 255) / 256;
  p.order = TileOrder{n_qp, a->B * a->H, a->B * a->H};
  const long long grid = static_cast<long long>(n_qp) * a->H * a->B;
  cudaStream_t s = static_cast<cudaStream_t>(a->stream);
  if (a->dk > 64)
    return a->dv > 64 ? launch_fwd<2, 0, 128, true>(tq, tk, tv, tq, tk, p, grid, s)
                      : launch_fwd<2, 0, 64, true>(tq, tk, tv, tq, tk, p, grid, s);
  return a->dv > 64 ? launch_fwd<1, 0, 128, true>(tq, tk, tv, tq, tk, p, grid, s)
                    : launch_fwd<1, 0, 64, true>(tq, tk, tv, tq, tk, p, grid, s);
}
