// Flash-attention backward for sm_100a: one fused kernel, five GEMMs per (q tile, kv tile) pair.
//
// One CTA owns a 128-row KV tile of one (batch, head); K and V stay resident in shared memory and
// the CTA walks the visible 128-row query tiles i:
//     S^T  = K Q_i^T            (SS)  -> TMEM [0,128)
//     dP^T = V dO_i^T           (SS)  -> TMEM [128,256)
//     P^T  = exp2(S^T*c - lse)        -> packed bf16 over S^T (TMEM)
//     dS^T = P^T (dP^T - delta)       -> bf16 in shared memory (128-byte swizzle); the 1/sqrt(D)
//                                        factor is applied when dQ and dK leave TMEM
//     dV  += P^T dO_i           (A from TMEM)        -> TMEM [256,256+D)
//     dK  += dS^T Q_i           (A = dS^T, K-major)  -> TMEM [384,384+D)
//     dQ_i = dS K               (A = dS^T read MN-major, B = K MN-major) -> TMEM over dP^T
// dQ_i is added to an fp32 buffer with bulk tensor reductions (TMA, staged through shared memory); dK/dV leave through the epilogue as
// bf16, fp32 or as fp32 reductions into (possibly a peer GPU's) accumulators, which is how the
// ring backward returns gradients to the owner of the KV block.
//
//   warps 0-3    producer group (registers trimmed): warp 0 TMA (K,V once; Q_i + lse/delta
//                double-buffered; dO_i), warp 1 tcgen05.mma issuer
//   warps 4-11   softmax/dS group: two warps per TMEM lane quadrant, 64 q-columns each
//   warps 12-15  dQ drain group (registers raised): tcgen05.ld, early release, bulk reduce-add
#pragma once
#include "attn_api.h"
#include "attn_common.cuh"
#include "common/host_util.h"

namespace ra {
namespace attn {

constexpr int BWD_THREADS = 512;
// Register re-balancing: the CTA owns 512 x 128 registers (launch bounds); setmaxnreg.inc blocks
// until registers are free, so the per-group budgets must fit in that allocation.
constexpr int BWD_REGS_PRODUCER = 80;  // warps 0-3
constexpr int BWD_REGS_SOFTMAX = 144;  // warps 4-11
constexpr int BWD_REGS_DRAIN = 144;    // warps 12-15
static_assert(128 * BWD_REGS_PRODUCER + 256 * BWD_REGS_SOFTMAX + 128 * BWD_REGS_DRAIN <= BWD_THREADS * 128,
              "setmaxnreg budgets exceed the registers the CTA was launched with");

struct BwdParams {
  int B, H;
  TileOrder order;  // of the 128-row kv tiles
  MaskParams mask;
  float scale;       // 1/sqrt(D)
  float scale_log2;  // log2(e)/sqrt(D)
  const float* lse2;   // (B, H, Sq_pad): -lse*log2(e), -inf for fully masked / padded rows
  const float* delta;  // (B, H, Sq_pad): rowsum(dO * O)
  int Sq_pad;
  float* dq_acc;       // (B, Sq, H, D) fp32 contiguous, accumulated with reductions
  void* dk; void* dv;  // (B, Sk, H, D) with strides below
  long long dkv_sb, dkv_ss, dkv_sh;
  int dkv_mode;        // 0: store bf16, 1: store fp32, 2: fp32 reduction (system scope)
  const uint4* copy_src;
  uint4* copy_dst;
  long long copy_n16;
  int copy_ctas;
  int* status;
  long long* trace;  // optional phase timestamps of the first compute CTA: [role 0..3][64 iterations][4]
  ShapeParams shape;  // SHAPED: shaped scores
};

template <int D>
struct BwdSmem {
  static constexpr int TILE_BYTES = 128 * D * 2;
  static constexpr int SLAB_BYTES = 128 * 64 * 2;
  static constexpr int K_OFF = 0;
  static constexpr int V_OFF = K_OFF + TILE_BYTES;
  static constexpr int Q_OFF = V_OFF + TILE_BYTES;        // 2 stages
  static constexpr int DO_OFF = Q_OFF + 2 * TILE_BYTES;   // 1 stage
  static constexpr int DS_OFF = DO_OFF + TILE_BYTES;      // 128 x 128 bf16
  static constexpr int DQ_OFF = DS_OFF + 128 * 128 * 2;   // dQ staging: 128 rows x 32 fp32, swizzled
  static constexpr int LSE_OFF = DQ_OFF + 128 * 32 * 4;   // [2 stages][lse2 128 | delta 128]
  static constexpr int SEG_OFF = LSE_OFF + 2 * 256 * 4;   // [2][128] int
  static constexpr int BAR_OFF = SEG_OFF + 2 * 128 * 4;
  static constexpr int VIS_OFF = BAR_OFF + 256;  // [VIS_WORDS] visibility of the q tiles
  static constexpr int TOTAL = VIS_OFF + VIS_WORDS * 4 + 1024;
};

__device__ __forceinline__ void bulk_load_1d(void* dst, const void* src, uint32_t bytes,
                                             uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void red_add_v4(float* addr, float a, float b, float c, float d) {
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(addr), "f"(a), "f"(b), "f"(c),
               "f"(d)
               : "memory");
}
__device__ __forceinline__ void red_add_v4_sys(float* addr, float a, float b, float c, float d) {
  asm volatile("red.relaxed.sys.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(addr), "f"(a),
               "f"(b), "f"(c), "f"(d)
               : "memory");
}

// Phase timestamps (SM clock) for pipeline analysis; only the first compute CTA records, only its
// first 64 iterations, and only when the launch was given a trace buffer (RaAttnBwdArgs::trace).
__device__ __forceinline__ void trace_event(long long* trace, bool on, int role, int it, int slot) {
  if (on && it < 64) trace[(role * 64 + it) * 4 + slot] = clock64();
}

// SHAPE (bits of the scores' shape): the scores are made again as the forward made them; dS gets the derivative of the cap, 1 - tanh^2, which is multiplied into
// the probabilities that wait for dP (their unmultiplied copy, P^T for dV, is in TMEM by then).
template <int D, int SHAPE>
__global__ void __launch_bounds__(BWD_THREADS, 1)
attn_bwd_kernel(const __grid_constant__ CUtensorMap tma_q, const __grid_constant__ CUtensorMap tma_k,
                const __grid_constant__ CUtensorMap tma_v, const __grid_constant__ CUtensorMap tma_do,
                const __grid_constant__ CUtensorMap tma_dq, const BwdParams p) {
  using SM = BwdSmem<D>;
  constexpr int NSLAB = D / 64;
  constexpr bool SHAPED = SHAPE != 0;

  // A failure recorded earlier on this stream (for example a ring barrier that timed out) turns
  // every later attention kernel into a no-op, so nothing touches the memory of a lost peer.
  if (p.status && *reinterpret_cast<const volatile int*>(p.status) != 0) return;

  if (static_cast<int>(blockIdx.x) < p.copy_ctas) {
    const long long stride = static_cast<long long>(p.copy_ctas) * BWD_THREADS;
    long long i = static_cast<long long>(blockIdx.x) * BWD_THREADS + threadIdx.x;
    // 16 loads of 16 bytes in flight per thread (the pull is bound by bytes in flight over NVLink)
    for (; i + 15 * stride < p.copy_n16; i += 16 * stride) {
      uint4 r[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) r[u] = p.copy_src[i + u * stride];
#pragma unroll
      for (int u = 0; u < 16; ++u) p.copy_dst[i + u * stride] = r[u];
    }
    for (; i < p.copy_n16; i += stride) p.copy_dst[i] = p.copy_src[i];
    return;
  }

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sK = smem + SM::K_OFF;
  uint8_t* sV = smem + SM::V_OFF;
  uint8_t* sQ = smem + SM::Q_OFF;
  uint8_t* sDO = smem + SM::DO_OFF;
  uint8_t* sDS = smem + SM::DS_OFF;
  uint8_t* sDQ = smem + SM::DQ_OFF;
  float* sLse = reinterpret_cast<float*>(smem + SM::LSE_OFF);  // [stage][-lse2 128 | delta 128]
  int* sSegQ = reinterpret_cast<int*>(smem + SM::SEG_OFF);     // [buf][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::BAR_OFF);
  uint64_t* kv_full = bars;        // 1
  uint64_t* q_full = bars + 1;     // 2
  uint64_t* q_empty = bars + 3;    // 2
  uint64_t* do_full = bars + 5;
  uint64_t* do_empty = bars + 6;
  uint64_t* s_full = bars + 7;
  uint64_t* dp_full = bars + 8;
  uint64_t* p_ready = bars + 9;    // 256 arrivals
  uint64_t* ds_ready = bars + 10;  // 256 arrivals
  uint64_t* dq_full = bars + 11;
  uint64_t* dq_empty = bars + 12;  // 128 arrivals
  uint64_t* acc_full = bars + 13;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const WaitCtx wc{abort_flag, p.status};
  const MaskParams& mk = p.mask;

  const int nqt = (mk.Sq + 127) / 128;
  const int idx = static_cast<int>(blockIdx.x) - p.copy_ctas;
  int bh, jt;
  p.order(idx, jt, bh);  // kv tile; low tiles see the most queries under a causal mask
  const int h = bh % p.H;
  const int b = bh / p.H;
  const int k0 = jt * 128;
  const bool tr = p.trace != nullptr && idx == 0;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
    }
    mbar_init(do_full, 1);
    mbar_init(do_empty, 1);
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_ready, 256);
    mbar_init(ds_ready, 256);
    mbar_init(dq_full, 1);
    mbar_init(dq_empty, 128);
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tma_q);
    tma_prefetch_desc(&tma_k);
    tma_prefetch_desc(&tma_v);
    tma_prefetch_desc(&tma_do);
    tma_prefetch_desc(&tma_dq);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // which q tiles this kv tile is seen by
  uint32_t* sVis = reinterpret_cast<uint32_t*>(smem + SM::VIS_OFF);
  const bool use_vis = nqt <= 32 * VIS_WORDS;
  // a tile of keys whose bias is -inf throughout (padding) is seen by no query
  bool dead = false;
  if (mk.bias) {
    const int kj = k0 + static_cast<int>(threadIdx.x);
    const float* bias = mk.bias + b * mk.bias_stride_b + h * mk.bias_stride_h;
    dead = __syncthreads_and(threadIdx.x >= 128 || kj >= mk.Sk || bias[kj] * kLog2e == -INFINITY) != 0;
  }
  const int prefix = SHAPED && p.shape.prefix ? p.shape.prefix[b] : 0;
  if (use_vis)
    fill_visibility(sVis, nqt, static_cast<int>(threadIdx.x), BWD_THREADS,
                    [&](int i) { return !dead && tile_visible<SHAPED>(mk, b, h, i * 128, k0, prefix); });
  // next q tile at or after i that sees this kv tile, or nqt; every role walks the same mask
  auto next_vis = [&](int i) -> int {
    if (use_vis) return vis_next(sVis, i, nqt);
    if (dead) return nqt;
    for (; i < nqt; ++i)
      if (tile_visible<SHAPED>(mk, b, h, i * 128, k0, prefix)) break;
    return i;
  };
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tS = tmem_base;         // S^T, then packed P^T (cols 0-31 and 64-95)
  const uint32_t tDP = tmem_base + 128;  // dP^T, then dQ_i
  const uint32_t tDV = tmem_base + 256;
  const uint32_t tDK = tmem_base + 384;

  if (warp < 4) {
    // ================================================================ producer warpgroup
    setmaxnreg_dec<BWD_REGS_PRODUCER>();
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- TMA producer
      mbar_arrive_expect_tx(kv_full, 2 * SM::TILE_BYTES);
#pragma unroll
      for (int s = 0; s < NSLAB; ++s) {
        tma_load_4d(sK + s * SM::SLAB_BYTES, &tma_k, kv_full, s * 64, h, k0, b);
        tma_load_4d(sV + s * SM::SLAB_BYTES, &tma_v, kv_full, s * 64, h, k0, b);
      }
      int it = 0;
      for (int i = next_vis(0); i < nqt; i = next_vis(i + 1)) {
        const int qi0 = i * 128;
        const int st = it & 1;
        if (!mbar_wait_relaxed(&q_empty[st], ((it >> 1) & 1) ^ 1u, wc, kTimeoutSmemEmpty)) break;
        mbar_arrive_expect_tx(&q_full[st], SM::TILE_BYTES + 1024);
#pragma unroll
        for (int s = 0; s < NSLAB; ++s)
          tma_load_4d(sQ + st * SM::TILE_BYTES + s * SM::SLAB_BYTES, &tma_q, &q_full[st], s * 64, h,
                      qi0, b);
        const long long row_off = (static_cast<long long>(b) * p.H + h) * p.Sq_pad + qi0;
        bulk_load_1d(sLse + st * 256, p.lse2 + row_off, 512, &q_full[st]);
        bulk_load_1d(sLse + st * 256 + 128, p.delta + row_off, 512, &q_full[st]);
        if (it > 0 && !mbar_wait_relaxed(do_empty, (it - 1) & 1, wc, kTimeoutSmemEmpty)) break;
        mbar_arrive_expect_tx(do_full, SM::TILE_BYTES);
#pragma unroll
        for (int s = 0; s < NSLAB; ++s)
          tma_load_4d(sDO + s * SM::SLAB_BYTES, &tma_do, do_full, s * 64, h, qi0, b);
        ++it;
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA issuer (warp-uniform flow)
      const bool leader = elect_one();
      constexpr uint32_t idesc_s = make_idesc_bf16(128, 128, 0, 0);
      constexpr uint32_t idesc_dv = make_idesc_bf16(128, D, 0, 1);
      constexpr uint32_t idesc_dq = make_idesc_bf16(128, D, 1, 1);
      constexpr uint32_t SLAB = SM::SLAB_BYTES;
      // descriptor bases: *_k = K-major view (rows of 128 B along the reduction dim),
      // *_mn = MN-major view of the same bytes (64-wide slabs SLAB bytes apart)
      const uint64_t k_k = make_smem_desc(smem_u32(sK), 16, 1024);
      const uint64_t k_mn = make_smem_desc(smem_u32(sK), SLAB, 1024);
      const uint64_t v_k = make_smem_desc(smem_u32(sV), 16, 1024);
      const uint64_t do_k = make_smem_desc(smem_u32(sDO), 16, 1024);
      const uint64_t do_mn = make_smem_desc(smem_u32(sDO), SLAB, 1024);
      const uint64_t ds_mn = make_smem_desc(smem_u32(sDS), SLAB, 1024);
      const uint64_t q_k[2] = {make_smem_desc(smem_u32(sQ), 16, 1024),
                               make_smem_desc(smem_u32(sQ + SM::TILE_BYTES), 16, 1024)};
      const uint64_t q_mn[2] = {make_smem_desc(smem_u32(sQ), SLAB, 1024),
                                make_smem_desc(smem_u32(sQ + SM::TILE_BYTES), SLAB, 1024)};
      auto issue_st = [&](int st) {  // S^T = K Q^T
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * SLAB + (kk & 3) * 32;
          if (leader)
            umma_ss(tS, desc_advance(k_k, off), desc_advance(q_k[st], off), idesc_s, kk != 0 ? 1u : 0u);
        }
        if (leader) umma_commit(s_full);
      };
      auto next_visible = [&](int i) { return next_vis(i); };
      bool ok = mbar_wait(kv_full, 0, wc, kTimeoutSmemFull);
      int i = next_visible(0);
      int it = 0;
      if (ok && i < nqt) {
        ok = mbar_wait(&q_full[0], 0, wc, kTimeoutSmemFull);
        if (ok) {
          tc_fence_after();
          issue_st(0);
        }
      }
      while (ok && i < nqt) {
        const int st = it & 1;
        const uint32_t par = it & 1;
        // dP^T = V dO^T (its region doubles as dQ: wait until the previous dQ left TMEM)
        if (!mbar_wait(do_full, par, wc, kTimeoutSmemFull)) break;
        if (it > 0 && !mbar_wait(dq_empty, (it - 1) & 1, wc, kTimeoutTmemEmpty)) break;
        tc_fence_after();
        trace_event(p.trace, tr && leader, 0, it, 0);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * SLAB + (kk & 3) * 32;
          if (leader)
            umma_ss(tDP, desc_advance(v_k, off), desc_advance(do_k, off), idesc_s, kk != 0 ? 1u : 0u);
        }
        if (leader) umma_commit(dp_full);
        // dV += P^T dO
        if (!mbar_wait(p_ready, par, wc, kTimeoutTmemFull)) break;
        tc_fence_after();
        trace_event(p.trace, tr && leader, 0, it, 1);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t a_col = tS + (kk < 4 ? kk * 8 : 64 + (kk - 4) * 8);
          if (leader)
            umma_ts(tDV, a_col, desc_advance(do_mn, kk * 2048), idesc_dv, (it != 0 || kk != 0) ? 1u : 0u);
        }
        if (leader) umma_commit(do_empty);
        // next S^T right away (P^T was consumed by the dV MMAs just issued), so that the softmax
        // group can work on it while dK/dQ of this iteration run
        const int in = next_visible(i + 1);
        if (in < nqt) {
          const int stn = (it + 1) & 1;
          if (!mbar_wait(&q_full[stn], ((it + 1) >> 1) & 1, wc, kTimeoutSmemFull)) break;
          tc_fence_after();
          issue_st(stn);
        }
        // dK += dS^T Q ; dQ_i = dS K
        if (!mbar_wait(ds_ready, par, wc, kTimeoutTmemFull)) break;
        tc_fence_after();
        trace_event(p.trace, tr && leader, 0, it, 2);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t a_col = tDP + (kk < 4 ? kk * 8 : 64 + (kk - 4) * 8);  // dS^T in TMEM, laid out like P^T
          if (leader)
            umma_ts(tDK, a_col, desc_advance(q_mn[st], kk * 2048), idesc_dv, (it != 0 || kk != 0) ? 1u : 0u);
        }
        if (leader) umma_commit(&q_empty[st]);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          if (leader)
            umma_ss(tDP, desc_advance(ds_mn, kk * 2048), desc_advance(k_mn, kk * 2048), idesc_dq,
                    kk != 0 ? 1u : 0u);
        if (leader) umma_commit(dq_full);
        trace_event(p.trace, tr && leader, 0, it, 3);
        i = in;
        ++it;
      }
      if (leader) umma_commit(acc_full);
    }
    __syncwarp();
  } else if (warp < 12) {
    // ================================================================ softmax / dS group
    setmaxnreg_inc<BWD_REGS_SOFTMAX>();
    const int quad = warp & 3;
    const int half = (warp - 4) >> 2;  // which 64 q-columns
    const int sm_tid = (warp - 4) * 32 + lane;
    const int row = quad * 32 + lane;  // kv row inside the tile
    const int kj = k0 + row;
    const bool row_valid = kj < mk.Sk;
    const int kpos = mk.kmap(row_valid ? kj : mk.Sk - 1);
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const int my_seg = (mk.seg_k && row_valid) ? mk.seg_k[static_cast<long long>(b) * mk.Sk + kj] : -1;
    const float my_bias2 =
        (mk.bias && row_valid) ? mk.bias[b * mk.bias_stride_b + h * mk.bias_stride_h + kj] * kLog2e : 0.f;
    const unsigned int bh_u = static_cast<unsigned int>(b * p.H + h);
    uint8_t* ds_row = sDS + half * SM::SLAB_BYTES + row * 128;
    const int swz = row & 7;
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    const uint64_t bias2 = f2_pack(my_bias2, my_bias2);
    const bool biased = __any_sync(0xffffffffu, my_bias2 != 0.f);  // no row of this warp has one: nothing to add
    const float slope2 = (SHAPE & kShapeSlopes) ? p.shape.slopes[h] * kLog2e : 0.f;
    const int dist0 = kpos - ((SHAPE & kShapeSlopes) ? query_from(p.shape, b) : 0);  // key position less the queries' first one

    // kinds of this kv tile's bitmap tiles, as in the forward
    const int kinds_row = (mk.Sk + 127) >> 7;
    const uint8_t* tile_kinds = mk.keep_tiles && !mk.drop_threshold
                                    ? mk.keep_tiles + b * mk.keep_tiles_sb + h * mk.keep_tiles_sh + (k0 >> 7) : nullptr;
    const bool bits = mk.drop_threshold || mk.keep;
    auto minus_delta = [](uint64_t dp, uint64_t delta) { return (SHAPE & kShapeCap) ? f2_sub(delta, dp) : f2_sub(dp, delta); };
    int it = 0;
    bool alive = true;
    for (int i = next_vis(0); i < nqt && alive; i = next_vis(i + 1)) {
      const int qi0 = i * 128;
      const int st = it & 1;
      const uint32_t par = it & 1;
      const int kind = tile_mask<SHAPED>(mk, b, tile_kinds ? tile_kinds[static_cast<long long>(i) * kinds_row] != 1 : bits, qi0, k0, prefix);
      if (kind & kMaskSeg) {
        if (sm_tid < 128)
          sSegQ[st * 128 + sm_tid] =
              (qi0 + sm_tid) < mk.Sq ? mk.seg_q[static_cast<long long>(b) * mk.Sq + qi0 + sm_tid] : -2;
        named_bar_sync(1, 256);
      }
      // a wait that gives up must end the loop for the whole warp: the TMEM loads and stores below are
      // warp-collective
      if (!__all_sync(0xffffffffu, mbar_wait(&q_full[st], (it >> 1) & 1, wc, kTimeoutSmemFull))) { alive = false; break; }
      const float4* nl4 = reinterpret_cast<const float4*>(sLse + st * 256 + half * 64);
      const float4* dl4 = reinterpret_cast<const float4*>(sLse + st * 256 + 128 + half * 64);
      if (!__all_sync(0xffffffffu, mbar_wait(s_full, par, wc, kTimeoutTmemFull))) { alive = false; break; }
      tc_fence_after();
      trace_event(p.trace, tr && sm_tid == 0, 1, it, 0);

      // causal rule transposed: column (q index) c is hidden iff c < lo; all of them if the row is padding
      const bool special = kind != 0 || biased;
      int lo = 0;
      if (kind & kMaskEdge) {
        if (!row_valid) {
          lo = 128;
        } else if (mk.cbs && !(SHAPED && kpos < prefix)) {
          const long long kstart = static_cast<long long>(kpos / mk.cbs) * mk.cbs;
          const long long v = kstart - mk.qmap(qi0);
          lo = static_cast<int>(v < 0 ? 0 : (v > 128 ? 128 : v));
        }
      }
      const unsigned int qpos0 = static_cast<unsigned int>(mk.qmap(qi0));
      uint64_t pv[32];  // 64 probabilities of this thread's row, as fp32 pairs
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t s[32];
        tmem_ld_x32(tS + lane_base + half * 64 + c * 32, s);
        tmem_ld_wait();
        trace_event(p.trace, tr && sm_tid == 0, 3, it, c * 2);
        uint64_t x[16];
        uint64_t mul2 = scale2;
        if constexpr ((SHAPE & kShapeCap) != 0) {  // s = tanh
          float zm = 0.f;
#pragma unroll
          for (int e = 0; e < 32; e += 2) zm = max3(zm, fabsf(__uint_as_float(s[e])), fabsf(__uint_as_float(s[e + 1])));
          auto turn = [&](const float (&cf)[5]) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float t0, t1;
              f2_unpack(tanh_near2(f2_pack_u(s[2 * e], s[2 * e + 1]), cf), t0, t1);
              s[2 * e] = __float_as_uint(t0);
              s[2 * e + 1] = __float_as_uint(t1);
            }
          };
          auto turn_any = [&] {
            tanh_in_tmem(tS + lane_base + half * 64 + c * 32, 32, p.shape.tanh.scale);
            tmem_ld_x32(tS + lane_base + half * 64 + c * 32, s);
            tmem_ld_wait();
          };
          if constexpr ((SHAPE & kShapeSlopes) != 0) {
            // The polynomial in one piece with what follows, so that it fills the pauses of the exponentials; where TMEM holds the tanh already it
            // is the identity. (Cap 20 with slopes, 32 heads x 4096 x 128 559 us, as a branch of its own 575; 2 x 4096 x 16 heads of 64 472 and
            // 484. For a cap alone it is no gain: 529 and 538, D 64 447 and 443.)
            float cf[5] = {p.shape.tanh.c[0], p.shape.tanh.c[1], p.shape.tanh.c[2], p.shape.tanh.c[3], p.shape.tanh.c[4]};
            if (!__all_sync(0xffffffffu, zm <= p.shape.tanh.near_max)) {
              turn_any();
              cf[0] = 1.f;
              cf[1] = cf[2] = cf[3] = cf[4] = 0.f;
            }
            turn(cf);
          } else if (__all_sync(0xffffffffu, zm <= p.shape.tanh.near_max)) {
            turn(p.shape.tanh.c);
          } else {
            turn_any();
          }
          mul2 = f2_pack(p.shape.cap_log2, p.shape.cap_log2);
        }
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const float4 n = nl4[c * 8 + g];
          x[2 * g] = f2_fma(f2_pack_u(s[4 * g], s[4 * g + 1]), mul2, f2_pack(n.x, n.y));
          x[2 * g + 1] = f2_fma(f2_pack_u(s[4 * g + 2], s[4 * g + 3]), mul2, f2_pack(n.z, n.w));
        }
        if constexpr ((SHAPE & kShapeSlopes) != 0) {  // as in the forward
          const float d0 = static_cast<float>(mk.qmap(qi0) + half * 64 + c * 32 - dist0);
          const uint64_t away = f2_pack(-slope2, -slope2), two = f2_pack(2.f, 2.f);
          uint64_t d = f2_pack(d0, d0 + 1.f);
          if (!p.shape.two_sided) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              x[e] = f2_fma(d, away, x[e]);
              d = f2_add(d, two);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float e0, e1;
              f2_unpack(d, e0, e1);
              x[e] = f2_fma(f2_pack(fabsf(e0), fabsf(e1)), away, x[e]);
              d = f2_add(d, two);
            }
          }
        }
        if (special) {
          // keepw bit e: column base + e survives. Gathered before the element loop, as in the forward, and the loop only
          // runs for words with a hole; the dropout hash is a small rolled loop that only runs when dropout is on.
          const int base = half * 64 + c * 32;
          const int n = lo - base;
          uint32_t keepw = n <= 0 ? 0xffffffffu : (n >= 32 ? 0u : ~((1u << n) - 1u));
          if (kind & kMaskBits) {
            if (mk.keep && RA_IN_BOUNDS((qi0 + base) >> 5, 1, mk.keep_sr, kTagAttnMaskBits))
              keepw &= mk.keep[b * mk.keep_sb + h * mk.keep_sh + static_cast<long long>(row_valid ? kj : mk.Sk - 1) * mk.keep_sr +
                               ((qi0 + base) >> 5)];
            if (mk.drop_threshold) {
              uint32_t drop = 0;
#pragma unroll 1
              for (int e = 0; e < 32; ++e)
                drop |= static_cast<uint32_t>(dropout_hash(mk.seed_lo, mk.seed_hi, bh_u, qpos0 + base + e,
                                                           static_cast<unsigned int>(kpos)) < mk.drop_threshold)
                        << e;
              keepw &= ~drop;
            }
          }
          if (kind & kMaskSeg) keep_segment<1>(&keepw, sSegQ + st * 128 + base, my_seg, lane);
          if (biased) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = f2_add(x[e], bias2);
          }
          if (!__all_sync(0xffffffffu, keepw == 0xffffffffu)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float x0, x1;
              f2_unpack(x[e], x0, x1);
              x[e] = f2_pack((keepw >> (2 * e)) & 1u ? x0 : -INFINITY, (keepw >> (2 * e + 1)) & 1u ? x1 : -INFINITY);
            }
          }
        }
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1;
          f2_unpack(x[e], x0, x1);
          const float p0 = exp2_approx(x0), p1 = exp2_approx(x1);
          pv[c * 16 + e] = f2_pack(p0, p1);
          pk[e] = pack_bf16x2(p0, p1);
        }
        if constexpr ((SHAPE & kShapeCap) != 0) {  // times t^2 - 1, the derivative's negative: dS takes delta - dP for it
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t t = f2_pack_u(s[2 * e], s[2 * e + 1]);
            pv[c * 16 + e] = f2_mul(pv[c * 16 + e], f2_fma(t, t, f2_pack(-1.f, -1.f)));
          }
        }
        tmem_st_x16(tS + lane_base + half * 64 + c * 16, pk);
        trace_event(p.trace, tr && sm_tid == 0, 3, it, c * 2 + 1);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_ready);
      trace_event(p.trace, tr && sm_tid == 0, 1, it, 1);

      if (!__all_sync(0xffffffffu, mbar_wait(dp_full, par, wc, kTimeoutTmemFull))) { alive = false; break; }
      // the dS buffer is still being read by the previous dK/dQ MMAs until dq_full fires
      if (it > 0 && !__all_sync(0xffffffffu, mbar_wait(dq_full, (it - 1) & 1, wc, kTimeoutTmemFull))) { alive = false; break; }
      tc_fence_after();
      trace_event(p.trace, tr && sm_tid == 0, 1, it, 2);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t dp[32];
        uint32_t dsw[16];
        tmem_ld_x32(tDP + lane_base + half * 64 + c * 32, dp);
        tmem_ld_wait();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 d0 = dl4[c * 8 + 2 * g], d1 = dl4[c * 8 + 2 * g + 1];
          const uint64_t t0 = f2_mul(pv[c * 16 + 4 * g], minus_delta(f2_pack_u(dp[8 * g], dp[8 * g + 1]), f2_pack(d0.x, d0.y)));
          const uint64_t t1 = f2_mul(pv[c * 16 + 4 * g + 1], minus_delta(f2_pack_u(dp[8 * g + 2], dp[8 * g + 3]), f2_pack(d0.z, d0.w)));
          const uint64_t t2 = f2_mul(pv[c * 16 + 4 * g + 2], minus_delta(f2_pack_u(dp[8 * g + 4], dp[8 * g + 5]), f2_pack(d1.x, d1.y)));
          const uint64_t t3 = f2_mul(pv[c * 16 + 4 * g + 3], minus_delta(f2_pack_u(dp[8 * g + 6], dp[8 * g + 7]), f2_pack(d1.z, d1.w)));
          float a0, a1, a2, a3, a4, a5, a6, a7;
          f2_unpack(t0, a0, a1);
          f2_unpack(t1, a2, a3);
          f2_unpack(t2, a4, a5);
          f2_unpack(t3, a6, a7);
          uint4 v;
          v.x = pack_bf16x2(a0, a1);
          v.y = pack_bf16x2(a2, a3);
          v.z = pack_bf16x2(a4, a5);
          v.w = pack_bf16x2(a6, a7);
          const int chunk = c * 4 + g;  // 16-byte chunk inside the 128-byte row
          *reinterpret_cast<uint4*>(ds_row + ((chunk ^ swz) << 4)) = v;
          dsw[4 * g] = v.x;
          dsw[4 * g + 1] = v.y;
          dsw[4 * g + 2] = v.z;
          dsw[4 * g + 3] = v.w;
        }
        // dS^T also goes back over the dP^T columns this thread has already read, packed like P^T, and feeds
        // the dK MMA from TMEM: one 32 KB shared-memory operand read less per iteration
        tmem_st_x16(tDP + lane_base + half * 64 + c * 16, dsw);
      }
      tmem_st_wait();
      tc_fence_before();
      fence_proxy_async_smem();
      mbar_arrive(ds_ready);
      trace_event(p.trace, tr && sm_tid == 0, 1, it, 3);
      ++it;
    }

    // ---- epilogue: dV (half 0) / dK (half 1) for this warp's 32 kv rows. dS carried no softmax
    // scale, so dK is scaled here.
    if (alive) alive = mbar_wait(acc_full, 0, wc, kTimeoutTmemFull);
    alive = __all_sync(0xffffffffu, alive);  // TMEM loads below are warp-collective
    tc_fence_after();
    if (alive && !(it == 0 && p.dkv_mode == 2)) {
      const uint32_t tacc = (half == 0 ? tDV : tDK) + lane_base;
      void* base = half == 0 ? p.dv : p.dk;
      const float mul = half == 0 ? 1.0f : p.scale;
      const long long off = b * p.dkv_sb + static_cast<long long>(kj) * p.dkv_ss + h * p.dkv_sh;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        if (it > 0) {
          tmem_ld_x32(tacc + c * 32, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = 0u;
        }
        if (!row_valid) continue;
        if (!(RA_IN_BOUNDS(kj, 1, mk.Sk, kTagAttnBwdDkv) && RA_IN_BOUNDS(c * 32, 32, D, kTagAttnBwdDkv))) continue;
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = __uint_as_float(r[e]) * mul;
        if (p.dkv_mode == 0) {
          __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(base) + off + c * 32;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint4 v;
            v.x = pack_bf16x2(f[8 * g], f[8 * g + 1]);
            v.y = pack_bf16x2(f[8 * g + 2], f[8 * g + 3]);
            v.z = pack_bf16x2(f[8 * g + 4], f[8 * g + 5]);
            v.w = pack_bf16x2(f[8 * g + 6], f[8 * g + 7]);
            *reinterpret_cast<uint4*>(dst + 8 * g) = v;
          }
        } else {
          float* dst = reinterpret_cast<float*>(base) + off + c * 32;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            if (p.dkv_mode == 1)
              *reinterpret_cast<float4*>(dst + 4 * g) =
                  make_float4(f[4 * g], f[4 * g + 1], f[4 * g + 2], f[4 * g + 3]);
            else
              red_add_v4_sys(dst + 4 * g, f[4 * g], f[4 * g + 1], f[4 * g + 2], f[4 * g + 3]);
          }
        }
      }
    }
  } else {
    // ================================================================ dQ drain group
    setmaxnreg_inc<BWD_REGS_DRAIN>();
    const int quad = warp & 3;
    const int row = quad * 32 + lane;  // q row inside the tile
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    int it = 0;
    for (int i = next_vis(0); i < nqt; i = next_vis(i + 1)) {
      const int qi0 = i * 128;
      bool ok = mbar_wait_relaxed(dq_full, it & 1, wc, kTimeoutTmemFull, 32);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      trace_event(p.trace, tr && warp == 12 && lane == 0, 2, it, 0);
      // pull the whole dQ tile into registers and hand the TMEM region back at once; then move it
      // to global memory with bulk tensor reductions staged through one 16 KiB shared buffer
      uint32_t r[D];
#pragma unroll
      for (int c = 0; c < D / 32; ++c) tmem_ld_x32(tDP + lane_base + c * 32, r + c * 32);
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive(dq_empty);
      trace_event(p.trace, tr && warp == 12 && lane == 0, 2, it, 1);
      uint8_t* dq_row = sDQ + row * 128;
      const int swz = row & 7;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        if (warp == 12 && lane == 0) tma_store_wait_read<0>();  // staging buffer free again
        named_bar_sync(2, 128);
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const float4 v = make_float4(__uint_as_float(r[c * 32 + 4 * g]) * p.scale,
                                       __uint_as_float(r[c * 32 + 4 * g + 1]) * p.scale,
                                       __uint_as_float(r[c * 32 + 4 * g + 2]) * p.scale,
                                       __uint_as_float(r[c * 32 + 4 * g + 3]) * p.scale);
          *reinterpret_cast<float4*>(dq_row + ((g ^ swz) << 4)) = v;
        }
        fence_proxy_async_smem();
        named_bar_sync(2, 128);
        if (warp == 12 && lane == 0) {
          tma_reduce_add_4d(&tma_dq, sDQ, c * 32, h, qi0, b);
          tma_store_commit();
        }
      }
      trace_event(p.trace, tr && warp == 12 && lane == 0, 2, it, 2);
      ++it;
    }
    if (warp == 12 && lane == 0) tma_store_wait_all<0>();  // reductions complete before the CTA retires
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) bounded_drain_pause();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// The kernel for scores of this shape (kShape bits); in attn_bwd_shaped_sm100.cu.
using BwdKernel = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap, const BwdParams);
BwdKernel bwd_kernel_shaped(int D, int shape);

}  // namespace attn
}  // namespace ra
