// Backward hop of attention with modified scores (capped by a tanh, biased by distance, masked by documents and prefixes).
//
//   z = cap * tanh(x / cap) - slope |i - j|,  x = scale * q.k;   P = exp(z - lse);   dP = dO V^T;   dZ = P (dP - delta)
//   dX = dZ (1 - tanh^2(x / cap));   dV = P^T dO;   dK = scale dX^T Q;   dQ = scale dX K
//
// The structure is that of the plain backward hop: a CTA owns 128 keys of one K/V head and walks the query tiles of the
// head group, five products per tile in the transposed orientation, dK and dV resident in tensor memory, dQ^T added to an
// fp32 accumulator.  What differs:
//  * The key rows of a CTA have intervals of queries that see them; their hull gives the query tiles it walks, and a thread
//    (= key row) compares a query with its own interval in the tiles that are not inside all of them.
//  * What the second half of a tile's work needs of the scores is one factor, W = P (1 - tanh^2), kept as pairs of fp16 in the
//    registers that hold P in the plain hop; P itself goes to tensor memory at once.
//  * The issuing warp clears the padding rows of K, Q and dO tiles on the border between real rows and padding.
//  * A key tile that no query sees writes zeros.
//
// Bound, as the plain hop, by the serial order of a tile's steps (tensor pipe 52 % busy with documents, 34 % at head dim 64);
// with a cap by the elementwise warps, which issue some fourteen instructions more per pair.  Whole backward pass, causal, us:
// S 4096, 32/8 heads of 128: no change 391, bias 392, cap 471, both 502; 16 heads of 64: 158, 165, 218, 228; 16/8 heads of 256: 560, 550, 570,
// 570.  (A cap with a running bias of 0 instead of an instantiation of its own: 499, 230, 578.)
// Taking the tile coordinates out of registers (BwdPlan) was worth 12 to 20 %: 199 -> 159 us (16 heads of 64 with a bias).  A
// polynomial for the tanh, as in the forward hop, loses here: 517 -> 556 us; the special-function unit is not what binds.
// dQ and dK carry roundings to 16 bits of W (there are registers for pairs, not for fp32; fp16 whatever the operands are, see
// weight_shift), of dX (an operand of the products) and of the result, and delta that of out: relative error 2.5e-3 to 3.0e-3 in
// bf16 (3.0e-3 to 3.6e-3 with W in bf16, no faster but for plain scores at head dim 128: 386 for 392 us), 4e-4 to 5e-4 in fp16; the
// result's rounding alone gives 1.7e-3 and 2.1e-4.
#include <initializer_list>
#include <type_traits>

#include "bwd_common.cuh"
#include "bwd_tile.cuh"
#include "scored.cuh"

namespace rfa {

// With bf16 operands P and dX are 2^15 times themselves (the results are scaled back), which lets W, whose type no product
// sees, be fp16: 11 bits instead of 8 down to weights of 2^-29, less below.
template <typename T>
__host__ __device__ constexpr int weight_shift() { return Pack2<T>::kIsBf16 ? 15 : 0; }

// Two of them.  Scores of 10^7 and more leave lse, and with it P, off by factors: above 2 they end there and not in an infinity.
// (Ending P itself at 1 takes two operations a pair more: 386 -> 395 us without a bias, S 4096, 32/8 heads of 128.)
template <typename T>
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  if constexpr (!Pack2<T>::kIsBf16) return Pack2<__half>::pack(lo, hi);
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

struct ScoredBwdParams {
  BwdParams p;
  ScoreParams sc;
};

// What a CTA works on.  Worked out once and kept in shared memory: each role takes into registers what it needs.
struct BwdPlan {
  int kvt, hf, part, hkv, b;
  int i_begin, n_i;          // query tiles that some key of the tile is seen by
  int full_lo, full_hi;      // rows [full_lo, full_hi) of the query block see every key of the tile
  int t0, t_total;           // this CTA's run of the G * n_i query tiles, head-major
  int real_lo, real_hi;      // rows of the whole sequence that are no padding
};
// Query head and tile of step t of a run.
struct BwdWalk {
  int t0, n_i, i_begin, head0;
  __device__ __forceinline__ BwdWalk(const BwdPlan& x, int G) : t0(x.t0), n_i(x.n_i), i_begin(x.i_begin), head0(x.hkv * G) {}
  __device__ __forceinline__ int head(int t) const { return head0 + (t0 + t) / n_i; }
  __device__ __forceinline__ int tile(int t) const { return i_begin + (t0 + t) % n_i; }
};

template <int DP, int DH, int BQ>
__device__ __forceinline__ void make_plan(const ScoredBwdParams& prm, BwdPlan& plan) {
  const BwdParams& p = prm.p;
  const ScoreParams& sc = prm.sc;
  constexpr int kHalves = DP / DH;
  // Key tile first, so that the CTAs with the most visible queries start first (with a mask: in the order of its work list)
  // and the tail of the grid evens out (head after head instead, a third of the DRAM traffic but a long tail: 1.00 -> 1.09 ms
  // at S 16384, 32/8 heads of 128 in documents of 2048); blocks that every query sees go head group first, which keeps the dQ accumulator of
  // the resident CTAs in L2.  The ordered mode needs key tiles in rising block order.
  const bool worklist = sc.has_mask && p.dq_order == nullptr;
  const int nkvt = (p.Skv + 127) / 128;
  int kvt, hf, part, hkv, b;
  {
    int rem = static_cast<int>(blockIdx.x);
    hf = rem % kHalves;
    rem /= kHalves;
    if (p.causal || sc.has_mask) {
      part = rem % p.nsplit;  // CTAs that share a K/V tile are adjacent (the tile stays in L2)
      rem /= p.nsplit;
      hkv = rem % p.Hkv;
      rem /= p.Hkv;
      if (worklist) {
        rem = __ldg(sc.mask.order_k + rem);
        b = rem / nkvt;
        kvt = rem % nkvt;
      } else {
        b = rem % p.B;
        kvt = rem / p.B;
      }
    } else {
      kvt = rem % nkvt;
      rem /= nkvt;
      part = rem % p.nsplit;
      rem /= p.nsplit;
      hkv = rem % p.Hkv;
      b = rem / p.Hkv;
    }
  }
  const int G = p.Hq / p.Hkv;
  const int n0 = kvt * 128;
  const int nQtiles = (p.Sq + BQ - 1) / BQ;
  // Query rows of the block: [lo, hi) is the hull of what the keys of this tile are seen by, [full_lo, full_hi) what sees
  // them all.  The ordered mode visits every tile of a masked block: its counters expect every key tile.
  int i_begin, i_end, full_lo, full_hi;
  {
    const int4 hull = key_hull(sc, b, nkvt, kvt, p.Skv);
    const int lo = max(hull.x - sc.q_pos, 0), hi = min(hull.w - sc.q_pos, p.Sq);
    i_begin = lo / BQ;
    i_end = lo < hi ? (hi + BQ - 1) / BQ : i_begin;
    full_lo = max(hull.y, sc.q_pos) - sc.q_pos;
    full_hi = hull.z - sc.q_pos;
    if (sc.has_mask && !worklist) {
      i_begin = 0;
      i_end = nQtiles;
    }
  }
  const int n_i = i_end - i_begin;
  // The G * n_i query tiles of the K/V tile, head-major, are dealt out to nsplit CTAs in equal runs.
  const int t0 = static_cast<int>(static_cast<long long>(G) * n_i * part / p.nsplit);
  const int t_total = static_cast<int>(static_cast<long long>(G) * n_i * (part + 1) / p.nsplit) - t0;
  const int real_lo = sc.has_mask ? __ldg(sc.mask.real + 2 * b) : 0;
  const int real_hi = sc.has_mask ? __ldg(sc.mask.real + 2 * b + 1) : sc.len;
  if ((threadIdx.x & 31) == 0) plan = BwdPlan{kvt, hf, part, hkv, b, i_begin, n_i, full_lo, full_hi, t0, t_total, real_lo, real_hi};
}

template <int DP, int DH, int BQ, int NSQ, int NSO, typename T, int kKind>
__global__ void __launch_bounds__(640, 1)
    scored_bwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                      const ScoredBwdParams prm) {
  const BwdParams& p = prm.p;
  const ScoreParams& sc = prm.sc;
  using Cfg = BwdCfg<DP, DH, BQ, NSQ, NSO>;
  constexpr bool kBf16 = Pack2<T>::kIsBf16;
  constexpr int kShift = weight_shift<T>();
  constexpr int kPanelK = 128 * 128;  // bytes per panel of a 128-row tile
  constexpr int kPanelQ = BQ * 128;   // bytes per panel of a BQ-row tile

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t bar_kv_full, bar_k_tmem;
  __shared__ uint64_t bar_q_full[NSQ], bar_q_empty[NSQ], bar_do_full[NSO], bar_do_empty[NSO];
  __shared__ uint64_t bar_s_full, bar_p_ready, bar_dp_full, bar_ds_ready, bar_dq_full, bar_dq_drained, bar_final;
  __shared__ uint32_t tmem_holder;
  __shared__ BwdPlan plan;
  __shared__ int abort_flag, skip_flag;

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const uint32_t smem_base = smem_u32(smem_raw);
  const uint32_t s_k = smem_base + Cfg::kOffK;
  const uint32_t s_v = smem_base + Cfg::kOffV;
  const uint32_t s_q = smem_base + Cfg::kOffQ;
  const uint32_t s_do = smem_base + Cfg::kOffDO;
  const uint32_t s_ds = smem_base + Cfg::kOffDS;
  const uint32_t s_stat = smem_base + Cfg::kOffStat;
  uint8_t* const stat_ptr = smem_raw + Cfg::kOffStat;
  uint8_t* const ds_ptr = smem_raw + Cfg::kOffDS;
  uint8_t* const dq_ptr = smem_raw + Cfg::kOffDQ;

  if (tid == 0) {
    abort_flag = ((smem_base & 1023u) != 0) ? 1 : 0;  // operand tiles need 1024-byte alignment
    mbar_init(&bar_kv_full, 1);
    mbar_init(&bar_k_tmem, 256);
    for (int i = 0; i < NSQ; ++i) {
      mbar_init(&bar_q_full[i], 1);
      mbar_init(&bar_q_empty[i], 1);
    }
    for (int i = 0; i < NSO; ++i) {
      mbar_init(&bar_do_full[i], 1);
      mbar_init(&bar_do_empty[i], 1);
    }
    mbar_init(&bar_s_full, 1);
    mbar_init(&bar_p_ready, 256);
    mbar_init(&bar_dp_full, 1);
    mbar_init(&bar_ds_ready, 256);
    mbar_init(&bar_dq_full, 1);
    mbar_init(&bar_dq_drained, 256);
    mbar_init(&bar_final, 1);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_holder, 512);
    tmem_relinquish();
  }
  pdl_wait();  // nothing above touches global memory

  if (warp == 0) make_plan<DP, DH, BQ>(prm, plan);
  if (tid == 0) skip_flag = *reinterpret_cast<volatile int*>(p.status);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_holder;
  if (skip_flag != 0) {  // an earlier kernel gave up
    if (warp == 0) tmem_dealloc(tmem_base, 512);
    return;
  }
  volatile int* abort_p = &abort_flag;
  const bool run = (abort_flag == 0) && (plan.t_total > 0);

  const int G = p.Hq / p.Hkv;
  // Register budget.  The launch gives every thread 96 registers (640 x 96 = 61440, the pool the warpgroups trade
  // inside); each role changes its own allowance on entry: 4 service warps x 64, 8 elementwise warps x 128,
  // 8 reduction warps x 80.  The raise waits until the other roles have lowered theirs, so the sum must fit the pool.
  static_assert(128 * 64 + 256 * 128 + 256 * 80 <= 640 * 96, "register allowances exceed what the launch allocated");
  if (warp < 4) {
    setmaxnreg_dec<64>();
    if (warp == 0) {
      // =========================== TMA producer ===========================
      if (lane == 0 && run) {
        const BwdWalk walk(plan, G);
        const int hkv = plan.hkv, b = plan.b, hf = plan.hf, n0 = plan.kvt * 128, T_total = plan.t_total;
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        tma_prefetch_desc(&tm_do);
        mbar_expect_tx(&bar_kv_full, Cfg::kKSmemBytes + Cfg::kVBytes);
        constexpr int kPanelsK = Cfg::kKTmem ? DH / 64 : Cfg::kPanels;
        const int k_col0 = Cfg::kKTmem ? hf * DH : 0;
#pragma unroll
        for (int pn = 0; pn < kPanelsK; ++pn)
          tma_load_4d(s_k + pn * kPanelK, &tm_k, &bar_kv_full, k_col0 + pn * 64, hkv, n0, b);
#pragma unroll
        for (int pn = 0; pn < Cfg::kPanels; ++pn)
          tma_load_4d(s_v + pn * kPanelK, &tm_v, &bar_kv_full, pn * 64, hkv, n0, b);
        auto load_do = [&](int t, int hq, int i) {
          const int so = t % NSO;
          if (!mbar_wait(&bar_do_empty[so], ((t / NSO) & 1) ^ 1, abort_p)) return false;
          mbar_expect_tx(&bar_do_full[so], Cfg::kQBytes);
#pragma unroll
          for (int pn = 0; pn < Cfg::kPanels; ++pn)
            tma_load_4d(s_do + so * Cfg::kQBytes + pn * kPanelQ, &tm_do, &bar_do_full[so], pn * 64, hq, i * BQ, b);
          return true;
        };
        auto load_q = [&](int t, int hq, int i) {
          const int st = t % NSQ;
          if (!mbar_wait(&bar_q_empty[st], ((t / NSQ) & 1) ^ 1, abort_p)) return false;
          mbar_expect_tx(&bar_q_full[st], Cfg::kQBytes + Cfg::kStatBytes);
#pragma unroll
          for (int pn = 0; pn < Cfg::kPanels; ++pn)
            tma_load_4d(s_q + st * Cfg::kQBytes + pn * kPanelQ, &tm_q, &bar_q_full[st], pn * 64, hq, i * BQ, b);
          const size_t stat_off = (static_cast<size_t>(b) * p.Hq + hq) * p.Spad + static_cast<size_t>(i) * BQ;
          bulk_load_1d(s_stat + st * Cfg::kStatBytes, p.lse2 + stat_off, BQ * 4, &bar_q_full[st]);
          bulk_load_1d(s_stat + st * Cfg::kStatBytes + BQ * 4, p.delta + stat_off, BQ * 4, &bar_q_full[st]);
          return true;
        };
        for (int t = 0; t < T_total; ++t) {
          const int hq = walk.head(t);
          const int i = walk.tile(t);
          // With as many dO slots as Q slots the dO slot frees first (after the dV product, the Q slot after dK); with fewer
          // the Q slot of tile t has been free since dK of tile t - 2.
          const bool ok = (NSO < NSQ) ? (load_q(t, hq, i) && load_do(t, hq, i)) : (load_do(t, hq, i) && load_q(t, hq, i));
          if (!ok) break;
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // =========================== MMA issuer ===========================
      // The whole warp runs the loop converged (cheap, warp-uniform descriptor arithmetic); the elected lane issues.
      if (run) {
        const BwdWalk walk(plan, G);
        const int hf = plan.hf, T_total = plan.t_total;
        const uint32_t el = elect_one();
        constexpr uint32_t idesc_s = make_idesc(128, BQ, kBf16, false, false);   // K-major x K-major
        // dV and dK (A from tensor memory / K-major, B MN-major) are as wide as the head dim, not as its padded size (head dim
        // 256 keeps a constant width: one more live register costs it 2 %).  With dQ^T reduced only by warps that hold
        // columns of the head dim: B 2, S 1500, 16/4 heads of 96, diagonal / full 71.4 / 116 -> 66.2 / 106 us; S 4096, 16 heads
        // of 32 130 / 257 -> 125 / 246; B 2, S 4096, 16 heads of 160 1166 / 1935 -> 1126 / 1898.  S^T and dP^T do run over
        // the padding: a predicate per step costs the issuer more (25 % at head dim 256) than the steps it saves.
        const uint32_t idesc_dv = make_idesc(128, DP > 128 ? DH : min((p.D + 15) / 16 * 16, DH), kBf16, false, true);
        constexpr uint32_t idesc_dq = make_idesc(128, BQ, kBf16, true, true);    // both MN-major
        const uint32_t tm_s = tmem_base + Cfg::kTmS;
        const uint32_t tm_dp = tmem_base + Cfg::kTmDP;
        const uint32_t tm_dv = tmem_base + Cfg::kTmDV;
        const uint32_t tm_dk = tmem_base + Cfg::kTmDK;

        // Descriptor low words of the resident tiles; offsets below are in 16-byte units.
        const uint32_t k_km = desc_lo_kmajor(s_k);                                   // K as K-major A (S^T), unless in TMEM
        const uint32_t tm_k = tmem_base + Cfg::kTmK;
        const uint32_t v_km = desc_lo_kmajor(s_v);                                   // V as K-major A (dP^T)
        const uint32_t k_mn = desc_lo_mnmajor(s_k + (Cfg::kKTmem ? 0 : hf * (DH / 64) * kPanelK), kPanelK);  // K^T as MN-major A (dQ^T)
        const uint32_t ds_km = desc_lo_kmajor(s_ds);                                 // dS^T as K-major A (dK)
        const uint32_t ds_mn = desc_lo_mnmajor(s_ds, kPanelK);                       // dS^T as MN-major B (dQ^T)
        auto q_km = [&](int st) { return desc_lo_kmajor(s_q + st * Cfg::kQBytes); };
        auto do_km = [&](int st) { return desc_lo_kmajor(s_do + st * Cfg::kQBytes); };
        auto q_mn = [&](int st) {
          return desc_lo_mnmajor(s_q + st * Cfg::kQBytes + hf * (DH / 64) * kPanelQ, kPanelQ);
        };
        auto do_mn = [&](int st) {
          return desc_lo_mnmajor(s_do + st * Cfg::kQBytes + hf * (DH / 64) * kPanelQ, kPanelQ);
        };

        // S^T[128 x BQ] = K[128 x DP] * Q[BQ x DP]^T
        auto issue_s = [&](int st) {
          const uint32_t bq = q_km(st);
#pragma unroll
          for (int ks = 0; ks < DP / 16; ++ks)
            if constexpr (Cfg::kKTmem)
              mma_ts_lo_e(tm_s, tm_k + ks * 8, bq + (((ks >> 2) * kPanelQ + (ks & 3) * 32) >> 4), idesc_s, ks > 0 ? 1u : 0u, el);
            else
              mma_ss_lo_e(tm_s, k_km + (((ks >> 2) * kPanelK + (ks & 3) * 32) >> 4),
                          bq + (((ks >> 2) * kPanelQ + (ks & 3) * 32) >> 4), idesc_s, ks > 0 ? 1u : 0u, el);
        };
        // dP^T[128 x BQ] = V[128 x DP] * dO[BQ x DP]^T
        auto issue_dp = [&](int st) {
          const uint32_t bo = do_km(st);
#pragma unroll
          for (int ks = 0; ks < DP / 16; ++ks)
            mma_ss_lo_e(tm_dp, v_km + (((ks >> 2) * kPanelK + (ks & 3) * 32) >> 4),
                      bo + (((ks >> 2) * kPanelQ + (ks & 3) * 32) >> 4), idesc_s, ks > 0 ? 1u : 0u, el);
        };
        // dV[128 x DH] += P^T[128 x BQ] (tensor memory) * dO[BQ x DH]
        auto issue_dv = [&](int st, bool acc) {
          const uint32_t bo = do_mn(st);
#pragma unroll
          for (int ks = 0; ks < BQ / 16; ++ks) {
            // P^T of query columns [16ks, 16ks+16): each elementwise group packs its half over its own S^T columns
            const int grp = (ks * 16) / (BQ / 2);
            const uint32_t pa = tm_s + grp * (BQ / 2) + ((ks * 16) % (BQ / 2)) / 2;
            mma_ts_lo_e(tm_dv, pa, bo + ((ks * 2048) >> 4), idesc_dv, (acc || ks > 0) ? 1u : 0u, el);
          }
        };
        // dK[128 x DH] += dS^T[128 x BQ] (shared memory, K-major) * Q[BQ x DH]
        auto issue_dk = [&](int st, bool acc) {
          const uint32_t bq = q_mn(st);
#pragma unroll
          for (int ks = 0; ks < BQ / 16; ++ks)
            mma_ss_lo_e(tm_dk, ds_km + (((ks >> 2) * kPanelK + (ks & 3) * 32) >> 4), bq + ((ks * 2048) >> 4), idesc_dv,
                        (acc || ks > 0) ? 1u : 0u, el);
        };
        // dQ^T[128 (d) x BQ] = K^T[d x 128 (kv)] * dS^T[128 (kv) x BQ]; for head dim 64 the upper 64
        // rows of the A operand run into the V tile (results in those lanes are ignored).
        auto issue_dq = [&]() {
#pragma unroll
          for (int ks = 0; ks < 128 / 16; ++ks)
            mma_ss_lo_e(tmem_base + Cfg::kTmDQ, k_mn + ((ks * 2048) >> 4), ds_mn + ((ks * 2048) >> 4), idesc_dq, ks > 0 ? 1u : 0u, el);
        };

        // Padding rows are cleared before the first product that reads them: those of K, Q and dO because a product contracts
        // over them, those of V because dP of a padding key meets a weight of 0 (delta of a padding query is 0 as well).
        const bool border_q = sc.has_mask && (plan.real_lo > sc.q_pos + plan.i_begin * BQ ||
                                              plan.real_hi < sc.q_pos + (plan.i_begin + plan.n_i) * BQ);
        auto clear_tile = [&](uint32_t tile, int panels, int rows, int pos) {
          if (plan.real_lo > pos || plan.real_hi < pos + rows)
            clear_padding_rows(tile, panels, rows, plan.real_lo - pos, plan.real_hi - pos, lane);
        };
        auto start_s = [&](int t, int st) {
          tc_fence_after_sync();
          if (border_q) clear_tile(s_q + st * Cfg::kQBytes, Cfg::kPanels, BQ, sc.q_pos + walk.tile(t) * BQ);
          issue_s(st);
          mma_commit_e(&bar_s_full, el);
        };
        auto start_dp = [&](int t, int so) {
          tc_fence_after_sync();
          if (border_q) clear_tile(s_do + so * Cfg::kQBytes, Cfg::kPanels, BQ, sc.q_pos + walk.tile(t) * BQ);
          issue_dp(so);
          mma_commit_e(&bar_dp_full, el);
        };

        bool ok = mbar_wait_warp(&bar_kv_full, 0, abort_p);
        if (ok && sc.has_mask) {
          clear_tile(s_k, Cfg::kKSmemBytes / kPanelK, 128, sc.k_pos + plan.kvt * 128);
          clear_tile(s_v, Cfg::kPanels, 128, sc.k_pos + plan.kvt * 128);
        }
        if (ok && Cfg::kKTmem) ok = mbar_wait_warp(&bar_k_tmem, 0, abort_p);
        if (ok) ok = mbar_wait_warp(&bar_q_full[0], 0, abort_p);
        if (ok) {
          start_s(0, 0);
          ok = mbar_wait_warp(&bar_do_full[0], 0, abort_p);
        }
        if (ok) {
          start_dp(0, 0);
        }
        for (int t = 0; t < T_total && ok; ++t) {
          const int st = t % NSQ;
          const int st_n = (t + 1) % NSQ;
          const uint32_t par_n = ((t + 1) / NSQ) & 1;
          const int so = t % NSO;
          const int so_n = (t + 1) % NSO;
          const uint32_t par_on = ((t + 1) / NSO) & 1;
          const bool more = (t + 1 < T_total);
          if (!mbar_wait_warp(&bar_p_ready, t & 1, abort_p)) break;
          tc_fence_after_sync();
          issue_dv(so, t > 0);
          mma_commit_e(&bar_do_empty[so], el);
          // S^T of the next tile goes out now if its Q tile has landed (a non-blocking probe); otherwise it is the
          // first thing issued once dS^T is ready.
          bool s_issued = !more;
          if (more && __all_sync(0xffffffffu, mbar_test_wait(&bar_q_full[st_n], par_n))) {
            start_s(t + 1, st_n);
            s_issued = true;
          }
          if (!mbar_wait_warp(&bar_ds_ready, t & 1, abort_p)) break;
          tc_fence_after_sync();
          if (!s_issued) {
            // the elementwise warps have nothing to do until S^T of the next tile exists: it goes first
            if (!mbar_wait_warp(&bar_q_full[st_n], par_n, abort_p)) break;
            start_s(t + 1, st_n);
          }
          if (Cfg::kOwnDQ) {
            // dP^T of the next tile does not have to wait for dQ^T: the elementwise warps find it ready
            if (more) {
              if (!mbar_wait_warp(&bar_do_full[so_n], par_on, abort_p)) break;
              start_dp(t + 1, so_n);
            }
            issue_dk(st, t > 0);
            mma_commit_e(&bar_q_empty[st], el);
            if (t > 0 && !mbar_wait_warp(&bar_dq_drained, (t - 1) & 1, abort_p)) break;
            tc_fence_after_sync();
            issue_dq();
            mma_commit_e(&bar_dq_full, el);
            if (!more) mma_commit_e(&bar_final, el);
            continue;
          }
          // dK before dQ^T: it releases the Q slot ~500 cycles earlier, which matters more than the reduction
          // starting earlier (a Q tile load takes 1500-3000 cycles under the L2 load of the reductions and only two
          // Q stages fit in shared memory).
          issue_dk(st, t > 0);
          mma_commit_e(&bar_q_empty[st], el);
          issue_dq();
          mma_commit_e(&bar_dq_full, el);
          if (more) {
            if (!mbar_wait_warp(&bar_do_full[so_n], par_on, abort_p)) break;
            if (!mbar_wait_warp(&bar_dq_drained, t & 1, abort_p)) break;
            start_dp(t + 1, so_n);
          } else {
            mma_commit_e(&bar_final, el);
          }
        }
      }
      __syncwarp();
    }
  } else if (warp < 12) {
    // =========================== elementwise warpgroups ===========================
    // Two warpgroups share every tile: group cw owns query columns [cw*BQ/2, (cw+1)*BQ/2).
    setmaxnreg_inc<128>();
    constexpr int kHalfCols = BQ / 2;
    constexpr int NCH = kHalfCols / 32;  // 32-column chunks per thread
    const int cw = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // kv row inside the tile
    const BwdWalk walk(plan, G);
    const int b = plan.b, hkv = plan.hkv, hf = plan.hf, n0 = plan.kvt * 128, T_total = plan.t_total;
    const int full_lo = plan.full_lo, full_hi = n0 + 128 > p.Skv ? INT_MIN : plan.full_hi;
    const int kvpos = n0 + row;
    // Queries of the block that see this key: [lo, lo + width).  Rows behind the block's end are seen by none.
    int lo = 0, width = 0;
    if (kvpos < p.Skv) {
      int hi = p.Sq;
      if (sc.has_mask) {
        const size_t at = static_cast<size_t>(b) * sc.len + sc.k_pos + kvpos;
        lo = max(__ldg(sc.mask.k_lo + at) - sc.q_pos, 0);
        hi = min(__ldg(sc.mask.k_hi + at) - sc.q_pos, p.Sq);
      } else if (sc.causal) {
        lo = max(sc.k_pos + kvpos - sc.q_pos, 0);
      }
      width = max(hi - lo, 0);
    }
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int col0 = cw * kHalfCols;
    const uint32_t a_s = tmem_base + lane_addr + Cfg::kTmS + col0;
    const uint32_t a_dp = tmem_base + lane_addr + Cfg::kTmDP + col0;
    const uint64_t nscale2 = pack_f2(-p.scale_log2, -p.scale_log2);
    const float cap_log2 = sc.cap * kLog2e;
    const float in_scale = has_cap(kKind) ? 2.f * p.scale_log2 / sc.cap : 0.f;  // raw score to the exponent of the tanh
    const int ahead = sc.q_pos + col0 - (sc.k_pos + kvpos);  // of query column col0 of tile 0 over this key
    bool ok = run;
    if (Cfg::kKTmem && run) {
      // K (16 bit, two per column) into tensor memory: each thread copies half of its row from global memory, once per CTA (zeros
      // for a key that no query sees: padding, or behind the block's end)
      const T* krow = static_cast<const T*>(p.k) + ((static_cast<size_t>(b) * p.Skv + kvpos) * p.Hkv + hkv) * p.D;
#pragma unroll 1
      for (int c = 0; c < DP / 4; c += 32) {
        uint32_t u[32];
        const int col = cw * (DP / 2) + 2 * c;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (width > 0 && col + k * 8 < p.D) w = *reinterpret_cast<const uint4*>(krow + col + k * 8);
          u[4 * k + 0] = w.x; u[4 * k + 1] = w.y; u[4 * k + 2] = w.z; u[4 * k + 3] = w.w;
        }
        tmem_st32(tmem_base + lane_addr + Cfg::kTmK + col / 2, u);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(&bar_k_tmem);
    }
    for (int t = 0; t < T_total && ok; ++t) {
      const int st = t % NSQ;
      const int i = walk.tile(t);
      const float* lse2_s = reinterpret_cast<const float*>(stat_ptr + st * Cfg::kStatBytes) + col0;
      const float* delta_s = lse2_s + BQ;
      if (!mbar_wait_warp(&bar_q_full[st], (t / NSQ) & 1, abort_p)) { ok = false; break; }
      if (!mbar_wait_warp(&bar_s_full, t & 1, abort_p)) { ok = false; break; }
      tc_fence_after_sync();
      const int q0 = i * BQ + col0;
      const bool masked = i * BQ < full_lo || i * BQ + BQ > full_hi;
      uint32_t pk[NCH * 16];  // W = P (1 - tanh^2) for dX, in fp16
      {
        uint32_t r[NCH][32];
#pragma unroll
        for (int c = 0; c < NCH; ++c) tmem_ld32(a_s + c * 32, r[c]);
        tmem_ld_wait32(r[0]);
#pragma unroll
        for (int c = 1; c < NCH; ++c) reg_fence32(r[c]);
        // P^T = exp2(z - lse2) = exp2(-y); the distance term slope |i - j| is linear in the query where all queries of the
        // tile lie on one side of all keys.
        const float slope = has_bias(kKind) ? slope_log2(sc, b, p.Hq, walk.head(t)) : 0.f;
        const int d0 = sc.q_pos + i * BQ - (sc.k_pos + n0);  // of the first query over the first key
        const bool linear = !has_bias(kKind) || d0 >= 127 || d0 + BQ - 1 <= 0 || slope == 0.f;
        const float sign_slope = d0 >= 127 ? slope : -slope;
        auto p_phase = [&](auto mask_tag, auto linear_tag) {
          constexpr bool kMask = decltype(mask_tag)::value;
          constexpr bool kLinear = decltype(linear_tag)::value;
          const uint64_t step = pack_f2(2.f * sign_slope, 2.f * sign_slope);
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            uint32_t u[16];
            const int d = ahead + i * BQ + c * 32;
            uint64_t bias = 0;
            if (kKind > 0 || kShift > 0) {
              // what y has beside lse2: the distance, the constant of the tanh, the power of two on P
              const float b0 = (has_bias(kKind) && kLinear ? static_cast<float>(d) * sign_slope : 0.f) - (has_cap(kKind) ? cap_log2 + kShift : kShift);
              bias = pack_f2(b0, has_bias(kKind) && kLinear ? b0 + sign_slope : b0);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float2 l2 = *reinterpret_cast<const float2*>(lse2_s + c * 32 + k * 2);
              uint64_t y2 = pack_f2(l2.x, l2.y);
              if (kKind > 0 || kShift > 0) {
                y2 = add2(y2, bias);
                if (has_bias(kKind) && kLinear) bias = add2(bias, step);
                else if (has_bias(kKind)) y2 = add2(y2, pack_f2(slope * fabsf(static_cast<float>(d + 2 * k)), slope * fabsf(static_cast<float>(d + 2 * k + 1))));
              }
              uint64_t jac2 = 0;
              if constexpr (has_cap(kKind)) {
                // cap tanh(x / cap) = cap - cap g and 1 - tanh^2 = g (2 - g) with g = 2 / (exp(2 x / cap) + 1)
                float a0, a1;
                unpack_f2(mul2(pack_u2(r[c][2 * k], r[c][2 * k + 1]), pack_f2(in_scale, in_scale)), a0, a1);
                const uint64_t half2 = pack_f2(0.5f, 0.5f);
                unpack_f2(fma2(pack_f2(fast_exp2(a0), fast_exp2(a1)), half2, half2), a0, a1);
                const uint64_t g2 = pack_f2(fast_rcp(a0), fast_rcp(a1));
                y2 = fma2(g2, pack_f2(cap_log2, cap_log2), y2);
                jac2 = mul2(g2, sub2(pack_f2(2.f, 2.f), g2));
              } else {
                y2 = fma2(pack_u2(r[c][2 * k], r[c][2 * k + 1]), nscale2, y2);
              }
              float y0, y1;
              unpack_f2(y2, y0, y1);
              float e0 = fast_exp2(-y0), e1 = fast_exp2(-y1);
              if (kMask) {
                const int qp = q0 + c * 32 + k * 2 - lo;
                if (static_cast<unsigned>(qp) >= static_cast<unsigned>(width)) e0 = 0.f;
                if (static_cast<unsigned>(qp + 1) >= static_cast<unsigned>(width)) e1 = 0.f;
              }
              u[k] = Pack2<T>::pack(e0, e1);
              if constexpr (has_cap(kKind)) {
                float w0, w1;
                unpack_f2(mul2(pack_f2(e0, e1), jac2), w0, w1);
                pk[c * 16 + k] = pack_weights<T>(w0, w1);
              } else {
                pk[c * 16 + k] = kBf16 ? pack_weights<T>(e0, e1) : u[k];
              }
            }
            // P^T (16 bit, two per column) goes over the start of this group's own S^T columns, all of which are in registers
            tmem_st16(a_s + c * 16, u);
          }
        };
        if (has_bias(kKind) && !linear) {
          if (masked) p_phase(std::true_type{}, std::false_type{});
          else p_phase(std::false_type{}, std::false_type{});
        } else {
          if (masked) p_phase(std::true_type{}, std::true_type{});
          else p_phase(std::false_type{}, std::true_type{});
        }
      }
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(&bar_p_ready);

      if (!mbar_wait_warp(&bar_dp_full, t & 1, abort_p)) { ok = false; break; }
      tc_fence_after_sync();
      {
        uint32_t r[NCH][32];
#pragma unroll
        for (int c = 0; c < NCH; ++c) tmem_ld32(a_dp + c * 32, r[c]);
        tmem_ld_wait32(r[0]);
#pragma unroll
        for (int c = 1; c < NCH; ++c) reg_fence32(r[c]);
        // the products that read the previous dS^T have retired (with dQ^T in dP^T's columns, dP^T itself says so)
        if (Cfg::kOwnDQ && t > 0 && !mbar_wait_warp(&bar_dq_full, (t - 1) & 1, abort_p)) { ok = false; break; }
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float4 d4 = *reinterpret_cast<const float4*>(delta_s + c * 32 + k * 4);
            const float2 p01 = Pack2<__half>::unpack(pk[c * 16 + 2 * k + 0]);
            const float2 p23 = Pack2<__half>::unpack(pk[c * 16 + 2 * k + 1]);
            float s0, s1, s2, s3;
            unpack_f2(mul2(pack_f2(p01.x, p01.y),
                           sub2(pack_u2(r[c][4 * k + 0], r[c][4 * k + 1]), pack_f2(d4.x, d4.y))), s0, s1);
            unpack_f2(mul2(pack_f2(p23.x, p23.y),
                           sub2(pack_u2(r[c][4 * k + 2], r[c][4 * k + 3]), pack_f2(d4.z, d4.w))), s2, s3);
            w[2 * k + 0] = Pack2<T>::pack(s0, s1);
            w[2 * k + 1] = Pack2<T>::pack(s2, s3);
          }
          // 32 columns = 64 bytes = four 16-byte chunks inside the panel that holds column col0 + c*32
          const int colg = col0 + c * 32;
          uint8_t* panel = ds_ptr + (colg / 64) * kPanelK;
          const int chunk0 = (colg % 64) / 8;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint4 v4 = make_uint4(w[4 * k + 0], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
            *reinterpret_cast<uint4*>(panel + sw128_offset(row, chunk0 + k)) = v4;
          }
        }
      }
      fence_proxy_async_smem();
      tc_fence_before_sync();
      mbar_arrive(&bar_ds_ready);
    }
    // ---- epilogue: group 0 writes dV, group 1 writes dK (scaled) ----
    if (ok) ok = mbar_wait_warp(&bar_final, 0, abort_p);
    // Ordered mode with a split tile: the runs add in the order of their index (one counter per warp and tile), so that
    // dK and dV are bit-reproducible too.  The run waited for has a lower block index: it was dispatched before.
    int* part_sem = nullptr;
    if (p.dq_order != nullptr && p.nsplit > 1) {
      part_sem = p.dq_order + static_cast<size_t>(p.B) * p.Hq * ((p.Sq + BQ - 1) / BQ) * Cfg::kHalves * 8 +
                 (((static_cast<size_t>(b) * p.Hkv + hkv) * ((p.Skv + 127) / 128) + plan.kvt) * Cfg::kHalves + hf) * 8 + (warp - 4);
      if ((ok || !run) && !wait_count(part_sem, plan.part, lane == 0, abort_p)) ok = false;
    }
    const bool unseen = T_total <= 0 && !p.reduce_out;  // no query sees any of these keys: zeros
    if (ok || unseen) {
      tc_fence_after_sync();
      const bool row_ok = kvpos < p.Skv;
      const int which = (cw == 0) ? 1 : 0;  // packed buffer: [0] = dK, [1] = dV
      const float mul = (cw == 0) ? 1.0f / (1 << kShift) : p.scale;
      const uint32_t a_acc = tmem_base + lane_addr + (cw == 0 ? Cfg::kTmDV : Cfg::kTmDK);
      T* const out16 = static_cast<T*>(cw == 0 ? p.dv16 : p.dk16);
      const size_t base16 = ((static_cast<size_t>(b) * p.Skv + kvpos) * p.Hkv + hkv) * p.D + hf * DH;
      const size_t base = (((static_cast<size_t>(which) * p.B + b) * p.Skv + kvpos) * p.Hkv + hkv) * p.D + hf * DH;
#pragma unroll 1
      for (int c = 0; c < DH / 32; ++c) {
        uint32_t r[32];
        if (ok) {
          tmem_ld32(a_acc + c * 32, r);
          tmem_ld_wait32(r);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0;
        }
        if (row_ok && out16 != nullptr) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (hf * DH + c * 32 + k * 8 < p.D) {
              uint4 w;
              w.x = Pack2<T>::pack(__uint_as_float(r[8 * k + 0]) * mul, __uint_as_float(r[8 * k + 1]) * mul);
              w.y = Pack2<T>::pack(__uint_as_float(r[8 * k + 2]) * mul, __uint_as_float(r[8 * k + 3]) * mul);
              w.z = Pack2<T>::pack(__uint_as_float(r[8 * k + 4]) * mul, __uint_as_float(r[8 * k + 5]) * mul);
              w.w = Pack2<T>::pack(__uint_as_float(r[8 * k + 6]) * mul, __uint_as_float(r[8 * k + 7]) * mul);
              *reinterpret_cast<uint4*>(out16 + base16 + c * 32 + k * 8) = w;
            }
          }
        } else if (row_ok) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int d = hf * DH + c * 32 + k * 4;
            if (d < p.D) {
              float4 v = make_float4(__uint_as_float(r[4 * k + 0]) * mul, __uint_as_float(r[4 * k + 1]) * mul,
                                     __uint_as_float(r[4 * k + 2]) * mul, __uint_as_float(r[4 * k + 3]) * mul);
              if (p.reduce_out) {
                // several CTAs (one per run of the query tiles) add into the same rows; the host prepared dkdv_out
                red_add_v4_f32(p.dkdv_out + base + c * 32 + k * 4, v.x, v.y, v.z, v.w);
              } else {
                *reinterpret_cast<float4*>(p.dkdv_out + base + c * 32 + k * 4) = v;
              }
            }
          }
        }
      }
    }
    if (part_sem != nullptr) {
      __threadfence();
      __syncwarp();
      if (lane == 0) red_release_gpu_add(part_sem, 1);
    }
    __syncwarp();
  } else {
    // =========================== dQ reduction warpgroups ===========================
    // Two warpgroups, each owning half of the query columns of dQ^T.  A thread pulls its whole share into registers
    // with one batch of loads and releases the tensor-memory columns at once (the next dP^T product is waiting for
    // them); the reductions into global memory (bulk, or vector ones at head dim 256 and in the ordered mode), which
    // drain at the rate the L2 can add, then overlap the next tile's products instead of sitting in front of them.
    setmaxnreg_dec<80>();
    constexpr int kRedCols = BQ / 2;
    constexpr int NCR = kRedCols / 32;
    const int half = (warp - 12) >> 2;
    const int quarter = warp & 3;
    const int drow = quarter * 32 + lane;  // row of dQ^T = head-dim index inside this CTA's half
    const BwdWalk walk(plan, G);
    const int b = plan.b, hf = plan.hf, T_total = plan.t_total;
    const int d = hf * DH + drow;
    const bool d_ok = (drow < DH) && (hf * DH + quarter * 32 < p.D);  // the same for the whole warp
    // Warps with nothing but padding in their rows only take part in releasing the columns: in a loop of their own, except
    // at head dim 64, where half of the warps have no rows at all (143 us inside the common loop, 147 apart: S 4096, 16
    // heads; head dim 128 spills fewer registers with it apart).
    constexpr bool kApart = (DP > 64);
    if (kApart && !d_ok) {
      for (int t = 0; t < T_total && run; ++t) {
        if (!mbar_wait_warp(&bar_dq_full, t & 1, abort_p)) break;
        mbar_arrive(&bar_dq_drained);
      }
    }
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t a_dq = tmem_base + lane_addr + Cfg::kTmDQ + half * kRedCols;
    // dQ accumulator layout (fp32, private): [b][hq][Spad/128 tiles][DP/32][32 groups of 4 rows][32][4].  Lane = head-dim
    // index, four consecutive registers = four consecutive query rows: 512 contiguous bytes per warp and row group, and
    // what a warp adds for a tile is one contiguous run.
    constexpr size_t kTileElems = static_cast<size_t>(128) * DP;
    const int nQt128 = p.Spad / 128;
    bool ok = run && (!kApart || d_ok);
    for (int t = 0; t < T_total && ok; ++t) {
      const int hq = walk.head(t);
      const int q0 = walk.tile(t) * BQ;
      if (!mbar_wait_warp(&bar_dq_full, t & 1, abort_p)) { ok = false; break; }
      tc_fence_after_sync();
      float* base = p.dq_acc + ((static_cast<size_t>(b) * p.Hq + hq) * nQt128 + q0 / 128) * kTileElems +
                    (d / 32) * 4096 + (q0 % 128 + half * kRedCols) / 4 * 128;  // of the warp's 32 head-dim columns
      uint32_t r[NCR][32];
      if (kApart || d_ok) {
#pragma unroll
        for (int c = 0; c < NCR; ++c) tmem_ld32(a_dq + c * 32, r[c]);
        tmem_ld_wait32(r[0]);
#pragma unroll
        for (int c = 1; c < NCR; ++c) reg_fence32(r[c]);
      }
      // every read of this half of dQ^T has completed: the columns may be overwritten by the next dP^T
      tc_fence_before_sync();
      mbar_arrive(&bar_dq_drained);
      // Ordered mode (bit-reproducible dQ): the contributions of the kv tiles to one accumulator tile are added in
      // kv-tile order.  One counter per (head, query tile, warp slice); the CTA of kv tile j adds after j earlier
      // tiles have.  The CTA of the previous kv tile (same heads) always has a lower block index, so it was
      // dispatched before this one: it is resident or finished, never pending behind the waiter.
      int* order_sem = nullptr;
      if (p.dq_order != nullptr) {
        order_sem = p.dq_order +
                    ((((static_cast<size_t>(b) * p.Hq + hq) * ((p.Sq + BQ - 1) / BQ) + q0 / BQ) * Cfg::kHalves + hf) * 2 + half) * 4 +
                    quarter;
        if (!wait_count(order_sem, plan.kvt, lane == 0 && d_ok, abort_p)) { ok = false; break; }
      }
      if (!kApart && !d_ok) continue;
      if (Cfg::kStageDQ && order_sem == nullptr) {
        constexpr int kChunks = kRedCols / 4 / Cfg::kDQGroups;
        const uint32_t wbuf = ((half * (Cfg::kDQWarps / 2) + quarter) * 2) * Cfg::kDQBufBytes;
        static_for<0, kChunks>([&](auto ck_) {
          constexpr int ck = decltype(ck_)::value;
          const uint32_t buf = wbuf + ((kChunks % 2 == 0) ? (ck & 1) : (t & 1)) * Cfg::kDQBufBytes;
          float4* stage = reinterpret_cast<float4*>(dq_ptr + buf) + lane;
          if (lane == 0) bulk_wait_read<1>();  // the reduction before the last one has read this buffer
          __syncwarp();
#pragma unroll
          for (int k = 0; k < Cfg::kDQGroups; ++k) {
            constexpr int g0 = ck * Cfg::kDQGroups;
            const uint32_t* v = &r[(g0 + k) / 8][((g0 + k) % 8) * 4];
            stage[k * 32] = make_float4(__uint_as_float(v[0]) * p.scale, __uint_as_float(v[1]) * p.scale,
                                        __uint_as_float(v[2]) * p.scale, __uint_as_float(v[3]) * p.scale);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            bulk_reduce_add_f32(base + ck * Cfg::kDQGroups * 128, smem_base + Cfg::kOffDQ + buf, Cfg::kDQBufBytes);
            bulk_commit();
          }
        });
      } else {
        // rows beyond Sq and head-dim columns beyond D hold exact zeros (zero-filled operands, P = 0)
#pragma unroll
        for (int c = 0; c < NCR; ++c) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            red_add_v4_f32(base + (c * 8 + k) * 128 + lane * 4, __uint_as_float(r[c][4 * k + 0]) * p.scale,
                           __uint_as_float(r[c][4 * k + 1]) * p.scale, __uint_as_float(r[c][4 * k + 2]) * p.scale,
                           __uint_as_float(r[c][4 * k + 3]) * p.scale);
            if (order_sem == nullptr) __nanosleep(kRedSleepNs);
          }
        }
        if (order_sem != nullptr) {
          __threadfence();  // this lane's reductions are performed before the counter moves
          __syncwarp();
          if (lane == 0) red_release_gpu_add(order_sem, 1);
        }
      }
    }
    if (Cfg::kStageDQ && lane == 0) bulk_wait<0>();
    __syncwarp();
  }

  // ---- teardown ----
  tc_fence_before_sync();
  __syncthreads();
  if (abort_flag) {
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    if (tid == 0) atomicExch(p.status, kStatusWaitTimeout);
  }
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int DP, int DH, int BQ, int NSQ, int NSO, typename T, int kKind>
static int launch_scored_bwd(const void* q, const void* k, const void* v, const void* dout, const ScoredBwdParams& prm,
                             int dtype, cudaStream_t stream) {
  using Cfg = BwdCfg<DP, DH, BQ, NSQ, NSO>;
  const BwdParams& p = prm.p;
  CUtensorMap tq, tk, tv, tdo;
  int rc;
  if ((rc = make_tmap_bshd(&tq, q, dtype, p.B, p.Sq, p.Hq, p.D, BQ)) != RFA_OK) return rc;
  if ((rc = make_tmap_bshd(&tdo, dout, dtype, p.B, p.Sq, p.Hq, p.D, BQ)) != RFA_OK) return rc;
  if ((rc = make_tmap_bshd(&tk, k, dtype, p.B, p.Skv, p.Hkv, p.D, 128)) != RFA_OK) return rc;
  if ((rc = make_tmap_bshd(&tv, v, dtype, p.B, p.Skv, p.Hkv, p.D, 128)) != RFA_OK) return rc;
  auto kern = scored_bwd_kernel<DP, DH, BQ, NSQ, NSO, T, kKind>;
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) { cudaGetLastError(); return RFA_ERR_CUDA; }
  if (!attr_done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
    if (e != cudaSuccess) { cudaGetLastError(); return RFA_ERR_CUDA; }
    // A raise of the warpgroups' registers that the launch's pool cannot satisfy would wait forever: a build whose register
    // count does not cover the allowances is refused.
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) { cudaGetLastError(); return RFA_ERR_CUDA; }
    if (fa.numRegs * Cfg::kThreads < 128 * 64 + 256 * 128 + 256 * 80) return RFA_ERR_UNSUPPORTED;
    attr_done[dev] = true;
  }
  const unsigned grid = static_cast<unsigned>(ceil_div(p.Skv, 128)) * p.Hkv * p.B * Cfg::kHalves * p.nsplit;
  return launch_chained(kern, grid, Cfg::kThreads, Cfg::kSmemBytes, stream, tq, tk, tv, tdo, prm);
}

template <typename T, int kKind>
static int dispatch_dim(const void* q, const void* k, const void* v, const void* dout, const ScoredBwdParams& prm, int dtype,
                        cudaStream_t stream) {
  switch (padded_head_dim(prm.p.D)) {
    case 64: return launch_scored_bwd<64, 64, 128, 2, 2, T, kKind>(q, k, v, dout, prm, dtype, stream);
    case 128: return launch_scored_bwd<128, 128, 128, 2, 1, T, kKind>(q, k, v, dout, prm, dtype, stream);
    case 256: return launch_scored_bwd<256, 128, 64, 2, 1, T, kKind>(q, k, v, dout, prm, dtype, stream);
    default: return RFA_ERR_UNSUPPORTED;
  }
}

template <typename T>
static int dispatch_kind(const void* q, const void* k, const void* v, const void* dout, const ScoredBwdParams& prm, int dtype,
                         cudaStream_t stream) {
  switch (score_kind(prm.sc)) {
    case 0: return dispatch_dim<T, 0>(q, k, v, dout, prm, dtype, stream);
    case 1: return dispatch_dim<T, 1>(q, k, v, dout, prm, dtype, stream);
    case 2: return dispatch_dim<T, 2>(q, k, v, dout, prm, dtype, stream);
    default: return dispatch_dim<T, 3>(q, k, v, dout, prm, dtype, stream);
  }
}

static int scored_dispatch(const void* q, const void* k, const void* v, const void* dout, const ScoredBwdParams& prm,
                           int dtype, cudaStream_t stream) {
  if (dtype == RFA_DTYPE_BF16) return dispatch_kind<__nv_bfloat16>(q, k, v, dout, prm, dtype, stream);
  return dispatch_kind<__half>(q, k, v, dout, prm, dtype, stream);
}

static int scored_bwd_params(const void* k, const float* lse2, const float* delta, float* dq_acc, float* dkdv_out, int B,
                             int S, int Hq, int Hkv, int D, int dtype, const rfa_score_args* args, int* dq_order, int* status,
                             ScoredBwdParams* prm) {
  const int rc = make_score_params(args, B, S, &prm->sc);
  if (rc != RFA_OK) return rc;
  BwdParams& p = prm->p;
  p = BwdParams{};
  p.k = k;
  p.lse2 = lse2;
  p.delta = delta;
  p.dq_acc = dq_acc;
  p.dkdv_out = dkdv_out;
  p.B = B;
  p.Sq = p.Skv = p.kv_len = S;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.D = D;
  p.Spad = round_up(S, 128);
  // of dQ and dK
  p.scale = args->softmax_scale / (1 << (dtype == RFA_DTYPE_BF16 ? weight_shift<__nv_bfloat16>() : weight_shift<__half>()));
  p.scale_log2 = args->softmax_scale * kLog2e;
  // the shape of the work that the split of the K/V tiles is chosen for: documents only shorten it
  p.causal = prm->sc.causal && prm->sc.q_pos == prm->sc.k_pos ? 1 : 0;
  p.dq_order = dq_order;
  p.status = status;
  const int dp = padded_head_dim(D), halves = dp == 256 ? 2 : 1;
  const long long units = static_cast<long long>(ceil_div(S, 128)) * Hkv * B * halves;
  if (units * 16 > INT_MAX) return RFA_ERR_TOO_LARGE;
  choose_split(p, units, dp == 256 ? 64 : 128);
  return RFA_OK;
}

// Bytes of the ordering counters that a launch uses: per query tile, and per K/V tile where the tiles are split.
static size_t order_bytes(const BwdParams& p) {
  const int dp = padded_head_dim(p.D), halves = dp == 256 ? 2 : 1;
  size_t n = static_cast<size_t>(p.B) * p.Hq * ceil_div(p.Sq, dp == 256 ? 64 : 128) * halves * 8;
  if (p.nsplit > 1) n += static_cast<size_t>(p.B) * p.Hkv * ceil_div(p.Skv, 128) * halves * 8;
  return n * sizeof(int);
}

static bool misaligned(std::initializer_list<const void*> ptrs) {
  for (const void* x : ptrs)
    if (reinterpret_cast<uintptr_t>(x) & 15u) return true;
  return false;
}

}  // namespace rfa

extern "C" int rfa_scored_bwd_hop(const void* q, const void* k, const void* v, const void* dout, const float* lse2,
                                  const float* delta, float* dq_acc, float* dkdv_out, int B, int S, int Hq, int Hkv, int D,
                                  int dtype, const rfa_score_args* args, int* dq_order, int* status, void* stream) {
  using namespace rfa;
  if (!dq_acc || !args) return RFA_ERR_INVALID_ARG;
  int rc = bwd_check_args(q, k, v, dout, lse2, delta, nullptr, dkdv_out, B, S, S, Hq, Hkv, D, dtype, args->softmax_scale, 0,
                          0, 0, S, status);
  if (rc != RFA_OK) return rc;
  if (misaligned({dq_acc, k}) || (reinterpret_cast<uintptr_t>(dq_order) & 3u)) return RFA_ERR_INVALID_ARG;
  ScoredBwdParams prm;
  rc = scored_bwd_params(k, lse2, delta, dq_acc, dkdv_out, B, S, Hq, Hkv, D, dtype, args, dq_order, status, &prm);
  if (rc != RFA_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if ((rc = prepare_dkdv(prm.p, s)) != RFA_OK) return rc;
  if (dq_order != nullptr && (rc = cuda_status(cudaMemsetAsync(dq_order, 0, order_bytes(prm.p), s))) != RFA_OK) return rc;
  return scored_dispatch(q, k, v, dout, prm, dtype, s);
}

// Three launches, as in rfa_bwd_local: delta, lse2 and the cleared buffers; the hop; the conversions.
extern "C" int rfa_scored_bwd_local(const void* q, const void* k, const void* v, const void* out, const void* dout,
                                    const float* lse, float* delta, float* lse2, float* dq_acc, float* dkdv, void* dq,
                                    void* dk, void* dv, int B, int S, int Hq, int Hkv, int D, int dtype,
                                    const rfa_score_args* args, int* dq_order, int* status, void* stream) {
  using namespace rfa;
  if (!out || !lse || !dq_acc || !dq || !dk || !dv || !args) return RFA_ERR_INVALID_ARG;
  int rc = bwd_check_args(q, k, v, dout, lse2, delta, nullptr, dkdv, B, S, S, Hq, Hkv, D, dtype, args->softmax_scale, 0, 0, 0,
                          S, status);
  if (rc != RFA_OK) return rc;
  if (misaligned({dq_acc, dq, dk, dv, dq_order, out, dout, k})) return RFA_ERR_INVALID_ARG;
  ScoredBwdParams prm;
  rc = scored_bwd_params(k, lse2, delta, dq_acc, dkdv, B, S, Hq, Hkv, D, dtype, args, dq_order, status, &prm);
  if (rc != RFA_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ClearList clear;
  clear.add(dq_acc, rfa_dq_acc_elems(B, S, Hq, D) * sizeof(float));
  if (prm.p.reduce_out) {
    clear.add(dkdv, static_cast<size_t>(2) * B * S * Hkv * D * sizeof(float));
  } else {
    prm.p.dk16 = dk;
    prm.p.dv16 = dv;
  }
  if (dq_order != nullptr) clear.add(dq_order, order_bytes(prm.p));
  if ((rc = launch_bwd_prepare(out, dout, lse, delta, lse2, B, S, Hq, D, dtype, clear, s)) != RFA_OK) return rc;
  if ((rc = scored_dispatch(q, k, v, dout, prm, dtype, s)) != RFA_OK) return rc;
  return launch_bwd_finish(dq_acc, dq, prm.p.reduce_out ? dkdv : nullptr, dk, dv, B, S, S, Hq, Hkv, D, dtype, s);
}
