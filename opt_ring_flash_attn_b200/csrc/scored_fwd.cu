// Forward hop of attention with modified scores: capped by a tanh, biased by distance, masked by documents and prefixes.
//
//   x = scale * q.k;   y = cap * tanh(x / cap);   z = y - slope |i - j|;   O, lse = online softmax over the visible keys
//
// The structure of a CTA is that of the plain forward hop (a TMA warp, an issuing warp, one softmax warpgroup per tile of
// 128 queries; tensor memory holds O and the scores), with these differences.
//  * A CTA walks the range of key tiles that the hull of its rows' intervals gives, each of its query tiles its own part of
//    it, so what no row sees is neither loaded nor multiplied.  With a mask the blocks take their tiles from its work list,
//    long ones first.
//  * Scores are brought to log2 units before the row maximum is taken, where a cap or a bias stands between them and it.
//  * A tile inside every row's interval needs no test; in the others a row compares the key with its own interval.
//  * A row that has seen no key keeps the finite maximum kNoKey, and ends with out = 0, lse = -inf.
//  * The issuing warp clears the padding rows of a V tile that holds the border between real rows and padding.
//  * Without a ring, few heads share the key tiles of a row among several CTAs; a second kernel joins their states.
//
// Bound, as the plain hop, by the chain of one query tile (scores, softmax, products), which two tiles per CTA overlap; by the
// start and end of CTAs where documents are short (5 us of a CTA's 30 at 13 key tiles a pair); and with a cap by the arithmetic
// units, whose phases (cap, maximum, exponentials) a warpgroup goes through in turn.  Forward hop, causal, us: S 4096, 32/8
// heads of 128: no change 132, bias 173, cap 195, both 232; 16 heads of 64: 63, 77, 98, 118; 16/8 heads of 256: 122, 153, 154, 186.
// S 16384, 32/8 heads of 128, ten documents: 422 us = 832 TFLOP/s of visible pairs, tensor pipe 48 % busy.
#include "fwd_common.cuh"
#include "scored.cuh"

namespace rfa {

struct ScoredFwdParams {
  float* acc;
  float* m;
  float* l;
  void* out;
  float* lse;
  int B, S, Hq, Hkv, D;
  int Spad, nT;
  int first, last;
  int nsplit;  // CTAs that share the key tiles of a pair of query tiles; each leaves its state in a copy of its own
  size_t acc_split, ml_split;  // elements between the copies
  int* status;
  ScoreParams sc;
};

// Scores of 32 keys in log2 units: the cap and the bias.  `bias` holds what is added to the first two keys, `step` what it
// grows by from pair to pair (bias and step include the constant of the tanh).
template <int kKind>
__device__ __forceinline__ void transform32(uint32_t (&r)[32], uint64_t scale2, uint64_t gain2, uint64_t bias, uint64_t step) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    uint64_t y;
    if constexpr (!has_cap(kKind)) {
      y = fma2(pack_u2(r[2 * i], r[2 * i + 1]), scale2, bias);
    } else {
      // cap * tanh(x / cap) = cap - 2 cap / (exp(2 x / cap) + 1); scale2 turns the raw score into the exponent, gain2 is
      // -2 cap, cap itself is in the bias.  Both ends of the range come out as they should: exp2 gives 0 or an infinity.
      float a0, a1;
      unpack_f2(mul2(pack_u2(r[2 * i], r[2 * i + 1]), scale2), a0, a1);
      float e0, e1;
      unpack_f2(add2(pack_f2(fast_exp2(a0), fast_exp2(a1)), pack_f2(1.f, 1.f)), e0, e1);
      y = fma2(pack_f2(fast_rcp(e0), fast_rcp(e1)), gain2, bias);
    }
    unpack_u2(y, r[2 * i], r[2 * i + 1]);
    if (has_bias(kKind)) bias = add2(bias, step);
  }
}

// cap * tanh(x) for |x| <= 0.8 on the FMA pipe: x times a polynomial of degree 4 in x^2 (least squares on [0, 0.8], reweighted
// to even out the absolute error of the tanh: 3.5e-7).  The formula with exp2 and a reciprocal takes two turns on the
// special-function unit per score, beside the one of the softmax, which makes it the unit that a tile waits for.  Forward hop,
// scores of 3.2 on average, caps of 50 / 20 / 5 (where no, few and most chunks leave the range), by the formula alone: S 4096,
// 32/8 heads of 128 262 / 260 / 259 us, with the polynomial 219 / 217 / 289; 16 heads of 64 133 / 133 / 132 and 113 / 110 / 145
// (before the masks became cheaper).
// The coefficients take ten registers, which is why the softmax keeps to exp2 beside a cap.  They hold the powers of `in`, which
// turns a raw score into x, so the polynomial is one of the raw score; where the ninth power would leave fp32 (or its product
// with the cap its normal numbers), which no ordinary scale and cap do, every tile takes the formula.
struct TanhPoly {
  float limit;  // of the square of a raw score
  bool usable;
  uint64_t c[5];
  __device__ __forceinline__ TanhPoly(float in, float cap) {
    usable = in > 2e-4f && in < 1e3f;
    limit = 0.64f / (in * in);
    float power = cap * in;
    const float k[5] = {0.9999951124191284f, -0.3331742584705353f, 0.13186223804950714f, -0.04826141893863678f,
                        0.011464733630418777f};
#pragma unroll
    for (int i = 0; i < 5; ++i, power *= in * in) c[i] = pack_f2(power * k[i], power * k[i]);
  }
  // `top` follows the largest square
  __device__ __forceinline__ uint64_t operator()(uint64_t score, uint64_t bias, float& top) const {
    const uint64_t u = mul2(score, score);
    float u0, u1;
    unpack_f2(u, u0, u1);
    top = max3_nan(top, u0, u1);
    uint64_t y = fma2(c[4], u, c[3]);
    y = fma2(y, u, c[2]);
    y = fma2(y, u, c[1]);
    y = fma2(y, u, c[0]);
    return fma2(score, y, bias);
  }
};

template <int kKind>
__device__ __forceinline__ void cap32(uint32_t (&r)[32], const TanhPoly& poly, uint64_t bias, uint64_t step, float& top) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    unpack_u2(poly(pack_u2(r[2 * i], r[2 * i + 1]), bias, top), r[2 * i], r[2 * i + 1]);
    if (has_bias(kKind)) bias = add2(bias, step);
  }
}

// The lowest n of 32 bits; none for n < 0, all for n > 32.
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (1u << max(n, 0)) - 1u; }

// Largest of 32 scores (independent partial maxima keep the dependency chains short).
__device__ __forceinline__ float max32(const uint32_t (&r)[32]) {
  float a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
#pragma unroll
  for (int i = 2; i < 30; i += 4) {
    a = max3_nan(a, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
    b = max3_nan(b, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
  }
  return max_nan(max3_nan(a, __uint_as_float(r[30]), __uint_as_float(r[31])), b);
}

// Softmax warpgroups per query tile.  Where a CTA holds one tile only (head dim 256) and there is a cap, two of them share its
// keys, half each, and compare their maxima: one alone has a warp per scheduler for all of the arithmetic.  S 4096, 16/8 heads of
// 256, us, one and two: cap 181, 166; with a bias too 210, 189 (before the polynomial became shorter).  Without a cap one keeps up with the
// copies and the products, and the comparing costs: 129, 132; with a bias 153, 153.  With two tiles per CTA it loses, 104 registers
// per thread being too few: 32/8 heads of 128 233, 284.
constexpr int fwd_share(int NQ, int kind) { return NQ == 1 && has_cap(kind) ? 2 : 1; }
constexpr int fwd_threads(int NQ, int kind) { return 128 + NQ * fwd_share(NQ, kind) * 128; }

template <int DP, int BN, int NQ, int NS, typename T, int kKind>
__global__ void __launch_bounds__(fwd_threads(NQ, kKind), 1)
    scored_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const ScoredFwdParams p) {
  using Cfg = FwdCfg<DP, BN, NQ, NS>;
  constexpr int kSlots = Cfg::kSlots;
  constexpr bool kBf16 = Pack2<T>::kIsBf16;
  constexpr int kPvParts = (DP == 64) ? 2 : 4;     // P is handed to the issuer in parts, as in the plain hop
  constexpr int kPartChunks = BN / 32 / kPvParts;
  constexpr int kShare = fwd_share(NQ, kKind);
  constexpr int kPolyEvery = (NQ == 2 && !has_cap(kKind)) ? kFwdPolyEvery : 0;  // a cap keeps the FMA pipe busy

  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_q_full;
  __shared__ uint64_t bar_kv_full[kSlots];
  __shared__ uint64_t bar_kv_empty[kSlots];
  __shared__ uint64_t bar_s_full[NQ * NS];
  __shared__ uint64_t bar_p_ready[NQ * NS * kPvParts];
  __shared__ uint64_t bar_pv_done[NQ];
  __shared__ uint64_t bar_pair[4];                          // two warps with the same rows of a tile
  __shared__ float pair_value[kShare == 2 ? 2 : 1][128];    // maximum or sum of each half of a row's keys
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag, skip_flag;

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t s_q = smem_base;
  const uint32_t s_kv = smem_base + NQ * Cfg::kQBytes;

  if (tid == 0) {
    abort_flag = 0;
    mbar_init(&bar_q_full, 1);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&bar_kv_full[i], 1);
      mbar_init(&bar_kv_empty[i], 1);
    }
    for (int i = 0; i < NQ * NS; ++i) {
      mbar_init(&bar_s_full[i], 1);
      for (int h = 0; h < kPvParts; ++h) mbar_init(&bar_p_ready[i * kPvParts + h], 128);
    }
    for (int i = 0; i < NQ; ++i) mbar_init(&bar_pv_done[i], 1);
    for (int i = 0; i < 4; ++i) mbar_init(&bar_pair[i], 2);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_holder, 512);
    tmem_relinquish();
  }
  pdl_wait();  // nothing above touches global memory

  // ---- tile coordinates: most work first, heads fastest ----
  const int nQs = (p.nT + NQ - 1) / NQ;
  const int split = blockIdx.x % p.nsplit, block = blockIdx.x / p.nsplit;
  int b, h, qs;
  if (p.sc.has_mask) {
    const int item = __ldg((NQ == 2 ? p.sc.mask.order_q2 : p.sc.mask.order_q) + block / p.Hq);
    h = block % p.Hq;
    b = item / nQs;
    qs = item % nQs;
  } else {
    const int per_qs = p.Hq * p.B, rem = block % per_qs;
    qs = nQs - 1 - block / per_qs;
    b = rem / p.Hq;
    h = rem % p.Hq;
  }
  const int hkv = h / (p.Hq / p.Hkv);

  // Range of key tiles of each query tile: tiles [j0 + t_lo[q], j0 + t_hi[q]) of the block, j0 the first of the CTA.
  int m0[NQ], t_lo[NQ], t_hi[NQ], full_lo[NQ], full_hi[NQ];  // keys [full_lo, full_hi) of the block are seen by every row
  int j0 = INT_MAX, j1 = 0;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    m0[q] = (qs * NQ + q) * 128;
    t_lo[q] = t_hi[q] = full_lo[q] = full_hi[q] = 0;
    if (m0[q] < p.S) {
      const int4 hull = query_hull(p.sc, b, p.nT, qs * NQ + q, p.S);
      const int lo = max(hull.x - p.sc.k_pos, 0), hi = min(hull.w - p.sc.k_pos, p.S);
      full_lo[q] = max(hull.y, p.sc.k_pos) - p.sc.k_pos;
      full_hi[q] = min(hull.z - p.sc.k_pos, p.S);
      if (lo < hi) {
        t_lo[q] = lo / BN;
        t_hi[q] = (hi + BN - 1) / BN;
        j0 = min(j0, t_lo[q]);
        j1 = max(j1, t_hi[q]);
      }
    }
  }
  if (j0 > j1) j0 = j1;  // nothing to do
  if (p.nsplit > 1) {  // this CTA's run of them
    const int n = j1 - j0, from = j0 + n * split / p.nsplit, to = j0 + n * (split + 1) / p.nsplit;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      t_lo[q] = max(t_lo[q], from);
      t_hi[q] = min(t_hi[q], to);
      if (t_lo[q] >= t_hi[q]) t_lo[q] = t_hi[q] = 0;
    }
    j0 = from;
    j1 = to;
  }
  const int nmax = j1 - j0;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    t_lo[q] = t_hi[q] > 0 ? t_lo[q] - j0 : 0;
    t_hi[q] = t_hi[q] > 0 ? t_hi[q] - j0 : 0;
  }
  // rows of the key block that are no padding
  const int real_lo = p.sc.has_mask ? __ldg(p.sc.mask.real + 2 * b) - p.sc.k_pos : 0;
  const int real_hi = p.sc.has_mask ? __ldg(p.sc.mask.real + 2 * b + 1) - p.sc.k_pos : p.S;

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

  if (warp < 4) {
    if constexpr (NQ == 2) setmaxnreg_dec<Cfg::kServiceRegs>();
    if (warp == 0) {
      // =========================== TMA producer ===========================
      if (lane == 0 && nmax > 0) {
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        int nvalid = 0;
#pragma unroll
        for (int q = 0; q < NQ; ++q) nvalid += (t_hi[q] > 0) ? 1 : 0;
        mbar_expect_tx(&bar_q_full, static_cast<uint32_t>(nvalid) * Cfg::kQBytes);
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          if (t_hi[q] > 0) {
#pragma unroll
            for (int pn = 0; pn < Cfg::kPanels; ++pn)
              tma_load_4d(s_q + q * Cfg::kQBytes + pn * (128 * 128), &tm_q, &bar_q_full, pn * 64, h, m0[q], b);
          }
        }
        SlotWalk<kSlots> w;
        auto load = [&](int which, int j) {
#pragma unroll
          for (int pc = 0; pc < Cfg::kPieces; ++pc, w.next()) {
            if (!mbar_wait(&bar_kv_empty[w.slot], w.phase ^ 1, abort_p)) return false;
            mbar_expect_tx(&bar_kv_full[w.slot], Cfg::kKVBytes);
#pragma unroll
            for (int pn = 0; pn < Cfg::kPanels / Cfg::kPieces; ++pn)
              tma_load_4d(s_kv + w.slot * Cfg::kKVBytes + pn * (BN * 128), which ? &tm_v : &tm_k, &bar_kv_full[w.slot],
                          (Cfg::kPanels / Cfg::kPieces * pc + pn) * 64, hkv, (j0 + j) * BN, b);
          }
          return true;
        };
        if constexpr (NS == 2) {  // in the order in which the products use them: K0, K1, V0, K2, V1, ...
          bool ok = load(0, 0);
          for (int j = 0; j < nmax && ok; ++j) ok = (j + 1 == nmax || load(0, j + 1)) && load(1, j);
        } else {
          bool ok = true;
          for (int j = 0; j < nmax && ok; ++j) ok = load(0, j) && load(1, j);
        }
      }
      __syncwarp();
    } else if (warp == 1 && nmax > 0) {
      // =========================== MMA issuer ===========================
      const uint32_t el = elect_one();
      const int d16 = (p.D + 15) / 16 * 16;
      constexpr uint32_t idesc_qk = make_idesc(128, BN, kBf16, false, false);
      // A tile on the border between real rows and padding: what its products would multiply by 0 is cleared first.
      auto clear_v = [&](int slot, int j) {
        const int r0 = (j0 + j) * BN;
        if (real_lo > r0 || real_hi < min(r0 + BN, p.S))
          clear_padding_rows(s_kv + slot * Cfg::kKVBytes, Cfg::kPanels / Cfg::kPieces, BN, real_lo - r0, real_hi - r0, lane);
      };
      if constexpr (NS == 2) {
        auto idesc_pv = [&](int pc) { return make_idesc(128, min(d16 - pc * 128, 128), kBf16, false, true); };
        const uint32_t q_lo = desc_lo_kmajor(s_q);
        SlotWalk<kSlots> w;
        auto s_tm = [&](int j) { return tmem_base + Cfg::kTmS + (j & 1) * BN; };
        auto qk = [&](int j) {
          bool got = true;
          static_for<0, Cfg::kPieces>([&](auto pc_) {
            constexpr int pc = decltype(pc_)::value;
            if (!got) return;
            got = mbar_wait_warp(&bar_kv_full[w.slot], w.phase, abort_p);
            if (!got) return;
            tc_fence_after_sync();
            issue_qk<128, BN>(s_tm(j), q_lo + pc * (2 * 128 * 128 / 16), desc_lo_kmajor(s_kv + w.slot * Cfg::kKVBytes),
                              idesc_qk, el, pc > 0);
            mma_commit_e(&bar_kv_empty[w.slot], el);
            w.next();
          });
          if (got) mma_commit_e(&bar_s_full[j & 1], el);
          return got;
        };
        bool ok = mbar_wait_warp(&bar_q_full, 0, abort_p) && qk(0);
        for (int j = 0; j < nmax && ok; ++j) {
          // Score buffer (j+1)&1 is free: P_{j-1} was consumed by the PV issued last iteration.
          if (j + 1 < nmax && !qk(j + 1)) break;
          uint32_t v_lo[Cfg::kPieces];
          int v_slot[Cfg::kPieces];
#pragma unroll
          for (int pc = 0; pc < Cfg::kPieces; ++pc, w.next()) {
            v_slot[pc] = w.slot;
            v_lo[pc] = desc_lo_mnmajor(s_kv + w.slot * Cfg::kKVBytes, BN * 128);
            ok = ok && mbar_wait_warp(&bar_kv_full[w.slot], w.phase, abort_p);
            if (ok) clear_v(w.slot, j);
          }
          static_for<0, kPvParts>([&](auto h_) {
            constexpr int h = decltype(h_)::value;
            ok = ok && mbar_wait_warp(&bar_p_ready[(j & 1) * kPvParts + h], (j >> 1) & 1, abort_p);
            if (!ok) return;
            tc_fence_after_sync();
#pragma unroll
            for (int pc = 0; pc < Cfg::kPieces; ++pc)
              issue_pv<128, BN, 2 * kPartChunks * h, 2 * kPartChunks * (h + 1)>(
                  tmem_base + Cfg::kTmO + pc * 128, s_tm(j), v_lo[pc], idesc_pv(pc), (h > 0) || (j > 0) || (p.first == 0), el);
          });
          if (!ok) break;
          mma_commit_e(&bar_pv_done[0], el);
#pragma unroll
          for (int pc = 0; pc < Cfg::kPieces; ++pc) mma_commit_e(&bar_kv_empty[v_slot[pc]], el);
        }
      } else {
        const uint32_t idesc_pv = make_idesc(128, d16, kBf16, false, true);
        auto slot_of = [&](int u) { return u % kSlots; };
        auto par_of = [&](int u) { return static_cast<uint32_t>((u / kSlots) & 1); };
        auto k_lo = [&](int u) { return desc_lo_kmajor(s_kv + slot_of(u) * Cfg::kKVBytes); };
        auto v_lo = [&](int u) { return desc_lo_mnmajor(s_kv + slot_of(u) * Cfg::kKVBytes, BN * 128); };
        uint32_t q_lo[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) q_lo[q] = desc_lo_kmajor(s_q + q * Cfg::kQBytes);
        auto s_tm = [&](int q) { return tmem_base + Cfg::kTmS + q * BN; };
        auto o_tm = [&](int q) { return tmem_base + Cfg::kTmO + q * DP; };
        auto wait_tile = [&](int u) { return mbar_wait_warp(&bar_kv_full[slot_of(u)], par_of(u), abort_p); };
        bool ok = mbar_wait_warp(&bar_q_full, 0, abort_p) && wait_tile(0);
        if (ok) {
          tc_fence_after_sync();
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            if (t_lo[q] == 0 && t_hi[q] > 0) {
              issue_qk<DP, BN>(s_tm(q), q_lo[q], k_lo(0), idesc_qk, el);
              mma_commit_e(&bar_s_full[q], el);
            }
          }
          mma_commit_e(&bar_kv_empty[slot_of(0)], el);
        }
        for (int j = 0; j < nmax && ok; ++j) {
          const int uv = 2 * j + 1, uk = 2 * (j + 1);
          if (!wait_tile(uv)) break;
          clear_v(slot_of(uv), j);
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            if (j >= t_lo[q] && j < t_hi[q]) {
              static_for<0, kPvParts>([&](auto h_) {
                constexpr int h = decltype(h_)::value;
                if (ok) {
                  if (!mbar_wait_warp(&bar_p_ready[q * kPvParts + h], (j - t_lo[q]) & 1, abort_p)) {
                    ok = false;
                  } else {
                    tc_fence_after_sync();
                    issue_pv<DP, BN, 2 * kPartChunks * h, 2 * kPartChunks * (h + 1)>(
                        o_tm(q), s_tm(q), v_lo(uv), idesc_pv, (h > 0) || (j > t_lo[q]) || (p.first == 0), el);
                  }
                }
              });
              if (!ok) break;
              if (j + 1 == t_hi[q]) mma_commit_e(&bar_pv_done[q], el);
            }
            if (j + 1 >= t_lo[q] && j + 1 < t_hi[q]) {
              if (!wait_tile(uk)) { ok = false; break; }
              tc_fence_after_sync();
              issue_qk<DP, BN>(s_tm(q), q_lo[q], k_lo(uk), idesc_qk, el);
              mma_commit_e(&bar_s_full[q], el);
            }
          }
          if (!ok) break;
          mma_commit_e(&bar_kv_empty[slot_of(uv)], el);
          if (j + 1 < nmax) {
            if (!wait_tile(uk)) break;  // also where no query tile uses it: a slot is released only once it is filled
            mma_commit_e(&bar_kv_empty[slot_of(uk)], el);
          }
        }
      }
      __syncwarp();
    }
  } else {
    // =========================== softmax warpgroups ===========================
    if constexpr (NQ == 2) setmaxnreg_inc<Cfg::kSoftmaxRegs>();
    const int q = kShare == 2 ? 0 : (warp - 4) >> 2;
    const int share = kShare == 2 ? (warp - 4) >> 2 : 0;  // half of the keys of a tile, and of the columns of O
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    // selected, not indexed: an array indexed at run time would live in local memory for the issuer as well
    const bool second = NQ == 2 && q == 1;
    const int t_first = second ? t_lo[NQ - 1] : t_lo[0];
    const int n = (second ? t_hi[NQ - 1] : t_hi[0]) - t_first;
    const int m0_q = second ? m0[NQ - 1] : m0[0];
    const int full_lo_q = second ? full_lo[NQ - 1] : full_lo[0];
    const int full_hi_q = second ? full_hi[NQ - 1] : full_hi[0];
    const int n_c32 = (p.D + 31) / 32;
    const int o_first = kShare == 2 && share == 1 ? (n_c32 + 1) / 2 : 0, o_end = kShare == 2 && share == 0 ? (n_c32 + 1) / 2 : n_c32;
    const int row_g = m0_q + row;
    const uint32_t o_addr = tmem_base + lane_addr + Cfg::kTmO + q * DP;
    const size_t bh = static_cast<size_t>(b) * p.Hq + h;
    float* acc_tile = p.acc + split * p.acc_split + ((bh * p.nT + (qs * NQ + q)) * (DP / 4)) * 512;  // [DP/4][128][4]
    const size_t ml_idx = bh * p.Spad + row_g + split * p.ml_split;

    if (m0_q < p.S && !(n == 0 && !p.first && !p.last)) {
      bool ok = true;
      float m_used = kNoKey;
      float l_sum = 0.f;
      if (!p.first || n == 0) {  // the state of the hops before, or of none
        if (!p.first) {
          m_used = p.m[ml_idx];
          if (share == 0) l_sum = p.l[ml_idx];
        }
#pragma unroll 1
        for (int c = o_first; c < o_end; ++c) {
          uint32_t r[32];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (!p.first) v = *reinterpret_cast<const float4*>(acc_tile + ((c * 8 + k) * 128 + row) * 4);
            r[4 * k + 0] = __float_as_uint(v.x);
            r[4 * k + 1] = __float_as_uint(v.y);
            r[4 * k + 2] = __float_as_uint(v.z);
            r[4 * k + 3] = __float_as_uint(v.w);
          }
          tmem_st32(o_addr + c * 32, r);
        }
        tmem_st_wait();
      }
      // Keys of the block that this row sees: [lo, lo + width).
      int lo = 0, width = p.S;
      if (row_g < p.S) {
        int hi = p.S;
        if (p.sc.has_mask) {
          const size_t at = static_cast<size_t>(b) * p.sc.len + p.sc.q_pos + row_g;
          lo = max(__ldg(p.sc.mask.q_lo + at) - p.sc.k_pos, 0);
          hi = min(__ldg(p.sc.mask.q_hi + at) - p.sc.k_pos, p.S);
        } else if (p.sc.causal) {
          hi = min(p.sc.q_pos + row_g + 1 - p.sc.k_pos, p.S);
        }
        width = max(hi - lo, 0);
      }
      const Exp2Poly exp2_poly;
      const float scale_log2 = p.sc.scale * kLog2e;
      const float cap_log2 = p.sc.cap * kLog2e;
      const float slope = has_bias(kKind) ? slope_log2(p.sc, b, p.Hq, h) : 0.f;
      const int ahead = p.sc.q_pos + row_g - p.sc.k_pos;  // position of this row, from the first key of the block
      // what a raw score is multiplied by, and the tanh's -2 cap
      const float in_scale = has_cap(kKind) ? 2.f * scale_log2 / p.sc.cap : scale_log2;
      const TanhPoly tanh_poly(p.sc.scale / p.sc.cap, cap_log2);
      int direct = tanh_poly.usable ? 0 : INT_MAX;  // tiles that take the formula at once
      uint32_t pair_par = 0;
      // Waits for the other warp with these rows; what either wrote before, tensor memory included, the other sees after.
      auto pair_sync = [&]() {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_pair[quarter]);
        const bool got = mbar_wait_warp(&bar_pair[quarter], pair_par, abort_p);
        pair_par ^= 1;
        tc_fence_after_sync();
        return got;
      };

#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        const int sb = (NS == 2) ? (j & 1) : 0;
        const uint32_t par = (NS == 2) ? ((j >> 1) & 1) : (j & 1);
        if (!mbar_wait_warp(&bar_s_full[q * NS + sb], par, abort_p)) { ok = false; break; }
        tc_fence_after_sync();
        constexpr int NCH = BN / 32 / kShare, kKeys = BN / kShare;
        const uint32_t s_tile = tmem_base + lane_addr + Cfg::kTmS + (q * NS + sb) * BN;
        const uint32_t s_addr = s_tile + share * kKeys;
        const int n0 = (j0 + t_first + j) * BN + share * kKeys;
        const bool masked = n0 < full_lo_q || n0 + kKeys > full_hi_q;

        uint32_t r[NCH][32];
#pragma unroll
        for (int c = 0; c < NCH; ++c) tmem_ld32(s_addr + c * 32, r[c]);
        tmem_ld_wait32(r[0]);
#pragma unroll
        for (int c = 1; c < NCH; ++c) reg_fence32(r[c]);
        float mx;
        auto mask_and_max = [&]() {
          if (masked) {
            // One word of bits per 32 keys, and nothing for those that the whole warp sees: beside a compare per key and row,
            // S 16384, documents of 2048, 32/8 heads of 128: no change 347 -> 340 us, cap 525 -> 485, both 606 -> 572.
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
              const int from = lo - (n0 + c * 32);
              const uint32_t seen = low_bits(from + width) & ~low_bits(from);
              if (!__all_sync(0xffffffffu, seen == 0xffffffffu)) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!(seen >> i & 1u)) r[c][i] = __float_as_uint(-INFINITY);
              }
            }
          }
          mx = max32(r[0]);
#pragma unroll
          for (int c = 1; c < NCH; ++c) mx = max_nan(mx, max32(r[c]));
        };
        if constexpr (kKind == 0) {
          mask_and_max();
        } else {
          // Keys all before or all after the warp's queries: the distance is linear in the key, sign * (ahead - key).  (To tell
          // that apart for every 32 keys of a tile costs more than it saves: 77 us for 76, S 4096, 16 heads of 64 with a bias.)
          const int d0 = p.sc.q_pos + m0_q + quarter * 32 - p.sc.k_pos;  // of the warp's first row
          const bool before = n0 + kKeys - 1 <= d0, after = n0 >= d0 + 31;
          const bool linear = !has_bias(kKind) || before || after || slope == 0.f;
          const float sign_slope = before ? slope : after ? -slope : 0.f;
          const uint64_t step = pack_f2(2.f * sign_slope, 2.f * sign_slope);
          const float first = static_cast<float>(n0 - ahead);  // minus the distance of the first key
          auto bias_of = [&](int c, float constant) {
            if (!has_bias(kKind)) return pack_f2(constant, constant);
            const float b0 = fmaf(first + c * 32, sign_slope, constant);
            return pack_f2(b0, b0 + sign_slope);
          };
          auto formula_chunk = [&](int c) {
            transform32<kKind>(r[c], pack_f2(in_scale, in_scale), pack_f2(-2.f * cap_log2, -2.f * cap_log2),
                               bias_of(c, has_cap(kKind) ? cap_log2 : 0.f), step);
          };
          auto formula = [&]() {
#pragma unroll
            for (int c = 0; c < NCH; ++c) formula_chunk(c);
          };
          auto finish = [&]() {
            if (!linear) {
              const float d = static_cast<float>(ahead - n0);
#pragma unroll
              for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  r[c][i] = __float_as_uint(fmaf(-slope, fabsf(d - static_cast<float>(c * 32 + i)), __uint_as_float(r[c][i])));
            }
            mask_and_max();
          };
          if (!has_cap(kKind) || direct > 0) {
            formula();
            finish();
            if (has_cap(kKind)) --direct;
          } else if constexpr (has_cap(kKind)) {
            // The polynomial first; chunks in which some lane left its range (garbage in masked places counts) are done again
            // from the scores, which are still in tensor memory.
            float top[NCH];
            mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
              top[c] = 0.f;
              cap32<kKind>(r[c], tanh_poly, bias_of(c, 0.f), step, top[c]);
              mx = max_nan(mx, max32(r[c]));  // fills the gaps of the arithmetic; good where nothing changes any more
            }
            float most = top[0];
#pragma unroll
            for (int c = 1; c < NCH; ++c) most = max_nan(most, top[c]);
            // (a NaN, of padding or not, tells nothing about the others: the formula again)
            const bool again = __any_sync(0xffffffffu, !(most <= tanh_poly.limit));
            if (again) {
              int count = 0;
#pragma unroll
              for (int c = 0; c < NCH; ++c)
                if (__any_sync(0xffffffffu, !(top[c] <= tanh_poly.limit))) {
                  tmem_ld32(s_addr + c * 32, r[c]);
                  tmem_ld_wait32(r[c]);
                  formula_chunk(c);
                  ++count;
                }
              direct = count >= NCH / 2 ? 8 : 0;  // a tile that left it in many places: the next ones will, too
            }
            if (again || masked || !linear) finish();
          }
        }
        if constexpr (kShare == 2) {
          // The other half's maximum.  Its warp has read what this one left for the last tile once its first part of that P
          // is there; and this half of P may only go over the other's scores once those are read.
          if (j > 0 && !mbar_wait_warp(&bar_p_ready[((j - 1) & 1) * kPvParts + (1 - share) * (kPvParts / 2)], ((j - 1) >> 1) & 1, abort_p)) {
            ok = false;
            break;
          }
          pair_value[share][row] = mx;
          if (!pair_sync()) { ok = false; break; }
          mx = max_nan(mx, pair_value[1 - share][row]);
        }
        const float m_new = max_nan(m_used, kKind == 0 ? mx * scale_log2 : mx);

        // lazy rescale: only when the maximum grew by more than 2^8, or is no number
        bool need;
        if (j == 0 && p.first) {
          m_used = m_new;
          need = false;
        } else {
          need = !(m_new - m_used <= 8.0f);
        }
        if (__any_sync(0xffffffffu, need)) {
          const float alpha = need ? fast_exp2(m_used - m_new) : 1.0f;
          if (need) m_used = m_new + (m_new - m_new);
          l_sum *= alpha;
          // With one score buffer the arrival on bar_s_full that let this iteration start was committed after
          // O += P_{j-1} V_{j-1} was issued, so that product has retired; with two buffers it has its own barrier.
          if (NS == 2 && j > 0) {
            if (!mbar_wait_warp(&bar_pv_done[q], (j - 1) & 1, abort_p)) { ok = false; break; }
            tc_fence_after_sync();
          }
#pragma unroll 1
          for (int c = 2 * o_first; c < 2 * o_end; ++c) {
            uint32_t o16[16];
            tmem_ld16(o_addr + c * 16, o16);
            tmem_ld_wait16(o16);
#pragma unroll
            for (int i = 0; i < 16; ++i) o16[i] = __float_as_uint(__uint_as_float(o16[i]) * alpha);
            tmem_st16(o_addr + c * 16, o16);
          }
          tmem_st_wait();
          if (kShare == 2 && !pair_sync()) { ok = false; break; }  // all of O, before either's P is added to it
        }

        // P = exp2(z - m_used), packed to 16 bit over the start of S (rounded for the product, as in the plain hop; the sum
        // is taken before).  The polynomial gives a masked key 2^-125 where exp2 gives 0: beside a real key nothing.
        const uint64_t scale2 = pack_f2(scale_log2, scale_log2);
        const uint64_t negm2 = pack_f2(-m_used, -m_used);
        uint64_t lp2[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          uint32_t u[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t s2 = pack_u2(r[c][2 * i], r[c][2 * i + 1]);
            const uint64_t x2 = kKind == 0 ? fma2(s2, scale2, negm2) : add2(s2, negm2);
            uint64_t p2;
            float p0, p1;
            if (kPolyEvery > 0 && (i % (kPolyEvery > 0 ? kPolyEvery : 1)) == kPolyEvery - 1) {
              p2 = exp2_poly(x2);
              unpack_f2(p2, p0, p1);
            } else {
              float x0, x1;
              unpack_f2(x2, x0, x1);
              p0 = fast_exp2(x0);
              p1 = fast_exp2(x1);
              p2 = pack_f2(p0, p1);
            }
            lp2[i & 1] = add2(lp2[i & 1], p2);
            u[i] = Pack2<T>::pack(p0, p1);
          }
          if (c > 0 && c % kPartChunks == 0) {
            // the previous part of P has landed: the issuer may start O += P V on them
            tmem_st_wait();
            tc_fence_before_sync();
            mbar_arrive(&bar_p_ready[(q * NS + sb) * kPvParts + (share * NCH + c) / kPartChunks - 1]);
          }
          tmem_st16(s_tile + (share * NCH + c) * 16, u);
        }
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive(&bar_p_ready[(q * NS + sb) * kPvParts + (share + 1) * kPvParts / kShare - 1]);
        {
          float a0, a1, b0, b1;
          unpack_f2(lp2[0], a0, a1);
          unpack_f2(lp2[1], b0, b1);
          l_sum += (a0 + a1) + (b0 + b1);
        }
      }

      // ---- epilogue: wait for the last PV, then spill state or write the result ----
      // With two score buffers the last scores only prove that O += P_{n-3} V_{n-3} has retired: a wait for the parity of
      // the last product alone would also be satisfied by the phase before the one of tile n-2.
      if (NS == 2 && ok && n > 1) ok = mbar_wait_warp(&bar_pv_done[q], (n - 2) & 1, abort_p);
      if (ok && n > 0) ok = mbar_wait_warp(&bar_pv_done[q], (NS == 2) ? ((n - 1) & 1) : 0, abort_p);
      if (kShare == 2 && ok) {  // every maximum has been read: the products of all P are done
        pair_value[share][row] = l_sum;
        ok = pair_sync();
        l_sum = pair_value[0][row] + pair_value[kShare - 1][row];
      }
      if (ok) {
        tc_fence_after_sync();
        l_sum += m_used - m_used;  // nothing, or NaN
        if (p.last) {
          const bool empty = m_used == kNoKey;
          const float inv = 1.0f / l_sum;
          const bool row_ok = row_g < p.S;
          T* orow = reinterpret_cast<T*>(p.out) + ((static_cast<size_t>(b) * p.S + row_g) * p.Hq + h) * p.D;
#pragma unroll 1
          for (int c = o_first; c < o_end; ++c) {
            uint32_t r[32];
            tmem_ld32(o_addr + c * 32, r);
            tmem_ld_wait32(r);
            if (row_ok) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (c * 32 + k * 8 < p.D) {
                  uint4 w;
                  w.x = Pack2<T>::pack(__uint_as_float(r[8 * k + 0]) * inv, __uint_as_float(r[8 * k + 1]) * inv);
                  w.y = Pack2<T>::pack(__uint_as_float(r[8 * k + 2]) * inv, __uint_as_float(r[8 * k + 3]) * inv);
                  w.z = Pack2<T>::pack(__uint_as_float(r[8 * k + 4]) * inv, __uint_as_float(r[8 * k + 5]) * inv);
                  w.w = Pack2<T>::pack(__uint_as_float(r[8 * k + 6]) * inv, __uint_as_float(r[8 * k + 7]) * inv);
                  if (empty) w = make_uint4(0, 0, 0, 0);
                  *reinterpret_cast<uint4*>(orow + c * 32 + k * 8) = w;
                }
              }
            }
          }
          if (row_ok && share == 0) p.lse[ml_idx] = empty ? -INFINITY : (m_used + log2f(l_sum)) * 0.6931471805599453f;
        } else {
#pragma unroll 1
          for (int c = o_first; c < o_end; ++c) {
            uint32_t r[32];
            tmem_ld32(o_addr + c * 32, r);
            tmem_ld_wait32(r);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              float4 v;
              v.x = __uint_as_float(r[4 * k + 0]);
              v.y = __uint_as_float(r[4 * k + 1]);
              v.z = __uint_as_float(r[4 * k + 2]);
              v.w = __uint_as_float(r[4 * k + 3]);
              *reinterpret_cast<float4*>(acc_tile + ((c * 8 + k) * 128 + row) * 4) = v;
            }
          }
          if (share == 0) {
            p.m[ml_idx] = m_used;
            p.l[ml_idx] = l_sum;
          }
        }
      }
    }
    __syncwarp();
  }

  // ---- teardown: every role arrives here, also after an abort ----
  tc_fence_before_sync();
  __syncthreads();
  if (abort_flag) {
    // Give copies that are still in flight time to land before the CTA's shared memory is released.
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    if (tid == 0) atomicExch(p.status, kStatusWaitTimeout);
  }
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

constexpr int kMaxSplit = 16;

// The states that the CTAs of a split left, into out and lse.  One block per tile of 128 rows: thread = row, and half of the
// head dim.  A few megabytes; bound by latency.
template <typename T>
__global__ void __launch_bounds__(256) join_splits_kernel(const ScoredFwdParams p) {
  pdl_wait();
  const int tile = blockIdx.x % p.nT, h = blockIdx.x / p.nT % p.Hq, b = blockIdx.x / p.nT / p.Hq;
  const int row = threadIdx.x & 127, row_g = tile * 128 + row;
  if (row_g >= p.S) return;
  const size_t bh = static_cast<size_t>(b) * p.Hq + h, ml_idx = bh * p.Spad + row_g;
  float weight[kMaxSplit], top = kNoKey, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxSplit; ++i)
    if (i < p.nsplit) top = max_nan(top, p.m[ml_idx + i * p.ml_split]);
#pragma unroll
  for (int i = 0; i < kMaxSplit; ++i)
    if (i < p.nsplit) {
      const float m = p.m[ml_idx + i * p.ml_split];
      weight[i] = m == kNoKey ? 0.f : fast_exp2(m - top);  // what stands beside that maximum is no sum
      if (weight[i] != 0.f) sum = fmaf(weight[i], p.l[ml_idx + i * p.ml_split], sum);
    }
  const bool empty = top == kNoKey;
  const float inv = 1.0f / sum;
  const int DP = static_cast<int>(p.acc_split / p.ml_split), half = (p.D / 8 + 1) / 2 * 8;
  const float* acc = p.acc + (bh * p.nT + tile) * (static_cast<size_t>(DP) * 128) + row * 4;
  T* orow = static_cast<T*>(p.out) + ((static_cast<size_t>(b) * p.S + row_g) * p.Hq + h) * p.D;
  const int begin = threadIdx.x < 128 ? 0 : half, end = threadIdx.x < 128 ? half : p.D;
  for (int d = begin; d < end; d += 8) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
#pragma unroll
    for (int i = 0; i < kMaxSplit; ++i)
      if (i < p.nsplit && weight[i] != 0.f) {
        const float* from = acc + i * p.acc_split + d / 4 * 512;
        const float4 u = *reinterpret_cast<const float4*>(from), w = *reinterpret_cast<const float4*>(from + 512);
        const float f = weight[i];
        x = make_float4(fmaf(u.x, f, x.x), fmaf(u.y, f, x.y), fmaf(u.z, f, x.z), fmaf(u.w, f, x.w));
        y = make_float4(fmaf(w.x, f, y.x), fmaf(w.y, f, y.y), fmaf(w.z, f, y.z), fmaf(w.w, f, y.w));
      }
    uint4 r = make_uint4(Pack2<T>::pack(x.x * inv, x.y * inv), Pack2<T>::pack(x.z * inv, x.w * inv),
                         Pack2<T>::pack(y.x * inv, y.y * inv), Pack2<T>::pack(y.z * inv, y.w * inv));
    if (empty) r = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(orow + d) = r;
  }
  if (threadIdx.x < 128) p.lse[ml_idx] = empty ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// Few heads: the longest row of tiles is as long as the pass, and most SMs wait.  Its key tiles are shared by so many CTAs that
// it is no longer than the mean load of an SM, where that pays for the second launch and the states in between (some kJoin
// tiles).  `typical_keys` (0: all) is how far a query may see: shorter rows need no split.  Measured, causal, us in one launch
// and split (CTAs per row): S 2048, 1 head of 64 33 -> 23 (3); 8 heads of 128 35 -> 34, with a cap 62 -> 41 (3); S 4096, 4 heads
// of 128 58 -> 39 (3); 8 heads 60 -> 52 (2); S 8192, 4 heads 109 -> 74 (2); S 16384, 1 head 204 -> 76 (4), 4 heads 217 (no
// split).  At S 1536, 4 heads, the two are even (27).
static int fwd_split(int B, int S, int Hq, int D, int causal, int typical_keys) {
  constexpr int kSMs = 148;
  constexpr double kCta = 3.0, kJoin = 5.0;  // in key tiles (1.6 us): start and end of a CTA; the join
  const int pair = padded_head_dim(D) == 256 ? 1 : 2, nT = ceil_div(S, 128);
  const double ctas = static_cast<double>(ceil_div(nT, pair)) * Hq * B;
  double longest = nT;
  if (typical_keys > 0 && typical_keys < S) longest = ceil_div(typical_keys, 128) + 1;
  const double mean = causal ? 0.5 * longest : longest;
  int best = 1;
  double best_t = 0;
  for (int n = 1; n <= kMaxSplit && (n == 1 || longest >= 4 * n); ++n) {
    const double load = ctas * (mean + n * kCta) / kSMs, chain = longest / n + kCta;
    const double t = (load > chain ? load : chain) + (n > 1 ? kJoin : 0);
    if (n == 1 || t < 0.9 * best_t) {
      best = n;
      best_t = t;
    }
  }
  return best;
}
// fp32 elements of one state: O, maxima and sums.
static size_t state_elems(int B, int S, int Hq, int D) {
  return static_cast<size_t>(B) * Hq * round_up(S, 128) * (padded_head_dim(D) + 2);
}

template <int DP, int BN, int NQ, int NS, typename T, int kKind>
static int launch_scored_fwd(const void* q, const void* k, const void* v, const ScoredFwdParams& prm, int dtype,
                             cudaStream_t stream) {
  using Cfg = FwdCfg<DP, BN, NQ, NS>;
  CUtensorMap tq, tk, tv;
  int rc;
  if ((rc = make_tmap_bshd(&tq, q, dtype, prm.B, prm.S, prm.Hq, prm.D, 128)) != RFA_OK) return rc;
  if ((rc = make_tmap_bshd(&tk, k, dtype, prm.B, prm.S, prm.Hkv, prm.D, BN)) != RFA_OK) return rc;
  if ((rc = make_tmap_bshd(&tv, v, dtype, prm.B, prm.S, prm.Hkv, prm.D, BN)) != RFA_OK) return rc;
  auto kern = scored_fwd_kernel<DP, BN, NQ, NS, T, kKind>;
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) { cudaGetLastError(); return RFA_ERR_CUDA; }
  if (!attr_done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
    if (e != cudaSuccess) { cudaGetLastError(); return RFA_ERR_CUDA; }
    if (NQ == 2) {
      // A raise that the launch's pool (threads x registers per thread) cannot satisfy would wait forever: a build whose
      // register count does not cover the allowances is refused.
      cudaFuncAttributes fa;
      e = cudaFuncGetAttributes(&fa, kern);
      if (e != cudaSuccess) { cudaGetLastError(); return RFA_ERR_CUDA; }
      if (fa.numRegs * fwd_threads(NQ, kKind) < Cfg::kPoolRegs) return RFA_ERR_UNSUPPORTED;
    }
    attr_done[dev] = true;
  }
  const unsigned grid = static_cast<unsigned>((prm.nT + NQ - 1) / NQ) * prm.Hq * prm.B * prm.nsplit;
  return launch_chained(kern, grid, fwd_threads(NQ, kKind), Cfg::kSmemBytes, stream, tq, tk, tv, prm);
}

template <typename T, int kKind>
static int dispatch_scored_fwd(const void* q, const void* k, const void* v, const ScoredFwdParams& prm, int dtype,
                               cudaStream_t stream) {
  switch (padded_head_dim(prm.D)) {
    case 64: return launch_scored_fwd<64, 128, 2, 1, T, kKind>(q, k, v, prm, dtype, stream);
    case 128: return launch_scored_fwd<128, 128, 2, 1, T, kKind>(q, k, v, prm, dtype, stream);
    case 256: return launch_scored_fwd<256, 128, 1, 2, T, kKind>(q, k, v, prm, dtype, stream);
    default: return RFA_ERR_UNSUPPORTED;
  }
}

template <typename T>
static int dispatch_scored_kind(const void* q, const void* k, const void* v, const ScoredFwdParams& prm, int dtype,
                                cudaStream_t stream) {
  switch (score_kind(prm.sc)) {
    case 0: return dispatch_scored_fwd<T, 0>(q, k, v, prm, dtype, stream);
    case 1: return dispatch_scored_fwd<T, 1>(q, k, v, prm, dtype, stream);
    case 2: return dispatch_scored_fwd<T, 2>(q, k, v, prm, dtype, stream);
    default: return dispatch_scored_fwd<T, 3>(q, k, v, prm, dtype, stream);
  }
}

}  // namespace rfa

extern "C" int rfa_scored_fwd_hop(const void* q, const void* k, const void* v, float* acc, float* m, float* l, void* out,
                                  float* lse, int B, int S, int Hq, int Hkv, int D, int dtype, const rfa_score_args* args,
                                  int first, int last, int* status, void* stream) {
  using namespace rfa;
  if (!q || !k || !v || !status) return RFA_ERR_INVALID_ARG;
  if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0) return RFA_ERR_INVALID_ARG;
  if (!(first && last) && (!acc || !m || !l)) return RFA_ERR_INVALID_ARG;
  if (last && (!out || !lse)) return RFA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(acc) & 15u) || (reinterpret_cast<uintptr_t>(out) & 15u)) return RFA_ERR_INVALID_ARG;
  if (padded_head_dim(D) == 0) return RFA_ERR_UNSUPPORTED;
  if (dtype != RFA_DTYPE_BF16 && dtype != RFA_DTYPE_FP16) return RFA_ERR_UNSUPPORTED;
  ScoredFwdParams prm;
  const int rc = make_score_params(args, B, S, &prm.sc);
  if (rc != RFA_OK) return rc;
  prm.acc = acc;
  prm.m = m;
  prm.l = l;
  prm.out = out;
  prm.lse = lse;
  prm.B = B;
  prm.S = S;
  prm.Hq = Hq;
  prm.Hkv = Hkv;
  prm.D = D;
  prm.Spad = round_up(S, 128);
  prm.nT = prm.Spad / 128;
  prm.first = first ? 1 : 0;
  prm.last = last ? 1 : 0;
  prm.nsplit = 1;
  prm.acc_split = prm.ml_split = 0;
  prm.status = status;
  if (static_cast<long long>(prm.nT) * Hq * B > INT_MAX) return RFA_ERR_TOO_LARGE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == RFA_DTYPE_BF16) return dispatch_scored_kind<__nv_bfloat16>(q, k, v, prm, dtype, s);
  return dispatch_scored_kind<__half>(q, k, v, prm, dtype, s);
}

extern "C" size_t rfa_scored_fwd_scratch_elems(int B, int S, int Hq, int D, int causal, int typical_keys) {
  using namespace rfa;
  if (B <= 0 || S <= 0 || Hq <= 0 || padded_head_dim(D) == 0) return 0;
  const int n = fwd_split(B, S, Hq, D, causal, typical_keys);
  return n > 1 ? n * state_elems(B, S, Hq, D) : 0;
}

extern "C" int rfa_scored_fwd_local(const void* q, const void* k, const void* v, void* out, float* lse, float* scratch, int B,
                                    int S, int Hq, int Hkv, int D, int dtype, const rfa_score_args* args, int typical_keys,
                                    int* status, void* stream) {
  using namespace rfa;
  if (!args) return RFA_ERR_INVALID_ARG;
  if (scratch == nullptr || B <= 0 || S <= 0 || Hq <= 0 || padded_head_dim(D) == 0)
    return rfa_scored_fwd_hop(q, k, v, nullptr, nullptr, nullptr, out, lse, B, S, Hq, Hkv, D, dtype, args, 1, 1, status, stream);
  const int n = fwd_split(B, S, Hq, D, args->causal, typical_keys);
  if (n == 1)
    return rfa_scored_fwd_hop(q, k, v, nullptr, nullptr, nullptr, out, lse, B, S, Hq, Hkv, D, dtype, args, 1, 1, status, stream);
  if (!q || !k || !v || !status || !out || !lse || Hkv <= 0 || Hq % Hkv != 0) return RFA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(scratch) & 15u) || (reinterpret_cast<uintptr_t>(out) & 15u)) return RFA_ERR_INVALID_ARG;
  if (dtype != RFA_DTYPE_BF16 && dtype != RFA_DTYPE_FP16) return RFA_ERR_UNSUPPORTED;
  ScoredFwdParams prm;
  int rc = make_score_params(args, B, S, &prm.sc);
  if (rc != RFA_OK) return rc;
  const size_t acc = static_cast<size_t>(B) * Hq * round_up(S, 128) * padded_head_dim(D);
  const size_t ml = static_cast<size_t>(B) * Hq * round_up(S, 128);
  prm.acc = scratch;
  prm.m = scratch + n * acc;
  prm.l = prm.m + n * ml;
  prm.out = out;
  prm.lse = lse;
  prm.B = B;
  prm.S = S;
  prm.Hq = Hq;
  prm.Hkv = Hkv;
  prm.D = D;
  prm.Spad = round_up(S, 128);
  prm.nT = prm.Spad / 128;
  prm.first = 1;
  prm.last = 0;
  prm.nsplit = n;
  prm.acc_split = acc;
  prm.ml_split = ml;
  prm.status = status;
  if (static_cast<long long>(prm.nT) * Hq * B * n > INT_MAX) return RFA_ERR_TOO_LARGE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = dtype == RFA_DTYPE_BF16 ? dispatch_scored_kind<__nv_bfloat16>(q, k, v, prm, dtype, s)
                               : dispatch_scored_kind<__half>(q, k, v, prm, dtype, s);
  if (rc != RFA_OK) return rc;
  const unsigned grid = static_cast<unsigned>(prm.nT) * Hq * B;
  return dtype == RFA_DTYPE_BF16 ? launch_chained(join_splits_kernel<__nv_bfloat16>, grid, 256, 0, s, prm)
                                 : launch_chained(join_splits_kernel<__half>, grid, 256, 0, s, prm);
}
