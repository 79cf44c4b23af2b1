// Tile configuration, product issue and slot bookkeeping that the forward kernels share.
#pragma once

#include "common.h"
#include "tc05.cuh"

namespace rfa {

// Every n-th pair of exponentials of the softmax on the FMA pipe (a quartic) instead of the special-function unit, which
// needs as many cycles per K/V tile as the tensor pipe does; 0 = none.  Diagonal / full block: S 8192, 32/8 heads of 128:
// every 2nd 553 / 1044 us, 3rd 502 / 953, 4th 510 / 976, none 518 / 991; S 4096, 16 heads of 64: 59.5 / 115.5, 55.5 / 105.3,
// 55.8 / 106.4, 56.2 / 107.6.  Head dim 256 has one softmax warpgroup to two tiles of tensor work: every 2nd 316 / 574 us,
// 4th 305 / 559, none 304 / 556.
constexpr int kFwdPolyEvery = 3;

template <int DP, int BN, int NQ, int NS>
struct FwdCfg {
  static constexpr int kBM = 128;
  static constexpr int kPanels = DP / 64;
  static constexpr int kQBytes = kBM * DP * 2;
  static constexpr int kPieces = (NS == 2) ? DP / 128 : 1;  // a K/V tile arrives in as many slots
  static constexpr int kKVBytes = BN * DP * 2 / kPieces;
  static constexpr int kSlots = (DP == 64) ? 8 : (NS == 2) ? 5 : 4;
  static constexpr int kSmemTiles = NQ * kQBytes + kSlots * kKVBytes;
  static constexpr int kSmemBytes = kSmemTiles + 1024;  // slack for 1024-byte alignment
  static constexpr int kThreads = 128 + NQ * 128;
  static constexpr int kServiceRegs = 72, kSoftmaxRegs = 216;  // per thread, two-tile variants
  static constexpr int kPoolRegs = 128 * kServiceRegs + NQ * 128 * kSoftmaxRegs;
  static_assert(NQ == 1 || kPoolRegs <= kThreads * 168, "register allowances exceed what the launch allocates");
  static constexpr int kTmO = 0;
  static constexpr int kTmS = NQ * DP;
  static_assert(kTmS + NQ * NS * BN <= 512, "tensor memory over budget");
  static_assert(kSmemBytes >= 120 * 1024, "one CTA per SM is assumed (whole TMEM is allocated)");
};

// S[128 x BN] = Q[128 x DP] * K[BN x DP]^T, both operands K-major.
template <int DP, int BN>
__device__ __forceinline__ void issue_qk(uint32_t s_tmem, uint32_t q_smem, uint32_t k_smem, uint32_t idesc,
                                         uint32_t el, bool accumulate = false) {
  // q_smem / k_smem are descriptor low words of the tile bases; offsets are in 16-byte units
  static_for<0, DP / 16>([&](auto ks_) {
    constexpr int ks = decltype(ks_)::value;
    mma_ss_off_e<(((ks / 4) * (128 * 128) + (ks % 4) * 32) / 16), (((ks / 4) * (BN * 128) + (ks % 4) * 32) / 16)>(
        s_tmem, q_smem, k_smem, idesc, (accumulate || ks > 0) ? 1u : 0u, el);
  });
}

// O[128 x DP] (+)= P[128 x BN] * V[BN x DP] over the K-steps [KS0, KS1) of 16 keys each; P in tensor memory,
// V MN-major.  The product of one K/V tile is issued in kPvParts pieces so that the first keys of P are consumed
// while the softmax warps still exponentiate the rest of the row.
template <int DP, int BN, int KS0, int KS1>
__device__ __forceinline__ void issue_pv(uint32_t o_tmem, uint32_t p_tmem, uint32_t v_smem, uint32_t idesc,
                                         bool accumulate, uint32_t el) {
  static_for<KS0, KS1>([&](auto ks_) {
    constexpr int ks = decltype(ks_)::value;
    mma_ts_off_e<(ks * 8), (ks * 128)>(o_tmem, p_tmem, v_smem, idesc, (accumulate || ks > KS0) ? 1u : 0u, el);
  });
}

// Position in the ring of K/V slots, advanced one slot at a time (for a count that is no power of two).
template <int kSlots>
struct SlotWalk {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == kSlots) {
      slot = 0;
      phase ^= 1;
    }
  }
};

}  // namespace rfa
