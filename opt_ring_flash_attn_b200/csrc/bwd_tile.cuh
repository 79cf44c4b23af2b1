// Tile configuration, the pause of the vector reductions and the wait of the ordered mode, which the backward kernels share.
#pragma once

#include "common.h"
#include "tc05.cuh"

namespace rfa {

// Pause (ns) a reduction warp takes after each vector reduction (head dim 256; up to 128 the copy engine reduces).  An SM
// can push 32 B per clock towards the L2; unpaced, the eight reduction warps keep the load/store queue full of reductions
// and every shared-memory or tensor-memory access of the elementwise warps waits behind them.  The optimum is sharp (150 ns
// behaves like 200; 0 / 20 / 50 / 100 / 150 / 200 ns, hop alone, us: B 2, S 4096, 16 heads of 256, full
// 2297 / 2197 / 2177 / 1990 / 2288 / 2288; 16 heads of 160, diagonal 1143 / 1121 / 1121 / 1085 / 1241 / 1240, full 1980 /
// 1934 / 1920 / 1790 / 2250 / 2250; S 700, 16 heads of 256, full 73.8 / 71.7 / 71.7 / 69.7 / 75.8 / 75.8).  The ordered mode
// never pauses: the next K/V tile is waiting for the addition (head dims up to 128, diagonal / full, paced and not: S 2048,
// 16/2 heads of 128 177 / 226 -> 164 / 208 us; S 4096, 16 heads of 64 323 / 973 -> 238 / 744; S 8192, 32/8 heads
// 2.27 / 4.25 -> 2.20 / 3.93 ms).
constexpr unsigned kRedSleepNs = 100;

// Bounded wait of one lane until a counter in global memory has reached `target`; the whole warp gets the answer
// (false: the CTA is aborting).
__device__ __forceinline__ bool wait_count(const int* sem, int target, bool waiter, volatile int* abort_p) {
  bool got = true;
  if (waiter) {
    const unsigned long long since = global_timer_ns();
    uint32_t spins = 0;
    while (ld_acquire_gpu(sem) < target) {
      if (((++spins) & 0x3fu) == 0) {
        if (*abort_p) { got = false; break; }
        if (global_timer_ns() - since > kWaitLimitNs) { *abort_p = 1; got = false; break; }
      }
      __nanosleep(64);
    }
  }
  return __all_sync(0xffffffffu, got);
}

template <int DP, int DH, int BQ, int NSQ, int NSO>
struct BwdCfg {
  static constexpr int kPanels = DP / 64;
  static constexpr int kHalves = DP / DH;
  // Head dim 256: K is the A operand of S^T from tensor memory (64 KB, 128 columns), so that shared memory only holds the
  // half of its columns that dQ^T needs and there is room for a second Q stage.
  static constexpr bool kKTmem = (DP == 256);
  static constexpr int kKSmemBytes = 128 * (kKTmem ? DH : DP) * 2;
  static constexpr int kVBytes = 128 * DP * 2;
  static constexpr int kQBytes = BQ * DP * 2;
  static constexpr int kDSBytes = 128 * BQ * 2;
  static constexpr int kStatBytes = 2 * BQ * 4;
  static constexpr int kOffK = 0;
  static constexpr int kOffV = kKSmemBytes;
  static constexpr int kOffQ = kOffV + kVBytes;
  static constexpr int kOffDO = kOffQ + NSQ * kQBytes;
  static constexpr int kOffDS = kOffDO + NSO * kQBytes;
  static constexpr int kOffStat = kOffDS + kDSBytes;
  // dQ^T staging for bulk reductions (head dims up to 128): per reduction warp two buffers of kDQGroups row groups.  Vector
  // reductions from registers share the load/store queue with every shared-memory access and special-function instruction
  // of the elementwise warps; the copy engine does not.  S 4096, 16 heads of 64, full block: vector reductions 350 us
  // (paced 100 ns) / 300 us (20 ns), bulk reductions 291.  At head dim 128 the 32 KB come from the second dO stage (dO of
  // the next tile is wanted after dQ^T has been drained, some 2500 cycles after dV released the slot).  Steady state, which
  // is power-limited at 950 W (S 8192, 32/8 heads, diagonal / full): 1.62 / 3.25 ms with paced vector reductions,
  // 1.51 / 2.93 with bulk ones; 1 KB instead of 2 KB per reduction costs 4 %.  Head dim 256 has 17 KB left, enough for
  // buffers of 1 KB; it keeps vector reductions, bulk ones have not been measured there.
  static constexpr bool kStageDQ = (DP <= 128);
  static constexpr int kDQGroups = (DP == 64) ? BQ / 8 : 4;      // row groups (of 4 query rows) per bulk reduction
  static constexpr int kDQBufBytes = kDQGroups * 512;            // one warp: 32 lanes x 16 bytes per row group
  static constexpr int kDQWarps = 2 * (DP < 128 ? DP : 128) / 32;
  static constexpr int kOffDQ = (kOffStat + NSQ * kStatBytes + 127) / 128 * 128;
  static constexpr int kSmemUsed = kOffDQ + (kStageDQ ? kDQWarps * 2 * kDQBufBytes : 0);
  // Pad to more than half of the SM's shared memory so that two CTAs never share an SM
  // (each CTA allocates the whole tensor memory).
  static constexpr int kSmemBytes = kSmemUsed < 120 * 1024 ? 120 * 1024 : kSmemUsed;
  static constexpr int kThreads = 640;
  static constexpr int kTmS = 0;
  static constexpr int kTmDP = BQ;
  static constexpr int kTmDV = 2 * BQ;
  static constexpr int kTmDK = 2 * BQ + DH;
  // dQ^T has columns of its own where tensor memory has room for them (head dim 64), so that the next dP^T need not wait
  // until it is drained; otherwise it takes over those of dP^T.
  static constexpr bool kOwnDQ = (DP == 64);
  static constexpr int kTmDQ = kOwnDQ ? 2 * BQ + 2 * DH : kTmDP;
  static constexpr int kTmK = 2 * BQ + 2 * DH;
  static_assert(2 * BQ + 2 * DH + (kOwnDQ ? BQ : 0) + (kKTmem ? DP / 2 : 0) <= 512, "tensor memory over budget");
  static_assert(kSmemBytes <= 232448 - 1024, "shared memory over budget");
};

}  // namespace rfa
