// What the kernels of attention with modified scores share: the parameters, the layout of a mask buffer and the scores.
//
// Documents, the causal rule and prefixes leave every query an interval of keys and every key an interval of queries, so a
// mask is two pairs of int32 per position instead of S x S truth values: a thread that owns a query row (forward) or a key
// row (backward) holds its interval in two registers, and the hull of a tile's intervals gives the range of tiles it meets
// and which of them need no test.
#pragma once

#include <limits.h>

#include "common.h"
#include "tc05.cuh"

namespace rfa {

constexpr float kLog2e = 1.4426950408889634f;
// Largest cap: cap * tanh comes out of cap - 2 cap / (exp + 1) with an error of up to 9 * 2^-24 of the cap (exp2 2^-22, reciprocal
// 2^-23, three roundings), or of a polynomial with 3.5e-7 (scored_fwd.cu): 5e-4 of a weight here, about what its rounding to fp16 is.
constexpr float kMaxCap = 1000.f;
// Running maximum of a row that has seen no key: finite, so that exp2(-inf - kNoKey) is 0 and not NaN, and far below any
// score in log2 units that could matter, so that the first real one rescales what was there by 0.
constexpr float kNoKey = -1e30f;

// Mask buffer (int32): per position of the whole sequence the interval of keys a query sees (q_lo, q_hi) and the interval
// of queries that see a key (k_lo, k_hi), [B][shards * S] each, empty as (0, 0); per tile of 128 rows of a shard the hull
// (smallest lo, largest lo, smallest hi, largest hi) of either, [B][shards][nT] int4, with largest lo = INT_MAX where a row
// is empty; per shard the (b, tile) pairs by falling work, for query tiles, pairs of query tiles and key tiles; per batch
// row the positions [begin, end) that are no padding.
struct MaskView {
  const int* q_lo;
  const int* q_hi;
  const int* k_lo;
  const int* k_hi;
  const int4* q_tile;
  const int4* k_tile;
  const int* order_q;   // [shards][B * nT]
  const int* order_q2;  // [shards][B * ceil(nT / 2)]
  const int* order_k;   // [shards][B * nT]
  const int* real;      // [B][2]
};

__host__ __device__ inline size_t mask_rows(int B, int S, int shards) {  // of one interval array, a multiple of 4
  return (static_cast<size_t>(B) * S * shards + 3) / 4 * 4;
}
__host__ __device__ inline size_t mask_elems(int B, int S, int shards) {
  const size_t nT = (static_cast<size_t>(S) + 127) / 128, tiles = static_cast<size_t>(B) * shards * nT;
  return 4 * mask_rows(B, S, shards) + 8 * tiles + 2 * tiles + static_cast<size_t>(B) * shards * ((nT + 1) / 2) +
         2 * static_cast<size_t>(B);
}
__host__ __device__ inline MaskView mask_view(const int* base, int B, int S, int shards) {
  const size_t n = mask_rows(B, S, shards), nT = (static_cast<size_t>(S) + 127) / 128;
  const size_t tiles = static_cast<size_t>(B) * shards * nT, pairs = static_cast<size_t>(B) * shards * ((nT + 1) / 2);
  MaskView v;
  v.q_lo = base;
  v.q_hi = base + n;
  v.k_lo = base + 2 * n;
  v.k_hi = base + 3 * n;
  v.q_tile = reinterpret_cast<const int4*>(base + 4 * n);
  v.k_tile = v.q_tile + tiles;
  v.order_q = base + 4 * n + 8 * tiles;
  v.order_q2 = v.order_q + tiles;
  v.order_k = v.order_q2 + pairs;
  v.real = v.order_k + tiles;
  return v;
}

// The scores of one launch.  Positions are those of the whole sequence; tiles and rows are those of the block.
struct ScoreParams {
  float scale, cap;
  const float* slopes;
  int slopes_per_batch;
  int causal;
  int has_mask;
  int q_pos, k_pos;  // of the first query and key row of the block
  int len;           // of the whole sequence
  MaskView mask;
};

// What the kernels multiply raw scores with has to be a number: scale * log2(e) and, for the tanh, 2 * scale * log2(e) / cap.
inline bool scores_fit(float scale, float cap) {
  return cap <= kMaxCap && 1.45 * scale <= 3.4e38 && (!(cap > 0.f) || 2.9 * scale <= 3.4e38 * cap);
}

// Checks and unpacks the arguments of an entry point.
inline int make_score_params(const rfa_score_args* a, int B, int S, ScoreParams* out) {
  if (!a || !(a->softmax_scale > 0.f) || !(a->softcap >= 0.f)) return RFA_ERR_INVALID_ARG;
  if (!scores_fit(a->softmax_scale, a->softcap)) return RFA_ERR_INVALID_ARG;
  if (a->shards < 1 || a->q_shard < 0 || a->q_shard >= a->shards || a->k_shard < 0 || a->k_shard >= a->shards)
    return RFA_ERR_INVALID_ARG;
  if (static_cast<long long>(S) * a->shards > INT_MAX / 2) return RFA_ERR_TOO_LARGE;
  if (reinterpret_cast<uintptr_t>(a->mask) & 15u) return RFA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(a->slopes) & 3u) return RFA_ERR_INVALID_ARG;
  out->scale = a->softmax_scale;
  out->cap = a->softcap;
  out->slopes = a->slopes;
  out->slopes_per_batch = a->slopes_per_batch;
  out->causal = a->causal;
  out->has_mask = a->mask != nullptr;
  out->q_pos = a->q_shard * S;
  out->k_pos = a->k_shard * S;
  out->len = S * a->shards;
  out->mask = MaskView{};
  if (a->mask) {
    MaskView v = mask_view(a->mask, B, S, a->shards);
    const int nT = ceil_div(S, 128);
    v.q_tile += static_cast<size_t>(a->q_shard) * nT;  // the batch stride stays shards * nT
    v.k_tile += static_cast<size_t>(a->k_shard) * nT;
    v.order_q += static_cast<size_t>(a->q_shard) * B * nT;
    v.order_q2 += static_cast<size_t>(a->q_shard) * B * ((nT + 1) / 2);
    v.order_k += static_cast<size_t>(a->k_shard) * B * nT;
    out->mask = v;
  }
  return RFA_OK;
}

// Kind of scores a kernel is instantiated for: 0 as they are, 1 with a distance bias, 2 capped, 3 both.  Separate
// instantiations, because a bias costs a tile two operations per pair of scores and a cap several.
inline int score_kind(const ScoreParams& s) { return (s.cap > 0.f ? 2 : 0) + (s.slopes ? 1 : 0); }
__host__ __device__ constexpr bool has_cap(int kind) { return kind >= 2; }
__host__ __device__ constexpr bool has_bias(int kind) { return kind % 2 == 1; }

__device__ __forceinline__ float slope_log2(const ScoreParams& s, int b, int Hq, int h) {
  return s.slopes ? __ldg(s.slopes + (s.slopes_per_batch ? static_cast<size_t>(b) * Hq : 0) + h) * kLog2e : 0.f;
}

__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Hull of the intervals of a tile, in rows of the other block (see MaskView), without a mask: the causal rule.
__device__ __forceinline__ int4 query_hull(const ScoreParams& s, int b, int nT, int tile, int S) {
  if (s.has_mask) {
    const int shards = s.len / S;
    return __ldg(s.mask.q_tile + static_cast<size_t>(b) * shards * nT + tile);
  }
  if (!s.causal) return make_int4(0, 0, s.len, s.len);
  const int first = s.q_pos + tile * 128;
  return make_int4(0, 0, first + 1, s.q_pos + min(tile * 128 + 128, S));
}
__device__ __forceinline__ int4 key_hull(const ScoreParams& s, int b, int nT, int tile, int S) {
  if (s.has_mask) {
    const int shards = s.len / S;
    return __ldg(s.mask.k_tile + static_cast<size_t>(b) * shards * nT + tile);
  }
  if (!s.causal) return make_int4(0, 0, s.len, s.len);
  const int first = s.k_pos + tile * 128;
  return make_int4(first, s.k_pos + min(tile * 128 + 127, S - 1), s.len, s.len);
}

// Rows [first, 128) or [0, first) of a swizzled operand tile that are padding, cleared by one warp: whatever they hold meets
// weights that are exactly 0, but 0 times an infinity or a NaN is no 0.  `begin` and `end` bound the real rows of the tile.
__device__ __forceinline__ void clear_padding_rows(uint32_t tile, int panels, int rows, int begin, int end, int lane) {
  for (int pn = 0; pn < panels; ++pn)
    for (int c = lane; c < rows * 8; c += 32) {
      const int row = c >> 3;
      if (row < begin || row >= end)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + pn * rows * 128 + c * 16), "r"(0) : "memory");
    }
  fence_proxy_async_smem();
  __syncwarp();
}

}  // namespace rfa
