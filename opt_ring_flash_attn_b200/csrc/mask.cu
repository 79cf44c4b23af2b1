// Document masks: the intervals, hulls and work orders of a mask buffer (scored.cuh) from document borders.
// Both kernels are bound by latency: S 16384 in 10 documents takes two launches of a few microseconds, once per batch
// of documents; every layer and both directions of a training step read the same buffer.
#include "scored.cuh"

namespace rfa {

__device__ __forceinline__ int clamp_pos(int x, int len) { return min(max(x, 0), len); }

// One block per (b, shard, tile): thread = row.  The document of a position by bisection over its borders.
__global__ void __launch_bounds__(128) mask_rows_kernel(const int* __restrict__ cu, const int* __restrict__ prefix,
                                                        int cu_rows, int n_docs, int B, int S, int shards, int causal,
                                                        int* __restrict__ mask) {
  const MaskView v = mask_view(mask, B, S, shards);
  const int nT = (S + 127) / 128, len = S * shards;
  const int tile = blockIdx.x % nT, shard = blockIdx.x / nT % shards, b = blockIdx.x / nT / shards;
  const int row = tile * 128 + threadIdx.x, pos = shard * S + row;
  const int* c = cu + (cu_rows == 1 ? 0 : static_cast<size_t>(b) * (n_docs + 1));
  int q_lo = 0, q_hi = 0, k_lo = 0, k_hi = 0;
  if (row < S) {
    int a = 0, z = n_docs;  // the number of documents that end at or before pos
    while (a < z) {
      const int mid = (a + z) / 2;
      if (c[mid + 1] <= pos) a = mid + 1;
      else z = mid;
    }
    if (a < n_docs && c[a] <= pos) {
      const int start = clamp_pos(c[a], len), end = clamp_pos(c[a + 1], len);
      int seen = start;  // keys before it are seen by the whole document
      if (prefix) {
        const int p = prefix[(cu_rows == 1 ? 0 : static_cast<size_t>(b) * n_docs) + a];
        seen = start + min(max(p, 0), end - start);
      }
      q_lo = start;
      q_hi = causal ? max(pos + 1, seen) : end;
      k_lo = causal && pos >= seen ? pos : start;
      k_hi = end;
    }
    const size_t at = static_cast<size_t>(b) * len + pos;
    const_cast<int*>(v.q_lo)[at] = q_lo;
    const_cast<int*>(v.q_hi)[at] = q_hi;
    const_cast<int*>(v.k_lo)[at] = k_lo;
    const_cast<int*>(v.k_hi)[at] = k_hi;
  }
  __shared__ int part[4][8];
  const bool some = q_lo < q_hi, counts = row < S;
  int r[8];
  r[0] = some ? q_lo : INT_MAX;
  r[1] = !counts ? INT_MIN : some ? q_lo : INT_MAX;
  r[2] = !counts ? INT_MAX : some ? q_hi : 0;
  r[3] = some ? q_hi : 0;
  r[4] = some ? k_lo : INT_MAX;
  r[5] = !counts ? INT_MIN : some ? k_lo : INT_MAX;
  r[6] = !counts ? INT_MAX : some ? k_hi : 0;
  r[7] = some ? k_hi : 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r[i] = (i % 4 == 0 || i % 4 == 2) ? __reduce_min_sync(0xffffffffu, r[i]) : __reduce_max_sync(0xffffffffu, r[i]);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][i] = r[i];
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    int h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = part[0][threadIdx.x * 4 + i];
      for (int w = 1; w < 4; ++w) {
        const int x = part[w][threadIdx.x * 4 + i];
        h[i] = (i == 0 || i == 2) ? min(h[i], x) : max(h[i], x);
      }
    }
    if (h[0] == INT_MAX) h[0] = 0;  // nothing but empty rows: the range of tiles is [0, 0)
    const size_t at = (static_cast<size_t>(b) * shards + shard) * nT + tile;
    const_cast<int4*>(threadIdx.x == 0 ? v.q_tile : v.k_tile)[at] = make_int4(h[0], h[1], h[2], h[3]);
  }
  if (tile == 0 && shard == 0 && threadIdx.x == 0) {
    const int begin = clamp_pos(c[0], len);
    const_cast<int*>(v.real)[2 * b] = begin;
    const_cast<int*>(v.real)[2 * b + 1] = max(begin, clamp_pos(c[n_docs], len));
  }
}

// Tiles of the other side that a tile (or a pair of them) meets.
__device__ __forceinline__ int tiles_met(const int4* hulls, int n) {
  int lo = INT_MAX, hi = 0;
  for (int i = 0; i < n; ++i)
    if (hulls[i].w > hulls[i].x) {
      lo = min(lo, hulls[i].x);
      hi = max(hi, hulls[i].w);
    }
  return hi > 0 ? (hi + 127) / 128 - lo / 128 : 0;
}

// The rank of every item by falling work: counting, which needs no sorting network and no scratch.  Work lists have a few
// hundred items; they are read by the blocks that run the long items first.
__global__ void __launch_bounds__(256) mask_order_kernel(int B, int S, int shards, int* __restrict__ mask) {
  const MaskView v = mask_view(mask, B, S, shards);
  const int nT = (S + 127) / 128;
  const int list = blockIdx.y % 3, shard = blockIdx.y / 3;
  const int width = list == 1 ? 2 : 1, per_row = list == 1 ? (nT + 1) / 2 : nT, n = B * per_row;
  const int4* hulls = (list == 2 ? v.k_tile : v.q_tile) + static_cast<size_t>(shard) * nT;
  auto work = [&](int i) {
    const int b = i / per_row, t = i % per_row * width;
    return tiles_met(hulls + static_cast<size_t>(b) * shards * nT + t, min(width, nT - t));
  };
  __shared__ int others[256];
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (blockIdx.x * 256 >= n) return;  // the same for the whole block
  const int mine = i < n ? work(i) : 0;
  int rank = 0;
  for (int j0 = 0; j0 < n; j0 += 256) {
    const int j = j0 + threadIdx.x;
    __syncthreads();
    others[threadIdx.x] = j < n ? work(j) : -1;
    __syncthreads();
    const int m = min(256, n - j0);
    for (int k = 0; k < m; ++k) rank += (others[k] > mine || (others[k] == mine && j0 + k < i)) ? 1 : 0;
  }
  if (i < n) {
    int* order = const_cast<int*>(list == 0 ? v.order_q + static_cast<size_t>(shard) * n
                                  : list == 1 ? v.order_q2 + static_cast<size_t>(shard) * n
                                              : v.order_k + static_cast<size_t>(shard) * n);
    order[rank] = i;
  }
}

}  // namespace rfa

extern "C" size_t rfa_mask_elems(int B, int S, int shards) {
  if (B <= 0 || S <= 0 || shards <= 0 || static_cast<long long>(S) * shards > INT_MAX / 2) return 0;
  if (static_cast<long long>(B) * shards * ((S + 127) / 128) > INT_MAX / 2 || shards > 65535 / 3) return 0;
  return rfa::mask_elems(B, S, shards);
}

extern "C" int rfa_document_mask(const int* cu, const int* prefix, int cu_rows, int n_docs, int B, int S, int shards,
                                 int causal, int* mask, void* stream) {
  using namespace rfa;
  if (!cu || !mask || n_docs < 1 || n_docs > INT_MAX / 4) return RFA_ERR_INVALID_ARG;
  if (cu_rows != 1 && cu_rows != B) return RFA_ERR_INVALID_ARG;
  if (rfa_mask_elems(B, S, shards) == 0) return RFA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(mask) & 15u) || (reinterpret_cast<uintptr_t>(cu) & 3u) ||
      (reinterpret_cast<uintptr_t>(prefix) & 3u))
    return RFA_ERR_INVALID_ARG;
  const int nT = ceil_div(S, 128);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  mask_rows_kernel<<<static_cast<unsigned>(B) * shards * nT, 128, 0, s>>>(cu, prefix, cu_rows, n_docs, B, S, shards, causal,
                                                                          mask);
  mask_order_kernel<<<dim3(ceil_div(B * nT, 256), 3 * shards), 256, 0, s>>>(B, S, shards, mask);
  return cuda_status(cudaGetLastError());
}
