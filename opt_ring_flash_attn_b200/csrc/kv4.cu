// K/V cache held in 4 bits: append, read-back, and the attention of new tokens over it.
//
// A group of 32 channels of a token and head is u = rint((x - min) / sc) in 0..15 with sc = (max - min) / 15 and min held in
// the cache's 16-bit type; it stands for u * sc + min.  A page holds 64 tokens of every head:
//   codes [page][head][K, V][64][D / 2] bytes,  meta [page][head][K, V][64][D / 32][sc, min]
// so that what one head needs of a page is two runs of memory, which the copy engine brings in with two untiled copies.
// Inside a row the codes lie in the order in which a warp's matrix products want them (NG = D / 32 groups): K as words of 8
// channels, channels [32 g + 8 c, + 8) at word c * NG + g; V as half words of 4, [32 g + 4 c, + 4) at c * NG + g.
#include <limits.h>

#include "scored.cuh"

namespace rfa {

constexpr int kPage = 64;    // tokens
constexpr int kGroup = 32;   // channels
constexpr int kSmCount = 148;

// ----------------------------------------------------------------------------
// Append and read-back: four lanes per group, eight channels each.  Bound by memory: 2 x 16 bytes in and 2 x 5 out per lane.
// ----------------------------------------------------------------------------
template <typename T>
struct Kv4Type;
template <>
struct Kv4Type<__nv_bfloat16> {
  static __device__ __forceinline__ uint16_t bits(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
  static __device__ __forceinline__ float value(uint16_t u) { return __uint_as_float(static_cast<uint32_t>(u) << 16); }
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};
template <>
struct Kv4Type<__half> {
  static __device__ __forceinline__ uint16_t bits(float x) { return __half_as_ushort(__float2half_rn(x)); }
  static __device__ __forceinline__ float value(uint16_t u) { return __half2float(__ushort_as_half(u)); }
  static __device__ __forceinline__ float lo(uint32_t w) { return value(static_cast<uint16_t>(w)); }
  static __device__ __forceinline__ float hi(uint32_t w) { return value(static_cast<uint16_t>(w >> 16)); }
};

struct Kv4Pages {
  uint8_t* codes;
  void* meta;
  const int* table;   // [B][max_pages]
  const int* first;   // [B]: position of token 0
  const int* counts;  // [B] or null: tokens of the row that count
  int n_pages, max_pages;
  int B, T, Hkv, D;
};

// The row (page, head, K, token) of token t of sequence b, or -1 where there is none.
__device__ __forceinline__ long long kv4_row(const Kv4Pages& p, int b, int t, int h) {
  if (p.counts && t >= __ldg(p.counts + b)) return -1;
  const long long pos = static_cast<long long>(__ldg(p.first + b)) + t;
  if (pos < 0 || pos / kPage >= p.max_pages) return -1;
  const int page = __ldg(p.table + static_cast<size_t>(b) * p.max_pages + pos / kPage);
  if (page < 0 || page >= p.n_pages) return -1;
  return ((static_cast<long long>(page) * p.Hkv + h) * 2) * kPage + pos % kPage;
}

// Codes of 8 channels (one lane), low bits first, and the group's (sc, min) in T's bits.
template <typename T>
__device__ __forceinline__ uint32_t quantize8(const uint4& raw, uint32_t& meta) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = Kv4Type<T>::lo(w[i]);
    x[2 * i + 1] = Kv4Type<T>::hi(w[i]);
  }
  // a NaN anywhere makes the group NaN, an infinity gives it an infinite scale: either way it does not read back as numbers
  float hi = x[0], lo = -x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    hi = max_nan(hi, x[i]);
    lo = max_nan(lo, -x[i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = max_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  lo = -lo;
  const uint16_t sb = Kv4Type<T>::bits((hi - lo) / 15.f);
  const float sc = Kv4Type<T>::value(sb);
  meta = static_cast<uint32_t>(sb) | (static_cast<uint32_t>(Kv4Type<T>::bits(lo)) << 16);
  if (!(sc > 0.f)) return 0;
  const float inv = 1.f / sc;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // (x - lo) * (1 / sc) is off by less than 3e-6 in 15; where it lies within 1e-5 of a border between two codes the
    // quotient itself decides, in 64 bits (16-bit inputs hit borders exactly, about one in a thousand)
    float t = (x[i] - lo) * inv;
    if (fabsf(fabsf(t - floorf(t)) - 0.5f) < 1e-5f) t = static_cast<float>(rint((static_cast<double>(x[i]) - lo) / sc));
    const int u = __float2int_rn(fminf(fmaxf(t, 0.f), 15.f));
    codes |= static_cast<uint32_t>(u) << (4 * i);
  }
  return codes;
}

template <typename T>
__global__ void __launch_bounds__(256) kv4_append_kernel(const T* __restrict__ k, const T* __restrict__ v, Kv4Pages p,
                                                         longlong3 ks, longlong3 vs, long long lanes) {
  pdl_wait();
  const int NG = p.D / kGroup;
  const long long id = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const bool in = id < lanes;
  const long long i = in ? id : 0;
  const int c = static_cast<int>(i & 3);
  const int g = static_cast<int>((i >> 2) % NG);
  const long long row = (i >> 2) / NG;
  const int h = static_cast<int>(row % p.Hkv);
  const int t = static_cast<int>(row / p.Hkv % p.T);
  const int b = static_cast<int>(row / p.Hkv / p.T);
  const int ch = g * kGroup + c * 8;
  const uint4 kr = __ldg(reinterpret_cast<const uint4*>(k + b * ks.x + t * ks.y + h * ks.z + ch));
  const uint4 vr = __ldg(reinterpret_cast<const uint4*>(v + b * vs.x + t * vs.y + h * vs.z + ch));
  const long long at = kv4_row(p, b, t, h);
  uint32_t km, vm;
  const uint32_t kc = quantize8<T>(kr, km);
  const uint32_t vc = quantize8<T>(vr, vm);
  if (!in || at < 0) return;
  const size_t half = p.D / 2;
  uint8_t* kd = p.codes + at * half;
  uint8_t* vd = kd + kPage * half;
  *reinterpret_cast<uint32_t*>(kd + 4 * (c * NG + g)) = kc;
  *reinterpret_cast<uint16_t*>(vd + 2 * (2 * c * NG + g)) = static_cast<uint16_t>(vc);
  *reinterpret_cast<uint16_t*>(vd + 2 * ((2 * c + 1) * NG + g)) = static_cast<uint16_t>(vc >> 16);
  uint32_t* md = static_cast<uint32_t*>(p.meta);
  if (c == 0) md[at * NG + g] = km;
  if (c == 1) md[(at + kPage) * NG + g] = vm;
}

template <typename T>
__device__ __forceinline__ uint4 dequantize8(uint32_t codes, uint32_t meta) {
  const float sc = Kv4Type<T>::lo(meta), mn = Kv4Type<T>::hi(meta);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = Pack2<T>::pack(fmaf(static_cast<float>((codes >> (8 * i)) & 15u), sc, mn),
                          fmaf(static_cast<float>((codes >> (8 * i + 4)) & 15u), sc, mn));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__global__ void __launch_bounds__(256) kv4_gather_kernel(T* __restrict__ k, T* __restrict__ v, Kv4Pages p, long long lanes) {
  pdl_wait();
  const int NG = p.D / kGroup;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= lanes) return;
  const int c = static_cast<int>(i & 3);
  const int g = static_cast<int>((i >> 2) % NG);
  const long long row = (i >> 2) / NG;
  const int h = static_cast<int>(row % p.Hkv);
  const int t = static_cast<int>(row / p.Hkv % p.T);
  const int b = static_cast<int>(row / p.Hkv / p.T);
  const long long at = kv4_row(p, b, t, h);
  uint4 ko = make_uint4(0, 0, 0, 0), vo = ko;
  if (at >= 0) {
    const size_t half = p.D / 2;
    const uint8_t* kd = p.codes + at * half;
    const uint8_t* vd = kd + kPage * half;
    const uint32_t* md = static_cast<const uint32_t*>(p.meta);
    const uint32_t kc = *reinterpret_cast<const uint32_t*>(kd + 4 * (c * NG + g));
    const uint32_t v0 = *reinterpret_cast<const uint16_t*>(vd + 2 * (2 * c * NG + g));
    const uint32_t v1 = *reinterpret_cast<const uint16_t*>(vd + 2 * ((2 * c + 1) * NG + g));
    ko = dequantize8<T>(kc, md[at * NG + g]);
    vo = dequantize8<T>(v0 | (v1 << 16), md[(at + kPage) * NG + g]);
  }
  *reinterpret_cast<uint4*>(k + i * 8) = ko;  // lanes run over [B][T][Hkv][D / 8]
  *reinterpret_cast<uint4*>(v + i * 8) = vo;
}

// ----------------------------------------------------------------------------
// Attention of new tokens over the cache
// ----------------------------------------------------------------------------
// Bound by reading the cache (160 bytes per key and head at D = 128), so everything is arranged around a page once it is in
// shared memory, and the pages of all sequences and heads are dealt out evenly: with units (b, kv head, tile of query rows)
// laid end to end, block i takes pages [i q, (i + 1) q) of them all, whatever the lengths are.  A unit that several blocks
// share is joined by a second kernel from at most two partial results per block.
//
// A block has a copying warp, which keeps kStages pages in flight, and four warps of 16 tokens each.  A warp computes, with
// tokens as the 16 rows and query rows (tokens x heads of the group, 8 or 16) as the columns of m16n8k16 products,
//   S[token][row] = sum over groups of sc_k * (u_k . q) + min_k * sum(q)        one accumulator per group
//   O[channel][row] += u_v (P sc_v),   plus sum(P min_v) per group and row      sc_v folded into P
// so the codes enter the tensor cores as they are: 4-bit codes become 16-bit floats by placing them in the mantissa of a power
// of two (one logic operation per two codes).  K keeps that power in its products and takes it out through min; V subtracts
// it, since there the sum runs over all tokens.  P sc_v is rounded to 16 bits like the P of the other kernels.
struct Kv4AttnParams {
  const void* q;
  const uint8_t* codes;
  const void* meta;
  const int* table;
  const int* lens;
  void* out;
  float* lse;
  float* part_o;   // [2 * blocks][rows][D]
  float* part_ml;  // [2 * blocks][rows][2]
  long long q_b, q_t, q_h;  // strides of q, in elements
  int B, T, Hq, Hkv, D;
  int n_pages, max_pages, units, blocks;  // units: (kv head, row tile) pairs of a sequence
  float scale_log2, cap_log2, cap_in;     // cap_in: raw score to the exponent of the tanh
  const float* slopes;
  int slopes_per_batch;
  int* status;
};

__device__ __forceinline__ int kv4_len(const Kv4AttnParams& p, int b) {
  return min(max(__ldg(p.lens + b), 0), p.max_pages * kPage);
}
__device__ __forceinline__ int pages_of(int len) { return (len + kPage - 1) / kPage; }

// Pages of all units, by the whole block (its threads are a multiple of 32, `red` has a slot per warp).
__device__ __forceinline__ long long kv4_total(const Kv4AttnParams& p, int before, long long* red, long long* sum_before) {
  long long all = 0, prior = 0;
  for (int b = threadIdx.x; b < p.B; b += blockDim.x) {
    const int n = pages_of(kv4_len(p, b));
    all += n;
    if (b < before) prior += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    prior += __shfl_xor_sync(0xffffffffu, prior, o);
  }
  if ((threadIdx.x & 31) == 0) {
    red[2 * (threadIdx.x >> 5)] = all;
    red[2 * (threadIdx.x >> 5) + 1] = prior;
  }
  __syncthreads();
  all = prior = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    all += red[2 * w];
    prior += red[2 * w + 1];
  }
  *sum_before = prior * p.units;
  return all * p.units;
}

// A position in the units laid end to end.
struct Kv4Cursor {
  int b, u, page, pages, len;
  __device__ __forceinline__ void open(const Kv4AttnParams& p) {
    len = kv4_len(p, b);
    pages = pages_of(len);
  }
  // the unit's run of pages is done: to the first page of the next unit that has any (p.B: none is left)
  __device__ __forceinline__ void next_unit(const Kv4AttnParams& p) {
    page = 0;
    if (++u < p.units) return;
    u = 0;
    do {
      if (++b >= p.B) return;
      open(p);
    } while (pages == 0);
  }
};

// Page `at` of all; one warp, converged.
__device__ __forceinline__ Kv4Cursor kv4_seek(const Kv4AttnParams& p, long long at) {
  const int lane = threadIdx.x & 31;
  long long base = 0;
  for (int b0 = 0;; b0 += 32) {
    const int n = b0 + lane < p.B ? pages_of(kv4_len(p, b0 + lane)) : 0;
    long long upto = static_cast<long long>(n) * p.units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + upto > at);
    if (past != 0 || b0 + 32 >= p.B) {
      const int l = past != 0 ? __ffs(past) - 1 : 31;
      const long long before = l == 0 ? 0 : __shfl_sync(0xffffffffu, upto, l - 1 < 0 ? 0 : l - 1);
      Kv4Cursor c;
      c.b = min(b0 + l, p.B - 1);
      c.open(p);
      const long long in = at - base - before;
      c.u = c.pages > 0 ? static_cast<int>(in / c.pages) : 0;
      c.page = c.pages > 0 ? static_cast<int>(in % c.pages) : 0;
      return c;
    }
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
}

// 4-bit codes at bits 0-3 and 16-19 of w, shifted there by `e` places of four, as a pair of 16-bit floats kBias + u.
template <typename T, int e>
__device__ __forceinline__ uint32_t codes_pair(uint32_t w) {
  uint32_t r;
  if constexpr (Pack2<T>::kIsBf16) {  // 128 + u: the code in the lowest bits of the 7-bit mantissa
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(e ? w >> (4 * e) : w), "r"(0x000f000fu), "r"(0x43004300u));
  } else {  // 64 + u: at bits 4-7 of the 10-bit mantissa
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(e == 0 ? w << 4 : e == 1 ? w : w >> (4 * e - 4)), "r"(0x00f000f0u), "r"(0x54005400u));
  }
  return r;
}
template <typename T>
__device__ __forceinline__ constexpr float codes_bias() { return Pack2<T>::kIsBf16 ? 128.f : 64.f; }
template <typename T>
__device__ __forceinline__ uint32_t minus_bias(uint32_t x) {
  if constexpr (Pack2<T>::kIsBf16) {
    const uint32_t b = 0x43004300u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const uint32_t b = 0x54005400u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Pack2<T>::kIsBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// N 32-bit words from shared memory, as wide as their alignment (N words) allows.
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], const uint8_t* src) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 x = reinterpret_cast<const uint4*>(src)[i];
      w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 x = reinterpret_cast<const uint2*>(src)[i];
      w[2 * i] = x.x; w[2 * i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(src)[i];
  }
}
// N half words, two to a word (the last word of an odd count has its upper half empty).
template <int N>
__device__ __forceinline__ void lds_halves(uint32_t (&w)[(N + 1) / 2], const uint8_t* src) {
  if constexpr (N % 2 == 0) {
    lds_words<N / 2>(w, src);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t x = reinterpret_cast<const uint16_t*>(src)[i];
      w[i / 2] = (i % 2) ? (w[i / 2] | (x << 16)) : x;
    }
  }
}

template <int NG, int NT>
struct Kv4Cfg {
  static constexpr int kD = NG * kGroup;
  static constexpr int kRows = 8 * NT;
  static constexpr int kCodeBytes = 2 * kPage * kD / 2;
  static constexpr int kMetaBytes = 2 * kPage * NG * 4;
  static constexpr int kStageBytes = kCodeBytes + kMetaBytes;
  static constexpr int kStages = NG <= 2 ? 6 : NG <= 4 ? 4 : 3;
  static constexpr int kBlocksPerSm = NG * NT <= 4 ? 3 : 2;
  static constexpr int kOffJoin = kStages * kStageBytes;           // [kRows][kD] fp32
  static constexpr int kOffMl = kOffJoin + kRows * kD * 4;         // [4 warps][kRows][2]
  static constexpr int kSmemBytes = kOffMl + 4 * kRows * 2 * 4;
  static_assert(kBlocksPerSm * (kSmemBytes + 1024) <= 228 * 1024, "shared memory over budget");
};

template <typename T, int NG, int NT>
__global__ void __launch_bounds__(160, Kv4Cfg<NG, NT>::kBlocksPerSm) kv4_attn_kernel(const Kv4AttnParams p) {
  using Cfg = Kv4Cfg<NG, NT>;
  constexpr int kStages = Cfg::kStages, kRows = Cfg::kRows, D = Cfg::kD;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bar_full[kStages], bar_empty[kStages];
  __shared__ int page_ok[kStages];
  __shared__ long long red[2 * 5];
  __shared__ int abort_flag, skip_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_empty[i], 4);
    }
    mbar_fence_init();
  }
  pdl_wait();
  pdl_trigger();  // the joining kernel waits for this one's results itself
  if (threadIdx.x == 0) skip_flag = *reinterpret_cast<volatile int*>(p.status);
  long long unused;
  const long long total = kv4_total(p, 0, red, &unused);  // a block barrier inside: the barriers are ready behind it
  if (skip_flag != 0) return;
  const long long quota = (total + p.blocks - 1) / p.blocks;
  const long long begin = min(quota * blockIdx.x, total), end = min(begin + quota, total);
  if (begin >= end) return;
  volatile int* abort_p = &abort_flag;
  Kv4Cursor at = kv4_seek(p, begin);
  int left = static_cast<int>(end - begin);
  const int n_row_tiles = p.units / p.Hkv;

  if (warp == 4) {
    // =========================== copying warp ===========================
    int n = 0;
    bool ok = true;
    while (left > 0 && ok) {
      const int run = min(left, at.pages - at.page);
      const int head = at.u / n_row_tiles;
      for (int i0 = 0; i0 < run && ok; i0 += 32) {
        const int mine = i0 + lane < run ? __ldg(p.table + static_cast<size_t>(at.b) * p.max_pages + at.page + i0 + lane) : -1;
        for (int i = 0; i < min(32, run - i0); ++i, ++n) {
          const int page = __shfl_sync(0xffffffffu, mine, i);
          const int st = n % kStages;
          if (lane == 0) {
            ok = mbar_wait(&bar_empty[st], ((n / kStages) & 1) ^ 1, abort_p);
            if (ok) {
              uint8_t* dst = smem + st * Cfg::kStageBytes;
              const bool good = page >= 0 && page < p.n_pages;
              page_ok[st] = good;
              if (good) {
                const size_t slab = static_cast<size_t>(page) * p.Hkv + head;
                mbar_expect_tx(&bar_full[st], Cfg::kStageBytes);
                bulk_load_1d(smem_u32(dst), p.codes + slab * Cfg::kCodeBytes, Cfg::kCodeBytes, &bar_full[st]);
                bulk_load_1d(smem_u32(dst + Cfg::kCodeBytes), static_cast<const uint8_t*>(p.meta) + slab * Cfg::kMetaBytes,
                             Cfg::kMetaBytes, &bar_full[st]);
              } else {
                mbar_arrive(&bar_full[st]);  // a page outside the pool: its tokens are not there
              }
            }
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
          if (!ok) break;
        }
      }
      left -= run;
      at.next_unit(p);
    }
  } else {
    // =========================== the warps that compute ===========================
    const int r = lane >> 2, c = lane & 3;  // S row / O row group, and column pair
    const int G = p.Hq / p.Hkv;
    const float bias = codes_bias<T>();
    int n = 0;
    bool ok = true;  // after a wait that ran out nothing is computed, but every barrier of the block is still met
    while (left > 0) {
      const int run = min(left, at.pages - at.page);
      const int head = at.u / n_row_tiles, row0 = at.u % n_row_tiles * kRows;
      const int n_rows = p.T * G;
      // Query rows as the B operand: lane holds channels [32 g + 8 c, + 8) of row r of each column tile, and the group sums
      uint32_t qf[NT][NG][4];
      float qsum[NT][NG][2], slope[NT][2];
      int lim[NT][2];  // last key that the row sees
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + nt * 8 + r;
        const T* src = static_cast<const T*>(p.q) + at.b * p.q_b + (row / G) * p.q_t + (head * G + row % G) * p.q_h + c * 8;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (row < n_rows) x = __ldg(reinterpret_cast<const uint4*>(src + g * kGroup));
          // pairs (0,4) (1,5) (2,6) (3,7): the order in which shifts bring the codes of a word out
          qf[nt][g][0] = __byte_perm(x.x, x.z, 0x5410);
          qf[nt][g][1] = __byte_perm(x.x, x.z, 0x7632);
          qf[nt][g][2] = __byte_perm(x.y, x.w, 0x5410);
          qf[nt][g][3] = __byte_perm(x.y, x.w, 0x7632);
          float s = (Kv4Type<T>::lo(x.x) + Kv4Type<T>::hi(x.x)) + (Kv4Type<T>::lo(x.y) + Kv4Type<T>::hi(x.y)) +
                    (Kv4Type<T>::lo(x.z) + Kv4Type<T>::hi(x.z)) + (Kv4Type<T>::lo(x.w) + Kv4Type<T>::hi(x.w));
          s += __shfl_xor_sync(0xffffffffu, s, 1);
          s += __shfl_xor_sync(0xffffffffu, s, 2);
          qsum[nt][g][0] = __shfl_sync(0xffffffffu, s, (2 * c) * 4);  // of the columns 2 c and 2 c + 1 that this lane has in S
          qsum[nt][g][1] = __shfl_sync(0xffffffffu, s, (2 * c + 1) * 4);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int col = row0 + nt * 8 + 2 * c + i;
          lim[nt][i] = col < n_rows ? at.len - p.T + col / G : -1;
          slope[nt][i] = 0.f;
          if (p.slopes && col < n_rows)
            slope[nt][i] = __ldg(p.slopes + (p.slopes_per_batch ? static_cast<size_t>(at.b) * p.Hq : 0) + head * G + col % G) * kLog2e;
        }
      }
      float o[NT][NG][2][4], corr[NT][NG][2], m[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][g][0][i] = o[nt][g][1][i] = 0.f;
          corr[nt][g][0] = corr[nt][g][1] = 0.f;
        }
        m[nt][0] = m[nt][1] = kNoKey;
        l[nt][0] = l[nt][1] = 0.f;
      }

      for (int i = 0; i < run; ++i, ++n) {
        const int st = n % kStages;
        ok = ok && mbar_wait_warp(&bar_full[st], (n / kStages) & 1, abort_p);
        if (!ok) continue;
        const uint8_t* stage = smem + st * Cfg::kStageBytes;
        const int pos0 = (at.page + i) * kPage + warp * 16;  // of the warp's first token
        const int there = page_ok[st] ? at.len - pos0 : 0;   // tokens of the warp that exist
        if (there > 0) {
          const bool tail = pos0 + 15 > at.len - p.T;  // some row does not see all of them
          const uint8_t* kc = stage + (warp * 16 + r) * (D / 2) + c * NG * 4;
          const uint8_t* km = stage + Cfg::kCodeBytes + (warp * 16 + r) * (NG * 4);
          // ---- S ----
          float s[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) s[nt][x] = 0.f;
          uint32_t w0[NG], w1[NG], e0[NG], e1[NG];
          lds_words<NG>(w0, kc);
          lds_words<NG>(w1, kc + 8 * (D / 2));
          lds_words<NG>(e0, km);
          lds_words<NG>(e1, km + 8 * (NG * 4));
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint32_t a0[4] = {codes_pair<T, 0>(w0[g]), codes_pair<T, 0>(w1[g]), codes_pair<T, 1>(w0[g]), codes_pair<T, 1>(w1[g])};
            const uint32_t a1[4] = {codes_pair<T, 2>(w0[g]), codes_pair<T, 2>(w1[g]), codes_pair<T, 3>(w0[g]), codes_pair<T, 3>(w1[g])};
            const float sc0 = Kv4Type<T>::lo(e0[g]), mn0 = fmaf(-bias, sc0, Kv4Type<T>::hi(e0[g]));
            const float sc1 = Kv4Type<T>::lo(e1[g]), mn1 = fmaf(-bias, sc1, Kv4Type<T>::hi(e1[g]));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float acc[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816<T>(acc, a0, qf[nt][g][0], qf[nt][g][1]);
              mma16816<T>(acc, a1, qf[nt][g][2], qf[nt][g][3]);
              s[nt][0] = fmaf(acc[0], sc0, fmaf(mn0, qsum[nt][g][0], s[nt][0]));
              s[nt][1] = fmaf(acc[1], sc0, fmaf(mn0, qsum[nt][g][1], s[nt][1]));
              s[nt][2] = fmaf(acc[2], sc1, fmaf(mn1, qsum[nt][g][0], s[nt][2]));
              s[nt][3] = fmaf(acc[3], sc1, fmaf(mn1, qsum[nt][g][1], s[nt][3]));
            }
          }
          // ---- scores in log2 units, masks, running maximum ----
          bool grow = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              float z = s[nt][x];
              const int ahead = lim[nt][x & 1] - (pos0 + r + (x < 2 ? 0 : 8));  // of the row over this key
              if (p.cap_log2 > 0.f) z = fmaf(-2.f * p.cap_log2, fast_rcp(fast_exp2(z * p.cap_in) + 1.f), p.cap_log2);
              else z *= p.scale_log2;
              if (p.slopes) z = fmaf(-slope[nt][x & 1], static_cast<float>(ahead), z);
              if (tail && ahead < 0) z = -INFINITY;
              s[nt][x] = z;
              // the maximum follows when a score is more than 2^2 above it (P sc_v then stays below the largest fp16), or
              // is no number
              grow = grow || !(z - m[nt][x & 1] <= 2.f);
            }
          if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                float top = max3_nan(m[nt][x], s[nt][x], s[nt][x + 2]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float alpha = fast_exp2(m[nt][x] - top);
                m[nt][x] = top;
                l[nt][x] *= alpha;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                  corr[nt][g][x] *= alpha;
                  o[nt][g][0][x] *= alpha;
                  o[nt][g][0][x + 2] *= alpha;
                  o[nt][g][1][x] *= alpha;
                  o[nt][g][1][x + 2] *= alpha;
                }
              }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              s[nt][x] = fast_exp2(s[nt][x] - m[nt][x & 1]);
              l[nt][x & 1] += s[nt][x];
            }
          // ---- O ----
          const uint8_t* vc = stage + kPage * (D / 2) + (warp * 16 + 2 * c) * (D / 2) + r * NG * 2;
          lds_words<NG>(e0, km + kPage * (NG * 4));
          lds_words<NG>(e1, km + (kPage + 8) * (NG * 4));
          if (r >= there) {  // tokens behind the last: their scales may be anything
#pragma unroll
            for (int g = 0; g < NG; ++g) e0[g] = 0;
          }
          if (r + 8 >= there) {
#pragma unroll
            for (int g = 0; g < NG; ++g) e1[g] = 0;
          }
          uint32_t t0[(NG + 1) / 2], t1[(NG + 1) / 2], t8[(NG + 1) / 2], t9[(NG + 1) / 2];
          lds_halves<NG>(t0, vc);
          lds_halves<NG>(t1, vc + D / 2);
          lds_halves<NG>(t8, vc + 8 * (D / 2));
          lds_halves<NG>(t9, vc + 9 * (D / 2));
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint32_t lo = __byte_perm(t0[g / 2], t1[g / 2], g % 2 ? 0x7632 : 0x5410);
            const uint32_t hi = __byte_perm(t8[g / 2], t9[g / 2], g % 2 ? 0x7632 : 0x5410);
            const uint32_t a0[4] = {minus_bias<T>(codes_pair<T, 0>(lo)), minus_bias<T>(codes_pair<T, 1>(lo)),
                                    minus_bias<T>(codes_pair<T, 0>(hi)), minus_bias<T>(codes_pair<T, 1>(hi))};
            const uint32_t a1[4] = {minus_bias<T>(codes_pair<T, 2>(lo)), minus_bias<T>(codes_pair<T, 3>(lo)),
                                    minus_bias<T>(codes_pair<T, 2>(hi)), minus_bias<T>(codes_pair<T, 3>(hi))};
            const float sc0 = Kv4Type<T>::lo(e0[g]), mn0 = Kv4Type<T>::hi(e0[g]);
            const float sc1 = Kv4Type<T>::lo(e1[g]), mn1 = Kv4Type<T>::hi(e1[g]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint32_t b0 = transpose8x8(Pack2<T>::pack(s[nt][0] * sc0, s[nt][1] * sc0));
              const uint32_t b1 = transpose8x8(Pack2<T>::pack(s[nt][2] * sc1, s[nt][3] * sc1));
              corr[nt][g][0] = fmaf(s[nt][0], mn0, fmaf(s[nt][2], mn1, corr[nt][g][0]));
              corr[nt][g][1] = fmaf(s[nt][1], mn0, fmaf(s[nt][3], mn1, corr[nt][g][1]));
              mma16816<T>(o[nt][g][0], a0, b0, b1);
              mma16816<T>(o[nt][g][1], a1, b0, b1);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_empty[st]);
      }

      // ---- the four warps' results of this run into one ----
      float* join = reinterpret_cast<float*>(smem + Cfg::kOffJoin);
      float* ml = reinterpret_cast<float*>(smem + Cfg::kOffMl);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], d);
#pragma unroll
            for (int g = 0; g < NG; ++g) corr[nt][g][x] += __shfl_xor_sync(0xffffffffu, corr[nt][g][x], d);
          }
          if (r == 0) {
            ml[(warp * kRows + nt * 8 + 2 * c + x) * 2] = m[nt][x];
            ml[(warp * kRows + nt * 8 + 2 * c + x) * 2 + 1] = l[nt][x];
          }
        }
      consumers_sync();
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          top[nt][x] = kNoKey;
          for (int w = 0; w < 4; ++w) top[nt][x] = max_nan(top[nt][x], ml[(w * kRows + nt * 8 + 2 * c + x) * 2]);
        }
      for (int w = 0; w < 4; ++w) {  // in the order of the warps: the same sum every time
        if (w == warp) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float f = fast_exp2(m[nt][x] - top[nt][x]);
#pragma unroll
              for (int g = 0; g < NG; ++g) {  // channels 32 g + 4 r + (0..3)
                float4* dst = reinterpret_cast<float4*>(join + (nt * 8 + 2 * c + x) * D + g * kGroup + 4 * r);
                const float4 old = w == 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *dst;
                *dst = make_float4(fmaf(o[nt][g][0][x] + corr[nt][g][x], f, old.x), fmaf(o[nt][g][0][x + 2] + corr[nt][g][x], f, old.y),
                                   fmaf(o[nt][g][1][x] + corr[nt][g][x], f, old.z), fmaf(o[nt][g][1][x + 2] + corr[nt][g][x], f, old.w));
              }
            }
        }
        consumers_sync();
      }
      const bool whole = at.page == 0 && run == at.pages;
      const int slot = 2 * blockIdx.x + (at.page > 0 ? 0 : 1);
      for (int i = threadIdx.x; i < kRows * D / 8; i += 128) {
        const int row = i / (D / 8), ch = i % (D / 8) * 8, rg = row0 + row;
        if (rg >= n_rows) continue;
        float mm = kNoKey, ll = 0.f;
        for (int w = 0; w < 4; ++w) mm = max_nan(mm, ml[(w * kRows + row) * 2]);
        for (int w = 0; w < 4; ++w) ll += ml[(w * kRows + row) * 2 + 1] * fast_exp2(ml[(w * kRows + row) * 2] - mm);
        const float4 x = *reinterpret_cast<const float4*>(join + row * D + ch);
        const float4 y = *reinterpret_cast<const float4*>(join + row * D + ch + 4);
        if (whole) {
          const int t = rg / G, h = head * G + rg % G;
          const float inv = ll == 0.f ? 0.f : 1.f / ll;
          T* dst = static_cast<T*>(p.out) + ((static_cast<size_t>(at.b) * p.T + t) * p.Hq + h) * D + ch;
          *reinterpret_cast<uint4*>(dst) = make_uint4(Pack2<T>::pack(x.x * inv, x.y * inv), Pack2<T>::pack(x.z * inv, x.w * inv),
                                                      Pack2<T>::pack(y.x * inv, y.y * inv), Pack2<T>::pack(y.z * inv, y.w * inv));
          if (p.lse && ch == 0)
            p.lse[(static_cast<size_t>(at.b) * p.Hq + h) * p.T + t] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) / kLog2e;
        } else {
          float* dst = p.part_o + (static_cast<size_t>(slot) * kRows + row) * D + ch;
          *reinterpret_cast<float4*>(dst) = x;
          *reinterpret_cast<float4*>(dst + 4) = y;
          if (ch == 0) *reinterpret_cast<float2*>(p.part_ml + (static_cast<size_t>(slot) * kRows + row) * 2) = make_float2(mm, ll);
        }
      }
      consumers_sync();  // the next run writes the same buffers
      left -= run;
      at.next_unit(p);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && abort_flag) {
    // Give copies that are still in flight time to land before the block's shared memory is released.
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    atomicExch(p.status, kStatusWaitTimeout);
  }
}

// One block per (b, unit, row): joins the partial results of a unit that several blocks shared, and answers for sequences
// without keys.
template <typename T>
__global__ void __launch_bounds__(128) kv4_join_kernel(const Kv4AttnParams p, int tile_rows) {
  __shared__ long long red[2 * 4];
  pdl_wait();
  const int n_row_tiles = p.units / p.Hkv, G = p.Hq / p.Hkv;
  const int row = blockIdx.x % tile_rows;
  const int u = blockIdx.x / tile_rows % p.units, b = blockIdx.x / tile_rows / p.units;
  const int rg = u % n_row_tiles * tile_rows + row;
  if (rg >= p.T * G) return;
  const int t = rg / G, h = u / n_row_tiles * G + rg % G;
  T* dst = static_cast<T*>(p.out) + ((static_cast<size_t>(b) * p.T + t) * p.Hq + h) * p.D;
  float* lse = p.lse ? p.lse + (static_cast<size_t>(b) * p.Hq + h) * p.T + t : nullptr;
  const int pages = pages_of(kv4_len(p, b));
  const int d = threadIdx.x * 2;
  if (pages == 0) {
    if (d < p.D) *reinterpret_cast<uint32_t*>(dst + d) = 0;
    if (lse && d == 0) *lse = -INFINITY;
    return;
  }
  long long first;
  const long long total = kv4_total(p, b, red, &first);
  const long long quota = (total + p.blocks - 1) / p.blocks;
  first += static_cast<long long>(u) * pages;
  const int c0 = static_cast<int>(first / quota), c1 = static_cast<int>((first + pages - 1) / quota);
  if (c0 == c1) return;  // written by that block
  auto slot = [&](int c) { return static_cast<size_t>(2 * c + (c == c0 ? 1 : 0)) * tile_rows + row; };
  float top = kNoKey;
  for (int c = c0; c <= c1; ++c) top = max_nan(top, p.part_ml[slot(c) * 2]);
  float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) {
    const size_t s = slot(c);
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + s * 2);
    const float f = fast_exp2(ml.x - top);
    sum = fmaf(ml.y, f, sum);
    if (d < p.D) {
      const float2 v = *reinterpret_cast<const float2*>(p.part_o + s * p.D + d);
      x = fmaf(v.x, f, x);
      y = fmaf(v.y, f, y);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (d < p.D) *reinterpret_cast<uint32_t*>(dst + d) = Pack2<T>::pack(x * inv, y * inv);
  if (lse && d == 0) *lse = sum == 0.f ? -INFINITY : (top + log2f(sum)) / kLog2e;
}

// Column tiles of 8 query rows: two where there are more rows than one holds and registers for both.
static int kv4_tiles(int T, int G, int D) { return T * G > 8 && D <= 128 ? 2 : 1; }
static int kv4_blocks(int D, int nt) { return kSmCount * (D / kGroup * nt <= 4 ? 3 : 2); }
static bool kv4_dim(int D) { return D == 64 || D == 96 || D == 128 || D == 192 || D == 256; }

template <typename T, int NG, int NT>
static int launch_kv4_attn(const Kv4AttnParams& p, cudaStream_t s) {
  using Cfg = Kv4Cfg<NG, NT>;
  auto kern = kv4_attn_kernel<T, NG, NT>;
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) { cudaGetLastError(); return RFA_ERR_CUDA; }
  if (!attr_done[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes) != cudaSuccess) {
      cudaGetLastError();
      return RFA_ERR_CUDA;
    }
    attr_done[dev] = true;
  }
  const int rc = launch_chained(kern, static_cast<unsigned>(p.blocks), 160, Cfg::kSmemBytes, s, p);
  if (rc != RFA_OK) return rc;
  return launch_chained(kv4_join_kernel<T>, static_cast<unsigned>(p.B) * p.units * Cfg::kRows, 128, 0, s, p,
                        static_cast<int>(Cfg::kRows));
}

template <typename T>
static int dispatch_kv4_attn(const Kv4AttnParams& p, int nt, cudaStream_t s) {
  switch (p.D) {
    case 64: return nt == 2 ? launch_kv4_attn<T, 2, 2>(p, s) : launch_kv4_attn<T, 2, 1>(p, s);
    case 96: return nt == 2 ? launch_kv4_attn<T, 3, 2>(p, s) : launch_kv4_attn<T, 3, 1>(p, s);
    case 128: return nt == 2 ? launch_kv4_attn<T, 4, 2>(p, s) : launch_kv4_attn<T, 4, 1>(p, s);
    case 192: return launch_kv4_attn<T, 6, 1>(p, s);
    case 256: return launch_kv4_attn<T, 8, 1>(p, s);
    default: return RFA_ERR_UNSUPPORTED;
  }
}

static int kv4_check(const void* codes, const void* meta, int n_pages, const int* table, int max_pages, const int* rows, int B,
                     int T, int Hkv, int D, int dtype) {
  if (!codes || !meta || !table || !rows) return RFA_ERR_INVALID_ARG;
  if (n_pages <= 0 || max_pages <= 0 || B <= 0 || T <= 0 || Hkv <= 0) return RFA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(codes) & 15u) || (reinterpret_cast<uintptr_t>(meta) & 15u) ||
      (reinterpret_cast<uintptr_t>(table) & 3u) || (reinterpret_cast<uintptr_t>(rows) & 3u))
    return RFA_ERR_INVALID_ARG;
  if (!kv4_dim(D)) return RFA_ERR_UNSUPPORTED;
  if (dtype != RFA_DTYPE_BF16 && dtype != RFA_DTYPE_FP16) return RFA_ERR_UNSUPPORTED;
  if (max_pages > INT_MAX / kPage) return RFA_ERR_TOO_LARGE;
  return RFA_OK;
}

}  // namespace rfa

extern "C" int rfa_kv4_append(const void* k, const void* v, const long long* k_strides, const long long* v_strides,
                              void* codes, void* meta, int n_pages, const int* table, int max_pages, const int* positions,
                              const int* counts, int B, int T, int Hkv, int D, int dtype, void* stream) {
  using namespace rfa;
  if (!k || !v || !k_strides || !v_strides) return RFA_ERR_INVALID_ARG;
  const int rc = kv4_check(codes, meta, n_pages, table, max_pages, positions, B, T, Hkv, D, dtype);
  if (rc != RFA_OK) return rc;
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0) return RFA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(k) & 15u) || (reinterpret_cast<uintptr_t>(v) & 15u) ||
      (reinterpret_cast<uintptr_t>(counts) & 3u))
    return RFA_ERR_INVALID_ARG;
  const long long lanes = static_cast<long long>(B) * T * Hkv * (D / 8);
  if (lanes > 256ll * INT_MAX) return RFA_ERR_TOO_LARGE;
  const Kv4Pages p{static_cast<uint8_t*>(codes), meta, table, positions, counts, n_pages, max_pages, B, T, Hkv, D};
  const longlong3 ks = make_longlong3(k_strides[0], k_strides[1], k_strides[2]);
  const longlong3 vs = make_longlong3(v_strides[0], v_strides[1], v_strides[2]);
  const unsigned grid = static_cast<unsigned>((lanes + 255) / 256);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == RFA_DTYPE_BF16)
    return launch_chained(kv4_append_kernel<__nv_bfloat16>, grid, 256, 0, s, static_cast<const __nv_bfloat16*>(k),
                          static_cast<const __nv_bfloat16*>(v), p, ks, vs, lanes);
  return launch_chained(kv4_append_kernel<__half>, grid, 256, 0, s, static_cast<const __half*>(k),
                        static_cast<const __half*>(v), p, ks, vs, lanes);
}

extern "C" int rfa_kv4_gather(void* k, void* v, const void* codes, const void* meta, int n_pages, const int* table,
                              int max_pages, const int* positions, const int* counts, int B, int T, int Hkv, int D, int dtype,
                              void* stream) {
  using namespace rfa;
  if (!k || !v) return RFA_ERR_INVALID_ARG;
  const int rc = kv4_check(codes, meta, n_pages, table, max_pages, positions, B, T, Hkv, D, dtype);
  if (rc != RFA_OK) return rc;
  if ((reinterpret_cast<uintptr_t>(k) & 15u) || (reinterpret_cast<uintptr_t>(v) & 15u) ||
      (reinterpret_cast<uintptr_t>(counts) & 3u))
    return RFA_ERR_INVALID_ARG;
  const long long lanes = static_cast<long long>(B) * T * Hkv * (D / 8);
  if (lanes > 256ll * INT_MAX) return RFA_ERR_TOO_LARGE;
  const Kv4Pages p{static_cast<uint8_t*>(const_cast<void*>(codes)), const_cast<void*>(meta), table, positions, counts,
                   n_pages, max_pages, B, T, Hkv, D};
  const unsigned grid = static_cast<unsigned>((lanes + 255) / 256);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == RFA_DTYPE_BF16)
    return launch_chained(kv4_gather_kernel<__nv_bfloat16>, grid, 256, 0, s, static_cast<__nv_bfloat16*>(k),
                          static_cast<__nv_bfloat16*>(v), p, lanes);
  return launch_chained(kv4_gather_kernel<__half>, grid, 256, 0, s, static_cast<__half*>(k), static_cast<__half*>(v), p, lanes);
}

extern "C" size_t rfa_kv4_scratch_elems(int T, int Hq, int Hkv, int D) {
  using namespace rfa;
  if (T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || !kv4_dim(D)) return 0;
  const int nt = kv4_tiles(T, Hq / Hkv, D);
  return static_cast<size_t>(2) * kv4_blocks(D, nt) * 8 * nt * (D + 2);
}

extern "C" int rfa_kv4_attn(const void* q, const long long* q_strides, const void* codes, const void* meta, int n_pages,
                            const int* table, int max_pages, const int* lens, void* out, float* lse, float* scratch, int B,
                            int T, int Hq, int Hkv, int D, int dtype, float softmax_scale, float softcap, const float* slopes,
                            int slopes_per_batch, int* status, void* stream) {
  using namespace rfa;
  if (!q || !q_strides || !out || !scratch || !status) return RFA_ERR_INVALID_ARG;
  const int rc = kv4_check(codes, meta, n_pages, table, max_pages, lens, B, T, Hkv, D, dtype);
  if (rc != RFA_OK) return rc;
  if (Hq <= 0 || Hq % Hkv != 0) return RFA_ERR_INVALID_ARG;
  if (!(softmax_scale > 0.f) || !(softmax_scale <= 3.0e38f) || !(softcap >= 0.f) || !(softcap <= 3.0e38f))
    return RFA_ERR_INVALID_ARG;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 != 0) return RFA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(q) & 15u) || (reinterpret_cast<uintptr_t>(out) & 15u) ||
      (reinterpret_cast<uintptr_t>(scratch) & 15u) || (reinterpret_cast<uintptr_t>(lse) & 3u) ||
      (reinterpret_cast<uintptr_t>(slopes) & 3u))
    return RFA_ERR_INVALID_ARG;
  const int nt = kv4_tiles(T, Hq / Hkv, D), rows = 8 * nt;
  const long long row_tiles = (static_cast<long long>(T) * (Hq / Hkv) + rows - 1) / rows;
  const long long units = row_tiles * Hkv;
  if (static_cast<long long>(T) * Hq > INT_MAX / 2 || units * rows * B > INT_MAX / 2) return RFA_ERR_TOO_LARGE;
  Kv4AttnParams p{};
  p.q = q;
  p.codes = static_cast<const uint8_t*>(codes);
  p.meta = meta;
  p.table = table;
  p.lens = lens;
  p.out = out;
  p.lse = lse;
  p.q_b = q_strides[0];
  p.q_t = q_strides[1];
  p.q_h = q_strides[2];
  p.B = B;
  p.T = T;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.D = D;
  p.n_pages = n_pages;
  p.max_pages = max_pages;
  p.units = static_cast<int>(units);
  // no more blocks than pages there can be; a block's share must fit an int
  const long long most = static_cast<long long>(max_pages) * units * B;
  p.blocks = static_cast<int>(most < kv4_blocks(D, nt) ? most : kv4_blocks(D, nt));
  if (most / p.blocks >= INT_MAX) return RFA_ERR_TOO_LARGE;
  p.part_o = scratch;
  p.part_ml = scratch + static_cast<size_t>(2) * p.blocks * rows * D;
  p.scale_log2 = softmax_scale * kLog2e;
  p.cap_log2 = softcap * kLog2e;
  p.cap_in = softcap > 0.f ? 2.f * softmax_scale * kLog2e / softcap : 0.f;
  p.slopes = slopes;
  p.slopes_per_batch = slopes_per_batch;
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == RFA_DTYPE_BF16 ? dispatch_kv4_attn<__nv_bfloat16>(p, nt, s) : dispatch_kv4_attn<__half>(p, nt, s);
}
