// K/V cache held in 4 bits: append, read-back, and the attention of new tokens over it.
//
// A group of 32 channels of a token and head is u = rint((x - min) / sc) in 0..15 with sc = (max - min) / 15 and min held in
// the cache's 16-bit type; it stands for u * sc + min.  A page holds 64 tokens of every head:
//   codes [page][head][K, V][64][D / 2] bytes,  meta [page][head][K, V][64][D / 32][sc, min]
// so that what one head needs of a page is two runs of memory, which the copy engine brings in with two untiled copies.
// Inside a row the codes lie in the order in which a warp's matrix products want them (NG = D / 32 groups): K as words of 8
// channels, channels [32 g + 8 c, + 8) at word c * NG + g; V as half words of 4, [32 g + 4 c, + 4) at c * NG + g.
#include <limits.h>

#include <type_traits>

#include "scored.cuh"

namespace rfa {

constexpr int kPage = 64;    // tokens
constexpr int kGroup = 32;   // channels
constexpr int kSmCount = 148;
constexpr int kMaxParts = kSmCount * 4;  // blocks of a launch at most

// ----------------------------------------------------------------------------
// Append and read-back: four lanes per group, eight channels each.  8192 tokens of 8 heads of 128 in 22 and 13 us, 2.0 and 3.3 TB/s
// of 44 MB each: bound by instructions (issue 72 % busy, the logic unit 52 and 64 %), of which a border between two codes in one
// group of many takes a fourth.  One token of 64 sequences: 6.3 us for both, launches.  Four tokens per lane instead of one, to
// share the index arithmetic, keep too few warps resident: 33 us.
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

// Larger ones of two pairs; NaN where either is.
template <typename T>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (Pack2<T>::kIsBf16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

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

// The code of an x that lies next to a border between two (16-bit inputs hit borders exactly, about one in a thousand): the
// sign of x - lo - border * sc decides.  The product is exact (5 bits times 11), its difference from x - lo is (they are nearly
// equal), and what rounding x - lo left over is known.  A call, because unrolled into its caller it outgrows the instruction
// cache.
__device__ __noinline__ float border_code(float x, float lo, float sc, float t) {
  const float d = x - lo;
  const float below = floorf(t), border = below + 0.5f;
  const float part_x = d + lo, part_lo = d - part_x;  // d = x - lo + what the two parts lack
  const float left = (x - part_x) + (-lo - part_lo);
  const float side = fmaf(-border, sc, d) + left;
  const bool up = side > 0.f || (side == 0.f && (static_cast<int>(below) & 1));
  return fminf(up ? below + 1.f : below, 15.f);
}

// Scales below the smallest normal number of their type keep fewer bits, and 15 of them may fall short of the range.
template <typename T>
constexpr float kSmallScale = Pack2<T>::kIsBf16 ? 1.1754944e-38f * 18446744073709551616.f : 6.103515625e-5f;

// Codes of 8 channels (one lane), low bits first, and the group's (sc, min) in T's bits.
template <typename T>
__device__ __forceinline__ uint32_t quantize8(const uint4& raw, uint32_t& meta) {
  // Maximum and (negated) minimum as pairs of 16 bits.  A NaN anywhere makes the group NaN, an infinity gives it an infinite
  // scale: either way it does not read back as numbers.
  const uint32_t top2 = max2_nan<T>(max2_nan<T>(raw.x, raw.y), max2_nan<T>(raw.z, raw.w));
  constexpr uint32_t sign = 0x80008000u;
  const uint32_t low2 = max2_nan<T>(max2_nan<T>(raw.x ^ sign, raw.y ^ sign), max2_nan<T>(raw.z ^ sign, raw.w ^ sign));
  uint32_t ends = max2_nan<T>(__byte_perm(top2, low2, 0x5410), __byte_perm(top2, low2, 0x7632));  // (max, -min)
  ends = max2_nan<T>(ends, __shfl_xor_sync(0xffffffffu, ends, 1));
  ends = max2_nan<T>(ends, __shfl_xor_sync(0xffffffffu, ends, 2));
  const float hi = Kv4Type<T>::lo(ends);
  float lo = -Kv4Type<T>::hi(ends);
  // (hi - lo) / 15, correctly rounded: the quotient with a rounded reciprocal, put right by its exact remainder
  const float span = hi - lo;
  const float q = span * 0.06666667f;
  const uint16_t sb = Kv4Type<T>::bits(span < INFINITY ? fmaf(fmaf(-15.f, q, span), 0.06666667f, q) : span);
  float sc = Kv4Type<T>::value(sb);
  meta = static_cast<uint32_t>(sb) | ((ends ^ sign) & 0xffff0000u);
  if (!(sc > 0.f)) return 0;
  // channels i and i + 4 as a pair
  float x[8] = {Kv4Type<T>::lo(raw.x), Kv4Type<T>::hi(raw.x), Kv4Type<T>::lo(raw.y), Kv4Type<T>::hi(raw.y),
                Kv4Type<T>::lo(raw.z), Kv4Type<T>::hi(raw.z), Kv4Type<T>::lo(raw.w), Kv4Type<T>::hi(raw.w)};
  if (sc < 1e-30f) {  // its reciprocal would leave fp32 (bf16 only): the same codes under a power of two
    constexpr float up = 18446744073709551616.f;
    sc *= up;
    lo *= up;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= up;
  }
  // (x - lo) * (1 / sc) is off by less than 6e-6 in 15, so its nearest whole number is the code unless it lies within 1e-5
  // of a border between two codes, or beyond 15 because a small scale lost bits.
  const float inv = fast_rcp(sc);
  const uint64_t inv2 = pack_f2(inv, inv), lo2 = pack_f2(lo, lo);
  constexpr float magic = 12582912.f;  // 1.5 * 2^23: adding it rounds to a whole number, ties to even
  const uint64_t magic2 = pack_f2(magic, magic);
  float u[8], away = 0.f;
  uint64_t four = 0;  // four codes each, as numbers of 16 bits
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    const uint64_t t = mul2(sub2(pack_f2(x[i], x[i + 4]), lo2), inv2);
    const uint64_t w = sub2(add2(t, magic2), magic2);
    float a0, a1;
    unpack_f2(sub2(t, w), a0, a1);
    away = fmaxf(away, fmaxf(fabsf(a0), fabsf(a1)));
    unpack_f2(w, u[i], u[i + 4]);
    four = fma2(four, pack_f2(16.f, 16.f), w);
  }
  float p0, p1;
  unpack_f2(four, p0, p1);
  if (away > 0.49999f || sc < kSmallScale<T>) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = (x[i] - lo) * inv;
      if (fabsf(t - u[i]) > 0.49999f) u[i] = border_code(x[i], lo, sc, t);
      u[i] = fminf(u[i], 15.f);
    }
    p0 = fmaf(fmaf(fmaf(u[3], 16.f, u[2]), 16.f, u[1]), 16.f, u[0]);
    p1 = fmaf(fmaf(fmaf(u[7], 16.f, u[6]), 16.f, u[5]), 16.f, u[4]);
  }
  return static_cast<uint32_t>(__float2int_rn(p0)) | (static_cast<uint32_t>(__float2int_rn(p1)) << 16);
}

// Lane i of sequence b: channels [32 g + 8 c, + 8) of head h of token t, in the order of memory.
template <int NG>
struct Kv4Lane {
  int c, g, h, t;
  __device__ __forceinline__ Kv4Lane(unsigned i, unsigned Hkv) {
    c = i & 3;
    const unsigned group = i >> 2, row = group / NG;
    g = group % NG;
    h = row % Hkv;
    t = row / Hkv;
  }
};

template <typename T, int NG>
__global__ void __launch_bounds__(256) kv4_append_kernel(const T* __restrict__ k, const T* __restrict__ v, Kv4Pages p,
                                                         longlong3 ks, longlong3 vs, unsigned lanes) {
  pdl_wait();
  pdl_trigger();  // what follows on the stream waits for the results itself
  const unsigned id = blockIdx.x * 256u + threadIdx.x;
  const bool in = id < lanes;
  const Kv4Lane<NG> at_lane(in ? id : 0, p.Hkv);
  const int c = at_lane.c, g = at_lane.g;
  const int ch = g * kGroup + c * 8;
  constexpr size_t half = NG * kGroup / 2;
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const uint4 kr = __ldg(reinterpret_cast<const uint4*>(k + b * ks.x + at_lane.t * ks.y + at_lane.h * ks.z + ch));
    const uint4 vr = __ldg(reinterpret_cast<const uint4*>(v + b * vs.x + at_lane.t * vs.y + at_lane.h * vs.z + ch));
    const long long at = kv4_row(p, b, at_lane.t, at_lane.h);
    uint32_t km, vm;
    const uint32_t kc = quantize8<T>(kr, km);
    const uint32_t vc = quantize8<T>(vr, vm);
    if (!in || at < 0) continue;
    uint8_t* kd = p.codes + at * half;
    uint8_t* vd = kd + kPage * half;
    *reinterpret_cast<uint32_t*>(kd + 4 * (c * NG + g)) = kc;
    *reinterpret_cast<uint16_t*>(vd + 2 * (2 * c * NG + g)) = static_cast<uint16_t>(vc);
    *reinterpret_cast<uint16_t*>(vd + 2 * ((2 * c + 1) * NG + g)) = static_cast<uint16_t>(vc >> 16);
    uint32_t* md = static_cast<uint32_t*>(p.meta);
    if (c == 0) md[at * NG + g] = km;
    if (c == 1) md[(at + kPage) * NG + g] = vm;
  }
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

template <typename T, int NG>
__global__ void __launch_bounds__(256) kv4_gather_kernel(T* __restrict__ k, T* __restrict__ v, Kv4Pages p, unsigned lanes) {
  pdl_wait();
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= lanes) return;
  const Kv4Lane<NG> lane(i, p.Hkv);
  const int c = lane.c, g = lane.g;
  constexpr size_t half = NG * kGroup / 2;
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const long long at = kv4_row(p, b, lane.t, lane.h);
    uint4 ko = make_uint4(0, 0, 0, 0), vo = ko;
    if (at >= 0) {
      const uint8_t* kd = p.codes + at * half;
      const uint8_t* vd = kd + kPage * half;
      const uint32_t* md = static_cast<const uint32_t*>(p.meta);
      const uint32_t kc = *reinterpret_cast<const uint32_t*>(kd + 4 * (c * NG + g));
      const uint32_t v0 = *reinterpret_cast<const uint16_t*>(vd + 2 * (2 * c * NG + g));
      const uint32_t v1 = *reinterpret_cast<const uint16_t*>(vd + 2 * ((2 * c + 1) * NG + g));
      ko = dequantize8<T>(kc, md[at * NG + g]);
      vo = dequantize8<T>(v0 | (v1 << 16), md[(at + kPage) * NG + g]);
    }
    const size_t to = (static_cast<size_t>(b) * lanes + i) * 8;  // lanes run over [T][Hkv][D / 8]
    *reinterpret_cast<uint4*>(k + to) = ko;
    *reinterpret_cast<uint4*>(v + to) = vo;
  }
}

// ----------------------------------------------------------------------------
// Attention of new tokens over the cache
// ----------------------------------------------------------------------------
// What it cannot do without is one read of the cache (160 bytes per key and head at D = 128); what limits it beside that is
// the logic unit, which works at half the rate of the others and has to take the codes apart.  So the arrangement is around
// how few of its operations a code needs, and the pages of all sequences and heads are dealt out evenly: with units (b, kv
// head, tile of query rows) laid end to end, block i takes pages [i q, (i + 1) q) of them all, whatever the lengths are.  A
// unit that several blocks share is joined by a second kernel from at most two partial results per block.
//
// Measured (pages scattered, lengths to 8192 / two of 131072; 32/8 heads of 128): 93 and 81 us for 335 and 286 MB, 3.6 TB/s; the
// longer the cache the nearer to 4.7 TB/s (8 x as long), the copies alone take 72 and 62.  The logic unit is 52 % busy, issue
// 55 %; some 15 us are the start, the joining of warps and the second launch.  One sequence of 1000: 12 us.  Steps on the way:
// a fifth warp for the copies 144 / 118 us (it costs registers: five warps on four schedulers); products in e4m3 161 / 126; fp16
// subnormals 141 / 104; parts of a unit read with loads in flight instead of in turn 104 -> 89; a cost per unit in the sharing
// out 139 -> 97; columns folded 97 / 84 -> 92 / 79; powers of V's scales per group 92 / 80 -> 93 / 81.  More work for the warps that an SM favours (the older ones) changes nothing.
//
// A block has two pairs of warps; a pair takes every other page of a run, a warp 32 of its 64 tokens, and the pair's first
// warp keeps its pages coming through a ring of its own.  Tokens are the 16 rows, query rows (tokens x heads of the group, 8
// or 16) the columns of the products:
//   S[token][row] = sum over groups g of sc (u . q)  +  sum of min_g sum_g(q)
//   O[channel][row] += u (P sc)  +  sum(P min) per group and row
// A code in bits 0-3 or 4-7 of a half word read as fp16 is u 2^-24 or u 2^-20 (subnormal numbers, which the products take as
// they are), so one logic operation takes two codes out and two of four need no shift.  (The same nibble as an e4m3 byte is
// u 2^-9, one operation for four codes, but products of e4m3 are widened to fp16 on the same logic unit: 57 million
// instructions instead of 42.)
//   q enters as fp16, each row under a power of two and the channels of odd codes under 2^-4 of it: exact for fp16 and bf16.
//   The minima meet the group sums of q, split in two 16-bit parts, in one more product with the meta words as they are.
//   P sc is rounded to fp16 (11 bits, for bf16 caches too), under a power of two per group of 32 channels that brings the
//   largest scale of V that the run has met to 2^4 or more (weights are 4 at most).  So P sc loses bits where it is less than 2^-18 of the
//   group's largest scale, at most 2^-29 of that scale a token.  (One power for all groups took the bits from the small ones: beside
//   a group 2^17 times as large, results were off by 7 %.)  The powers lie in shared memory: in registers, of which the kernel has none
//   to spare, the first case above takes 97 us.
//   For fp16 results u - 8 stands in for u, which halves what that rounding weighs (min + 8 sc makes up for it): relative error of fp16
//   results 2.8e-4 instead of 4.8e-4, where rounding the result alone gives 2.1e-4.
constexpr float kMostDown = 2.6584559915698317e36f;  // 2^121, what scales of V are multiplied with before any was seen
constexpr float kDownLimit = 4096.f;                 // of a scale times its power: with weights up to 2^2 far inside fp16

// 1 / x of a power of two in [2^-126, 2^126].
__device__ __forceinline__ float power_rcp(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }

struct Kv4AttnParams {
  const void* q;
  const uint8_t* codes;
  const void* meta;
  const int* table;
  const int* lens;
  const int* after;  // [B] or null: tokens of each sequence that lie behind those of this cache, in other parts of it
  void* out;
  float* lse;
  float* part_o;   // [2 * blocks][rows][D]
  float* part_ml;  // [2 * blocks][rows][2]
  int* opened;     // [blocks]: the unit that the block begins and leaves to others, or -1
  int* last_block; // [B][units]: the block that ends the unit
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

// The work of a unit in pages: its own, and kUnitCost for what comes with each unit (its queries, joining four warps' results,
// writing them).  B 64, lengths to 8192: without it blocks with short sequences end at 126 us, the others at 79.
constexpr int kUnitCost = 3;
__device__ __forceinline__ int unit_work(int pages) { return pages > 0 ? pages + kUnitCost : 0; }

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
  // Pages of this unit for a block that has `work` left from here on, and what is left then.  A block that ends before the
  // first page of a unit leaves the unit to the next one.
  __device__ __forceinline__ int take(int& work, int& skip) const {
    const int head = page == 0 ? kUnitCost - skip : 0;  // `skip`: of the unit's cost lies before the block
    skip = 0;
    const int n = max(0, min(work - head, pages - page));
    work -= head + n;
    return n;
  }
};

// Work of all units, and the position `begin(total)` of it, with the part of the unit's cost that lies before the position;
// one warp, converged.  Lengths of up to 32 sequences are read once.
template <typename F>
__device__ __forceinline__ Kv4Cursor kv4_seek(const Kv4AttnParams& p, F begin, int& total, int& skip) {
  const int lane = threadIdx.x & 31;
  const int first = lane < p.B ? pages_of(kv4_len(p, lane)) : 0;
  int sum = unit_work(first);
  for (int b = lane + 32; b < p.B; b += 32) sum += unit_work(pages_of(kv4_len(p, b)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  total = sum * p.units;
  const int at = begin(total);
  int base = 0;
  for (int b0 = 0;; b0 += 32) {
    const int n = b0 == 0 ? first : b0 + lane < p.B ? pages_of(kv4_len(p, b0 + lane)) : 0;
    int upto = unit_work(n) * p.units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + upto > at);
    if (past != 0 || b0 + 32 >= p.B) {
      const int l = past != 0 ? __ffs(past) - 1 : 31;
      const int before = l == 0 ? 0 : __shfl_sync(0xffffffffu, upto, l - 1 < 0 ? 0 : l - 1);
      Kv4Cursor c;
      c.b = min(b0 + l, p.B - 1);
      c.len = kv4_len(p, c.b);
      c.pages = pages_of(c.len);
      const int in = at - base - before, each = max(unit_work(c.pages), 1);
      c.u = in / each;
      c.page = max(in % each - kUnitCost, 0);
      skip = min(in % each, kUnitCost);
      return c;
    }
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
}

// Where the share of block i begins, in work of all units.  Every block that takes part has some: between the first and the
// last block of a unit there is none without a part of it.
__device__ __forceinline__ int block_start(const Kv4AttnParams& p, int total, int i) {
  const int n = max(min(p.blocks, total), 1);
  return static_cast<int>(static_cast<long long>(total) * min(i, n) / n);
}

// The pages that a pair of warps copies: every other one of each run.
struct Kv4Fetch {
  Kv4Cursor at;  // start of the run
  int work, run, next, count;
  // to the next page from `next` on, over the ends of runs; its number (read here, looked at one step later)
  __device__ __forceinline__ int settle(const Kv4AttnParams& p, int first) {
    while (next >= run) {
      if (work <= 0) {
        run = -1;
        return -1;
      }
      at.next_unit(p);
      int skip = 0;
      run = at.take(work, skip);
      next = first;
    }
    return __ldg(p.table + static_cast<size_t>(at.b) * p.max_pages + at.page + next);
  }
};

// Codes e and e + 4 of a word (one per half word) as fp16, (u - 8) or u times 2^-24 (e even) or 2^-20 (e odd).
template <bool kCentred, int e>
__device__ __forceinline__ uint32_t codes_fp16(uint32_t w) {
  const uint32_t x = (e >= 2 ? w >> 8 : w) & (e % 2 ? 0x00f000f0u : 0x000f000fu);
  if constexpr (!kCentred) return x;
  const uint32_t eight = e % 2 ? 0x00800080u : 0x00080008u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&eight));
  return *reinterpret_cast<const uint32_t*>(&r);
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
__device__ __forceinline__ float4 add4(const float4& a, const float4& b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

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
  static constexpr int kBlocksPerSm = NG * NT <= 4 ? 4 : NG * NT <= 6 ? 3 : 2;
  static constexpr int kRing = NG <= 2 ? 4 : NG * NT <= 4 ? 2 : NG * NT <= 6 ? 2 : NG <= 4 ? 4 : 2;  // pages of a pair
  static constexpr int kOffJoin = 2 * kRing * kStageBytes;         // [2 pairs][kRows][kD] fp32
  static constexpr int kOffMl = kOffJoin + 2 * kRows * kD * 4;     // [4 warps][kRows][2]
  static constexpr int kSmemBytes = kOffMl + 4 * kRows * 2 * 4;
  static_assert(kBlocksPerSm * (kSmemBytes + 1024 + 256) <= 228 * 1024, "shared memory over budget");
};

template <typename T, int NG, int NT, bool kHalf>
__global__ void __launch_bounds__(128, Kv4Cfg<NG, NT>::kBlocksPerSm) kv4_attn_kernel(const Kv4AttnParams p) {
  using Cfg = Kv4Cfg<NG, NT>;
  constexpr int kRing = Cfg::kRing, kRows = Cfg::kRows, D = Cfg::kD;
  constexpr bool kCentred = !Pack2<T>::kIsBf16;
  // With four query rows or fewer, columns 0-3 are the rows over the first 16 of a warp's 32 tokens and columns 4-7 the same
  // rows over the others (kSets token sets per S tile): half the work from the scores to P, and a sum of two at the end.
  static_assert(!kHalf || NT == 1, "half columns are for one column tile");
  constexpr int kJ = kHalf ? 1 : 2;               // S tiles of 16 tokens that are held apart
  constexpr int kUsedRows = kHalf ? 4 : kRows;
  constexpr int kQuads = (NG + 3) / 4;
  constexpr float q_down = 1.f / 16777216.f;  // codes are u 2^-24
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bar_full[2][kRing], bar_empty[2][kRing];
  __shared__ int page_ok[2][kRing];
  __shared__ Kv4Fetch fetcher[2];
  // per warp, in shared memory because registers are short: powers of two on the scales of V per group, slopes per column
  __shared__ __align__(16) uint32_t v_down_s[4][NG];  // (as bits)
  __shared__ float slope_s[4][8 * NT];
  __shared__ int abort_flag, skip_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pair = warp >> 1, side = warp & 1;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < 2 * kRing; ++i) {
      mbar_init(&bar_full[0][i], 1);
      mbar_init(&bar_empty[0][i], 1);
    }
    mbar_fence_init();
  }
  pdl_wait();
  pdl_trigger();  // the joining kernel waits for this one's results itself
  if (threadIdx.x == 0) skip_flag = *reinterpret_cast<volatile int*>(p.status);
  volatile int* abort_p = &abort_flag;
  int total, skip;
  Kv4Cursor at = kv4_seek(p, [&](int all) { return block_start(p, all, blockIdx.x); }, total, skip);
  int work = block_start(p, total, blockIdx.x + 1) - block_start(p, total, blockIdx.x);
  __syncthreads();  // the barriers are ready
  if (skip_flag != 0) return;
  const int n_row_tiles = p.units / p.Hkv;
  uint8_t* const ring = smem + pair * (kRing * Cfg::kStageBytes);

  // ---- the copies of a pair: lane 0 of its first warp walks the same pages, kRing ahead ----
  // Its state lives in shared memory (one lane needs it), and the number of the next page is read one step early (in a register:
  // a store of it would wait for the load).
  int next_page = -1;
  bool ok = true;  // after a wait that ran out nothing is computed, but every barrier of the block is still met
  auto fetch = [&]() {  // the next page of the pair, if there is one, into the slot that has its turn
    Kv4Fetch& f = fetcher[pair];
    if (f.run < 0) return true;
    const int slot = f.count % kRing;
    if (f.count >= kRing && !mbar_wait(&bar_empty[pair][slot], (f.count / kRing - 1) & 1, abort_p)) return false;
    const bool good = next_page >= 0 && next_page < p.n_pages;
    page_ok[pair][slot] = good;
    if (good) {
      const size_t slab = static_cast<size_t>(next_page) * p.Hkv + f.at.u / n_row_tiles;
      uint8_t* dst = ring + slot * Cfg::kStageBytes;
      mbar_expect_tx(&bar_full[pair][slot], Cfg::kStageBytes);
      bulk_load_1d(smem_u32(dst), p.codes + slab * Cfg::kCodeBytes, Cfg::kCodeBytes, &bar_full[pair][slot]);
      bulk_load_1d(smem_u32(dst + Cfg::kCodeBytes), static_cast<const uint8_t*>(p.meta) + slab * Cfg::kMetaBytes,
                   Cfg::kMetaBytes, &bar_full[pair][slot]);
    } else {
      mbar_arrive(&bar_full[pair][slot]);  // a page outside the pool: its tokens are not there
    }
    ++f.count;
    f.next += 2;
    next_page = f.settle(p, pair);
    return true;
  };
  if (side == 0 && lane == 0 && work > 0) {
    Kv4Fetch& f = fetcher[pair];
    int f_skip = skip;
    f.at = at;
    f.work = work;
    f.run = at.take(f.work, f_skip);
    f.next = pair;
    f.count = 0;
    next_page = f.settle(p, pair);
    for (int i = 0; i < kRing; ++i) fetch();  // no waits yet
  }

  const int r = lane >> 2, c = lane & 3;  // S row / O row group, and column pair
  // S row r is token rt of each 8: V's loads then take tokens 0, 3, 4, 7 at a time, which lie in different banks by twos.
  const int rt = r ^ ((r >> 1) & 1);
  const int far = kHalf ? (c >> 1) * 16 : 0;           // of this lane's tokens in S
  const uint32_t first_set = r < 4 ? 0xffffffffu : 0;  // kHalf: columns (rows of the B operand's lanes) of the first set
  const int G = p.Hq / p.Hkv;
  const int n_rows = p.T * G;
  int n = 0;         // pages of the pair so far
  int opened = -1;
  while (work > 0) {
    const int run = at.take(work, skip);
    if (run == 0) {  // the share ends before the first page of this unit, or begins behind the last of the one before
      at.next_unit(p);
      continue;
    }
    const int head = at.u / n_row_tiles, row0 = at.u % n_row_tiles * kRows;
    __syncwarp();  // the last run's slopes and powers have been read
    // Query rows as the B operand: this lane holds channels [32 g + 8 c, + 8) of row r of each column tile.
    uint32_t qf[NT][NG][4], qs[NT][kQuads][2];
    float zs[NT][2];
    int lim[NT][2];  // position of the row, the last that it sees (in another part of the cache, where tokens lie behind this one)
    const int end = at.len + (p.after ? min(max(__ldg(p.after + at.b), 0), INT_MAX - at.len) : 0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + nt * 8 + (kHalf ? r & 3 : r);
      const T* src = static_cast<const T*>(p.q) + at.b * p.q_b + (row / G) * p.q_t + (head * G + row % G) * p.q_h + c * 8;
      uint4 x[NG];
      float top = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        x[g] = make_uint4(0, 0, 0, 0);
        if (row < n_rows) x[g] = __ldg(reinterpret_cast<const uint4*>(src + g * kGroup));
        const uint32_t w[4] = {x[g].x, x[g].y, x[g].z, x[g].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max3_nan(top, fabsf(Kv4Type<T>::lo(w[i])), fabsf(Kv4Type<T>::hi(w[i])));
      }
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e with which the row's largest element comes to [2^12, 2^13): what lies 2^22 below it keeps its bits
      const int ex = static_cast<int>(__float_as_uint(top) >> 23);  // 255: no number
      const int e = ex == 255 ? 0 : min(139 - ex, 126);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23), up_odd = 0.0625f * up;
#pragma unroll
      for (int k = 0; k < kQuads; ++k) qs[nt][k][0] = qs[nt][k][1] = 0;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float v0 = Kv4Type<T>::lo(x[g].x) * up, v1 = Kv4Type<T>::hi(x[g].x) * up_odd;
        const float v2 = Kv4Type<T>::lo(x[g].y) * up, v3 = Kv4Type<T>::hi(x[g].y) * up_odd;
        const float v4 = Kv4Type<T>::lo(x[g].z) * up, v5 = Kv4Type<T>::hi(x[g].z) * up_odd;
        const float v6 = Kv4Type<T>::lo(x[g].w) * up, v7 = Kv4Type<T>::hi(x[g].w) * up_odd;
        // pairs (0,4) (1,5) (2,6) (3,7): the order in which the codes of a word come out
        qf[nt][g][0] = Pack2<__half>::pack(v0, v4);
        qf[nt][g][1] = Pack2<__half>::pack(v1, v5);
        qf[nt][g][2] = Pack2<__half>::pack(v2, v6);
        qf[nt][g][3] = Pack2<__half>::pack(v3, v7);
        float sum = fmaf(16.f, (v1 + v3) + (v5 + v7), (v0 + v2) + (v4 + v6));
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (g % 4 == c) {  // beside the minimum (upper half of a meta word) the sum of q, in two parts
          sum *= q_down;
          const uint16_t hi = Kv4Type<T>::bits(sum);
          qs[nt][g / 4][0] = static_cast<uint32_t>(hi) << 16;
          qs[nt][g / 4][1] = static_cast<uint32_t>(Kv4Type<T>::bits(sum - Kv4Type<T>::value(hi))) << 16;
        }
      }
      // what brings the row's scores back, and a row that holds no number makes all of its scores none
      const float back = ex == 255 ? __uint_as_float(0x7fc00000u) : 1.f / (up * q_down);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = row0 + nt * 8 + (kHalf ? (2 * c + i) & 3 : 2 * c + i);
        zs[nt][i] = __shfl_sync(0xffffffffu, back, (2 * c + i) * 4) * (p.cap_log2 > 0.f ? p.cap_in : p.scale_log2);
        lim[nt][i] = col < n_rows ? end - p.T + col / G : -1;
        if (p.slopes && r == 0)
          slope_s[warp][nt * 8 + 2 * c + i] = col < n_rows ? __ldg(p.slopes + (p.slopes_per_batch ? static_cast<size_t>(at.b) * p.Hq : 0) + head * G + col % G) * kLog2e : 0.f;
      }
    }
    float o[NT][NG][2][4], corr[NT][NG][2], m[NT][2], l[NT][2];
    if (lane < NG) v_down_s[warp][lane] = __float_as_uint(kMostDown);
    __syncwarp();
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

    for (int i = pair; i < run; i += 2, ++n) {
      const int slot = n % kRing;
      if (side == 0 && n > 0) {  // refill the slot before this one: the partner is done with it, or nearly
        if (lane == 0 && ok) ok = fetch();
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      }
      ok = ok && mbar_wait_warp(&bar_full[pair][slot], (n / kRing) & 1, abort_p);
      if (!ok) continue;
      const uint8_t* stage = ring + slot * Cfg::kStageBytes;
      const int pos0 = (at.page + i) * kPage + side * 32;         // of the warp's first token
      const int there = page_ok[pair][slot] ? at.len - pos0 : 0;  // tokens of the warp that exist
      if (there > 0) {
        const uint8_t* kc = stage + (side * 32 + rt) * (D / 2) + c * NG * 4;
        const uint8_t* km = stage + Cfg::kCodeBytes + (side * 32 + rt) * (NG * 4);
        // ---- S, tokens pos0 + 16 j + r and + 8 ----
        float s[kJ][NT][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float sj[NT][4];
          uint32_t w0[NG], w1[NG], e0[NG], e1[NG];
          lds_words<NG>(w0, kc + j * 16 * (D / 2));
          lds_words<NG>(w1, kc + (j * 16 + 8) * (D / 2));
          lds_words<NG>(e0, km + j * 16 * (NG * 4));
          lds_words<NG>(e1, km + (j * 16 + 8) * (NG * 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) sj[nt][x] = 0.f;
#pragma unroll
          for (int k = 0; k < kQuads; ++k) {
            const bool any = k * 4 + c < NG;
            const uint32_t a = any ? *reinterpret_cast<const uint32_t*>(km + j * 16 * (NG * 4) + (k * 4 + c) * 4) : 0;
            const uint32_t b = any ? *reinterpret_cast<const uint32_t*>(km + (j * 16 + 8) * (NG * 4) + (k * 4 + c) * 4) : 0;
            const uint32_t mw[4] = {a, b, a, b};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<T>(sj[nt], mw, qs[nt][k][0], qs[nt][k][1]);
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint32_t a0[4] = {codes_fp16<false, 0>(w0[g]), codes_fp16<false, 0>(w1[g]), codes_fp16<false, 1>(w0[g]), codes_fp16<false, 1>(w1[g])};
            const uint32_t a1[4] = {codes_fp16<false, 2>(w0[g]), codes_fp16<false, 2>(w1[g]), codes_fp16<false, 3>(w0[g]), codes_fp16<false, 3>(w1[g])};
            const float sc0 = Kv4Type<T>::lo(e0[g]), sc1 = Kv4Type<T>::lo(e1[g]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float acc[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816<__half>(acc, a0, qf[nt][g][0], qf[nt][g][1]);
              mma16816<__half>(acc, a1, qf[nt][g][2], qf[nt][g][3]);
              sj[nt][0] = fmaf(acc[0], sc0, sj[nt][0]);
              sj[nt][1] = fmaf(acc[1], sc0, sj[nt][1]);
              sj[nt][2] = fmaf(acc[2], sc1, sj[nt][2]);
              sj[nt][3] = fmaf(acc[3], sc1, sj[nt][3]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              if (kHalf) s[0][nt][x] = j == 0 || c < 2 ? (j == 0 ? sj[nt][x] : s[0][nt][x]) : sj[nt][x];
              else s[j][nt][x] = sj[nt][x];
            }
        }
        // ---- scores in log2 units, masks ----
        if (p.cap_log2 > 0.f) {
#pragma unroll
          for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                s[j][nt][x] = fmaf(-2.f * p.cap_log2, fast_rcp(fast_exp2(s[j][nt][x] * zs[nt][x & 1]) + 1.f), p.cap_log2);
        } else {
#pragma unroll
          for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int x = 0; x < 4; ++x) s[j][nt][x] *= zs[nt][x & 1];
        }
        if (p.slopes) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float slope = slope_s[warp][nt * 8 + 2 * c + x];
              const float ahead = static_cast<float>(lim[nt][x] - (pos0 + far + rt));  // of the row over its first key here
#pragma unroll
              for (int j = 0; j < kJ; ++j) {
                s[j][nt][x] = fmaf(-slope, ahead - 16.f * j, s[j][nt][x]);
                s[j][nt][x + 2] = fmaf(-slope, ahead - (16.f * j + 8.f), s[j][nt][x + 2]);
              }
            }
        }
        if (there < 31 + p.T) {  // some row may not see all of them
#pragma unroll
          for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                if (far + j * 16 + rt + (x < 2 ? 0 : 8) > min(lim[nt][x & 1] - pos0, there - 1)) s[j][nt][x] = -INFINITY;
        }
        // ---- running maximum: it follows when a score is more than 2^2 above it, or is no number ----
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float hi = max_nan(s[0][nt][x], s[0][nt][x + 2]);
            if (!kHalf) hi = max3_nan(hi, s[kJ - 1][nt][x], s[kJ - 1][nt][x + 2]);
            grow = grow || !(hi - m[nt][x] <= 2.f);
          }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float top = max3_nan(m[nt][x], s[0][nt][x], s[0][nt][x + 2]);
              if (!kHalf) top = max3_nan(top, s[kJ - 1][nt][x], s[kJ - 1][nt][x + 2]);
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
        for (int j = 0; j < kJ; ++j)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              s[j][nt][x] = fast_exp2(s[j][nt][x] - m[nt][x & 1]);
              l[nt][x & 1] += s[j][nt][x];
            }
        // ---- O ----
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          const uint8_t* vm = km + (kPage + far + j * 16) * (NG * 4);
          uint32_t e0[NG], e1[NG];
          lds_words<NG>(e0, vm);
          lds_words<NG>(e1, vm + 8 * (NG * 4));
          if (there < 32) {  // tokens behind the last: their scales may be anything
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              if (far + j * 16 + rt >= there) e0[g] = 0;
              if (far + j * 16 + rt + 8 >= there) e1[g] = 0;
            }
          }
          float sc0[NG], sc1[NG], most = 0.f, v_down[NG];
          uint32_t down_bits[NG];
          lds_words<NG>(down_bits, reinterpret_cast<const uint8_t*>(v_down_s[warp]));
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            v_down[g] = __uint_as_float(down_bits[g]);
            sc0[g] = Kv4Type<T>::lo(e0[g]) * v_down[g];
            sc1[g] = Kv4Type<T>::lo(e1[g]) * v_down[g];
            most = fmaxf(fmaxf(most, fabsf(sc0[g])), fabsf(sc1[g]));
          }
          if (__any_sync(0xffffffffu, most > kDownLimit)) {
            // A group whose scales outgrew their power, as the first ones do (or that holds no number: it tells nothing about
            // the others, and changes nothing): the power is chosen again, the largest of the group comes to [2^4, 2^5).
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const float a = fabsf(Kv4Type<T>::lo(e0[g])), b = fabsf(Kv4Type<T>::lo(e1[g]));
              const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(a < INFINITY ? a : 0.f, b < INFINITY ? b : 0.f)));
              const bool change = __uint_as_float(top) * v_down[g] > kDownLimit;
              const float down = change ? __uint_as_float((258u - (top >> 23)) << 23) : v_down[g];
              const float f = down * power_rcp(v_down[g]);
              v_down[g] = down;
              if (lane == 0) v_down_s[warp][g] = __float_as_uint(down);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  o[nt][g][0][x] *= f;
                  o[nt][g][1][x] *= f;
                }
              sc0[g] = Kv4Type<T>::lo(e0[g]) * v_down[g];
              sc1[g] = Kv4Type<T>::lo(e1[g]) * v_down[g];
            }
            __syncwarp();
          }
          // P sc as the B operand, in fp16
          uint32_t pb[NT][NG][2];
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            float mn0 = Kv4Type<T>::hi(e0[g]), mn1 = Kv4Type<T>::hi(e1[g]);
            if (kCentred) {
              mn0 = fmaf(8.f, Kv4Type<T>::lo(e0[g]), mn0);
              mn1 = fmaf(8.f, Kv4Type<T>::lo(e1[g]), mn1);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              pb[nt][g][0] = transpose8x8(Pack2<__half>::pack(s[j][nt][0] * sc0[g], s[j][nt][1] * sc0[g]));
              pb[nt][g][1] = transpose8x8(Pack2<__half>::pack(s[j][nt][2] * sc1[g], s[j][nt][3] * sc1[g]));
              corr[nt][g][0] = fmaf(s[j][nt][0], mn0, fmaf(s[j][nt][2], mn1, corr[nt][g][0]));
              corr[nt][g][1] = fmaf(s[j][nt][1], mn0, fmaf(s[j][nt][3], mn1, corr[nt][g][1]));
            }
          }
#pragma unroll
          for (int set = 0; set < 3 - kJ; ++set) {  // kHalf: both token sets, each with its columns of P
            const uint8_t* vc = stage + kPage * (D / 2) + (side * 32 + (j + set) * 16 + 2 * c + (c & 1)) * (D / 2) + r * NG * 2;
            const int v_next = (c & 1) ? -(D / 2) : D / 2;  // to the odd one of the two tokens
            const uint32_t keep = set == 0 ? first_set : ~first_set;
            uint32_t t0[(NG + 1) / 2], t1[(NG + 1) / 2], t8[(NG + 1) / 2], t9[(NG + 1) / 2];
            lds_halves<NG>(t0, vc);
            lds_halves<NG>(t1, vc + v_next);
            lds_halves<NG>(t8, vc + 8 * (D / 2));
            lds_halves<NG>(t9, vc + 8 * (D / 2) + v_next);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const uint32_t lo = __byte_perm(t0[g / 2], t1[g / 2], g % 2 ? 0x7632 : 0x5410);
              const uint32_t hi = __byte_perm(t8[g / 2], t9[g / 2], g % 2 ? 0x7632 : 0x5410);
              const uint32_t a0[4] = {codes_fp16<kCentred, 0>(lo), codes_fp16<kCentred, 1>(lo), codes_fp16<kCentred, 0>(hi), codes_fp16<kCentred, 1>(hi)};
              const uint32_t a1[4] = {codes_fp16<kCentred, 2>(lo), codes_fp16<kCentred, 3>(lo), codes_fp16<kCentred, 2>(hi), codes_fp16<kCentred, 3>(hi)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint32_t b0 = kHalf ? pb[nt][g][0] & keep : pb[nt][g][0], b1 = kHalf ? pb[nt][g][1] & keep : pb[nt][g][1];
                mma16816<__half>(o[nt][g][0], a0, b0, b1);
                mma16816<__half>(o[nt][g][1], a1, b0, b1);
              }
            }
          }
        }
      }
      __syncwarp();
      if (side == 1 && lane == 0) mbar_arrive(&bar_empty[pair][slot]);
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
    __syncthreads();
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        top[nt][x] = kNoKey;
        for (int w = 0; w < 4; ++w) {
          const float* at_row = ml + (w * kRows + nt * 8 + (kHalf ? (2 * c + x) & 3 : 2 * c + x)) * 2;
          top[nt][x] = max_nan(top[nt][x], at_row[0]);
          if (kHalf) top[nt][x] = max_nan(top[nt][x], at_row[8]);
        }
      }
    for (int w = 0; w < 2; ++w) {  // in a fixed order: the same sum every time
      if (w == side) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float f = fast_exp2(m[nt][x] - top[nt][x]);
#pragma unroll
            for (int g = 0; g < NG; ++g) {  // channels 32 g + 4 r + (0..3); even codes carry 2^24, odd ones 2^20
              const float up = f * power_rcp(__uint_as_float(v_down_s[warp][g]));
              float4* dst = reinterpret_cast<float4*>(join + (pair * kRows + nt * 8 + 2 * c + x) * D + g * kGroup + 4 * r);
              const float4 old = w == 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *dst;
              const float rest = corr[nt][g][x] * f;
              *dst = make_float4(fmaf(o[nt][g][0][x] * 16777216.f, up, rest) + old.x,
                                 fmaf(o[nt][g][0][x + 2] * 1048576.f, up, rest) + old.y,
                                 fmaf(o[nt][g][1][x] * 16777216.f, up, rest) + old.z,
                                 fmaf(o[nt][g][1][x + 2] * 1048576.f, up, rest) + old.w);
            }
          }
      }
      __syncthreads();
    }
    const bool whole = at.page == 0 && run == at.pages;
    const int slot = 2 * blockIdx.x + (at.page > 0 ? 0 : 1);
    if (at.page == 0 && !whole) opened = at.b * p.units + at.u;
    if (threadIdx.x == 0 && at.page > 0 && at.page + run == at.pages)
      p.last_block[static_cast<size_t>(at.b) * p.units + at.u] = blockIdx.x;
    for (int i = threadIdx.x; i < kUsedRows * D / 8; i += 128) {
      const int row = i / (D / 8), ch = i % (D / 8) * 8, rg = row0 + row;
      if (rg >= n_rows) continue;
      float mm = kNoKey, ll = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
#pragma unroll
      for (int set = 0; set < 3 - kJ; ++set)
        for (int w = 0; w < 4; ++w) mm = max_nan(mm, ml[(w * kRows + set * 4 + row) * 2]);
#pragma unroll
      for (int set = 0; set < 3 - kJ; ++set) {
        for (int w = 0; w < 4; ++w) {
          const float* at_row = ml + (w * kRows + set * 4 + row) * 2;
          ll += at_row[1] * fast_exp2(at_row[0] - mm);
        }
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) {
          const float* from = join + (pr * kRows + set * 4 + row) * D + ch;
          x = add4(x, *reinterpret_cast<const float4*>(from));
          y = add4(y, *reinterpret_cast<const float4*>(from + 4));
        }
      }
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
    __syncthreads();  // the next run writes the same buffers
    at.next_unit(p);
  }
  if (threadIdx.x == 0) p.opened[blockIdx.x] = opened;
  // sequences without keys
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (kv4_len(p, b) > 0) continue;
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + static_cast<size_t>(b) * p.T * p.Hq * D);
    for (int i = threadIdx.x; i < p.T * p.Hq * (D / 8); i += 128) dst[i] = make_uint4(0, 0, 0, 0);
    if (p.lse)
      for (int i = threadIdx.x; i < p.T * p.Hq; i += 128) p.lse[static_cast<size_t>(b) * p.Hq * p.T + i] = -INFINITY;
  }
  if (threadIdx.x == 0 && abort_flag) {
    // Give copies that are still in flight time to land before the block's shared memory is released.
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    atomicExch(p.status, kStatusWaitTimeout);
  }
}

// Joins the partial results of the units that several blocks shared: one block per query row and block of the other kernel,
// which has something to do where that one began a unit and left it.
template <typename T>
__global__ void __launch_bounds__(128) kv4_join_kernel(const Kv4AttnParams p, int tile_rows, int used_rows) {
  pdl_wait();
  const int row = blockIdx.x % used_rows, c0 = blockIdx.x / used_rows;
  const int unit = p.opened[c0];
  if (unit < 0 || unit >= p.B * p.units) return;
  const int c1 = p.last_block[unit];
  if (c1 <= c0 || c1 >= p.blocks) return;  // the other kernel gave up
  const int n_row_tiles = p.units / p.Hkv, G = p.Hq / p.Hkv;
  const int u = unit % p.units, b = unit / p.units;
  const int rg = u % n_row_tiles * tile_rows + row;
  if (rg >= p.T * G) return;
  const int t = rg / G, h = u / n_row_tiles * G + rg % G;
  T* dst = static_cast<T*>(p.out) + ((static_cast<size_t>(b) * p.T + t) * p.Hq + h) * p.D;
  float* lse = p.lse ? p.lse + (static_cast<size_t>(b) * p.Hq + h) * p.T + t : nullptr;
  // Maximum and weights of the parts first, by all threads; then each warp sums every fourth part, loads of
  // several parts in flight (one thread per channel pair walking all parts took 29 us for 37 of them).
  __shared__ float weight[kMaxParts];
  __shared__ float4 sums[128];
  __shared__ float stat[2 * 4];
  const int parts = c1 - c0 + 1;
  auto slot = [&](int i) { return static_cast<size_t>(2 * (c0 + i) + (i == 0 ? 1 : 0)) * tile_rows + row; };
  float top = kNoKey;
  for (int i = threadIdx.x; i < parts; i += 128) top = max_nan(top, p.part_ml[slot(i) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) stat[threadIdx.x >> 5] = top;
  __syncthreads();
  top = max_nan(max_nan(stat[0], stat[1]), max_nan(stat[2], stat[3]));
  float sum = 0.f;
  for (int i = threadIdx.x; i < parts; i += 128) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot(i) * 2);
    weight[i] = fast_exp2(ml.x - top);
    sum = fmaf(ml.y, weight[i], sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) stat[4 + (threadIdx.x >> 5)] = sum;
  __syncthreads();
  sum = (stat[4] + stat[5]) + (stat[6] + stat[7]);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (lse && threadIdx.x == 0) *lse = sum == 0.f ? -INFINITY : (top + log2f(sum)) / kLog2e;
  // a warp for every fourth part, lanes of 4 channels (two rounds for head dims above 128)
  for (int d0 = 0; d0 < p.D; d0 += 128) {
    const int d = d0 + (threadIdx.x & 31) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d < p.D) {
#pragma unroll 4
      for (int i = threadIdx.x >> 5; i < parts; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p.part_o + slot(i) * p.D + d);
        const float w = weight[i];
        x = make_float4(fmaf(v.x, w, x.x), fmaf(v.y, w, x.y), fmaf(v.z, w, x.z), fmaf(v.w, w, x.w));
      }
    }
    sums[threadIdx.x] = x;
    __syncthreads();
    if (threadIdx.x < 32 && d < p.D) {
      x = add4(add4(sums[threadIdx.x], sums[threadIdx.x + 32]), add4(sums[threadIdx.x + 64], sums[threadIdx.x + 96]));
      *reinterpret_cast<uint2*>(dst + d) = make_uint2(Pack2<T>::pack(x.x * inv, x.y * inv), Pack2<T>::pack(x.z * inv, x.w * inv));
    }
    __syncthreads();
  }
}

// Column tiles of 8 query rows: two where there are more rows than one holds and registers for both.
static int kv4_tiles(int T, int G, int D) { return T * G > 8 && D <= 128 ? 2 : 1; }
static int kv4_blocks(int D, int nt) { return kSmCount * (D / kGroup * nt <= 4 ? 4 : D / kGroup * nt <= 6 ? 3 : 2); }
static bool kv4_dim(int D) { return D == 64 || D == 96 || D == 128 || D == 192 || D == 256; }

// f(a value of the 16-bit type, the number of channel groups)
template <typename F>
static int kv4_by_groups(int D, F&& f) {
  switch (D / kGroup) {
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 8: return f(std::integral_constant<int, 8>{});
    default: return RFA_ERR_UNSUPPORTED;
  }
}
template <typename F>
static int kv4_by_type(int dtype, int D, F&& f) {
  if (dtype == RFA_DTYPE_BF16) return kv4_by_groups(D, [&](auto groups) { return f(__nv_bfloat16{}, groups); });
  return kv4_by_groups(D, [&](auto groups) { return f(__half{}, groups); });
}

template <typename T, int NG, int NT, bool kHalf = false>
static int launch_kv4_attn(const Kv4AttnParams& p, cudaStream_t s) {
  using Cfg = Kv4Cfg<NG, NT>;
  auto kern = kv4_attn_kernel<T, NG, NT, kHalf>;
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
  const int rc = launch_chained(kern, static_cast<unsigned>(p.blocks), 128, Cfg::kSmemBytes, s, p);
  if (rc != RFA_OK) return rc;
  const int rows = p.T * (p.Hq / p.Hkv);
  const int used = rows < Cfg::kRows ? rows : Cfg::kRows;
  return launch_chained(kv4_join_kernel<T>, static_cast<unsigned>(p.blocks) * used, 128, 0, s, p, static_cast<int>(Cfg::kRows),
                        used);
}

// Four query rows or fewer fold the columns (see the kernel); more take one or two column tiles.
template <typename T>
static int dispatch_kv4_attn(const Kv4AttnParams& p, int nt, cudaStream_t s) {
  return kv4_by_groups(p.D, [&](auto groups) {
    constexpr int NG = decltype(groups)::value;
    if (p.T * (p.Hq / p.Hkv) <= 4) return launch_kv4_attn<T, NG, 1, true>(p, s);
    if constexpr (NG <= 4)
      if (nt == 2) return launch_kv4_attn<T, NG, 2>(p, s);
    return launch_kv4_attn<T, NG, 1>(p, s);
  });
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
  if (static_cast<long long>(T) * Hkv * (D / 8) > INT_MAX - 256) return RFA_ERR_TOO_LARGE;
  const unsigned lanes = static_cast<unsigned>(T) * Hkv * (D / 8);  // of a sequence
  const Kv4Pages p{static_cast<uint8_t*>(codes), meta, table, positions, counts, n_pages, max_pages, B, T, Hkv, D};
  const longlong3 ks = make_longlong3(k_strides[0], k_strides[1], k_strides[2]);
  const longlong3 vs = make_longlong3(v_strides[0], v_strides[1], v_strides[2]);
  const dim3 grid((lanes + 255) / 256, B < 65535 ? B : 65535);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return kv4_by_type(dtype, D, [&](auto type, auto groups) {
    using T16 = decltype(type);
    return launch_chained(kv4_append_kernel<T16, decltype(groups)::value>, grid, 256, 0, s, static_cast<const T16*>(k),
                          static_cast<const T16*>(v), p, ks, vs, lanes);
  });
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
  if (static_cast<long long>(T) * Hkv * (D / 8) > INT_MAX - 256) return RFA_ERR_TOO_LARGE;
  const unsigned lanes = static_cast<unsigned>(T) * Hkv * (D / 8);  // of a sequence
  const Kv4Pages p{static_cast<uint8_t*>(const_cast<void*>(codes)), const_cast<void*>(meta), table, positions, counts,
                   n_pages, max_pages, B, T, Hkv, D};
  const dim3 grid((lanes + 255) / 256, B < 65535 ? B : 65535);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return kv4_by_type(dtype, D, [&](auto type, auto groups) {
    using T16 = decltype(type);
    return launch_chained(kv4_gather_kernel<T16, decltype(groups)::value>, grid, 256, 0, s, static_cast<T16*>(k),
                          static_cast<T16*>(v), p, lanes);
  });
}

extern "C" size_t rfa_kv4_scratch_elems(int B, int T, int Hq, int Hkv, int D) {
  using namespace rfa;
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || !kv4_dim(D)) return 0;
  const int nt = kv4_tiles(T, Hq / Hkv, D);
  const size_t units = (static_cast<size_t>(T) * (Hq / Hkv) + 8 * nt - 1) / (8 * nt) * Hkv;
  return static_cast<size_t>(2) * kv4_blocks(D, nt) * 8 * nt * (D + 2) + kv4_blocks(D, nt) + units * B;
}

extern "C" int rfa_kv4_attn(const void* q, const long long* q_strides, const void* codes, const void* meta, int n_pages,
                            const int* table, int max_pages, const int* lens, void* out, float* lse, float* scratch, int B,
                            int T, int Hq, int Hkv, int D, int dtype, float softmax_scale, float softcap, const float* slopes,
                            int slopes_per_batch, int* status, void* stream) {
  return rfa_kv4_attn_part(q, q_strides, codes, meta, n_pages, table, max_pages, lens, nullptr, out, lse, scratch, B, T, Hq, Hkv,
                           D, dtype, softmax_scale, softcap, slopes, slopes_per_batch, status, stream);
}

extern "C" int rfa_kv4_attn_part(const void* q, const long long* q_strides, const void* codes, const void* meta, int n_pages,
                                 const int* table, int max_pages, const int* lens, const int* after, void* out, float* lse,
                                 float* scratch, int B, int T, int Hq, int Hkv, int D, int dtype, float softmax_scale,
                                 float softcap, const float* slopes, int slopes_per_batch, int* status, void* stream) {
  using namespace rfa;
  if (!q || !q_strides || !out || !scratch || !status) return RFA_ERR_INVALID_ARG;
  const int rc = kv4_check(codes, meta, n_pages, table, max_pages, lens, B, T, Hkv, D, dtype);
  if (rc != RFA_OK) return rc;
  if (Hq <= 0 || Hq % Hkv != 0) return RFA_ERR_INVALID_ARG;
  if (!(softmax_scale > 0.f) || !(softcap >= 0.f) || !scores_fit(softmax_scale, softcap))
    return RFA_ERR_INVALID_ARG;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 != 0) return RFA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(q) & 15u) || (reinterpret_cast<uintptr_t>(out) & 15u) ||
      (reinterpret_cast<uintptr_t>(scratch) & 15u) || (reinterpret_cast<uintptr_t>(lse) & 3u) ||
      (reinterpret_cast<uintptr_t>(slopes) & 3u) || (reinterpret_cast<uintptr_t>(after) & 3u))
    return RFA_ERR_INVALID_ARG;
  const int nt = kv4_tiles(T, Hq / Hkv, D), rows = 8 * nt;
  const long long row_tiles = (static_cast<long long>(T) * (Hq / Hkv) + rows - 1) / rows;
  const long long units = row_tiles * Hkv;
  if (static_cast<long long>(T) * Hq * (D / 8) > INT_MAX - 128 || units * rows * B > INT_MAX / 2) return RFA_ERR_TOO_LARGE;
  Kv4AttnParams p{};
  p.q = q;
  p.codes = static_cast<const uint8_t*>(codes);
  p.meta = meta;
  p.table = table;
  p.lens = lens;
  p.after = after;
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
  // no more blocks than pages there can be; all of the work is counted in an int
  const long long most = static_cast<long long>(max_pages) * units * B;
  if ((static_cast<long long>(max_pages) + kUnitCost) * units * B > INT_MAX) return RFA_ERR_TOO_LARGE;
  p.blocks = static_cast<int>(most < kv4_blocks(D, nt) ? most : kv4_blocks(D, nt));
  p.part_o = scratch;
  p.part_ml = scratch + static_cast<size_t>(2) * p.blocks * rows * D;
  p.opened = reinterpret_cast<int*>(p.part_ml + static_cast<size_t>(2) * p.blocks * rows * 2);
  p.last_block = p.opened + p.blocks;
  p.scale_log2 = softmax_scale * kLog2e;
  p.cap_log2 = softcap * kLog2e;
  p.cap_in = softcap > 0.f ? 2.f * softmax_scale * kLog2e / softcap : 0.f;
  p.slopes = slopes;
  p.slopes_per_batch = slopes_per_batch;
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == RFA_DTYPE_BF16 ? dispatch_kv4_attn<__nv_bfloat16>(p, nt, s) : dispatch_kv4_attn<__half>(p, nt, s);
}
