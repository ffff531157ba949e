// Sampling from given random numbers, one token per row of logits:
//
//   w_i = e^((l_i - max) / T) in 64 bits; tokens in the order of their logits,
//   largest first, equal ones by index; of these
//     the first top_k;
//     those whose sum of w before them is below top_p of the sum;
//     those with w >= min_p (the first always stays);
//   the token is the first whose running sum passes u times the sum.
//
// T not above 0: the largest logit.  NaN counts as -inf, -inf is never drawn, a
// row of nothing else gives -1.
//
// Sums are of w in steps of 2^-44 in 64-bit integers: the order of the additions
// does not change them, so a row gives the same token every time (2^18 tokens of
// w = 1 stay below 2^62; a sum of 150000 is off by about 2^-27 of one token's
// largest weight at the very most, by 2^-36 where the roundings fall at random).
//
// Nothing is sorted.  A place in the order is a border: the keys above a key, and
// the first of those that equal it (Border).  Three launches:
//
//   sample_top_kernel: per chunk of 4096 logits the largest (with its index) and
//     the smallest;
//   sample_bins_kernel: per chunk the logits by value into 512 bins between the
//     row's largest and smallest (or 32 T below, where w rounds to 0): their
//     number and sum of w per bin, and their indices in the bins' order;
//   sample_pick_kernel: a block per row adds the chunks' bins up and finds the
//     bin of each border; that bin's elements come from their chunks into LDS,
//     where the border is found by fixing the key's bits from the top, 8 at a
//     time, from a histogram of those that agree so far.
//
// A bin of more than kCap elements (what a block's LDS has room for) is searched by the
// same steps over the whole row, one block reading it 4 to 7 times a border.  Rows that
// get there: most logits within 1/512 of the row's span, or equal ones.  One or 16 rows of
// 151936 that spread by 0.01 beside one logit of 20, at a temperature of 10, take 0.33 ms
// (0.02 with a spread of 2) and 0.6 with top-p; of equal logits with top-p 2.3, as every
// one of them adds to the same count.
//
// Rows of 151936: one with top-k and top-p takes 3 + 5.2 + 9.5 us in the three kernels, 16
// nuclei 4.4 + 9.9 + 16.1, 128 mixed ones 15 + 37 + 18.4.  Chunks of 8192 gave the same
// within 2%, with twice the room for a row's tail.
#include <type_traits>

#include "ec_device.h"
#include "ec_expf.h"
#include "ec_kernels.h"

namespace ec {

namespace {

typedef unsigned long long u64;

constexpr double kOne = 17592186044416.0;  // 2^44: w = 1
constexpr int kChunk = 4096, kBins = 512, kCap = 4096, kSorted = 256, kFew = 32, kBinThreads = 512, kTopThreads = 256;
constexpr int kMaxChunks = (1 << 18) / kChunk;  // one per lane of a wave
static_assert(kMaxChunks <= 64 && kChunk <= 65535, "chunks per lane, counts in 16 bits");
constexpr float kNats = 32.0f;  // e^-32 is 0 in steps of 2^-44

// an order-preserving image of the logit; NaN as -inf, -0 as +0
__device__ __forceinline__ uint32_t key_of(float v) {
  v = v != v ? -__builtin_inff() : v + 0.0f;
  const uint32_t u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
constexpr uint32_t kNegInf = 0x007FFFFFu, kPosInf = 0xFF800000u;  // key_of(-inf), key_of(inf)

// e^x in steps of 2^-44, rounded to nearest, for x <= 0: x = k ln2 / 32 + r with
// |r| <= ln2 / 64, 2^(k / 32) from the table (ec_exp2_32, a copy in LDS) and e^r by
// its series to r^5 (r^6 / 720 is 2^-49 of it).  The method, exponent and table index
// from the low bits of x * 32 / ln2 + a large constant, is that of ec_expf.h, which names
// its source.  About 15 instructions where the library's exp and conversion take 60.
__device__ __forceinline__ u64 exp_steps(double x, const uint64_t *tab) {
  constexpr double kInv = 46.16624130844683;                // 32 / ln2
  constexpr double kStep = 0x1.62e42fefa39efp-6;            // ln2 / 32 (k of it off by 2^-48 at most)
  constexpr double kShift = 0x1.8p52;
  x = fmax(x, -40.0);
  double kd = __builtin_fma(x, kInv, kShift);
  const uint64_t ki = __builtin_bit_cast(uint64_t, kd);
  kd -= kShift;
  const double r = __builtin_fma(-kd, kStep, x);
  double p = __builtin_fma(r, 1.0 / 120.0, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  // the table's entries leave out the exponent that k's low bits add; 2^44 on top
  const double s = __builtin_bit_cast(double, tab[ki % 32] + (ki << 47) + (44ull << 52));
  return __builtin_bit_cast(uint64_t, __builtin_fma(s, p, kShift)) - __builtin_bit_cast(uint64_t, kShift);
}

// What a row's weights and bins are made of.  A logit's bin is number (max - l) *
// per of the 512, the last one open (in 32 bits: every step of it keeps the order).
struct Scale {
  uint32_t top;  // key of the largest
  double max, neg_inv_t;
  float max32, per;
};
__device__ __forceinline__ Scale scale_of(uint32_t top, uint32_t low, float T) {
  Scale b;
  b.top = top;
  b.max32 = key_value(top);
  b.max = (double)b.max32;
  b.neg_inv_t = -1.0 / (double)T;  // T is 2^-149 at least
  const float span = fminf(b.max32 - key_value(low), kNats * T);
  b.per = span > 0.0f ? fminf(kBins / span, 0x1p127f) : 0.0f;
  return b;
}
// Of a value (-inf weighs nothing).  Where the largest is infinite it alone weighs.
template <bool INF>
__device__ __forceinline__ u64 weight_of(const Scale &b, float v, const uint64_t *tab) {
  if (INF) return v == __builtin_inff() ? (u64)kOne : 0;
  return exp_steps((b.max - (double)v) * b.neg_inv_t, tab);
}
template <bool INF>
__device__ __forceinline__ int bin_at(const Scale &b, float v) {
  if (INF) return v == __builtin_inff() ? 0 : kBins - 1;
  return (int)fminf((b.max32 - v) * b.per, (float)(kBins - 1));
}
__device__ __forceinline__ u64 weight(const Scale &b, float v, const uint64_t *tab) {
  return b.top == kPosInf ? weight_of<true>(b, v, tab) : weight_of<false>(b, v, tab);
}
__device__ __forceinline__ int bin_of(const Scale &b, float v) {
  return b.top == kPosInf ? bin_at<true>(b, v) : bin_at<false>(b, v);
}

// scratch of a batch of rows
struct Scratch {
  u64 *sum;         // [rows][chunks][kBins]
  u64 *top;         // [rows][chunks] key << 32 | ~index of the largest
  uint32_t *low;    // [rows][chunks] key of the smallest above -inf
  uint32_t *live;   // [rows][chunks] elements above -inf
  uint16_t *start;  // [rows][chunks][kBins]: a bin's first place in the chunk's order
  uint16_t *at;     // [rows][chunks][kChunk]: indices within the chunk in the bins' order
};
size_t scratch_row(int nb) { return (size_t)nb * (8 + 4 + 4 + kBins * (8 + 2) + kChunk * 2); }
Scratch scratch_of(void *p, int rows, int nb) {
  const size_t n = (size_t)rows * nb;
  Scratch s;
  char *c = (char *)p;
  s.sum = (u64 *)c, c += n * kBins * 8;
  s.top = (u64 *)c, c += n * 8;
  s.low = (uint32_t *)c, c += n * 4;
  s.live = (uint32_t *)c, c += n * 4;
  s.start = (uint16_t *)c, c += n * kBins * 2;
  s.at = (uint16_t *)c;
  return s;
}

// f of all lanes' values, by DPP: within the row of 16 (lane pairs, quads, then mirrored
// halves and rows), then the rows' by lane
template <class T, class F>
__device__ __forceinline__ T wave_join(T v, F f) {
  v = f(v, dpp_mov<0xB1>(v));
  v = f(v, dpp_mov<0x4E>(v));
  v = f(v, dpp_mov<0x141>(v));
  v = f(v, dpp_mov<0x140>(v));
  return f(f(readlane(v, 0), readlane(v, 16)), f(readlane(v, 32), readlane(v, 48)));
}
__device__ __forceinline__ u64 wave_max64(u64 v) {
  return wave_join(v, [](u64 x, u64 y) { return x > y ? x : y; });
}
__device__ __forceinline__ uint32_t wave_max32(uint32_t v) {
  return wave_join(v, [](uint32_t x, uint32_t y) { return max(x, y); });
}
__device__ __forceinline__ uint32_t wave_min32(uint32_t v) {
  return wave_join(v, [](uint32_t x, uint32_t y) { return min(x, y); });
}

// Bound by memory: 128 rows of 151936, 78 MB, in 15.4 us (5.0 TB/s).  One row is a launch
// and one round of loads.
__global__ __launch_bounds__(kTopThreads) void sample_top_kernel(SampleArgs a, Scratch s, int row0) {
  __shared__ u64 s_top[kTopThreads / 64];
  __shared__ uint32_t s_low[kTopThreads / 64];
  const int t = threadIdx.x, c0 = blockIdx.x * kChunk, nb = gridDim.x;
  const float *l = a.logits + (size_t)(row0 + blockIdx.y) * a.ld;
  uint32_t low = ~0u, big = 0;
  int at = 0;
  float v[kChunk / kTopThreads];
#pragma unroll
  for (int j = 0; j < kChunk / kTopThreads; j++) v[j] = l[min(c0 + t + kTopThreads * j, a.V - 1)];
#pragma unroll
  for (int j = 0; j < kChunk / kTopThreads; j++) {
    const uint32_t k = key_of(v[j]);
    if (k > big) big = k, at = j;  // the first of equal ones
    if (k > kNegInf) low = min(low, k);
  }
  u64 top = ((u64)big << 32) | (uint32_t)~min(c0 + t + kTopThreads * at, a.V - 1);
  top = wave_max64(top);
  low = wave_min32(low);
  if ((t & 63) == 0) {
    s_top[t >> 6] = top;
    s_low[t >> 6] = low;
  }
  __syncthreads();
  if (t == 0) {
    for (int i = 1; i < kTopThreads / 64; i++) {
      top = s_top[i] > top ? s_top[i] : top;
      low = min(low, s_low[i]);
    }
    s.top[(size_t)blockIdx.y * nb + blockIdx.x] = top;
    s.low[(size_t)blockIdx.y * nb + blockIdx.x] = low;
  }
}

// the row's largest (key << 32 | ~index) and smallest, by every wave: read, then joined
struct Ends {
  u64 top;
  uint32_t low;
};
__device__ __forceinline__ Ends read_ends(const Scratch &s, int row, int nb) {
  const size_t at = (size_t)row * nb + min((int)(threadIdx.x & 63), nb - 1);
  return Ends{s.top[at], s.low[at]};
}
__device__ __forceinline__ Ends row_ends(Ends e) { return Ends{wave_max64(e.top), wave_min32(e.low)}; }

__device__ __forceinline__ float temp_of(const SampleArgs &a, int row) { return a.temp ? a.temp[row] : 1.0f; }

// the keys alone
struct KeyEnds {
  uint32_t top, low;
};
__device__ __forceinline__ KeyEnds key_ends(const Scratch &s, int row, int nb) {
  const size_t at = (size_t)row * nb + min((int)(threadIdx.x & 63), nb - 1);
  return KeyEnds{wave_max32(((const uint32_t *)s.top)[2 * at + 1]), wave_min32(s.low[at])};
}

// In straight code: what is not to be counted goes to a spare bin of its lane, whose
// place is behind the chunk's indices (37 us for 128 rows of 151936; with branches 43).
// Bound by the vector ALU: about 45 instructions an element, 13 of them in 64 bits.
__global__ __launch_bounds__(kBinThreads) void sample_bins_kernel(SampleArgs a, Scratch s, int row0) {
  constexpr int PT = kChunk / kBinThreads, kSpare = 64;
  __shared__ u64 s_sum[kBins + kSpare];
  __shared__ int s_cnt[kBins + kSpare], s_at[kBins + kSpare], s_wave[kBinThreads / 64];
  __shared__ __attribute__((aligned(4))) uint16_t s_idx[kChunk + PT * kBinThreads / 64];
  __shared__ uint64_t s_tab[32];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, row = blockIdx.y, c0 = blockIdx.x * kChunk, nb = gridDim.x;
  const float *l = a.logits + (size_t)(row0 + row) * a.ld + c0;
  const int n = min(a.V - c0, kChunk);
  float v[PT];
  if (n == kChunk) {
#pragma unroll
    for (int j = 0; j < PT; j++) v[j] = (l + kBinThreads * j)[t];
  } else {
#pragma unroll
    for (int j = 0; j < PT; j++) {
      const int at = kBinThreads * j + t;
      v[j] = l[min(at, n - 1)];
      if (at >= n) v[j] = -__builtin_inff();
    }
  }
  const float T = temp_of(a, row0 + row);
  const KeyEnds ends = key_ends(s, row, nb);
  if (!(T > 0.0f) || ends.top == kNegInf) return;  // the largest logit, or none: nothing to weigh
  const Scale sc = scale_of(ends.top, ends.low, T);
  static_assert(kBins == kBinThreads && kSpare <= 64, "a bin per thread");
  s_sum[t] = 0;
  s_cnt[t] = 0;
  if (t < kSpare) {
    s_cnt[kBins + t] = 0;
    s_at[kBins + t] = kChunk;
  }
  if (t < 32) s_tab[t] = ec_exp2_32[t];
  __syncthreads();
  int bin[PT], place[PT];
  auto weigh = [&](auto inf) {
    u64 x[PT];
#pragma unroll
    for (int j = 0; j < PT; j++) {
      const int b = bin_at<decltype(inf)::value>(sc, v[j]);
      x[j] = weight_of<decltype(inf)::value>(sc, v[j], s_tab);
      bin[j] = v[j] > -__builtin_inff() ? b : kBins + lane;
    }
#pragma unroll
    for (int j = 0; j < PT; j++) {
      place[j] = atomicAdd(&s_cnt[bin[j]], 1);
      atomicAdd(&s_sum[x[j] ? bin[j] : kBins + lane], x[j]);
    }
  };
  if (ends.top == kPosInf) weigh(std::true_type{});
  else weigh(std::false_type{});
  __syncthreads();
  const int mine = s_cnt[t], upto = (int)wave_scan((uint32_t)mine);
  if (lane == 63) s_wave[w] = upto;
  __syncthreads();
  int first = upto - mine, total = 0;
  for (int i = 0; i < kBinThreads / 64; i++) {
    if (i < w) first += s_wave[i];
    total += s_wave[i];
  }
  s_at[t] = first;
  const size_t ch = (size_t)row * nb + blockIdx.x;
  s.sum[ch * kBins + t] = s_sum[t];
  s.start[ch * kBins + t] = (uint16_t)first;
  if (t == 0) s.live[ch] = (uint32_t)total;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PT; j++) s_idx[s_at[bin[j]] + place[j]] = (uint16_t)(t + kBinThreads * j);
  __syncthreads();
  // two indices a store (one past the end at most, in the chunk's own room)
  for (int i = 2 * t; i < total; i += 2 * kBinThreads)
    *reinterpret_cast<uint32_t *>(s.at + ch * kChunk + i) = *reinterpret_cast<const uint32_t *>(s_idx + i);
}

// A block's LDS for a row.
struct Pick {
  // the row's bins: number and sum of w of the elements before a bin
  int cnt[kBins + 1];
  u64 sum[kBins + 1];
  __attribute__((aligned(4))) uint16_t start[kMaxChunks][kBins];  // a bin's first place in each chunk's order
  int live[64];
  // the elements of a run of bins, in any order; up to kSorted of them in order
  // instead, with the sum of w up to each
  uint32_t key[kCap], idx[kCap];
  u64 w[kCap], upto[kSorted];
  int seg[64], first[64];
  // a step's histogram, and what it found
  int hc[256];
  u64 hw[256];
  int found, found_cnt, found_equal, few, few_at[kFew];
  u64 found_sum;
  u64 wave_w[16];
  uint32_t differ;
  uint64_t tab[32];
};

// One row, and which of its bins are in LDS: lo .. hi, n elements.
struct Row {
  const float *l;
  const Scratch *s;
  size_t ch0;  // the row's first chunk in the scratch
  int V, nb;
  Scale sc;
  int lo, hi, n;
};

// Up to kSorted listed elements into their order, with running sums: four threads
// count the elements before each.
__device__ void sort_list(Pick &k, const Row &r) {
  const int t = threadIdx.x, i = t >> 2;
  auto order = [&](int j) { return ((u64)k.key[j] << 32) | ~k.idx[j]; };
  uint32_t key = 0, idx = 0;
  u64 w = 0;
  int before = 0;
  if (i < r.n) {
    key = k.key[i], idx = k.idx[i], w = k.w[i];
    const u64 mine = order(i);
    // eight reads a round (behind the list, but in the arrays: not counted)
    for (int j0 = t & 3; j0 < r.n; j0 += 32) {
      u64 o[8];
#pragma unroll
      for (int j = 0; j < 8; j++) o[j] = order(j0 + 4 * j);
#pragma unroll
      for (int j = 0; j < 8; j++) before += j0 + 4 * j < r.n && o[j] > mine;
    }
  }
  before += dpp_mov<0xB1>(before);
  before += dpp_mov<0x4E>(before);
  __syncthreads();
  if (i < r.n && (t & 3) == 0) k.key[before] = key, k.idx[before] = idx, k.w[before] = w;
  __syncthreads();
  static_assert(kSorted == 256, "four a lane");
  if (t < 64) {
    u64 v[4], all = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      v[j] = 4 * t + j < r.n ? k.w[4 * t + j] : 0;
      all += v[j];
    }
    u64 x = k.sum[r.lo] + wave_scan(all) - all;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x += v[j];
      k.upto[4 * t + j] = x;
    }
  }
  __syncthreads();
}

// Bin b's elements into LDS, with those of all bins before it where they are few
// (the next border is among them then); false where b's are too many.
__device__ bool load_bin(Pick &k, Row &r, int b) {
  const int t = threadIdx.x, lane = t & 63;
  if (r.lo <= b && b <= r.hi) return true;
  if (k.cnt[b + 1] - k.cnt[b] > kCap) return false;
  r.lo = k.cnt[b + 1] <= kSorted ? 0 : b;
  r.hi = b;
  r.n = k.cnt[b + 1] - k.cnt[r.lo];
  __syncthreads();
  if (t < 64) {
    const int c = min(lane, r.nb - 1), from = k.start[c][r.lo];
    const int m = lane < r.nb ? (b + 1 < kBins ? k.start[c][b + 1] : k.live[c]) - from : 0;
    k.seg[lane] = (int)wave_scan((uint32_t)m) - m;
    k.first[lane] = from;
    if (t == 0) k.differ = 0;
  }
  __syncthreads();
  uint32_t d = 0, first = 0;
  for (int i = t; i < r.n; i += 1024) {
    int c = 0;  // the last chunk whose elements start at i or before it
#pragma unroll
    for (int step = 32; step > 0; step >>= 1)
      if (c + step < r.nb && k.seg[c + step] <= i) c += step;
    const int at = c * kChunk + r.s->at[(r.ch0 + c) * kChunk + k.first[c] + (i - k.seg[c])];
    const float v = r.l[at];
    const uint32_t key = key_of(v);
    k.key[i] = key;
    k.idx[i] = (uint32_t)at;
    k.w[i] = weight(r.sc, v, k.tab);
    if (i == t) first = key;
    d |= key ^ first;
  }
  if (r.n <= kSorted) {
    __syncthreads();
    sort_list(k, r);
    return true;
  }
  // bits in which any two keys differ: from the wave's first key, and that from the list's
  const uint32_t lead = (uint32_t)readlane((int)first, 0);
  if (t < r.n) d |= first ^ lead;
  __syncthreads();
  if ((t & ~63) < r.n) d |= lead ^ k.key[0];
  d = wave_join(d, [](uint32_t x, uint32_t y) { return x | y; });
  if (lane == 0 && d) atomicOr(&k.differ, d);
  __syncthreads();
  return true;
}

// A key with what is before it in the order: their number and sum of w; and how
// many have it.
struct Border {
  uint32_t key;
  int equal, above;
  u64 sum;
};

// Fixes the bits of a key below `bits`, 8 at a time, until the element is found at
// which the running count reaches want (BY_SUM false) or the running sum passes
// target, over the elements that each(f) hands to f(key, weight) and whose upper
// bits are prefix's.  cnt, sum: what comes before them all.  It ends when all bits are
// fixed or at most `few` elements agree in those that are (bits: how many are not).
template <bool BY_SUM, class Each>
__device__ Border fix_bits(Pick &k, const Each &each, uint32_t prefix, int &bits, int cnt, u64 sum, int want, u64 target,
                           int few = 0) {
  const int t = threadIdx.x, lane = t & 63;
  int equal = few + 1;
  while (bits > 0 && equal > few) {
    const int take = bits < 8 ? bits : 8, shift = bits - take;
    __syncthreads();
    if (t < 256) {
      k.hc[t] = 0;
      k.hw[t] = 0;
    }
    __syncthreads();
    each([&](uint32_t key, u64 w) {
      if (bits < 32 && (key >> bits) != prefix) return;
      const int bin = (key >> shift) & ((1 << take) - 1);
      atomicAdd(&k.hc[bin], 1);
      if (w) atomicAdd(&k.hw[bin], w);
    });
    __syncthreads();
    if (t < 64) {
      // four bins a lane, the largest first
      int c[4], call = 0;
      u64 w[4], wall = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        c[j] = k.hc[255 - 4 * lane - j];
        w[j] = k.hw[255 - 4 * lane - j];
        call += c[j];
        wall += w[j];
      }
      int cb = cnt + (int)wave_scan((uint32_t)call) - call;
      u64 wb = sum + wave_scan(wall) - wall;
      int hit = -1, hc = 0, he = 0;
      u64 hw = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (hit < 0 && (BY_SUM ? wb + w[j] > target : cb + c[j] >= want)) hit = 255 - 4 * lane - j, hc = cb, hw = wb, he = c[j];
        cb += c[j];
        wb += w[j];
      }
      const uint64_t m = __ballot(hit >= 0);
      if (m && lane == __ffsll((unsigned long long)m) - 1) {
        k.found = hit;
        k.found_cnt = hc;
        k.found_sum = hw;
        k.found_equal = he;
      }
    }
    __syncthreads();
    prefix = (prefix << take) | (uint32_t)k.found;
    cnt = k.found_cnt;
    sum = k.found_sum;
    equal = k.found_equal;
    bits = shift;
  }
  return Border{prefix, equal, cnt, sum};
}

// An element of the row: the sum of w up to it and itself, its weight, and (TOKEN)
// its index.
struct Place {
  u64 upto, w;
  int token;
};

// The element among at.equal (kFew at most) of the list whose keys agree with at.key
// above `bits`: a wave compares each with all.
template <bool BY_SUM>
__device__ Place find_few(Pick &k, const Row &r, const Border &at, int bits, int want, u64 target) {
  const int t = threadIdx.x;
  __syncthreads();
  if (t == 0) k.few = 0;
  __syncthreads();
  for (int i = t; i < r.n; i += 1024)
    if ((k.key[i] >> bits) == at.key) k.few_at[atomicAdd(&k.few, 1)] = i;
  __syncthreads();
  if (t < 64) {
    const int i = t < at.equal ? k.few_at[t] : -1;
    const u64 mine = i < 0 ? 0 : ((u64)k.key[i] << 32) | ~k.idx[i], w = i < 0 ? 0 : k.w[i];
    int cnt = at.above;
    u64 sum = at.sum;
    for (int j = 0; j < at.equal; j++)
      if (readlane(mine, j) > mine) cnt++, sum += readlane(w, j);
    if (i >= 0 && (BY_SUM ? sum <= target && sum + w > target : cnt + 1 == want)) {
      k.found = i;
      k.found_sum = sum + w;
    }
  }
  __syncthreads();
  const int i = k.found;
  return Place{k.found_sum, k.w[i], (int)k.idx[i]};
}

// The element at which the running count reaches want, or the running sum passes
// target (there is one).
template <bool BY_SUM, bool TOKEN>
__device__ Place find_place(Pick &k, Row &r, int want, u64 target) {
  const int t = threadIdx.x;
  __syncthreads();
  if (t < kBins) {
    const bool hit = BY_SUM ? k.sum[t] <= target && k.sum[t + 1] > target : k.cnt[t] < want && k.cnt[t + 1] >= want;
    if (hit) k.found = t;
  }
  __syncthreads();
  const int b = k.found;
  Place p{0, 0, 0};
  const bool listed = load_bin(k, r, b);
  if (listed && r.n <= kSorted) {
    __syncthreads();
    if (t < r.n) {
      const u64 before = t ? k.upto[t - 1] : k.sum[r.lo];
      if (BY_SUM ? before <= target && k.upto[t] > target : k.cnt[r.lo] + t + 1 == want) k.found = t;
    }
    __syncthreads();
    const int i = k.found;
    p.upto = k.upto[i];
    p.w = k.w[i];
    p.token = (int)k.idx[i];
    return p;
  }
  Border at;
  if (listed) {
    int bits = k.differ ? 32 - __clz(k.differ) : 0;
    if (bits == 0) {
      at = Border{k.key[0], r.n, k.cnt[b], k.sum[b]};
    } else {
      at = fix_bits<BY_SUM>(
          k,
          [&](auto f) {
            for (int i = t; i < r.n; i += 1024) f(k.key[i], k.w[i]);
          },
          bits < 32 ? k.key[0] >> bits : 0, bits, k.cnt[b], k.sum[b], want, target, kFew);
      if (at.equal <= kFew) return find_few<BY_SUM>(k, r, at, bits, want, target);
    }
  } else {
    int bits = 32;
    at = fix_bits<BY_SUM>(
        k,
        [&](auto f) {
          for (int i = t; i < r.V; i += 1024) {
            const float v = r.l[i];
            if (v > -__builtin_inff() && bin_of(r.sc, v) == b) f(key_of(v), weight(r.sc, v, k.tab));
          }
        },
        0, bits, k.cnt[b], k.sum[b], want, target);
  }
  // of the elements with the key, the number of those before this one
  p.w = weight(r.sc, key_value(at.key), k.tab);
  int ties = want - at.above - 1;
  if (BY_SUM) {
    const u64 before = p.w ? (target - at.sum) / p.w : 0;
    ties = before < (u64)at.equal ? (int)before : at.equal - 1;
  }
  p.upto = at.sum + (u64)(ties + 1) * p.w;
  if (!TOKEN) return p;
  // number `ties` by index: the largest complement of the index but for so many
  constexpr int kIdxBits = 18;
  constexpr uint32_t kIdx = (1u << kIdxBits) - 1;
  static_assert(kMaxChunks * kChunk <= 1 << kIdxBits, "an index's bits");
  int bits = kIdxBits;
  const Border i = fix_bits<false>(
      k,
      [&](auto f) {
        if (listed) {
          for (int j = t; j < r.n; j += 1024)
            if (k.key[j] == at.key) f(~k.idx[j] & kIdx, 0);
        } else {
          for (int j = t; j < r.V; j += 1024)
            if (key_of(r.l[j]) == at.key) f(~(uint32_t)j & kIdx, 0);
        }
      },
      0, bits, 0, 0, ties + 1, 0);
  p.token = (int)(~i.key & kIdx);
  return p;
}

// the smallest key whose weight reaches min_p (at most the largest one's)
__device__ uint32_t least_key(const Scale &sc, double min_p) {
  auto reaches = [&](uint32_t c) {
    return c >= sc.top || (c > kNegInf && sc.top != kPosInf && exp((sc.max - (double)key_value(c)) * sc.neg_inv_t) >= min_p);
  };
  // near max + T log min_p: 64 keys at a time
  const int lane = threadIdx.x & 63;
  const uint32_t g = key_of((float)(sc.max - log(min_p) / sc.neg_inv_t));
  if (g > kNegInf + 64 && g < sc.top) {
    const uint64_t m = __ballot(reaches(g - 32 + lane));
    if (m && !(m & 1)) return g - 32 + (uint32_t)__ffsll((unsigned long long)m) - 1;
  }
  uint32_t thr = 0;
  for (int bit = 31; bit >= 0; bit--)
    if (!reaches(thr | ((1u << bit) - 1u))) thr |= 1u << bit;
  return thr;
}

// Bound by latency, a block per row: the ends 1.5 us, the chunks' bins 2.1, then for each
// border not among the elements already there its bin 2.1 (two dependent reads past
// the L2) and the search: 0.4 to 0.8 in a sorted list, else 0.9 a round of 8 bits and 0.5
// for the few that are left (all 32 bits in rounds took 18.1 us for the nuclei).
__global__ __launch_bounds__(1024) void sample_pick_kernel(SampleArgs a, Scratch s, int row0, int nb) {
  __shared__ Pick k;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, row = row0 + blockIdx.x;
  // The chunks' bins: two of them a thread, every fourth chunk, kRead chunks read at
  // a time (the chunks' blocks ran on other XCDs, so every read goes past this one's
  // L2), and the row's ends before them.
  constexpr int kRead = 10, kGroups = 1024 / (kBins / 2);
  const int b2 = 2 * (t & (kBins / 2 - 1)), group = t / (kBins / 2);
  const size_t ch0 = (size_t)blockIdx.x * nb;
  typedef u64 u64x2 __attribute__((ext_vector_type(2)));
  u64x2 x[kRead];
  uint32_t y[kRead];
  auto read = [&](int c0) {
#pragma unroll
    for (int i = 0; i < kRead; i++) {
      const size_t ch = ch0 + min(c0 + kGroups * i, nb - 1);
      x[i] = *reinterpret_cast<const u64x2 *>(s.sum + ch * kBins + b2);
      y[i] = *reinterpret_cast<const uint32_t *>(s.start + ch * kBins + b2);
    }
  };
  const Ends part = read_ends(s, blockIdx.x, nb);
  const float T = temp_of(a, row);
  read(group);
  const Ends ends = row_ends(part);
  const uint32_t tk = (uint32_t)(ends.top >> 32);
  if (tk == kNegInf || !(T > 0.0f)) {
    if (t == 0) {
      const bool none = tk == kNegInf;
      a.token[row] = none ? -1 : (int)~(uint32_t)ends.top;
      if (a.prob) a.prob[row] = none ? 0.0f : 1.0f;
    }
    return;
  }
  Row r;
  r.l = a.logits + (size_t)row * a.ld;
  r.s = &s;
  r.ch0 = ch0;
  r.V = a.V;
  r.nb = nb;
  r.sc = scale_of(tk, ends.low, T);
  r.lo = 0;
  r.hi = -1;
  r.n = 0;
  const int top_k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;
  const double u = a.u[row];

  // Added up.  A bin's first place, added over the chunks, is the number of elements
  // before it.
  {
    u64 sum0 = 0, sum1 = 0;
    int before0 = 0, before1 = 0;
    for (int c0 = group; c0 < nb; c0 += kGroups * kRead) {
      if (c0 != group) read(c0);
#pragma unroll
      for (int i = 0; i < kRead; i++)
        if (c0 + kGroups * i < nb) {
          sum0 += x[i].x;
          sum1 += x[i].y;
          before0 += (int)(y[i] & 0xFFFFu);
          before1 += (int)(y[i] >> 16);
          *reinterpret_cast<uint32_t *>(&k.start[c0 + kGroups * i][b2]) = y[i];
        }
    }
    // the groups' sums in the place of the elements, which come later
    u64(*part_sum)[kBins] = reinterpret_cast<u64(*)[kBins]>(k.w);
    int(*part_cnt)[kBins] = reinterpret_cast<int(*)[kBins]>(k.key);
    static_assert(kGroups * kBins <= kCap, "room for them");
    part_sum[group][b2] = sum0;
    part_sum[group][b2 + 1] = sum1;
    part_cnt[group][b2] = before0;
    part_cnt[group][b2 + 1] = before1;
    if (t < 64) {
      const int n = t < nb ? (int)s.live[r.ch0 + t] : 0;
      k.live[t] = n;
      const int all = (int)wave_scan((uint32_t)n);
      if (t == 63) k.cnt[kBins] = all;
    }
    if (t < 32) k.tab[t] = ec_exp2_32[t];
    __syncthreads();
    u64 sum = 0, upto = 0;
    int before = 0;
    if (t < kBins) {
#pragma unroll
      for (int g = 0; g < kGroups; g++) {
        sum += part_sum[g][t];
        before += part_cnt[g][t];
      }
      upto = wave_scan(sum);
      if (lane == 63) k.wave_w[w] = upto;
    }
    __syncthreads();
    if (t < kBins) {
      for (int i = 0; i < w; i++) upto += k.wave_w[i];
      k.sum[t + 1] = upto;
      k.cnt[t] = before;
      if (t == 0) k.sum[0] = 0;
    }
    __syncthreads();
  }
  // the sum of those that stay
  u64 total = k.sum[kBins];
  if (top_k > 0 && top_k < k.cnt[kBins]) total = find_place<false, false>(k, r, top_k, 0).upto;
  if (top_p < 1.0f) {
    // up to the element at which the sum reaches top_p of it: passes ceil(top_p sum) - 1
    const double at = ceil((double)top_p * (double)total) - 1.0;
    u64 target = at > 0.0 ? (u64)at : 0;
    if (target >= total) target = total - 1;
    total = find_place<true, false>(k, r, 0, target).upto;
  }
  if (min_p > 0.0f) {
    // those from the least key on, as far as they are among those that stay
    const uint32_t thr = least_key(r.sc, (double)min_p);
    const int b = bin_of(r.sc, key_value(thr));
    u64 sum = 0;
    int from = b;
    if (load_bin(k, r, b)) {
      for (int i = t; i < r.n; i += 1024)
        if (k.key[i] >= thr) sum += k.w[i];
      from = r.lo;
    } else {
      for (int i = t; i < r.V; i += 1024) {
        const float v = r.l[i];
        if (key_of(v) >= thr && bin_of(r.sc, v) == b) sum += weight(r.sc, v, k.tab);
      }
    }
    sum = wave_scan(sum);
    __syncthreads();
    if (lane == 63) k.wave_w[w] = sum;
    __syncthreads();
    sum = k.sum[from];
    for (int i = 0; i < 16; i++) sum += k.wave_w[i];
    total = sum < total ? sum : total;
  }
  // the draw: running sum above u total
  const double at = u * (double)total;
  u64 target = at > 0.0 ? at < (double)total ? (u64)at : total - 1 : u == u ? 0 : total - 1;
  if (target >= total) target = total - 1;
  const Place p = find_place<true, true>(k, r, 0, target);
  if (t == 0) {
    a.token[row] = p.token;
    if (a.prob) a.prob[row] = (float)((double)p.w / (double)total);
  }
}

int chunks_of(int V) { return (V + kChunk - 1) / kChunk; }

}  // namespace

// rows of a batch: some rounds of chunks for every CU, a scratch of about 110 MB at most
int sample_batch(int V) { return 8192 / chunks_of(V); }

size_t sample_workspace(int rows, int V) {
  const int n = sample_batch(V);
  return scratch_row(chunks_of(V)) * (rows < n ? rows : n);
}

hipError_t sample_top(const SampleArgs &a, void *ws, int row0, int n, hipStream_t st) {
  const int nb = chunks_of(a.V);
  klaunch(sample_top_kernel, dim3(nb, n), dim3(kTopThreads), 0, st, a, scratch_of(ws, n, nb), row0);
  return hipGetLastError();
}

hipError_t sample_bins(const SampleArgs &a, void *ws, int row0, int n, hipStream_t st) {
  const int nb = chunks_of(a.V);
  klaunch(sample_bins_kernel, dim3(nb, n), dim3(kBinThreads), 0, st, a, scratch_of(ws, n, nb), row0);
  return hipGetLastError();
}

hipError_t sample_pick(const SampleArgs &a, void *ws, int row0, int n, hipStream_t st) {
  const int nb = chunks_of(a.V);
  klaunch(sample_pick_kernel, dim3(n), dim3(1024), 0, st, a, scratch_of(ws, n, nb), row0, nb);
  return hipGetLastError();
}

}  // namespace ec
