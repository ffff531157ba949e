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
// Nothing is sorted.  A place in the order is a border (Border below): the keys
// above a key, and the first of those that equal it.  It is found by fixing the
// key's bits from the top, 8 at a time, from a histogram of counts or of sums
// over the elements that agree in the bits so far.  Sums are of w in steps of
// 2^-44 in 64-bit integers: the order of the additions does not change them, so
// a row gives the same token every time (2^18 tokens of w = 1 stay below 2^62;
// a sum of 150000 is off by about 2^-27 of one token's largest weight at the
// very most, by 2^-36 where the roundings fall at random).
#include "ec_device.h"
#include "ec_kernels.h"

namespace ec {

namespace {

typedef unsigned long long u64;

constexpr double kOne = 17592186044416.0;  // 2^44: w = 1

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

// a logit's weight in steps of 2^-44
__device__ __forceinline__ u64 weight(uint32_t key, uint32_t top, double inv_t) {
  if (key == top) return (u64)kOne;
  if (key <= kNegInf || top == kPosInf) return 0;
  const double x = ((double)key_value(key) - (double)key_value(top)) * inv_t;
  return (u64)__double2ll_rn(exp(x) * kOne);
}

// The elements before a place in the order: those with a key above `key`, and
// the first `ties` of the `equal` ones that have it; `sum`: the weights of the
// keys above.
struct Border {
  uint32_t key;
  int ties, above;
  u64 sum;
};

struct RowBlock {
  u64 hist[256];
  int count[256];
  u64 scan_sum;
  int scan_bin, scan_count, found;
};

// The border of the place where the running count reaches `want` elements
// (BY_SUM false), or where the running sum passes `target` (true), within the
// elements before `lim`.  Every thread of the block calls it.
template <bool BY_SUM>
__device__ Border find_border(RowBlock &s, const float *l, int V, uint32_t top, double inv_t, int want, double target,
                              const Border &lim) {
  uint32_t prefix = 0;
  u64 sum = 0;
  int cnt = 0, equal = 0;
  const int t = threadIdx.x;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (t < 256) {
      s.hist[t] = 0;
      s.count[t] = 0;
    }
    __syncthreads();
    for (int i = t; i < V; i += 1024) {
      const uint32_t k = key_of(l[i]);
      if (k < lim.key || (k == lim.key && !lim.ties) || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
      const int bin = (k >> shift) & 255;
      atomicAdd(&s.count[bin], 1);
      atomicAdd(&s.hist[bin], weight(k, top, inv_t));
    }
    __syncthreads();
    if (t == 0) {
      int bin = 255, c = cnt, last = -1;
      u64 w = sum;
      int at_c = cnt;
      u64 at_w = sum;
      for (; bin >= 0; bin--) {
        if (BY_SUM ? s.hist[bin] != 0 : s.count[bin] != 0) {
          last = bin;
          at_c = c;
          at_w = w;
          c += s.count[bin];
          w += s.hist[bin];
          if (BY_SUM ? (double)w > target : c >= want) break;
        }
      }
      // never passed: the last element
      s.scan_bin = last;
      s.scan_count = at_c;
      s.scan_sum = at_w;
      s.found = last < 0 ? 0 : s.count[last];
    }
    __syncthreads();
    prefix = (prefix << 8) | (uint32_t)s.scan_bin;
    cnt = s.scan_count;
    sum = s.scan_sum;
    equal = s.found;
    __syncthreads();
  }
  if (prefix == lim.key) equal = min(equal, lim.ties);
  Border b;
  b.key = prefix;
  b.above = cnt;
  b.sum = sum;
  if (!BY_SUM) {
    b.ties = min(equal, want - cnt);
  } else {
    const u64 w = weight(prefix, top, inv_t);
    const double r = w ? floor((target - (double)sum) / (double)w) : (double)equal;
    b.ties = r < 0.0 ? 0 : r < (double)equal ? (int)r : equal - 1;  // elements of this key before the one that passes
  }
  return b;
}

__global__ __launch_bounds__(1024) void sample_rows_kernel(SampleArgs a) {
  __shared__ RowBlock s;
  __shared__ uint32_t s_max[16];
  __shared__ u64 s_sum[16];
  __shared__ int s_cnt[16], s_token;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, row = blockIdx.x;
  const float *l = a.logits + (size_t)row * a.ld;
  uint32_t mx = 0;
  for (int i = t; i < a.V; i += 1024) mx = max(mx, key_of(l[i]));
  for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
  if (lane == 0) s_max[w] = mx;
  __syncthreads();
  uint32_t top = s_max[0];
  for (int j = 1; j < 16; j++) top = max(top, s_max[j]);
  const float T = a.temp ? a.temp[row] : 1.0f;
  const bool none = top == kNegInf, greedy = !(T > 0.0f);
  Border at{top, 0, 0, 0};
  double p = 1.0;
  if (!none && !greedy) {
    const double inv_t = 1.0 / (double)T;
    // what stays: at first all but -inf
    Border keep{kNegInf, 0, 0, 0};
    const int k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < a.V) keep = find_border<false>(s, l, a.V, top, inv_t, k, 0.0, keep);
    auto sum_of = [&](const Border &b) {
      u64 sum = 0;
      for (int i = t; i < a.V; i += 1024) {
        const uint32_t key = key_of(l[i]);
        if (key > b.key) sum += weight(key, top, inv_t);
      }
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
      __syncthreads();
      if (lane == 0) s_sum[w] = sum;
      __syncthreads();
      sum = 0;
      for (int j = 0; j < 16; j++) sum += s_sum[j];
      return sum + (u64)b.ties * weight(b.key, top, inv_t);
    };
    u64 total = sum_of(keep);
    const float tp = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? a.min_p[row] : 0.0f;
    if (tp < 1.0f) {
      // the element at which the sum reaches top_p of it is the last one that stays
      const double target = (double)tp * (double)total;
      // of the elements up to the one that passes the target that one stays too, if it starts below it
      keep = find_border<true>(s, l, a.V, top, inv_t, 0, target, keep);
      const u64 wb = weight(keep.key, top, inv_t);
      if ((double)(keep.sum + (u64)keep.ties * wb) < target || keep.ties + keep.above == 0) keep.ties++;
      total = sum_of(keep);
    }
    if (mp > 0.0f) {
      // the smallest key whose weight reaches min_p, by its bits
      uint32_t thr = 0;
      for (int bit = 31; bit >= 0; bit--) {
        const uint32_t c = thr | ((1u << bit) - 1u);  // the largest key with this bit clear
        double x = ((double)key_value(c) - (double)key_value(top)) * inv_t;
        const bool reaches = c >= top || (c > kNegInf && exp(x) >= (double)mp);  // min_p above 1: the largest alone
        if (!reaches) thr |= 1u << bit;
      }
      thr = min(thr, top);
      if (thr > keep.key) {
        keep = Border{thr - 1, 0, 0, 0};
        total = sum_of(keep);
      }
    }
    at = find_border<true>(s, l, a.V, top, inv_t, 0, a.u[row] * (double)total, keep);
    p = (double)weight(at.key, top, inv_t) / (double)total;
  }
  // the element number at.ties of those that have the key, by index
  int left = at.ties;
  if (t == 0) s_token = -1;
  for (int i0 = 0; i0 < a.V; i0 += 1024) {
    const int i = i0 + t;
    const bool hit = i < a.V && key_of(l[i]) == at.key;
    const uint64_t m = __ballot(hit);
    __syncthreads();
    if (lane == 0) s_cnt[w] = __popcll(m);
    __syncthreads();
    int before = 0, all = 0;
    for (int j = 0; j < 16; j++) {
      if (j < w) before += s_cnt[j];
      all += s_cnt[j];
    }
    if (hit && before + __popcll(m & ((1ull << lane) - 1)) == left) s_token = i;
    if (left < all) break;
    left -= all;
  }
  __syncthreads();
  if (t == 0) {
    a.token[row] = none ? -1 : s_token;
    if (a.prob) a.prob[row] = none ? 0.0f : (float)p;
  }
}

}  // namespace

hipError_t sample_rows(const SampleArgs &a, hipStream_t st) {
  klaunch(sample_rows_kernel, dim3(a.rows), dim3(1024), 0, st, a);
  return hipGetLastError();
}

}  // namespace ec
