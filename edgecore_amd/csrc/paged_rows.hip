// Rows in and out of a paged cache (ec_pages.h) whose elements are 16 or 8 bits
// wide, 8-bit ones with a scale per row and KV head:
//
//   paged_append: one token's q|k|v row, per head of q and k
//       y = x / sqrt(mean x^2 + eps) * gamma           (gamma null: y = x)
//       a_i = (past + i) f_i, in 64 bits
//       (y_i, y_j) -> factor (y_i cos a_i - y_j sin a_i, y_i sin a_i + y_j cos a_i)
//     over the pairs (i, i + rot / 2) or (2 i, 2 i + 1) of the first rot
//     elements; q goes to its own rows in fp32, k and v to the pages: in fp16, or
//       s = max |y| / Q, the next fp16 from there up,  c = y / s to the nearest
//     with Q = 127 (int8) or 448 (e4m3).  A row stands for the fp16 values c s.
//   paged_read: the values that rows of the pages stand for, into the fp16 slot cache.
//
// k is computed in 64 bits: a code is a step of 1/127 of a row's largest, so that a
// key near the border of two would show 32-bit roundings in all that is read.
#include "ec_device.h"
#include "ec_kernels.h"
#include "paged_cache.h"

namespace ec {

namespace {

// What a row's threads know of it: its sequence, its position, its place in the pages.
struct PagedRow {
  bool mine, ok;  // a sequence's row; of one that takes part, with a page
  int pos;
  uint32_t row;  // of KV head 0; KV head h's is page * h further on
};
__device__ __forceinline__ PagedRow paged_row(const EcPageBatch &t, int m) {
  PagedRow r{false, false, 0, 0};
  const int b = page_seq_of(t, m);
  if (b < 0) return r;
  const EcPageSeq s = ec_page_seq(&t, b);
  r.mine = ec_page_seq_mine(&t, s) && m >= s.start && m - s.start < s.n;
  if (!r.mine || !ec_page_seq_ok(&t, s, EC_PAGES_ROWS)) return r;
  r.pos = s.past + (m - s.start);
  bool bad = false;
  r.row = page_row(t, page_id(t, b, r.pos), r.pos, 0, &bad);
  r.ok = !bad;
  return r;
}

// cos and sin of a = pos * f, times factor, in 64 bits
__device__ __forceinline__ double2 rope_cs64(int pos, double f, double factor) {
  const double turns = (double)pos * f * 0.15915494309189533577;
  double s, c;
  sincospi(2.0 * (turns - rint(turns)), &s, &c);
  return make_double2(c * factor, s * factor);
}

// The form for any head size and alignment: one block per token, a wave a head at
// a time, its elements through the wave's row in LDS.
constexpr int kAppendMaxHd = 512;
__global__ __launch_bounds__(256) void paged_append_any_kernel(PagedAppendArgs a) {
  __shared__ double row[4][kAppendMaxHd];
  __shared__ double2 cs[kAppendMaxHd / 2];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, hd = a.c.hd, KVH = a.c.t.KVH;
  const PagedRow rr = paged_row(a.c.t, blockIdx.x);
  if (!rr.mine) return;
  const size_t m = blockIdx.x;
  float *q = a.q + m * a.ldq;
  if (!rr.ok) {
    for (int e = t; e < a.H * hd; e += 256) q[e] = __builtin_nanf("");
    return;
  }
  const int half = a.rot >> 1;
  for (int e = t; e < half; e += 256) cs[e] = rope_cs64(rr.pos, a.inv_freq[e], a.factor);
  __syncthreads();
  const float *x = a.x + m * a.ldx;
  // a uniform count of rounds: the waves meet at barriers in each
  for (int h0 = 0; h0 < a.H + 2 * KVH; h0 += 4) {
    const int h = h0 + w;
    const bool on = h < a.H + 2 * KVH, isv = h >= a.H + KVH, isq = h < a.H;
    const float *gamma = isq ? a.q_gamma : isv ? nullptr : a.k_gamma;
    double r = 1.0;
    if (on) {
      double sum = 0.0;
      for (int e = lane; e < hd; e += 64) {
        const double v = x[(size_t)h * hd + e];
        row[w][e] = v;
        sum = __builtin_fma(v, v, sum);
      }
      if (gamma) r = 1.0 / sqrt(wave_sum(sum) / hd + a.eps);
    }
    __syncthreads();
    if (on) {
      double y[kAppendMaxHd / 64], top = 0.0;
      bool nan = false;
#pragma unroll
      for (int i = 0; i < kAppendMaxHd / 64; i++) {
        const int e = lane + 64 * i;
        if (e >= hd) break;
        auto at = [&](int j) {
          const double v = row[w][j];
          return gamma ? v * r * gamma[j] : v;
        };
        y[i] = at(e);
        if (!isv && e < a.rot) {
          const bool second = a.layout ? e & 1 : e >= half;
          const int f = a.layout ? e >> 1 : second ? e - half : e;
          const double o = at(a.layout ? e ^ 1 : second ? e - half : e + half);
          y[i] = second ? o * cs[f].y + y[i] * cs[f].x : y[i] * cs[f].x - o * cs[f].y;
        }
        top = fmax(top, fabs(y[i]));
        nan |= y[i] != y[i];
      }
      const int kvh = isv ? h - a.H - KVH : h - a.H;
      const size_t at = rr.row + (size_t)kvh * a.c.t.page;
      uint16_t sc = 0;
      if (!isq && a.c.type != CACHE_F16) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmax(top, __shfl_xor(top, o, 64));
        sc = __ballot(nan) ? 0x7E00 : cache_scale(top, a.c.type);
        if (lane == 0) (isv ? a.c.vs : a.c.ks)[at] = sc;
      }
#pragma unroll
      for (int i = 0; i < kAppendMaxHd / 64; i++) {
        const int e = lane + 64 * i;
        if (e >= hd) break;
        if (isq) q[(size_t)h * hd + e] = (float)y[i];
        else cache_store(isv ? a.c.v : a.c.k, a.c.type, at * hd + e, y[i], sc);
      }
    }
    __syncthreads();
  }
}

// whether sequence b's rows of its slot share one with those of an earlier sequence
__device__ __forceinline__ bool read_clashes(const PagedReadArgs &a, int b, EcTreeSeq s) {
  if (!a.slot) return false;
  bool hit = false;
  for (int c = threadIdx.x & 63; c < b; c += 64) {
    const EcTreeSeq o{a.slot[c], a.to ? a.to[c] : 0, a.count[c]};
    hit |= ec_tree_seq_ok(&a.t, o) && ec_tree_clash(s, o);
  }
  return __ballot(hit) != 0;
}

// One block per 16 rows of a sequence, an element a thread.
constexpr int kReadRows = 16;
__global__ __launch_bounds__(256) void paged_read_any_kernel(PagedReadArgs a) {
  const int b = blockIdx.y, t = threadIdx.x, hd = a.c.hd, KVH = a.c.t.KVH;
  const EcTreeSeq s{a.slot ? a.slot[b] : b, a.to ? a.to[b] : 0, a.count[b]};
  const int first = a.first[b];
  if (!ec_tree_seq_ok(&a.t, s) || first < 0 || s.n > a.c.t.rows || first > a.c.t.rows - s.n || read_clashes(a, b, s)) return;
  for (int i = blockIdx.x * kReadRows; i < min(s.n, (int)(blockIdx.x + 1) * kReadRows); i++) {
    const int p = first + i;
    bool bad = false;
    const size_t row = page_row(a.c.t, page_id(a.c.t, b, p), p, 0, &bad);
    const size_t to = ((size_t)s.slot * a.t.C + (s.past + i)) * ((size_t)KVH * hd);
    for (int e = t; e < KVH * hd; e += 256) {
      const int h = e / hd;
      const size_t at = row + (size_t)h * a.c.t.page;
      a.kc[to + e] = bad ? 0x7E00 : cache_value(a.c.k, a.c.ks, a.c.type, at, hd, e - h * hd);
      a.vc[to + e] = bad ? 0x7E00 : cache_value(a.c.v, a.c.vs, a.c.type, at, hd, e - h * hd);
    }
  }
}

}  // namespace

int paged_append_max_hd() { return kAppendMaxHd; }

hipError_t paged_append(const PagedAppendArgs &a, hipStream_t st) {
  klaunch(paged_append_any_kernel, dim3(a.c.t.M), dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t paged_read(const PagedReadArgs &a, hipStream_t st) {
  klaunch(paged_read_any_kernel, dim3((a.t.N + kReadRows - 1) / kReadRows, a.t.B), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ec
