// Attention of new tokens over a paged cache (ec_pages.h, paged_cache.h): the token at
// position t of its text sees the positions p <= t, with a window those with p > t -
// window and the first `sinks`:
//
//   x_p = scale q . k_p
//   o   = sum_p e^(x_p - m) v_p / sum_p e^(x_p - m),  m = max_p x_p
//
// in fp32.  What a token does not see does not reach it, finite or not.
#include <cfloat>

#include "ec_device.h"
#include "ec_kernels.h"
#include "paged_cache.h"

namespace ec {

namespace {

// The form for any head size and alignment: one block per (token, head), tiles
// of 256 positions, a position per thread for the scores and an element of the
// head per thread for the sums, with the running maximum and sum.
constexpr int kPagedMaxHd = 512;
__global__ __launch_bounds__(256) void attn_paged_any_kernel(PagedAttnArgs a) {
  __shared__ float q[kPagedMaxHd], p_s[256], red[4];
  __shared__ float part[256];
  __shared__ uint32_t row_s[256];
  const int t = threadIdx.x, hd = a.c.hd;
  const int h = blockIdx.y, m = blockIdx.x, kvh = h / (a.H / a.c.t.KVH);
  const int b = page_seq_of(a.c.t, m);
  if (b < 0) return;
  const EcPageSeq s = ec_page_seq(&a.c.t, b);
  if (!ec_page_seq_mine(&a.c.t, s) || m < s.start || m - s.start >= s.n) return;
  float *out = a.out + (size_t)m * a.ldo + (size_t)h * hd;
  bool bad = !ec_page_seq_ok(&a.c.t, s, a.max_past);
  const int pos = s.past + (m - s.start), lo = a.window && pos >= a.window ? pos - a.window + 1 : 0;
  for (int e = t; e < hd; e += 256) q[e] = a.q[(size_t)m * a.ldq + (size_t)h * hd + e];
  __syncthreads();
  // elements per round and the groups of positions that share one
  const int width = hd < 256 ? hd : 256, groups = 256 / width;
  const int g = t / width, d0 = t - g * width;
  float mx = -FLT_MAX, sum = 0.0f, acc[kPagedMaxHd / 256] = {0.0f, 0.0f};
  const int sinks = min(a.sinks, lo), seen = bad ? 0 : sinks + (pos - lo + 1);
  for (int i0 = 0; i0 < seen; i0 += 256) {
    const int i = i0 + t, p = i < sinks ? i : i - sinks + lo;
    const bool on = i < seen;
    float x = 0.0f;
    if (on) {
      const uint32_t row = page_row(a.c.t, page_id(a.c.t, b, p), p, kvh, &bad);
      row_s[t] = row;
      for (int e = 0; e < hd; e++) x = __builtin_fmaf(q[e], h2f(cache_value(a.c.k, a.c.ks, a.c.type, row, hd, e)), x);
      x *= a.scale;
    }
    const float mt = fmaxf(mx, block_max256(on ? x : -FLT_MAX, red));
    const float e = on ? expf(x - mt) : 0.0f, back = expf(mx - mt);
    p_s[t] = e;
    sum = sum * back + block_sum256(e, red);
    mx = mt;
    const int n = min(256, seen - i0);
    for (int r = 0, d = d0; r < kPagedMaxHd / 256; r++, d += 256) {
      acc[r] *= back;
      if (g < groups && d < hd)
        for (int j = g; j < n; j += groups)
          acc[r] = __builtin_fmaf(p_s[j], h2f(cache_value(a.c.v, a.c.vs, a.c.type, row_s[j], hd, d)), acc[r]);
    }
    __syncthreads();
  }
  const float inv = __syncthreads_or(bad) ? __builtin_nanf("") : 1.0f / sum;
  for (int r = 0, d = d0; r < kPagedMaxHd / 256; r++, d += 256) {
    part[t] = acc[r];
    __syncthreads();
    if (g == 0 && d < hd) {
      float o = 0.0f;
      for (int j = 0; j < groups; j++) o += part[j * width + d0];
      out[d] = o * inv;
    }
    __syncthreads();
  }
}

}  // namespace

int attention_paged_max_hd() { return kPagedMaxHd; }

hipError_t attention_paged(const PagedAttnArgs &a, hipStream_t st) {
  klaunch(attn_paged_any_kernel, dim3(a.c.t.M, a.H), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ec
