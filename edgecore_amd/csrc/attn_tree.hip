// Attention of drafted tokens over the fp16 slot cache (ec_tree.h): node i of
// a sequence sees the cached text, within its window, and of the nodes its
// ancestors and itself, within the window as well:
//
//   x_p = scale q . k_p        p < past, or p - past an ancestor of i or i
//   o   = sum_p e^(x_p - m) v_p / sum_p e^(x_p - m),  m = max_p x_p
//
// in fp32 (a row that sees nothing gives 0).  What a row does not see does not
// reach it, finite or not.
#include <cfloat>

#include "ec_device.h"
#include "ec_kernels.h"

namespace ec {

namespace {

// The form for any head size and alignment: one block per (node, head), tiles
// of 256 positions, a position per thread for the scores and an element of the
// head per thread for the sums, with the running maximum and sum.
constexpr int kTreeMaxHd = 512;
__global__ __launch_bounds__(256) void attn_tree_any_kernel(TreeAttnArgs a) {
  __shared__ float q[kTreeMaxHd], p_s[256], red[4];
  __shared__ float part[256];
  const int t = threadIdx.x;
  const int h = blockIdx.y, b = blockIdx.x / a.t.N, i = blockIdx.x - b * a.t.N;
  const int kvh = h / (a.H / a.KVH);
  const EcTreeSeq s = ec_tree_seq(&a.t, b);
  if (i >= ec_tree_rows(&a.t, s)) return;
  const size_t m = blockIdx.x;
  float *out = a.out + m * a.ldo + (size_t)h * a.hd;
  bool ok = ec_tree_seq_ok(&a.t, s);
  uint64_t see = 0;
  int depth = 0, mydepth = 0;
  if (ok) {
    const int p = tree_parent(a.t, b, s.n, &ok);
    if (ok) {
      const uint64_t anc = tree_ancestors(p, &depth);
      see = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(anc >> 32), i, 64) << 32) |
            (uint32_t)__shfl((int)(uint32_t)anc, i, 64);
      mydepth = __shfl(depth, i, 64);
      // the nodes within the window
      if (a.window) see &= __ballot(mydepth - depth < a.window);
    }
  }
  if (!ok) {
    for (int e = t; e < a.hd; e += 256) out[e] = __builtin_nanf("");
    return;
  }
  const int lo = a.window && s.past + mydepth >= a.window ? min(s.past + mydepth - a.window + 1, s.past) : 0;
  const int end = s.past + s.n;
  const size_t kv = (size_t)a.KVH * a.hd, base = (size_t)s.slot * a.t.C * kv + (size_t)kvh * a.hd;
  for (int e = t; e < a.hd; e += 256) q[e] = a.q[m * a.ldq + (size_t)h * a.hd + e];
  __syncthreads();
  // elements per round and the groups of positions that share one
  const int width = a.hd < 256 ? a.hd : 256, groups = 256 / width;
  const int g = t / width, d0 = t - g * width;
  float mx = -FLT_MAX, sum = 0.0f, acc[kTreeMaxHd / 256] = {0.0f, 0.0f};
  for (int p0 = lo; p0 < end; p0 += 256) {
    const int p = p0 + t;
    bool on = p < s.past;
    if (!on && p < end) on = (see >> (p - s.past)) & 1;
    float x = 0.0f;
    if (on) {
      const uint16_t *k = a.kc + base + (size_t)p * kv;
      for (int e = 0; e < a.hd; e++) x = __builtin_fmaf(q[e], h2f(k[e]), x);
      x *= a.scale;
    }
    const float mt = fmaxf(mx, block_max256(on ? x : -FLT_MAX, red));
    const float e = on ? expf(x - mt) : 0.0f, back = expf(mx - mt);
    p_s[t] = on ? e : -1.0f;  // a sign for what is not seen
    sum = sum * back + block_sum256(e, red);
    mx = mt;
    const int n = min(256, end - p0);
    for (int r = 0, d = d0; r < kTreeMaxHd / 256; r++, d += 256) {
      acc[r] *= back;
      if (g < groups && d < a.hd)
        for (int j = g; j < n; j += groups)
          if (p_s[j] >= 0.0f) acc[r] = __builtin_fmaf(p_s[j], h2f(a.vc[base + (size_t)(p0 + j) * kv + d]), acc[r]);
    }
    __syncthreads();
  }
  const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
  for (int r = 0, d = d0; r < kTreeMaxHd / 256; r++, d += 256) {
    part[t] = acc[r];
    __syncthreads();
    if (g == 0 && d < a.hd) {
      float o = 0.0f;
      for (int j = 0; j < groups; j++) o += part[j * width + d0];
      out[d] = o * inv;
    }
    __syncthreads();
  }
}

}  // namespace

int attention_tree_max_hd() { return kTreeMaxHd; }

size_t attention_tree_workspace(const TreeAttnArgs &) { return 0; }

hipError_t attention_tree(const TreeAttnArgs &a, hipStream_t st) {
  klaunch(attn_tree_any_kernel, dim3(a.t.B * a.t.N, a.H), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ec
