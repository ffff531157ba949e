// Rows of drafted tokens in and out of the fp16 slot cache (ec_tree.h):
//
//   qk_norm_rope: one token's q|k|v row, per head of q and k
//       y = x / sqrt(mean x^2 + eps) * gamma           (gamma null: y = x)
//       a_i = (past + depth) f_i, in 64 bits
//       (y_i, y_j) -> factor (y_i cos a_i - y_j sin a_i, y_i sin a_i + y_j cos a_i)
//     over the pairs (i, i + rot / 2) or (2 i, 2 i + 1) of the first rot
//     elements; q goes to its own rows in fp32, k and v to the cache in fp16
//     (one rounding: the cache's type).
//   tree_accept: from node 0 to the child whose token its parent's logits
//     gave, while there is one; the path's rows of the cache, in all layers,
//     move to the front of the nodes' rows.
#include "ec_device.h"
#include "ec_kernels.h"

namespace ec {

namespace {

// cos and sin of a = pos * f, times factor.  The turns a / 2 pi are formed in
// 64 bits (at a million positions their error is 2^-33 of a turn) and reduced
// to [-1/2, 1/2] there; what is left fits 32 bits.
__device__ __forceinline__ float2 rope_cs(int pos, double f, float factor) {
  const double turns = (double)pos * f * 0.15915494309189533577;
  const float x = (float)(2.0 * (turns - rint(turns)));
  float s, c;
  sincospif(x, &s, &c);
  return make_float2(c * factor, s * factor);
}

// One block per token.  A wave takes a head at a time, its elements through
// the wave's row in LDS.
constexpr int kRopeMaxHd = 512;
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormRopeArgs a) {
  __shared__ float row[4][kRopeMaxHd];
  __shared__ float2 cs[kRopeMaxHd / 2];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int b = blockIdx.x / a.t.N, i = blockIdx.x - b * a.t.N;
  const EcTreeSeq s = ec_tree_seq(&a.t, b);
  if (i >= ec_tree_rows(&a.t, s)) return;
  bool ok = ec_tree_seq_ok(&a.t, s);
  int depth = i;
  if (ok && a.t.parent) {
    bool pok;
    const int p = tree_parent(a.t, b, s.n, &pok);
    ok = pok;
    if (ok) {
      int d;
      tree_ancestors(p, &d);
      depth = __shfl(d, i, 64);
    }
  }
  ok = ok && !tree_clashes(a.t, b, s);
  const size_t m = blockIdx.x;
  float *q = a.q + m * a.ldq;
  if (!ok) {
    for (int e = t; e < a.H * a.hd; e += 256) q[e] = __builtin_nanf("");
    return;
  }
  const int half = a.rot >> 1;
  for (int e = t; e < half; e += 256) cs[e] = rope_cs(s.past + depth, a.inv_freq[e], a.factor);
  __syncthreads();
  const float *x = a.x + m * a.ldx;
  const size_t crow = ((size_t)s.slot * a.t.C + (s.past + i)) * ((size_t)a.KVH * a.hd);
  // a uniform count of rounds: the waves meet at barriers in each
  for (int h0 = 0; h0 < a.H + 2 * a.KVH; h0 += 4) {
    const int h = h0 + w;
    const bool on = h < a.H + 2 * a.KVH, isv = h >= a.H + a.KVH, isq = h < a.H;
    const float *gamma = isq ? a.q_gamma : isv ? nullptr : a.k_gamma;
    float r = 1.0f;
    if (on) {
      float sum = 0.0f;
      for (int e = lane; e < a.hd; e += 64) {
        const float v = x[(size_t)h * a.hd + e];
        row[w][e] = v;
        sum += v * v;
      }
      if (gamma) r = 1.0f / sqrtf(wave_sum(sum) / (float)a.hd + a.eps);
    }
    __syncthreads();
    if (on) {
      for (int e = lane; e < a.hd; e += 64) {
        auto at = [&](int j) {
          const float v = row[w][j];
          return gamma ? v * r * gamma[j] : v;
        };
        float y = at(e);
        if (!isv && e < a.rot) {
          const bool second = a.layout ? e & 1 : e >= half;
          const int f = a.layout ? e >> 1 : second ? e - half : e;
          const float o = at(a.layout ? e ^ 1 : second ? e - half : e + half);
          y = second ? o * cs[f].y + y * cs[f].x : y * cs[f].x - o * cs[f].y;
        }
        if (isq) q[(size_t)h * a.hd + e] = y;
        else if (isv) a.vc[crow + (size_t)(h - a.H - a.KVH) * a.hd + e] = f2h(y);
        else a.kc[crow + (size_t)(h - a.H) * a.hd + e] = f2h(y);
      }
    }
    __syncthreads();
  }
}

// The walk by one wave: a node per lane, the next node by a ballot over the
// lanes whose parent and token fit.  Returns the path's length; lane j has the
// path's node j in *node (-1 past its end).  All of it is uniform but *node.
__device__ __forceinline__ int accept_walk(const AcceptArgs &a, int b, int n, int parent, int *node, int *next) {
  const int i = threadIdx.x & 63;
  const size_t row = (size_t)b * a.t.N + i;
  const int tok = i < n ? a.token[row] : -1, smp = i < n ? a.sampled[row] : -1;
  int cur = 0, len = 1;
  *node = i == 0 ? 0 : -1;
  for (;;) {
    const int want = __shfl(smp, cur, 64);
    // a parent comes before its child, so the walk ends after at most n steps
    const uint64_t fit = __ballot(i > cur && i < n && parent == cur && tok == want && want >= 0);
    *next = want;
    if (!fit) return len;
    cur = __ffsll((unsigned long long)fit) - 1;
    if (i == len) *node = cur;
    len++;
  }
}

// One block per (layer, sequence).  Every thread owns columns of the rows and
// moves them in the path's order: row j's source is at j or behind it, and the
// sources ascend, so no row is written before it has been read.
template <typename T>
__global__ __launch_bounds__(256) void tree_accept_kernel(AcceptArgs a, int cols) {
  __shared__ int path[EC_TREE_MAX];
  __shared__ int s_len;
  const int t = threadIdx.x, layer = blockIdx.x, b = blockIdx.y;
  const EcTreeSeq s = ec_tree_seq(&a.t, b);
  if (t < 64) {
    int len = 0, node = -1, next = -1;
    if (ec_tree_seq_ok(&a.t, s) && s.n > 0) {
      bool ok;
      const int p = tree_parent(a.t, b, s.n, &ok);
      if (ok && !tree_clashes(a.t, b, s)) len = accept_walk(a, b, s.n, p, &node, &next);
    }
    path[t] = node;
    if (t == 0) s_len = len;
    if (layer == 0) {
      if (t < a.t.N) a.path[(size_t)b * a.t.N + t] = node;
      if (t == 0) {
        a.npath[b] = len;
        a.next[b] = next;
        a.new_past[b] = s.past + len;
      }
    }
  }
  __syncthreads();
  const int len = s_len;
  if (len < 2) return;
  const size_t base = (((size_t)layer * a.t.nslots + s.slot) * a.t.C + s.past) * cols;
  for (int c = t; c < 2 * cols; c += 256) {
    T *rows = c < cols ? (T *)a.kc + base + c : (T *)a.vc + base + (c - cols);
    for (int j = 1; j < len; j++)
      if (path[j] != j) rows[(size_t)j * cols] = rows[(size_t)path[j] * cols];
  }
}

}  // namespace

int qk_norm_rope_max_hd() { return kRopeMaxHd; }

hipError_t qk_norm_rope(const NormRopeArgs &a, hipStream_t st) {
  klaunch(qk_norm_rope_kernel, dim3(a.t.B * a.t.N), dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t tree_accept(const AcceptArgs &a, hipStream_t st) {
  klaunch(tree_accept_kernel<uint16_t>, dim3(a.layers, a.t.B), dim3(256), 0, st, a, a.kv);
  return hipGetLastError();
}

}  // namespace ec
