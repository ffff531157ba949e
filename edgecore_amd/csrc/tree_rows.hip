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

// What a row's threads know of it: its cache row, and the position it stands at.
struct RopeRow {
  bool mine, ok;  // a node's row; of a sequence that takes part
  int pos;
  size_t crow;  // first element in the caches
};
__device__ __forceinline__ RopeRow rope_row(const NormRopeArgs &a, int m) {
  const int b = m / a.t.N, i = m - b * a.t.N;
  const EcTreeSeq s = ec_tree_seq(&a.t, b);
  RopeRow r;
  r.mine = i < ec_tree_rows(&a.t, s);
  r.ok = r.mine && ec_tree_seq_ok(&a.t, s);
  int depth = i;
  if (r.ok && a.t.parent) {
    const int p = tree_parent(tree_parent_read(a.t, b), s.n, &r.ok);
    if (r.ok) {
      int d;
      tree_ancestors(p, &d);
      depth = __shfl(d, i, 64);
    }
  }
  r.ok = r.ok && !tree_clashes(a.t, b, s);
  r.pos = r.ok ? s.past + depth : 0;
  r.crow = r.ok ? ((size_t)s.slot * a.t.C + (s.past + i)) * ((size_t)a.KVH * a.hd) : 0;
  return r;
}

// The form for any head size and alignment: one block per token, a wave a head at
// a time, its elements through the wave's row in LDS.  Three prompts of up to 333 rows,
// 10 + 2 x 5 heads of 80, take 9.7 us here, 6.3 in the form below.  Bound by latency:
// three barriers for every four heads, stores of 2 bytes.
constexpr int kRopeMaxHd = 512;
__global__ __launch_bounds__(256) void qk_norm_rope_any_kernel(NormRopeArgs a) {
  __shared__ float row[4][kRopeMaxHd];
  __shared__ float2 cs[kRopeMaxHd / 2];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const RopeRow rr = rope_row(a, blockIdx.x);
  if (!rr.mine) return;
  const size_t m = blockIdx.x;
  float *q = a.q + m * a.ldq;
  if (!rr.ok) {
    for (int e = t; e < a.H * a.hd; e += 256) q[e] = __builtin_nanf("");
    return;
  }
  const int half = a.rot >> 1;
  for (int e = t; e < half; e += 256) cs[e] = rope_cs(rr.pos, a.inv_freq[e], a.factor);
  __syncthreads();
  const float *x = a.x + m * a.ldx;
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
        else if (isv) a.vc[rr.crow + (size_t)(h - a.H - a.KVH) * a.hd + e] = f2h(y);
        else a.kc[rr.crow + (size_t)(h - a.H) * a.hd + e] = f2h(y);
      }
    }
    __syncthreads();
  }
}

// The form for head sizes that are multiples of 4 up to 256 and rows of whole
// 16-byte chunks: a block per row, LPH lanes a head, four elements a lane, the next
// head's on their way while one is worked on.  The norm's sum goes over the head's
// lanes; a pair's other element is in the same lane (layout 1) or in lane +- rot / 8,
// which holds its four (layout 0, rot a multiple of 8).  Every element is read and
// written once: 2048 rows of 12 + 2 x 2 heads of 128, 27.5 MB, take 8.7 us (3.2 TB/s;
// a copy of as much 5.4), 128 rows of 14 + 2 x 2 of 64 take 5.2, a launch and the
// chain before the first store (a sequence's numbers, its tree, the angles), which
// blocks of their own overlap best: with two rows a block the prompt's rows took 3%
// longer, with four 24%, with four heads of a lane ahead 14%.  The form for any size
// takes 17.3 and 8.2.
template <int LPH>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormRopeArgs a) {
  __shared__ float4 cs[64];  // four cosines, then four sines, of four frequencies
  __shared__ RopeRow info;
  const int t = threadIdx.x, li = t % LPH, e = 4 * li, heads = a.H + 2 * a.KVH, groups = blockDim.x / LPH;
  const size_t m = blockIdx.x;
  const int half = a.rot >> 1;
  const bool in = e < a.hd;
  const float *row = a.x + m * a.ldx + e;
  auto read = [&](int h) {
    float4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (in && h < heads) x = *reinterpret_cast<const float4 *>(row + (size_t)h * a.hd);
    return x;
  };
  int h = t / LPH;
  float4 next = read(h);
  double f = 0.0;
  if (t < half) f = a.inv_freq[t];
  if (t < 64) {
    const RopeRow rr = rope_row(a, blockIdx.x);
    if (t == 0) info = rr;
  }
  __syncthreads();
  const RopeRow rr = info;
  if (!rr.mine) return;
  for (int j = t; j < half; j += blockDim.x) {
    const float2 c = rope_cs(rr.pos, j == t ? f : a.inv_freq[j], a.factor);
    float *p = reinterpret_cast<float *>(cs + 2 * (j >> 2)) + (j & 3);
    p[0] = c.x;
    p[4] = c.y;
  }
  __syncthreads();
  // a uniform count of rounds: the lanes of a wave exchange their elements in each
  for (int h0 = 0; h0 < heads; h0 += groups, h += groups) {
    float4 x = next;
    next = read(h + groups);
    const bool isq = h < a.H, isv = h >= a.H + a.KVH;
    const float *gamma = isq ? a.q_gamma : isv ? nullptr : a.k_gamma;
    float sum = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w;
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (gamma && in) {
      const float s = 1.0f / sqrtf(sum / (float)a.hd + a.eps);
      const float4 g = *reinterpret_cast<const float4 *>(gamma + e);
      x.x = x.x * s * g.x;
      x.y = x.y * s * g.y;
      x.z = x.z * s * g.z;
      x.w = x.w * s * g.w;
    }
    if (a.layout) {
      if (!isv && e < a.rot) {
        // frequencies 2 li and 2 li + 1; where rot ends inside the lane, the first alone
        const float *c = reinterpret_cast<const float *>(cs + 2 * (li >> 1)) + 2 * (li & 1);
        const float a0 = x.x, b0 = x.y, a1 = x.z, b1 = x.w;
        x.x = a0 * c[0] - b0 * c[4];
        x.y = a0 * c[4] + b0 * c[0];
        if (e + 2 < a.rot) {
          x.z = a1 * c[1] - b1 * c[5];
          x.w = a1 * c[5] + b1 * c[1];
        }
      }
    } else if (a.rot) {
      const int far = half >> 2;  // lanes from an element to its pair's other one
      const bool first = li < far;
      const int src = ((t & 63) + (first ? far : -far)) & 63;
      float4 o;
      o.x = __shfl(x.x, src, 64);
      o.y = __shfl(x.y, src, 64);
      o.z = __shfl(x.z, src, 64);
      o.w = __shfl(x.w, src, 64);
      if (!isv && e < a.rot) {
        const int k = first ? li : li - far;
        const float4 c = cs[2 * k], s = cs[2 * k + 1];
        const float sg = first ? -1.0f : 1.0f;
        x.x = x.x * c.x + sg * (o.x * s.x);
        x.y = x.y * c.y + sg * (o.y * s.y);
        x.z = x.z * c.z + sg * (o.z * s.z);
        x.w = x.w * c.w + sg * (o.w * s.w);
      }
    }
    if (!in || h >= heads) continue;
    if (isq) {
      const float nan = __builtin_nanf("");
      if (!rr.ok) x = make_float4(nan, nan, nan, nan);
      *reinterpret_cast<float4 *>(a.q + m * a.ldq + (size_t)h * a.hd + e) = x;
    } else if (rr.ok) {
      uint16_t *to = isv ? a.vc + rr.crow + (size_t)(h - a.H - a.KVH) * a.hd + e : a.kc + rr.crow + (size_t)(h - a.H) * a.hd + e;
      uint2 p;
      p.x = (uint32_t)f2h(x.x) | (uint32_t)f2h(x.y) << 16;
      p.y = (uint32_t)f2h(x.z) | (uint32_t)f2h(x.w) << 16;
      *reinterpret_cast<uint2 *>(to) = p;
    }
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

// One block per (layer, sequence).  Every thread owns columns of the rows (16
// bytes where the rows allow it) and moves them in the path's order, kMoves rows
// read before they are written: row j's source is at j or behind it, and the
// sources ascend, so no row is written before it has been read.  Bound by latency:
// the sequence's numbers, the tree, the rows, one after the other: 3.8 us for one
// sequence's 8 nodes in 24 layers, 5.4 for 16 wide trees in 28 (3.7 MB at most); 6.1
// with one row at a time, 6.7 with 2-byte columns.
constexpr int kMoves = 8;
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
      const int p = tree_parent(tree_parent_read(a.t, b), s.n, &ok);
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
  for (int c = t; c < 2 * cols; c += blockDim.x) {
    T *rows = c < cols ? (T *)a.kc + base + c : (T *)a.vc + base + (c - cols);
    for (int j = 1; j < len; j += kMoves) {
      T v[kMoves];
#pragma unroll
      for (int i = 0; i < kMoves; i++) v[i] = rows[(size_t)path[min(j + i, len - 1)] * cols];
#pragma unroll
      for (int i = 0; i < kMoves; i++)
        if (j + i < len && path[j + i] != j + i) rows[(size_t)(j + i) * cols] = v[i];
    }
  }
}

}  // namespace

int qk_norm_rope_max_hd() { return kRopeMaxHd; }

// rows that the vector form's 16-byte (caches: 8-byte) accesses can take
static bool rope_vector_ok(const NormRopeArgs &a) {
  const uintptr_t p = (uintptr_t)a.x | (uintptr_t)a.q | (uintptr_t)a.q_gamma | (uintptr_t)a.k_gamma;
  return a.hd % 4 == 0 && a.hd <= 256 && a.ldx % 4 == 0 && a.ldq % 4 == 0 && !(p & 15) &&
         !(((uintptr_t)a.kc | (uintptr_t)a.vc) & 7) && (a.layout || a.rot % 8 == 0);
}

template <int LPH>
static void launch_rope(const NormRopeArgs &a, hipStream_t st) {
  const long threads = (long)(a.H + 2 * a.KVH) * LPH;
  const int block = threads >= 256 ? 256 : (int)(threads + 63) / 64 * 64;
  klaunch(qk_norm_rope_kernel<LPH>, dim3(a.t.B * a.t.N), dim3(block), 0, st, a);
}

hipError_t qk_norm_rope(const NormRopeArgs &a, hipStream_t st) {
  if (!rope_vector_ok(a)) klaunch(qk_norm_rope_any_kernel, dim3(a.t.B * a.t.N), dim3(256), 0, st, a);
  else if (a.hd <= 32) launch_rope<8>(a, st);
  else if (a.hd <= 64) launch_rope<16>(a, st);
  else if (a.hd <= 128) launch_rope<32>(a, st);
  else launch_rope<64>(a, st);
  return hipGetLastError();
}

hipError_t tree_accept(const AcceptArgs &a, hipStream_t st) {
  const dim3 grid(a.layers, a.t.B);
  auto block = [](int cols) { return dim3(2 * cols <= 64 ? 64 : 2 * cols <= 128 ? 128 : 256); };
  if (a.kv % 8 == 0 && !(((uintptr_t)a.kc | (uintptr_t)a.vc) & 15))
    klaunch(tree_accept_kernel<v4u>, grid, block(a.kv / 8), 0, st, a, a.kv / 8);
  else
    klaunch(tree_accept_kernel<uint16_t>, grid, block(a.kv), 0, st, a, a.kv);
  return hipGetLastError();
}

}  // namespace ec
