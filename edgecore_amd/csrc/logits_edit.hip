// Logits before they are sampled: penalties for tokens that the text has already,
// biases, masks.  Per row, with c(t) the number of times that token t occurs in the
// text behind the prompt and among the row's node and its ancestors, and the tokens
// of the prompt seen as well:
//
//   y = x > 0 ? x / r : x r    where t is seen, else x
//   y = y - f c - p [c > 0] + bias(t),    -inf where the mask's bit of t is 0
#include "ec_device.h"
#include "ec_kernels.h"

namespace ec {

namespace {

// One block per 1024 tokens of the vocabulary and 8 of a sequence's rows.  The text is
// counted into a table of the chunk in LDS (whole numbers: the order does not show), from
// which every thread takes its tokens' counts and biases into registers, for all rows; a token
// that is also a node's is marked, and its count of a row's line is added where it comes up.
// So the rows need no barrier, and each is read while the one before it is worked on.  VEC:
// rows of whole 16-byte chunks, four tokens of a thread beside each other; otherwise they
// stand 256 apart.  STREAM: rows that are more than the L2s hold go past them.
//
// Bound by memory: 112 of 128 rows of 151936, 138 MB, with texts of 4000 tokens, biases and
// masks, take 30 us where three inputs take turns, 4.6 TB/s (a copy of 1 GiB 5.1), and 39 where
// eight do; through the L2s 37 and 40.  As many rows of 50257 take 20, at 2.2 TB/s: they begin at
// any address, and a thread's tokens are read one by one.  Every block reads its sequence's
// whole text: with one row a sequence that is more than the row's part from 2000 tokens on (128
// rows: 33 us for texts of 500, 56 for 8000; of 50257 tokens 17 and 26).  One row takes as long
// as the shortest kernels.
constexpr int kEditChunk = 1024, kEditRows = 8;
constexpr uint32_t kSeen = 1u << 31, kNode = 1u << 30;  // of the prompt; the token of a node
constexpr double kL2 = 32 << 20;                        // bytes of the 8 L2s together

template <bool VEC, bool STREAM>
__global__ __launch_bounds__(256) void logits_edit_kernel(EditArgs a) {
  __shared__ uint32_t count[kEditChunk], bias_at[kEditChunk];  // bias_at: the entry's index and 1
  __shared__ uint64_t line[EC_TREE_MAX];
  __shared__ int node[EC_TREE_MAX];
  const int t = threadIdx.x, v0 = blockIdx.x * kEditChunk, nv = min(kEditChunk, a.V - v0);
  const int b = blockIdx.y, i0 = blockIdx.z * kEditRows;
  const int nodes = a.nodes ? a.nodes[b] : a.N, rows = nodes >= 0 && nodes <= a.N ? nodes : a.N;
  if (i0 >= rows) return;
  const int len = a.len ? a.len[b] : 0, prompt = a.prompt ? a.prompt[b] : 0, nbias = a.nbias ? a.nbias[b] : a.max_bias;
  bool ok = nodes == rows && len >= 0 && len <= a.ldt && nbias >= 0 && nbias <= a.max_bias;
  // the k-th token of this thread, in the chunk
  const auto tok = [&](int k) { return VEC ? 4 * t + k : 256 * k + t; };
  struct Row {
    float x[4];
    uint32_t allow[VEC ? 1 : 4];
  };
  const auto read = [&](int i, Row &row) {
    const size_t r = (size_t)b * a.N + i;
    if constexpr (VEC) {
      if (tok(0) >= nv) return;
      const float4 y = *reinterpret_cast<const float4 *>(a.logits + r * a.ld + v0 + tok(0));
      row.x[0] = y.x, row.x[1] = y.y, row.x[2] = y.z, row.x[3] = y.w;
      if (a.mask) row.allow[0] = a.mask[r * a.ldm + ((v0 + tok(0)) >> 5)];
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (tok(k) < nv) {
          row.x[k] = a.logits[r * a.ld + v0 + tok(k)];
          if (a.mask) row.allow[k] = a.mask[r * a.ldm + ((v0 + tok(k)) >> 5)];
        }
    }
  };
  const float rep = a.repetition ? a.repetition[b] : 1.0f, freq = a.frequency ? a.frequency[b] : 0.0f,
              pres = a.presence ? a.presence[b] : 0.0f;
  Row next;
  read(i0, next);
  for (int e = t; e < kEditChunk; e += 256) {
    count[e] = 0;
    if (a.max_bias) bias_at[e] = 0;
  }
  if (a.token && t < 64) {
    int parent = t - 1;
    if (a.parent && t < a.N) parent = a.parent[(size_t)b * a.N + t];
    bool good;
    parent = tree_parent(parent, rows, &good);
    int depth;
    line[t] = good ? tree_ancestors(parent, &depth) : 0;
    node[t] = t < rows ? a.token[(size_t)b * a.N + t] : -1;
  }
  __syncthreads();
  if (a.token) ok = ok && line[0] != 0;
  if (ok) {
    const int *text = a.text + (size_t)b * a.ldt;
    constexpr int UN = 8;  // mostly none of them is of the chunk: one test for all
    for (int j0 = t; j0 < len; j0 += 256 * UN) {
      uint32_t e[UN], least = ~0u;
#pragma unroll
      for (int u = 0; u < UN; u++) e[u] = (uint32_t)text[min(j0 + 256 * u, len - 1)] - (uint32_t)v0;
#pragma unroll
      for (int u = 0; u < UN; u++) least = min(least, e[u]);
      if (least >= (uint32_t)nv) continue;
#pragma unroll
      for (int u = 0; u < UN; u++)
        if (e[u] < (uint32_t)nv && j0 + 256 * u < len) {
          if (j0 + 256 * u < prompt) atomicOr(&count[e[u]], kSeen);
          else atomicAdd(&count[e[u]], 1u);
        }
    }
    if (a.token && t < rows && t < 64) {
      const uint32_t e = (uint32_t)node[t] - (uint32_t)v0;
      if (e < (uint32_t)nv) atomicOr(&count[e], kNode);
    }
    for (int j = t; j < nbias; j += 256) {
      const uint32_t e = (uint32_t)a.bias_token[(size_t)b * a.max_bias + j] - (uint32_t)v0;
      if (e < (uint32_t)nv) atomicMax(&bias_at[e], (uint32_t)j + 1);
    }
    __syncthreads();
  }
  uint32_t c[4];
  float bias[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    c[k] = count[tok(k)];
    const uint32_t at = ok && nbias ? bias_at[tok(k)] : 0;
    bias[k] = at ? a.bias[(size_t)b * a.max_bias + (at - 1)] : 0.0f;
  }
  const int i1 = min(rows, i0 + kEditRows);
  for (int i = i0; i < i1; i++) {
    Row row = next;
    if (i + 1 < i1) read(i + 1, next);
#pragma unroll
    for (int k = 0; k < 4; k++) {
      uint32_t n = c[k] & ~(kSeen | kNode);
      bool seen = (c[k] & ~kNode) != 0;
      if (__builtin_expect((c[k] & kNode) != 0, 0)) {
        uint32_t more = 0;
#pragma unroll 1
        for (uint64_t up = line[i]; up; up &= up - 1) more += node[__ffsll((unsigned long long)up) - 1] == v0 + tok(k);
        n += more;
        seen |= more != 0;
      }
      float y = row.x[k];
      if (seen) y = y > 0.0f ? y / rep : y * rep;
      if (n) y = (y - freq * (float)n) - pres;
      if (bias[k] != 0.0f) y += bias[k];
      if (a.mask && !((row.allow[VEC ? 0 : k] >> ((v0 + tok(k)) & 31)) & 1)) y = -__builtin_inff();
      row.x[k] = ok ? y : __builtin_nanf("");
    }
    float *out = a.out + ((size_t)b * a.N + i) * a.ldo + v0;
    if constexpr (VEC) {
      typedef float v4f __attribute__((ext_vector_type(4)));
      const v4f y = {row.x[0], row.x[1], row.x[2], row.x[3]};
      v4f *to = reinterpret_cast<v4f *>(out + tok(0));
      if (tok(0) < nv) {
        if constexpr (STREAM) __builtin_nontemporal_store(y, to);
        else *to = y;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (tok(k) < nv) {
          if constexpr (STREAM) __builtin_nontemporal_store(row.x[k], out + tok(k));
          else out[tok(k)] = row.x[k];
        }
    }
  }
}

}  // namespace

hipError_t logits_edit(const EditArgs &a, hipStream_t st) {
  const dim3 grid((a.V + kEditChunk - 1) / kEditChunk, a.B, (a.N + kEditRows - 1) / kEditRows);
  const bool vec = a.V % 4 == 0 && a.ld % 4 == 0 && a.ldo % 4 == 0 && !(((uintptr_t)a.logits | (uintptr_t)a.out) & 15);
  const bool stream = (double)a.B * a.N * a.V * 4 > kL2;
  if (vec && stream) klaunch((logits_edit_kernel<true, true>), grid, dim3(256), 0, st, a);
  else if (vec) klaunch((logits_edit_kernel<true, false>), grid, dim3(256), 0, st, a);
  else if (stream) klaunch((logits_edit_kernel<false, true>), grid, dim3(256), 0, st, a);
  else klaunch((logits_edit_kernel<false, false>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ec
