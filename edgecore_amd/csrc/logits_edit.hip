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

// One block per chunk of the vocabulary and some of a sequence's rows: the text is
// counted into a table of the chunk in LDS (whole numbers: the order does not show),
// a row's nodes are added for the row and taken out again.
constexpr int kEditChunk = 4096, kEditRows = 4;
constexpr uint32_t kSeen = 1u << 31;  // of the prompt

__global__ __launch_bounds__(256) void logits_edit_kernel(EditArgs a) {
  __shared__ uint32_t count[kEditChunk];
  __shared__ uint32_t bias_at[kEditChunk];  // the entry's index and 1
  __shared__ uint64_t line[EC_TREE_MAX];
  __shared__ int node[EC_TREE_MAX];
  const int t = threadIdx.x, v0 = blockIdx.x * kEditChunk, nv = min(kEditChunk, a.V - v0);
  const int b = blockIdx.y, i0 = blockIdx.z * kEditRows;
  const int nodes = a.nodes ? a.nodes[b] : a.N, rows = nodes >= 0 && nodes <= a.N ? nodes : a.N;
  if (i0 >= rows) return;
  const int len = a.len ? a.len[b] : 0, prompt = a.prompt ? a.prompt[b] : 0, nbias = a.nbias ? a.nbias[b] : a.max_bias;
  bool ok = nodes == rows && len >= 0 && len <= a.ldt && nbias >= 0 && nbias <= a.max_bias;
  for (int e = t; e < nv; e += 256) count[e] = bias_at[e] = 0;
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
    for (int j = t; j < len; j += 256) {
      const uint32_t e = (uint32_t)a.text[(size_t)b * a.ldt + j] - (uint32_t)v0;
      if (e < (uint32_t)nv) {
        if (j < prompt) atomicOr(&count[e], kSeen);
        else atomicAdd(&count[e], 1u);
      }
    }
    for (int j = t; j < nbias; j += 256) {
      const uint32_t e = (uint32_t)a.bias_token[(size_t)b * a.max_bias + j] - (uint32_t)v0;
      if (e < (uint32_t)nv) atomicMax(&bias_at[e], (uint32_t)j + 1);
    }
  }
  const float rep = a.repetition ? a.repetition[b] : 1.0f, freq = a.frequency ? a.frequency[b] : 0.0f,
              pres = a.presence ? a.presence[b] : 0.0f;
  for (int i = i0; i < min(rows, i0 + kEditRows); i++) {
    const size_t r = (size_t)b * a.N + i;
    uint32_t mine = ~0u;  // of the chunk: the token of a node of this row's line
    if (a.token && ok && t < 64 && ((line[i] >> t) & 1)) mine = (uint32_t)node[t] - (uint32_t)v0;
    __syncthreads();
    if (mine < (uint32_t)nv) atomicAdd(&count[mine], 1u);
    __syncthreads();
    for (int e = t; e < nv; e += 256) {
      float x = a.logits[r * a.ld + v0 + e];
      const uint32_t c = count[e], n = c & ~kSeen, k = bias_at[e];
      if (c) x = x > 0.0f ? x / rep : x * rep;
      if (n) x = (x - freq * (float)n) - pres;
      if (k) x += a.bias[(size_t)b * a.max_bias + (k - 1)];
      if (a.mask && !((a.mask[r * a.ldm + ((v0 + e) >> 5)] >> ((v0 + e) & 31)) & 1)) x = -__builtin_inff();
      if (!ok) x = __builtin_nanf("");
      a.out[r * a.ldo + v0 + e] = x;
    }
    __syncthreads();
    if (mine < (uint32_t)nv) atomicSub(&count[mine], 1u);
  }
}

}  // namespace

hipError_t logits_edit(const EditArgs &a, hipStream_t st) {
  klaunch(logits_edit_kernel, dim3((a.V + kEditChunk - 1) / kEditChunk, a.B, (a.N + kEditRows - 1) / kEditRows), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ec
