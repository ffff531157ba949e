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

// One block per CHUNK tokens of the vocabulary and some of a sequence's rows: the text is
// counted into a table of the chunk in LDS (whole numbers: the order does not show), a
// row's nodes are added for the row and taken out again.  VEC: rows of whole 16-byte
// chunks, four tokens of a thread beside each other; otherwise they stand 256 apart.
constexpr int kEditRows = 4;
constexpr uint32_t kSeen = 1u << 31;  // of the prompt

template <int CHUNK, bool VEC>
__global__ __launch_bounds__(256) void logits_edit_kernel(EditArgs a) {
  constexpr int Q = CHUNK / 1024;  // fours of a thread
  __shared__ __attribute__((aligned(16))) uint32_t count[CHUNK];
  __shared__ __attribute__((aligned(16))) uint32_t bias_at[CHUNK];  // the entry's index and 1, then its value
  __shared__ uint64_t line[EC_TREE_MAX];
  __shared__ int node[EC_TREE_MAX];
  const int t = threadIdx.x, v0 = blockIdx.x * CHUNK, nv = min(CHUNK, a.V - v0);
  const int b = blockIdx.y, i0 = blockIdx.z * kEditRows;
  const int nodes = a.nodes ? a.nodes[b] : a.N, rows = nodes >= 0 && nodes <= a.N ? nodes : a.N;
  if (i0 >= rows) return;
  const int len = a.len ? a.len[b] : 0, prompt = a.prompt ? a.prompt[b] : 0, nbias = a.nbias ? a.nbias[b] : a.max_bias;
  bool ok = nodes == rows && len >= 0 && len <= a.ldt && nbias >= 0 && nbias <= a.max_bias;
  // the k-th token of the q-th four of this thread, in the chunk
  const auto tok = [&](int q, int k) { return VEC ? 1024 * q + 4 * t + k : 1024 * q + 256 * k + t; };
  float x[Q][4];
  uint32_t allow[Q][4];
  const auto read = [&](int i) {
    const size_t r = (size_t)b * a.N + i;
#pragma unroll
    for (int q = 0; q < Q; q++) {
      if constexpr (VEC) {
        if (tok(q, 0) >= nv) break;
        const float4 y = *reinterpret_cast<const float4 *>(a.logits + r * a.ld + v0 + tok(q, 0));
        x[q][0] = y.x, x[q][1] = y.y, x[q][2] = y.z, x[q][3] = y.w;
        if (a.mask) allow[q][0] = a.mask[r * a.ldm + ((v0 + tok(q, 0)) >> 5)];
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (tok(q, k) < nv) {
            x[q][k] = a.logits[r * a.ld + v0 + tok(q, k)];
            if (a.mask) allow[q][k] = a.mask[r * a.ldm + ((v0 + tok(q, k)) >> 5)];
          }
      }
    }
  };
  read(i0);
  for (int e = t; e < CHUNK; e += 256) {
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
    constexpr int UN = 8;
    for (int j0 = t; j0 < len; j0 += 256 * UN) {
      uint32_t e[UN];
#pragma unroll
      for (int u = 0; u < UN; u++) e[u] = (uint32_t)text[min(j0 + 256 * u, len - 1)] - (uint32_t)v0;
#pragma unroll
      for (int u = 0; u < UN; u++)
        if (e[u] < (uint32_t)nv && j0 + 256 * u < len) {
          if (j0 + 256 * u < prompt) atomicOr(&count[e[u]], kSeen);
          else atomicAdd(&count[e[u]], 1u);
        }
    }
    for (int j = t; j < nbias; j += 256) {
      const uint32_t e = (uint32_t)a.bias_token[(size_t)b * a.max_bias + j] - (uint32_t)v0;
      if (e < (uint32_t)nv) atomicMax(&bias_at[e], (uint32_t)j + 1);
    }
    if (nbias) {
      __syncthreads();
      for (int e = t; e < nv; e += 256)
        if (bias_at[e]) bias_at[e] = __float_as_uint(a.bias[(size_t)b * a.max_bias + (bias_at[e] - 1)]);
    }
  }
  const float rep = a.repetition ? a.repetition[b] : 1.0f, freq = a.frequency ? a.frequency[b] : 0.0f,
              pres = a.presence ? a.presence[b] : 0.0f;
  const bool biased = ok && nbias;
  for (int i = i0; i < min(rows, i0 + kEditRows); i++) {
    const size_t r = (size_t)b * a.N + i;
    uint32_t mine = ~0u;  // of the chunk: the token of a node of this row's line
    if (a.token && ok && t < 64 && ((line[i] >> t) & 1)) mine = (uint32_t)node[t] - (uint32_t)v0;
    __syncthreads();
    if (a.token) {
      if (mine < (uint32_t)nv) atomicAdd(&count[mine], 1u);
      __syncthreads();
    }
#pragma unroll
    for (int q = 0; q < Q; q++) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int e = tok(q, k);
        const uint32_t c = count[e], n = c & ~kSeen;
        float y = x[q][k];
        if (c) y = y > 0.0f ? y / rep : y * rep;
        if (n) y = (y - freq * (float)n) - pres;
        if (biased && bias_at[e]) y += __uint_as_float(bias_at[e]);
        if (a.mask && !((allow[q][VEC ? 0 : k] >> ((v0 + e) & 31)) & 1)) y = -__builtin_inff();
        x[q][k] = ok ? y : __builtin_nanf("");
      }
      if constexpr (VEC) {
        if (tok(q, 0) < nv)
          *reinterpret_cast<float4 *>(a.out + r * a.ldo + v0 + tok(q, 0)) = make_float4(x[q][0], x[q][1], x[q][2], x[q][3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (tok(q, k) < nv) a.out[r * a.ldo + v0 + tok(q, k)] = x[q][k];
      }
    }
    if (i + 1 < min(rows, i0 + kEditRows)) read(i + 1);
    if (a.token) {
      __syncthreads();
      if (mine < (uint32_t)nv) atomicSub(&count[mine], 1u);
    }
  }
}

}  // namespace

template <int CHUNK>
static void launch_edit(const EditArgs &a, hipStream_t st) {
  const dim3 grid((a.V + CHUNK - 1) / CHUNK, a.B, (a.N + kEditRows - 1) / kEditRows);
  const bool vec = a.V % 4 == 0 && a.ld % 4 == 0 && a.ldo % 4 == 0 && !(((uintptr_t)a.logits | (uintptr_t)a.out) & 15);
  if (vec) klaunch((logits_edit_kernel<CHUNK, true>), grid, dim3(256), 0, st, a);
  else klaunch((logits_edit_kernel<CHUNK, false>), grid, dim3(256), 0, st, a);
}

hipError_t logits_edit(const EditArgs &a, hipStream_t st) {
  const long blocks = (long)((a.V + 4095) / 4096) * a.B * ((a.N + kEditRows - 1) / kEditRows);
  if (blocks >= 512) launch_edit<4096>(a, st);
  else launch_edit<1024>(a, st);
  return hipGetLastError();
}

}  // namespace ec
