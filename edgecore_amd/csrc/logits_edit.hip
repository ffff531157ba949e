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

// One block per CHUNK tokens of the vocabulary and some of a sequence's rows.  The text is
// counted into a table of the chunk in LDS (whole numbers: the order does not show), from
// which every thread takes its tokens' counts and biases into registers, for all rows; a token
// that is also a node's is marked, and its count of a row's line is added where it comes up.
// So the rows need no barrier, and each is read while the one before it is worked on.  VEC:
// rows of whole 16-byte chunks, four tokens of a thread beside each other; otherwise they
// stand 256 apart.
constexpr int kEditRows = 8;
constexpr uint32_t kSeen = 1u << 31, kNode = 1u << 30;  // of the prompt; the token of a node

template <int CHUNK, bool VEC>
__global__ __launch_bounds__(256) void logits_edit_kernel(EditArgs a) {
  constexpr int Q = CHUNK / 1024;  // fours of a thread
  __shared__ uint32_t count[CHUNK], bias_at[CHUNK];  // bias_at: the entry's index and 1
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
  struct Row {
    float x[Q][4];
    uint32_t allow[Q][VEC ? 1 : 4];
  };
  const auto read = [&](int i, Row &row) {
    const size_t r = (size_t)b * a.N + i;
#pragma unroll
    for (int q = 0; q < Q; q++) {
      if constexpr (VEC) {
        if (tok(q, 0) >= nv) break;
        const float4 y = *reinterpret_cast<const float4 *>(a.logits + r * a.ld + v0 + tok(q, 0));
        row.x[q][0] = y.x, row.x[q][1] = y.y, row.x[q][2] = y.z, row.x[q][3] = y.w;
        if (a.mask) row.allow[q][0] = a.mask[r * a.ldm + ((v0 + tok(q, 0)) >> 5)];
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (tok(q, k) < nv) {
            row.x[q][k] = a.logits[r * a.ld + v0 + tok(q, k)];
            if (a.mask) row.allow[q][k] = a.mask[r * a.ldm + ((v0 + tok(q, k)) >> 5)];
          }
      }
    }
  };
  const float rep = a.repetition ? a.repetition[b] : 1.0f, freq = a.frequency ? a.frequency[b] : 0.0f,
              pres = a.presence ? a.presence[b] : 0.0f;
  Row next;
  read(i0, next);
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
  uint32_t c[Q][4];
  float bias[Q][4];
#pragma unroll
  for (int q = 0; q < Q; q++)
#pragma unroll
    for (int k = 0; k < 4; k++) {
      c[q][k] = count[tok(q, k)];
      const uint32_t at = ok && nbias ? bias_at[tok(q, k)] : 0;
      bias[q][k] = at ? a.bias[(size_t)b * a.max_bias + (at - 1)] : 0.0f;
    }
  const int i1 = min(rows, i0 + kEditRows);
  for (int i = i0; i < i1; i++) {
    const size_t r = (size_t)b * a.N + i;
    Row row = next;
    if (i + 1 < i1) read(i + 1, next);
#pragma unroll
    for (int q = 0; q < Q; q++) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        uint32_t n = c[q][k] & ~(kSeen | kNode);
        bool seen = (c[q][k] & ~kNode) != 0;
        if (__builtin_expect((c[q][k] & kNode) != 0, 0)) {
          uint32_t more = 0;
#pragma unroll 1
          for (uint64_t up = line[i]; up; up &= up - 1) more += node[__ffsll((unsigned long long)up) - 1] == v0 + tok(q, k);
          n += more;
          seen |= more != 0;
        }
        float y = row.x[q][k];
        if (seen) y = y > 0.0f ? y / rep : y * rep;
        if (n) y = (y - freq * (float)n) - pres;
        if (bias[q][k] != 0.0f) y += bias[q][k];
        if (a.mask && !((row.allow[q][VEC ? 0 : k] >> ((v0 + tok(q, k)) & 31)) & 1)) y = -__builtin_inff();
        row.x[q][k] = ok ? y : __builtin_nanf("");
      }
      if constexpr (VEC) {
        if (tok(q, 0) < nv)
          *reinterpret_cast<float4 *>(a.out + r * a.ldo + v0 + tok(q, 0)) = make_float4(row.x[q][0], row.x[q][1], row.x[q][2], row.x[q][3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (tok(q, k) < nv) a.out[r * a.ldo + v0 + tok(q, k)] = row.x[q][k];
      }
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
  const long blocks = (long)((a.V + 2047) / 2048) * a.B * ((a.N + kEditRows - 1) / kEditRows);
  if (blocks >= 512) launch_edit<2048>(a, st);
  else launch_edit<1024>(a, st);
  return hipGetLastError();
}

}  // namespace ec
