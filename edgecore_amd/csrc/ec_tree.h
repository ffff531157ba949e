/*
 * The batch that the operators for drafted tokens take: B sequences of N rows,
 * row b * N + i being node i of sequence b.  Per sequence a cache slot, the
 * number of rows already cached there (past) and the number of its nodes; per
 * node its parent.  Node i's key and value live at row past + i of the slot;
 * its place in the text is past + depth.  The arrays are in device memory, so
 * what they hold is checked where they are read, by the functions here: a
 * sequence that fails takes no part in the call.
 *
 * C and C++ (host) and HIP (device) compatible.
 */
#ifndef EC_TREE_H
#define EC_TREE_H

#include <stdint.h>

#if defined(__HIP__)
#define EC_TREE_FN __host__ __device__ static inline
#else
#define EC_TREE_FN static inline
#endif

/* the most nodes of a sequence with parents: one per lane of a wave */
#define EC_TREE_MAX 64

typedef struct {
    int B, N;
    const int *slot, *past, *nodes, *parent; /* past alone is never NULL */
    int nslots, C, max_past;
} EcTreeBatch;

typedef struct {
    int slot, past, n;
} EcTreeSeq;

EC_TREE_FN EcTreeSeq ec_tree_seq(const EcTreeBatch *t, int b)
{
    EcTreeSeq s;
    s.slot = t->slot ? t->slot[b] : b;
    s.past = t->past[b];
    s.n = t->nodes ? t->nodes[b] : t->N;
    return s;
}

/* whether the sequence's numbers name rows of the cache (no sum that could
 * pass the largest int) */
EC_TREE_FN int ec_tree_seq_ok(const EcTreeBatch *t, EcTreeSeq s)
{
    return s.slot >= 0 && s.slot < t->nslots && s.n >= 0 && s.n <= t->N && s.past >= 0 && s.past <= t->max_past &&
           s.n <= t->C && s.past <= t->C - s.n;
}

/* rows of the call that the sequence owns: its nodes, or all N where their
 * number is none (then they are marked as failed) */
EC_TREE_FN int ec_tree_rows(const EcTreeBatch *t, EcTreeSeq s)
{
    return s.n >= 0 && s.n <= t->N ? s.n : t->N;
}

/* node i's parent comes before it, or is none (-1) */
EC_TREE_FN int ec_tree_parent_ok(int parent, int i)
{
    return parent >= -1 && parent < i;
}

/* whether two sequences (both ec_tree_seq_ok) have a node's row in common */
EC_TREE_FN int ec_tree_clash(EcTreeSeq a, EcTreeSeq b)
{
    return a.slot == b.slot && a.n > 0 && b.n > 0 && a.past < b.past + b.n && b.past < a.past + a.n;
}

#if defined(__HIP__)
namespace ec {

/* Every lane of the wave calls the functions below. */

/* whether sequence b's nodes share a row with those of an earlier sequence, written
 * or not: what the earlier ones' parents and clashes are is not followed (never where
 * every sequence has its own slot).  Four sequences a lane at a time, so that
 * a round is one wait */
__device__ __forceinline__ bool tree_clashes(const EcTreeBatch &t, int b, EcTreeSeq s) {
  if (!t.slot) return false;
  for (int c0 = 0; c0 < b; c0 += 256) {
    EcTreeSeq o[4];
#pragma unroll
    for (int k = 0; k < 4; k++) o[k] = ec_tree_seq(&t, min(c0 + 64 * k + (int)(threadIdx.x & 63), b - 1));
    bool hit = false;
#pragma unroll
    for (int k = 0; k < 4; k++) hit |= ec_tree_seq_ok(&t, o[k]) && ec_tree_clash(s, o[k]);
    if (__ballot(hit)) return true;
  }
  return false;
}

/* lane i's entry of the parents, read ahead of its check (any value behind the rows) */
__device__ __forceinline__ int tree_parent_read(const EcTreeBatch &t, int b) {
  const int i = threadIdx.x & 63;
  return t.parent ? t.parent[(size_t)b * t.N + min(i, t.N - 1)] : i - 1;
}
/* lane i's parent (-1 past the nodes) from what it read; *ok: whether every node's is valid */
__device__ __forceinline__ int tree_parent(int read, int n, bool *ok) {
  const int i = threadIdx.x & 63, p = i < n ? read : -1;
  *ok = __ballot(!ec_tree_parent_ok(p, i)) == 0;
  return p;
}

/* lane i's ancestors and itself, and its depth, from valid parents: every
 * round doubles the distance that a lane has looked up the tree */
__device__ __forceinline__ uint64_t tree_ancestors(int parent, int *depth) {
  const int i = threadIdx.x & 63;
  uint64_t m = 1ull << i;
  int p = parent;
  for (int r = 0; r < 6; r++) {
    const int at = p < 0 ? i : p;
    const uint64_t mo = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(m >> 32), at, 64) << 32) |
                        (uint32_t)__shfl((int)(uint32_t)m, at, 64);
    const int po = __shfl(p, at, 64);
    if (p >= 0) {
      m |= mo;
      p = po;
    }
  }
  *depth = __popcll(m) - 1;
  return m;
}

}  // namespace ec
#endif

#endif /* EC_TREE_H */
