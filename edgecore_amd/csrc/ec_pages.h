/*
 * The batch that the operators over a paged cache take: B sequences whose new
 * rows stand one behind the other in a call of M rows, and the pages that hold
 * their cached rows.  Row i of sequence b's new ones is row start[b] + i of the
 * call and row past[b] + i of its text; row p of a text is row p % page of page
 * table[b][p / page].  The arrays are in device memory, so what they hold is
 * checked where they are read, by the functions here: a sequence that fails
 * takes no part in the call.
 *
 * C and C++ (host) and HIP (device) compatible.
 */
#ifndef EC_PAGES_H
#define EC_PAGES_H

#include <stdint.h>

#if defined(__HIP__)
#define EC_PAGES_FN __host__ __device__ static inline
#else
#define EC_PAGES_FN static inline
#endif

/* rows of a text, at most: sums of two of them stay below 2^31 */
#define EC_PAGES_ROWS (1 << 30)

typedef struct {
    int B, M;
    const int *start, *past; /* start NULL: a row each */
    const int *table;
    int ldt, npages, page, KVH;
    int rows; /* that a table has room for, at most EC_PAGES_ROWS */
    uint32_t mul, shift; /* p / page = p mul >> shift, for p < 2^31 */
} EcPageBatch;

typedef struct {
    int start, n, past;
} EcPageSeq;

/* mul and shift of a page size: 2^shift / page rounded up, off by less than
 * page <= 2^(shift - 31), so that the quotients of 31 bits are exact */
EC_PAGES_FN void ec_pages_divide(EcPageBatch *t)
{
    uint32_t s = 0;
    while (((uint32_t)1 << s) < (uint32_t)t->page) s++;
    t->shift = 31 + s;
    t->mul = (uint32_t)((((uint64_t)1 << t->shift) + (uint32_t)t->page - 1) / (uint32_t)t->page);
}

EC_PAGES_FN int ec_page_of(const EcPageBatch *t, int p)
{
    return (int)(((uint64_t)(uint32_t)p * t->mul) >> t->shift);
}

EC_PAGES_FN EcPageSeq ec_page_seq(const EcPageBatch *t, int b)
{
    EcPageSeq s;
    s.start = t->start ? t->start[b] : b;
    /* in 64 bits: the difference of two ints may pass the largest one */
    const int64_t n = t->start ? (int64_t)t->start[b + 1] - s.start : 1;
    s.n = n < 0 || n > t->M ? -1 : (int)n;
    s.past = t->past[b];
    return s;
}

/* whether the sequence's new rows are rows of the call */
EC_PAGES_FN int ec_page_seq_mine(const EcPageBatch *t, EcPageSeq s)
{
    return s.start >= 0 && s.n > 0 && s.start <= t->M - s.n;
}

/* whether its table has room for its text (no sum that could pass the largest int) */
EC_PAGES_FN int ec_page_seq_ok(const EcPageBatch *t, EcPageSeq s, int max_past)
{
    return s.past >= 0 && s.past <= max_past && s.n <= t->rows && s.past <= t->rows - s.n;
}

#if defined(__HIP__)
namespace ec {

/* row p of sequence b's text, as a row of the cache's [npages][KVH][page] of KV
 * head h (below 2^31: the host checks the product).  *bad: its page is none */
__device__ __forceinline__ uint32_t page_row(const EcPageBatch &t, int id, int p, int h, bool *bad) {
  const bool b = (uint32_t)id >= (uint32_t)t.npages;
  *bad |= b;
  const int pg = ec_page_of(&t, p);
  return ((b ? 0u : (uint32_t)id) * (uint32_t)t.KVH + (uint32_t)h) * (uint32_t)t.page + (uint32_t)(p - pg * t.page);
}
__device__ __forceinline__ int page_id(const EcPageBatch &t, int b, int p) {
  return t.table[(size_t)b * t.ldt + ec_page_of(&t, p)];
}

/* The sequence that row m of the call belongs to, or -1: the last one that starts at
 * m or before it (empty ones aside: the last of equal starts).  Every lane of the wave
 * calls it with the same m: 64 starts a round. */
__device__ __forceinline__ int page_seq_of(const EcPageBatch &t, int m) {
  if (!t.start) return m < t.B ? m : -1;
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = t.B;  // of these
  if (t.start[0] > m) return -1;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, b = lo + lane * step;
    const uint64_t in = __ballot(b < hi && t.start[b < hi ? b : lo] <= m);
    // where the starts ascend these are the first lanes
    const int k = in ? 63 - __clzll((long long)in) : 0;
    lo += k * step;
    hi = hi < lo + step ? hi : lo + step;
  }
  return lo;
}

}  // namespace ec
#endif

#endif /* EC_PAGES_H */
