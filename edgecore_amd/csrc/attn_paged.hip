// Attention of new tokens over a paged cache (ec_pages.h, paged_cache.h): the token at
// position t of its text sees the positions p <= t, with a window those with p > t -
// window and the first `sinks`:
//
//   x_p = scale q . k_p
//   o   = sum_p e^(x_p - m) v_p / sum_p e^(x_p - m),  m = max_p x_p
//
// in fp32.  What a token does not see does not reach it, finite or not.
//
// One pass over the keys and values with the running maximum and sum; tiles of them meet 16
// rows (single tokens: bound by the cache's bytes) or 128 (chunks: by the matrix cores and the
// vector ALUs, which a wave uses in turn and two waves of a SIMD in part beside each other).
// Texts are split into parts where their row tiles do not fill the chip, and the parts joined
// by a second launch.  Times below are kernels' in us by the library's timing, by which the
// shortest kernels take 4; cases are sequences x tokens, query / KV heads x head size, rows of the texts.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "attn_parts.h"
#include "ec_device.h"
#include "ec_kernels.h"
#include "paged_cache.h"

namespace ec {

namespace {

// The form for any head size and alignment: one block per (token, head), tiles
// of 256 positions, a position per thread for the scores and an element of the
// head per thread for the sums, with the running maximum and sum.  Every query head reads
// its keys again, by elements: right, not fast (64 x 1, 12 / 2 x 126, 4000: 1410; at 128 the matrix cores'
// forms take 31).
constexpr int kPagedMaxHd = 512;
__global__ __launch_bounds__(256) void attn_paged_any_kernel(PagedAttnArgs a) {
  __shared__ float q[kPagedMaxHd], p_s[256], red[4];
  __shared__ float part[256];
  __shared__ uint32_t row_s[256];
  const int t = threadIdx.x, hd = a.c.hd;
  const int h = blockIdx.y, m = blockIdx.x, kvh = h / a.G;
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
      // in sums of 16 positions, these in the tile's: one by one, weights below half a step of
      // what there is would be lost (32000 positions beside one that has 0.999: 2e-4 of the outputs)
      float tile = 0.0f;
      if (g < groups && d < hd)
        for (int j0 = g; j0 < n; j0 += 16 * groups) {
          float some = 0.0f;
          for (int j = j0; j < min(n, j0 + 16 * groups); j += groups)
            some = __builtin_fmaf(p_s[j], h2f(cache_value(a.c.v, a.c.vs, a.c.type, row_s[j], hd, d)), some);
          tile += some;
        }
      acc[r] = __builtin_fmaf(acc[r], back, tile);
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

// ---------------------------------------------------------------------------
// The matrix-core forms (head sizes that are multiples of 16 up to 128, in LDS and
// registers filled up with zeros to one of 32).  A unit of work is a tile of RT rows of one
// KV head of one sequence (row r: token r / G, query head r % G of the G = H / KVH that
// share it) and a part of the 64-position tiles that they see.
// ---------------------------------------------------------------------------
constexpr int kTp = 64;          // positions per tile
constexpr float kRoom = 3.0f;    // how far scores may pass the running maximum (powers of two)
constexpr float kLift = 12.0f;   // the weights are 2^kLift e^(x - m)
static_assert(kLift + kRoom < 16.0f, "weights below 65504");
constexpr long kGridRow = 1L << 20;
typedef float v16f __attribute__((ext_vector_type(16)));

// places: units per KV head that run at once (512: two blocks a CU); target: parts per KV head that
// the texts are split into where there is no room for all at once (0: they are not split); least:
// tiles of a part, at least
struct PagedGrid {
  long units;
  int places, target, least;
};

// The tiles that rows of tokens ta .. tb see: those of the first tokens that are not among
// the window's, then the window's.
struct Tiles {
  int lo, sinks;     // positions from lo on and below sinks are seen
  int front, first, n;  // tiles of the first tokens, the window's first one, all
  __device__ __forceinline__ int at(int i) const { return (i < front ? i : i - front + first) * kTp; }
};
__device__ __forceinline__ Tiles tiles_of(const PagedAttnArgs &a, const EcPageSeq &s, int ta, int tb) {
  Tiles t;
  t.lo = a.window && s.past + ta >= a.window ? s.past + ta - a.window + 1 : 0;
  t.sinks = min(a.sinks, t.lo);
  t.first = t.lo / kTp;
  t.front = min((t.sinks + kTp - 1) / kTp, t.first);
  t.n = t.front + (s.past + tb) / kTp - t.first + 1;
  return t;
}

// A sequence's row tiles, and no fewer tiles of positions than any of them has
template <int RT>
__device__ __forceinline__ int row_tiles(const PagedAttnArgs &a, const EcPageSeq &s) {
  return ec_page_seq_mine(&a.c.t, s) ? (s.n * a.G + RT - 1) / RT : 0;
}
template <int RT>
__device__ __forceinline__ int most_tiles(const PagedAttnArgs &a, const EcPageSeq &s) {
  if (!ec_page_seq_ok(&a.c.t, s, a.max_past)) return 1;
  const int all = (s.past + s.n - 1) / kTp + 1;
  if (!a.window) return all;
  // the tokens of a row tile, the tiles of the positions that they see
  const int tokens = min((RT + a.G - 2) / a.G + 1, s.n);
  const long seen = ((long)a.window + tokens) / kTp + 2 + ((long)min(a.sinks, s.past + s.n) + kTp - 1) / kTp;
  return (int)min((long)all, seen);
}

// What a block does: part j of n of row tile rt of sequence c and KV head kvh.  at: the
// unit of part 0 (the parts are KVH units from each other).
struct Unit {
  int c, rt, kvh, j, n;
  uint32_t at;
  EcPageSeq s;
};
__device__ __forceinline__ EcPageSeq lane_seq(EcPageSeq s, int l) {
  return EcPageSeq{readlane(s.start, l), readlane(s.n, l), readlane(s.past, l)};
}
// By a wave, a sequence per lane.  The parts: as many of a row tile as its sequence's tiles are
// times a share of all tiles of the call, so that the units are alike, and a text that is longer
// than the others is not what the call waits for.  The share is the smallest with which all units
// run at once: with as many units as places on average, some of them start when others end (a call
// of 6 x 256, 12 / 12 x 64, window 1000: 39.4 against 33.9; 64 x 1, 12 / 2 x 128, 4000: 38.2 against 34.5).
// The search takes 0.4 to 1 us.  Within a sequence the last
// row tiles, which see most, come first, and the units of one part of the positions stand 8
// apart where there are as many parts: on one XCD, whose L2 they share.
template <int RT>
__device__ __forceinline__ Unit find_unit(const PagedAttnArgs &a, const PagedGrid &gr, long x) {
  const int lane = threadIdx.x & 63, B = a.c.t.B, KVH = a.c.t.KVH;
  Unit u{-1, 0, 0, 0, 1, 0, {0, 0, 0}};
  if (!gr.target) {
    // sequence b's row tiles are among places start[b] G / RT + b and on, up to the next one's
    const long places = gr.units / KVH, place = places - 1 - x / KVH;
    const auto base = [&](int b) {
      return (long)(a.c.t.start ? a.c.t.start[b] : b) * a.G / RT + b;
    };
    int lo = 0, hi = B;
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64, b = lo + lane * step;
      const uint64_t in = __ballot(b < hi && base(min(b, B - 1)) <= place);
      const int k = in ? 63 - __clzll((long long)in) : 0;
      lo += k * step;
      hi = min(hi, lo + step);
    }
    u.s = ec_page_seq(&a.c.t, lo);
    const long rt = place - base(lo);
    if (rt < 0 || rt >= row_tiles<RT>(a, u.s)) return u;
    u.c = lo;
    u.rt = (int)rt;
    u.kvh = (int)(x % KVH);
    return u;
  }
  EcPageSeq s0{0, 0, 0};
  int rt0 = 0, tiles0 = 0;
  const auto seq = [&](int c, EcPageSeq &s, int &rt, int &tiles) {
    s = ec_page_seq(&a.c.t, min(c, B - 1));
    rt = c < B ? row_tiles<RT>(a, s) : 0;
    tiles = rt ? most_tiles<RT>(a, s) : 0;
  };
  seq(lane, s0, rt0, tiles0);
  unsigned long long all = 0, least = 0;
  for (int c0 = 0; c0 < B; c0 += 64) {
    EcPageSeq s;
    int rt = rt0, tiles = tiles0;
    if (c0) seq(c0 + lane, s, rt, tiles);
    all += readlane(wave_scan((unsigned long long)rt * tiles), 63);
    least += readlane(wave_scan((uint32_t)rt), 63);
  }
  // the smallest share whose units all have a place at once; where none of a few has, one
  // whose units are no more than target and the row tiles
  uint32_t share = (uint32_t)fmin(fmax(ceil((double)all / gr.places), (double)gr.least), 0x1p30);
  for (int k = 0;; k++) {
    unsigned long long units = least;
    for (int c0 = 0; c0 < B && least <= (unsigned long long)gr.places; c0 += 64) {
      if (!c0) units = 0;
      EcPageSeq s;
      int rt = rt0, tiles = tiles0;
      if (c0) seq(c0 + lane, s, rt, tiles);
      units += readlane(wave_scan((unsigned long long)rt * (((uint32_t)tiles + share - 1) / share)), 63);
    }
    if (units <= (unsigned long long)gr.places) break;
    if (k == 8 || least > (unsigned long long)gr.places) {
      share = (uint32_t)fmin(fmax(ceil((double)all / gr.target), (double)gr.least), 0x1p30);
      break;
    }
    share += max(1u, share >> 4);
  }
  unsigned long long before = 0;
  for (int c0 = 0; c0 < B; c0 += 64) {
    EcPageSeq s = s0;
    int rt = rt0, tiles = tiles0;
    if (c0) seq(c0 + lane, s, rt, tiles);
    const int n = (int)(((uint32_t)tiles + share - 1) / share);
    const unsigned long long mine = (unsigned long long)rt * n * KVH, upto = before + wave_scan(mine);
    const uint64_t hit = __ballot(mine && upto > (unsigned long long)x);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      u.s = lane_seq(s, l);
      u.c = c0 + l;
      u.n = readlane(n, l);
      const uint32_t i = (uint32_t)((unsigned long long)x - (readlane(upto, l) - readlane(mine, l))), groups = u.n * KVH;
      u.rt = readlane(rt, l) - 1 - (int)(i / groups);
      const uint32_t g = i % groups;
      u.j = (int)(g / KVH);
      u.kvh = (int)(g - u.j * KVH);
      u.at = (uint32_t)x - u.j * KVH;
      return u;
    }
    before = readlane(upto, 63);
  }
  return u;
}

// where part i of n parts of the tiles starts (products below 2^48: the quotient's floor is exact)
__device__ __forceinline__ int part_at(int tiles, int i, int n) {
  return n == 1 ? (i ? tiles : 0) : (int)((double)tiles * i / n);
}

// The parts' results: which rows of the call there are, per row and query head the place of
// its part 0 and the number of parts, then per unit and row maxima and sums, outputs.
struct PartRows {
  int *rows;
  uint2 *where;
  float2 *ml;
  float *o;
};
__device__ __forceinline__ PartRows part_rows(const PagedAttnArgs &a, const PagedGrid &gr, int rt) {
  PartRows p;
  p.rows = (int *)a.ws;
  p.where = (uint2 *)(p.rows + 4);
  p.ml = (float2 *)(p.where + (((size_t)a.c.t.M * a.H + 1) & ~(size_t)1));
  p.o = (float *)(p.ml + (size_t)gr.units * rt);
  return p;
}
size_t part_bytes(const PagedAttnArgs &a, const PagedGrid &gr, int rt, int hdp) {
  return 16 + 8 * (((size_t)a.c.t.M * a.H + 1) & ~(size_t)1) + (size_t)gr.units * rt * (8 + 4 * (size_t)hdp);
}

// q in units of log2, so that a product is an exponent, in two 16-bit parts.  A row is
// brought into the parts' range by a power of two (up; down: its inverse) where its largest
// is outside [2^-4, 2^15) (below, the low parts' steps of 2^-24 would count).
template <int N>
__device__ __forceinline__ void split_row(float (&v)[N][8], float big, v4u (&hi)[N], v4u (&lo)[N], float *up, float *down, bool *plain) {
  int e = 0;
  if (!(big >= 0.0625f && big < 32768.0f) && big > 0.0f)
    e = min(max(14 - ((int)(__float_as_uint(big) >> 23) - 127), -126), 100);
  *up = __uint_as_float((uint32_t)(e + 127) << 23);
  *down = __uint_as_float((uint32_t)(127 - e) << 23);
  *plain = __ballot(e != 0) == 0;
#pragma unroll
  for (int k = 0; k < N; k++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float x = v[k][2 * j] * *up, y = v[k][2 * j + 1] * *up;
      const Parts f = split2(x, y);
      hi[k][j] = f.hi;
      lo[k][j] = (uint32_t)f2h(x - h2f((uint16_t)f.hi)) | (uint32_t)f2h(y - h2f((uint16_t)(f.hi >> 16))) << 16;
    }
}
__device__ __forceinline__ void read8(float (&v)[8], const float *q, bool in, float f, float &big) {
  float4 x = {0.0f, 0.0f, 0.0f, 0.0f}, y = x;
  if (in) {
    x = *reinterpret_cast<const float4 *>(q);
    y = *reinterpret_cast<const float4 *>(q + 4);
  }
  v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    v[j] *= f;
    big = fmaxf(big, fabsf(v[j]));
  }
}

// two weights in two 16-bit parts each, the nearest and the nearest of the rest
__device__ __forceinline__ Parts split_near(float x, float y, float minus) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2h hi = __builtin_convertvector((v2f{x, y}), v2h);
  const v2f lo = {__builtin_fmaf((float)hi.x, minus, x), __builtin_fmaf((float)hi.y, minus, y)};
  return Parts{__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, __builtin_convertvector(lo, v2h))};
}
// -1, unknown to the compiler: it would make two instructions of a mixed-precision difference
__device__ __forceinline__ float minus_one() {
  float m = -1.0f;
  asm volatile("" : "+s"(m));
  return m;
}

// which of the positions p0 .. p0 + 63 the token at position t sees
__device__ __forceinline__ uint64_t tile_mask(const PagedAttnArgs &a, int p0, int t) {
  uint64_t m = low_bits(t - p0 + 1);
  if (a.window && t >= a.window) m &= ~low_bits(t - a.window + 1 - p0) | low_bits(min(a.sinks, t) - p0);
  return m;
}

// values that are not finite become 0; whether there was one
__device__ __forceinline__ bool only_finite(v4u &v) {
  uint32_t hit = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    // an exponent of all ones carries out of its field
    const uint32_t e = v[j] & 0x7C007C00u;
    const uint32_t bad = ((e & 0x7C00u) + 0x0400u) & 0x8000u, bad2 = ((e >> 16) + 0x0400u) & 0x8000u;
    v[j] &= ~((bad ? 0xFFFFu : 0u) | (bad2 ? 0xFFFF0000u : 0u));
    hit |= bad | bad2;
  }
  return hit != 0;
}

// the maximum and the sum over lanes l and l + 32
__device__ __forceinline__ float pair_max(float v) {
  const v2u x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x.x), __uint_as_float(x.y));
}
__device__ __forceinline__ float pair_sum(float v) {
  const v2u x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x.x) + __uint_as_float(x.y);
}

__device__ __forceinline__ v16f mma32(v4u a, v4u b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// The wait between the last of the scores' products and what reads them, 12 states for these
// instructions (8 passes): in a block behind a branch the compiler can leave it out (it did for
// the maximum, behind the test of `plain`: heads of 65 to 128 came out without the last products' low
// parts, now and then)
__device__ __forceinline__ void settle(v16f (&v)[1]) { asm volatile("s_nop 11" : "+v"(v[0])); }
__device__ __forceinline__ void settle(v16f (&v)[2]) { asm volatile("s_nop 11" : "+v"(v[0]), "+v"(v[1])); }
// and for those of 4 passes, 8 states
__device__ __forceinline__ void settle(v4f (&v)[2]) { asm volatile("s_nop 7" : "+v"(v[0]), "+v"(v[1])); }
__device__ __forceinline__ void settle(v4f (&v)[4]) { asm volatile("s_nop 7" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3])); }

// The operand of 32 elements' values at 16 positions, two reads of four rows of the tile:
// lane l of 16 names 8 bytes of row l / 4 and gets element l of the four rows.
template <int HD>
__device__ __forceinline__ v4u read_v32(uint32_t at, int row) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4s lv4s;
  const v2u x = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s *)(uintptr_t)(at + 2 * HD * row)));
  const v2u y = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s *)(uintptr_t)(at + 2 * HD * (row + 8))));
  return v4u{x.x, x.y, y.x, y.y};
}

// Rows of a unit that takes no part
template <int RT>
__device__ __forceinline__ void mark_rows(const PagedAttnArgs &a, const PagedGrid &gr, const Unit &u) {
  const int G = a.G, hd = a.c.hd, r0 = u.rt * RT, n = min(u.s.n * G - r0, RT);
  for (int e = threadIdx.x; e < n * hd; e += blockDim.x) {
    const int r = r0 + e / hd;
    a.out[(size_t)(u.s.start + r / G) * a.ldo + (size_t)(u.kvh * G + r % G) * hd + e % hd] = __builtin_nanf("");
  }
  if (gr.target)
    for (int e = threadIdx.x; e < n; e += blockDim.x)
      part_rows(a, gr, RT).where[(size_t)(u.s.start + (r0 + e) / G) * a.H + u.kvh * G + (r0 + e) % G] = make_uint2(0, 1);
}
__device__ __forceinline__ void mark_call(const PagedAttnArgs &a, const PagedGrid &gr, long x) {
  if (gr.target && x == 0 && threadIdx.x == 0) {
    int *rows = (int *)a.ws;
    rows[0] = a.c.t.start ? a.c.t.start[0] : 0;
    rows[1] = a.c.t.start ? a.c.t.start[a.c.t.B] : a.c.t.M;
  }
}

// Single tokens: 16 rows of one KV head a block.  Each of its NW waves takes every
// NW-th of the part's steps of TP positions, without a barrier: keys come from the cache
// as the matrix instruction's operand, values through the wave's own tile in LDS, which
// transposes them; the next step's are on their way while a wave works on one.  The waves'
// results are joined in LDS.
// The chunks' kernel takes it for sequences of that few rows among others (24 sequences, one
// of 333 tokens, 14 / 2 x 64, 1500: 22.2 a call; with tiles of 128 for all 24.8).
//
// 64 x 1, 12 / 2 x 128 of int8, 4000: 32 where three caches take turns, 29.5 over and over on one, 118
// MB at 3.7 and 4.0 TB/s (a plain sum over and over on as many bytes 26.4); two steps on their way
// instead of one 33.  One sequence, 14 / 2 x 64 of fp16, 700: 10.3, the chain of the starts, the
// table, two steps' keys and the waves' join.
template <int HDP, int NW>
constexpr int step_lds() {
  const int tile = (HDP <= 64 ? 64 : 32) * HDP * 2, joined = 16 * (HDP + 4) * 4;
  return NW * (tile > joined ? tile : joined);
}
// URT: rows of a unit's places in the workspace
template <int HDP, int TYPE, int NW, int URT>
__device__ __forceinline__ void step_unit(const PagedAttnArgs &a, const PagedGrid &gr, const Unit &un, long x, char *lds, float2 (&ml)[NW][16]) {
  constexpr int RT = 16, NT = 64 * NW, TP = HDP <= 64 ? 64 : 32, PT = TP / 16, CPR = HDP / 8, KS = HDP / 32, DT = HDP / 16, ND = DT % 4 ? 2 : 4;
  constexpr int EB = TYPE == CACHE_F16 ? 2 : 1, VC = TYPE == CACHE_F16 ? 1 : 2;  // chunks of 8 elements in 16 bytes
  constexpr int LV = TP * CPR / VC / 64, PER = kTp / TP;
  constexpr bool WIDE = TYPE != CACHE_F16 && KS % 2 == 0;  // two chunks of keys in 16 bytes
  constexpr int LDO = HDP + 4;
  const EcPageSeq s = un.s;
  const int t = threadIdx.x, lane = t & 63, lr = lane & 15, lg = lane >> 4, hd = a.c.hd;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int G = a.G, rows = s.n * G, r0 = un.rt * RT;
  const int ta = r0 / G, tb = (min(rows, r0 + RT) - 1) / G;
  const Tiles tl = tiles_of(a, s, ta, tb);
  const int tile0 = part_at(tl.n, un.j, un.n), tile1 = part_at(tl.n, un.j + 1, un.n);
  const int steps = (tile1 - tile0) * PER;
  const auto pos_of = [&](int i) { return tl.at(tile0 + i / PER) + i % PER * TP; };

  // ---- a step's keys and values ----
  bool bad = false;
  int pos = 0, id = 0;
  uint32_t crow = 0;  // lane l's position's row in the cache
  v4u kr[PT][WIDE ? KS / 2 : KS], vr[LV];
  uint16_t ksc[PT], vsc[LV];
  const auto find = [&](int i) {
    const int p = pos_of(i) + (lane & (TP - 1));
    pos = p >= tl.lo || p < tl.sinks ? min(p, s.past + tb) : tl.lo;
    id = page_id(a.c.t, un.c, pos);
  };
  const auto load = [&] {
    crow = page_row(a.c.t, id, pos, un.kvh, &bad);
#pragma unroll
    for (int pt = 0; pt < PT; pt++) {
      const uint32_t row = (uint32_t)__shfl((int)crow, 16 * pt + lr, 64);
      const char *k = (const char *)a.c.k + (size_t)row * hd * EB;
      if constexpr (TYPE != CACHE_F16) ksc[pt] = a.c.ks[row];
#pragma unroll
      for (int c = 0; c < (WIDE ? KS / 2 : KS); c++) {
        kr[pt][c] = v4u{0, 0, 0, 0};
        if constexpr (TYPE == CACHE_F16) {
          if (32 * c + 8 * lg < hd) kr[pt][c] = *(const v4u *)(k + 2 * (32 * c + 8 * lg));
        } else if constexpr (WIDE) {
          if (lg * (HDP / 4) + 16 * c < hd) kr[pt][c] = *(const v4u *)(k + lg * (HDP / 4) + 16 * c);
        } else {
          if (lg * (HDP / 4) + 8 * c < hd) {
            const v2u y = *(const v2u *)(k + lg * (HDP / 4) + 8 * c);
            kr[pt][c].x = y.x;
            kr[pt][c].y = y.y;
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < LV; u++) {
      const int ch = u * 64 + lane, r = ch / (CPR / VC), cc = ch % (CPR / VC) * VC;
      const uint32_t row = (uint32_t)__shfl((int)crow, r, 64);
      vr[u] = v4u{0, 0, 0, 0};
      if (8 * cc < hd) vr[u] = *(const v4u *)((const char *)a.c.v + ((size_t)row * hd + 8 * cc) * EB);
      if constexpr (TYPE != CACHE_F16) vsc[u] = a.c.vs[row];
    }
  };
  if (w < steps) {
    find(w);
    load();
    if (w + NW < steps) find(w + NW);
  }

  // ---- this lane's row of q; its elements in the order that the keys' have ----
  const int row = r0 + lr, rq = min(row, rows - 1), token = rq / G, head = un.kvh * G + (rq - token * G);
  const int qpos = s.past + token;
  v4u qh[KS], ql[KS];
  float up, down;
  bool plain;
  {
    const float *q = a.q + (size_t)(s.start + token) * a.ldq + (size_t)head * hd;
    float v[KS][8], big = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; k++) {
      const int e = TYPE == CACHE_F16 ? 32 * k + 8 * lg : lg * (HDP / 4) + 8 * k;
      read8(v[k], q + e, e < hd, a.scale * 1.44269504f, big);
    }
    split_row(v, row_max(big), qh, ql, &up, &down, &plain);
  }

  // the values' LDS addresses in the tile's first 32 rows
  typedef __attribute__((address_space(3))) void lvoid;
  _Float16 *V = reinterpret_cast<_Float16 *>(lds) + w * TP * HDP;
  const uint32_t vbase = (uint32_t)(uintptr_t)(lvoid *)V;
  uint32_t vcol[DT];
#pragma unroll
  for (int d = 0; d < DT; d++) {
    const int r = 4 * lg + (lr >> 2);
    vcol[d] = (uint32_t)(r * HDP + ((2 * d + ((lr & 3) >> 1)) ^ swz<HDP>(r)) * 8 + 4 * (lr & 1)) * 2;
  }

  v4f o[DT], from = {0.0f, 0.0f, 0.0f, 0.0f};  // from: what the row's products start at
  const float minus = minus_one();
  float mx = -FLT_MAX, lim = -FLT_MAX, sum = 0.0f;
#pragma unroll
  for (int d = 0; d < DT; d++) o[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  for (int i = w; i < steps; i += NW) {
    const int p0 = pos_of(i);
    const bool edge = !(p0 + TP - 1 <= s.past + ta && (!a.window || p0 > s.past + tb - a.window || p0 + TP <= a.sinks));
    const uint32_t srow = crow;
    // ---- scores: sc[pt][r] of position 16 pt + 4 lg + r ----
    v4f sc[PT];
#pragma unroll
    for (int pt = 0; pt < PT; pt++) {
      sc[pt] = from;
#pragma unroll
      for (int k = 0; k < KS; k++) {
        v4u kf;
        if constexpr (TYPE == CACHE_F16) kf = kr[pt][k];
        else if constexpr (WIDE) kf = to_f16<TYPE>(k & 1 ? v2u{kr[pt][k / 2].z, kr[pt][k / 2].w} : v2u{kr[pt][k / 2].x, kr[pt][k / 2].y}, ksc[pt]);
        else kf = to_f16<TYPE>(v2u{kr[pt][k].x, kr[pt][k].y}, ksc[pt]);
        sc[pt] = mma(kf, qh[k], sc[pt]);
        sc[pt] = mma(kf, ql[k], sc[pt]);
      }
    }
    // ---- values into LDS ----
    bool inf = false;
#pragma unroll
    for (int u = 0; u < LV; u++) {
      const int ch = u * 64 + lane, r = ch / (CPR / VC), cc = ch % (CPR / VC) * VC;
#pragma unroll
      for (int c = 0; c < VC; c++) {
        v4u v;
        if constexpr (TYPE == CACHE_F16) v = vr[u];
        else v = to_f16<TYPE>(c ? v2u{vr[u].z, vr[u].w} : v2u{vr[u].x, vr[u].y}, vsc[u]);
        if (edge) inf |= only_finite(v);
        *reinterpret_cast<v4u *>(V + r * HDP + ((cc + c) ^ swz<HDP>(r)) * 8) = v;
      }
    }
    if (i + NW < steps) {
      load();
      if (i + 2 * NW < steps) find(i + 2 * NW);
    }

    // ---- weights ----
    settle(sc);
    if (edge) {
      const uint64_t on = tile_mask(a, p0, qpos) >> (4 * lg);
#pragma unroll
      for (int pt = 0; pt < PT; pt++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (!((on >> (16 * pt + r)) & 1)) sc[pt][r] = -__builtin_inff();
    }
    if (__builtin_expect(!plain, 0)) {
#pragma unroll
      for (int pt = 0; pt < PT; pt++)
#pragma unroll
        for (int r = 0; r < 4; r++) sc[pt][r] *= down;
    }
    float top = -FLT_MAX;
#pragma unroll
    for (int pt = 0; pt < PT; pt++)
#pragma unroll
      for (int r = 0; r < 4; r++) top = fmaxf(top, sc[pt][r]);
    if (__builtin_expect(__ballot(top > lim) != 0, 0)) {
      const float big = row_max(top);
      const bool first = mx == -FLT_MAX, move = big > (first ? -FLT_MAX : kLift);
      const float by = move ? big - kLift : 0.0f, back = first ? 0.0f : __builtin_amdgcn_exp2f(-by);
      if (move) {
        mx = first ? big : mx + by;
        lim = kLift + kRoom;
      }
      const float f = move || !first ? (kLift - mx) * up : 0.0f;
      from = v4f{f, f, f, f};
      sum *= back;
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int r = 0; r < 4; r++) o[d][r] *= back;
#pragma unroll
      for (int pt = 0; pt < PT; pt++)
#pragma unroll
        for (int r = 0; r < 4; r++) sc[pt][r] -= by;
    }
    v4u ph[PT / 2], pl[PT / 2];
    float here = 0.0f;
#pragma unroll
    for (int pt = 0; pt < PT; pt++) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        p[r] = __builtin_amdgcn_exp2f(sc[pt][r]);
        here += p[r];
      }
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const Parts f = split_near(p[2 * r], p[2 * r + 1], minus);
        ph[pt >> 1][2 * (pt & 1) + r] = f.hi;
        pl[pt >> 1][2 * (pt & 1) + r] = f.lo;
      }
    }
    sum += here;

    // ---- outputs: o[d][r] of element 16 d + 4 lg + r ----
#pragma unroll
    for (int u = 0; u < TP / 32; u++)
#pragma unroll
      for (int d = 0; d < DT; d += ND) {
        v4u vf[ND];
        if (u == 0) read_v<HDP, ND>(vcol + d, vbase, 0, vf);
        else read_v<HDP, ND>(vcol + d, vbase, 1, vf);
#pragma unroll
        for (int e = 0; e < ND; e++) {
          o[d + e] = mma(vf[e], ph[u], o[d + e]);
          o[d + e] = mma(vf[e], pl[u], o[d + e]);
        }
      }

    // values that are not finite, for the rows that see them
    if (__builtin_expect(__ballot(inf) != 0, 0)) {
      const uint64_t on = tile_mask(a, p0, qpos);
      for (int pp = 0; pp < TP; pp++) {
        const uint32_t r = (uint32_t)__shfl((int)srow, pp, 64);
        if ((on >> pp) & 1) {
#pragma unroll
          for (int d = 0; d < DT; d++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const int e = 16 * d + 4 * lg + k;
              if (e < hd && (cache_value(a.c.v, a.c.vs, TYPE, r, hd, e) & 0x7C00u) == 0x7C00u) o[d][k] = __builtin_nanf("");
            }
        }
      }
    }
  }

  // ---- the waves' results together ----
  float l = row_sum(sum);
  if (__ballot(bad)) l = __builtin_nanf("");
  __syncthreads();  // every wave is done with its tile
  float *wo = reinterpret_cast<float *>(lds) + (w * RT + lr) * LDO + 4 * lg;
#pragma unroll
  for (int d = 0; d < DT; d++) *reinterpret_cast<v4f *>(wo + 16 * d) = o[d];
  if (lg == 0) ml[w][lr] = make_float2(mx, l);
  __syncthreads();
  constexpr int LPR = NT / RT;
  const int jr = t / LPR, jc = t % LPR, jrow = r0 + jr;
  if (jrow >= rows) return;
  const int jt = jrow / G, jh = un.kvh * G + (jrow - jt * G);
  float m = -FLT_MAX, f[NW], jl = 0.0f;
#pragma unroll
  for (int k = 0; k < NW; k++) m = fmaxf(m, ml[k][jr].x);
#pragma unroll
  for (int k = 0; k < NW; k++) {
    f[k] = __builtin_amdgcn_exp2f(ml[k][jr].x - m);
    jl = __builtin_fmaf(ml[k][jr].y, f[k], jl);
  }
  float scale = 1.0f;
  float *to;
  if (gr.target) {
    const PartRows pr = part_rows(a, gr, URT);
    if (un.j == 0 && jc == 0) pr.where[(size_t)(s.start + jt) * a.H + jh] = make_uint2(un.at * URT + jr, un.n);
    to = pr.o + ((size_t)x * URT + jr) * HDP;
    if (un.n > 1 && jc == 0) pr.ml[(size_t)x * URT + jr] = make_float2(m, jl);
  }
  if (!gr.target || un.n == 1) {
    to = a.out + (size_t)(s.start + jt) * a.ldo + (size_t)jh * hd;
    scale = jl > 0.0f || jl != jl ? 1.0f / jl : 0.0f;
  }
  for (int e = 4 * jc; e < hd; e += 4 * LPR) {
    v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NW; k++) {
      const v4f y = *reinterpret_cast<const v4f *>(reinterpret_cast<const float *>(lds) + (k * RT + jr) * LDO + e);
#pragma unroll
      for (int c = 0; c < 4; c++) v[c] = __builtin_fmaf(y[c], f[k], v[c]);
    }
    *reinterpret_cast<v4f *>(to + e) = v * scale;
  }
}

template <int HDP, int TYPE, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn_step_kernel(PagedAttnArgs a, PagedGrid gr) {
  __shared__ __attribute__((aligned(16))) char lds[step_lds<HDP, NW>()];
  __shared__ float2 ml[NW][16];
  const long x = (long)blockIdx.y * gridDim.x + blockIdx.x;
  mark_call(a, gr, x);
  if (x >= gr.units) return;
  const Unit un = find_unit<16>(a, gr, x);
  if (un.c < 0) return;
  if (!ec_page_seq_ok(&a.c.t, un.s, a.max_past)) mark_rows<16>(a, gr, un);
  else step_unit<HDP, TYPE, NW, 16>(a, gr, un, x, lds, ml);
}

// Chunks of tokens: 128 rows of one KV head a block, 32 a wave; the waves share tiles of
// keys and values that the block brings to LDS in fp16, the next tile on its way into
// registers while the waves work on one.
//
// Products run transposed, K Q^T and V^T P^T, so that a lane keeps one row (lane & 31):
// the scores' accumulators hold 16 of each 32 positions, its maximum and sum need one
// exchange, with the lane 32 further on, and the weights are the second product's operand
// as they stand: half h of the lanes takes 4 h .. 4 h + 3 of every run of 8 positions.  The
// values, rows of the cache, are read for it by the transposing LDS load.
//
// fp32 by two 16-bit parts of q and of the weights (the keys and values are fp16 as they
// are): the parts' second products are a quarter of the time.  The scores' sums start at kLift -
// m (`from`, here and in the single tokens' form), so that they are exponents as they come; a
// step's rounding is then that of a number of up to kLift and the maximum's size instead of the
// sum's own.  Modelled on the CPU (2000 positions, queries and keys of unit variance) the
// outputs are 4.7e-7 off with it and 2.3e-7 without for heads of 64, 6.5e-7 and 2.7e-7 for
// 128; sums from 0 would take an addition a score, and their tests' bounds hold both.
//
// 1 x 512, 14 / 2 x 64 of e4m3, 7500: 44 to 47 by card, 0.60 to 0.65 PFLOP/s of products in two parts (a
// library's fp16 product reaches 1.15); up to 4 x 2048, 12 / 2 x 128 of fp16 from their start: 120 to 125 for
// 42 GFLOP, 132 for 47, 0.67 to 0.71; 10 to 20 more in the first tens of calls.  Matrix cores 34 to 44% and
// vector ALUs 45 to 53% busy: a tile takes a wave 2.3 us beside another wave, 1.5 alone.  Measured and not
// taken: tiles of 32 positions at 64 elements (chunk 51), with three waves a SIMD (57: spills),
// blocks of 256 rows (chunk 45, prompt 135), wave priorities, loads behind the barrier, keys a
// step ahead (all the same), a join by the last block of a row tile (chunk 52, 24 mixed sequences 32).
template <int HDP, int TYPE>
__global__ __launch_bounds__(256, 2) void attn_chunk_kernel(PagedAttnArgs a, PagedGrid gr) {
  constexpr int RT = 128, NT = 256, TP = HDP <= 64 ? 64 : 32, PT = TP / 32, PER = kTp / TP, CPR = HDP / 8, KS = HDP / 16, DT = HDP / 32,
                LPT = (TP * CPR + NT - 1) / NT;
  extern __shared__ __attribute__((aligned(16))) _Float16 lds[];  // [2 buffers][K, V][TP][HDP]
  __shared__ __attribute__((aligned(16))) int infinite[2][4];  // of a buffer: which wave brought values that are not finite
  const long x = (long)blockIdx.y * gridDim.x + blockIdx.x;
  mark_call(a, gr, x);
  if (x >= gr.units) return;
  const Unit un = find_unit<RT>(a, gr, x);
  if (un.c < 0) return;
  const EcPageSeq s = un.s;
  if (!ec_page_seq_ok(&a.c.t, s, a.max_past)) {
    mark_rows<RT>(a, gr, un);
    return;
  }
  if (s.n * a.G <= 16) {
    __shared__ float2 ml[4][16];
    step_unit<HDP, TYPE, 4, RT>(a, gr, un, x, (char *)lds, ml);
    return;
  }
  const int t = threadIdx.x, lane = t & 63, ln = lane & 31, h = lane >> 5, hd = a.c.hd;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int G = a.G, rows = s.n * G, r0 = un.rt * RT;
  const int ta = r0 / G, tb = (min(rows, r0 + RT) - 1) / G;
  const Tiles tl = tiles_of(a, s, ta, tb);
  const int tile0 = part_at(tl.n, un.j, un.n), tile1 = part_at(tl.n, un.j + 1, un.n);
  const int steps = (tile1 - tile0) * PER;
  const auto pos_of = [&](int i) { return tl.at(tile0 + i / PER) + i % PER * TP; };

  // ---- the tiles' way into LDS ----
  // a thread's chunks of 8 elements; rows that no token of the block sees are another's that is
  bool bad = false;
  int pos[LPT], id[LPT];
  Raw8<TYPE> kr[LPT], vr[LPT];
  uint16_t ksc[LPT], vsc[LPT];
  const auto find = [&](int i) {
#pragma unroll
    for (int u = 0; u < LPT; u++) {
      const int p = pos_of(i) + min((u * NT + t) / CPR, TP - 1);
      pos[u] = p >= tl.lo || p < tl.sinks ? min(p, s.past + tb) : tl.lo;
      id[u] = page_id(a.c.t, un.c, pos[u]);
    }
  };
  const auto load = [&] {
#pragma unroll
    for (int u = 0; u < LPT; u++) {
      const uint32_t row = page_row(a.c.t, id[u], pos[u], un.kvh, &bad);
      const int cc = (u * NT + t) % CPR;
      kr[u] = vr[u] = Raw8<TYPE>{};
      if (8 * cc < hd) {
        constexpr int B = TYPE == CACHE_F16 ? 2 : 1;
        const size_t at = ((size_t)row * hd + 8 * cc) * B;
        kr[u] = *(const Raw8<TYPE> *)((const char *)a.c.k + at);
        vr[u] = *(const Raw8<TYPE> *)((const char *)a.c.v + at);
      }
      if constexpr (TYPE != CACHE_F16) {
        ksc[u] = a.c.ks[row];
        vsc[u] = a.c.vs[row];
      }
    }
  };
  if (steps) {
    find(0);
    load();
    if (steps > 1) find(1);
  }

  // ---- this lane's row of q ----
  const int row = r0 + 32 * w + ln, rq = min(row, rows - 1), token = rq / G, head = un.kvh * G + (rq - token * G);
  const int qpos = s.past + token;
  v4u qh[KS], ql[KS];
  float up, down;
  bool plain;  // no row of the wave scaled
  {
    const float *q = a.q + (size_t)(s.start + token) * a.ldq + (size_t)head * hd + 8 * h;
    float v[KS][8], big = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; k++) read8(v[k], q + 16 * k, 16 * k + 8 * h < hd, a.scale * 1.44269504f, big);
    split_row(v, pair_max(big), qh, ql, &up, &down, &plain);
  }

  // the values' LDS addresses in a tile's first 8 rows (rows 8, 16 .. further on have the
  // same swizzle)
  typedef __attribute__((address_space(3))) void lvoid;
  const uint32_t vbase = (uint32_t)(uintptr_t)(lvoid *)lds + 2 * TP * HDP;
  uint32_t vcol[DT];
#pragma unroll
  for (int d = 0; d < DT; d++) {
    const int l = lane & 15, r = 4 * h + (l >> 2);
    vcol[d] = (uint32_t)(r * HDP + ((4 * d + 2 * ((lane >> 4) & 1) + ((l & 3) >> 1)) ^ swz<HDP>(r)) * 8 + 4 * (l & 1)) * 2;
  }

  uint64_t nans = 0;  // elements of o that an infinity or NaN reaches
  v16f o[DT];
  const float minus = minus_one();
  v16f from;  // what the row's products start at, as the matrix instruction takes it
#pragma unroll
  for (int i = 0; i < 16; i++) from[i] = 0.0f;
  float mx = -FLT_MAX, lim = -FLT_MAX, sum = 0.0f;
#pragma unroll
  for (int d = 0; d < DT; d++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[d][i] = 0.0f;

  constexpr int kBuf = 2 * TP * HDP;  // elements of a buffer: K, then V
  // Step i's tile from registers into LDS, the next one on its way.  EDGE: a tile that some
  // rows see in part: what they do not see has weight 0, and its values must be finite for that
  // to be nothing.  Whether one was not.
  const auto stage = [&](auto edge, int i) {
    constexpr bool EDGE = decltype(edge)::value;
    _Float16 *K = lds + (i & 1) * kBuf, *V = K + TP * HDP;
    bool inf = false;
#pragma unroll
    for (int u = 0; u < LPT; u++) {
      const int r = (u * NT + t) / CPR, cc = (u * NT + t) % CPR, at = r * HDP + (cc ^ swz<HDP>(r)) * 8;
      if (TP * CPR % NT && r >= TP) break;
      *reinterpret_cast<v4u *>(K + at) = to_f16<TYPE>(kr[u], ksc[u]);
      v4u v = to_f16<TYPE>(vr[u], vsc[u]);
      if constexpr (EDGE) inf |= only_finite(v);
      *reinterpret_cast<v4u *>(V + at) = v;
    }
    if (i + 1 < steps) {
      load();
      if (i + 2 < steps) find(i + 2);
    }
    if constexpr (EDGE) {
      const int any = __ballot(inf) != 0;
      if (lane == 0) infinite[i & 1][w] = any;
    }
    // the tile is there, and every wave is done with the one before it; the loads of the next
    // one go on
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  const auto compute = [&](auto edge, int i) {
    constexpr bool EDGE = decltype(edge)::value;
    const int p0 = pos_of(i);
    const _Float16 *K = lds + (i & 1) * kBuf;
    uint32_t vat[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) vat[d] = vbase + 2 * (uint32_t)((i & 1) * kBuf) + vcol[d];

    // ---- scores: sc[pt][i] of position 32 pt + 8 (i / 4) + 4 h + i % 4 ----
    v16f sc[PT];
#pragma unroll
    for (int pt = 0; pt < PT; pt++) sc[pt] = from;
#pragma unroll
    for (int k = 0; k < KS; k++) {
      v4u kf[PT];
#pragma unroll
      for (int pt = 0; pt < PT; pt++) {
        const int r = 32 * pt + ln;
        kf[pt] = *reinterpret_cast<const v4u *>(K + r * HDP + ((2 * k + h) ^ swz<HDP>(r)) * 8);
      }
#pragma unroll
      for (int pt = 0; pt < PT; pt++) sc[pt] = mma32(kf[pt], qh[k], sc[pt]);
#pragma unroll
      for (int pt = 0; pt < PT; pt++) sc[pt] = mma32(kf[pt], ql[k], sc[pt]);
    }
    settle(sc);

    // ---- weights ----
    if constexpr (EDGE) {
      const uint64_t on = tile_mask(a, p0, qpos) >> (4 * h);
#pragma unroll
      for (int pt = 0; pt < PT; pt++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (!((on >> (32 * pt + 8 * (i >> 2) + (i & 3))) & 1)) sc[pt][i] = -__builtin_inff();
    }
    if (__builtin_expect(!plain, 0)) {
#pragma unroll
      for (int pt = 0; pt < PT; pt++)
#pragma unroll
        for (int i = 0; i < 16; i++) sc[pt][i] *= down;
    }
    // exponents of the weights already (the sums began at kLift - mx): kRoom above kLift the
    // maximum moves
    float top = -FLT_MAX;
#pragma unroll
    for (int pt = 0; pt < PT; pt++)
#pragma unroll
      for (int i = 0; i < 16; i++) top = fmaxf(top, sc[pt][i]);
    if (__builtin_expect(__ballot(top > lim) != 0, 0)) {
      const float big = pair_max(top);
      const bool first = mx == -FLT_MAX, move = big > (first ? -FLT_MAX : kLift);
      const float by = move ? big - kLift : 0.0f, back = first ? 0.0f : __builtin_amdgcn_exp2f(-by);
      if (move) {
        mx = first ? big : mx + by;
        lim = kLift + kRoom;
      }
      const float f = move || !first ? (kLift - mx) * up : 0.0f;
#pragma unroll
      for (int i = 0; i < 16; i++) from[i] = f;
      sum *= back;
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] *= back;
#pragma unroll
      for (int pt = 0; pt < PT; pt++)
#pragma unroll
        for (int i = 0; i < 16; i++) sc[pt][i] -= by;
    }
    // the tile's weights are added up before they meet the sum so far: one by one, those
    // below half a step of it would be lost
    v4u ph[PT][2], pl[PT][2];
    float here[2] = {0.0f, 0.0f};
#pragma unroll
    for (int pt = 0; pt < PT; pt++)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float p = __builtin_amdgcn_exp2f(sc[pt][i]), q = __builtin_amdgcn_exp2f(sc[pt][i + 1]);
        here[0] += p;
        here[1] += q;
        const Parts f = split_near(p, q, minus);
        ph[pt][i >> 3][(i & 7) >> 1] = f.hi;
        pl[pt][i >> 3][(i & 7) >> 1] = f.lo;
      }
    sum += here[0] + here[1];

    // ---- outputs: o[d][i] of element 32 d + 8 (i / 4) + 4 h + i % 4 ----
#pragma unroll
    for (int pt = 0; pt < PT; pt++) {
      v4u vf[2][DT];
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int d = 0; d < DT; d++) vf[c][d] = read_v32<HDP>(vat[d], 32 * pt + 16 * c);
#pragma unroll
      for (int c = 0; c < 2; c++) {
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = mma32(vf[c][d], ph[pt][c], o[d]);
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = mma32(vf[c][d], pl[pt][c], o[d]);
      }
    }

    // values that are not finite, for the rows that see them
    v4i any = {0, 0, 0, 0};
    if constexpr (EDGE) any = *reinterpret_cast<const v4i *>(infinite[i & 1]);
    if (EDGE && __builtin_expect((any.x | any.y | any.z | any.w) != 0, 0)) {
      const uint64_t on = tile_mask(a, p0, qpos);
      for (int pp = 0; pp < TP && p0 + pp <= s.past + tb; pp++) {
        if (!((on >> pp) & 1)) continue;
        bool none = false;
        const uint32_t r = page_row(a.c.t, page_id(a.c.t, un.c, p0 + pp), p0 + pp, un.kvh, &none);
        for (int e = 0; e < 16 * DT; e++) {
          const int at = 32 * (e >> 4) + 8 * ((e & 15) >> 2) + 4 * h + (e & 3);
          if (at < hd && (cache_value(a.c.v, a.c.vs, TYPE, r, hd, at) & 0x7C00u) == 0x7C00u) nans |= 1ull << e;
        }
      }
    }
  };
  // the steps whose tiles every token sees whole, and those in front of and behind them (the
  // first tokens' always: they are few)
  const int low = max(a.window ? s.past + tb - a.window + 1 : 0, 0) - tl.first * kTp, step0 = (tl.front - tile0) * PER;
  const int whole0 = min(max(step0 + (max(low, 0) + TP - 1) / TP, 0), steps);
  const int whole1 = min(max(step0 + (s.past + ta + 1 - tl.first * kTp) / TP, whole0), steps);
  if (r0 + 32 * w < rows) {
    int i = 0;
    for (; i < whole0; i++) {
      stage(std::true_type{}, i);
      compute(std::true_type{}, i);
    }
    for (; i < whole1; i++) {
      stage(std::false_type{}, i);
      compute(std::false_type{}, i);
    }
    for (; i < steps; i++) {
      stage(std::true_type{}, i);
      compute(std::true_type{}, i);
    }
  } else {  // no row of the wave's own: it brings its share of the tiles
    for (int i = 0; i < steps; i++)
      if (i < whole0 || i >= whole1) stage(std::true_type{}, i);
      else stage(std::false_type{}, i);
  }
  if (__builtin_expect(nans != 0, 0)) {
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
      for (int i = 0; i < 16; i++)
        if ((nans >> (16 * d + i)) & 1) o[d][i] = __builtin_nanf("");
  }

  const bool none = __syncthreads_or(bad);
  const float l = none ? __builtin_nanf("") : pair_sum(sum);
  if (row >= rows) return;
  if (gr.target) {
    const PartRows pr = part_rows(a, gr, RT);
    if (un.j == 0 && h == 0)
      pr.where[(size_t)(s.start + token) * a.H + head] = make_uint2(un.at * RT + 32 * w + ln, un.n);
    if (un.n > 1) {
      const size_t at = (size_t)x * RT + 32 * w + ln;
      if (h == 0) pr.ml[at] = make_float2(mx, l);
      if (tile0 == tile1) return;
      float *po = pr.o + at * HDP + 4 * h;
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          *reinterpret_cast<float4 *>(po + 32 * d + 8 * i) = make_float4(o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
      return;
    }
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  float *out = a.out + (size_t)(s.start + token) * a.ldo + (size_t)head * hd + 4 * h;
#pragma unroll
  for (int d = 0; d < DT; d++)
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (32 * d + 8 * i + 4 * h < hd)
        *reinterpret_cast<float4 *>(out + 32 * d + 8 * i) =
            make_float4(o[d][4 * i] * inv, o[d][4 * i + 1] * inv, o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv);
}

// Joins the parts' outputs: per row the largest of their maxima, the sums and outputs
// brought to it.  HDP / 4 lanes a row (a power of two of them: 24 of 32 at 96).
template <int HDP>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(PagedAttnArgs a, PagedGrid gr, int rt) {
  constexpr int LPR = HDP == 96 ? 32 : HDP / 4, RPB = 256 / LPR, kRead = 8;
  const int li = threadIdx.x % LPR;
  const long r = (long)blockIdx.x * RPB + threadIdx.x / LPR;
  if (r >= (long)a.c.t.M * a.H) return;
  const PartRows pr = part_rows(a, gr, rt);
  const int token = (int)(r / a.H);
  if (token < pr.rows[0] || token >= pr.rows[1]) return;
  const uint2 where = pr.where[r];
  const size_t each = (size_t)a.c.t.KVH * rt;
  const int n = (int)where.y;
  // (where the starts do not ascend, a row's numbers may be an earlier call's)
  if (n < 2 || where.x + (size_t)(n - 1) * each >= (size_t)gr.units * rt || 4 * li >= a.c.hd) return;
  float m = -FLT_MAX, l = 0.0f;
  float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = 0; i0 < n; i0 += kRead) {
    float2 u[kRead];
    float4 v[kRead];
#pragma unroll
    for (int i = 0; i < kRead; i++) {
      const size_t at = where.x + (size_t)min(i0 + i, n - 1) * each;
      u[i] = pr.ml[at];
      v[i] = *reinterpret_cast<const float4 *>(pr.o + at * HDP + 4 * li);
    }
    float big = m;
#pragma unroll
    for (int i = 0; i < kRead; i++)
      if (i0 + i < n) big = fmaxf(big, u[i].x);
    const float back = __builtin_amdgcn_exp2f(m - big);
    m = big;
    l *= back;
    o = make_float4(o.x * back, o.y * back, o.z * back, o.w * back);
#pragma unroll
    for (int i = 0; i < kRead; i++)
      if (i0 + i < n && u[i].y != 0.0f) {  // (outputs of a part without tiles are not there)
        const float f = __builtin_amdgcn_exp2f(u[i].x - m);
        l = __builtin_fmaf(u[i].y, f, l);
        o.x = __builtin_fmaf(v[i].x, f, o.x);
        o.y = __builtin_fmaf(v[i].y, f, o.y);
        o.z = __builtin_fmaf(v[i].z, f, o.z);
        o.w = __builtin_fmaf(v[i].w, f, o.w);
      }
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  *reinterpret_cast<float4 *>(a.out + (size_t)token * a.ldo + (size_t)(r - (long)token * a.H) * a.c.hd + 4 * li) =
      make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// heads and rows that the matrix-core forms' tiles and 16-byte accesses can take, whose rows
// (of query heads) count in an int, and no more blocks of sequences without rows than that
bool tiles_ok(const PagedAttnArgs &a) {
  if ((long)a.c.t.M * a.H > 1L << 30 || (long)a.c.t.B * a.c.t.KVH > 1L << 30) return false;
  const uintptr_t p = (uintptr_t)a.q | (uintptr_t)a.c.k | (uintptr_t)a.c.v | (uintptr_t)a.out;
  return a.c.hd % 16 == 0 && a.c.hd <= 128 && !(p & 15) && a.ldq % 4 == 0 && a.ldo % 4 == 0;
}
int padded(int hd) { return (hd + 31) / 32 * 32; }

// Rows of a tile: 16 where a sequence has on average no more (8 x 1 and x 2, 12 / 2 x 128, 4000: 10.6 + 4.7
// and 11.1 + 4.7 with the join, in tiles of 128 10.8 + 6.8 and 12.0 + 6.8; 8 x 48, 12 / 12 x 64: 36 and 33).
// The average says little of the longest chunk: where one stands among single tokens either may be
// faster (12 / 12 x 64 over 4000, a call in tiles of 16 and of 128: 512 tokens among 64 sequences 112 and 109, among 40
// 84 and 101, among 35 78 and 62; 300 among 24 over 2000 30 and 58; 64 among 64 87 and 95; 12 / 2 x 128: 150 among 64 51
// and 57).  How long the chunks are is in device memory, which the host does not read.
int tile_rows(const PagedAttnArgs &a) { return (long)a.c.t.M * a.G <= 16L * a.c.t.B ? 16 : 128; }

PagedGrid paged_grid(const PagedAttnArgs &a) {
  const int rt = tile_rows(a), KVH = a.c.t.KVH;
  const long tiles = (long)a.c.t.M * a.G / rt + a.c.t.B, places = 512 / KVH;
  PagedGrid g;
  // (chunks: 1 x 8, 12 / 2 x 128, 4000: 11.7 + 6.9 with parts of two tiles, 15.6 + 4.6 of four)
  g.least = rt == 16 ? 4 : 2;
  long left = places - tiles;
  if (left < places / 2) left = places / 2;
  if (left < 1) left = 1;
  // Not split: texts that one block is through with before a join is, single tokens' up to 1024
  // positions (1 x 1, 14 / 2 x 64: 10.3 against 7.8 + 4.1 at 900, 14.8 against 7.9 + 3.9 at 2000), of wider heads 640
  // (12 / 2 x 128: 11.1 against 9.4 + 3.9 at 500, 15.3 against 9.9 + 4.0 at 900).  Whole calls of fp16 back to
  // back, unsplit against split, whose join's launch is then partly hidden: 8 / 1 x 32 8.1 against 8.6 at 1024, 9.6
  // against 8.7 at 1500; 14 / 2 x 64 9.9 against 10.4 at 640, 12.8 against 10.4 at 1024; 16 / 4 x 96 10.5 against 12.6 at
  // 500, 13.1 against 12.5 at 640; 12 / 2 x 128 13.4 against 14.8 at 500, 17.7 against 14.8 at 640.  And calls whose row tiles fill
  // the chip several times without (600 x 1, 12 / 2 x 128, 1000: 75, split 101; 60 x 100, 12 / 12 x 64, 1000: 79, split 72).
  const long new_rows = rt == 16 ? a.c.t.M / a.c.t.B + 1 : a.c.t.M;
  long span = a.max_past + new_rows;
  if (a.window && a.window + new_rows + a.sinks < span) span = a.window + new_rows + a.sinks;
  g.target = tiles * KVH <= (rt == 128 ? 2048 : 1024) && span > (rt == 128 ? g.least * kTp : a.c.hd <= 64 ? 1024 : 640) ? (int)left : 0;
  g.places = (int)(places < 1 ? 1 : places);
  g.units = (g.target && tiles + g.target < g.places ? g.places : tiles + g.target) * KVH;
  return g;
}

template <int HDP, int TYPE>
hipError_t launch_paged(const PagedAttnArgs &a, hipStream_t st) {
  const PagedGrid g = paged_grid(a);
  const long row = g.units < kGridRow ? g.units : kGridRow;
  const dim3 grid((unsigned)row, (unsigned)((g.units + row - 1) / row));
  // eight waves a block where every block has a CU to itself (64 x 1, 12 / 2 x 128, 300: 10.3, with four
  // 11.2), four where they share one (100 x 1, 12 / 12 x 64, 300: 27, with eight 39) or are joined
  if (tile_rows(a) == 16 && (g.target || g.units > 256)) klaunch((attn_step_kernel<HDP, TYPE, 4>), grid, dim3(256), 0, st, a, g);
  else if (tile_rows(a) == 16) klaunch((attn_step_kernel<HDP, TYPE, 8>), grid, dim3(512), 0, st, a, g);
  else klaunch((attn_chunk_kernel<HDP, TYPE>), grid, dim3(256), std::max(2 * 2 * (HDP <= 64 ? 64 : 32) * HDP * 2, step_lds<HDP, 4>()), st, a, g);
  return hipGetLastError();
}
template <int HDP>
hipError_t launch_paged(const PagedAttnArgs &a, hipStream_t st) {
  if (a.c.type == CACHE_F16) return launch_paged<HDP, CACHE_F16>(a, st);
  if (a.c.type == CACHE_I8) return launch_paged<HDP, CACHE_I8>(a, st);
  return launch_paged<HDP, CACHE_E4M3>(a, st);
}
template <int HDP>
hipError_t launch_join(const PagedAttnArgs &a, hipStream_t st) {
  constexpr int rpb = 256 / (HDP == 96 ? 32 : HDP / 4);
  klaunch((attn_paged_join_kernel<HDP>), dim3((unsigned)(((long)a.c.t.M * a.H + rpb - 1) / rpb)), dim3(256), 0, st, a, paged_grid(a),
          tile_rows(a));
  return hipGetLastError();
}

}  // namespace

int attention_paged_max_hd() { return kPagedMaxHd; }

bool attention_paged_joins(const PagedAttnArgs &a) { return tiles_ok(a) && paged_grid(a).target > 0; }

size_t attention_paged_workspace(const PagedAttnArgs &a) {
  return attention_paged_joins(a) ? part_bytes(a, paged_grid(a), tile_rows(a), padded(a.c.hd)) : 0;
}

hipError_t attention_paged(const PagedAttnArgs &a, hipStream_t st) {
  if (tiles_ok(a)) {
    if (a.c.hd <= 32) return launch_paged<32>(a, st);
    if (a.c.hd <= 64) return launch_paged<64>(a, st);
    if (a.c.hd <= 96) return launch_paged<96>(a, st);
    return launch_paged<128>(a, st);
  }
  klaunch(attn_paged_any_kernel, dim3(a.c.t.M, a.H), dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t attention_paged_join(const PagedAttnArgs &a, hipStream_t st) {
  if (a.c.hd <= 32) return launch_join<32>(a, st);
  if (a.c.hd <= 64) return launch_join<64>(a, st);
  if (a.c.hd <= 96) return launch_join<96>(a, st);
  return launch_join<128>(a, st);
}

}  // namespace ec
