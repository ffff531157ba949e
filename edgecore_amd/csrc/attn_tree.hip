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
#include <type_traits>

#include "attn_parts.h"
#include "ec_device.h"
#include "ec_kernels.h"

namespace ec {

namespace {

// the first cached position that a node of this depth sees
__device__ __forceinline__ int window_lo(int window, int past, int depth) {
  return window && past + depth >= window ? min(past + depth - window + 1, past) : 0;
}

// The form for any head size and alignment: one block per (node, head), tiles
// of 256 positions, a position per thread for the scores and an element of the
// head per thread for the sums, with the running maximum and sum.  Every query head
// reads its keys and values anew, a thread a whole key, and nothing is split over the
// positions: calls of 8 nodes of 14 / 2 heads over 700 rows take 41 us at head size 64
// (the matrix-core form and its join 10.6), 53 at 80, 75 at 112, 143 at 256; 16 one-token
// sequences of 12 / 12 heads over 1000 rows 96 (17), 124, 182 and 353; 8 trees of 16 nodes,
// 12 / 2 heads of 80, over 4000 rows 530 (22 at head size 96).
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
    const int p = tree_parent(tree_parent_read(a.t, b), s.n, &ok);
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
  const int lo = window_lo(a.window, s.past, mydepth);
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
      // in sums of 16 positions, these in the tile's: one by one, weights below half a step of
      // what there is would be lost (32000 positions beside one that has 0.99: 5e-5 of the outputs)
      float tile = 0.0f;
      if (g < groups && d < a.hd)
        for (int j0 = g; j0 < n; j0 += 16 * groups) {
          float some = 0.0f;
          for (int j = j0; j < min(n, j0 + 16 * groups); j += groups)
            if (p_s[j] >= 0.0f) some = __builtin_fmaf(p_s[j], h2f(a.vc[base + (size_t)(p0 + j) * kv + d]), some);
          tile += some;
        }
      acc[r] = __builtin_fmaf(acc[r], back, tile);
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

// The matrix-core form (head sizes 32, 64, 96, 128).  One KV head serves G = H /
// KVH query heads of n nodes: R = n G rows that share its keys and values.  A
// block of NW waves takes 16 NW rows of one KV head and a part of the positions, 64
// at a time: keys and values go from the cache straight into LDS, the next tile
// while the waves work on one.
//
// Products run transposed, K Q^T and V^T P^T, so that a lane keeps one row
// (lane & 15): the scores' accumulators hold 16 positions of it, its maximum and
// sum need two exchanges with the other three groups of 16 lanes, and the
// weights are the second product's operand as they stand: a matrix
// instruction's 32 positions may come in any order that both operands share, so
// lane group g takes 4 g .. 4 g + 3 of two runs of 16.  The values, rows of the
// cache, are read for it by the transposing LDS load.
//
// fp32 by two 16-bit parts: q = hi + lo (a row whose largest is outside [2^-4, 2^15)
// under a power of two that brings it to 2^14: its low part's steps of 2^-24 are below
// 2^-20 of the largest at worst), weights = hi + lo (off by 2^-23 of a weight or, below
// 2^-1, by 2^-24 at most); keys and values are 16 bits as they are, so two products give
// each sum.  The parts are of 2^12 times the weights, so that 2^-24 is 2^-36 of the
// running maximum's: behind a token that takes most of the weight stand thousands of
// small ones that matter together.  The maximum is raised only when a score passes it by a
// factor of 2^3 (the parts' room), and the accumulated outputs are scaled only then: mostly
// in a part's first tile (a room of 2^10 is no faster).  Over 1000 to 32600 positions of
// which the first takes 1/2 to 0.99 of the weight, in one part or many, errors are up to
// 2.1 times those of the same formula in plain fp32, over normal scores 0.2 to 0.9 times
// them, of a few positions up to 1.3 times.
//
// What bounds it.  Two sequences of 64 nodes, 14 / 2 heads of 64, over 32600 rows: 41
// us, 23 GFLOP of matrix products in two parts, 0.56 PFLOP/s.  The matrix cores are
// busy 37% of it, the vector ALUs (16 exponentials, maxima, sums and the weights'
// parts, 120 instructions a tile and wave, and the matrix instructions' issue) 59%; the
// two overlap in part only, and every wave waits for its LDS reads in four places a
// tile.  Half of the products left out (the low parts') saved 8 us, the exponentials 2,
// the loads none.  Slower or no faster: two tiles of rows a wave, a third buffer, the next
// tile's keys read or multiplied ahead, operands of all products read first (registers),
// priorities.  At head size 64 the 128 registers of 4 waves a SIMD spill 4 or 7, in front
// of the loop over the tiles alone.
// One-token sequences are bound by memory: 16 of 12 / 12 heads over 1000 rows, 43
// MB, take 13.5 us, 3.2 TB/s (a plain sum reads 4.0).
constexpr int kTp = 64;          // positions per tile
constexpr float kRoom = 3.0f;    // how far scores may pass the running maximum (powers of two)
constexpr int kLift = 12;        // the weights' parts are those of 2^kLift e^(x - m)
constexpr float kLifted = 1 << kLift;
static_assert(kLift + kRoom < 16.0f, "parts below 65504");

// where part i of a sequence's n parts starts, of its tiles
__device__ __forceinline__ int part_at(int tiles, int i, int n) { return (int)((int64_t)tiles * i / n); }

// which of the positions p0 .. p0 + 63 a row sees: those of the text from lo on,
// and the nodes of `see` behind it
__device__ __forceinline__ uint64_t tile_mask(int p0, int lo, int past, uint64_t see) {
  const int d = past - p0;
  const uint64_t nodes = d >= 64 ? 0 : d >= 0 ? see << d : d > -64 ? see >> -d : 0;
  return (low_bits(d) & ~low_bits(lo - p0)) | nodes;
}

// How the positions are split: `parts` blocks per KV head and row block, of which a
// sequence has as many as its tiles ask for, up to `most`.
constexpr long kGridRow = 1L << 20;
struct TreeGrid {
  int parts, most, rb, shift;  // rb: row blocks per KV head; tiles >> shift add up in 31 bits
};

// a sequence's tiles (one where it takes no part)
__device__ __forceinline__ int tree_tiles(const TreeAttnArgs &a, const EcTreeSeq &s) {
  return ec_tree_seq_ok(&a.t, s) ? (s.past + s.n - window_lo(a.window, s.past, 0) + kTp - 1) / kTp : 1;
}

// A sequence's parts: one, and of those left (parts - B) those between its tiles' share
// of the running sum of all sequences' and the next one's; of these as many as it has
// tiles, up to `most`.  By a wave, a sequence per lane.  Part i of the grid gets its
// sequence, its place j among the sequence's parts and their number n (b is -1 where
// it is none of them).
struct TreePart {
  int b, j, n;
  EcTreeSeq s;
};
__device__ __forceinline__ TreePart tree_part(const TreeAttnArgs &a, const TreeGrid &gr, int i) {
  const int lane = threadIdx.x & 63, B = a.t.B;
  const auto tiles_of = [&](int c, EcTreeSeq &s) {
    s = ec_tree_seq(&a.t, min(c, B - 1));
    return c < B ? tree_tiles(a, s) : 0;
  };
  EcTreeSeq s0, s;
  const int tiles0 = tiles_of(lane, s0);
  uint32_t all = 0;
  for (int c0 = 0; c0 < B; c0 += 64)
    all += readlane(wave_scan((uint32_t)((c0 ? tiles_of(c0 + lane, s) : tiles0) >> gr.shift)), 63);
  // exact: the products stay below 2^53, the quotients' steps above 2^-40
  const double left = (double)(gr.parts - B), per = (double)max(all, 1u);
  uint32_t sum = 0;
  for (int c0 = 0; c0 < B; c0 += 64) {
    s = s0;
    const int c = c0 + lane, tiles = c0 ? tiles_of(c, s) : tiles0;
    const uint32_t w = (uint32_t)(tiles >> gr.shift), upto = sum + wave_scan(w);
    const int first = c + (int)(left * (double)(upto - w) / per), next = c + 1 + (int)(left * (double)upto / per);
    const uint64_t hit = __ballot(c < B && first <= i && i < next);
    if (hit) {
      const int at = __ffsll((unsigned long long)hit) - 1, j = i - readlane(first, at);
      const int n = readlane(min(min(next - first, tiles), gr.most), at);
      return TreePart{j < n ? c0 + at : -1, j, n, EcTreeSeq{readlane(s.slot, at), readlane(s.past, at), readlane(s.n, at)}};
    }
    sum = readlane(upto, 63);
  }
  return TreePart{-1, 0, 0, {0, 0, 0}};
}
// The parts' results: outputs, then maxima and sums, [most][rows of the call], and each
// sequence's number of parts.
struct PartRows {
  float *o;
  float2 *ml;
  int *n;
  size_t all;
};
__device__ __forceinline__ PartRows part_rows(const TreeAttnArgs &a, const TreeGrid &gr, int hd) {
  PartRows p;
  p.all = (size_t)a.t.B * a.t.N * a.H;
  p.o = (float *)a.ws;
  p.ml = (float2 *)(p.o + gr.most * p.all * hd);
  p.n = (int *)(p.ml + gr.most * p.all);
  return p;
}



template <int HD, int NW, int OCC>
__global__ __launch_bounds__(NW * 64, OCC) void attn_tree_kernel(TreeAttnArgs a, TreeGrid gr) {
  constexpr int CPR = HD / 8, KS = HD / 32, DT = HD / 16, NT = NW * 64, LPT = (kTp * CPR + NT - 1) / NT,
                ND = DT % 4 ? 2 : 4;
  typedef __attribute__((address_space(1))) const void gvoid;
  typedef __attribute__((address_space(3))) void lvoid;
  extern __shared__ __attribute__((aligned(16))) _Float16 lds[];  // [2 buffers][K, V][kTp][HD]
  const int t = threadIdx.x, lane = t & 63, lr = lane & 15, lg = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  // blocks go to the 8 XCDs in turn: a part's row blocks, which read the same rows
  // of the cache, follow each other on one XCD
  const int x = blockIdx.y * gridDim.x + blockIdx.x, unit = ((x >> 3) / gr.rb) * 8 + (x & 7), rb = (x >> 3) % gr.rb;
  if (unit >= gr.parts * a.KVH) return;
  const int kvh = unit % a.KVH, part = unit / a.KVH;
  const int G = a.H / a.KVH, r0 = rb * 16 * NW;
  const bool joins = gr.parts > a.t.B;
  TreePart tp{part, 0, 1, {0, 0, 0}};
  if (joins && a.t.B > 1) {
    tp = tree_part(a, gr, part);
  } else if (joins) {
    tp.s = ec_tree_seq(&a.t, 0);
    tp.n = min(gr.most, tree_tiles(a, tp.s));
    tp.b = part < tp.n ? 0 : -1;
    tp.j = part;
  } else {
    tp.s = ec_tree_seq(&a.t, part);
  }
  const int b = tp.b;
  if (b < 0) return;
  const EcTreeSeq s = tp.s;
  const size_t m0 = (size_t)b * a.t.N;
  const int rows = ec_tree_rows(&a.t, s) * G;
  if (r0 >= rows) return;
  if (!ec_tree_seq_ok(&a.t, s)) {  // NaN, here or by the join
    if (!joins)
      for (int e = t; e < min(rows - r0, 16 * NW) * HD; e += NT) {
        const int r = r0 + e / HD;
        a.out[(m0 + r / G) * a.ldo + (size_t)(kvh * G + r % G) * HD + e % HD] = __builtin_nanf("");
      }
    return;
  }
  const int end = s.past + s.n, lo0 = window_lo(a.window, s.past, 0), lo_all = window_lo(a.window, s.past, s.n - 1);
  const int tiles = (end - lo0 + kTp - 1) / kTp;
  const int tile0 = part_at(tiles, tp.j, tp.n), tile1 = part_at(tiles, tp.j + 1, tp.n);

  // the parents and this lane's row of q (of a node that there is), both before the
  // first tile
  const int parent = tree_parent_read(a.t, b);
  const int row = r0 + w * 16 + lr, node = row / G, head = kvh * G + (row - node * G);
  float4 qr[KS][2];
  {
    const float *q = a.q + (m0 + min(node, a.t.N - 1)) * a.ldq + (size_t)head * HD + 8 * lg;
#pragma unroll
    for (int k = 0; k < KS; k++) {
      qr[k][0] = *reinterpret_cast<const float4 *>(q + 32 * k);
      qr[k][1] = *reinterpret_cast<const float4 *>(q + 32 * k + 4);
    }
  }

  // The tiles' way into LDS: a wave's instruction fills 64 chunks, lane l the l-th
  // of them, with the chunk that the swizzle puts there.  In the sequence's last
  // tile the rows behind the nodes are the last node's again (no row sees them).
  const size_t kv = (size_t)a.KVH * HD, base = (size_t)s.slot * a.t.C * kv + (size_t)kvh * HD;
  const int rest = end - lo0 - (tiles - 1) * kTp;  // rows of the last tile
  uint32_t off[LPT], off_last[LPT];
#pragma unroll
  for (int u = 0; u < LPT; u++) {
    const int ch = (w * LPT + u) * 64 + lane, r = ch / CPR, cc = 8 * ((ch - r * CPR) ^ swz<HD>(r));
    off[u] = (uint32_t)r * (uint32_t)kv + cc;
    off_last[u] = (uint32_t)min(r, rest - 1) * (uint32_t)kv + cc;
  }
  constexpr int kBuf = 2 * kTp * HD;  // elements of a buffer: K, then V
  const uint16_t *kn = a.kc + base + (size_t)(lo0 + tile0 * kTp) * kv, *vn = a.vc + base + (size_t)(lo0 + tile0 * kTp) * kv;
  auto load = [&](bool last, int to) {
#pragma unroll
    for (int u = 0; u < LPT; u++) {
      const int first = (w * LPT + u) * 64;
      if (kTp * CPR % NT && first >= kTp * CPR) break;
      const uint32_t o = last ? off_last[u] : off[u];
      __builtin_amdgcn_global_load_lds((gvoid *)(kn + o), (lvoid *)(lds + to + first * 8), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((gvoid *)(vn + o), (lvoid *)(lds + to + kTp * HD + first * 8), 16, 0, 0);
    }
    kn += kTp * kv;
    vn += kTp * kv;
  };
  load(tile0 + 1 == tiles, 0);

  // the nodes' ancestors, where a tile of this block has rows that not all see (from
  // parents that are not valid some mask: the rows are NaN in the end)
  uint64_t anc = 0;
  int depth = 0;
  bool ok = true;
  const bool edges = lo0 + tile1 * kTp > s.past || lo0 + tile0 * kTp < lo_all;
  if (edges) {
    anc = tree_ancestors(tree_parent(parent, s.n, &ok), &depth);
    if (a.window > 0 && a.window < EC_TREE_MAX)
      for (int j = 0; j < s.n; j++)
        if (depth - __shfl(depth, j, 64) >= a.window) anc &= ~(1ull << j);
  }

  const bool work = r0 + w * 16 < rows, live = row < rows;
  const int src = min(node, EC_TREE_MAX - 1);
  const uint64_t see = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(anc >> 32), src, 64) << 32) |
                       (uint32_t)__shfl((int)(uint32_t)anc, src, 64);
  const int lo = window_lo(a.window, s.past, __shfl(depth, src, 64));
  // q in units of log2, so that a product is an exponent.  A row is brought
  // into the parts' range by a power of two where its largest is outside [2^-4,
  // 2^15) (below, the low parts' steps of 2^-24 would count).
  v4u qh[KS], ql[KS];
  float up, down;
  bool plain;  // no row of the wave scaled
  {
    float v[KS][8], big = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; k++) {
      const float4 u0 = qr[k][0], u1 = qr[k][1];
      v[k][0] = u0.x, v[k][1] = u0.y, v[k][2] = u0.z, v[k][3] = u0.w;
      v[k][4] = u1.x, v[k][5] = u1.y, v[k][6] = u1.z, v[k][7] = u1.w;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        v[k][j] *= a.scale * 1.44269504f;
        big = fmaxf(big, fabsf(v[k][j]));
      }
    }
    big = row_max(big);
    int e = 0;
    if (!(big >= 0.0625f && big < 32768.0f) && big > 0.0f)
      e = min(max(14 - ((int)(__float_as_uint(big) >> 23) - 127), -126), 100);
    up = __uint_as_float((uint32_t)(e + 127) << 23);
    down = __uint_as_float((uint32_t)(127 - e) << 23);
    plain = __ballot(e != 0) == 0;
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float x = v[k][2 * j] * up, y = v[k][2 * j + 1] * up;
        const Parts f = split2(x, y);
        qh[k][j] = f.hi;
        // once a block, so the low parts are the nearest here
        ql[k][j] = (uint32_t)f2h(x - h2f((uint16_t)f.hi)) | (uint32_t)f2h(y - h2f((uint16_t)(f.hi >> 16))) << 16;
      }
  }

  // the values' LDS addresses in a buffer's first 32 rows (rows 16 and 32 further
  // on have the same swizzle)
  const uint32_t vbase = (uint32_t)(uintptr_t)(lvoid *)lds + 2 * kTp * HD;
  uint32_t vcol[DT];
#pragma unroll
  for (int d = 0; d < DT; d++) {
    const int r = 4 * lg + (lr >> 2);
    vcol[d] = (uint32_t)(r * HD + ((2 * d + ((lr & 3) >> 1)) ^ swz<HD>(r)) * 8 + 4 * (lr & 1)) * 2;
  }

  v4f o[DT], from = {0.0f, 0.0f, 0.0f, 0.0f};  // from: what the row's products start at
  float mx = -FLT_MAX, lim = -FLT_MAX, sum = 0.0f;
#pragma unroll
  for (int d = 0; d < DT; d++) o[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  int buf = 0;  // of this tile: 0 or kBuf
  // One tile.  EDGE: one that some rows see in part: what they do not see has weight
  // 0, and its values must be finite for that to be nothing.
  auto step = [&](auto edge, int tile) {
    constexpr bool EDGE = decltype(edge)::value;
    const int p0 = lo0 + tile * kTp;
    // this tile has landed, and every wave is done with the one before it
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("s_barrier" ::: "memory");
    if (tile + 1 < tile1) load(tile + 2 == tiles, kBuf - buf);
    _Float16 *K = lds + buf, *V = K + kTp * HD;
    const uint32_t vat = vbase + 2 * (uint32_t)buf;
    buf = kBuf - buf;
    bool inf = false;
    if constexpr (EDGE) {
      for (int ch = t; ch < kTp * CPR; ch += NT) {
        v4u *at = reinterpret_cast<v4u *>(V) + ch, v = *at;
        uint32_t hit = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          // an exponent of all ones carries out of its field
          const uint32_t e = v[j] & 0x7C007C00u;
          const uint32_t bad = ((e & 0x7C00u) + 0x0400u) & 0x8000u, bad2 = ((e >> 16) + 0x0400u) & 0x8000u;
          v[j] &= ~((bad ? 0xFFFFu : 0u) | (bad2 ? 0xFFFF0000u : 0u));
          hit |= bad | bad2;
        }
        if (hit) {
          *at = v;
          inf = true;
        }
      }
      inf = __syncthreads_or(inf);
    }
    if (!work) return;

    // ---- scores: sc[pt][r] of position 16 pt + 4 lg + r ----
    v4f sc[4];
#pragma unroll
    for (int pt = 0; pt < 4; pt++) {
      sc[pt] = from;
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const int r = 16 * pt + lr;
        const v4u kf = *reinterpret_cast<const v4u *>(K + r * HD + ((4 * k + lg) ^ swz<HD>(r)) * 8);
        sc[pt] = mma(kf, qh[k], sc[pt]);
        sc[pt] = mma(kf, ql[k], sc[pt]);
      }
    }

    // ---- weights ----
    if constexpr (EDGE) {
      const uint64_t on = tile_mask(p0, lo, s.past, see) >> (4 * lg);
#pragma unroll
      for (int pt = 0; pt < 4; pt++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (!((on >> (16 * pt + r)) & 1)) sc[pt][r] = -__builtin_inff();
    }
    if (__builtin_expect(!plain, 0)) {
#pragma unroll
      for (int pt = 0; pt < 4; pt++)
#pragma unroll
        for (int r = 0; r < 4; r++) sc[pt][r] *= down;
    }
    // exponents of the weights already (the sums began at -mx): above kRoom the maximum
    // moves
    float top = -FLT_MAX;
#pragma unroll
    for (int pt = 0; pt < 4; pt++)
#pragma unroll
      for (int r = 0; r < 4; r++) top = fmaxf(top, sc[pt][r]);
    if (__builtin_expect(__ballot(top > lim) != 0, 0)) {
      const float big = row_max(top);
      const bool first = mx == -FLT_MAX, move = big > (first ? -FLT_MAX : 0.0f);
      const float by = move ? big : 0.0f, back = first ? 0.0f : __builtin_amdgcn_exp2f(-by);
      if (move) {
        mx = first ? big : mx + by;
        lim = kRoom;
      }
      const float f = move || !first ? -mx * up : 0.0f;
      from = v4f{f, f, f, f};
      sum *= back;
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int r = 0; r < 4; r++) o[d][r] *= back;
#pragma unroll
      for (int pt = 0; pt < 4; pt++)
#pragma unroll
        for (int r = 0; r < 4; r++) sc[pt][r] -= by;
    }
    // the tile's weights are added up before they meet the sum so far: one by one, those
    // below half a step of it would be lost
    v4u ph[2], pl[2];
    float here = 0.0f;
#pragma unroll
    for (int pt = 0; pt < 4; pt++) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        p[r] = __builtin_amdgcn_exp2f(sc[pt][r]);
        here += p[r];
      }
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const Parts f = split2<kLift>(p[2 * r], p[2 * r + 1]);
        ph[pt >> 1][2 * (pt & 1) + r] = f.hi;
        pl[pt >> 1][2 * (pt & 1) + r] = f.lo;
      }
    }
    sum += here;

    // ---- outputs: o[d][r] of element 16 d + 4 lg + r ----
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int d = 0; d < DT; d += ND) {
        v4u vf[ND];
        read_v<HD, ND>(vcol + d, vat, u, vf);
#pragma unroll
        for (int e = 0; e < ND; e++) {
          o[d + e] = mma(vf[e], ph[u], o[d + e]);
          o[d + e] = mma(vf[e], pl[u], o[d + e]);
        }
      }

    // values that are not finite, for the rows that see them, one by one
    if (EDGE && __builtin_expect(inf, 0)) {
      const uint64_t on = tile_mask(p0, lo, s.past, see);
      for (int pp = 0; pp < kTp && p0 + pp < end; pp++) {
        float wgt = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (32 * u + 16 * (e >> 2) + (e & 3) == (pp & ~12)) wgt = half_of(ph[u], e) + half_of(pl[u], e);
        wgt = __shfl(wgt, (((pp & 15) >> 2) << 4) | lr, 64);  // from the lane that has this row's weight of it
        if ((on >> pp) & 1) {
#pragma unroll
          for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              const uint16_t v = a.vc[base + (size_t)(p0 + pp) * kv + 16 * d + 4 * lg + r];
              if ((v & 0x7C00u) == 0x7C00u) o[d][r] += wgt * h2f(v);
            }
        }
      }
    }
  };
  // the tiles that every row sees whole, and those in front of and behind them
  const int whole0 = min(max(lo_all - lo0 + kTp - 1, 0) / kTp, tile1), whole1 = max(s.past - lo0, 0) / kTp;
  int tile = tile0;
  for (; tile < whole0; tile++) step(std::true_type{}, tile);
  for (; tile < min(whole1, tile1); tile++) step(std::false_type{}, tile);
  for (; tile < tile1; tile++) step(std::true_type{}, tile);

  if (!edges) tree_parent(parent, s.n, &ok);
  const float l = ok ? row_sum(sum) * kLifted : __builtin_nanf("");  // as the outputs
  if (!live) return;
  if (!joins) {
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    float *out = a.out + (m0 + node) * a.ldo + (size_t)head * HD + 4 * lg;
#pragma unroll
    for (int d = 0; d < DT; d++)
      *reinterpret_cast<float4 *>(out + 16 * d) =
          make_float4(o[d][0] * inv, o[d][1] * inv, o[d][2] * inv, o[d][3] * inv);
  } else {
    const PartRows pr = part_rows(a, gr, HD);
    const size_t at = tp.j * pr.all + (m0 + node) * a.H + head;
    float *po = pr.o + at * HD + 4 * lg;
#pragma unroll
    for (int d = 0; d < DT; d++) *reinterpret_cast<float4 *>(po + 16 * d) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
    if (lg == 0) pr.ml[at] = make_float2(mx, l);
    if (tp.j == 0 && kvh == 0 && rb == 0 && t == 0) pr.n[b] = tp.n;
  }
}

// Joins the parts' outputs: per row the largest of their maxima, the sums and outputs
// brought to it.  HD / 4 lanes a row (a power of two of them: 24 of 32 at 96).  Latency
// is all of it: the reads do not wait for the sequence's numbers, and those of the next
// parts do not for these (3.6 us for 8 nodes, 6.4 for the 30 to 34 parts of 2 x 64
// nodes; one set of 16 parts 7.9).  The last block of a row's parts could join them,
// without this launch; but what it counts arrivals with lives from call to call, and a
// run that ends half way would leave it wrong for good.
template <int HD>
__global__ __launch_bounds__(256) void attn_tree_join_kernel(TreeAttnArgs a, TreeGrid gr) {
  constexpr int LPR = HD == 96 ? 32 : HD / 4, RPB = 256 / LPR;
  constexpr int kRead = 12;  // parts read at a time, in two sets by turns
  const int t = threadIdx.x, b = blockIdx.y, li = t % LPR;
  const int r = blockIdx.x * RPB + t / LPR;
  const PartRows pr = part_rows(a, gr, HD);
  const size_t row = (size_t)b * a.t.N * a.H + min(r, a.t.N * a.H - 1);
  struct Read {
    float2 u[kRead];
    float4 v[kRead];
  } x[2];
  const auto read = [&](Read &x, int j0, int n) {
#pragma unroll
    for (int i = 0; i < kRead; i++) {
      const size_t at = (size_t)min(j0 + i, n - 1) * pr.all + row;
      x.u[i] = pr.ml[at];
      x.v[i] = *reinterpret_cast<const float4 *>(pr.o + at * HD + 4 * min(li, HD / 4 - 1));
    }
  };
  read(x[0], 0, gr.most);  // before it is known how many there are
  const EcTreeSeq s = ec_tree_seq(&a.t, b);
  const bool ok = ec_tree_seq_ok(&a.t, s);  // (bad parents: the parts' sums are NaN)
  const int rows = ec_tree_rows(&a.t, s) * a.H, n = pr.n[b];
  if (blockIdx.x * RPB >= rows) return;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (ok) {
    float m = -FLT_MAX, l = 0.0f;
    const auto use = [&](const Read &x, int i0) {
      float big = m;
#pragma unroll
      for (int i = 0; i < kRead; i++)
        if (i0 + i < n) big = fmaxf(big, x.u[i].x);
      const float back = __builtin_amdgcn_exp2f(m - big);
      m = big;
      l *= back;
      o = make_float4(o.x * back, o.y * back, o.z * back, o.w * back);
#pragma unroll
      for (int i = 0; i < kRead; i++)
        if (i0 + i < n) {
          const float f = __builtin_amdgcn_exp2f(x.u[i].x - m);
          l = __builtin_fmaf(x.u[i].y, f, l);
          o.x = __builtin_fmaf(x.v[i].x, f, o.x);
          o.y = __builtin_fmaf(x.v[i].y, f, o.y);
          o.z = __builtin_fmaf(x.v[i].z, f, o.z);
          o.w = __builtin_fmaf(x.v[i].w, f, o.w);
        }
    };
    for (int i0 = 0; i0 < n; i0 += 2 * kRead) {
      if (i0 + kRead < n) read(x[1], i0 + kRead, n);
      use(x[0], i0);
      if (i0 + kRead >= n) break;
      if (i0 + 2 * kRead < n) read(x[0], i0 + 2 * kRead, n);
      use(x[1], i0 + kRead);
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  } else {
    o.x = o.y = o.z = o.w = __builtin_nanf("");
  }
  const int node = r / a.H;
  if (r < rows && li < HD / 4)
    *reinterpret_cast<float4 *>(a.out + ((size_t)b * a.t.N + node) * a.ldo + (size_t)(r - node * a.H) * HD + 4 * li) = o;
}

// heads and rows that the matrix-core form's tiles and 16-byte accesses can take, and
// whose blocks (no more than query heads in all) count in an int (both sides' times stand
// at the form for any size)
bool tiles_ok(const TreeAttnArgs &a) {
  if ((long)a.t.B * a.t.N * a.H > 1L << 30) return false;
  const uintptr_t p = (uintptr_t)a.q | (uintptr_t)a.kc | (uintptr_t)a.vc | (uintptr_t)a.out;
  return (a.hd == 32 || a.hd == 64 || a.hd == 96 || a.hd == 128) && !(p & 15) && a.ldq % 4 == 0 && a.ldo % 4 == 0;
}

// Waves per block: 4 (64 rows) or 8 (128), by the rows that share a KV head.  Up to 64
// rows, 8 waves would load faster but for more blocks' places: 15.7 instead of 13.5 us
// for the one-token sequences above.  Over 64, 4 waves read the cache twice as often:
// 45 instead of 41 us for the two long contexts, 20.0 instead of 18.2 for 8 trees of
// 16 nodes, 12 / 2 heads of 128, over 4000 rows.
int tree_waves(const TreeAttnArgs &a) { return (long)a.t.N * (a.H / a.KVH) <= 64 ? 4 : 8; }

// Row blocks and parts: blocks for the CUs' places, of at least a tile each.  Two a CU, at
// head sizes above 64 with 8 waves one (180 registers leave room for no second: two a
// CU, one after the other, take 24 + 7.0 us (the join's) instead of 18.2 + 5.6 for the
// trees over 4000 rows), at those up to 64 with 4 waves three: 16 one-token sequences of
// 12 / 12 heads over 1000 rows take 15.1 + 4.0 us with two, 13.5 + 4.2 with three, 13.7 +
// 4.1 with four, 32 of 14 / 2 heads over 2000 rows took 13.1, 13.0 and 14.3 in all.  Three
// and four a CU for 8 waves take 45 + 8.1 and 46 + 9.5 us instead of 41 + 6.4 for the long
// contexts.  With no parts at all these take 520 us, the trees 106, 8 nodes over 700 rows
// 16 instead of 7.4 + 3.6.  Where the sequences alone fill the places there are no parts,
// whatever their lengths: 64 one-token sequences of 12 / 12 heads, one over 30000 rows
// and 63 over 300, take 380 us, 16 of them (split) 32.
TreeGrid tree_grid(const TreeAttnArgs &a) {
  TreeGrid g;
  const int waves = tree_waves(a), per = 16 * waves;
  g.rb = (int)(((long)a.t.N * (a.H / a.KVH) + per - 1) / per);
  long span = (long)a.t.max_past + a.t.N;
  if (a.window > 0 && (long)a.window + a.t.N < span) span = (long)a.window + a.t.N;
  const long tiles = (span + kTp - 1) / kTp, full = a.hd <= 64 ? (waves == 4 ? 768 : 512) : waves == 4 ? 512 : 256;
  const long want = full / ((long)a.KVH * g.rb), most = tiles * a.t.B;
  g.parts = (int)(want < a.t.B ? a.t.B : want < most ? want : most);
  // of a sequence, four times its even share at most: the join's rows have room for that
  const long share = 4 * ((g.parts + a.t.B - 1) / a.t.B);
  g.most = (int)(share < g.parts - a.t.B + 1 ? share : g.parts - a.t.B + 1);
  g.shift = 0;
  while ((tiles >> g.shift) * a.t.B >= 1L << 31) g.shift++;
  return g;
}

template <int HD>
hipError_t launch_tree(const TreeAttnArgs &a, hipStream_t st) {
  const TreeGrid g = tree_grid(a);
  // a multiple of 8 blocks in x (the XCDs' turns), as many as a dimension's 2^32 threads
  // have room for
  const long blocks = ((long)g.parts * a.KVH + 7) / 8 * 8 * g.rb, row = blocks < kGridRow ? blocks : kGridRow;
  const dim3 grid((unsigned)row, (unsigned)((blocks + row - 1) / row));
  const uint32_t lds = 2 * 4 * kTp * HD;
  if (tree_waves(a) == 4) klaunch((attn_tree_kernel<HD, 4, HD <= 64 ? 4 : 2>), grid, dim3(256), lds, st, a, g);
  else klaunch((attn_tree_kernel<HD, 8, HD <= 64 ? 4 : 2>), grid, dim3(512), lds, st, a, g);
  return hipGetLastError();
}

template <int HD>
hipError_t launch_join(const TreeAttnArgs &a, hipStream_t st) {
  constexpr int rpb = 256 / (HD == 96 ? 32 : HD / 4);
  klaunch((attn_tree_join_kernel<HD>), dim3((a.t.N * a.H + rpb - 1) / rpb, a.t.B), dim3(256), 0, st, a, tree_grid(a));
  return hipGetLastError();
}

}  // namespace

int attention_tree_max_hd() { return kTreeMaxHd; }

size_t attention_tree_workspace(const TreeAttnArgs &a) {
  if (!attention_tree_joins(a)) return 0;
  return (size_t)a.t.B * ((size_t)tree_grid(a).most * a.t.N * a.H * (a.hd + 2) * sizeof(float) + sizeof(int));
}

hipError_t attention_tree(const TreeAttnArgs &a, hipStream_t st) {
  if (tiles_ok(a)) {
    if (a.hd == 64) return launch_tree<64>(a, st);
    if (a.hd == 128) return launch_tree<128>(a, st);
    if (a.hd == 96) return launch_tree<96>(a, st);
    return launch_tree<32>(a, st);
  }
  klaunch(attn_tree_any_kernel, dim3(a.t.B * a.t.N, a.H), dim3(256), 0, st, a);
  return hipGetLastError();
}

bool attention_tree_joins(const TreeAttnArgs &a) { return tiles_ok(a) && tree_grid(a).parts > a.t.B; }

hipError_t attention_tree_join(const TreeAttnArgs &a, hipStream_t st) {
  if (a.hd == 64) return launch_join<64>(a, st);
  if (a.hd == 128) return launch_join<128>(a, st);
  if (a.hd == 96) return launch_join<96>(a, st);
  return launch_join<32>(a, st);
}

}  // namespace ec
