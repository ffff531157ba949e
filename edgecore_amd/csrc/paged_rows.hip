// Rows in and out of a paged cache (ec_pages.h) whose elements are 16 or 8 bits
// wide, 8-bit ones with a scale per row and KV head:
//
//   paged_append: one token's q|k|v row, per head of q and k
//       y = x / sqrt(mean x^2 + eps) * gamma           (gamma null: y = x)
//       a_i = (past + i) f_i, in 64 bits
//       (y_i, y_j) -> factor (y_i cos a_i - y_j sin a_i, y_i sin a_i + y_j cos a_i)
//     over the pairs (i, i + rot / 2) or (2 i, 2 i + 1) of the first rot
//     elements; q goes to its own rows in fp32, k and v to the pages: in fp16, or
//       s = max |y| / Q, the next fp16 from there up,  c = y / s to the nearest
//     with Q = 127 (int8) or 448 (e4m3).  A row stands for the fp16 values c s.
//   paged_read: the values that rows of the pages stand for, into the fp16 slot cache.
//
// k is computed in 64 bits: a code is a step of 1/127 of a row's largest, so that a
// key near the border of two would show 32-bit roundings in all that is read.
#include <algorithm>
#include <type_traits>

#include "ec_device.h"
#include "ec_kernels.h"
#include "paged_cache.h"

namespace ec {

namespace {

// What a row's threads know of it: its sequence, its position, its place in the pages.
struct PagedRow {
  bool mine, ok;  // a sequence's row; of one that takes part, with a page
  int pos;
  uint32_t row;  // of KV head 0; KV head h's is page * h further on
};
__device__ __forceinline__ PagedRow paged_row(const EcPageBatch &t, int m) {
  PagedRow r{false, false, 0, 0};
  const int b = page_seq_of(t, m);
  if (b < 0) return r;
  const EcPageSeq s = ec_page_seq(&t, b);
  r.mine = ec_page_seq_mine(&t, s) && m >= s.start && m - s.start < s.n;
  if (!r.mine || !ec_page_seq_ok(&t, s, EC_PAGES_ROWS)) return r;
  r.pos = s.past + (m - s.start);
  bool bad = false;
  r.row = page_row(t, page_id(t, b, r.pos), r.pos, 0, &bad);
  r.ok = !bad;
  return r;
}

// cos and sin of a = pos * f, times factor, in 64 bits
__device__ __forceinline__ double2 rope_cs64(int pos, double f, double factor) {
  const double turns = (double)pos * f * 0.15915494309189533577;
  double s, c;
  sincospi(2.0 * (turns - rint(turns)), &s, &c);
  return make_double2(c * factor, s * factor);
}

// The form for any head size and alignment: one block per token, a wave a head at
// a time, its elements through the wave's row in LDS.
constexpr int kAppendMaxHd = 512;
constexpr long kGridRow = 1L << 20;
constexpr double kL2 = 32 << 20;  // bytes of the 8 L2s together
__global__ __launch_bounds__(256) void paged_append_any_kernel(PagedAppendArgs a) {
  __shared__ double row[4][kAppendMaxHd];
  __shared__ double2 cs[kAppendMaxHd / 2];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, hd = a.c.hd, KVH = a.c.t.KVH;
  const PagedRow rr = paged_row(a.c.t, blockIdx.x);
  if (!rr.mine) return;
  const size_t m = blockIdx.x;
  float *q = a.q + m * a.ldq;
  if (!rr.ok) {
    for (int e = t; e < a.H * hd; e += 256) q[e] = __builtin_nanf("");
    return;
  }
  const int half = a.rot >> 1;
  for (int e = t; e < half; e += 256) cs[e] = rope_cs64(rr.pos, a.inv_freq[e], a.factor);
  __syncthreads();
  const float *x = a.x + m * a.ldx;
  // a uniform count of rounds: the waves meet at barriers in each
  for (int h0 = 0; h0 < a.H + 2 * KVH; h0 += 4) {
    const int h = h0 + w;
    const bool on = h < a.H + 2 * KVH, isv = h >= a.H + KVH, isq = h < a.H;
    const float *gamma = isq ? a.q_gamma : isv ? nullptr : a.k_gamma;
    double r = 1.0;
    if (on) {
      double sum = 0.0;
      for (int e = lane; e < hd; e += 64) {
        const double v = x[(size_t)h * hd + e];
        row[w][e] = v;
        sum = __builtin_fma(v, v, sum);
      }
      if (gamma) r = 1.0 / sqrt(wave_sum(sum) / hd + a.eps);
    }
    __syncthreads();
    if (on) {
      double y[kAppendMaxHd / 64], top = 0.0;
      bool nan = false;
#pragma unroll
      for (int i = 0; i < kAppendMaxHd / 64; i++) {
        const int e = lane + 64 * i;
        if (e >= hd) break;
        auto at = [&](int j) {
          const double v = row[w][j];
          return gamma ? v * r * gamma[j] : v;
        };
        y[i] = at(e);
        if (!isv && e < a.rot) {
          const bool second = a.layout ? e & 1 : e >= half;
          const int f = a.layout ? e >> 1 : second ? e - half : e;
          const double o = at(a.layout ? e ^ 1 : second ? e - half : e + half);
          y[i] = second ? o * cs[f].y + y[i] * cs[f].x : y[i] * cs[f].x - o * cs[f].y;
        }
        top = fmax(top, fabs(y[i]));
        nan |= y[i] != y[i];
      }
      const int kvh = isv ? h - a.H - KVH : h - a.H;
      const size_t at = rr.row + (size_t)kvh * a.c.t.page;
      uint16_t sc = 0;
      if (!isq && a.c.type != CACHE_F16) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmax(top, __shfl_xor(top, o, 64));
        sc = __ballot(nan) ? 0x7E00 : cache_scale(top, a.c.type);
        if (lane == 0) (isv ? a.c.vs : a.c.ks)[at] = sc;
      }
#pragma unroll
      for (int i = 0; i < kAppendMaxHd / 64; i++) {
        const int e = lane + 64 * i;
        if (e >= hd) break;
        if (isq) q[(size_t)h * hd + e] = (float)y[i];
        else cache_store(isv ? a.c.v : a.c.k, a.c.type, at * hd + e, y[i], sc);
      }
    }
    __syncthreads();
  }
}

// The form for head sizes that are multiples of 4 up to 256 and rows of whole
// 16-byte chunks: a block per row, LPH lanes a head, four elements a lane.  A wave takes 64
// / LPH heads at a time, of q (in 32 bits) or of k and v (in 64), those of k and v first:
// they take longest.  Bound by the chain of start, length and page in front of the stores and
// by the 64-bit roundings: 2 x 1500 rows of 14 + 2 2 heads of 64 in 12.9 us (fp16 10.9), 12 + 2 2
// of 128 in 15.4; the form for any size takes 30 at heads of 62 and 37 at 126.  64 rows take 5, as
// the shortest kernels do.  A pair's other element is in the same lane (layout 1) or in lane +-
// rot / 8, which holds its four (layout 0, rot a multiple of 8).
template <int LPH, int TYPE>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
  constexpr int GPW = 64 / LPH;  // heads of a wave
  __shared__ double cosines[128], sines[128];
  const int t = threadIdx.x, lane = t & 63, li = lane % LPH, e = 4 * li, hd = a.c.hd, KVH = a.c.t.KVH, H = a.H;
  const int kvw = (2 * KVH + GPW - 1) / GPW, all = kvw + (H + GPW - 1) / GPW, waves = blockDim.x >> 6;
  const size_t m = blockIdx.x;
  const int half = a.rot >> 1;
  const bool in = e < hd;
  const float *x = a.x + m * a.ldx + e;
  // the head of slot i's lanes: k and v, then q
  const auto head_of = [&](int i) {
    const int g = lane / LPH, h = i < kvw ? H + i * GPW + g : (i - kvw) * GPW + g;
    return i < kvw ? (h < H + 2 * KVH ? h : -1) : h < H && i < all ? h : -1;
  };
  const auto read = [&](int h) {
    float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (in && h >= 0) v = *reinterpret_cast<const float4 *>(x + (size_t)h * hd);
    return v;
  };
  int i = t >> 6, h = head_of(i);
  float4 next = read(h);
  double f = 0.0;
  if (t < half) f = a.inv_freq[t];
  const PagedRow rr = paged_row(a.c.t, blockIdx.x);
  if (!rr.mine) return;
  for (int j = t; j < half; j += blockDim.x) {
    const double2 c = rope_cs64(rr.pos, j == t ? f : a.inv_freq[j], a.factor);
    cosines[j] = c.x;
    sines[j] = c.y;
  }
  __syncthreads();
  const int far = half >> 2;  // lanes from an element to its pair's other one (layout 0)
  const bool first = li < far;
  const int src = (lane + (first ? far : -far)) & 63;
  // four elements turned; in q's width or in 64 bits
  const auto turn = [&](auto *v) {
    using T = std::remove_pointer_t<decltype(v)>;
    if (a.layout) {
      if (e < a.rot)
#pragma unroll
        for (int k = 0; k < 4; k += 2)
          if (e + k < a.rot) {
            const T c = (T)cosines[2 * li + k / 2], s = (T)sines[2 * li + k / 2], p = v[k], q = v[k + 1];
            v[k] = p * c - q * s;
            v[k + 1] = p * s + q * c;
          }
    } else if (a.rot) {
      T o[4];
#pragma unroll
      for (int k = 0; k < 4; k++) o[k] = __shfl(v[k], src, 64);
      if (e < a.rot)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int j = 4 * (first ? li : li - far) + k;
          const T c = (T)cosines[j], s = (T)sines[j];
          v[k] = first ? v[k] * c - o[k] * s : v[k] * c + o[k] * s;
        }
    }
  };
  for (; i < all; i += waves) {
    const float4 xv = next;
    const int mine = h;
    h = head_of(i + waves);
    next = read(h);
    if (i < kvw) {
      const bool isv = mine >= H + KVH;
      double y[4] = {xv.x, xv.y, xv.z, xv.w};
      if (a.k_gamma) {
        double sum = y[0] * y[0] + y[1] * y[1] + y[2] * y[2] + y[3] * y[3];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (in && !isv) {
          const double s = 1.0 / sqrt(sum / hd + a.eps);
          const float4 g = *reinterpret_cast<const float4 *>(a.k_gamma + e);
          y[0] = y[0] * s * g.x;
          y[1] = y[1] * s * g.y;
          y[2] = y[2] * s * g.z;
          y[3] = y[3] * s * g.w;
        }
      }
      double z[4] = {y[0], y[1], y[2], y[3]};
      turn(z);
      if (!isv)
#pragma unroll
        for (int k = 0; k < 4; k++) y[k] = z[k];
      const int kvh = isv ? mine - H - KVH : mine - H;
      const size_t at = rr.row + (size_t)kvh * a.c.t.page;
      void *to = isv ? a.c.v : a.c.k;
      if constexpr (TYPE == CACHE_F16) {
        if (in && mine >= 0 && rr.ok)
          *reinterpret_cast<uint2 *>((uint16_t *)to + at * hd + e) =
              make_uint2((uint32_t)cache_f16(y[0]) | (uint32_t)cache_f16(y[1]) << 16, (uint32_t)cache_f16(y[2]) | (uint32_t)cache_f16(y[3]) << 16);
      } else {
        // the row's largest by its bits: a NaN's are above every number's
        uint64_t top = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) top = max(top, __builtin_bit_cast(uint64_t, y[k]) & ~(1ull << 63));
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) top = max(top, (uint64_t)__shfl_xor((unsigned long long)top, o, 64));
        const double largest = __builtin_bit_cast(double, top);
        const uint16_t sc = largest != largest ? 0x7E00 : cache_scale(largest, TYPE);
        const double s = h2f(sc);
        uint32_t w = 0;
        if constexpr (TYPE == CACHE_I8) {
#pragma unroll
          for (int k = 0; k < 4; k++) w |= (uint32_t)(cache_code_i8(y[k], s) & 255) << (8 * k);
        } else {
          w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cache_code_e4m3(y[0], s), cache_code_e4m3(y[1], s), 0, false);
          w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cache_code_e4m3(y[2], s), cache_code_e4m3(y[3], s), (int)w, true);
        }
        if (in && mine >= 0 && rr.ok) {
          *reinterpret_cast<uint32_t *>((uint8_t *)to + at * hd + e) = w;
          if (li == 0) (isv ? a.c.vs : a.c.ks)[at] = sc;
        }
      }
    } else {
      float y[4] = {xv.x, xv.y, xv.z, xv.w};
      if (a.q_gamma) {
        float sum = y[0] * y[0] + y[1] * y[1] + y[2] * y[2] + y[3] * y[3];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (in) {
          const float s = 1.0f / sqrtf(sum / (float)hd + (float)a.eps);
          const float4 g = *reinterpret_cast<const float4 *>(a.q_gamma + e);
          y[0] = y[0] * s * g.x;
          y[1] = y[1] * s * g.y;
          y[2] = y[2] * s * g.z;
          y[3] = y[3] * s * g.w;
        }
      }
      turn(y);
      if (in && mine >= 0) {
        const float nan = __builtin_nanf("");
        *reinterpret_cast<float4 *>(a.q + m * a.ldq + (size_t)mine * hd + e) =
            rr.ok ? make_float4(y[0], y[1], y[2], y[3]) : make_float4(nan, nan, nan, nan);
      }
    }
  }
}

// whether sequence b's rows of its slot share one with those of an earlier sequence
__device__ __forceinline__ bool read_clashes(const PagedReadArgs &a, int b, EcTreeSeq s) {
  if (!a.slot) return false;
  bool hit = false;
  for (int c = threadIdx.x & 63; c < b; c += 64) {
    const EcTreeSeq o{a.slot[c], a.to ? a.to[c] : 0, a.count[c]};
    hit |= ec_tree_seq_ok(&a.t, o) && ec_tree_clash(s, o);
  }
  return __ballot(hit) != 0;
}

// The form for any head size and alignment: one block per `per` rows of a sequence, an
// element a thread.
__global__ __launch_bounds__(256) void paged_read_any_kernel(PagedReadArgs a, int per) {
  const int b = blockIdx.y, t = threadIdx.x, hd = a.c.hd, KVH = a.c.t.KVH;
  const EcTreeSeq s{a.slot ? a.slot[b] : b, a.to ? a.to[b] : 0, a.count[b]};
  const int first = a.first[b];
  if (!ec_tree_seq_ok(&a.t, s) || first < 0 || s.n > a.c.t.rows || first > a.c.t.rows - s.n || read_clashes(a, b, s)) return;
  const int i0 = blockIdx.x * per;
  for (int i = i0; i < min(s.n, i0 + per); i++) {
    const int p = first + i;
    bool bad = false;
    const size_t row = page_row(a.c.t, page_id(a.c.t, b, p), p, 0, &bad);
    const size_t to = ((size_t)s.slot * a.t.C + (s.past + i)) * ((size_t)KVH * hd);
    for (int e = t; e < KVH * hd; e += 256) {
      const int h = e / hd;
      const size_t at = row + (size_t)h * a.c.t.page;
      a.kc[to + e] = bad ? 0x7E00 : cache_value(a.c.k, a.c.ks, a.c.type, at, hd, e - h * hd);
      a.vc[to + e] = bad ? 0x7E00 : cache_value(a.c.v, a.c.vs, a.c.type, at, hd, e - h * hd);
    }
  }
}

// The form for head sizes that are multiples of 8: eight elements a thread at a time,
// those of a KV head's rows one behind the other, as they stand in a page.  STREAM: rows that
// are more than the L2s hold go past them.  Bound by memory: 112000 rows of 2 heads of 128
// from e4m3, 173 MB, take 27 us where three caches take turns, 6.3 TB/s with what the last-level
// cache holds of them (a copy of 172 MiB over and over 5.3), and 35 where eight do; through the L2s
// 37 and 38.
template <int TYPE, bool STREAM>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedReadArgs a, int per) {
  const int b = blockIdx.y, t = threadIdx.x, hd = a.c.hd, KVH = a.c.t.KVH;
  const EcTreeSeq s{a.slot ? a.slot[b] : b, a.to ? a.to[b] : 0, a.count[b]};
  const int first = a.first[b], i0 = blockIdx.x * per;
  if (!ec_tree_seq_ok(&a.t, s) || i0 >= s.n || first < 0 || s.n > a.c.t.rows || first > a.c.t.rows - s.n || read_clashes(a, b, s)) return;
  const int n = min(per, s.n - i0), cpr = hd / 8, items = KVH * n * cpr;
  const size_t base = ((size_t)s.slot * a.t.C + (s.past + i0)) * ((size_t)KVH * hd);
  constexpr int UN = 2;
  for (int j0 = t; j0 < items; j0 += 256 * UN) {
    Raw8<TYPE> k[UN], v[UN];
    uint16_t ks[UN], vs[UN];
    size_t to[UN];
    bool bad[UN];
#pragma unroll
    for (int u = 0; u < UN; u++) {
      const int j = min(j0 + 256 * u, items - 1), r = j / cpr, cc = j - r * cpr, h = r / n, p = first + i0 + (r - h * n);
      bad[u] = false;
      const size_t row = page_row(a.c.t, page_id(a.c.t, b, p), p, h, &bad[u]);
      constexpr int B = TYPE == CACHE_F16 ? 2 : 1;
      k[u] = *(const Raw8<TYPE> *)((const char *)a.c.k + (row * hd + 8 * cc) * B);
      v[u] = *(const Raw8<TYPE> *)((const char *)a.c.v + (row * hd + 8 * cc) * B);
      if constexpr (TYPE != CACHE_F16) {
        ks[u] = a.c.ks[row];
        vs[u] = a.c.vs[row];
      }
      to[u] = base + (size_t)(r - h * n) * (KVH * hd) + h * hd + 8 * cc;
    }
#pragma unroll
    for (int u = 0; u < UN; u++) {
      if (j0 + 256 * u >= items) break;
      const v4u none = {0x7E007E00u, 0x7E007E00u, 0x7E007E00u, 0x7E007E00u};
      const v4u ko = bad[u] ? none : to_f16<TYPE>(k[u], ks[u]), vo = bad[u] ? none : to_f16<TYPE>(v[u], vs[u]);
      v4u *kt = reinterpret_cast<v4u *>(a.kc + to[u]), *vt = reinterpret_cast<v4u *>(a.vc + to[u]);
      if constexpr (STREAM) {
        __builtin_nontemporal_store(ko, kt);
        __builtin_nontemporal_store(vo, vt);
      } else {
        *kt = ko;
        *vt = vo;
      }
    }
  }
}

}  // namespace

int paged_append_max_hd() { return kAppendMaxHd; }

// rows that the vector form's 16-byte (caches: of four elements) accesses can take
static bool append_vector_ok(const PagedAppendArgs &a) {
  const uintptr_t p = (uintptr_t)a.x | (uintptr_t)a.q | (uintptr_t)a.q_gamma | (uintptr_t)a.k_gamma;
  return a.c.hd % 4 == 0 && a.c.hd <= 256 && a.ldx % 4 == 0 && a.ldq % 4 == 0 && !(p & 15) &&
         !(((uintptr_t)a.c.k | (uintptr_t)a.c.v) & (a.c.type == CACHE_F16 ? 7 : 3)) && (a.layout || a.rot % 8 == 0);
}

template <int LPH>
static void launch_append(const PagedAppendArgs &a, hipStream_t st) {
  constexpr int gpw = 64 / LPH;
  const int slots = (a.H + gpw - 1) / gpw + (2 * a.c.t.KVH + gpw - 1) / gpw;
  const dim3 grid(a.c.t.M), block(slots < 4 ? 64 * slots : 256);
  if (a.c.type == CACHE_F16) klaunch((paged_append_kernel<LPH, CACHE_F16>), grid, block, 0, st, a);
  else if (a.c.type == CACHE_I8) klaunch((paged_append_kernel<LPH, CACHE_I8>), grid, block, 0, st, a);
  else klaunch((paged_append_kernel<LPH, CACHE_E4M3>), grid, block, 0, st, a);
}

hipError_t paged_append(const PagedAppendArgs &a, hipStream_t st) {
  if (!append_vector_ok(a)) klaunch(paged_append_any_kernel, dim3(a.c.t.M), dim3(256), 0, st, a);
  else if (a.c.hd <= 32) launch_append<8>(a, st);
  else if (a.c.hd <= 64) launch_append<16>(a, st);
  else if (a.c.hd <= 128) launch_append<32>(a, st);
  else launch_append<64>(a, st);
  return hipGetLastError();
}

template <int TYPE>
static void launch_read(const PagedReadArgs &a, dim3 grid, int per, bool stream, hipStream_t st) {
  if (stream) klaunch((paged_read_kernel<TYPE, true>), grid, dim3(256), 0, st, a, per);
  else klaunch((paged_read_kernel<TYPE, false>), grid, dim3(256), 0, st, a, per);
}

hipError_t paged_read(const PagedReadArgs &a, hipStream_t st) {
  const int al = a.c.type == CACHE_F16 ? 15 : 7;
  const bool vec = a.c.hd % 8 == 0 && !(((uintptr_t)a.c.k | (uintptr_t)a.c.v) & al) && !(((uintptr_t)a.kc | (uintptr_t)a.vc) & 15);
  // blocks of 16 rows (27.1 us for the rows above, 28.3 with 64), of 8 where that would leave CUs
  // without one; of more where they would be more than a grid's dimension has room for
  const long most = std::min({(long)a.t.N, (long)a.c.t.rows, (long)a.t.C});
  const long per = std::max(most * a.t.B < 16384 ? 8L : 16L, (most + kGridRow - 1) / kGridRow);
  const bool stream = (double)most * a.t.B * a.c.t.KVH * a.c.hd * 4 > kL2;
  const dim3 grid((unsigned)((most + per - 1) / per), a.t.B);
  if (!vec) klaunch(paged_read_any_kernel, grid, dim3(256), 0, st, a, (int)per);
  else if (a.c.type == CACHE_F16) launch_read<CACHE_F16>(a, grid, (int)per, stream, st);
  else if (a.c.type == CACHE_I8) launch_read<CACHE_I8>(a, grid, (int)per, stream, st);
  else launch_read<CACHE_E4M3>(a, grid, (int)per, stream, st);
  return hipGetLastError();
}

}  // namespace ec
