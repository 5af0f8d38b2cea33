// Attention of new rows over a paged K/V cache on gfx950 (layouts in trf_hip.h).
//
// For request r with n new rows, the last of its len positions, row i at position p = len - n + i:
//     O = gate * sum_j 2^(c (q.k_j) - m) v_j / sum_j 2^(c (q.k_j) - m),   c = scale * log2(e),
// over the keys j < len that the row sees (causal: j <= p; a window w: j > p - w), in one pass over the keys with a
// running m.  The query heads that share a K/V head and the request's rows are the columns of the same products:
// column x of K/V head h is row x / group, head h * group + x % group.
//
// S^T = K . Q^T puts keys on MFMA rows and columns on MFMA columns, O^T += V^T . P^T features on rows.  A 16-key
// group of the cache holds K and V in exactly the order the A operands want, so operands come from memory (or LDS)
// in 256- and 512-byte runs; key rows go in with bits 2 and 3 of their number swapped, so that the registers of S^T
// are the B operand of P.V as they stand (key_slot).
#include <algorithm>

#include "trf_device.h"

namespace trf {
namespace {

constexpr int kCols = 32;   // columns of an MFMA tile
constexpr int kWaves = 4;   // waves of a workgroup
// P may exceed 1 by this power of two before the running maximum is raised: fewer rescales, no loss (fp32 sums; P of
// at most 256 is well inside fp16).
constexpr float kRaise = 8.0f;

struct Args {
  PagedAttnArgs a;
  int32_t n_pages, kv_heads, group, gpp_shift, page_shift;  // gpp_shift: log2 of the 16-key groups of a page
  int32_t search;  // column tiles are numbered over all requests (0: a request has one)
  int32_t splits;  // parts that a tile's keys are cut into, each a workgroup's
  float* part_o;   // splits > 1: O before the division, [split][row][head][D] ...
  float* part_ml;  // ... and (m, l), [split][row][head][2]
};

// Tables do not change while a kernel runs: scalar loads.
__device__ __forceinline__ int scalar_load(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)(p);
}

__device__ __forceinline__ int key_slot(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }
// Key of register r of half-wave hh in its 32-key tile.
__device__ __forceinline__ int key_in_tile(int r, int hh) { return r < 8 ? 8 * hh + r : 8 + 8 * hh + r; }

template <bool F16>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return mfma32h(a, b, c);
  else
    return mfma32(a, b, c);
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return F16 ? pk_f16(a, b) : pk_bf16(a, b);
}

// Both halves of x with every infinity and NaN made zero; `any` collects whether there was one.
template <bool F16>
__device__ __forceinline__ uint32_t finite2(uint32_t x, bool& any) {
  constexpr uint32_t e = F16 ? 0x7c00u : 0x7f80u;
  const bool lo = (x & e) == e, hi = ((x >> 16) & e) == e;
  any |= lo | hi;
  return (lo ? 0u : x & 0xffffu) | (hi ? 0u : x & 0xffff0000u);
}

// What a workgroup's column tile is: its request, columns and the keys that any (lo, hi) and all (lo_all, hi_all) of
// its columns see.
struct Tile {
  int r, h, col0, cols;  // first column of the tile, columns of the request
  int first, rows, len;  // first row of the request, its rows, its length
  int lo, hi, lo_all, hi_all;
};

// Request whose tiles hold tile t, where request r's begin at starts[r] * group / width + r: that many tiles lie
// before it at least, and it has room for its own.  A wave looks at 64 places at a time.
__device__ __forceinline__ int request_of_tile(const Args& g, int t, int width, int& base) {
  const int lane = threadIdx.x & 63, R = g.a.n_requests;
  auto begin = [&](int r) {
    return int(int64_t(min(max(g.a.starts[r], 0), g.a.n_rows)) * g.group / width) + r;
  };
  int lo = 0, n = R;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int at = lo + lane * step;
    const uint64_t below = __ballot(lane * step < n && begin(min(at, R - 1)) <= t);
    const int k = 63 - __builtin_clzll(below | 1);
    n = min(step, lo + n - (lo + k * step));
    lo += k * step;
  }
  base = begin(lo);
  return lo;
}

__device__ __forceinline__ int clamp_key(const Tile& t, int64_t x) { return int(min(max(x, int64_t(0)), int64_t(t.len))); }

// Keys that any and all of the columns col0 .. last of the tile's request see.
__device__ __forceinline__ void key_range(const Args& g, const Tile& t, int col0, int last, int& lo, int& hi, int& lo_all,
                                          int& hi_all) {
  const int64_t base = int64_t(t.len) - t.rows, p0 = base + col0 / g.group, p1 = base + last / g.group;
  hi = g.a.causal ? clamp_key(t, p1 + 1) : t.len;
  hi_all = g.a.causal ? clamp_key(t, p0 + 1) : t.len;
  lo = g.a.window ? clamp_key(t, p0 - g.a.window + 1) : 0;
  lo_all = g.a.window ? clamp_key(t, p1 - g.a.window + 1) : 0;
}

__device__ __forceinline__ bool find_tile(const Args& g, int tile, int h, int width, Tile& t) {
  int k = 0;
  t.r = tile;
  t.h = h;
  if (g.search) {
    int base;
    t.r = __builtin_amdgcn_readfirstlane(request_of_tile(g, tile, width, base));
    k = tile - __builtin_amdgcn_readfirstlane(base);
  }
  t.first = min(max(g.a.starts[t.r], 0), g.a.n_rows);
  t.rows = min(max(g.a.starts[t.r + 1], t.first), g.a.n_rows) - t.first;
  t.cols = t.rows * g.group;
  t.col0 = k * width;
  if (t.col0 < 0 || t.col0 >= t.cols) return false;
  t.len = min(max(g.a.lens[t.r], 0), g.a.max_pages << g.page_shift);
  key_range(g, t, t.col0, min(t.col0 + width, t.cols) - 1, t.lo, t.hi, t.lo_all, t.hi_all);
  return true;
}

// What a wave carries for its columns: lane j and j + 32 hold column j of a 32-column tile.
template <int D>
struct Acc {
  f32x16 o[D / 32];
  float m, l;  // m in the scores' own units; l is this half-wave's part of the sum
};

template <int D>
__device__ __forceinline__ void clear(Acc<D>& s) {
#pragma unroll
  for (int d = 0; d < D / 32; ++d) s.o[d] = zero16();
  s.m = -INFINITY;
  s.l = 0.f;
}

// The keys that a column sees: lo .. lo + n - 1.
struct Mask {
  int lo;
  uint32_t n;
  __device__ __forceinline__ bool operator()(int key) const { return uint32_t(key - lo) < n; }
};

__device__ __forceinline__ Mask mask_of(const Args& g, const Tile& t, int col) {
  const int64_t pos = int64_t(t.len) - t.rows + col / g.group;
  const int lo = g.a.window ? clamp_key(t, pos - g.a.window + 1) : 0, hi = g.a.causal ? clamp_key(t, pos + 1) : t.len;
  return Mask{lo, uint32_t(max(hi - lo, 0))};
}

// Scores -> P as two B operands; raises m, with o and l, where a score is far above it.
template <int D, bool F16>
__device__ __forceinline__ void softmax_tile(const f32x16& s, float c, Acc<D>& acc, u32x4& p0, u32x4& p1) {
  float top = s[0];
#pragma unroll
  for (int r = 1; r < 15; r += 2) top = fmaxf(fmaxf(top, s[r]), s[r + 1]);
  top = halfwave_max(fmaxf(top, s[15]));
  const bool raise = top > acc.m && (top - acc.m) * c > (acc.m == -INFINITY ? 0.f : kRaise);
  if (__any(raise)) {
    const float m = raise ? top : acc.m;
    const float f = raise ? __builtin_amdgcn_exp2f((acc.m - m) * c) : 1.f;
    acc.m = m;
    acc.l *= f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc.o[d][r] *= f;
  }
  const float shift = acc.m == -INFINITY ? 0.f : acc.m * c;
  float e[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    e[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -shift));
    acc.l += e[r];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p0[i] = pack2<F16>(e[2 * i], e[2 * i + 1]);
    p1[i] = pack2<F16>(e[8 + 2 * i], e[8 + 2 * i + 1]);
  }
}

// Sum of the halves of a column.
__device__ __forceinline__ float halfwave_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float value16(uint16_t v, bool f16) {
  return f16 ? float(__builtin_bit_cast(_Float16, v)) : bf16_to_f32(v);
}

// What V lacks in the product of a tile that not all columns see whole.  0 * infinity is NaN, so V went in with its
// infinities and NaN as zeros; the columns that see them get them here, feature by feature.  at(u) is the tile's group
// u of 16 keys, as the cache has it.
template <int D, bool F16, class Group, class Seen>
__device__ __forceinline__ void add_infinities(Acc<D>& acc, Group at, Seen seen, int hh) {
  constexpr uint16_t e = F16 ? 0x7c00 : 0x7f80;
#pragma unroll 1
  for (int k = 0; k < 32; ++k) {
    if (!seen(k)) continue;
    const uint16_t* v = at(k >> 4) + ((k & 15) >> 3) * D * 8 + (k & 7);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint16_t x = v[(32 * d + row_of_group(q, hh) + i) * 8];
          acc.o[d][4 * q + i] += (x & e) == e ? value16(x, F16) : 0.f;
        }
        asm volatile("" ::: "memory");  // four loads at a time: this is rare, and registers are not
      }
  }
}

// Operands of column tile `col0`: q of row and head of each lane's column, zeros past the request's columns.
template <int D>
__device__ __forceinline__ void load_q(const Args& g, const Tile& t, int col, int hh, u32x4 (&qb)[D / 16]) {
  const bool valid = col < t.cols;
  const int row = valid ? col / g.group : 0, head = t.h * g.group + (valid ? col % g.group : 0);
  const uint16_t* q = g.a.q + (t.first + row) * g.a.q_stride + head * D + hh * 8;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) qb[ks] = valid ? *reinterpret_cast<const u32x4*>(q + ks * 16) : zero4();
}

// Columns' rows out: four features of a column, divided by its sum and gated; zeros for a row that saw no key.
template <int D, bool F16>
__device__ __forceinline__ void store4(const Args& g, int64_t out, int quad, const f32x4& o, float m, float l) {
  const float f = m > -INFINITY ? (g.a.gate ? g.a.gate[out] : 1.f) / l : 0.f;
  const u32x2 y = m > -INFINITY ? u32x2{pack2<F16>(o[0] * f, o[1] * f), pack2<F16>(o[2] * f, o[3] * f)} : u32x2{0u, 0u};
  *reinterpret_cast<u32x2*>(g.a.o + out * D + 4 * quad) = y;
}

// Row of O (times heads, plus the head) that is column col of the tile's request.
__device__ __forceinline__ int64_t out_row(const Args& g, const Tile& t, int col) {
  return int64_t(t.first + col / g.group) * g.a.heads + t.h * g.group + col % g.group;
}

// Key tiles (of `width` keys) of split blockIdx.y of the tile.
__device__ __forceinline__ void split_range(const Args& g, const Tile& t, int width, int& k0, int& k1) {
  k0 = t.lo / width;
  k1 = (t.hi + width - 1) / width;
  if (g.splits > 1) {
    const int each = (max(k1 - k0, 0) + g.splits - 1) / g.splits;
    k0 += each * blockIdx.y;
    k1 = min(k1, k0 + each);
  }
}

}  // namespace

// ============================================================ few columns
// A workgroup has one tile of 32 columns; its four waves take every fourth 32-key tile, K and V^T operands straight
// from the cache into registers, and join their sums in LDS at the end.
template <int D, bool F16>
__global__ __launch_bounds__(64 * kWaves) void k_paged_attn_few(Args g) {
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int kQuad = kCols + 1;  // columns of a feature quad in LDS, padded
  __shared__ f32x4 lds_o[kWaves][D / 4 * kQuad];
  __shared__ float lds_m[kWaves][kCols], lds_l[kWaves][kCols];
  const int lane = threadIdx.x & 63, wave = wave_id(), j = lane & 31, hh = lane >> 5;
  Tile t;
  if (!find_tile(g, blockIdx.x / g.kv_heads, blockIdx.x % g.kv_heads, kCols, t)) return;
  const int col = t.col0 + j;
  u32x4 qb[KS];
  load_q<D>(g, t, col, hh, qb);
  const Mask mask = mask_of(g, t, col);
  Acc<D> acc;
  clear(acc);
  const int32_t* table = g.a.table + int64_t(t.r) * g.a.max_pages;
  const int gpp_mask = (1 << g.gpp_shift) - 1;
  int k0, k1;
  split_range(g, t, 32, k0, k1);
  for (int kt = k0 + wave; kt < k1; kt += kWaves) {
    const int key0 = kt * 32;
    const uint16_t *Kg[2], *Vg[2];
    bool page_ok[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int group = 2 * kt + u;
      // the second group of the last tile may lie past the table's end
      int page = scalar_load(table + min(group >> g.gpp_shift, g.a.max_pages - 1));
      page_ok[u] = uint32_t(page) < uint32_t(g.n_pages);
      if (!page_ok[u]) page = 0;
      const int64_t base = ((((int64_t(page) * g.kv_heads + t.h) << g.gpp_shift) + (group & gpp_mask)) * 16) * D;
      Kg[u] = g.a.K + base;
      Vg[u] = g.a.V + base;
    }
    const uint16_t* Kl = (j < 16 ? Kg[0] : Kg[1]) + (hh * 16 + key_slot(j & 15)) * 8;
    u32x4 ka[KS], va[DT][2];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ka[ks] = *reinterpret_cast<const u32x4*>(Kl + ks * 256);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int d = 0; d < DT; ++d) va[d][u] = *reinterpret_cast<const u32x4*>(Vg[u] + (hh * D + 32 * d + j) * 8);
    f32x16 s = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mfma<F16>(ka[ks], qb[ks], s);
    const bool whole = key0 >= t.lo_all && key0 + 32 <= t.hi_all && page_ok[0] && page_ok[1];
    bool odd = false;  // an infinity or NaN among V that some column may not see
    auto seen = [&](int k) { return mask(key0 + k) && page_ok[k >> 4]; };
    if (!whole) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = seen(key_in_tile(r, hh)) ? s[r] : -INFINITY;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) va[d][u][i] = finite2<F16>(va[d][u][i], odd);
    }
    u32x4 p0, p1;
    softmax_tile<D, F16>(s, g.a.scale_log2, acc, p0, p1);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      acc.o[d] = mfma<F16>(va[d][0], p0, acc.o[d]);
      acc.o[d] = mfma<F16>(va[d][1], p1, acc.o[d]);
    }
    if (__any(odd)) add_infinities<D, F16>(acc, [&](int u) { return Vg[u]; }, seen, hh);
  }
  acc.l = halfwave_sum(acc.l);
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      lds_o[wave][(8 * d + 2 * q + hh) * kQuad + j] =
          f32x4{acc.o[d][4 * q], acc.o[d][4 * q + 1], acc.o[d][4 * q + 2], acc.o[d][4 * q + 3]};
  if (hh == 0) {
    lds_m[wave][j] = acc.m;
    lds_l[wave][j] = acc.l;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < kCols * (D / 4); x += 64 * kWaves) {
    const int cc = x / (D / 4), quad = x % (D / 4);
    if (t.col0 + cc >= t.cols) break;
    float m = -INFINITY, l = 0.f;
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, lds_m[w][cc]);
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < kWaves; ++w) {
      if (lds_m[w][cc] == -INFINITY) continue;
      const float f = __builtin_amdgcn_exp2f((lds_m[w][cc] - m) * g.a.scale_log2);
      l += f * lds_l[w][cc];
      o += f * lds_o[w][quad * kQuad + cc];
    }
    const int64_t out = out_row(g, t, t.col0 + cc);
    if (g.splits == 1) {
      store4<D, F16>(g, out, quad, o, m, l);
    } else {
      const int64_t at = int64_t(blockIdx.y) * g.a.n_rows * g.a.heads + out;
      *reinterpret_cast<f32x4*>(g.part_o + at * D + 4 * quad) = o;
      if (quad == 0) {
        g.part_ml[2 * at] = m;
        g.part_ml[2 * at + 1] = l;
      }
    }
  }
}

// ============================================================ many columns
// A workgroup has 4 x 32 QT columns, 32 QT a wave.  Tiles of 64 keys stream through a ring of LDS buffers, loaded
// global->LDS directly: the tile's four 16-key groups lie one after the other, each as the cache has it, and wave w
// loads group w, of one page.  A wave computes the tiles that its own columns see and meets every barrier.
template <int D, bool F16, int QT>
__global__ __launch_bounds__(64 * kWaves, 2) void k_paged_attn_many(Args g) {
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int kGroup = 2 * D;               // 16-byte chunks of a 16-key group, K or V
  constexpr int kLoads = kGroup / 64;         // 1 KB loads of one
  constexpr int kWidth = kWaves * kCols * QT;
  constexpr int kBufs = D == 64 ? 3 : 2;
  __shared__ u32x4 lds[kBufs][2][4 * kGroup];
  const int lane = threadIdx.x & 63, wave = wave_id(), j = lane & 31, hh = lane >> 5;
  Tile t;
  if (!find_tile(g, blockIdx.x / g.kv_heads, blockIdx.x % g.kv_heads, kWidth, t)) return;
  const int32_t* table = g.a.table + int64_t(t.r) * g.a.max_pages;
  const int gpp_mask = (1 << g.gpp_shift) - 1;
  int k0, k1;
  split_range(g, t, 64, k0, k1);

  // this wave's columns: the keys that any and all of them see
  const int col0 = t.col0 + wave * kCols * QT, last = min(col0 + kCols * QT, t.cols) - 1;
  const bool active = col0 < t.cols;
  int lo = 0, hi = 0, lo_all = 0, hi_all = 0;
  if (active) key_range(g, t, col0, last, lo, hi, lo_all, hi_all);

  u32x4 qb[QT][KS];
  Acc<D> acc[QT];
  Mask mask[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int col = col0 + kCols * qt + j;
    load_q<D>(g, t, col, hh, qb[qt]);
    mask[qt] = mask_of(g, t, col);
    clear(acc[qt]);
  }

  auto page_of = [&](int kt) {
    return scalar_load(table + min((4 * kt + wave) >> g.gpp_shift, g.a.max_pages - 1));
  };
  auto stage = [&](int kt, int page) {  // this wave's share of tile kt: zeros for what is no page
    const bool ok = uint32_t(page) < uint32_t(g.n_pages);
    const int64_t at = ((((int64_t(ok ? page : 0) * g.kv_heads + t.h) << g.gpp_shift) + ((4 * kt + wave) & gpp_mask)) * 16) * D;
    const int bytes = ok ? 32 * D : 0;
    const __amdgpu_buffer_rsrc_t Kr = buffer_rsrc(g.a.K + at, bytes), Vr = buffer_rsrc(g.a.V + at, bytes);
    u32x4* dst = &lds[(kt - k0) % kBufs][0][wave * kGroup];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      buffer_load_lds16(Kr, (64 * i + lane) * 16, dst + 64 * i);
      buffer_load_lds16(Vr, (64 * i + lane) * 16, dst + 4 * kGroup + 64 * i);
    }
  };
  // tile kt's operands from LDS, scores, P and P.V, for every column tile
  auto compute = [&](int kt) {
    const u32x4* Kl = lds[(kt - k0) % kBufs][0];
    const u32x4* Vl = lds[(kt - k0) % kBufs][1];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int key0 = 64 * kt + 32 * half;
      if (key0 >= hi || key0 + 32 <= lo) continue;
      bool page_ok[2];
      bool whole = key0 >= lo_all && key0 + 32 <= hi_all;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        page_ok[u] = uint32_t(scalar_load(table + min((4 * kt + 2 * half + u) >> g.gpp_shift, g.a.max_pages - 1))) <
                     uint32_t(g.n_pages);
        whole &= page_ok[u];
      }
      u32x4 ka[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        ka[ks] = Kl[(2 * half + (j >> 4)) * kGroup + (2 * ks + hh) * 16 + key_slot(j & 15)];
      u32x4 p0[QT], p1[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        f32x16 s = zero16();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = mfma<F16>(ka[ks], qb[qt][ks], s);
        if (!whole) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int k = key_in_tile(r, hh);
            s[r] = mask[qt](key0 + k) && page_ok[k >> 4] ? s[r] : -INFINITY;
          }
        }
        softmax_tile<D, F16>(s, g.a.scale_log2, acc[qt], p0[qt], p1[qt]);
      }
      bool odd = false;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        u32x4 v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          v[u] = Vl[(2 * half + u) * kGroup + hh * D + 32 * d + j];
          if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[u][i] = finite2<F16>(v[u][i], odd);
          }
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          acc[qt].o[d] = mfma<F16>(v[0], p0[qt], acc[qt].o[d]);
          acc[qt].o[d] = mfma<F16>(v[1], p1[qt], acc[qt].o[d]);
        }
      }
      if (__any(odd)) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
          add_infinities<D, F16>(
              acc[qt], [&](int u) { return reinterpret_cast<const uint16_t*>(Vl + (2 * half + u) * kGroup); },
              [&](int k) { return mask[qt](key0 + k) && page_ok[k >> 4]; }, hh);
      }
    }
  };

  if (k0 < k1) {
#pragma unroll
    for (int i = 0; i < kBufs - 1; ++i)
      if (k0 + i < k1) stage(k0 + i, page_of(k0 + i));
    int next = page_of(min(k0 + kBufs - 1, k1));  // page of the tile to be staged next, read a tile ahead
    for (int kt = k0; kt < k1; ++kt) {
      if (kBufs > 2 && kt + kBufs - 2 < k1)  // the younger tiles' loads stay in flight
        vmcnt_barrier<2 * kLoads*(kBufs - 2)>();
      else
        vmcnt_barrier<0>();
      if (kt + kBufs - 1 < k1) {
        stage(kt + kBufs - 1, next);
        next = page_of(kt + kBufs);
      }
      if (active) compute(kt);
    }
  }
  if (!active) return;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int col = col0 + kCols * qt + j;
    const float l = halfwave_sum(acc[qt].l);
    if (col >= t.cols) continue;
    const int64_t out = out_row(g, t, col), at = int64_t(blockIdx.y) * g.a.n_rows * g.a.heads + out;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 o{acc[qt].o[d][4 * q], acc[qt].o[d][4 * q + 1], acc[qt].o[d][4 * q + 2], acc[qt].o[d][4 * q + 3]};
        const int quad = 8 * d + 2 * q + hh;
        if (g.splits == 1)
          store4<D, F16>(g, out, quad, o, acc[qt].m, l);
        else
          *reinterpret_cast<f32x4*>(g.part_o + at * D + 4 * quad) = o;
      }
    if (g.splits > 1 && hh == 0) {
      g.part_ml[2 * at] = acc[qt].m;
      g.part_ml[2 * at + 1] = l;
    }
  }
}

// ============================================================ joining the splits
// Splits in ascending order, so that the sums do not depend on which finished first.
template <int D, bool F16>
__global__ __launch_bounds__(256) void k_paged_attn_join(Args g, int width) {
  Tile t;
  if (!find_tile(g, blockIdx.x / g.kv_heads, blockIdx.x % g.kv_heads, width, t)) return;
  const int64_t stride = int64_t(g.a.n_rows) * g.a.heads;
  for (int x = threadIdx.x; x < width * (D / 4); x += 256) {
    const int cc = x / (D / 4), quad = x % (D / 4);
    if (t.col0 + cc >= t.cols) break;
    const int64_t out = out_row(g, t, t.col0 + cc);
    float m = -INFINITY, l = 0.f;
    for (int s = 0; s < g.splits; ++s) m = fmaxf(m, g.part_ml[2 * (s * stride + out)]);
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < g.splits; ++s) {
      const int64_t at = s * stride + out;
      const float ms = g.part_ml[2 * at];
      const float f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ms - m) * g.a.scale_log2);
      l += f * g.part_ml[2 * at + 1];
      o += f * *reinterpret_cast<const f32x4*>(g.part_o + at * D + 4 * quad);
    }
    store4<D, F16>(g, out, quad, o, m, l);
  }
}

namespace {

// How a call is run, from what the host knows of it.
struct Plan {
  int qt;  // 0: the kernel for few columns; else 32-column tiles per wave of the one for many
  int width, tiles, search, splits;
};

Plan plan_of(const PagedShape& s, const PagedAttnArgs& a) {
  Plan p{};
  const int group = a.heads / s.kv_heads;
  const int64_t most = int64_t(a.max_new) * group;  // columns of a request, at most
  p.qt = most <= 32 ? 0 : s.head_dim == 128 || most <= kWaves * kCols ? 1 : 2;
  p.width = p.qt ? kWaves * kCols * p.qt : kCols;
  p.search = most > p.width;
  p.tiles = p.search ? int(int64_t(a.n_rows) * group / p.width) + a.n_requests : a.n_requests;
  // Parts of the keys: enough workgroups for four on each CU (two of the kernel for many columns), parts of 512 keys
  // at least.
  const int64_t blocks = int64_t(p.tiles) * s.kv_heads, want = int64_t(device_cu_count()) * (p.qt ? 2 : 4);
  p.splits = int(std::max<int64_t>(1, std::min<int64_t>({want / blocks, a.max_len / 512, 64})));
  return p;
}

}  // namespace

size_t paged_attention_workspace(const PagedShape& s, const PagedAttnArgs& a) {
  const Plan p = plan_of(s, a);
  return p.splits == 1 ? 0 : size_t(p.splits) * a.n_rows * a.heads * (s.head_dim + 2) * 4;
}

template <int D, bool F16>
void launch(const Plan& p, const Args& g, hipStream_t st) {
  const dim3 grid(unsigned(int64_t(p.tiles) * g.kv_heads), unsigned(p.splits));
  if (p.qt == 0)
    k_paged_attn_few<D, F16><<<grid, 64 * kWaves, 0, st>>>(g);
  else if (p.qt == 1)
    k_paged_attn_many<D, F16, 1><<<grid, 64 * kWaves, 0, st>>>(g);
  else if constexpr (D == 64)
    k_paged_attn_many<D, F16, 2><<<grid, 64 * kWaves, 0, st>>>(g);
  if (p.splits > 1) k_paged_attn_join<D, F16><<<grid.x, 256, 0, st>>>(g, p.width);
}

void launch_paged_attention(const PagedShape& s, const PagedAttnArgs& a, void* workspace, hipStream_t st) {
  const Plan p = plan_of(s, a);
  Args g{};
  g.a = a;
  g.n_pages = s.n_pages;
  g.kv_heads = s.kv_heads;
  g.group = a.heads / s.kv_heads;
  g.page_shift = s.page_shift;
  g.gpp_shift = s.page_shift - 4;
  g.search = p.search;
  g.splits = p.splits;
  g.part_o = static_cast<float*>(workspace);
  g.part_ml = g.part_o + size_t(p.splits) * a.n_rows * a.heads * s.head_dim;
  if (s.head_dim == 64)
    s.f16 ? launch<64, true>(p, g, st) : launch<64, false>(p, g, st);
  else
    s.f16 ? launch<128, true>(p, g, st) : launch<128, false>(p, g, st);
}

}  // namespace trf
