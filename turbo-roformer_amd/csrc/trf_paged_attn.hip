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

constexpr int kCols = 32;  // columns of a wave's tile
// P may exceed 1 by this power of two before the running maximum is raised: fewer rescales, no loss (fp32 sums; P of
// at most 256 is well inside fp16).
constexpr float kRaise = 8.0f;

struct Args {
  PagedAttnArgs a;
  int32_t n_pages, kv_heads, group, gpp_shift, page_shift;  // gpp_shift: log2 of the 16-key groups of a page
  int32_t tiles;   // column tiles: of the requests one after the other, or one each (search = 0)
  int32_t search;
};

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
  const int last = min(t.col0 + width, t.cols) - 1;
  const int64_t p0 = int64_t(t.len) - t.rows + t.col0 / g.group, p1 = int64_t(t.len) - t.rows + last / g.group;
  auto key = [&](int64_t x) { return int(min(max(x, int64_t(0)), int64_t(t.len))); };
  t.hi = g.a.causal ? key(p1 + 1) : t.len;
  t.hi_all = g.a.causal ? key(p0 + 1) : t.len;
  t.lo = g.a.window ? key(p0 - g.a.window + 1) : 0;
  t.lo_all = g.a.window ? key(p1 - g.a.window + 1) : 0;
  return true;
}

// One 32-key, 32-column tile's state of a column: lane j and j + 32 hold column j.
template <int D>
struct Acc {
  f32x16 o[D / 32];
  float m, l;  // m is in the scores' own units; l is this half-wave's part of the sum
};

template <int D>
__device__ __forceinline__ void clear(Acc<D>& s) {
#pragma unroll
  for (int d = 0; d < D / 32; ++d) s.o[d] = zero16();
  s.m = -INFINITY;
  s.l = 0.f;
}

// Scores -> P as two B operands; raises m, with o and l, where a score is far above it.
template <int D, bool F16>
__device__ __forceinline__ void softmax_tile(const f32x16& s, float c, Acc<D>& acc, u32x4& p0, u32x4& p1) {
  float top = s[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
  top = halfwave_max(top);
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

}  // namespace

// ============================================================ few columns
// A workgroup has one tile of 32 columns; its four waves take every fourth 32-key tile, K and V^T operands straight
// from the cache into registers, and join their sums in LDS at the end.
template <int D, bool F16>
__global__ __launch_bounds__(256) void k_paged_attn_few(Args g) {
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int kQuad = kCols + 1;  // columns of a feature quad in LDS, padded
  __shared__ f32x4 lds_o[4][D / 4 * kQuad];
  __shared__ float lds_m[4][kCols], lds_l[4][kCols];
  const int lane = threadIdx.x & 63, wave = wave_id(), j = lane & 31, hh = lane >> 5;
  Tile t;
  if (!find_tile(g, blockIdx.x / g.kv_heads, blockIdx.x % g.kv_heads, kCols, t)) return;

  const int col = t.col0 + j;
  const bool valid = col < t.cols;
  const int row = col / g.group, head = t.h * g.group + col % g.group;
  const int64_t pos = int64_t(t.len) - t.rows + row;
  u32x4 qb[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
    qb[ks] = valid ? *reinterpret_cast<const u32x4*>(g.a.q + (t.first + row) * g.a.q_stride + head * D + (2 * ks + hh) * 8)
                   : zero4();
  Acc<D> acc;
  clear(acc);
  const float c = g.a.scale_log2;
  const int32_t* table = g.a.table + int64_t(t.r) * g.a.max_pages;
  const int gpp_mask = (1 << g.gpp_shift) - 1;
  for (int kt = (t.lo >> 5) + wave; kt * 32 < t.hi; kt += 4) {
    const int key0 = kt * 32;
    const uint16_t *Kg[2], *Vg[2];
    bool page_ok[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int group = 2 * kt + u;
      // the second group of the last tile may lie past the table's end
      const int at = min(group >> g.gpp_shift, g.a.max_pages - 1);
      int page = table[at];
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
      for (int d = 0; d < DT; ++d)
        va[d][u] = *reinterpret_cast<const u32x4*>(Vg[u] + (hh * D + 32 * d + j) * 8);
    f32x16 s = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mfma<F16>(ka[ks], qb[ks], s);
    const bool whole = key0 >= t.lo_all && key0 + 32 <= t.hi_all && page_ok[0] && page_ok[1];
    bool odd = false;  // an infinity or NaN among V that some column may not see
    auto seen = [&](int k) {
      const int key = key0 + k;
      return key < t.len && page_ok[k >> 4] && (!g.a.causal || key <= pos) && (!g.a.window || key > pos - g.a.window);
    };
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
    softmax_tile<D, F16>(s, c, acc, p0, p1);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      acc.o[d] = mfma<F16>(va[d][0], p0, acc.o[d]);
      acc.o[d] = mfma<F16>(va[d][1], p1, acc.o[d]);
    }
    if (__any(odd)) {
      // 0 * infinity is NaN, so V went into the product with its infinities and NaN as zeros; the columns that see
      // them get them here, feature by feature.
      for (int k = 0; k < 32; ++k) {
        if (!seen(k)) continue;
        const uint16_t* v = (k < 16 ? Vg[0] : Vg[1]) + ((k & 15) >> 3) * D * 8 + (k & 7);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const uint16_t x = v[(32 * d + row_of_group(r >> 2, hh) + (r & 3)) * 8];
            constexpr uint16_t e = F16 ? 0x7c00 : 0x7f80;
            if ((x & e) == e) acc.o[d][r] += value16(x, F16);
          }
      }
    }
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
  for (int x = threadIdx.x; x < kCols * (D / 4); x += 256) {
    const int cc = x / (D / 4), quad = x % (D / 4);
    if (t.col0 + cc >= t.cols) break;
    float m = -INFINITY, l = 0.f;
    for (int w = 0; w < 4; ++w) m = fmaxf(m, lds_m[w][cc]);
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    if (m > -INFINITY)
      for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f((lds_m[w][cc] - m) * c);
        if (lds_m[w][cc] == -INFINITY) continue;
        l += f * lds_l[w][cc];
        o += f * lds_o[w][quad * kQuad + cc];
      }
    const int rr = (t.col0 + cc) / g.group, hd = t.h * g.group + (t.col0 + cc) % g.group;
    const int64_t out = int64_t(t.first + rr) * g.a.heads + hd;
    // a row that sees no key is zero
    const float f = m > -INFINITY ? (g.a.gate ? g.a.gate[out] : 1.f) / l : 0.f;
    const u32x2 y = m > -INFINITY ? u32x2{pack2<F16>(o[0] * f, o[1] * f), pack2<F16>(o[2] * f, o[3] * f)} : u32x2{0u, 0u};
    *reinterpret_cast<u32x2*>(g.a.o + out * D + 4 * quad) = y;
  }
}

size_t paged_attention_workspace(const PagedShape&, const PagedAttnArgs&) { return 0; }

void launch_paged_attention(const PagedShape& s, const PagedAttnArgs& a, void*, hipStream_t st) {
  Args g{};
  g.a = a;
  g.n_pages = s.n_pages;
  g.kv_heads = s.kv_heads;
  g.group = a.heads / s.kv_heads;
  g.page_shift = s.page_shift;
  g.gpp_shift = s.page_shift - 4;
  g.search = int64_t(a.max_new) * g.group > kCols;
  g.tiles = g.search ? int(int64_t(a.n_rows) * g.group / kCols) + a.n_requests : a.n_requests;
  const auto kernel = s.head_dim == 64 ? (s.f16 ? k_paged_attn_few<64, true> : k_paged_attn_few<64, false>)
                                       : (s.f16 ? k_paged_attn_few<128, true> : k_paged_attn_few<128, false>);
  kernel<<<unsigned(int64_t(g.tiles) * s.kv_heads), 256, 0, st>>>(g);
}

}  // namespace trf
