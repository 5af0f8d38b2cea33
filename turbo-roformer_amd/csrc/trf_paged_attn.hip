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
#include <type_traits>

#include "trf_device.h"

namespace trf {
namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kCols = 32;   // columns of an MFMA tile
constexpr int kWaves = 4;   // waves of a workgroup
// P may exceed its value at the running maximum by this power of two before that is raised: fewer rescales, no loss (fp32
// sums).  fp16 reaches from 2^-24 to 2^16: there P is 2^7 at the maximum, so that it keeps to 2^15 and weights down to
// 2^-31 of the largest are not lost (of 131,071 keys with 2^-26 of it each, together 2^-9 of the sum, nothing was left).
constexpr float kRaise = 8.0f;
template <bool F16>
constexpr float kAtMax = F16 ? 7.0f : 0.0f;
// What the shift and the limit are rounded by grows with the scores: past this, times the scale, every larger one raises
// the maximum.
constexpr float kLargeScore = 4194304.0f;

struct Args {
  PagedAttnArgs a;
  int32_t n_pages, kv_heads, group, gpp_shift, page_shift;  // gpp_shift: log2 of the 16-key groups of a page
  int32_t search;  // column tiles are numbered over all requests: 1 in their order, 2 the ones with most keys first (0: a
                   // request has one)
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

// The same for at most 64 requests, in the order of the keys that their tiles see, most first: with a few rounds of
// workgroups of unequal lengths the long ones must not come last (us, in their order and so: 62 sequences of 200 to 4000
// keys, 50 to 200 rows 87 and 75; 16 of 1000 to 8000, 500 to 1000 rows 193 and 158).  A lane has a request.  False: all
// see as many, and their order will do.  r: -1 for a tile past the last; at: the tile's number within the request.
__device__ __forceinline__ bool request_by_length(const Args& g, int t, int width, int& r, int& at) {
  const int lane = threadIdx.x & 63, R = g.a.n_requests, mine = min(lane, R - 1);
  const int s0 = min(max(g.a.starts[mine], 0), g.a.n_rows), n = min(max(g.a.starts[mine + 1], s0), g.a.n_rows) - s0;
  const int len = min(max(g.a.lens[mine], 0), g.a.max_pages << g.page_shift);
  const int keys = g.a.window ? int(min(int64_t(len), int64_t(n) + g.a.window)) : len;
  if (__all(keys == __builtin_amdgcn_readfirstlane(keys))) return false;
  const int tiles = lane < R ? int((int64_t(n) * g.group + width - 1) / width) : 0;
  // keys (of 2^25 at most) and, for equal ones, the request: no two the same
  const int order = min(keys, (1 << 25) - 1) << 6 | (63 - lane);
  int first = 0;
  for (int q = 0; q < R; ++q)
    first += __builtin_amdgcn_readlane(order, q) > order ? __builtin_amdgcn_readlane(tiles, q) : 0;
  const uint64_t found = __ballot(t >= first && t < first + tiles);
  r = found ? __builtin_ctzll(found) : -1;
  // a causal request's last rows see the most
  if (found) at = __builtin_amdgcn_readlane(tiles, r) - 1 - (t - __builtin_amdgcn_readlane(first, r));
  return true;
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
  if (g.search == 2 && request_by_length(g, tile, width, t.r, k)) {
    if (t.r < 0) return false;
  } else if (g.search) {
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
  float m, shift;  // running maximum in the scores' own units, and times the scale, less kAtMax (0 while there is none)
  float limit;     // scores above this raise it: kRaise past it, in the scores' own units
  f32x4 sum[2];    // this lane's sums of P's first and second halves of 8, in each register (row_sum)
};

template <int D>
__device__ __forceinline__ void clear(Acc<D>& s) {
#pragma unroll
  for (int d = 0; d < D / 32; ++d) s.o[d] = zero16();
  s.m = -INFINITY;
  s.limit = -INFINITY;
  s.shift = 0.f;
  s.sum[0] = s.sum[1] = f32x4{0.f, 0.f, 0.f, 0.f};
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

// The sum of the rounded P, the weights that P.V applies, on the matrix pipe instead of by 16 additions a lane:
// v_mfma_f32_4x4x4 is 16 products of 4 x 4 matrices, lane l has column l % 4 of number l / 4, four values of it an
// operand.  With ones for A each lane gets the sum of its own values, in all four registers: a NaN among them reaches no
// other column, as it would with zeros in A (0 * NaN).  Two sums, so that no product waits for the one before it (the
// 17 s chunk 436 us with one, 434 with two; v_mfma_f32_16x16x32 with zeros took 433).
template <bool F16>
__device__ __forceinline__ f32x4 sum4(uint32_t a, uint32_t b, f32x4 c) {
  const u32x2 x{a, b}, ones = F16 ? u32x2{0x3c003c00u, 0x3c003c00u} : u32x2{0x3f803f80u, 0x3f803f80u};
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_4x4x4f16(__builtin_bit_cast(f16x4, ones), __builtin_bit_cast(f16x4, x), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(__builtin_bit_cast(s16x4, ones), __builtin_bit_cast(s16x4, x), c, 0, 0, 0);
}

template <bool F16, int D>
__device__ __forceinline__ void row_sum(Acc<D>& acc, u32x4 p0, u32x4 p1) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    acc.sum[0] = sum4<F16>(p0[i], p0[i + 1], acc.sum[0]);
    acc.sum[1] = sum4<F16>(p1[i], p1[i + 1], acc.sum[1]);
  }
}

// A column's sum, of its two lanes.
template <int D>
__device__ __forceinline__ float sum_of(const Acc<D>& acc) {
  const float l = acc.sum[0][0] + acc.sum[1][0];
  return l + __shfl_xor(l, 32);
}

// The largest score of this lane's half of a column.
__device__ __forceinline__ float half_max(const f32x16& s) {
  float top = s[0];
#pragma unroll
  for (int r = 1; r < 15; r += 2) top = fmaxf(fmaxf(top, s[r]), s[r + 1]);
  return fmaxf(top, s[15]);
}

// Whether any column of the wave has a score far above its maximum, or its first.
template <int D>
__device__ __forceinline__ bool above(const Acc<D>& acc, float top) {
  return __builtin_amdgcn_ballot_w64(top > acc.limit) != 0;
}

// Raises the maxima of the columns that are.
template <bool F16, int D>
__device__ __forceinline__ void raise(Acc<D>& acc, float half_top, float c) {
  const float top = halfwave_max(half_top);
  const bool up = top > acc.limit;
  const float f = up ? __builtin_amdgcn_exp2f((acc.m - top) * c) : 1.f;
  if (up) {
    acc.m = top;
    acc.shift = top * c - kAtMax<F16>;
    acc.limit = fabsf(acc.shift) < kLargeScore ? top + kRaise / c : top;
  }
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc.o[d][r] *= f;
  acc.sum[0] *= f;
  acc.sum[1] *= f;
}

// Half of a tile's scores -> P as a B operand: rounded to the type of V, as the matrix instruction takes both in one type.
// With the sum formed from the same values (row_sum) the weights that are applied still add to one.
template <bool F16, int HALF>
__device__ __forceinline__ u32x4 weights(const f32x16& s, float c, float shift) {
  float e[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[8 * HALF + r], c, -shift));
  return u32x4{pack2<F16>(e[0], e[1]), pack2<F16>(e[2], e[3]), pack2<F16>(e[4], e[5]), pack2<F16>(e[6], e[7])};
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

// Columns' rows out: four features of a column, divided by its sum and gated; zeros for a row that saw no key, whose sum
// is zero (where it is NaN so is o, and stays it).
template <int D, bool F16>
__device__ __forceinline__ void store4(const Args& g, int64_t out, int quad, const f32x4& o, float l) {
  const float f = __float_as_uint(l) << 1 ? (g.a.gate ? g.a.gate[out] : 1.f) / l : 0.f;
  *reinterpret_cast<u32x2*>(g.a.o + out * D + 4 * quad) = u32x2{pack2<F16>(o[0] * f, o[1] * f), pack2<F16>(o[2] * f, o[3] * f)};
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
// from the cache into registers (each byte of the cache is used once, so LDS would only pass it on), and join their sums
// in LDS at the end.  Bound by HBM, or by latency for short caches: single rows of 5 sequences of 100,000 to 131,000 keys,
// 32 and 8 heads of 128, 407-425 us by host with the join (5.5-5.7 TB/s; one tile at a time 408 + 20, as it came first 2475);
// one row of 62 sequences of 600 to 1701 keys, 8 heads of 64, 32 us (4.6 TB/s: two workgroups a CU of unequal lengths); one
// row of 17 keys 5.1 us.  Head dim 128 runs one wave a SIMD, with all its registers: at two, with one tile each, 443 us.
template <int D, bool F16>
__global__ __launch_bounds__(64 * kWaves, D == 64 ? 2 : 1) void k_paged_attn_few(Args g) {
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
  const float c = g.a.scale_log2;
  const int32_t* table = g.a.table + int64_t(t.r) * g.a.max_pages;
  const uint32_t page_bytes = uint32_t(g.kv_heads) * D * 2 << g.page_shift;
  const int64_t head_at = int64_t(t.h) * D << g.page_shift;
  const uint16_t *Kh = g.a.K + head_at, *Vh = g.a.V + head_at;
  struct Operands {
    u32x4 ka[KS], va[DT][2];
    uint64_t at0, at1;  // elements from the head's first to the two groups, and whether they are in a page
    bool ok0, ok1;
  };
  auto group_at = [&](int group, bool& ok) {
    // the second group of the last tile may lie past the table's end
    const int page = scalar_load(table + min(group >> g.gpp_shift, g.a.max_pages - 1));
    ok = uint32_t(page) < uint32_t(g.n_pages);
    return (uint64_t(uint32_t(ok ? page : 0)) * page_bytes + uint32_t((group & ((1 << g.gpp_shift) - 1)) * 32 * D)) / 2;
  };
  auto load = [&](Operands& x, int kt) {
    x.at0 = group_at(2 * kt, x.ok0);
    x.at1 = group_at(2 * kt + 1, x.ok1);
    const uint16_t* Kl = Kh + (j < 16 ? x.at0 : x.at1) + (hh * 16 + key_slot(j & 15)) * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) x.ka[ks] = *reinterpret_cast<const u32x4*>(Kl + ks * 256);
    const uint16_t* Vl = Vh + (hh * D + j) * 8;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      x.va[d][0] = *reinterpret_cast<const u32x4*>(Vl + x.at0 + 256 * d);
      x.va[d][1] = *reinterpret_cast<const u32x4*>(Vl + x.at1 + 256 * d);
    }
  };
  // EDGE: not all columns see all of the tile.
  auto tile = [&](auto edge, Operands& x, int key0) {
    constexpr bool EDGE = decltype(edge)::value;
    f32x16 s = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mfma<F16>(x.ka[ks], qb[ks], s);
    bool odd = false;  // an infinity or NaN among V that some column may not see
    const bool ok0 = x.ok0, ok1 = x.ok1;
    auto seen = [&](int k) { return mask(key0 + k) && (k < 16 ? ok0 : ok1); };
    if (EDGE) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = seen(key_in_tile(r, hh)) ? s[r] : -INFINITY;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) x.va[d][u][i] = finite2<F16>(x.va[d][u][i], odd);
    }
    const float top = half_max(s);
    if (above(acc, top)) raise<F16>(acc, top, c);
    const u32x4 p0 = weights<F16, 0>(s, c, acc.shift), p1 = weights<F16, 1>(s, c, acc.shift);
    row_sum<F16>(acc, p0, p1);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      acc.o[d] = mfma<F16>(x.va[d][0], p0, acc.o[d]);
      acc.o[d] = mfma<F16>(x.va[d][1], p1, acc.o[d]);
    }
    if (EDGE && __any(odd)) {
      const uint16_t *V0 = Vh + x.at0, *V1 = Vh + x.at1;
      add_infinities<D, F16>(acc, [&](int u) { return u ? V1 : V0; }, seen, hh);
    }
  };
  auto compute = [&](Operands& x, int kt) {
    const int key0 = kt * 32;
    if (key0 >= t.lo_all && key0 + 32 <= t.hi_all && x.ok0 && x.ok1)
      tile(std::integral_constant<bool, false>{}, x, key0);
    else
      tile(std::integral_constant<bool, true>{}, x, key0);
  };
  int k0, k1;
  split_range(g, t, 32, k0, k1);
  Operands even, odd;
  int kt = k0 + wave;
  // two tiles' operands in turn: one on its way from memory while the other is worked on
  if (kt < k1) load(even, kt);
  for (; kt < k1; kt += 2 * kWaves) {
    if (kt + kWaves < k1) load(odd, kt + kWaves);
    compute(even, kt);
    if (kt + kWaves >= k1) break;
    if (kt + 2 * kWaves < k1) load(even, kt + 2 * kWaves);
    compute(odd, kt + kWaves);
  }
  const float l = sum_of(acc);
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      lds_o[wave][(8 * d + 2 * q + hh) * kQuad + j] =
          f32x4{acc.o[d][4 * q], acc.o[d][4 * q + 1], acc.o[d][4 * q + 2], acc.o[d][4 * q + 3]};
  if (hh == 0) {
    lds_m[wave][j] = acc.m;
    lds_l[wave][j] = l;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < kCols * (D / 4); x += 64 * kWaves) {
    const int cc = x / (D / 4), quad = x % (D / 4);
    if (t.col0 + cc >= t.cols) break;
    float m = -INFINITY, l = 0.f;
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, lds_m[w][cc]);
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < kWaves; ++w) {
      const float f = lds_m[w][cc] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((lds_m[w][cc] - m) * c);
      l += f * lds_l[w][cc];
      o += f * lds_o[w][quad * kQuad + cc];
    }
    const int64_t out = out_row(g, t, t.col0 + cc);
    if (g.splits == 1) {
      store4<D, F16>(g, out, quad, o, l);
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
// A workgroup has 4 x 32 QT columns, 32 QT a wave.  K and V stream through a ring of LDS buffers, loaded global->LDS directly
// in stages of 64 (D = 64) or 32 (D = 128) keys: 16-key groups one after the other, each as the cache has it, so that
// a wave loads one page's part of a stage.
//
// A step is 32 keys (a unit) and 32 columns.  Matrix and vector work of one step depend on each other end to end
// (scores, maximum, P, P.V), so a wave works on three steps at once: while P of one is formed, the scores of the next
// and P.V of the one before run on the matrix pipe, in the shadow of the exponentials.  With QT = 2 the steps of a unit
// take turns on the two column tiles, and each K and V operand read from LDS feeds two products.  Raising the maximum,
// masks and infinities leave that path (rare).
//
// Bound by issue and by waits, about alike, beside a matrix pipe that is busy 44% of the cycles at 1.9-2.1 GHz: about 50
// vector instructions and 16 exponentials a step, for 12 (D = 64) or 20 MFMAs, 4 of them small; of a wave's cycles
// 47% (40% at D = 128) issue, 27% (35%) wait for their turn, 26% (24%) for loads and the stages' barriers.  Measured: 62
// sequences of 1701 rows over 1701 keys, 8 heads of 64, 432-444 us by host (830-850 TFLOP/s; a large library matrix product
// reaches 1190); 9 sequences of 300 to 600 rows over 2400 to 5800 keys, 32 and 8 heads of 128, 280-288 us (840-870
// TFLOP/s: 1104 workgroups in 2.2 rounds of 512); 8 of 700 rows over 6000 keys 524 us (990 TFLOP/s).  Steps on the way (us
// for the first and the second): K and V through LDS 566 and 371, three steps at once 521 and 344, two column tiles a wave
// and a loop without edges 486 and 331.
template <int D, int QT>
struct Many {
  static constexpr int kStageKeys = D == 64 ? 64 : 32, kUnits = kStageKeys / 32;  // keys and units of a stage
  static constexpr int kAhead = D == 64 && QT == 1 ? 1 : 2;  // stages whose loads are in flight past the one waited for
  // stages in LDS: V of unit i, K of i + 2, and the ones in flight (48 KB, 64 KB or 80 KB, for 3 or 2 workgroups a CU)
  static constexpr int kBufs = kAhead + 1 + 2 / kUnits;
  static constexpr int kGroup = 2 * D;              // 16-byte chunks of a 16-key group, K or V
  static constexpr int kStageGroups = kStageKeys / 16;
  static constexpr int kStage = 2 * kStageGroups * kGroup;  // chunks of a stage: K groups, then V groups
  static constexpr int kLoads = kStage / 64 / kWaves;       // 1 KB loads of a wave
};

template <int D, bool F16, int QT>
__global__ __launch_bounds__(64 * kWaves, D == 64 && QT == 1 ? 3 : 2) void k_paged_attn_many(Args g) {
  using M = Many<D, QT>;
  constexpr int KS = D / 16, DT = D / 32;
  __shared__ u32x4 lds[M::kBufs][M::kStage];
  const int lane = threadIdx.x & 63, wave = wave_id(), j = lane & 31, hh = lane >> 5;
  Tile t;
  if (!find_tile(g, blockIdx.x / g.kv_heads, blockIdx.x % g.kv_heads, kWaves * kCols * QT, t)) return;
  const int32_t* table = g.a.table + int64_t(t.r) * g.a.max_pages;
  const float c = g.a.scale_log2;
  int s0, s1;  // stages
  split_range(g, t, M::kStageKeys, s0, s1);
  const int n_stages = max(s1 - s0, 0), n_units = n_stages * M::kUnits, first_key = s0 * M::kStageKeys;

  // This wave's share of stage st: K and V of one 16-key group (D = 64), or one of the two (D = 128).
  constexpr int kGroupsEach = M::kLoads * 64 / M::kGroup;
  static_assert(kGroupsEach * kWaves == 2 * M::kStageGroups, "a wave loads whole groups");
  const int my_group = wave % M::kStageGroups, first_group = M::kStageGroups * s0 + my_group;
  const uint32_t page_bytes = uint32_t(g.kv_heads) * D * 2 << g.page_shift;
  const int64_t head = int64_t(t.h) * D << g.page_shift;
  const uint16_t *Kh = g.a.K + head, *Vh = g.a.V + head;
  auto page_of = [&](int st) {
    return scalar_load(table + min((first_group + M::kStageGroups * st) >> g.gpp_shift, g.a.max_pages - 1));
  };
  int slot = 0;  // where the next stage goes
  auto stage = [&](int st, int page) {  // zeros for what is no page
    const bool ok = uint32_t(page) < uint32_t(g.n_pages);
    const int in = (first_group + M::kStageGroups * st) & ((1 << g.gpp_shift) - 1);
    const uint64_t at = uint64_t(uint32_t(ok ? page : 0)) * page_bytes + uint32_t(in * 32 * D);
    const int bytes = ok ? 32 * D : 0;
    u32x4* dst = lds[0] + slot + my_group * M::kGroup;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      if (kGroupsEach == 1 && v != wave / M::kStageGroups) continue;
      const __amdgpu_buffer_rsrc_t r = buffer_rsrc(reinterpret_cast<const char*>(v ? Vh : Kh) + at, bytes);
#pragma unroll
      for (int i = 0; i < M::kGroup / 64; ++i)
        buffer_load_lds16(r, (64 * i + lane) * 16, dst + v * M::kStageGroups * M::kGroup + 64 * i);
    }
    slot = slot == (M::kBufs - 1) * M::kStage ? 0 : slot + M::kStage;
  };
  constexpr int kFirst = 2 / M::kUnits;  // stage that the end of step 0 waits for
  for (int st = 0; st < min(kFirst + M::kAhead, n_stages); ++st) stage(st, page_of(st));
  int next = page_of(kFirst + M::kAhead);

  // entries of these stages' keys that are no pages: then every unit looks its groups up
  bool bad = false;
  const int last = min(int64_t(t.hi), int64_t(s1) * M::kStageKeys);
  const int e1 = min(((last + 15) / 16 + (1 << g.gpp_shift) - 1) >> g.gpp_shift, g.a.max_pages);
  for (int e = (first_key >> g.page_shift) + lane; e < e1; e += 64) bad |= uint32_t(table[e]) >= uint32_t(g.n_pages);
  const bool any_bad = __any(bad);

  // this wave's columns, and its units a .. b - 1 (counted from the workgroup's first)
  const int col0 = t.col0 + wave * kCols * QT;
  const bool active = col0 < t.cols;
  int lo = 0, hi = 0, lo_all = 0, hi_all = 0;
  if (active) key_range(g, t, col0, min(col0 + kCols * QT, t.cols) - 1, lo, hi, lo_all, hi_all);
  const int a = min(max(lo - first_key, 0) / 32, n_units), b = min((max(hi - first_key, 0) + 31) / 32, n_units);
  u32x4 qb[QT][KS];
  Mask mask[QT];
  Acc<D> acc[QT];
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    load_q<D>(g, t, col0 + kCols * x + j, hh, qb[x]);
    mask[x] = mask_of(g, t, col0 + kCols * x + j);
    clear(acc[x]);
  }

  // places of units in the ring
  const int k_lane = (j >> 4) * M::kGroup + hh * 16 + key_slot(j & 15);
  const int v_lane = M::kStageGroups * M::kGroup + hh * D + j;
  auto place = [&](int i) { return (i / M::kUnits) % M::kBufs * M::kStage + i % M::kUnits * 2 * M::kGroup; };
  auto after = [&](int at, int i) {  // unit i's place, after unit i - 1's
    if (i % M::kUnits) return at + 2 * M::kGroup;
    at += M::kStage - 2 * M::kGroup * (M::kUnits - 1);
    return at == M::kBufs * M::kStage ? 0 : at;
  };
  // The end of step i, the same for all waves: unit i + 2 lies in LDS, and the next stage's loads are under way.
  auto advance = [&](int i) {
    if ((i + 2) % M::kUnits != 0 || i + 2 >= n_units) return;
    const int st = (i + 2) / M::kUnits;
    if (M::kAhead > 1 && st + M::kAhead - 1 < n_stages)
      vmcnt_barrier<M::kLoads*(M::kAhead - 1)>();
    else
      vmcnt_barrier<0>();
    if (st + M::kAhead < n_stages) {
      stage(st + M::kAhead, next);
      next = page_of(st + M::kAhead + 1);
    }
  };
  auto group_ok = [&](int key) {  // whether the key's group is in a page, where not all are
    return !any_bad || uint32_t(scalar_load(table + min(key >> 4 >> g.gpp_shift, g.a.max_pages - 1))) < uint32_t(g.n_pages);
  };

  // Operands of the step after the present one (K) and of the one before it (V, P: zeros before the first), and the
  // scores of the present step and the next.
  u32x4 ka[KS], va[DT][2], p0[QT], p1[QT];
  auto no_p_v = [&]() {
#pragma unroll
    for (int x = 0; x < QT; ++x) p0[x] = p1[x] = zero4();
#pragma unroll
    for (int d = 0; d < DT; ++d) va[d][0] = va[d][1] = zero4();
  };
  no_p_v();
  f32x16 s_even = zero16(), s_odd = zero16();
  auto load_k = [&](int at) {
    const u32x4* K = lds[0] + at + k_lane;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ka[ks] = K[ks * 32];
  };
  auto scores = [&](f32x16& s, int x) {
    s = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mfma<F16>(ka[ks], qb[x][ks], s);
  };
  auto p_v = [&](int x) {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      acc[x].o[d] = mfma<F16>(va[d][0], p0[x], acc[x].o[d]);
      acc[x].o[d] = mfma<F16>(va[d][1], p1[x], acc[x].o[d]);
    }
  };

  if (n_stages >= kFirst + M::kAhead)
    vmcnt_barrier<M::kLoads * (kFirst + M::kAhead - 2 / M::kUnits)>();  // units 0 and 1
  else
    vmcnt_barrier<0>();
  for (int i = 0; i < a; ++i) advance(i);
  if (a < b) {
    int at = place(a), at1 = after(at, a + 1);
    load_k(at);
    scores(s_even, 0);
    if (QT == 1) load_k(at1);
    // units all of whose keys all columns see
    const int w0 = (max(lo_all - first_key, 0) + 31) / 32, w1 = any_bad ? 0 : min(max(hi_all - first_key, 0) / 32, b);
    // Step of unit i and column tile x, whose scores are in s; before it came tile x of unit i - 1 (QT = 1) or the other
    // tile.  EDGE: not all columns see all of the unit.
    bool odd = false;  // EDGE: V of the unit has infinities or NaN, zeros in va
    auto step = [&](auto edge, int i, int x, f32x16& s, f32x16& s_next) {
      constexpr bool EDGE = decltype(edge)::value;
      const bool last = x == QT - 1;
      const int key0 = first_key + 32 * i;
      if (EDGE) {
        const bool ok0 = group_ok(key0), ok1 = group_ok(key0 + 16);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int k = key_in_tile(r, hh);
          s[r] = mask[x](key0 + k) && (k < 16 ? ok0 : ok1) ? s[r] : -INFINITY;
        }
      }
      const float top = half_max(s);
      if (above(acc[x], top)) {
        if (QT == 1) {  // P.V of the unit before belongs to the sums that are scaled here
          p_v(x);
          no_p_v();
        }
        raise<F16>(acc[x], top, c);
      }
      // two stretches of matrix work with vector work of about its length, and the operands' loads behind each
      scores(s_next, last ? 0 : x + 1);
      const u32x4 n0 = weights<F16, 0>(s, c, acc[x].shift);
      __builtin_amdgcn_sched_barrier(0);
      if (QT == 2 && !last) load_k(at1);
      p_v(QT - 1 - x);
      p1[x] = weights<F16, 1>(s, c, acc[x].shift);
      p0[x] = n0;
      __builtin_amdgcn_sched_barrier(0);
      row_sum<F16>(acc[x], p0[x], p1[x]);
      if (QT == 1) {  // K first: the next step begins with it
        advance(i);
        load_k(after(at1, i + 2));
      }
      if (x == 0) {
        const u32x4* V = lds[0] + at + v_lane;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int u = 0; u < 2; ++u) va[d][u] = V[u * M::kGroup + 32 * d];
        if (EDGE) {
          bool any = false;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int y = 0; y < 4; ++y) va[d][u][y] = finite2<F16>(va[d][u][y], any);
          odd = __any(any);
        }
      }
      if (EDGE && last && odd) {
        const u32x4* unit = lds[0] + at + M::kStageGroups * M::kGroup;
        auto group = [&](int u) { return reinterpret_cast<const uint16_t*>(unit + u * M::kGroup); };
#pragma unroll
        for (int y = 0; y < QT; ++y)
          add_infinities<D, F16>(acc[y], group, [&](int k) { return mask[y](key0 + k) && group_ok(key0 + (k & 16)); }, hh);
      }
      if (last) {
        if (QT == 2) advance(i);
        at = at1;
        at1 = after(at1, i + 2);
      }
    };
    const auto inner = std::integral_constant<bool, false>{};
    const auto edge = std::integral_constant<bool, true>{};
    for (int i = a; i < b;) {
      // the scores change places from step to step without being copied: two steps a turn
      if constexpr (QT == 1) {
        if (i >= w0)
          for (; i + 1 < w1; i += 2) {
            step(inner, i, 0, s_even, s_odd);
            step(inner, i + 1, 0, s_odd, s_even);
          }
        if (i < b) {
          step(edge, i++, 0, s_even, s_odd);
          s_even = s_odd;
        }
      } else {
        if (i >= w0)
          for (; i < w1; ++i) {
            step(inner, i, 0, s_even, s_odd);
            step(inner, i, 1, s_odd, s_even);
          }
        if (i < b) {
          step(edge, i, 0, s_even, s_odd);
          step(edge, i++, 1, s_odd, s_even);
        }
      }
    }
    p_v(QT - 1);
  }
  for (int i = max(a, b); i < n_units; ++i) advance(i);
  if (!active) return;
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const int col = col0 + kCols * x + j;
    const float l = sum_of(acc[x]);
    if (col >= t.cols) continue;
    const int64_t out = out_row(g, t, col), part = int64_t(blockIdx.y) * g.a.n_rows * g.a.heads + out;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16& o = acc[x].o[d];
        const f32x4 o4{o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]};
        const int quad = 8 * d + 2 * q + hh;
        if (g.splits == 1)
          store4<D, F16>(g, out, quad, o4, l);
        else
          *reinterpret_cast<f32x4*>(g.part_o + part * D + 4 * quad) = o4;
      }
    if (g.splits > 1 && hh == 0) {
      g.part_ml[2 * part] = acc[x].m;
      g.part_ml[2 * part + 1] = l;
    }
  }
}

// ============================================================ joining the splits
// Splits in ascending order, so that the sums do not depend on which finished first.  A workgroup has 256 / (D / 4)
// columns, four features of one a thread; reads of all splits are under way at once (one after the other they took 20 us
// for 25 splits).
constexpr int kMaxSplits = 32;

template <int D, bool F16>
__global__ __launch_bounds__(256) void k_paged_attn_join(Args g, int width) {
  constexpr int kColumns = 256 / (D / 4);
  __shared__ float2 ml[kMaxSplits][kColumns];
  Tile t;
  if (!find_tile(g, blockIdx.x / g.kv_heads, blockIdx.x % g.kv_heads, width, t)) return;
  const int c0 = t.col0 + blockIdx.y * kColumns, n = min(min(kColumns, t.col0 + width - c0), t.cols - c0);
  if (n <= 0) return;
  const int64_t stride = int64_t(g.a.n_rows) * g.a.heads;
  for (int x = threadIdx.x; x < g.splits * kColumns; x += 256) {
    const int s = x / kColumns, cc = x % kColumns;
    if (cc < n) ml[s][cc] = reinterpret_cast<const float2*>(g.part_ml)[s * stride + out_row(g, t, c0 + cc)];
  }
  __syncthreads();
  const int cc = threadIdx.x / (D / 4), quad = threadIdx.x % (D / 4);
  if (cc >= n) return;
  const int64_t out = out_row(g, t, c0 + cc);
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < g.splits; ++s) m = fmaxf(m, ml[s][cc].x);
  f32x4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = 0; s < g.splits; ++s) {
    const float2 p = ml[s][cc];
    const float f = p.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((p.x - m) * g.a.scale_log2);
    l += f * p.y;
    o += f * *reinterpret_cast<const f32x4*>(g.part_o + (s * stride + out) * D + 4 * quad);
  }
  store4<D, F16>(g, out, quad, o, l);
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
  // keys that a row sees, at most
  const int64_t keys = a.window ? std::min<int64_t>(a.max_len, int64_t(a.window) + (a.causal ? 0 : a.max_new)) : a.max_len;
  // Two column tiles a wave for many columns: half the LDS reads, but the last tile of 256 and the keys of a causal one,
  // whose rows end 256 / group keys apart, waste more. us for QT = 1 and 2, 62 sequences of 1701 with 8 heads of 64: 257
  // columns 89 and 126, 500 129 and 138, 900 212 and 223, 1701 278 and 288, not causal 436 and 413; 62 of 1100, all their
  // rows, 145 and 162, 10 of them 32 and 44; 8 of 8000, 2048 columns 270 and 250; 246 of 430, 412 rows of groups of 8 heads
  // 265 and 247.
  const bool two = most > 1024 && (!a.causal || keys * group > 2048);
  p.qt = most <= kCols ? 0 : s.head_dim == 128 || !two ? 1 : 2;
  p.width = p.qt ? kWaves * kCols * p.qt : kCols;
  p.search = most > p.width;
  p.tiles = p.search ? int(int64_t(a.n_rows) * group / p.width) + a.n_requests : a.n_requests;
  const int64_t blocks = int64_t(p.tiles) * s.kv_heads, want = int64_t(device_cu_count()) * 2;
  // A part has at least 256 of the keys that a tile's rows see, of many columns 128 up to one workgroup a CU: they have a
  // longer way per key, but more partial sums to write (us at 256, 128 and this: one of 700 keys, 300 rows, 16 and 4 heads
  // of 128 25, 18 and 18; four of them 27, 32 and 27; one of 1000 rows and keys, 8 heads of 64 14.3, 16.4 and 14.3).
  const int64_t seen = std::min<int64_t>(a.max_len, keys + p.width / group);
  int64_t parts = std::min(want / blocks, seen / 256);
  if (p.qt) parts = std::max(parts, std::min(want / 2 / blocks, seen / 128));
  p.splits = int(std::min<int64_t>(parts, kMaxSplits));
  if (p.splits < 3) p.splits = 1;
  // Requests by length where it matters: beyond some rounds of two workgroups a CU the last one is a small part of all.
  if (p.search && a.n_requests > 1 && a.n_requests <= 64 && blocks < 6 * want) p.search = 2;
  return p;
}

}  // namespace

// No more for a causal call or one with a window than without.
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
  constexpr int columns = 256 / (D / 4);
  if (p.splits > 1)
    k_paged_attn_join<D, F16><<<dim3(grid.x, (p.width + columns - 1) / columns), 256, 0, st>>>(g, p.width);
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
