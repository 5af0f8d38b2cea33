// Pages of the paged K/V cache on gfx950: dealing them to requests, taking them back, and the write of new K and V
// rows into them (the layouts are in trf_hip.h).
#include <algorithm>
#include <type_traits>

#include "trf_device.h"

namespace trf {

// ============================================================ prefix sums over the requests
// Every workgroup of a plan or a release forms the prefix sums over all requests itself: at most kPageRequests of
// them, read from L2, against a second launch or a wait between workgroups.  Thread t holds requests
// t * EACH .. t * EACH + EACH - 1 in registers.

// x of the lane that a DPP control names, 0 where there is none or the row is not in the mask.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_before(uint32_t x) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(x), CTRL, ROWS, 0xf, false));
}

// Inclusive prefix sum over the wave: within rows of 16 lanes, then of each row's last lane into the rows behind it.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x, uint32_t most) {
  x = min(x + lane_before<0x111, 0xf>(x), most);  // row_shr:1, 2, 4, 8
  x = min(x + lane_before<0x112, 0xf>(x), most);
  x = min(x + lane_before<0x114, 0xf>(x), most);
  x = min(x + lane_before<0x118, 0xf>(x), most);
  x = min(x + lane_before<0x142, 0xa>(x), most);  // row_bcast:15 into rows 1 and 3
  return min(x + lane_before<0x143, 0xc>(x), most);  // row_bcast:31 into rows 2 and 3
}

// Exclusive prefix sums of x and y over the workgroup's threads in thread order, and their totals.  Sums saturate at
// most_x and most_y (every term is at most that, and that at most 2^31 - 1), which is as associative as plain addition of
// whole numbers.  lds [2][THREADS / 64] is not used by anything else until the next barrier.
template <int THREADS>
__device__ __forceinline__ void block_scan(uint32_t& x, uint32_t& y, uint32_t most_x, uint32_t most_y, uint32_t* lds,
                                           uint32_t& total_x, uint32_t& total_y) {
  constexpr int W = THREADS / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t in_x = wave_scan(x, most_x), in_y = wave_scan(y, most_y);
  if (lane == 63) lds[wave] = in_x, lds[W + wave] = in_y;
  __syncthreads();
  uint32_t before_x = 0, before_y = 0;
  total_x = total_y = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w == wave) before_x = total_x, before_y = total_y;
    total_x = min(total_x + lds[w], most_x);
    total_y = min(total_y + lds[W + w], most_y);
  }
  x = min(before_x + lane_before<0x138, 0xf>(in_x), most_x);  // wave_shr:1
  y = min(before_y + lane_before<0x138, 0xf>(in_y), most_y);
}

// Last index r in [0, n) with a[r] <= v, for ascending a with a[0] <= v.
__device__ __forceinline__ int last_not_above(const uint32_t* a, int n, uint32_t v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int clamped_length(int len, const PagePlan& p) {
  return min(max(len, 0), p.max_pages << p.page_shift);
}

// ============================================================ plan
// One thread per new row: its request by binary search over the row starts in LDS, its page from the request's
// table row or, past the pages it has, from the pool; the row that opens a new page enters it in the table (a new
// page's first position is always a new row).  Bound by latency: a read of the lengths, two prefix sums, a search and
// a read of a page, one after the other.  Measured: 62 requests and rows 2.5 us, 4092 requests and 105,000 rows 9.4 (one
// sum after the other 3.0 and 10.8, and with the requests read again for each step 4.1 and 14.6; 512 threads of 8
// requests 13.2, 4 rows a thread 14.8).
template <int THREADS, int EACH>
__global__ __launch_bounds__(THREADS) void k_page_plan(PagePlan p, const int32_t* __restrict__ state,
                                                       const int32_t* __restrict__ n_new,
                                                       const int32_t* __restrict__ pool, int32_t* table,
                                                       int32_t* __restrict__ state_out, int32_t* __restrict__ starts,
                                                       int32_t* __restrict__ slots, int32_t* __restrict__ positions) {
  __shared__ uint32_t begin[THREADS * EACH];  // first row of each request
  __shared__ int2 request[THREADS * EACH];    // its length, and the pages dealt before it (-1: refused)
  __shared__ uint32_t sums[2][2 * THREADS / 64];
  __shared__ int32_t counts[2];               // pages dealt, requests refused
  const int R = p.n_requests, r0 = threadIdx.x * EACH, page = 1 << p.page_shift;
  const uint32_t beyond = uint32_t(p.n_rows) + 1;  // row sums end here
  if (threadIdx.x < 2) counts[threadIdx.x] = 0;
  uint32_t n[EACH], mine = 0;
  int len[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int r = min(r0 + e, R - 1);
    n[e] = r0 + e < R ? min(uint32_t(max(n_new[r], 0)), beyond) : 0;
    len[e] = clamped_length(state[2 + r], p);
  }
  const int free = min(max(state[0], 0), p.n_pages);
  // Pages are wanted by requests whose rows fit; that they all do is what both sums are formed on at once.
  uint32_t want[EACH], want_mine = 0;
  bool fits[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    fits[e] = r0 + e < R && int64_t(len[e]) + n[e] <= p.max_length;
    want[e] = fits[e] ? ((len[e] + n[e] + page - 1) >> p.page_shift) - ((len[e] + page - 1) >> p.page_shift) : 0;
    want_mine += want[e];
    mine = min(mine + n[e], beyond);
  }
  uint32_t row = mine, before = want_mine, rows, wanted;
  block_scan<THREADS>(row, before, beyond, 0x7fffffffu, sums[0], rows, wanted);
  uint32_t first[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    first[e] = row;
    row = min(row + n[e], beyond);
  }
  if (rows == beyond) {  // more rows than there is room for: once more, without the requests that do not fit
    want_mine = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      fits[e] &= first[e] + n[e] < beyond;
      if (!fits[e]) want[e] = 0;
      want_mine += want[e];
    }
    uint32_t none = 0;
    before = want_mine;
    block_scan<THREADS>(before, none, 0x7fffffffu, 0, sums[1], wanted, none);
  }
  int used = 0, refused = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int r = r0 + e;
    const bool ok = fits[e] && (want[e] == 0 || before + want[e] <= uint32_t(free));
    if (r < R) {
      begin[r] = first[e];
      request[r] = int2{len[e], ok ? int32_t(min(before, uint32_t(free))) : -1};
      if (blockIdx.x == 0) {
        starts[r] = min(first[e], uint32_t(p.n_rows));
        state_out[2 + r] = ok ? len[e] + n[e] : len[e];
      }
    }
    if (ok) used += want[e];
    refused += !ok && n[e] > 0;
    before += want[e];
  }
  if (blockIdx.x == 0) {
    if (used) atomicAdd(&counts[0], used);
    if (refused) atomicAdd(&counts[1], refused);
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    starts[R] = min(rows, uint32_t(p.n_rows));
    state_out[0] = free - counts[0];
    state_out[1] = counts[1];
  }
  for (int64_t i = int64_t(blockIdx.x) * THREADS + threadIdx.x; i < p.n_rows; i += int64_t(gridDim.x) * THREADS) {
    int pos = -1, slot = -1;
    if (uint32_t(i) < rows) {
      const int r = last_not_above(begin, R, uint32_t(i));
      const int2 q = request[r];
      if (q.y >= 0) {
        const int have = (q.x + page - 1) >> p.page_shift;
        pos = q.x + int(uint32_t(i) - begin[r]);
        const int at = pos >> p.page_shift;
        int32_t* entry = table + int64_t(r) * p.max_pages + at;
        const int pg = *(at < have ? entry : pool + (free - 1 - (q.y + at - have)));
        if (at >= have && (pos & (page - 1)) == 0) *entry = pg;
        if (uint32_t(pg) < uint32_t(p.n_pages)) slot = (pg << p.page_shift) + (pos & (page - 1));
      }
    }
    slots[i] = slot;
    positions[i] = pos;
  }
}

// Threads of a workgroup and requests of a thread: what holds them all (the fewer waves meet at a barrier the better).
template <class Run>
void by_requests(int32_t n, Run run) {
  using std::integral_constant;
  if (n <= 256)
    run(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (n <= 1024)
    run(integral_constant<int, 1024>{}, integral_constant<int, 1>{});
  else if (n <= 4096)
    run(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
  else
    run(integral_constant<int, 1024>{}, integral_constant<int, 8>{});
}
static_assert(kPageRequests <= 8 * 1024, "requests per thread");

void launch_page_plan(const PagePlan& p, const int32_t* state, const int32_t* n_new, const int32_t* pool,
                      int32_t* table, int32_t* state_out, int32_t* starts, int32_t* slots, int32_t* positions,
                      hipStream_t st) {
  by_requests(p.n_requests, [&](auto threads, auto each) {
    constexpr int T = decltype(threads)::value, E = decltype(each)::value;
    const int64_t blocks = (int64_t(p.n_rows) + T - 1) / T;
    const unsigned grid = unsigned(std::min<int64_t>(std::max<int64_t>(blocks, 1), 256));
    k_page_plan<T, E><<<grid, T, 0, st>>>(p, state, n_new, pool, table, state_out, starts, slots, positions);
  });
}

// ============================================================ release
// One thread per released page: its request by binary search over the prefix sums in LDS.  Measured: 62 of 124 requests
// 3.0 us, 1350 of 4092 with 346,000 pages 6.4.
template <int THREADS, int EACH>
__global__ __launch_bounds__(THREADS) void k_page_release(PagePlan p, const int32_t* __restrict__ state,
                                                          const uint8_t* __restrict__ done, int32_t* __restrict__ pool,
                                                          const int32_t* __restrict__ table,
                                                          int32_t* __restrict__ state_out) {
  __shared__ uint32_t before[THREADS * EACH];  // pages released before the request's
  __shared__ uint32_t sums[2 * THREADS / 64];
  const int R = p.n_requests, r0 = threadIdx.x * EACH, page = 1 << p.page_shift;
  const int free = min(max(state[0], 0), p.n_pages);
  uint32_t n[EACH], mine = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int r = min(r0 + e, R - 1), len = clamped_length(state[2 + r], p);
    const bool gone = done[r] != 0;
    n[e] = r0 + e < R && gone ? uint32_t(len + page - 1) >> p.page_shift : 0;
    if (blockIdx.x == 0 && r0 + e < R) state_out[2 + r] = gone ? 0 : len;
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) mine += n[e];
  uint32_t at = mine, none = 0, total;
  block_scan<THREADS>(at, none, 0x7fffffffu, 0, sums, total, none);
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (r0 + e < R) before[r0 + e] = at;
    at += n[e];
  }
  total = min(total, uint32_t(p.n_pages - free));
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    state_out[0] = free + int(total);
    state_out[1] = 0;
  }
  __syncthreads();
  for (uint32_t k = blockIdx.x * THREADS + threadIdx.x; k < total; k += gridDim.x * THREADS) {
    const int r = last_not_above(before, R, k);
    pool[free + k] = table[int64_t(r) * p.max_pages + (k - before[r])];
  }
}

void launch_page_release(const PagePlan& p, const int32_t* state, const uint8_t* done, int32_t* pool,
                         const int32_t* table, int32_t* state_out, hipStream_t st) {
  const int64_t most = std::min<int64_t>(int64_t(p.n_requests) * p.max_pages, p.n_pages);
  by_requests(p.n_requests, [&](auto threads, auto each) {
    constexpr int T = decltype(threads)::value, E = decltype(each)::value;
    const unsigned grid = unsigned(std::min<int64_t>((most + 2 * T - 1) / (2 * T), 256));
    k_page_release<T, E><<<grid, T, 0, st>>>(p, state, done, pool, table, state_out);
  });
}

// ============================================================ append
// Rows of k, v (and q) into the cache.  Memory wants a row's heads side by side where they come from, and 16 positions'
// chunks (K) or 8 positions' values (V) side by side where they go: a workgroup reads rows of 128 features of k and v,
// turns K on the way and lets both change direction in LDS.  It writes the 16-key groups whose first row of this call is
// one of its 16 rows, and for that reads up to 15 rows more: a group's lines are written whole, by one workgroup.  V goes
// out 16 bytes a feature, or in single values where the call does not fill an octet.  More features a workgroup leave
// fewer of them on a CU to cover the two waits of each (slots, then rows): us at 512, 256 and 128 features 247, 184 and
// 165 for the 17 s chunk, 92, 65 and 49 for the pieces.  Bound by HBM for many rows, where a large copy reaches 5.1 TB/s:
// 105,462 rows of 8 heads of 64 122 us (5.3 TB/s), 8,700 rows of 32 and 8 heads of 128 45 us (4.5 TB/s); 62 rows 4.8 us,
// latency.
constexpr int kAppendRows = 16, kAppendFeatures = 128;
constexpr int kMostRows = 2 * kAppendRows - 1;            // rows of the groups that a tile writes
constexpr int kKPad = kAppendFeatures / 8 + 1;            // 16-byte chunks of a K row in LDS

struct AppendArgs {
  const uint16_t *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements from row to row
  int32_t heads, kv_heads, n_rows, rope_len, slots, page_shift;
  const int32_t *slot, *position;
  const float* rope;
  uint16_t *q_out, *K, *V;
  int32_t heads_per, parts, kv_parts;  // heads of a workgroup; workgroups per tile, and those that write K and V (the others turn q)
};

// Row i's slot if it is written (a slot of the cache and, with a table, one of its positions), or -1.
__device__ __forceinline__ int live_slot(const AppendArgs& a, int i) {
  if (i < 0 || i >= a.n_rows) return -1;
  const int slot = a.slot[i];
  const bool live = uint32_t(slot) < uint32_t(a.slots) && (!a.rope || uint32_t(a.position[i]) < uint32_t(a.rope_len));
  return live ? slot : -1;
}

template <bool F16>
__device__ __forceinline__ u32x4 turn8(u32x4 x, const f32x4& c, const f32x4& s) {
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = x[i];  // a bit_cast of the vector's element itself takes element 0
    float a, b;
    if constexpr (F16) {
      const f16x2 v = __builtin_bit_cast(f16x2, w);
      a = float(v[0]), b = float(v[1]);
    } else {
      a = __uint_as_float(w << 16), b = __uint_as_float(w & 0xffff0000u);
    }
    const float ya = a * c[i] - b * s[i], yb = a * s[i] + b * c[i];
    y[i] = F16 ? pk_f16(ya, yb) : pk_bf16(ya, yb);
  }
  return y;
}

// The 8 features from chunk c of a head on, of a row at this position, turned by the table's angles.
template <int D, bool F16>
__device__ __forceinline__ u32x4 turned(const AppendArgs& a, u32x4 x, int position, int c) {
  if (!a.rope) return x;
  const float* t = a.rope + int64_t(position) * (D / 2) + 4 * c;
  return turn8<F16>(x, *reinterpret_cast<const f32x4*>(t),
                    *reinterpret_cast<const f32x4*>(t + int64_t(a.rope_len) * (D / 2)));
}

// What a large launch writes is more than the caches hold: non-temporal stores (165 and 160 us for the 17 s chunk, 49 and
// 47 for the pieces, without and with).
__device__ __forceinline__ void store_once(uint16_t* dst, const u32x4& x) {
  __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(dst));
}

template <int D, bool F16>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
  __shared__ u32x4 lds_k[kMostRows * kKPad];
  __shared__ u32x4 lds_v[kMostRows * kAppendFeatures / 8];
  __shared__ int2 rows[kMostRows];       // the rows that are written here, from row0 on, and their slots
  __shared__ int32_t octets[kMostRows];  // first of their rows in that list | their number << 8
  __shared__ int2 count;                 // rows and octets
  constexpr int kHead = D / 8;           // chunks of a head
  // A tile's parts run at the same time: its rows are read, and its groups written, in one go.  Workgroups are dealt to
  // the 8 XCDs in turn, and parts that write K and V move twice what the others do: the parts start one later in each tile
  // (150 and 122 us for the 17 s chunk).
  const int tile = blockIdx.x / a.parts, row0 = tile * kAppendRows, lane = threadIdx.x & 63;
  const int part = int((blockIdx.x + tile) % uint32_t(a.parts));
  const bool is_q = part >= a.kv_parts;
  const int h0 = (is_q ? part - a.kv_parts : part) * a.heads_per;
  const int nh = min(a.heads_per, (is_q ? a.heads : a.kv_heads) - h0), width = nh * kHead;  // chunks of a row
  if (is_q) {
    for (int x = threadIdx.x; x < kAppendRows * width; x += 256) {
      const int r = x / width, c = x - r * width;
      if (live_slot(a, row0 + r) < 0) continue;
      const int64_t i = row0 + r;
      const u32x4 y = *reinterpret_cast<const u32x4*>(a.q + i * a.q_stride + h0 * D + 8 * c);
      store_once(a.q_out + (i * a.heads + h0) * D + 8 * c, turned<D, F16>(a, y, a.rope ? a.position[i] : 0, c % kHead));
    }
    return;
  }
  if (threadIdx.x < 64) {
    // Lane l has row row0 - 1 + l, up to the last that a group of this tile can have.
    const int slot = lane <= kMostRows ? live_slot(a, row0 - 1 + lane) : -1, before = __shfl_up(slot, 1);
    // a row that continues the one before it in its group, or in its octet
    const bool cont = lane > 0 && slot >= 0 && (slot & 15) && before == slot - 1, cont8 = cont && (slot & 7);
    const uint64_t conts = __ballot(cont), conts8 = __ballot(cont8);
    const int leader = 63 - __builtin_clzll((~conts & ((2ull << lane) - 1)) | 1);
    const bool mine = slot >= 0 && leader >= 1 && leader <= kAppendRows;
    const uint64_t mines = __ballot(mine), first8 = __ballot(mine && !cont8), below = (1ull << lane) - 1;
    const int at = __popcll(mines & below);
    if (mine) rows[at] = int2{lane - 1, slot};
    if (mine && !cont8) octets[__popcll(first8 & below)] = at | (1 + __builtin_ctzll(~(conts8 >> lane >> 1))) << 8;
    if (lane == 0) count = int2{int(__popcll(mines)), int(__popcll(first8))};
  }
  __syncthreads();
  const int n_rows = count.x, n_octets = count.y;
  for (int x = threadIdx.x; x < n_rows * width; x += 256) {
    const int r = x / width, c = x - r * width;
    const int64_t i = row0 + rows[r].x;
    const u32x4 y = *reinterpret_cast<const u32x4*>(a.k + i * a.k_stride + h0 * D + 8 * c);
    lds_v[r * (kAppendFeatures / 8) + c] = *reinterpret_cast<const u32x4*>(a.v + i * a.v_stride + h0 * D + 8 * c);
    lds_k[r * kKPad + c] = turned<D, F16>(a, y, a.rope ? a.position[i] : 0, c % kHead);
  }
  __syncthreads();
  const int page_mask = (1 << a.page_shift) - 1;
  for (int x = threadIdx.x; x < n_rows * width; x += 256) {
    const int c = x / n_rows, r = x - c * n_rows, slot = rows[r].y, in = slot & page_mask;
    const int64_t head = int64_t(slot >> a.page_shift) * a.kv_heads + h0 + c / kHead;
    uint16_t* dst = a.K + (((head << a.page_shift) + (in & ~15)) * D + (c % kHead) * 128 + (in & 15) * 8);
    store_once(dst, lds_k[r * kKPad + c]);
  }
  const uint16_t* V = reinterpret_cast<const uint16_t*>(lds_v);
  for (int x = threadIdx.x; x < n_octets * nh * D; x += 256) {
    const int o = octets[x / (nh * D)], f = x % (nh * D), r = o & 255, n = o >> 8;
    const int slot = rows[r].y, in = slot & page_mask;
    const int64_t head = int64_t(slot >> a.page_shift) * a.kv_heads + h0 + f / D;
    uint16_t* dst = a.V + (((head << a.page_shift) + (in & ~7)) * D + (f % D) * 8);
    if (n == 8) {
      u32x4 y;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        y[k] = uint32_t(V[(r + 2 * k) * kAppendFeatures + f]) | uint32_t(V[(r + 2 * k + 1) * kAppendFeatures + f]) << 16;
      store_once(dst, y);
    } else {
      for (int k = 0; k < n; ++k) dst[(in & 7) + k] = V[(r + k) * kAppendFeatures + f];
    }
  }
}

void launch_paged_append(const PagedShape& s, const uint16_t* q, int64_t q_stride, int heads, const uint16_t* k,
                         int64_t k_stride, const uint16_t* v, int64_t v_stride, uint16_t* K, uint16_t* V,
                         const int32_t* slots, const int32_t* positions, int32_t n_rows, const float* rope,
                         int32_t rope_len, uint16_t* q_out, hipStream_t st) {
  AppendArgs a{};
  a.q = q, a.k = k, a.v = v;
  a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
  a.heads = q ? heads : 0, a.kv_heads = s.kv_heads, a.n_rows = n_rows, a.rope_len = rope_len;
  a.slots = s.n_pages << s.page_shift, a.page_shift = s.page_shift;
  a.slot = slots, a.position = positions, a.rope = rope;
  a.q_out = q_out, a.K = K, a.V = V;
  // Heads of a workgroup: as many as its tile holds, fewer while there are fewer than two workgroups per CU.
  const int tiles = (n_rows + kAppendRows - 1) / kAppendRows;
  a.heads_per = kAppendFeatures / s.head_dim;
  auto parts = [&](int n) { return (n + a.heads_per - 1) / a.heads_per; };
  while (a.heads_per > 1 && int64_t(tiles) * (parts(a.kv_heads) + parts(a.heads)) < 2 * device_cu_count()) a.heads_per /= 2;
  a.kv_parts = parts(a.kv_heads);
  a.parts = a.kv_parts + parts(a.heads);
  auto kernel = s.head_dim == 64 ? (s.f16 ? k_paged_append<64, true> : k_paged_append<64, false>)
                                 : (s.f16 ? k_paged_append<128, true> : k_paged_append<128, false>);
  kernel<<<unsigned(int64_t(tiles) * a.parts), 256, 0, st>>>(a);
}

}  // namespace trf
