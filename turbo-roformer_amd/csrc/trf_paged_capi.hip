// C ABI of the paged K/V cache (declared in include/trf_hip.h): argument checks.  Host code only; the kernels live in
// trf_pages.hip and trf_paged_attn.hip.
#include <math.h>

#include "trf_hip.h"
#include "trf_internal.h"

using trf::set_error;

namespace {

int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(TRF_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
  return TRF_OK;
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

#define TRF_REQUIRE_AT(ptr, name, al)                                                              \
  do {                                                                                             \
    if (!(ptr)) return set_error(TRF_ERR_ARG, "%s must not be NULL", name);                        \
    if (!aligned((ptr), al)) return set_error(TRF_ERR_ARG, "%s must be %d-byte aligned", name, al); \
  } while (0)

#define TRF_TRY(expr)                 \
  do {                                \
    if (int rc_ = (expr)) return rc_; \
  } while (0)

// log2 of a page size, or -1.
int page_shift(int32_t page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

int check_pages(int32_t n_pages, int32_t page_size) {
  if (page_shift(page_size) < 0)
    return set_error(TRF_ERR_ARG, "page_size must be 16, 32, 64, 128 or 256, got %d", page_size);
  if (n_pages < 1 || int64_t(n_pages) * page_size >= int64_t(1) << 31)
    return set_error(TRF_ERR_ARG, "n_pages must be >= 1 and n_pages * page_size below 2^31 (got %d pages of %d)", n_pages,
                     page_size);
  return TRF_OK;
}

int check_table(int32_t n_requests, int32_t max_pages, int32_t page_size) {
  if (n_requests < 1 || max_pages < 1 || int64_t(n_requests) * max_pages >= int64_t(1) << 31 ||
      int64_t(max_pages) * page_size > int64_t(1) << 30)
    return set_error(TRF_ERR_ARG,
                     "n_requests and max_pages must be >= 1, n_requests * max_pages below 2^31 and max_pages * page_size "
                     "at most 2^30 (got %d requests, %d pages of %d)", n_requests, max_pages, page_size);
  return TRF_OK;
}

int check_cache(int32_t dtype, int32_t n_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim,
                trf::PagedShape& s) {
  if (dtype != TRF_BF16 && dtype != TRF_F16) return set_error(TRF_ERR_ARG, "dtype must be 1 (bf16) or 2 (fp16), got %d", dtype);
  TRF_TRY(check_pages(n_pages, page_size));
  if (head_dim != 64 && head_dim != 128) return set_error(TRF_ERR_ARG, "head_dim must be 64 or 128, got %d", head_dim);
  if (kv_heads < 1 || kv_heads > 65535) return set_error(TRF_ERR_ARG, "kv_heads must be 1..65535, got %d", kv_heads);
  s = trf::PagedShape{n_pages, page_shift(page_size), kv_heads, head_dim, dtype == TRF_F16};
  return TRF_OK;
}

int check_rows(const char* name, const void* p, int64_t stride, int32_t heads, int32_t head_dim) {
  if (!p) return set_error(TRF_ERR_ARG, "%s must not be NULL", name);
  if (!aligned(p, 16) || stride % 8)
    return set_error(TRF_ERR_ARG, "%s must be 16-byte aligned, its row stride a multiple of 8 elements (got %lld)", name,
                     (long long)stride);
  if (stride < int64_t(heads) * head_dim)
    return set_error(TRF_ERR_ARG, "%s's rows are %lld elements apart, fewer than %d heads of %d", name, (long long)stride,
                     heads, head_dim);
  return TRF_OK;
}

// Rows out [n_rows][row] beside rows q: in the same place, if both lie alike, or apart.
int check_rows_out(const char* name, const void* out, const void* q, int64_t q_stride, int32_t n_rows, int64_t row) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(q), b = reinterpret_cast<uintptr_t>(out);
  const bool apart = b + uintptr_t(n_rows * row * 2) <= a || a + uintptr_t(((n_rows - 1) * q_stride + row) * 2) <= b;
  if (!apart && !(a == b && q_stride == row))
    return set_error(TRF_ERR_ARG, "%s must not overlap q, unless it is q with rows of heads * head_dim elements", name);
  return TRF_OK;
}

int check_state(const int32_t* state, const int32_t* state_out, int32_t n_requests) {
  TRF_REQUIRE_AT(state, "state", 4);
  TRF_REQUIRE_AT(state_out, "state_out", 4);
  const int64_t d = state_out - state, n = 2 + int64_t(n_requests);
  if (d > -n && d < n) return set_error(TRF_ERR_ARG, "state_out must not overlap state");
  return TRF_OK;
}

hipStream_t as_hip(trf_stream_t s) { return reinterpret_cast<hipStream_t>(s); }

}  // namespace

extern "C" {

int trf_page_plan(const int32_t* state, const int32_t* n_new, int32_t n_requests, int32_t n_rows, const int32_t* pool,
                  int32_t n_pages, int32_t page_size, int32_t* table, int32_t max_pages, int32_t* state_out,
                  int32_t* starts, int32_t* slots, int32_t* positions, trf_stream_t stream) {
  TRF_TRY(check_pages(n_pages, page_size));
  TRF_TRY(check_table(n_requests, max_pages, page_size));
  return trf_page_plan_limited(state, n_new, n_requests, n_rows, pool, n_pages, page_size, table, max_pages,
                               max_pages * page_size, state_out, starts, slots, positions, stream);
}

int trf_page_plan_limited(const int32_t* state, const int32_t* n_new, int32_t n_requests, int32_t n_rows,
                          const int32_t* pool, int32_t n_pages, int32_t page_size, int32_t* table, int32_t max_pages,
                          int32_t max_length, int32_t* state_out, int32_t* starts, int32_t* slots, int32_t* positions,
                          trf_stream_t stream) {
  TRF_TRY(check_pages(n_pages, page_size));
  TRF_TRY(check_table(n_requests, max_pages, page_size));
  if (max_length < 1 || max_length > max_pages * page_size)
    return set_error(TRF_ERR_ARG, "max_length must be 1..%d, got %d", max_pages * page_size, max_length);
  if (n_requests > trf::kPageRequests)
    return set_error(TRF_ERR_ARG, "n_requests must be at most %d, got %d", trf::kPageRequests, n_requests);
  if (n_rows < 0 || n_rows >= 1 << 30) return set_error(TRF_ERR_ARG, "n_rows must be 0..2^30 - 1, got %d", n_rows);
  TRF_TRY(check_state(state, state_out, n_requests));
  TRF_REQUIRE_AT(n_new, "n_new", 4);
  TRF_REQUIRE_AT(pool, "pool", 4);
  TRF_REQUIRE_AT(table, "table", 4);
  TRF_REQUIRE_AT(starts, "starts", 4);
  if (n_rows > 0) {
    TRF_REQUIRE_AT(slots, "slots", 4);
    TRF_REQUIRE_AT(positions, "positions", 4);
  }
  const trf::PagePlan p{n_requests, n_rows, n_pages, page_shift(page_size), max_pages, max_length};
  trf::launch_page_plan(p, state, n_new, pool, table, state_out, starts, slots, positions, as_hip(stream));
  return check_launch("page_plan");
}

int trf_page_release(const int32_t* state, const uint8_t* done, int32_t n_requests, int32_t* pool, int32_t n_pages,
                     int32_t page_size, const int32_t* table, int32_t max_pages, int32_t* state_out, trf_stream_t stream) {
  TRF_TRY(check_pages(n_pages, page_size));
  TRF_TRY(check_table(n_requests, max_pages, page_size));
  if (n_requests > trf::kPageRequests)
    return set_error(TRF_ERR_ARG, "n_requests must be at most %d, got %d", trf::kPageRequests, n_requests);
  TRF_TRY(check_state(state, state_out, n_requests));
  TRF_REQUIRE_AT(done, "done", 1);
  TRF_REQUIRE_AT(pool, "pool", 4);
  TRF_REQUIRE_AT(table, "table", 4);
  const trf::PagePlan p{n_requests, 0, n_pages, page_shift(page_size), max_pages, max_pages * page_size};
  trf::launch_page_release(p, state, done, pool, table, state_out, as_hip(stream));
  return check_launch("page_release");
}

int trf_paged_append(const uint16_t* q, int64_t q_stride, int32_t heads, const uint16_t* k, int64_t k_stride,
                     const uint16_t* v, int64_t v_stride, int32_t dtype, int32_t n_rows, const int32_t* slots,
                     const int32_t* positions, const float* rope, int32_t rope_len, uint16_t* K, uint16_t* V,
                     int32_t n_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim, uint16_t* q_out,
                     trf_stream_t stream) {
  trf::PagedShape s{};
  TRF_TRY(check_cache(dtype, n_pages, page_size, kv_heads, head_dim, s));
  if (q && (heads < 1 || heads > 65535)) return set_error(TRF_ERR_ARG, "heads must be 1..65535, got %d", heads);
  // a workgroup of 256 threads per 16 rows and head, and 32 bits for a launch's threads
  if (n_rows < 0 || (int64_t(n_rows) + 15) / 16 * (kv_heads + (q ? heads : 0)) >= int64_t(1) << 24)
    return set_error(TRF_ERR_ARG, "n_rows must be >= 0 and n_rows, up to the next 16, * (heads + kv_heads) below 2^28, got %d",
                     n_rows);
  if (rope && rope_len < 1) return set_error(TRF_ERR_ARG, "rope_len must be >= 1, got %d", rope_len);
  if (n_rows == 0) return TRF_OK;
  TRF_TRY(check_rows("k", k, k_stride, kv_heads, head_dim));
  TRF_TRY(check_rows("v", v, v_stride, kv_heads, head_dim));
  TRF_REQUIRE_AT(slots, "slots", 4);
  if (rope) {
    TRF_REQUIRE_AT(rope, "rope", 16);
    TRF_REQUIRE_AT(positions, "positions", 4);
  }
  TRF_REQUIRE_AT(K, "K", 16);
  TRF_REQUIRE_AT(V, "V", 16);
  if (q) {
    TRF_TRY(check_rows("q", q, q_stride, heads, head_dim));
    TRF_REQUIRE_AT(q_out, "q_out", 16);
    TRF_TRY(check_rows_out("q_out", q_out, q, q_stride, n_rows, int64_t(heads) * head_dim));
  }
  trf::launch_paged_append(s, q, q_stride, heads, k, k_stride, v, v_stride, K, V, slots, positions, n_rows, rope, rope_len,
                           q_out, as_hip(stream));
  return check_launch("paged_append");
}

static int attention_args(int32_t heads, int32_t dtype, int32_t n_pages, int32_t page_size, int32_t kv_heads,
                          int32_t head_dim, int32_t max_pages, int32_t n_requests, int32_t n_rows, int32_t max_new,
                          int32_t max_len, trf::PagedShape& s, trf::PagedAttnArgs& a) {
  TRF_TRY(check_cache(dtype, n_pages, page_size, kv_heads, head_dim, s));
  TRF_TRY(check_table(n_requests, max_pages, page_size));
  if (heads < 1 || heads > 65535 || heads % kv_heads)
    return set_error(TRF_ERR_ARG, "heads must be a multiple of kv_heads = %d, at most 65535, got %d", kv_heads, heads);
  if (n_rows < 0 || int64_t(n_rows) * heads >= int64_t(1) << 31)
    return set_error(TRF_ERR_ARG, "n_rows must be >= 0 and n_rows * heads below 2^31, got %d", n_rows);
  if (max_new < 0 || max_len < 0) return set_error(TRF_ERR_ARG, "max_new and max_len must be >= 0, got %d and %d", max_new, max_len);
  // a workgroup of 256 threads per column tile and K/V head, and 32 bits for a launch's threads
  if ((int64_t(n_rows) * (heads / kv_heads) / 32 + n_requests) * kv_heads >= int64_t(1) << 24)
    return set_error(TRF_ERR_ARG, "too many rows, requests and heads for one call");
  a.heads = heads;
  a.max_pages = max_pages;
  a.n_requests = n_requests;
  a.n_rows = n_rows;
  a.max_new = max_new < n_rows ? max_new : n_rows;
  a.max_len = max_len < max_pages * page_size ? max_len : max_pages * page_size;
  return TRF_OK;
}

size_t trf_paged_attention_workspace_bytes(int32_t heads, int32_t dtype, int32_t n_pages, int32_t page_size,
                                           int32_t kv_heads, int32_t head_dim, int32_t max_pages, int32_t n_requests,
                                           int32_t n_rows, int32_t max_new, int32_t max_len) {
  trf::PagedShape s{};
  trf::PagedAttnArgs a{};
  if (attention_args(heads, dtype, n_pages, page_size, kv_heads, head_dim, max_pages, n_requests, n_rows, max_new, max_len,
                     s, a))
    return 0;
  return trf::paged_attention_workspace(s, a);
}

int trf_paged_attention(const uint16_t* q, int64_t q_stride, int32_t heads, const uint16_t* K, const uint16_t* V,
                        int32_t dtype, int32_t n_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim,
                        const int32_t* table, int32_t max_pages, const int32_t* starts, const int32_t* lens,
                        int32_t n_requests, int32_t n_rows, int32_t max_new, int32_t max_len, float scale, int32_t causal,
                        int32_t window, const float* gate, uint16_t* O, void* workspace, size_t workspace_bytes,
                        trf_stream_t stream) {
  trf::PagedShape s{};
  trf::PagedAttnArgs a{};
  TRF_TRY(attention_args(heads, dtype, n_pages, page_size, kv_heads, head_dim, max_pages, n_requests, n_rows, max_new,
                         max_len, s, a));
  if (!(scale > 0.f) || !(scale < 1e30f)) return set_error(TRF_ERR_ARG, "scale must be positive and finite, got %g", double(scale));
  if (causal != 0 && causal != 1) return set_error(TRF_ERR_ARG, "causal must be 0 or 1, got %d", causal);
  if (window < 0) return set_error(TRF_ERR_ARG, "window must be 0 (none) or positive, got %d", window);
  if (n_rows == 0 || max_new == 0) return TRF_OK;
  TRF_TRY(check_rows("q", q, q_stride, heads, head_dim));
  TRF_REQUIRE_AT(K, "K", 16);
  TRF_REQUIRE_AT(V, "V", 16);
  TRF_REQUIRE_AT(table, "table", 4);
  TRF_REQUIRE_AT(starts, "starts", 4);
  TRF_REQUIRE_AT(lens, "lens", 4);
  if (gate) TRF_REQUIRE_AT(gate, "gate", 4);
  TRF_REQUIRE_AT(O, "O", 16);
  TRF_TRY(check_rows_out("O", O, q, q_stride, n_rows, int64_t(heads) * head_dim));
  a.causal = causal;
  a.window = window;
  const size_t need = trf::paged_attention_workspace(s, a);
  if (need) {
    if (!workspace || workspace_bytes < need)
      return set_error(TRF_ERR_WORKSPACE, "workspace is %zu bytes, need %zu", workspace ? workspace_bytes : size_t(0), need);
    TRF_REQUIRE_AT(workspace, "workspace", 16);
  }
  a.q = q, a.K = K, a.V = V, a.table = table, a.starts = starts, a.lens = lens, a.gate = gate, a.o = O;
  a.q_stride = q_stride;
  a.scale_log2 = scale * 1.44269504088896341f;
  trf::launch_paged_attention(s, a, workspace, as_hip(stream));
  return check_launch("paged_attention");
}

}  // extern "C"
