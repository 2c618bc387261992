// The C ABI of the paged cache (include/sa.h): argument checks and dispatch; the tables' and the cache write's
// kernels (the attention's are in sa_paged_bf16.hip, sa_paged_f16.hip and sa_paged_f32.hip).

#include <math.h>

#include "sa_paged.h"

using namespace sa_host;

namespace {

constexpr int64_t MAX_TOKENS = (int64_t)1 << 24, MAX_LEN = (int64_t)1 << 30;
constexpr int64_t GRID_THREADS = ((int64_t)1 << 32) - NTHREADS;   // threads of a launch's first dimension

// log2 of a page size, -1 if it is none: a power of two from 8 on
int page_shift(int64_t page_size) {
  if (page_size < 8 || page_size > (1 << 20) || (page_size & (page_size - 1))) return -1;
  return __builtin_ctzll((unsigned long long)page_size);
}
bool head_dim_ok(int64_t d) { return d == 16 || d == 32 || d == 64 || d == 128; }
int64_t elem_size(int dtype) { return dtype == SA_DTYPE_F32 ? 4 : dtype == SA_DTYPE_BF16 || dtype == SA_DTYPE_F16 ? 2 : 0; }
bool batch_ok(int64_t requests, int64_t tokens) {
  return requests >= 1 && requests < 65536 && tokens >= 1 && tokens < MAX_TOKENS;
}
bool aligned(const void* p) { return p && (uintptr_t)p % 16 == 0; }
// element strides of (token, head) rows that are read in 16-byte pieces, 128 rows within a buffer resource's 2 GiB
bool rows_ok(const void* p, int64_t token, int64_t head, int64_t head_dim, int64_t es) {
  return aligned(p) && token >= head_dim && token < ((int64_t)1 << 31) / (128 * es) && head >= 0 && token * es % 16 == 0 &&
         head * es % 16 == 0;
}

template <class S, class P>
void append(const AppendCall& c, int64_t head_dim, hipStream_t st) {
  const int64_t chunks = (int64_t)c.N * c.H * (head_dim / P::EPC);
  const dim3 grid((unsigned)cdiv(chunks, NTHREADS)), block(NTHREADS);
  if (head_dim == 16) hipLaunchKernelGGL((paged_append_kernel<S, P, 16>), grid, block, 0, st, c);
  else if (head_dim == 32) hipLaunchKernelGGL((paged_append_kernel<S, P, 32>), grid, block, 0, st, c);
  else if (head_dim == 64) hipLaunchKernelGGL((paged_append_kernel<S, P, 64>), grid, block, 0, st, c);
  else hipLaunchKernelGGL((paged_append_kernel<S, P, 128>), grid, block, 0, st, c);
}
template <class S>
void append_to(const AppendCall& c, int64_t head_dim, int dtype, hipStream_t st) {
  if (dtype == SA_DTYPE_BF16) append<S, PagedBF16>(c, head_dim, st);
  else if (dtype == SA_DTYPE_F16) append<S, PagedF16>(c, head_dim, st);
  else append<S, PagedF32>(c, head_dim, st);
}

}  // namespace

extern "C" {

int sa_page_plan(const int32_t* cached, const int32_t* new_tokens, const uint8_t* finished, int32_t* table, int64_t table_ld,
                 int32_t* free_pages, const int32_t* taken, int32_t* starts, int32_t* lengths, int32_t* cached_out,
                 int64_t* slots, int32_t* taken_out, int64_t requests, int64_t width, int64_t pool, int64_t tokens,
                 int64_t page_size, void* stream) {
  if (page_shift(page_size) < 0 || width < 1 || width > MAX_LEN / page_size) return SA_ERR_ARGUMENT;
  return sa_page_plan_within(cached, new_tokens, finished, table, table_ld, free_pages, taken, starts, lengths, cached_out, slots,
                             taken_out, requests, width, pool, tokens, page_size, std::max<int64_t>(tokens, 1), width * page_size,
                             stream);
}

int sa_page_plan_within(const int32_t* cached, const int32_t* new_tokens, const uint8_t* finished, int32_t* table, int64_t table_ld,
                        int32_t* free_pages, const int32_t* taken, int32_t* starts, int32_t* lengths, int32_t* cached_out,
                        int64_t* slots, int32_t* taken_out, int64_t requests, int64_t width, int64_t pool, int64_t tokens,
                        int64_t page_size, int64_t max_new, int64_t max_len, void* stream) {
  const int sh = page_shift(page_size);
  if (requests < 1 || requests >= 65536 || tokens < 0 || tokens >= MAX_TOKENS || sh < 0) return SA_ERR_ARGUMENT;
  if (width < 1 || table_ld < width || width > MAX_LEN / page_size || pool < 0 || pool > INT32_MAX) return SA_ERR_ARGUMENT;
  if (max_new < 1 || max_len < 1 || max_len > width * page_size) return SA_ERR_ARGUMENT;
  if (!cached || !new_tokens || !table || !taken || !starts || !lengths || !cached_out || !taken_out) return SA_ERR_ARGUMENT;
  if ((pool > 0 && !free_pages) || (tokens > 0 && !slots)) return SA_ERR_ARGUMENT;
  hipStream_t st = static_cast<hipStream_t>(stream);
  PlanCall c{};
  c.cached = cached;
  c.fresh = new_tokens;
  c.finished = finished;
  c.table = table;
  c.stack = free_pages;
  c.taken = taken;
  c.starts = starts;
  c.lengths = lengths;
  c.cached_out = cached_out;
  c.taken_out = taken_out;
  c.slots = slots;
  c.table_ld = table_ld;
  c.R = (int)requests;
  c.W = (int)width;
  c.F = (int)pool;
  c.N = (int)tokens;
  c.pshift = sh;
  c.max_new = (int)std::min(max_new, tokens);
  c.max_len = (int)max_len;
  c.slots_here = tokens <= PLAN_SLOTS;
  const int threads = (int)std::min<int64_t>(std::max<int64_t>(align_up(requests, 64), 256), PLAN_THREADS);
  hipLaunchKernelGGL(page_plan_kernel, dim3(1), dim3((unsigned)threads), 0, st, c);
  if (!c.slots_here)
    hipLaunchKernelGGL(page_slots_kernel, dim3((unsigned)cdiv(tokens, NTHREADS)), dim3(NTHREADS), 0, st, starts, lengths, table,
                       table_ld, slots, (int)requests, (int)width, (int)tokens, sh);
  return launch_status();
}

int sa_paged_append(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                    void* k_pages, void* v_pages, const int64_t* slots, int64_t tokens, int64_t heads, int64_t head_dim,
                    int64_t pages, int64_t page_size, int src_dtype, int dtype, void* stream) {
  const int sh = page_shift(page_size);
  const int64_t ss = elem_size(src_dtype), es = elem_size(dtype);
  if (!ss || !es) return SA_ERR_DTYPE;
  if (!head_dim_ok(head_dim)) return SA_ERR_HEAD_DIM;
  if (tokens < 0 || tokens >= MAX_TOKENS || heads < 1 || heads >= 65536 || pages < 1 || pages > INT32_MAX || sh < 0) return SA_ERR_ARGUMENT;
  if (tokens == 0) return SA_OK;
  if (!rows_ok(k, k_token, k_head, head_dim, ss) || !rows_ok(v, v_token, v_head, head_dim, ss) || !aligned(k_pages) ||
      !aligned(v_pages) || !slots)
    return SA_ERR_ARGUMENT;
  if (tokens * heads * (head_dim * es / 16) >= GRID_THREADS) return SA_ERR_ARGUMENT;
  AppendCall c{};
  c.k = k;
  c.v = v;
  c.k_pages = k_pages;
  c.v_pages = v_pages;
  c.slots = slots;
  c.k_token = k_token;
  c.k_head = k_head;
  c.v_token = v_token;
  c.v_head = v_head;
  c.total = pages << sh;
  c.N = (int)tokens;
  c.H = (int)heads;
  c.pshift = sh;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (src_dtype == SA_DTYPE_BF16) append_to<PagedBF16>(c, head_dim, dtype, st);
  else if (src_dtype == SA_DTYPE_F16) append_to<PagedF16>(c, head_dim, dtype, st);
  else append_to<PagedF32>(c, head_dim, dtype, st);
  return launch_status();
}

static bool paged_sizes_ok(int64_t requests, int64_t tokens, int64_t heads, int64_t groups, int64_t max_new, int64_t max_len) {
  return batch_ok(requests, tokens) && heads >= 1 && heads < 65536 && groups >= 1 && heads % groups == 0 && max_new >= 1 &&
         max_new <= tokens && max_len >= 1 && max_len < MAX_LEN && tokens * heads < ((int64_t)1 << 30) &&
         (requests * heads + requests * groups * cdiv(max_len, 4 * NTHREADS)) * NTHREADS < GRID_THREADS;
}

int64_t sa_paged_attention_workspace_bytes(int64_t requests, int64_t tokens, int64_t heads, int64_t groups, int64_t head_dim,
                                           int64_t max_new, int64_t max_len, int dtype) {
  const int64_t es = elem_size(dtype & ~SA_WIDE_WEIGHTS);
  if (!paged_sizes_ok(requests, tokens, heads, groups, max_new, max_len) || !head_dim_ok(head_dim) || !es) return -1;
  return paged_shape(requests, tokens, heads, groups, head_dim, es, max_new, max_len).total;
}

int sa_paged_attention(const void* q, int64_t q_token, int64_t q_head, const void* k_pages, const void* v_pages, void* out,
                       const int32_t* table, int64_t table_ld, const int32_t* lengths, const int32_t* starts, float* selected,
                       int64_t state_ld, void* workspace, int64_t workspace_bytes, int64_t requests, int64_t tokens,
                       int64_t heads, int64_t groups, int64_t head_dim, int64_t pages, int64_t page_size, int64_t width,
                       int64_t max_new, int64_t max_len, float scale, int dtype, int exempt, void* stream) {
  const int sh = page_shift(page_size);
  const bool wide = dtype & SA_WIDE_WEIGHTS;
  dtype &= ~SA_WIDE_WEIGHTS;
  const int64_t es = elem_size(dtype);
  if (!es) return SA_ERR_DTYPE;
  if (!head_dim_ok(head_dim)) return SA_ERR_HEAD_DIM;
  if (!paged_sizes_ok(requests, tokens, heads, groups, max_new, max_len) || sh < 0 || exempt < 1) return SA_ERR_ARGUMENT;
  if (pages < 1 || pages > INT32_MAX || width < 1 || table_ld < width || max_len > width * page_size || state_ld < max_len)
    return SA_ERR_ARGUMENT;
  if (!(scale > 0.f) || !(scale < INFINITY)) return SA_ERR_ARGUMENT;
  if (!rows_ok(q, q_token, q_head, head_dim, es) || !aligned(k_pages) || !aligned(v_pages) || !aligned(out) ||
      !table || !lengths || !starts || !selected)
    return SA_ERR_ARGUMENT;
  const int64_t need = sa_paged_attention_workspace_bytes(requests, tokens, heads, groups, head_dim, max_new, max_len, dtype);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need) return SA_ERR_WORKSPACE;
  PagedLaunch c{};
  c.q = q;
  c.k_pages = k_pages;
  c.v_pages = v_pages;
  c.out = out;
  c.table = table;
  c.lengths = lengths;
  c.starts = starts;
  c.selected = selected;
  c.q_token = q_token;
  c.q_head = q_head;
  c.table_ld = table_ld;
  c.state_ld = state_ld;
  c.ws = workspace;
  c.R = requests;
  c.N = tokens;
  c.H = heads;
  c.G = groups;
  c.pages = pages;
  c.max_new = max_new;
  c.max_len = max_len;
  c.pshift = sh;
  c.scale = scale;
  c.exempt = exempt;
  c.head_dim = (int)head_dim;
  c.wide = wide;
  c.st = static_cast<hipStream_t>(stream);
  return dtype == SA_DTYPE_BF16 ? paged_bf16(c) : dtype == SA_DTYPE_F16 ? paged_f16(c) : paged_f32(c);
}

}  // extern "C"
