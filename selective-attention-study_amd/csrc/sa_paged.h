// Selective Attention over a paged cache (gfx950): the step's tables, the cache write, and the attention of a
// ragged batch of new tokens over pages.
//
// A cache is k_pages, v_pages (pages, H, P, D): a page holds P consecutive positions of one request, every head's
// rows together, so that one head's keys of a page are P D contiguous elements. A request's positions are found
// through its table row: position j in page table[r][j / P], row j % P. The per-key selection state belongs to the
// request, not to the page (it depends on the request's own queries): (R, G, L) fp32 rows.
//
// Per request with c cached and n new tokens, t = c + n (operator: sa_kernels.h):
//   F[i, j] = state[j] (j < c, else 0) + sum over the chunk's queries r < i of relu(s q_sel[r].k_sel[j]),
//             exempt <= j < c + r;    out_h = softmax_j(s q_h.k_h - F) V_h;    state[j] = F after the last query
//
// Kernels:
//   page_plan, page_slots   the step's tables from the requests' lengths
//   paged_append            new rows into the pages
//   paged_carry             n > 1: each selector's history on entry to every 32-query tile, and the new state
//   paged_carry_join        the same where the queries are walked in segments: the segments' histories joined
//   paged_fwd, paged_fwd4   n > 1: a wavefront's 32 queries of one or two heads over the key tiles, or a part of them
//   paged_join              the parts of a query joined
//   paged_step, paged_step_join    n = 1: the cache read once in fp32 arithmetic, split over workgroups

#pragma once

#include "sa_kernels.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Cache element types: 16-byte chunks of a row are the unit that loads, LDS and the matrix operands share. mma
// contracts one chunk per lane (lanes 0-31 the even, lanes 32-63 the odd chunk of their row): one bf16 or fp16
// instruction, or four fp32 ones that take element e of both halves' chunks (the order of a contraction is free as
// long as both operands have the same).
//
// Softmax weights are taken 2^LIFT times their size beside the row's reference (the factor cancels in the normalisation): an
// fp16 number below 2^-14 has no more than its last bits, one below 2^-25 none, and a row's many small weights together
// may be what its output is made of. At 2^10 a weight keeps half a step of fp16 down to 2^-24 of the largest, and is off by 2^-35 of
// that at most below it: t keys by t 2^-35, half a step of an output at 2^24 of them.
struct PagedBF16 {
  typedef uint16_t elem;
  static constexpr int EPC = 8;
  static constexpr float LIFT = 0.f, BIG = 16384.f;   // (BIG: paged_fwd4_kernel)
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u32x4 pack(const f32x16& x, int s) {   // round to nearest even
    bf16x8 f;
#pragma unroll
    for (int t = 0; t < 8; ++t) f[t] = (bf16_t)x[8 * s + t];
    return __builtin_bit_cast(u32x4, f);
  }
  // what pack has rounded away, rounded in its turn (hi: pack's result): a weight as the sum of the two is off by 2^-16 of itself
  static __device__ __forceinline__ u32x4 rest(const f32x16& x, u32x4 hi, int s) {
    const bf16x8 h = __builtin_bit_cast(bf16x8, hi);
    bf16x8 f;
#pragma unroll
    for (int t = 0; t < 8; ++t) f[t] = (bf16_t)(x[8 * s + t] - (float)h[t]);
    return __builtin_bit_cast(u32x4, f);
  }
  static __device__ __forceinline__ float to_float(elem x) { return __uint_as_float((uint32_t)x << 16); }
  static __device__ __forceinline__ elem to_elem(float x) { return __builtin_bit_cast(elem, (bf16_t)x); }
};
struct PagedF16 {
  typedef uint16_t elem;
  static constexpr int EPC = 8;
  static constexpr float LIFT = 10.f, BIG = 32768.f;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u32x4 pack(const f32x16& x, int s) {
    f16x8 f;
#pragma unroll
    for (int t = 0; t < 8; ++t) f[t] = (_Float16)x[8 * s + t];
    return __builtin_bit_cast(u32x4, f);
  }
  // (off by 2^-22 of the weight, or 2^-25 LIFTed)
  static __device__ __forceinline__ u32x4 rest(const f32x16& x, u32x4 hi, int s) {
    const f16x8 h = __builtin_bit_cast(f16x8, hi);
    f16x8 f;
#pragma unroll
    for (int t = 0; t < 8; ++t) f[t] = (_Float16)(x[8 * s + t] - (float)h[t]);
    return __builtin_bit_cast(u32x4, f);
  }
  static __device__ __forceinline__ float to_float(elem x) { return (float)__builtin_bit_cast(_Float16, x); }
  static __device__ __forceinline__ elem to_elem(float x) { return __builtin_bit_cast(elem, (_Float16)x); }
};
struct PagedF32 {
  typedef float elem;
  static constexpr int EPC = 4;
  static constexpr float LIFT = 0.f;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ float to_float(elem x) { return x; }
  static __device__ __forceinline__ elem to_elem(float x) { return x; }
};

// ---------------------------------------------------------------------------------------------
// Requests of a ragged batch. Tiles of 1 << sh query rows are numbered without a table of their own: request r's
// tiles take the numbers from (starts[r] >> sh) + r on, as many as it can need (a request of n rows covers at most
// ((starts[r] + n) >> sh) - (starts[r] >> sh) + 1 tiles), so N rows of R requests have (N >> sh) + R numbers.
//
// The request that holds number x (ROWS: that holds row x): the last r with first(r) <= x. All 64 lanes probe at once, 64-fold narrower each
// round: one round of loads up to 64 requests, two up to 4096. Called by whole wavefronts; any contents of `starts`
// give an r in [0, R).
template <bool ROWS>
__device__ __forceinline__ int find_request(const int* starts, int R, int x, int sh) {
  const int lane = threadIdx.x & 63;
  int base = 0, n = R;
  while (n > 1) {
    const int stride = (n + 63) >> 6;
    const int i = lane * stride;
    bool at = false;
    if (i < n) {
      const int s = starts[base + i];
      at = ROWS ? s <= x : (s >> sh) + base + i <= x;
    }
    const int hit = max(__popcll(__ballot(at)), 1) - 1;
    base += hit * stride;
    n = min(stride, n - hit * stride);
    if (stride == 1) break;
  }
  return __builtin_amdgcn_readfirstlane(min(base, R - 1));
}

struct PagedCall {
  const void *q, *k_pages, *v_pages;
  void* out;
  const int *table, *lengths, *starts;
  float* selected;
  int64_t q_token, q_head, table_ld, state_ld;
  int R, N, H, G, pages, pshift;
  int max_new, max_len;
  float* totals;   // (R, G, segments, ld) what each segment of query tiles adds to the histories; of the first, with the state
  int segments, seg_tiles;   // of query tiles, whose histories are made independently (seg_tiles a multiple of four)
  int ones;   // several tokens: requests with one new token are left to the single-token kernels
  float *least, *kn;   // per key tile: least history on entry to a query tile, largest key norm; NULL: every tile is computed
  int64_t reach_ld;
  float scale;
  int exempt;
};

// One request's step: n new rows from token `first` on, c cached positions, t = c + n. A request that cannot be
// served is left out (live = false): fewer positions than new rows, more than the table row, the state row or the
// caller's bound holds, rows outside the batch, more new rows than the bound.
struct PagedRequest {
  int first, n, c, t;
  bool live;
};
__device__ __forceinline__ PagedRequest paged_request(const PagedCall& a, int r) {
  PagedRequest q;
  q.first = __builtin_amdgcn_readfirstlane(a.starts[r]);
  const int end = __builtin_amdgcn_readfirstlane(a.starts[r + 1]);
  q.t = __builtin_amdgcn_readfirstlane(a.lengths[r]);
  const bool rows = q.first >= 0 && end > q.first && end <= a.N;
  q.n = rows ? end - q.first : 0;
  q.c = q.t - q.n;
  q.live = rows && q.t >= q.n && q.t <= a.max_len && q.n <= a.max_new;   // (max_len: within the table and state rows)
  return q;
}

struct PagedTiles {   // what a workgroup of query tiles has to do
  PagedRequest rq;
  int r, row0;        // request, its first row
  int kt_hi;          // the key tiles that one of its rows sees
};

static __device__ uint4 paged_zero_row;   // what rows without a page read

// ---------------------------------------------------------------------------------------------
// The step's tables. One workgroup (a step's scans run over the requests, some hundreds); bound by its latency: two block
// scans and one round trip each for the lengths, the stack and the table. A step of 8 requests takes 2.9 us.
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_WAVES = PLAN_THREADS / 64;
// Tokens up to which the same workgroup makes the slot map (8 requests, us, against a second kernel: 5.7 and 6.7 at 2048
// tokens, 7.0 and 6.6 at 4096, 15.8 and 6.6 at 16384).
constexpr int PLAN_SLOTS = 2048;
constexpr int PLAN_BATCH = 8;      // loads of a table row under way at a time

struct PlanCall {
  const int *cached, *fresh;
  const uint8_t* finished;
  int* table;
  int* stack;
  const int* taken;
  int *starts, *lengths, *cached_out, *taken_out;
  int64_t* slots;
  int64_t table_ld;
  int R, W, F, N, pshift;
  int max_new, max_len;   // of a request with new tokens (max_len within the row's pages)
  bool slots_here;   // the slot map too; else page_slots_kernel makes it
};

// Inclusive sums over the workgroup's threads, in request order, and their totals: 32 bits within a wavefront (the callers'
// values are at most 2^24 each), 64 across.
struct Sum2 {
  int64_t a, b, ta, tb;
};
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int dpp_add(int x) { return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROW_MASK, 0xF, false); }
__device__ __forceinline__ int wave_scan_incl(int x) {
  x = dpp_add<0x111, 0xF>(x);   // row_shr:1, 2, 4, 8: within rows of 16 lanes
  x = dpp_add<0x112, 0xF>(x);
  x = dpp_add<0x114, 0xF>(x);
  x = dpp_add<0x118, 0xF>(x);
  x = dpp_add<0x142, 0xA>(x);   // row_bcast:15 into rows 1 and 3
  return dpp_add<0x143, 0xC>(x);   // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ Sum2 block_scan2(int a, int b, int (*sh)[2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  a = wave_scan_incl(a);
  b = wave_scan_incl(b);
  if (lane == 63) {
    sh[wave][0] = a;
    sh[wave][1] = b;
  }
  __syncthreads();
  Sum2 s{a, b, 0, 0};
  for (int w = 0; w < waves; ++w) {
    if (w < wave) {
      s.a += sh[w][0];
      s.b += sh[w][1];
    }
    s.ta += sh[w][0];
    s.tb += sh[w][1];
  }
  __syncthreads();
  return s;
}

// n integers by a wavefront, PLAN_BATCH loads under way
__device__ __forceinline__ void wave_copy(int* to, const int* from, int n) {
  for (int i0 = threadIdx.x & 63; i0 < n; i0 += 64 * PLAN_BATCH) {
    int x[PLAN_BATCH];
#pragma unroll
    for (int u = 0; u < PLAN_BATCH; ++u) x[u] = i0 + 64 * u < n ? from[i0 + 64 * u] : 0;
#pragma unroll
    for (int u = 0; u < PLAN_BATCH; ++u)
      if (i0 + 64 * u < n) to[i0 + 64 * u] = x[u];
  }
}

// Requests whose pages a whole wavefront moves, shared out over the workgroup's wavefronts: they come in any order and often
// next to each other (a batch's prompts behind its generating requests: 31 us at 51 of 512 requests, each wavefront its own;
// 11 shared out).
struct PlanJob {
  int r, n, c, need;   // (a finished request: need = its pages)
  int64_t from, first;   // entry of the stack, token row; c < 0: left out
};

__global__ __launch_bounds__(PLAN_THREADS) void page_plan_kernel(PlanCall a) {
  __shared__ int sh[PLAN_WAVES][2];
  __shared__ int64_t sMost[PLAN_WAVES];
  __shared__ PlanJob sJobs[PLAN_THREADS];
  __shared__ int sCount;
  const int tid = threadIdx.x, lane = tid & 63, threads = blockDim.x;
  const int P = 1 << a.pshift;
  const auto pages_of = [&](int64_t x) { return (int)((x + P - 1) >> a.pshift); };
  int64_t base = min(max(a.taken[0], 0), a.F);   // first free entry of the stack
  // the strip's jobs, each by one wavefront (`mine`: this thread's request is one); between barriers of their own
  auto share_out = [&](bool mine, const PlanJob& job, auto work) {
    if (tid == 0) sCount = 0;
    __syncthreads();
    const uint64_t all = __ballot(mine);
    int at = 0;
    if (lane == 0 && all) at = atomicAdd(&sCount, __popcll(all));
    at = __shfl(at, 0);
    if (mine) sJobs[at + __popcll(all & ((1ull << lane) - 1))] = job;
    __syncthreads();
    for (int i = tid >> 6; i < sCount; i += threads >> 6) work(sJobs[i]);
    __syncthreads();
  };

  // finished requests' pages go back, request after request
  if (a.finished) {
    auto back_of = [&](int r) { return r < a.R && a.finished[r] ? min(min(pages_of(max(a.cached[r], 0)), a.W), 1 << 24) : 0; };
    int64_t total = 0;
    for (int r0 = 0; r0 < a.R; r0 += threads) total += block_scan2(back_of(r0 + tid), 0, sh).ta;
    int64_t at = base - total;
    base = max(at, (int64_t)0);
    for (int r0 = 0; r0 < a.R; r0 += threads) {
      const int r = r0 + tid, back = back_of(r);
      const Sum2 s = block_scan2(back, 0, sh);
      const int64_t to = at + s.a - back;
      share_out(back > 0 && to >= 0, PlanJob{r, 0, 0, back, to, 0},
                [&](const PlanJob& j) { wave_copy(a.stack + j.from, a.table + j.r * a.table_ld, j.need); });
      at += s.ta;
    }
    __threadfence_block();
    __syncthreads();
  }

  // pages for the new tokens, in request order: all a request needs, or none
  int64_t row = 0, given = 0;   // rows and needs of the requests before this strip
  int64_t most = 0;             // needs up to the last request served
  const int64_t avail = a.F - base;
  for (int r0 = 0; r0 < a.R; r0 += threads) {
    const int r = r0 + tid;
    int c = 0, n = 0;
    if (r < a.R) {
      c = a.finished && a.finished[r] ? 0 : max(a.cached[r], 0);
      n = min(max(a.fresh[r], 0), a.N + 1);   // (one row more than there are is as many as any more)
    }
    const int64_t t = (int64_t)c + n;
    const int have = pages_of(c);
    const bool fits = r < a.R && (n > 0 ? n <= a.max_new && t <= a.max_len : t <= ((int64_t)a.W << a.pshift));
    const int need = fits ? pages_of(t) - have : 0;
    const Sum2 s = block_scan2(n, need, sh);
    const int64_t first = row + s.a - n, end = row + s.a, upto = given + s.b;
    const bool served = fits && end <= a.N && (need == 0 || upto <= avail);
    const int64_t from = base + upto - need;   // the request's first entry of the stack
    if (served && need) most = max(most, upto);
    if (r < a.R) {
      a.starts[r] = (int)min(first, (int64_t)a.N);
      a.lengths[r] = served ? (int)t : 0;
      a.cached_out[r] = served ? (int)t : c;
      if (r == a.R - 1) a.starts[a.R] = (int)min(end, (int64_t)a.N);
    }
    int* trow = a.table + (int64_t)r * a.table_ld;
    // the page of the first new token: the last one held, unless that is full
    const bool one = served && n <= 1;
    if (one && n == 1) {
      int page;
      if (need) {
        page = a.stack[from];
        trow[have] = page;
      } else {
        page = trow[c >> a.pshift];
      }
      if (a.slots_here) a.slots[first] = ((int64_t)page << a.pshift) + (c & (P - 1));
    }
    share_out(r < a.R && n > 0 && !one, PlanJob{r, n, served ? c : -1, need, from, first}, [&](const PlanJob& j) {
      int* tr = a.table + j.r * a.table_ld;
      const bool ok = j.c >= 0;
      const int hv = ok ? pages_of(j.c) : 0;
      if (ok) wave_copy(tr + hv, a.stack + j.from, j.need);
      if (a.slots_here)
        for (int i = lane; i < j.n && j.first + i < a.N; i += 64) {
          const int pos = j.c + i, p = pos >> a.pshift;
          const int page = !ok ? -1 : p < hv ? tr[p] : a.stack[j.from + p - hv];
          a.slots[j.first + i] = ok ? ((int64_t)page << a.pshift) + (pos & (P - 1)) : -1;
        }
    });
    row += s.ta;
    given += s.tb;
  }
  if (a.slots_here)
    for (int64_t i = row + tid; i < a.N; i += threads) a.slots[i] = -1;   // rows behind the last request
  // the last served request's needs: the largest over the threads
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) most = max(most, (int64_t)__shfl_xor(most, o));
  if (lane == 0) sMost[tid >> 6] = most;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < threads >> 6; ++w) most = max(most, sMost[w]);
    a.taken_out[0] = (int)(base + most);
  }
}

// The slot map of a long batch: a thread per token, its request found by bisection of `starts` (in the L2).
__global__ __launch_bounds__(NTHREADS) void page_slots_kernel(const int* __restrict__ starts, const int* __restrict__ lengths,
                                                              const int* __restrict__ table, int64_t table_ld,
                                                              int64_t* __restrict__ slots, int R, int W, int N, int pshift) {
  const int i = blockIdx.x * NTHREADS + threadIdx.x;
  if (i >= N) return;
  int lo = 0, hi = R;   // starts[lo] <= i < starts[hi]
  int64_t slot = -1;
  if (i < starts[R]) {
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= i) lo = mid;
      else hi = mid;
    }
    const int first = starts[lo], t = lengths[lo];
    const int pos = t - (starts[lo + 1] - first) + i - first;
    if (t > 0 && pos >= 0) slot = ((int64_t)table[lo * table_ld + (pos >> pshift)] << pshift) + (pos & ((1 << pshift) - 1));
  }
  slots[i] = slot;
}

// ---------------------------------------------------------------------------------------------
// New rows into the pages: a thread per 16-byte chunk of the cache (k's and v's), so that eight lanes write one
// head's row of a page and neighbouring lanes the next heads'. Bound by HBM. Rows whose slot is not in the cache
// are left out.
struct AppendCall {
  const void *k, *v;
  void *k_pages, *v_pages;
  const int64_t* slots;
  int64_t k_token, k_head, v_token, v_head;
  int64_t total;   // slots of the cache
  int N, H, pshift;
};

// `n` elements of type S from p as the cache's type.
template <class S, class P>
__device__ __forceinline__ u32x4 convert_chunk(const typename S::elem* p) {
  if constexpr (std::is_same<S, P>::value) {
    return *reinterpret_cast<const u32x4*>(p);
  } else {
    union {
      u32x4 u[2];
      typename S::elem e[32 / sizeof(typename S::elem)];
    } in;
    union {
      u32x4 u;
      typename P::elem e[P::EPC];
    } out;
    if constexpr (sizeof(typename S::elem) * P::EPC == 8) {   // four 16-bit elements to fp32
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      in.u[0][0] = x.x;
      in.u[0][1] = x.y;
    } else {
      in.u[0] = reinterpret_cast<const u32x4*>(p)[0];
      if constexpr (sizeof(typename S::elem) * P::EPC == 32) in.u[1] = reinterpret_cast<const u32x4*>(p)[1];
    }
#pragma unroll
    for (int e = 0; e < P::EPC; ++e) out.e[e] = P::to_elem(S::to_float(in.e[e]));
    return out.u;
  }
}

template <class S, class P, int D>
__global__ __launch_bounds__(NTHREADS) void paged_append_kernel(AppendCall a) {
  constexpr int CPR = D / P::EPC;
  const uint32_t per = (uint32_t)a.H * CPR;
  const uint64_t id = (uint64_t)blockIdx.x * NTHREADS + threadIdx.x;
  const int token = (int)(id / per);
  if (token >= a.N) return;
  const uint32_t x = (uint32_t)(id - (uint64_t)token * per);
  const int head = (int)(x / CPR), c = (int)(x % CPR);
  const int64_t slot = a.slots[token];
  if (slot < 0 || slot >= a.total) return;
  const int64_t page = slot >> a.pshift;
  const int rowi = (int)(slot & ((1 << a.pshift) - 1));
  const int64_t to = (((page * a.H + head) << a.pshift) + rowi) * D + c * P::EPC;
  typedef typename S::elem se;
  typedef typename P::elem pe;
  const u32x4 kc = convert_chunk<S, P>(static_cast<const se*>(a.k) + token * a.k_token + head * a.k_head + c * P::EPC);
  const u32x4 vc = convert_chunk<S, P>(static_cast<const se*>(a.v) + token * a.v_token + head * a.v_head + c * P::EPC);
  *reinterpret_cast<u32x4*>(static_cast<pe*>(a.k_pages) + to) = kc;
  *reinterpret_cast<u32x4*>(static_cast<pe*>(a.v_pages) + to) = vc;
}

// ---------------------------------------------------------------------------------------------
// Tiles of 32 rows in LDS, rows of CPR 16-byte chunks end to end, chunk c of row r stored at chunk c ^ swz(r): read
// both by lane-per-row fragments (16 rows, one logical chunk, per pass over the 64 banks) and transposed (four
// consecutive rows, two or four consecutive chunks of each). Rows of 256 bytes or more cover every bank, so four
// consecutive rows go to distinct quarters and the 16 rows of a pass to the 16 chunks; at 128 bytes two rows
// share the banks and the pattern is swzq's; at 64 and 32 bytes four and eight rows do.
template <int CPR>
__device__ __forceinline__ int paged_swz(int r) {
  if constexpr (CPR >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  else if constexpr (CPR == 8) return ((r & 3) << 1) ^ ((r >> 2) & 3);
  else if constexpr (CPR == 4) return (r >> 2) & 3;
  else return (r >> 3) & 1;
}

template <class P, int D>
struct PagedTile {
  typedef typename P::elem elem;
  static constexpr int ES = (int)sizeof(elem), RB = D * ES, CPR = RB / 16, BYTES = TILE * RB;
  static constexpr int NS = CPR / 2 > 0 ? CPR / 2 : 1;   // contraction steps of a row
  static constexpr int PARTS = BYTES / 1024;             // direct loads that fill a tile
  static constexpr int DB = D < 32 ? 1 : D / 32;         // 32-column blocks of a value row
  static_assert(CPR >= 2, "a row of at least two chunks");

  // the fragment of step s of row n
  static __device__ __forceinline__ u32x4 row_frag(const char* t, int n, int h, int s) {
    return *reinterpret_cast<const u32x4*>(t + n * RB + (((2 * s + h) ^ paged_swz<CPR>(n)) << 4));
  }
  // columns 32 db .. of the rows of step s, transposed (16-bit types): the operand of V^T P, rows in the accumulator's order
  // (the tile at t + at: one sum and one pointer step, since through a longer chain of them the compiler no longer knows
  // which LDS variable a transposing read is of, and waits for the loads into the others)
  static __device__ __forceinline__ u32x4 value_frag(const char* t, int at, int lane, int db, int s) {
    const int g = lane >> 4, k = lane & 15;
    // (a row of 16 columns: its upper 16 lanes read some of the same, for output rows that nobody keeps)
    const int c = (4 * db + 2 * (g & 1) + ((k & 3) >> 1)) & (CPR - 1);
    u32x4 f;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = 16 * s + 8 * hf + 4 * (g >> 1) + (k >> 2);
      typedef __attribute__((address_space(3))) short4v* lds_s4;
      const int off = at + r * RB + ((c ^ paged_swz<CPR>(r)) << 4) + 8 * (k & 1);
      const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(t + off));
      const uint2 u = __builtin_bit_cast(uint2, x);
      f[2 * hf] = u.x;
      f[2 * hf + 1] = u.y;
    }
    return f;
  }
  // o (columns 32 db ..) += V^T P for the tile's rows, P in the accumulator's layout (lane = query); of a 16-bit type pf, and with
  // WIDE pr, the weights' halves
  template <bool WIDE>
  static __device__ __forceinline__ f32x16 values(const char* t, int lane, int db, const u32x4* pf, const u32x4* pr, const f32x16& p,
                                                  f32x16 o) {
    if constexpr (ES == 2) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const u32x4 v = value_frag(t, 0, lane, db, s);
        o = P::mma(v, pf[s], o);
        if constexpr (WIDE) o = P::mma(v, pr[s], o);
      }
    } else {
      const int n = lane & 31, h = lane >> 5, d = (32 * db + n) & (D - 1);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = crow(i, h);
        const float x = *reinterpret_cast<const float*>(t + r * RB + (((d >> 2) ^ paged_swz<CPR>(r)) << 4) + 4 * (d & 3));
        o = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[i], o, 0, 0, 0);
      }
    }
    return o;
  }
};

__device__ __forceinline__ void g2l16(const void* g, void* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, lds_ptr(l), 16, 0, 0);
}

// 16 bytes per lane from p + off into LDS; zeros past `bytes`
__device__ __forceinline__ void b2l16(const char* p, int bytes, char* l, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(p, bytes), lds_ptr(l), 16, off, 0, 0, 0);
}

// The loads of the tiles that NW wavefronts fill together: part m of a tile (m = wave, wave + NW, ...) is 64 chunks,
// lane l's the chunk at 64 m + l, which holds logical chunk (l % CPR) ^ swz(row) of row (64 m + l) / CPR. A request's
// table is read one tile before its rows.
//
// A part of at most 8 rows lies in one page whatever the page size: its address is one number for the wavefront, the
// loads go through a buffer resource that starts at the part and ends with the request's last row (or holds nothing,
// where the table names no page), and the vector unit computes nothing per load. Narrower rows (16 or 32 rows per part)
// look up a page per lane and read zeros from a row of their own.
template <class P, int D, int NW>
struct PagedRows {
  typedef PagedTile<P, D> T;
  static constexpr int PER = (T::PARTS + NW - 1) / NW;
  static constexpr int ROWS = 64 / T::CPR;   // of a part
  static constexpr bool UNIFORM = ROWS <= 8;
  struct Place {     // of a part's rows in the cache, head 0
    int64_t at;      // byte offset (per lane: -1, none)
    int bytes;       // from there to the last row (uniform parts)
  };
  const int* trow;      // the request's table row
  int pshift, pages, t;
  int64_t page_bytes;   // all heads of a page
  int row[PER], col[PER];   // per lane: row of the tile, byte offset of its chunk (uniform parts: of the part)

  __device__ __forceinline__ PagedRows(const PagedCall& a, int r, int t_, int wave, int lane)
      : trow(a.table + r * a.table_ld), pshift(a.pshift), pages(a.pages), t(t_),
        page_bytes(((int64_t)a.H << a.pshift) * T::RB) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = 64 * (wave + NW * i) + lane;
      row[i] = UNIFORM ? ROWS * (wave + NW * i) : at / T::CPR;
      col[i] = ((at % T::CPR) ^ paged_swz<T::CPR>(at / T::CPR)) << 4;
      if (UNIFORM) col[i] += lane / T::CPR * T::RB;
    }
  }
  // the table entries of key tile kt's rows (-1: none; a tile before the first has none)
  __device__ __forceinline__ void pages_of(int kt, int (&pg)[PER]) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = kt * TILE + row[i];
      pg[i] = (kt >= 0 && j < t) ? trow[j >> pshift] : -1;
    }
  }
  __device__ __forceinline__ void places(int kt, const int (&pg)[PER], Place (&pl)[PER]) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = kt * TILE + row[i], in = (j & ((1 << pshift) - 1)) * T::RB;
      const int page = UNIFORM ? __builtin_amdgcn_readfirstlane(pg[i]) : pg[i];
      const bool ok = (uint32_t)page < (uint32_t)pages;
      if constexpr (UNIFORM) {
        pl[i].at = ok ? page * page_bytes + in : 0;
        pl[i].bytes = ok ? min(ROWS, t - j) * T::RB : 0;
      } else {
        pl[i].at = ok ? page * page_bytes + in + col[i] : -1;
      }
    }
  }
  // the rows of one head, whose rows of page 0 begin at `base`, into a tile
  __device__ __forceinline__ void load(char* tile, const char* base, const Place (&pl)[PER], int wave) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int m = wave + NW * i;
      if (T::PARTS % NW != 0 && m >= T::PARTS) continue;
      if constexpr (UNIFORM)
        b2l16(base + pl[i].at, pl[i].bytes, tile + 1024 * m, col[i]);
      else
        g2l16(pl[i].at >= 0 ? base + pl[i].at : reinterpret_cast<const char*>(&paged_zero_row), tile + 1024 * m);
    }
  }
};

// c + the products of two chunks' elements
template <class P>
__device__ __forceinline__ float chunk_dot(u32x4 x, u32x4 y, float c) {
  union {
    u32x4 u;
    typename P::elem e[P::EPC];
  } a{x}, b{y};
#pragma unroll
  for (int e = 0; e < P::EPC; ++e) c = fmaf(P::to_float(a.e[e]), P::to_float(b.e[e]), c);
  return c;
}

// The least of a wavefront's 64 values, in every lane.
__device__ __forceinline__ float least_of(float x) {
  auto with = [](float y, int z) { return fminf(y, __int_as_float(z)); };
  x = with(x, __builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x111, 0xF, 0xF, false));   // row_shr:1, 2, 4, 8
  x = with(x, __builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x112, 0xF, 0xF, false));
  x = with(x, __builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x114, 0xF, 0xF, false));
  x = with(x, __builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x118, 0xF, 0xF, false));
  x = with(x, __builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x142, 0xA, 0xF, false));   // row_bcast:15, 31
  x = with(x, __builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x143, 0xC, 0xF, false));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// The key tiles that a workgroup's rows can give weight to (as find_reach for the contiguous cache): for a tile
// before the rows, log2 weight <= s log2e |q| max |k| - log2e (least F) - (row maximum), the row maximum at least the row's logit
// of its own key, which has no history. Below -REACH_ZERO a weight is an exact fp32 zero (in one part of several: once they
// are joined; LIFTed ones: nothing beside the row's sum, at 2^-122 of it), and the tile is left out for all of the workgroup's heads together; tiles for which a NaN or an infinity enters
// the bound stay. A mask in LDS, bit i the i-th newest tile; past the mask's end every tile stays. A chunk of
// 4096 queries at 32768 keys, 16 heads, of N(0,1) inputs: 849 us -> 133, the whole call; where the histories leave the oldest fifth without
// weight 800 -> 770; where they are too small everywhere 98 -> 104 (prompts of 60 to 2000 tokens), the rows and norms for nothing.
//
// A part of several takes an equal share of the tiles that stay (of some SHARE_TILES at least: a short request's last parts may
// be empty). Shares of the key range itself leave the oldest part idle where tiles are left out there, and the last ones of short requests:
// the chunk above 824 -> 772 us, chunks of 300 to 700 queries of three requests, each of 8 heads selecting, 68 -> 63.
struct PagedLive {
  const uint64_t* mask;   // NULL: every tile
  int hi, at, left;       // tiles; the next one's number, counted from the newest; how many to come
  __device__ __forceinline__ int next() {   // -1: none
    if (left <= 0) return -1;
    --left;
    while (mask != nullptr) {
      const int word = at >> 6;
      if (word >= REACH_MASK_WORDS) break;
      const uint64_t m = uniform64(mask[word]) >> (at & 63);
      if (m) {
        at += __builtin_ctzll(m);
        break;
      }
      at = (word + 1) << 6;
    }
    return hi - 1 - at++;
  }
  // part z of `parts`
  __device__ __forceinline__ void share(int z, int parts) {
    const int lane = threadIdx.x & 63, words = min((hi + 63) >> 6, REACH_MASK_WORDS);
    int marked = 0, two = 0, upto = 0;   // tiles in the mask that stay; in the lane's pair of words; up to its end
    if (mask != nullptr) {
      static_assert(REACH_MASK_WORDS <= 128, "two words per lane");
#pragma unroll
      for (int i = 0; i < 2; ++i) two += 2 * lane + i < words ? __popcll(mask[2 * lane + i]) : 0;
      upto = wave_scan_incl(two);
      marked = __builtin_amdgcn_readlane(upto, 63);
    }
    const int total = mask == nullptr ? hi : marked + max(hi - 64 * words, 0);
    parts = max(min(parts, (total + SHARE_TILES - 1) / SHARE_TILES), 1);
    if (z >= parts) return;
    const int first = (int)((int64_t)total * z / parts);
    left = (int)((int64_t)total * (z + 1) / parts) - first;
    at = first;
    if (mask == nullptr) return;
    at = 64 * words + first - marked;
    if (first < marked) {
      const int pair = __popcll(__ballot(upto <= first));
      int rest = first - (__builtin_amdgcn_readlane(upto, pair) - __builtin_amdgcn_readlane(two, pair)), word = 2 * pair;
      uint64_t m = uniform64(mask[word]);
      if (rest >= __popcll(m)) {
        rest -= __popcll(m);
        m = uniform64(mask[++word]);
      }
      for (; rest > 0; --rest) m &= m - 1;
      at = 64 * word + __builtin_ctzll(m);
    }
  }
};

// Whether any of a sample of the first `tiles` has history enough for the search to pay.
__device__ __forceinline__ bool paged_live_worth(const float* least, int tiles) {
  if (tiles <= 0) return false;
  const int lane = threadIdx.x & 63, kt = (int)((int64_t)tiles * lane >> 6);
  return __any(least[kt] * REACH_F > REACH_WORTH);
}
// The larger of a row's two bounds over a wavefront's 32 rows of a head: largest |q|, least logit (log2 units) of a row's own key.
template <class P, int D>
__device__ __forceinline__ void paged_live_bounds(const PagedCall& a, const PagedRequest& rq, int r, int row, int head,
                                                  const u32x4 (&qf)[PagedTile<P, D>::NS], float (&bound)[2]) {
  const int h = (threadIdx.x >> 5) & 1, pos = rq.c + row;
  const bool in = row < rq.n;
  const int pg = in ? a.table[r * a.table_ld + (pos >> a.pshift)] : -1;
  const typename P::elem* k = static_cast<const typename P::elem*>(a.k_pages) +
                              ((((int64_t)pg * a.H + head) << a.pshift) + (pos & ((1 << a.pshift) - 1))) * D + h * P::EPC;
  const bool ok = (uint32_t)pg < (uint32_t)a.pages;
  float qq = 0.f, qk = 0.f;
#pragma unroll
  for (int s = 0; s < PagedTile<P, D>::NS; ++s) {
    qq = chunk_dot<P>(qf[s], qf[s], qq);
    if (ok) qk = chunk_dot<P>(qf[s], *reinterpret_cast<const u32x4*>(k + 2 * s * P::EPC), qk);
  }
  const Halves q2 = halves(qq), z2 = halves(qk);
  const float z = (z2.lo + z2.hi) * (a.scale * LOG2E);
  bound[0] = sqrtf(half_max(q2.lo + q2.hi < REACH_NORM2 ? q2.lo + q2.hi : INFINITY));
  bound[1] = -half_max(in ? (z > -3.0e38f ? -z : INFINITY) : -INFINITY);
}
// The mask, by WAVES wavefronts, a lane per key tile: bound[head][part] as above, `least` and `kn` the rows of the workgroup's
// first query tile and first head.
template <int WAVES, int HEADS, int PARTS>
__device__ __forceinline__ void paged_live_mask(const PagedCall& a, const PagedTiles& w, const float (*bound)[PARTS][2], const float* least,
                                                const float* kn, uint64_t* mask) {
  const int lane = threadIdx.x & 63, wave = wave_id();
  float qa[HEADS], zb[HEADS];
#pragma unroll
  for (int g = 0; g < HEADS; ++g) {
    qa[g] = bound[g][0][0];
    zb[g] = bound[g][0][1];
#pragma unroll
    for (int p = 1; p < PARTS; ++p) {
      qa[g] = fmaxf(qa[g], bound[g][p][0]);
      zb[g] = fminf(zb[g], bound[g][p][1]);
    }
    qa[g] *= a.scale * REACH_Q;
  }
  const int words = min((w.kt_hi + 63) >> 6, REACH_MASK_WORDS);
  for (int word = wave; word < words; word += WAVES) {
    const int kt = w.kt_hi - 1 - (word * 64 + lane);
    bool live = kt >= 0;
    if (live && (kt + 1) * TILE <= w.rq.c + w.row0) {
      const float f = least[kt] * REACH_F;
      if (f > REACH_WORTH) {   // (else a key norm may be missing)
        bool dead = true;
#pragma unroll
        for (int g = 0; g < HEADS; ++g) dead &= qa[g] * kn[g * a.reach_ld + kt] - f - zb[g] < -REACH_ZERO;
        live = !dead;
      }
    }
    const uint64_t m = __ballot(live);
    if (lane == 0) mask[word] = m;
  }
}

// The key norms of key tile kb, by a wavefront: `run` each key's history after the step (lane: key lane & 31).
template <class P, int D>
__device__ __forceinline__ void paged_key_norms(const PagedCall& a, const PagedRequest& rq, int r, int g, int kb, float run) {
  typedef typename P::elem elem;
  constexpr int NS = PagedTile<P, D>::NS;
  const int lane = threadIdx.x & 63, h = lane >> 5, j = kb * TILE + (lane & 31), hd = g * (a.H / a.G);
  if (a.least == nullptr || !(least_of(j < rq.t ? run : INFINITY) * REACH_F > REACH_WORTH)) return;
  const int pg = j < rq.t ? a.table[r * a.table_ld + (j >> a.pshift)] : -1;
  const bool ok = (uint32_t)pg < (uint32_t)a.pages;
  constexpr int HB = NS <= 4 ? 4 : NS == 8 ? 2 : 1;   // heads whose rows are on their way at a time
  for (int head = hd; head < hd + a.H / a.G; head += HB) {
    u32x4 kr[HB][NS], vr[HB][NS];
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      const int hb = min(head + b, hd + a.H / a.G - 1);
      const int64_t at = ((((int64_t)(ok ? pg : 0) * a.H + hb) << a.pshift) + (j & ((1 << a.pshift) - 1))) * D + h * P::EPC;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        kr[b][s] = *reinterpret_cast<const u32x4*>(static_cast<const elem*>(a.k_pages) + at + 2 * s * P::EPC);
        vr[b][s] = *reinterpret_cast<const u32x4*>(static_cast<const elem*>(a.v_pages) + at + 2 * s * P::EPC);
      }
    }
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      float kk = 0.f, vv = 0.f;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        kk = chunk_dot<P>(kr[b][s], kr[b][s], kk);
        vv = chunk_dot<P>(vr[b][s], vr[b][s], vv);
      }
      const Halves k2 = halves(kk), v2 = halves(vv);
      // (a row without a page is zeros)
      const float x = !ok ? 0.f : (k2.lo + k2.hi < REACH_NORM2 && v2.lo + v2.hi < REACH_NORM2) ? k2.lo + k2.hi : INFINITY;
      const float mx = -least_of(-x);
      if (lane == 0 && head + b < hd + a.H / a.G) a.kn[((int64_t)r * a.H + head + b) * a.reach_ld + kb] = sqrtf(mx);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// The selectors' histories of a step of several tokens: carry[tile][g][j], what key j has received before the
// tile's first query, and the state after the step. A wavefront owns 32 keys of one selector (rows in registers) and
// its workgroup walks the request's query tiles, as sel_carry64_kernel does, U tiles at a time: a step rarely has keys
// enough for more than one wavefront per SIMD, so the walk is bound by the latency of its own instructions and the U
// products and sums are kept independent; the rows are loaded into LDS three steps ahead, once for the workgroup. At 4096
// queries on 32768 keys (us, histories and state alone): 48; one tile at a time from the L2 105, four at a time 64, through LDS
// one step ahead 55. Rows of keys that no query of a tile sees hold no history: the forward masks those keys.
//
// With a.least, also what the forward needs to leave out key tiles without weight (PagedLive): each key tile's least history
// on entry to every fourth query tile, and, of key tiles whose least history at the end makes it possible, the largest
// |k| of every head of the group (infinity where a key or a value is not finite, or a product could overflow): 69 us, of that 16 to read the keys and values of 16 heads.
template <class P, int D>
__global__ __launch_bounds__(NTHREADS) void paged_carry_kernel(PagedCall a, float* __restrict__ carry, int64_t carry_ld) {
  typedef PagedTile<P, D> T;
  typedef typename P::elem elem;
  constexpr int NS = T::NS, U = T::BYTES > 8192 ? 1 : T::BYTES > 4096 ? 2 : 4, PER = U * T::PARTS / NWAVES;
  // The U tiles of step t are in buffer t mod 4 (variables of their own: a step's reads touch none of the others), filled
  // by loads that step t - 3 issues (the prologue for the first three). Every step issues PER loads (past the last tile: of
  // nothing), then U + 1 stores, so at its end the loads of step t + 1, issued in step t - 2, have landed once
  // no more than 2 PER + 3 (U + 1) newer operations run.
  __shared__ __attribute__((aligned(16))) char sQ0[U * T::BYTES], sQ1[U * T::BYTES], sQ2[U * T::BYTES], sQ3[U * T::BYTES];
  const int lane = threadIdx.x & 63, wave = wave_id(), n = lane & 31, h = lane >> 5;
  const int r = blockIdx.z, g = blockIdx.y, seg = blockIdx.x % a.segments;
  const PagedRequest rq = paged_request(a, r);
  if (!rq.live || (a.ones && rq.n == 1)) return;
  const int hd = g * (a.H / a.G);
  const int nkb = (rq.t + TILE - 1) / TILE, last = min((rq.n + TILE - 1) / TILE, (seg + 1) * a.seg_tiles);   // (its last query tile + 1)
  const elem* q = static_cast<const elem*>(a.q) + rq.first * a.q_token + hd * a.q_head;
  const int* trow = a.table + r * a.table_ld;
  float* state = a.selected + ((int64_t)r * a.G + g) * a.state_ld;
  const int64_t plane = a.G * carry_ld;   // from one tile's histories to the next's
  float* cr = carry + (int64_t)((rq.first >> 5) + r) * plane + g * carry_ld;
  // part m = wave + NWAVES i of the U tiles' 16-byte chunks; rows past the last read as zeros
  int off[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = 64 * (wave + NWAVES * i) + lane, row = at / T::CPR;
    off[i] = row * (int)a.q_token * T::ES + (((at % T::CPR) ^ paged_swz<T::CPR>(row % TILE)) << 4);
  }
  auto load_q = [&](int rb, char* buf) {
    const int left = max(min(rq.n - rb * TILE, U * TILE), 0);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      b2l16(reinterpret_cast<const char*>(q + rb * TILE * a.q_token), left * (int)a.q_token * T::ES, buf + 1024 * (wave + NWAVES * i), off[i]);
  };
  for (int kb0 = blockIdx.x / a.segments * NWAVES; kb0 < nkb; kb0 += gridDim.x / a.segments * NWAVES) {
    const int kb = kb0 + wave, j = kb * TILE + n;
    // tiles before this end before the workgroup's first key
    int rb = max((max(kb0 * TILE - rq.c, 0) / TILE) & ~3, seg * a.seg_tiles);   // (every fourth one begins a step)
    const bool any = rb < last;
    if (any) {
      load_q(rb, sQ0);
      load_q(rb + U, sQ1);
      load_q(rb + 2 * U, sQ2);
    }
    u32x4 kf[NS];
    {
      const int pg = j < rq.t ? trow[j >> a.pshift] : -1;
      const bool ok = (uint32_t)pg < (uint32_t)a.pages;
      const elem* k = static_cast<const elem*>(a.k_pages) +
                      ((((int64_t)(ok ? pg : 0) * a.H + hd) << a.pshift) + (j & ((1 << a.pshift) - 1))) * D;
#pragma unroll
      for (int s = 0; s < NS; ++s)
        kf[s] = ok ? *reinterpret_cast<const u32x4*>(k + (2 * s + h) * P::EPC) : u32x4{0, 0, 0, 0};
    }
    float run = j < rq.c && seg == 0 ? state[j] : 0.f;
    const int64_t lplane = a.G * a.reach_ld;
    float* least = a.least + ((int64_t)((rq.first >> 5) + r) * a.G + g) * a.reach_ld + kb;   // (not used without a.least)
    const uint32_t end = (uint32_t)rq.t * 4, own = h == 0 && j < rq.t ? (uint32_t)j * 4 : end;   // byte offset of the lane's key in a row of histories
    auto step = [&](const char* buf, char* next) {
      load_q(rb + 3 * U, next);
      f32x16 acc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) acc[u] = zero16();
#pragma unroll
      for (int s = 0; s < NS; ++s)   // (the U chains side by side)
#pragma unroll
        for (int u = 0; u < U; ++u) acc[u] = P::mma(T::row_frag(buf + u * T::BYTES, n, h, s), kf[s], acc[u]);
      float sum[U];
      const int qbase = rq.c + rb * TILE;
      // (one choice for the U tiles: their sums interleave too)
      if (qbase > kb * TILE + TILE - 1 && kb * TILE >= a.exempt) {
#pragma unroll
        for (int u = 0; u < U; ++u) sum[u] = block_selection_sum(acc[u], true, 0, a.scale);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
          sum[u] = block_selection_sum(acc[u], false, j >= a.exempt ? j - qbase - u * TILE - 4 * h : 32, a.scale);
      }
      {
        const bool kept = a.least != nullptr && seg == 0 && (rb & 3) == 0 && rb < last && kb < nkb;
        const float mn = kept ? least_of(j >= rq.t ? INFINITY : run == run ? run : -INFINITY) : 0.f;   // (a NaN keeps the tile)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(mn), rsrc(least + rb * lplane, kept ? 4 : 0), lane * 4, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {   // (every lane stores, past the row's end where it has no key or the tile is none)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(run), rsrc(cr + (rb + u) * plane, rb + u < last ? end : 0), own, 0, 0);
        run += sum[u];
      }
      rb += U;
      // (one asm block: at a barrier of its own the compiler waits for everything)
      __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * PER + 3 * (U + 1)) : "memory");
    };
    wait_loads();
    __syncthreads();
    while (any) {
      step(sQ0, sQ3);
      if (rb >= last) break;
      step(sQ1, sQ0);
      if (rb >= last) break;
      step(sQ2, sQ1);
      if (rb >= last) break;
      step(sQ3, sQ2);
      if (rb >= last) break;
    }
    wait_loads();   // nothing on its way into LDS when the workgroup ends or takes its next keys
    __syncthreads();
    if (a.segments == 1) {
      if (h == 0 && j < rq.t) state[j] = run;
      if (kb < nkb) paged_key_norms<P, D>(a, rq, r, g, kb, run);
    } else if (h == 0 && j < rq.t) {
      a.totals[(((int64_t)r * a.G + g) * a.segments + seg) * carry_ld + j] = run;
    }
  }
}

// The histories of the segments after the first, which begin at zero, raised by what the segments before have added; the
// state, and what paged_carry leaves to do of least histories and key norms. Workgroup: 256 keys, a thread each, of SEG_PART
// query tiles (the first two of the grid's y: the state and the norms).
constexpr int SEG_PART = 16;
template <class P, int D>
__global__ __launch_bounds__(NTHREADS) void paged_carry_join_kernel(PagedCall a, float* __restrict__ carry, int64_t carry_ld) {
  const int lane = threadIdx.x & 63, r = blockIdx.z / a.G, g = blockIdx.z % a.G, j = blockIdx.x * NTHREADS + threadIdx.x;
  const PagedRequest rq = paged_request(a, r);
  if (!rq.live || (a.ones && rq.n == 1) || (int)blockIdx.x * NTHREADS >= rq.t) return;
  const float* totals = a.totals + ((int64_t)r * a.G + g) * a.segments * carry_ld + min(j, rq.t - 1);
  auto before = [&](int seg) {
    float sum = 0.f;
    for (int i = 0; i < seg; ++i) sum += totals[i * carry_ld];
    return sum;
  };
  if (blockIdx.y < 2) {   // one of every wavefront's two key tiles
    const int kb = (j >> 6) * 2 + blockIdx.y;
    const float run = before(a.segments), x = __shfl(run, (lane & 31) + 32 * blockIdx.y);
    if (lane >> 5 == blockIdx.y && j < rq.t) a.selected[((int64_t)r * a.G + g) * a.state_ld + j] = run;
    if (kb * TILE < rq.t) paged_key_norms<P, D>(a, rq, r, g, kb, x);
    return;
  }
  const int rb0 = a.seg_tiles + ((int)blockIdx.y - 2) * SEG_PART, ntile = (rq.n + TILE - 1) / TILE;
  // (tiles before a key's hold nothing of it)
  const int first = max(rb0, (max((int)blockIdx.x * NTHREADS - rq.c, 0) / TILE) & ~3), last = min(rb0 + SEG_PART, ntile);
  if (first >= last) return;
  int seg = first / a.seg_tiles;
  float base = before(seg);
  const int64_t plane = a.G * carry_ld;
  float* cr = carry + (int64_t)((rq.first >> 5) + r) * plane + g * carry_ld + min(j, rq.t - 1);
  for (int rb = first; rb < last; rb += 4) {   // (segments begin at multiples of four)
    if (rb >= (seg + 1) * a.seg_tiles) base += totals[seg++ * carry_ld];
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = cr[min(rb + u, last - 1) * plane];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] += base;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (rb + u < last && j < rq.t) cr[(rb + u) * plane] = x[u];
    if (a.least != nullptr) {
      const float y = j >= rq.t ? INFINITY : x[0] == x[0] ? x[0] : -INFINITY;
      float* least = a.least + ((int64_t)((rq.first >> 5) + r + rb) * a.G + g) * a.reach_ld;
      const float lo = least_of(lane < 32 ? y : INFINITY), hi = least_of(lane < 32 ? INFINITY : y);
      if ((lane & 31) == 0 && j < rq.t) least[j / TILE] = lane < 32 ? lo : hi;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// The attention of a step of several tokens. Workgroup (HG heads of one selector and a part of the key tiles, NW x 32 query
// rows of one request, numbered as above, the last first): workgroups next to each other, which the XCDs take in turns, are of
// different heads and parts, so that an XCD's L2 holds few heads' keys. As fwd64_kernel: a wavefront's 32
// queries against one 32-key tile at a time, newest first, every operand loaded straight into LDS one tile ahead,
// the selection (-F, through the wavefront's LDS rows) one tile ahead of the softmax. What differs is where rows come
// from: each lane looks its row's page up one tile before the load.
//
// WHOLE: every head selects for itself (HG = 1): the wavefront's logits arrive with F already subtracted, and the
// key tile is loaded once.
//
// P is rounded to the cache's type for the product with V (by half a step at most: relative 2^-8 bf16, 2^-11 fp16, of fp16
// weights below 2^-24 of the largest 2^-35 of that; the size of the output's own rounding; fp32 not at all). WIDE: as the sum of
// two numbers of that type (2^-16, 2^-22), in twice the value products, which is what fp32 operands come to, q, k and v
// being of 16 bits as they are: a chunk of 4096 fp16 queries at 32768 keys, 16 heads, 757 -> 937 us, prompts of 60 to 2000
// tokens 114 -> 136, chunks of 300 to 700 queries of three requests, each of 8 heads selecting, 62 -> 64. Logits, F, row
// statistics and sums are fp32.

// The grid of the forward kernels: heads and parts, then query tiles, over y and z where a dimension's 65535 would not hold them.
inline dim3 tile_grid(int64_t per_tile, int64_t tiles) {
  const int64_t rounds = cdiv(tiles, 32768);
  return dim3((unsigned)per_tile, (unsigned)cdiv(tiles, rounds), (unsigned)rounds);
}
__device__ __forceinline__ int last_tile_first() { return gridDim.y * gridDim.z - 1 - (blockIdx.z * gridDim.y + blockIdx.y); }

// Workgroup number x (1 << SH rows, numbered as above), part z; false: nothing. Rows that no workgroup computes, those
// before the first request, behind the last and of requests left out, become zero here, COLS columns from col0 on, unless the parts are
// joined afterwards (the join does it).
template <class P, int SH, int COLS, int THREADS>
__device__ __forceinline__ bool paged_tiles(const PagedCall& a, int x, int z, int64_t row_elems, int col0, bool joined,
                                            PagedTiles& w) {
  auto clear = [&](int first, int count) {
    typename P::elem* out = static_cast<typename P::elem*>(a.out) + first * row_elems + col0;
    for (int i = threadIdx.x; i < count * COLS; i += THREADS) out[i / COLS * row_elems + i % COLS] = P::to_elem(0.f);
  };
  const bool zeros = !joined && z == 0;
  if (zeros) {
    const int first = x << SH, hi = min((x + 1) << SH, a.N), lo = min(max(first, a.starts[a.R]), hi);
    clear(lo, hi - lo);
    if (first < a.starts[0]) clear(first, min(hi, a.starts[0]) - first);
  }
  w.r = find_request<false>(a.starts, a.R, x, SH);
  w.rq = paged_request(a, w.r);
  w.row0 = (x - ((w.rq.first >> SH) + w.r)) << SH;
  if (w.row0 < 0 || w.row0 >= w.rq.n) return false;
  if (a.ones && w.rq.n == 1 && w.rq.live) return false;   // (paged_step's)
  if (!w.rq.live) {
    if (zeros) clear(w.rq.first + w.row0, min(1 << SH, w.rq.n - w.row0));
    return false;
  }
  w.kt_hi = (w.rq.c + min(w.row0 + (1 << SH), w.rq.n) - 1) / TILE + 1;
  return true;
}

// A wavefront's results for the request's row `row` (lane = row; o transposed, 4 columns per quarter): the output, or the
// part's share of it: reference m (log2 units), sum l, and the sums of weighted values.
template <class P, int D>
__device__ __forceinline__ void paged_write(const PagedCall& a, const PagedTiles& w, int row, int head, int z, float m, float l,
                                            const f32x16 (&o)[PagedTile<P, D>::DB], int h, float* part_ml, float* part_o) {
  typedef typename P::elem elem;
  const Halves lh = halves(l);
  if (row >= w.rq.n) return;
  const float ltot = lh.lo + lh.hi;
  const int64_t at = (int64_t)(w.rq.first + row) * a.H + head, part = (int64_t)z * a.N * a.H + at;
  const bool joined = part_o != nullptr;
  if (joined && h == 0) {
    part_ml[2 * part] = m;
    part_ml[2 * part + 1] = ltot;
  }
  const float inv = joined ? 1.f : 1.f / ltot;
#pragma unroll
  for (int db = 0; db < PagedTile<P, D>::DB; ++db) {
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int d = db * 32 + 8 * q4 + 4 * h;
      if (D < 32 && d >= D) continue;
      const float4 v4 = make_float4(o[db][4 * q4] * inv, o[db][4 * q4 + 1] * inv, o[db][4 * q4 + 2] * inv, o[db][4 * q4 + 3] * inv);
      elem* out = static_cast<elem*>(a.out) + at * D + d;
      if (joined) {
        *reinterpret_cast<float4*>(part_o + part * D + d) = v4;
      } else if constexpr (sizeof(elem) == 2) {
        *reinterpret_cast<uint2*>(out) = make_uint2((uint32_t)P::to_elem(v4.x) | ((uint32_t)P::to_elem(v4.y) << 16),
                                                    (uint32_t)P::to_elem(v4.z) | ((uint32_t)P::to_elem(v4.w) << 16));
      } else {
        *reinterpret_cast<float4*>(out) = v4;
      }
    }
  }
}

template <class P, int D, int HG, int NW>
struct FwdLds {
  typedef PagedTile<P, D> T;
  struct Tiles {
    __attribute__((aligned(16))) char k[HG][T::BYTES];
    __attribute__((aligned(16))) char v[HG][T::BYTES];
  };
};

template <class P, int D, int HG, int NW, bool WHOLE, bool WIDE>
__global__ __launch_bounds__(NW * 64, (NW == 1 ? 1 : (sizeof(typename P::elem) == 2 && D <= 64) ? (HG == 1 ? 3 : 2) : 1)) void paged_fwd_kernel(
    PagedCall a, const float* __restrict__ carry, int64_t carry_ld, int splits, float* __restrict__ part_ml,
    float* __restrict__ part_o) {
  typedef PagedTile<P, D> T;
  typedef typename P::elem elem;
  typedef PagedRows<P, D, NW> Rows;
  constexpr int NS = T::NS, DB = T::DB, PER = Rows::PER, LDF = TILE + 4;
  constexpr int SH = NW == 4 ? 7 : 5;   // rows of a workgroup: 1 << SH
  static_assert(!WHOLE || HG == 1, "a head that selects for itself alone");
  // separate variables, so that the compiler knows a step's reads do not touch the buffers being filled. Lifetimes as
  // in fwd64_kernel: sB0, sB1 the K and V rows of the t-th tile visited (buffer t mod 2; filled in step t - 1, read
  // in step t); sS0, sS1 its selector's K rows (filled in step t - 2, read by the selection at the end of step t - 1); sF
  // each wavefront's own. A step ends with every load landed and a barrier.
  __shared__ typename FwdLds<P, D, HG, NW>::Tiles sB0, sB1;
  __shared__ __attribute__((aligned(16))) char sS0[T::BYTES], sS1[T::BYTES];
  __shared__ __attribute__((aligned(16))) float sF[NW][TILE * LDF];
  __shared__ uint64_t sMask[NW == 1 ? 1 : REACH_MASK_WORDS];   // PagedLive
  __shared__ float sBound[HG][NW][2];

  const int tid = threadIdx.x, lane = tid & 63, wave = NW == 1 ? 0 : wave_id();
  const int n = lane & 31, h = lane >> 5;
  const int groups = a.H / HG, x = last_tile_first(), z = blockIdx.x / groups;
  const int hd0 = (blockIdx.x % groups) * HG, per = a.H / a.G, g0 = hd0 / per, hsel = g0 * per;
  PagedTiles w;
  if (!paged_tiles<P, SH, HG * D, NW * 64>(a, x, z, (int64_t)a.H * D, hd0 * D, part_o != nullptr, w)) return;
  const PagedRequest& rq = w.rq;
  const int r = w.r, row0 = w.row0, kt_hi = w.kt_hi;

  const int rb0 = row0 + wave * TILE;          // the wavefront's first row
  const int qpos0 = rq.c + rb0;                // and its position
  const int q_row = rb0 + n, q_pos = qpos0 + n;
  // tiles the wavefront needs: those up to its last row's
  const int my_end = rb0 < rq.n ? min((qpos0 + TILE - 1) / TILE + 1, kt_hi) : 0;

  u32x4 qf[HG][NS], qs[NS];
  {
    const elem* qt = static_cast<const elem*>(a.q) + (int64_t)(rq.first + q_row) * a.q_token;
    const bool ok = q_row < rq.n;
    auto frag = [&](int head, int s) -> u32x4 {
      return ok ? *reinterpret_cast<const u32x4*>(qt + head * a.q_head + (2 * s + h) * P::EPC) : u32x4{0, 0, 0, 0};
    };
#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
      for (int g = 0; g < HG; ++g) qf[g][s] = frag(hd0 + g, s);
      qs[s] = WHOLE ? qf[0][s] : frag(hsel, s);
    }
  }
  float m[HG], l[HG];
  f32x16 o[HG][DB];
#pragma unroll
  for (int g = 0; g < HG; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[g][db] = zero16();
  }
  const float sl2 = a.scale * LOG2E, neg_inv_scale = -1.f / a.scale;

  const Rows rows(a, r, rq.t, wave, lane);
  const int64_t head_bytes = (int64_t)T::RB << a.pshift;
  const char* kp = static_cast<const char*>(a.k_pages);
  const char* vp = static_cast<const char*>(a.v_pages);
  const float* crow_p = carry + ((int64_t)((rq.first >> 5) + r + (min(rb0, rq.n - 1) >> 5)) * a.G + g0) * carry_ld;

  auto load_tile = [&](typename FwdLds<P, D, HG, NW>::Tiles& B, const typename Rows::Place (&off)[PER]) {
#pragma unroll
    for (int g = 0; g < HG; ++g) {
      if (!WHOLE) rows.load(B.k[g], kp + (hd0 + g) * head_bytes, off, wave);
      rows.load(B.v[g], vp + (hd0 + g) * head_bytes, off, wave);
    }
  };
  auto load_sel = [&](char* S, const typename Rows::Place (&off)[PER]) { rows.load(S, kp + hsel * head_bytes, off, wave); };
  auto carry_of = [&](int kt) { return kt >= 0 ? crow_p[min(kt * TILE + n, rq.t - 1)] : 0.f; };

  // Tile kt's selection into the wavefront's F rows (fwd64_kernel's select)
  auto select = [&](int kt, const char* S, float entry) {
    const int kbase = kt * TILE;
    f32x16 l0 = zero16();
#pragma unroll
    for (int s = 0; s < NS; ++s) l0 = P::mma(qs[s], T::row_frag(S, n, h, s), l0);
    f32x16 sel;
#pragma unroll
    for (int i = 0; i < 16; ++i) sel[i] = __builtin_amdgcn_fmed3f(-l0[i], -3.0e38f, 0.f);
    if (kbase + TILE - 1 >= qpos0 || kbase < a.exempt) {
      const int jk = kbase + n, thr = jk >= a.exempt ? jk - qpos0 - 4 * h : 32;
#pragma unroll
      for (int i = 0; i < 16; ++i) sel[i] = crow(i, 0) > thr ? sel[i] : 0.f;
    }
    float run = entry * neg_inv_scale;
    float* fw = sF[wave];
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const Halves s4 = halves(((sel[4 * q4] + sel[4 * q4 + 1]) + sel[4 * q4 + 2]) + sel[4 * q4 + 3]);
      float p = (h == 0) ? run : run + s4.lo;
#pragma unroll
      for (int t2 = 0; t2 < 4; ++t2) {
        fw[crow(4 * q4 + t2, h) * LDF + n] = WHOLE ? p + l0[4 * q4 + t2] : p;
        p += sel[4 * q4 + t2];
      }
      run = (run + s4.lo) + s4.hi;
    }
  };

  PagedLive tiles{nullptr, kt_hi, 0, 0};
  if constexpr (NW > 1) {
    const float* least = a.least + ((int64_t)((rq.first >> 5) + r + (row0 >> 5)) * a.G + g0) * a.reach_ld;
    if (a.least != nullptr && paged_live_worth(least, (rq.c + row0) / TILE)) {
#pragma unroll
      for (int g = 0; g < HG; ++g) {
        float bound[2];
        paged_live_bounds<P, D>(a, rq, r, q_row, hd0 + g, qf[g], bound);
        if (lane == 0) {
          sBound[g][wave][0] = bound[0];
          sBound[g][wave][1] = bound[1];
        }
      }
      __syncthreads();
      paged_live_mask<NW, HG, NW>(a, w, sBound, least, a.kn + ((int64_t)r * a.H + hd0) * a.reach_ld, sMask);
      __syncthreads();
      tiles.mask = sMask;
    }
  }

  // the tiles, newest first: cur in the buffers, n1's selector rows too, n2's pages known (-1: none)
  tiles.share(z, splits);
  int cur = tiles.next(), n1 = tiles.next(), n2 = tiles.next();
  typename Rows::Place off1[PER], off2[PER];   // of tiles n1 and n2
  int pg[PER];
  {
    typename Rows::Place off0[PER];
    rows.pages_of(cur, pg);
    rows.places(cur, pg, off0);
    if (cur >= 0) {
      load_tile(sB0, off0);
      load_sel(sS0, off0);
    }
    rows.pages_of(n1, pg);
    rows.places(n1, pg, off1);
    if (n1 >= 0) load_sel(sS1, off1);
    rows.pages_of(n2, pg);
  }
  float entry1 = carry_of(n1);
  const float entry0 = carry_of(cur);
  wait_loads();
  __syncthreads();
  if (cur >= 0 && cur < my_end) select(cur, sS0, entry0);
  __syncthreads();   // every wavefront is past its reads of sS0, which the first step fills

  auto step = [&](auto odd_tag) __attribute__((always_inline)) {
    constexpr bool ODD = decltype(odd_tag)::value;
    auto& B = ODD ? sB1 : sB0;
    rows.places(n2, pg, off2);
    if (n1 >= 0) load_tile(ODD ? sB0 : sB1, off1);
    if (n2 >= 0) load_sel(ODD ? sS1 : sS0, off2);
    const int n3 = tiles.next();
    rows.pages_of(n3, pg);
    const float entry2 = carry_of(n2);
    if (cur < my_end) {
      const int kbase = cur * TILE;
      f32x16 fs;
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const float4 f4 = *reinterpret_cast<const float4*>(&sF[wave][n * LDF + 8 * q4 + 4 * h]);
        fs[4 * q4] = f4.x;
        fs[4 * q4 + 1] = f4.y;
        fs[4 * q4 + 2] = f4.z;
        fs[4 * q4 + 3] = f4.w;
      }
#pragma unroll
      for (int g = 0; g < HG; ++g) {
        f32x16 lg = fs;   // the product accumulates onto -F
        if (!WHOLE) {
#pragma unroll
          for (int s = 0; s < NS; ++s) lg = P::mma(T::row_frag(B.k[g], n, h, s), qf[g][s], lg);
        }
        if (kbase + TILE - 1 > qpos0) {   // keys past a query (those past the last position among them)
          const int thr = q_pos - kbase - 4 * h;
#pragma unroll
          for (int i = 0; i < 16; ++i) lg[i] = crow(i, 0) <= thr ? lg[i] : -INFINITY;
        }
        float zmax = lg[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) zmax = fmaxf(zmax, lg[i]);
        const Halves zh = halves(zmax);
        const float m_new = fmaxf(m[g], fmaxf(zh.lo, zh.hi) * sl2);
        if (__any(m_new > m[g])) {
          const float alpha = (m_new == -INFINITY) ? 1.f : fast_exp2(m[g] - m_new);
          m[g] = m_new;
          l[g] *= alpha;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[g][db][i] *= alpha;
        }
        const float mu = (m[g] == -INFINITY) ? 0.f : m[g], ref = P::LIFT == 0.f ? -mu : P::LIFT - mu;
        float psum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = fast_exp2(fmaf(lg[i], sl2, ref));
          lg[i] = p;
          psum += p;
        }
        l[g] += psum;
        u32x4 pf[2], pr[2];
        if constexpr (T::ES == 2) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            pf[s] = P::pack(lg, s);
            if constexpr (WIDE) pr[s] = P::rest(lg, pf[s], s);
          }
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) o[g][db] = T::template values<WIDE>(B.v[g], lane, db, pf, pr, lg, o[g][db]);
      }
    }
    if (n1 >= 0 && n1 < my_end) select(n1, ODD ? sS0 : sS1, entry1);
    entry1 = entry2;
#pragma unroll
    for (int i = 0; i < PER; ++i) off1[i] = off2[i];
    wait_loads();
    __syncthreads();
    cur = n1;
    n1 = n2;
    n2 = n3;
  };
  while (cur >= 0) {
    step(std::false_type{});
    if (cur < 0) break;
    step(std::true_type{});
  }

#pragma unroll
  for (int g = 0; g < HG; ++g) paged_write<P, D>(a, w, q_row, hd0 + g, z, m[g], l[g], o[g], h, part_ml, part_o);
}

// The same for groups of four heads or more at 16-bit head dim 64, the usual sizes of a long step: sixteen wavefronts, one
// workgroup per CU, query tiles 4 x 32 rows, four heads; wavefront w has head w % 4, query tile w / 4. Each tile's selection is
// made once for the four heads (every wavefront one tile in four, its own query tile's, in turns that give each SIMD one
// of the four selections of a step).
//
// What bounds paged_fwd_kernel is the vector unit: per head and tile 16 exponentials (256 cycles of a SIMD) and, of some 90
// other instructions, half of a selection's 105 and the running maximum's. Here a quarter of a selection, and no maximum: the
// weights are taken against the reference mu of the tiles before, and only where a row's sum of them over half a tile
// passes BIG (or a row has no reference yet) is the maximum looked for, mu moved and the tile's weights taken again.
// Any reference within 2^14 of the maximum gives the same bf16 weights to rounding; fp16's (LIFT times larger) stay within 2^5 of it,
// so that none passes the type's largest number.
// At 4096 queries on 32768 keys, 16 heads, every tile computed, under the profiler: 0.78 ms (657 TFLOP/s of the two products; 0.80
// before PagedLive's equal shares), paged_fwd_kernel 1.04, with the selection after the products 0.91, with eight wavefronts of two
// query tiles each 0.97 (0.91). What is left over is each step's common start and end: its LDS reads
// at once (0.46 ms without selection, value products and loads), and the wait for its last wavefront.
template <class P, bool WIDE>
__global__ __launch_bounds__(1024) void paged_fwd4_kernel(PagedCall a, const float* __restrict__ carry, int64_t carry_ld,
                                                          int splits, float* __restrict__ part_ml, float* __restrict__ part_o) {
  constexpr int D = 64, HG = 4, SH = 7, LDF = TILE + 4;
  typedef PagedTile<P, D> T;
  typedef typename P::elem elem;
  typedef PagedRows<P, D, 4> Rows;
  constexpr int NS = T::NS, DB = T::DB;
  static_assert(T::ES == 2 && Rows::PER == 1 && Rows::UNIFORM, "parts of eight rows, one per wavefront of four");
  // lifetimes as in paged_fwd_kernel; sF0, sF1 the four query tiles' F of the t-th tile visited (buffer t mod 2, written in step
  // t - 1, read in step t)
  struct Tiles {
    __attribute__((aligned(16))) char k[HG][T::BYTES];
    __attribute__((aligned(16))) char v[HG][T::BYTES];
  };
  __shared__ Tiles sB0, sB1;
  __shared__ __attribute__((aligned(16))) char sS0[T::BYTES], sS1[T::BYTES];
  __shared__ __attribute__((aligned(16))) float sF0[4][TILE * LDF], sF1[4][TILE * LDF];
  __shared__ u32x4 sQ[4][NS * 64];   // the selector's query fragments (written once: registers are short)
  __shared__ uint64_t sMask[REACH_MASK_WORDS];   // PagedLive
  __shared__ float sBound[HG][4][2];

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), n = lane & 31, h = lane >> 5;
  const int u = wave & 3, qt = wave >> 2;   // the wavefront's head and query tile
  const int groups = a.H / HG, x = last_tile_first(), z = blockIdx.x / groups;
  const int hd0 = (blockIdx.x % groups) * HG, per = a.H / a.G, g0 = hd0 / per, hsel = g0 * per;
  PagedTiles w;
  if (!paged_tiles<P, SH, HG * D, 1024>(a, x, z, (int64_t)a.H * D, hd0 * D, part_o != nullptr, w)) return;
  const PagedRequest& rq = w.rq;

  const int rb = w.row0 + qt * TILE, qpos0 = rq.c + rb;   // the query tile's first row and its position
  const int end = rb < rq.n ? (qpos0 + TILE - 1) / TILE + 1 : 0;   // tiles that it needs

  u32x4 qf[NS];
  {
    const int row = rb + n;
    const elem* qp = static_cast<const elem*>(a.q) + (int64_t)(rq.first + row) * a.q_token;
    auto frag = [&](int head, int s) -> u32x4 {
      return row < rq.n ? *reinterpret_cast<const u32x4*>(qp + head * a.q_head + (2 * s + h) * P::EPC) : u32x4{0, 0, 0, 0};
    };
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      qf[s] = frag(hd0 + u, s);
      if (u == 0) sQ[qt][s * 64 + lane] = frag(hsel, s);
    }
  }
  float mu = -1e30f, l = 0.f;   // (no reference yet: the first weights overflow)
  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = zero16();
  const float sl2 = a.scale * LOG2E, neg_inv_scale = -1.f / a.scale;

  // loads: the wavefront's part (qt) of its head's K and V tile; those of head hd0's of the selector's K tile too
  const Rows rows(a, w.r, rq.t, qt, lane);
  const int64_t head_bytes = (int64_t)T::RB << a.pshift;
  const char* kp = static_cast<const char*>(a.k_pages) + (hd0 + u) * head_bytes;
  const char* vp = static_cast<const char*>(a.v_pages) + (hd0 + u) * head_bytes;
  const char* kselp = static_cast<const char*>(a.k_pages) + hsel * head_bytes;
  auto load_tile = [&](Tiles& B, const typename Rows::Place (&pl)[1]) {
    rows.load(B.k[u], kp, pl, qt);
    rows.load(B.v[u], vp, pl, qt);
  };
  auto load_sel = [&](char* S, const typename Rows::Place (&pl)[1]) {
    if (u == 0) rows.load(S, kselp, pl, qt);
  };
  const float* crow_p = carry + ((int64_t)((rq.first >> 5) + w.r + (min(rb, rq.n - 1) >> 5)) * a.G + g0) * carry_ld;
  auto carry_of = [&](int kt) { return kt >= 0 ? crow_p[min(kt * TILE + n, rq.t - 1)] : 0.f; };

  auto select = [&](int kt, const char* S, float entry, float* fw) {   // paged_fwd_kernel's
    const int kbase = kt * TILE;
    f32x16 l0 = zero16();
#pragma unroll
    for (int s = 0; s < NS; ++s) l0 = P::mma(sQ[qt][s * 64 + lane], T::row_frag(S, n, h, s), l0);
    f32x16 sel;
#pragma unroll
    for (int i = 0; i < 16; ++i) sel[i] = __builtin_amdgcn_fmed3f(-l0[i], -3.0e38f, 0.f);
    if (kbase + TILE - 1 >= qpos0 || kbase < a.exempt) {
      const int jk = kbase + n, thr = jk >= a.exempt ? jk - qpos0 - 4 * h : 32;
#pragma unroll
      for (int i = 0; i < 16; ++i) sel[i] = crow(i, 0) > thr ? sel[i] : 0.f;
    }
    float run = entry * neg_inv_scale;
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const Halves s4 = halves(((sel[4 * q4] + sel[4 * q4 + 1]) + sel[4 * q4 + 2]) + sel[4 * q4 + 3]);
      float p = (h == 0) ? run : run + s4.lo;
#pragma unroll
      for (int t2 = 0; t2 < 4; ++t2) {
        fw[crow(4 * q4 + t2, h) * LDF + n] = p;
        p += sel[4 * q4 + t2];
      }
      run = (run + s4.lo) + s4.hi;
    }
  };

  auto attend = [&](int kt, const Tiles& B, const float* F) __attribute__((always_inline)) {
    auto logits = [&]() __attribute__((always_inline)) {
      f32x16 lg;
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const float4 f4 = *reinterpret_cast<const float4*>(F + n * LDF + 8 * q4 + 4 * h);
        lg[4 * q4] = f4.x;
        lg[4 * q4 + 1] = f4.y;
        lg[4 * q4 + 2] = f4.z;
        lg[4 * q4 + 3] = f4.w;
      }
#pragma unroll
      for (int s = 0; s < NS; ++s) lg = P::mma(T::row_frag(B.k[u], n, h, s), qf[s], lg);
      if (kt * TILE + TILE - 1 > qpos0) {   // keys past a query
        const int thr = qpos0 + n - kt * TILE - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) lg[i] = crow(i, 0) <= thr ? lg[i] : -INFINITY;
      }
      return lg;
    };
    f32x16 lg = logits();
    u32x4 pf[2], pr[2];
    float psum;
    auto weights = [&]() __attribute__((always_inline)) {
      f32x16 p;
      float s = 0.f;
      const float ref = P::LIFT == 0.f ? -mu : P::LIFT - mu;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = fast_exp2(fmaf(lg[i], sl2, ref));
        s += p[i];
      }
      psum = s;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        pf[t] = P::pack(p, t);
        if constexpr (WIDE) pr[t] = P::rest(p, pf[t], t);
      }
    };
    weights();
    if (__builtin_expect(__any(!(psum <= P::BIG)), 0)) {
      if constexpr (WIDE) {   // the logits again: kept, they would not fit the registers beside the weights' halves
        __asm__ volatile("" ::: "memory");   // (nor would what they were made from)
        lg = logits();
      }
      float zmax = lg[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) zmax = fmaxf(zmax, lg[i]);
      const Halves zh = halves(zmax);
      const float m_new = fmaxf(mu, fmaxf(zh.lo, zh.hi) * sl2);
      const float alpha = fast_exp2(mu - m_new);
      mu = m_new;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
      weights();
    }
    l += psum;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const u32x4 v = T::value_frag(reinterpret_cast<const char*>(&B), HG * T::BYTES + u * T::BYTES, lane, db, s);
        o[db] = P::mma(v, pf[s], o[db]);
        if constexpr (WIDE) o[db] = P::mma(v, pr[s], o[db]);
      }
  };

  PagedLive tiles{nullptr, w.kt_hi, 0, 0};
  {
    const float* least = a.least + ((int64_t)((rq.first >> 5) + w.r + (w.row0 >> 5)) * a.G + g0) * a.reach_ld;
    if (a.least != nullptr && paged_live_worth(least, (rq.c + w.row0) / TILE)) {
      float bound[2];
      paged_live_bounds<P, D>(a, rq, w.r, rb + n, hd0 + u, qf, bound);
      if (lane == 0) {
        sBound[u][qt][0] = bound[0];
        sBound[u][qt][1] = bound[1];
      }
      __syncthreads();
      paged_live_mask<16, HG, 4>(a, w, sBound, least, a.kn + ((int64_t)w.r * a.H + hd0) * a.reach_ld, sMask);
      __syncthreads();
      tiles.mask = sMask;
    }
  }

  // the tile of the step (the t-th: t mod 2 names the buffers), and the next two; -1: none
  tiles.share(z, splits);
  int cur = tiles.next(), n1 = tiles.next(), n2 = tiles.next();
  int turn = (u - qt) & 3;   // tiles until the wavefront's next selection (0: the tile at hand)
  typename Rows::Place at1[1], at2[1];
  int pg[1];
  {
    typename Rows::Place at0[1];
    rows.pages_of(cur, pg);
    rows.places(cur, pg, at0);
    if (cur >= 0) {
      load_tile(sB0, at0);
      load_sel(sS0, at0);
    }
    rows.pages_of(n1, pg);
    rows.places(n1, pg, at1);
    if (n1 >= 0) load_sel(sS1, at1);
    rows.pages_of(n2, pg);
  }
  float entry = carry_of(n1);   // of the next tile, a step ahead (every wavefront: a branch would have the compiler wait)
  const float entry0 = carry_of(cur);
  wait_loads();
  __syncthreads();
  if (turn == 0 && cur >= 0 && cur < end) select(cur, sS0, entry0, sF0[qt]);
  turn = (turn - 1) & 3;
  __syncthreads();

  auto step = [&](auto odd_tag) __attribute__((always_inline)) {
    constexpr bool ODD = decltype(odd_tag)::value;
    rows.places(n2, pg, at2);
    if (n1 >= 0) load_tile(ODD ? sB0 : sB1, at1);
    if (n2 >= 0) load_sel(ODD ? sS1 : sS0, at2);
    const int n3 = tiles.next();
    rows.pages_of(n3, pg);
    const float entry2 = carry_of(n2);
    if (turn == 0) {
      // the next tile's F: first, and ahead of the SIMD's other wavefronts, which wait for it at the step's end
      __builtin_amdgcn_s_setprio(1);
      if (n1 >= 0 && n1 < end) select(n1, ODD ? sS0 : sS1, entry, ODD ? sF0[qt] : sF1[qt]);
    }
    if (cur < end) attend(cur, ODD ? sB1 : sB0, ODD ? sF1[qt] : sF0[qt]);
    __builtin_amdgcn_s_setprio(0);
    turn = (turn - 1) & 3;
    at1[0] = at2[0];
    entry = entry2;
    wait_loads();
    __syncthreads();
    cur = n1;
    n1 = n2;
    n2 = n3;
  };
  while (cur >= 0) {
    step(std::false_type{});
    if (cur < 0) break;
    step(std::true_type{});
  }
  paged_write<P, D>(a, w, rb + n, hd0 + u, z, mu, l, o, h, part_ml, part_o);
}

// The parts of every query joined: out = sum_z 2^(m_z - M) o_z / sum_z 2^(m_z - M) l_z (a part of no key: l_z = 0). A
// workgroup per row, a thread per four output columns; bound by latency, so four parts are loaded at a time, the first
// while the row's request is looked for (twelve parts of 2 to 9 rows of 16 requests: 8.6 us a part at a time, 5.0 so).
template <class P, int D>
__global__ __launch_bounds__(NTHREADS) void paged_join_kernel(PagedCall a, int splits, const float* __restrict__ part_ml,
                                                              const float* __restrict__ part_o) {
  typedef typename P::elem elem;
  constexpr int U = 4;
  const int row = blockIdx.x, items = a.H * (D / 4);
  float2 ml[U];
  float4 x[U];
  auto load = [&](int i, int z0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (z0 + u >= splits) continue;
      const int64_t at = ((int64_t)(z0 + u) * a.N + row) * a.H + i / (D / 4);
      ml[u] = *reinterpret_cast<const float2*>(part_ml + 2 * at);
      x[u] = *reinterpret_cast<const float4*>(part_o + at * D + 4 * (i % (D / 4)));
    }
  };
  if ((int)threadIdx.x < items) load(threadIdx.x, 0);
  const int r = find_request<true>(a.starts, a.R, row, 0);
  const PagedRequest rq = paged_request(a, r);
  const bool live = rq.live && row >= rq.first && row < rq.first + rq.n;
  if (live && a.ones && rq.n == 1) return;   // (paged_step_join's)
  elem* out = static_cast<elem*>(a.out) + (int64_t)row * a.H * D;
  for (int i = threadIdx.x; i < items; i += NTHREADS) {
    float M = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int z0 = 0; live && z0 < splits; z0 += U) {
      if (z0 > 0 || i >= NTHREADS) load(i, z0);
      float m_new = M;
#pragma unroll
      for (int u = 0; u < U; ++u) m_new = fmaxf(m_new, z0 + u < splits ? ml[u].x : -INFINITY);
      const float alpha = M == -INFINITY ? 0.f : fast_exp2(M - m_new);
      M = m_new;
      l *= alpha;
      acc = make_float4(acc.x * alpha, acc.y * alpha, acc.z * alpha, acc.w * alpha);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (z0 + u >= splits) continue;
        const float w = ml[u].x == -INFINITY ? 0.f : fast_exp2(ml[u].x - M);
        l = fmaf(w, ml[u].y, l);
        acc.x = fmaf(w, x[u].x, acc.x);
        acc.y = fmaf(w, x[u].y, acc.y);
        acc.z = fmaf(w, x[u].z, acc.z);
        acc.w = fmaf(w, x[u].w, acc.w);
      }
    }
    const float inv = live ? 1.f / l : 0.f;
    const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
    for (int e = 0; e < 4; ++e) out[4 * i + e] = P::to_elem(y[e]);
  }
}

// ---------------------------------------------------------------------------------------------
// One new token per request. Workgroup (chunk, head, request) reads its chunk of the head's cached keys and
// values once, 16 bytes per lane, as decode_partial_kernel does (logits reduced over the lanes of a row, one
// probability per lane, values added into each lane's column slice); a lane looks up the pages of its rows one step
// ahead. The selector head's workgroups write the new state rows to the workspace, which paged_step_join copies
// over the state after every head has read the old one.
template <class P, int D>
struct StepLayout {
  static constexpr int EPC = P::EPC, LPK = D / EPC, KPI = 64 / LPK;
  static constexpr int NR = 8 < LPK ? 8 : LPK;
  static constexpr int DUP = LPK / NR, STEP = KPI * NR;
};

template <class P, int D>
__global__ __launch_bounds__(NTHREADS) void paged_step_kernel(PagedCall a, float* __restrict__ pm, float* __restrict__ pl,
                                                              float* __restrict__ po, float* __restrict__ next_state,
                                                              int64_t next_ld, int chunk, int nchunk) {
  using L = StepLayout<P, D>;
  typedef typename P::elem elem;
  constexpr int EPC = L::EPC, LPK = L::LPK, KPI = L::KPI, NR = L::NR, DUP = L::DUP, STEP = L::STEP;
  union Row {
    u32x4 u;
    elem e[EPC];
  };
  __shared__ __align__(16) float sP[NWAVES][STEP];
  __shared__ float sPart[NWAVES][D + 2];

  const int cidx = blockIdx.x;
  const int r = blockIdx.z, hd = blockIdx.y;
  const PagedRequest rq = paged_request(a, r);
  if (!rq.live || rq.n != 1 || cidx * chunk >= rq.t) return;
  const int t = rq.t, per = a.H / a.G;
  const int64_t sg = (int64_t)r * a.G + hd / per;
  const bool selector = (hd % per) == 0;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int kq = lane / LPK, dc = lane % LPK;
  const int ri = dc / DUP;
  const bool owner = dc % DUP == 0;
  const int wkeys = chunk / NWAVES;
  const int kw0 = cidx * chunk + wave * wkeys, kw_end = min(kw0 + wkeys, t);
  const float* selrow = a.selected + sg * a.state_ld;
  float* nextrow = next_state + sg * next_ld;
  const int* trow = a.table + r * a.table_ld;
  const int pmask = (1 << a.pshift) - 1;

  float qf[EPC];
  {
    Row qq;
    qq.u = *reinterpret_cast<const u32x4*>(static_cast<const elem*>(a.q) + rq.first * a.q_token + hd * a.q_head + EPC * dc);
#pragma unroll
    for (int e = 0; e < EPC; ++e) qf[e] = P::to_float(qq.e[e]) * a.scale;
  }
  float m = -INFINITY, l = 0.f, o[EPC];
#pragma unroll
  for (int e = 0; e < EPC; ++e) o[e] = 0.f;

  auto lookup = [&](int kw, int (&pg)[NR]) {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int j = kw + i * KPI + kq;
      pg[i] = j < kw_end ? trow[j >> a.pshift] : -1;
    }
  };
  int pg[NR];
  lookup(kw0, pg);
  for (int kw = kw0; kw < kw_end; kw += STEP) {
    Row kr[NR], vr[NR];
    int64_t off[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int j = kw + i * KPI + kq;
      const bool ok = (uint32_t)pg[i] < (uint32_t)a.pages;
      off[i] = ok ? ((((int64_t)pg[i] * a.H + hd) << a.pshift) + (j & pmask)) * D + EPC * dc : -1;
    }
#pragma unroll
    for (int i = 0; i < NR; ++i)
      kr[i].u = off[i] >= 0 ? *reinterpret_cast<const u32x4*>(static_cast<const elem*>(a.k_pages) + off[i]) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NR; ++i)
      vr[i].u = off[i] >= 0 ? *reinterpret_cast<const u32x4*>(static_cast<const elem*>(a.v_pages) + off[i]) : u32x4{0, 0, 0, 0};
    const int j = kw + ri * KPI + kq;
    const bool jok = j < kw_end;
    const float sel = j < t - 1 && jok ? selrow[j] : 0.f;
    if (kw + STEP < kw_end) lookup(kw + STEP, pg);
    float z1[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < EPC; ++e) s = fmaf(qf[e], P::to_float(kr[i].e[e]), s);
      z1[i] = s;
    }
#pragma unroll
    for (int st = 1; st < NR; st <<= 1) {   // reduce-scatter over the row's lanes (decode_partial_kernel)
      const int half = NR / (2 * st), s = LPK / (2 * st);
      const uint32_t up = (lane & s) ? 0xffffffffu : 0u;
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const uint32_t lo = __float_as_uint(z1[i]), hi = __float_as_uint(z1[i + half]);
        const float send = __uint_as_float((lo & up) | (hi & ~up));
        const float keep = __uint_as_float((hi & up) | (lo & ~up));
        z1[i] = keep + __shfl_xor(send, s);
      }
    }
#pragma unroll
    for (int s = DUP / 2; s >= 1; s >>= 1) z1[0] += __shfl_xor(z1[0], s);
    const float raw = z1[0];
    if (selector && owner && jok) nextrow[j] = sel + (j >= a.exempt && j < t - 1 ? fmaxf(raw, 0.f) : 0.f);
    const float z = jok ? (raw - sel) * LOG2E : -INFINITY;
    const float m_new = fmaxf(m, wave_max(z));
    const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m - m_new);
    const float p = z != -INFINITY ? fast_exp2(z - m_new) : 0.f;   // (not where no key has weight; NaN where only NaNs are)
    l = fmaf(l, alpha, owner ? p : 0.f);
#pragma unroll
    for (int e = 0; e < EPC; ++e) o[e] *= alpha;
    m = m_new;
    if (owner) sP[wave][kq * NR + ri] = p;
    lds_wave_sync();
    float pr[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) pr[i] = sP[wave][kq * NR + i];
    lds_wave_sync();
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < EPC; ++e) o[e] = fmaf(pr[i], P::to_float(vr[i].e[e]), o[e]);
  }
  l = wave_sum(l);
#pragma unroll
  for (int sh = LPK; sh < 64; sh <<= 1)
#pragma unroll
    for (int e = 0; e < EPC; ++e) o[e] += __shfl_xor(o[e], sh);
  if (kq == 0) {
#pragma unroll
    for (int e = 0; e < EPC; ++e) sPart[wave][2 + EPC * dc + e] = o[e];
  }
  if (lane == 0) {
    sPart[wave][0] = m;
    sPart[wave][1] = l;
  }
  __syncthreads();
  if (wave == 0) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < NWAVES; ++w) mx = fmaxf(mx, sPart[w][0]);
    const int64_t slot = ((int64_t)r * a.H + hd) * nchunk + cidx;
    for (int c = lane; c < D + 2; c += 64) {
      float acc = 0.f;
#pragma unroll
      for (int w = 0; w < NWAVES; ++w) {
        const float wt = sPart[w][0] == -INFINITY ? 0.f : fast_exp2(sPart[w][0] - mx);
        acc = fmaf(wt, sPart[w][c], acc);
      }
      if (c == 0) pm[slot] = mx;
      else if (c == 1) pl[slot] = acc;
      else po[slot * D + c - 2] = acc;
    }
  }
}

// Block (r, head) for the first R * H blocks: the request's chunks' partials joined; without `ones` (every row is here) also
// zeros for the rows of requests left out, and for those before the first request and behind the last, each block every R-th of them. Blocks
// from there on: the new state rows, `sblocks` blocks of 1024 keys each.
template <class P, int D>
__global__ __launch_bounds__(NTHREADS) void paged_step_join_kernel(PagedCall a, const float* __restrict__ pm,
                                                                   const float* __restrict__ pl, const float* __restrict__ po,
                                                                   const float* __restrict__ next_state, int64_t next_ld,
                                                                   int chunk, int nchunk, int sblocks) {
  typedef typename P::elem elem;
  constexpr int QPP = D / 4, SLOTS = NTHREADS / QPP;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int64_t out_blocks = (int64_t)a.R * a.H;
  if (blockIdx.x >= out_blocks) {
    const int64_t s = blockIdx.x - out_blocks;
    const int64_t sg = s / sblocks;
    const int j0 = (int)(s % sblocks) * (4 * NTHREADS);
    const PagedRequest rq = paged_request(a, (int)(sg / a.G));
    if (!rq.live || rq.n != 1) return;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + u * NTHREADS + tid;
      if (j < rq.t) a.selected[sg * a.state_ld + j] = next_state[sg * next_ld + j];
    }
    return;
  }
  __shared__ float sRed[NWAVES][2];
  __shared__ float4 sO[NWAVES][QPP];
  const int r = (int)(blockIdx.x / a.H), hd = (int)(blockIdx.x % a.H);
  const PagedRequest rq = paged_request(a, r);
  auto row_of = [&](int row) { return static_cast<elem*>(a.out) + ((int64_t)row * a.H + hd) * D; };
  if (!a.ones) {
    if (tid < D) {
      for (int64_t row = max(a.starts[a.R], 0) + (int64_t)r; row < a.N; row += a.R) row_of((int)row)[tid] = P::to_elem(0.f);
      for (int64_t row = r; row < min(a.starts[0], a.N); row += a.R) row_of((int)row)[tid] = P::to_elem(0.f);
      if (!rq.live)
        for (int i = 0; i < rq.n; ++i) row_of(rq.first + i)[tid] = P::to_elem(0.f);
    }
  }
  if (!rq.live || rq.n != 1) return;
  elem* out = row_of(rq.first);
  const int nparts = (rq.t + chunk - 1) / chunk;
  const int64_t at = ((int64_t)r * a.H + hd) * nchunk;
  float mx = -INFINITY;
  for (int i = tid; i < nparts; i += NTHREADS) mx = fmaxf(mx, pm[at + i]);
  mx = wave_max(mx);
  if (lane == 0) sRed[wave][0] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(sRed[0][0], sRed[1][0]), fmaxf(sRed[2][0], sRed[3][0]));
  float l = 0.f;
  for (int i = tid; i < nparts; i += NTHREADS) l = fmaf(fast_exp2(pm[at + i] - mx), pl[at + i], l);
  l = wave_sum(l);
  if (lane == 0) sRed[wave][1] = l;
  const int slot = tid / QPP, cq = tid % QPP;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = slot; i < nparts; i += SLOTS) {
    const float w = fast_exp2(pm[at + i] - mx);
    const float4 x = *reinterpret_cast<const float4*>(po + (at + i) * D + 4 * cq);
    acc.x = fmaf(w, x.x, acc.x);
    acc.y = fmaf(w, x.y, acc.y);
    acc.z = fmaf(w, x.z, acc.z);
    acc.w = fmaf(w, x.w, acc.w);
  }
#pragma unroll
  for (int sh = QPP; sh < 64; sh <<= 1) {
    acc.x += __shfl_xor(acc.x, sh);
    acc.y += __shfl_xor(acc.y, sh);
    acc.z += __shfl_xor(acc.z, sh);
    acc.w += __shfl_xor(acc.w, sh);
  }
  if (lane < QPP) sO[wave][lane] = acc;
  __syncthreads();
  if (tid < QPP) {
    l = (sRed[0][1] + sRed[1][1]) + (sRed[2][1] + sRed[3][1]);
    const float inv = 1.f / l;
    float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NWAVES; ++w) {
      y[0] += sO[w][tid].x;
      y[1] += sO[w][tid].y;
      y[2] += sO[w][tid].z;
      y[3] += sO[w][tid].w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) out[4 * tid + e] = P::to_elem(y[e] * inv);
  }
}

// ---------------------------------------------------------------------------------------------
// Launches (sizes: paged_shape, sa_host.h).
inline PagedCall paged_call(const PagedLaunch& c) {
  PagedCall a{};
  a.q = c.q;
  a.k_pages = c.k_pages;
  a.v_pages = c.v_pages;
  a.out = c.out;
  a.table = c.table;
  a.lengths = c.lengths;
  a.starts = c.starts;
  a.selected = c.selected;
  a.q_token = c.q_token;
  a.q_head = c.q_head;
  a.table_ld = c.table_ld;
  a.state_ld = c.state_ld;
  a.R = (int)c.R;
  a.N = (int)c.N;
  a.H = (int)c.H;
  a.G = (int)c.G;
  a.pages = (int)c.pages;
  a.pshift = c.pshift;
  a.max_new = (int)c.max_new;
  a.max_len = (int)c.max_len;
  a.scale = c.scale;
  a.exempt = c.exempt;
  return a;
}

template <class P, int D, int HG, int NW, bool WHOLE, bool WIDE>
void launch_paged_tiles(const PagedCall& a, const PagedShape& s, const float* carry, float* ml, float* o, hipStream_t st) {
  const int64_t tiles = (int64_t)(a.N >> (NW == 4 ? 7 : 5)) + a.R;
  hipLaunchKernelGGL((paged_fwd_kernel<P, D, HG, NW, WHOLE, WIDE>), tile_grid((int64_t)a.H / HG * s.splits, tiles), dim3(NW * 64), 0,
                     st, a, carry, s.ld, s.splits, ml, o);
}

template <class P, int D, bool WIDE>
void launch_paged_fwd(const PagedCall& a, const PagedShape& s, const float* carry, float* ml, float* o, hipStream_t st) {
  const bool whole = a.G == a.H;
  if constexpr (sizeof(typename P::elem) == 2 && D == 64) {
    if (s.hg == 4)
      hipLaunchKernelGGL((paged_fwd4_kernel<P, WIDE>), tile_grid((int64_t)a.H / 4 * s.splits, (a.N >> 7) + a.R), dim3(1024), 0, st, a,
                         carry, s.ld, s.splits, ml, o);
  }
  if constexpr (sizeof(typename P::elem) == 2 && D <= 64) {
    if (s.hg == 2) {
      if (s.nw == 4) launch_paged_tiles<P, D, 2, 4, false, WIDE>(a, s, carry, ml, o, st);
      else launch_paged_tiles<P, D, 2, 1, false, WIDE>(a, s, carry, ml, o, st);
    }
  }
  if (s.hg == 1) {
    if (s.nw == 4) {
      if (whole) launch_paged_tiles<P, D, 1, 4, true, WIDE>(a, s, carry, ml, o, st);
      else launch_paged_tiles<P, D, 1, 4, false, WIDE>(a, s, carry, ml, o, st);
    } else {
      if (whole) launch_paged_tiles<P, D, 1, 1, true, WIDE>(a, s, carry, ml, o, st);
      else launch_paged_tiles<P, D, 1, 1, false, WIDE>(a, s, carry, ml, o, st);
    }
  }
}

template <class P, int D>
void launch_paged_step(const PagedCall& a, const PagedShape& s, char* ws, hipStream_t st) {
  auto at = [&](int64_t off) { return reinterpret_cast<float*>(ws + off); };
  float *pm = at(s.step_m), *pl = at(s.step_l), *po = at(s.step_o), *next = at(s.step_state);
  const int nchunk = (int)cdiv(a.max_len, s.chunk), sblocks = (int)cdiv(a.max_len, 4 * NTHREADS);
  {
    TimedLaunch timed(SA_KERNEL_DECODE, st);
    hipLaunchKernelGGL((paged_step_kernel<P, D>), dim3((unsigned)nchunk, (unsigned)a.H, (unsigned)a.R), dim3(NTHREADS), 0, st, a, pm, pl,
                       po, next, s.ld, s.chunk, nchunk);
  }
  const int64_t blocks = (int64_t)a.R * a.H + (int64_t)a.R * a.G * sblocks;
  hipLaunchKernelGGL((paged_step_join_kernel<P, D>), dim3((unsigned)blocks), dim3(NTHREADS), 0, st, a, pm, pl, po, next, s.ld, s.chunk,
                     nchunk, sblocks);
}

template <class P, int D>
int paged_launch(const PagedLaunch& c) {
  PagedCall a = paged_call(c);
  const PagedShape s = paged_shape(c.R, c.N, c.H, c.G, D, sizeof(typename P::elem), c.max_new, c.max_len);
  char* ws = static_cast<char*>(c.ws);
  auto at = [&](int64_t off) { return reinterpret_cast<float*>(ws + off); };
  a.ones = s.several && s.ones;
  if (s.ones) launch_paged_step<P, D>(a, s, ws, c.st);
  if (!s.several) return launch_status();
  if (s.reach) {
    a.least = at(s.least);
    a.kn = at(s.kn);
    a.reach_ld = s.ld / TILE;
  }
  a.segments = s.segments;
  a.seg_tiles = s.seg_tiles;
  a.totals = s.segments > 1 ? at(s.totals) : nullptr;
  float *carry = at(s.carry), *ml = s.splits > 1 ? at(s.m) : nullptr, *o = s.splits > 1 ? at(s.o) : nullptr;
  {
    TimedLaunch timed(SA_KERNEL_SELECTION, c.st);
    hipLaunchKernelGGL((paged_carry_kernel<P, D>), dim3((unsigned)(s.carry_blocks * s.segments), (unsigned)a.G, (unsigned)a.R),
                       dim3(NTHREADS), 0, c.st, a, carry, s.ld);
    if (s.segments > 1)
      hipLaunchKernelGGL((paged_carry_join_kernel<P, D>), dim3((unsigned)cdiv(a.max_len, NTHREADS),
                         (unsigned)(2 + cdiv(cdiv(a.max_new, TILE) - s.seg_tiles, SEG_PART)), (unsigned)(a.R * a.G)), dim3(NTHREADS), 0,
                         c.st, a, carry, s.ld);
  }
  {
    TimedLaunch timed(SA_KERNEL_FORWARD, c.st);
    if constexpr (sizeof(typename P::elem) == 2) {
      if (c.wide) launch_paged_fwd<P, D, true>(a, s, carry, ml, o, c.st);
      else launch_paged_fwd<P, D, false>(a, s, carry, ml, o, c.st);
    } else {
      launch_paged_fwd<P, D, false>(a, s, carry, ml, o, c.st);
    }
  }
  if (s.splits > 1)
    hipLaunchKernelGGL((paged_join_kernel<P, D>), dim3((unsigned)a.N), dim3(NTHREADS), 0, c.st, a, s.splits, ml, o);
  return launch_status();
}

template <class P>
int paged_entry(const PagedLaunch& c) {
  if (c.head_dim == 16) return paged_launch<P, 16>(c);
  if (c.head_dim == 32) return paged_launch<P, 32>(c);
  if (c.head_dim == 64) return paged_launch<P, 64>(c);
  return paged_launch<P, 128>(c);
}

}  // namespace
