// Softmax cross entropy of a large vocabulary from hidden states and the output head's matrix (include/sa.h:
// sa_linear_xent), without the logits kept.
//
//   l[i, v] = x_i . W_v;   lse_i = log sum_v exp l[i, v];   loss_i = lse_i - l[i, t_i]
//   G[i, v] = exp(l[i, v] - lse_i) - [v = t_i];   dx_i = g_i sum_v G[i, v] W_v;   dW_v = sum_i g_i G[i, v] x_i
//
// Tokens whose target is ignored are taken out first (xent_rows: the kept tokens' numbers, in order, and how many; the
// count stays on the device and bounds the launches that follow), so they cost nothing and nothing in their rows (a NaN, an
// infinity) reaches a result.
//
//   xent_rows, xent_gather   the kept tokens' rows, in the products' type, padded to whole stages of the contraction
//   xent_logits              logits of a tile (vocabulary x tokens: a lane holds one token's, so its maximum and sum are taken in
//                            registers); a token's maximum, sum and target logit per tile of the vocabulary go to the workspace
//   xent_join, xent_sum      the tiles' statistics joined: lse, loss; the mean or the sum
//   xent_factors             backward: what the sums and G are multiplied by
//   xent_pass                a piece of the vocabulary at a time: the logits computed again, and G of them; beside it the products of
//                            the piece before, dX += G W_piece (fp32 in the workspace across the pieces), dW_piece = G^T X
//   xent_finish              the parts of a split contraction added, scaled, converted
//
// All products run through one tile loop on matrix instructions with fp32 accumulation (Mainloop). Statistics, lse and losses are
// fp32. Both passes take the logits from the same operands, so that the probabilities are the forward's whatever the rows hold. G is rounded to
// 11 bits (few tokens' with fp16 operands to 22, in two numbers): it is held in fp16 at 2^14 times its size (a vocabulary's probabilities lie below
// that type's normal range). Its products with bf16
// operands hold these in fp16 too, times the power of two that brings their largest to 2^14: exactly, but for numbers 2^31 times smaller
// than that, which are off by 2^-39 of it, and at the same rate. (With G in bf16 the gradients' error was 1.4 to 1.6 times that of their own
// rounding; so it is that rounding's.) The factors and a common g are applied to the fp32 sums. Tokens' own g_i (reduction none): G_i takes
// g_i over the power of two below it before it is rounded, the sum dx_i that power; dW sums over tokens, so it reads a copy of x whose rows have their
// powers (16-bit types; fp32 puts all of g_i into G_i).
//
// Bound by the matrix units and, with all of them busy, by power (1.8-1.9 GHz). Measured, 16384 tokens x 50304 x 768 bf16: the forward pass's products
// 1.2-1.4 ms (0.9-1.05 PFLOP/s with the statistics; torch's own product of that shape 1.13), the backward's eight passes 0.48-0.53
// each (three products: 0.95-1.0 PFLOP/s), all else 0.15. Few tokens: by the weight's way from HBM (8 tokens 15.8-20 us for 77 MB).

#pragma once

#include <math.h>

#include <type_traits>

#include "sa_lm.h"

namespace sa_host {

struct XentCall {
  const void *x, *w;            // the caller's rows
  const int64_t* targets;
  const float* dloss;
  float *loss, *lse;            // lse: the kept tokens' largest logits, then (from tokens on) 1 / sum of exp beside those; null where no
                                // backward pass follows
  int* rows;                    // [0] kept tokens, [64 ..] largest magnitudes (MAXIMA of weight, of x), [ROWS_HEAD ..] the kept tokens'
                                // numbers, [ROWS_HEAD + tokens ..] each token's place among them or -1
  void *dx, *dw;
  void* ws;
  int64_t x_ld, w_ld, tokens, vocab, width, ignore;
  int x_t, w_t, reduction;
  int cus;
  hipStream_t st;
};
int64_t xent_bytes_bf16(const XentCall& c, bool backward);
int64_t xent_bytes_f16(const XentCall& c, bool backward);
int64_t xent_bytes_f32(const XentCall& c, bool backward);
int xent_bf16(const XentCall& c, bool backward);
int xent_f16(const XentCall& c, bool backward);
int xent_f32(const XentCall& c, bool backward);

}  // namespace sa_host

namespace {

typedef float f32x16 __attribute__((__vector_size__(16 * sizeof(float))));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((__vector_size__(8 * sizeof(bf16_t))));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_void_ptr;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int MAXIMA = 512;                    // workgroups that look for the largest magnitude of a matrix
constexpr int ROWS_HEAD = 64 + 2 * MAXIMA;     // ints before the kept tokens' numbers
static_assert(ROWS_HEAD == SA_XENT_ROWS, "as the header says");

// ---------------------------------------------------------------------------------------------
// Operand types. A lane's operand of one step is 16 bytes of its row (lanes 0-31 the even, 32-63 the odd 16 bytes): one instruction for
// 16-bit types, four for fp32, each of which contracts element e of both halves' four (the order of a contraction is
// free as long as both operands have the same).

struct XF16;
struct XBF16 {
  typedef uint16_t elem;
  typedef XF16 Back;   // what G is held in, and what it is multiplied with
  static constexpr int CODE = SA_DTYPE_BF16;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
struct XF16 {
  typedef uint16_t elem;
  typedef XF16 Back;
  static constexpr int CODE = SA_DTYPE_F16;
  static constexpr float LIFT = 16384.f;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
struct XF32 {
  typedef float elem;
  typedef XF32 Back;
  static constexpr int CODE = SA_DTYPE_F32;
  static constexpr float LIFT = 1.f;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
// the same number in every lane, as a value the compiler keeps in a scalar register (after a division it would not know)
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ lds_void_ptr lds_at(const void* p) { return (lds_void_ptr)(uint32_t)(uintptr_t)p; }
// element i of a 32 x 32 accumulator: column lane % 32, row acc_row(i, lane / 32)
__device__ __forceinline__ constexpr int acc_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }
// Loads past `bytes` give zero; so does any at PAST or behind it, however much there is (what a tile means to read lies below).
constexpr int PAST = 0x7fffff00;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* p, int64_t bytes) {
  const int64_t most = PAST;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)(bytes < 0 ? 0 : bytes < most ? bytes : most), 0x00020000);
}

// ---------------------------------------------------------------------------------------------
// One operand of a tile: EDGE rows (or columns) of the result, KB = 64 bytes of the contraction per stage.
//
// Plain: the matrix has the contraction along its rows. A stage holds EDGE rows of 64 bytes; the 16-byte chunk c of row r sits at
// chunk c ^ (r / 4 mod 4): a fragment read takes one chunk of 16 rows a pass over 64 banks, and the four rows that share banks then
// take four chunks.
// Turned (TR): the matrix has the contraction down its columns (K, EDGE). A stage holds 64 / size rows of EDGE elements, and
// the fragments are read transposed: 16-bit types by ds_read_b64_tr_b16 (lane i of 16 gets as element t the element i % 4 of
// the 8 bytes that lane 4t + i/4 addresses: two groups of 16 read 64 bytes of each of four rows a pass, which sit at chunk c ^ 4 (r
// mod 4), in banks of their own), fp32 by one 4-byte read per instruction (32 neighbours of a row).
// (Measured on the bank-conflict counter: none. With chunks at c ^ (r mod 8) and c ^ 2 (r mod 4) every read took twice as long.)
//
// The loads go from memory straight into LDS: one instruction fills 64 consecutive 16-byte slots, and each lane fetches the
// chunk that belongs in its slot. Rows past the resource's end read as zeros.
constexpr int KB = 64;

template <class OP, int EDGE, bool TR, int WAVES>
struct Operand {
  static constexpr int ES = sizeof(typename OP::elem);
  static constexpr int BYTES = EDGE * KB;
  static constexpr int BK = KB / ES;
  static constexpr int ROW = TR ? EDGE * ES : KB;               // bytes of a staged row
  static constexpr int LANES = ROW / 16 < 64 ? ROW / 16 : 64;   // lanes of an instruction on one row
  static constexpr int RPI = 64 / LANES;                        // rows of an instruction
  static constexpr int IPR = ROW / (16 * LANES);                // instructions of a row
  static constexpr int LOADS = BYTES / 1024;                    // instructions of a stage
  static constexpr int PER = LOADS / WAVES;                     // and of a wavefront
  static_assert(LOADS % WAVES == 0, "whole loads per wavefront");

  __amdgpu_buffer_rsrc_t rs;
  int lane_off, ld;   // bytes

  // p: the tile's first row (plain) or column (turned), at the contraction's start; bytes: what may be read from there
  __device__ __forceinline__ void open(const void* p, int64_t bytes, int64_t ld_elems) {
    rs = resource(p, bytes);
    ld = (int)(ld_elems * ES);
    const int lane = threadIdx.x & 63;
    const int r = lane / LANES, pos = lane % LANES;
    lane_off = r * ld + (TR ? pos : pos ^ ((r >> 2) & 3)) * 16;   // (the turned swizzle: below)
  }
  // stage k of the contraction into `to` (the wavefront's share), zeros from stage `last` on
  __device__ __forceinline__ void load(uint8_t* to, int k, int last, int wave) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int n = wave * PER + i;
      int voff = lane_off, soff;
      if constexpr (!TR) {
        soff = n * RPI * ld + k * KB;
      } else {
        const int r0 = (n / IPR) * RPI;   // first row of the instruction
        if constexpr (ES == 2) {
          const int pos = lane % LANES + (n % IPR) * LANES, r = r0 + lane / LANES;
          voff = (lane / LANES) * ld + ((pos ^ ((r & 3) << 2)) * 16);
        } else {
          voff = lane_off + (n % IPR) * 1024;
        }
        soff = (k * BK + r0) * ld;
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds_at(to + 1024 * n), 16, voff, k < last ? soff : PAST, 0, 0);
    }
  }
  // the fragment of step j (two per stage) of rows (columns) first .. first + 31
  static __device__ __forceinline__ u32x4 frag(const uint8_t* t, int first, int j) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    if constexpr (!TR) {
      const int r = first + (lane & 31);
      return *reinterpret_cast<const u32x4*>(t + r * KB + (((2 * j + h) ^ ((lane >> 2) & 3)) << 4));
    } else if constexpr (ES == 2) {
      const int g = lane >> 4, k = lane & 15;
      u32x4 f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = 16 * j + 8 * (g >> 1) + 4 * hf + (k >> 2);
        const int c = (first >> 3) + 2 * (g & 1) + ((k & 3) >> 1);
        typedef __attribute__((address_space(3))) short4v* lds_s4;
        // (one sum: after a chain of additions the compiler no longer knows which variable is read, and waits for all loads in flight)
        const int at = r * ROW + ((c ^ ((r & 3) << 2)) << 4) + 8 * (k & 1);
        const short4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(t + at));
        const uint2 u = __builtin_bit_cast(uint2, v);
        f[2 * hf] = u.x;
        f[2 * hf + 1] = u.y;
      }
      return f;
    } else {
      u32x4 f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = *reinterpret_cast<const uint32_t*>(t + (8 * j + 4 * h + e) * ROW + (first + (lane & 31)) * 4);
      return f;
    }
  }
};

template <int A_BYTES, int B_BYTES>
struct StageOf {
  alignas(1024) uint8_t a[A_BYTES];
  alignas(1024) uint8_t b[B_BYTES];
};

// A tile of WM x WN wavefronts, each TM x TN squares of 32: acc[a][b] += A B^T over `stages` of the contraction. A ring of four stages in
// LDS, in variables of their own (one array indexed by the stage makes the compiler wait for the loads in flight before it
// reads): while one is multiplied, the loads of the next three are under way, since a stage of the larger tiles (32 KB, 1024
// cycles of the matrix units) is over before memory has answered.
template <class OP, int WM_, int WN_, int TM_, int TN_, bool TRA, bool TRB>
struct Mainloop {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int BM = WM * TM * 32, BN = WN * TN * 32;
  static constexpr bool TWO_NUMBERS = std::is_same<OP, XF16>::value;   // (halves_of)
  typedef Operand<OP, BM, TRA, WAVES> A;
  typedef Operand<OP, BN, TRB, WAVES> B;
  static constexpr int BK = A::BK, LOADS = A::PER + B::PER;
  typedef StageOf<A::BYTES, B::BYTES> Stage;
  struct Frags {
    u32x4 a[TM], b[TN];
  };
  f32x16 acc[TM][TN];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;
  }
  static __device__ __forceinline__ void read(Frags& f, const Stage& s, int j, int wm, int wn) {
#pragma unroll
    for (int a = 0; a < TM; ++a) f.a[a] = A::frag(s.a, (wm * TM + a) * 32, j);
#pragma unroll
    for (int b = 0; b < TN; ++b) f.b[b] = B::frag(s.b, (wn * TN + b) * 32, j);
    __builtin_amdgcn_sched_barrier(0);   // (the reads go out before the products that hide them)
  }
  __device__ __forceinline__ void multiply(const Frags& f) {
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b) acc[a][b] = OP::mma(f.a[a], f.b[b], acc[a][b]);
    __builtin_amdgcn_sched_barrier(0);
  }
  // everyone has read what they wanted, and all but everyone's last PENDING loads are there
  template <int PENDING>
  static __device__ __forceinline__ void arrive() {
    __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PENDING) : "memory");
  }
  static __device__ __forceinline__ void load(const A& oa, const B& ob, Stage& s, int k, int stages, int wave) {
    oa.load(s.a, k, stages, wave);
    ob.load(s.b, k, stages, wave);
  }
  // The products of stage k, in `now`, whose first step's operands are in f0. Each step's are read while the products of the step before
  // run, across the barrier too: the last step's are in registers by then, and `now` takes stage k + 4.
  __device__ __forceinline__ void stage(const A& oa, const B& ob, Stage& now, const Stage& next, int k, int stages, Frags& f0, Frags& f1,
                                        int wave, int wm, int wn) {
    read(f1, now, 1, wm, wn);
    multiply(f0);
    arrive<2 * LOADS>();
    load(oa, ob, now, k + 4, stages, wave);
    read(f0, next, 0, wm, wn);
    multiply(f1);
  }
  // (Stages past the last are of zeros: one way out of the loop keeps the sums in the registers they are in.)
  __device__ __forceinline__ void run(const A& oa, const B& ob, Stage& s0, Stage& s1, Stage& s2, Stage& s3, int stages) {
    const int wave = wave_index(), wm = wave / WN, wn = wave % WN;
    clear();
    load(oa, ob, s0, 0, stages, wave);
    load(oa, ob, s1, 1, stages, wave);
    load(oa, ob, s2, 2, stages, wave);
    load(oa, ob, s3, 3, stages, wave);
    arrive<3 * LOADS>();
    Frags f0, f1;
    read(f0, s0, 0, wm, wn);
    for (int k = 0; k < stages; k += 4) {
      stage(oa, ob, s0, s1, k, stages, f0, f1, wave, wm, wn);
      stage(oa, ob, s1, s2, k + 1, stages, f0, f1, wave, wm, wn);
      stage(oa, ob, s2, s3, k + 2, stages, f0, f1, wave, wm, wn);
      stage(oa, ob, s3, s0, k + 3, stages, f0, f1, wave, wm, wn);
    }
    arrive<0>();   // (the last loads, of zeros, are in: the LDS may be used)
  }
};

// The tile of workgroup `id` among mt x nt: every XCD (workgroups go to the eight in turn) takes a contiguous run of tiles, in
// bands of 8 along the first axis, so that the tiles that run together share rows in its L2. False past the last.
__device__ __forceinline__ bool tile_of(int64_t id, int mt, int nt, int& m, int& n) {
  const int64_t total = (int64_t)mt * nt, per = (total + 7) / 8;
  const int64_t t = (id & 7) * per + (id >> 3);
  if ((id >> 3) >= per || t >= total) return false;
  const int band = (int)(t / (8 * (int64_t)nt));
  const int high = min(8, mt - band * 8);
  const int in = (int)(t - (int64_t)band * 8 * nt);
  n = uniform(in / high);
  m = uniform(band * 8 + in - n * high);
  return true;
}
inline int64_t tiles_grid(int64_t mt, int64_t nt) { return 8 * cdiv(mt * nt, 8); }

// ---------------------------------------------------------------------------------------------
// The larger of two magnitudes, x's if it is a number: an infinity or a NaN has no say in what unit the others are held in.
__device__ __forceinline__ float larger(float most, float x) {
  const float a = fabsf(x);
  return a < INFINITY ? fmaxf(most, a) : most;
}
// The largest of the workgroup's values, as the workgroup's own number of `maxima`.
__device__ __forceinline__ void put_maximum(float most, float (&acc)[16], int* maxima, int at) {
#pragma unroll
  for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  if ((threadIdx.x & 63) == 0) acc[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < (int)blockDim.x / 64; ++w) most = fmaxf(most, acc[w]);
  maxima[at] = (int)__float_as_uint(most);
}

// The kept tokens, in order: the first workgroup, 8192 tokens a round. The others (a backward pass of bf16 operands follows) look for the
// largest magnitude of the weight meanwhile.

struct Matrix {
  const void* p;
  int64_t ld, rows;
  int width, dtype;
};
__global__ __launch_bounds__(1024) void xent_rows_kernel(const int64_t* targets, int64_t tokens, int64_t ignore, int* rows, float* each,
                                                         Matrix w) {
  __shared__ int count[16];
  __shared__ float acc[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x > 0) {
    // rows that follow each other are one; else a wavefront takes rows in turn
    const bool quads = (uintptr_t)w.p % (w.dtype == SA_DTYPE_F32 ? 16 : 8) == 0 && w.ld % 4 == 0 && w.width % 4 == 0;
    const bool flat = quads && w.ld == w.width;
    constexpr int64_t RUN = 2048;   // elements of a flat matrix's row: a wavefront's loads in flight
    const int64_t elements = w.rows * w.width, n = flat ? (elements + RUN - 1) / RUN : w.rows;
    float most = 0.f;
    constexpr int AHEAD = 8;   // loads in flight
    for (int64_t i = (int64_t)(blockIdx.x - 1) * 16 + wave; i < n; i += MAXIMA * 16) {
      const void* row = row_of(w.p, flat ? i * RUN : i, flat ? 1 : w.ld, w.dtype);
      const int width = flat ? (int)min(RUN, elements - i * RUN) : w.width;
      for (int e0 = 0; e0 < width; e0 += 256 * AHEAD) {
        Quad q[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int e = e0 + 256 * u + 4 * lane;
          q[u] = quads ? fetch<true>(row, w.dtype, e, 1, width) : fetch<false>(row, w.dtype, e, 1, width);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          float x[4];
          if (quads) numbers<true>(q[u], w.dtype, x);
          else numbers<false>(q[u], w.dtype, x);
#pragma unroll
          for (int j = 0; j < 4; ++j) most = larger(most, x[j]);
        }
      }
    }
    put_maximum(most, acc, rows + 64, blockIdx.x - 1);
    return;
  }
  int base = 0;
  for (int64_t i0 = 0; i0 < tokens; i0 += 8192) {
    bool kept[8];
    int n = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t i = i0 + wave * 512 + u * 64 + lane;
      kept[u] = i < tokens && targets[i] != ignore;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) n += (int)__popcll(__ballot(kept[u]));
    __syncthreads();
    if (lane == 0) count[wave] = n;
    __syncthreads();
    int at = base;
    for (int w = 0; w < 16; ++w) {
      at += w < wave ? count[w] : 0;
      base += count[w];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t i = i0 + wave * 512 + u * 64 + lane;
      const uint64_t mask = __ballot(kept[u]);
      const int mine = at + (int)__popcll(mask & (((uint64_t)1 << lane) - 1));
      if (kept[u]) rows[ROWS_HEAD + mine] = (int)i;
      if (i < tokens) {
        rows[ROWS_HEAD + tokens + i] = kept[u] ? mine : -1;
        if (each && !kept[u]) each[i] = 0.f;
      }
      at += (int)__popcll(mask);
    }
  }
  if (threadIdx.x == 0) rows[0] = base;
}

struct Factors {   // xent_factors_kernel
  float g, w, x, from_w, from_x;
};

// In how many numbers of 11 bits G holds the probabilities of `kept` tokens, where it has `held` rows. With one its rounding is beside the gradients' own
// with fp16 operands, the same for a whole row, so that few rows' errors do not even out: of 40 calls each, 1 / 2 / 8 / 32 / 64 tokens,
// dx's error was up to 2.5 / 1.8 / 1.6 / 1.5 / 1.46 times that rounding's, 1.3 at the median, as for more tokens; with two 1.03. (Forward and backward,
// us: 8 x 50304 x 768 113 -> 126, 64 x 50304 x 768 121 -> 140, 33 x 32000 x 2048 165 -> 191. held 0: one.)
constexpr int TWICE_TOKENS = 64;
__device__ __forceinline__ int halves_of(int kept, int64_t held) { return kept <= TWICE_TOKENS && 2 * (int64_t)kept <= held ? 2 : 1; }

// Rows in the products' type, zeros behind the width: to[i] = from[numbers ? numbers[i] : i], where `to` is not null. maxima: each workgroup's largest
// magnitude (MAXIMA workgroups then). also (null: none): the same rows, rounded to that type first, in the type that G is held in and *unit times; with
// `power` also times the row's power over *g, the largest number's (a row whose power is above that is none). held: where G has two
// numbers (halves_of) the rows that dW reads, also's or else to's, once more behind the last.
template <class OP>
__global__ __launch_bounds__(1024) void xent_gather_kernel(const void* from, int64_t ld, int dtype, int width, const int* numbers_of,
                                                           const int* count, int64_t most, int* maxima, typename OP::elem* to, int padded,
                                                           typename OP::Back::elem* also, const float* unit, const float* power, const float* g,
                                                           int64_t held) {
  __shared__ float acc[16];
  const int64_t rows = count ? *count : most;
  const bool twice = held && halves_of((int)rows, held) == 2;
  const int lane = threadIdx.x & 63;
  const bool quads = ((uintptr_t)from % (dtype == SA_DTYPE_F32 ? 16 : 8)) == 0 && ld % 4 == 0 && width % 4 == 0;
  float top = 0.f;
  constexpr int AHEAD = 4;   // loads in flight: a wavefront's of a row
  for (int64_t i = (int64_t)blockIdx.x * (blockDim.x / 64) + wave_index(); i < rows; i += (int64_t)gridDim.x * (blockDim.x / 64)) {
    const void* row = row_of(from, numbers_of ? numbers_of[i] : i, ld, dtype);
    const float by = !also ? 0.f : power ? fminf(power[i] / *g, 1.f) * *unit : *unit;
    for (int e0 = 4 * lane; e0 < padded; e0 += 256 * AHEAD) {
      Quad q[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        q[u] = quads ? fetch<true>(row, dtype, e0 + 256 * u, 1, width) : fetch<false>(row, dtype, e0 + 256 * u, 1, width);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        float x[4];
        if (quads) numbers<true>(q[u], dtype, x);
        else numbers<false>(q[u], dtype, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) top = larger(top, x[j]);
        if (to) put<true>(to + i * padded, OP::CODE, e0 + 256 * u, 1, padded, x);
        if (twice && !also) put<true>(to + (rows + i) * padded, OP::CODE, e0 + 256 * u, 1, padded, x);
        if (!also) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = stored(x[j], OP::CODE) * by;
        put<true>(also + i * padded, OP::Back::CODE, e0 + 256 * u, 1, padded, x);
        if (twice) put<true>(also + (rows + i) * padded, OP::Back::CODE, e0 + 256 * u, 1, padded, x);
      }
    }
  }
  if (maxima) put_maximum(top, acc, maxima, blockIdx.x);
}

// ---------------------------------------------------------------------------------------------
// Logits of a tile: rows of the vocabulary (M) x tokens (N).

struct LogitsCall {
  const void *w, *x;
  int64_t w_ld, x_ld;
  const int64_t* targets;
  const int* rows;          // null: tokens as they come, `tokens` of them
  int64_t tokens, vocab;    // vocab: of the whole table
  int64_t v0, v1;           // this launch's rows of it
  int stages;               // of the contraction
  int mt, nt;
  float *top, *sum, *at;    // (mt, tokens) statistics, the targets' logits
  const float* lse;         // backward: XentCall's
  const float* factor;      // backward: of each kept token's row of G; null: 1
  void* g;                  // (tokens, g_ld), or two rows of a token: halves_of(kept tokens, held)
  int64_t held;
  int64_t g_ld;
};

// (OP: what G is held in, of as many bits as the operands. Where G has two numbers, the second, what rounding the first leaves, is in as many
// rows again behind the kept tokens'.)
template <class OP, class L, bool GRAD>
__device__ __forceinline__ void logits_tile(const LogitsCall& c, int64_t id, typename L::Stage& s0, typename L::Stage& s1,
                                            typename L::Stage& s2, typename L::Stage& s3) {
  typedef typename OP::elem elem;
  constexpr int ES = sizeof(elem);
  const int64_t tokens = c.rows ? c.rows[0] : c.tokens;
  int m, n;
  if (!tile_of(id, c.mt, (int)((tokens + L::BN - 1) / L::BN), m, n)) return;
  const int64_t v0 = c.v0 + (int64_t)m * L::BM, n0 = (int64_t)n * L::BN;
  typename L::A oa;
  typename L::B ob;
  oa.open((const elem*)c.w + v0 * c.w_ld, ((c.v1 - v0 - 1) * c.w_ld + c.stages * L::BK) * ES, c.w_ld);
  ob.open((const elem*)c.x + n0 * c.x_ld, ((tokens - n0 - 1) * c.x_ld + c.stages * L::BK) * ES, c.x_ld);
  L l;
  l.run(oa, ob, s0, s1, s2, s3, c.stages);
  const int lane = threadIdx.x & 63, wave = wave_index(), h = lane >> 5, wm = wave / L::WN, wn = wave % L::WN;
  const int64_t vw = v0 + wm * L::TM * 32;   // the wavefront's first row of the vocabulary
  const bool edge = vw + L::TM * 32 > c.v1;
  if constexpr (!GRAD) {
    float* top = reinterpret_cast<float*>(s0.a);   // [WM][BN], then the sums (everyone is done with the stages)
    float* sum = top + L::WM * L::BN;
#pragma unroll
    for (int b = 0; b < L::TN; ++b) {
      const int col = (wn * L::TN + b) * 32 + (lane & 31);
      const int64_t i = n0 + col;
      const int64_t t = i < tokens ? c.targets[c.rows ? c.rows[ROWS_HEAD + i] : i] : -1;
      const int64_t tl = t - vw;
      const bool hit = i < tokens && t < c.v1 && tl >= 0 && tl < L::TM * 32 && ((tl >> 2) & 1) == h;
      if (__ballot(hit)) {
        const int want = (int)(hit ? tl : -1);
        float mine = 0.f;
#pragma unroll
        for (int a = 0; a < L::TM; ++a)
#pragma unroll
          for (int r = 0; r < 16; ++r) mine = want == a * 32 + acc_row(r, h) ? l.acc[a][b][r] : mine;
        if (hit) c.at[i] = mine;
      }
      if (edge) {
#pragma unroll
        for (int a = 0; a < L::TM; ++a)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (vw + a * 32 + acc_row(r, h) >= c.v1) l.acc[a][b][r] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int a = 0; a < L::TM; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, l.acc[a][b][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      // (Nothing but -inf: a sum of zeros, not of NaN. The difference is taken before the factor: as l LOG2E - round(mx LOG2E) in one instruction the
      // largest's own term is not 1, and a loss of 0 comes out off by up to 2^-24 of its logit, either way. What it costs: 16384 x 50304 x
      // 768 bf16 1230 -> 1241 us, 4096 x 50304 x 256 153 -> 157.)
      const float ref = mx == -INFINITY ? 0.f : mx;
      float s = 0.f;
#pragma unroll
      for (int a = 0; a < L::TM; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) s += __builtin_amdgcn_exp2f((l.acc[a][b][r] - ref) * LOG2E);
      s += __shfl_xor(s, 32);
      if (h == 0) top[wm * L::BN + col] = mx, sum[wm * L::BN + col] = s;
    }
    __syncthreads();
    for (int col = threadIdx.x; col < L::BN; col += L::THREADS) {
      const int64_t i = n0 + col;
      if (i >= tokens) continue;
      float mx = top[col], s = sum[col];
#pragma unroll
      for (int w = 1; w < L::WM; ++w) mx = fmaxf(mx, top[w * L::BN + col]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      s *= __builtin_amdgcn_exp2f((top[col] - ref) * LOG2E);
#pragma unroll
      for (int w = 1; w < L::WM; ++w) s += sum[w * L::BN + col] * __builtin_amdgcn_exp2f((top[w * L::BN + col] - ref) * LOG2E);
      c.top[m * c.tokens + i] = mx;
      c.sum[m * c.tokens + i] = s;
    }
  } else {
    // G of 32 tokens x the wavefront's rows goes through a part of LDS of its own, so that a token's row is stored in
    // 16-byte pieces side by side. Chunk c of token row r sits at c ^ (r mod 8, or mod as many as there are).
    constexpr int RB = L::TM * 32 * ES;   // bytes of a token's row
    constexpr int CPR = RB / 16, TURN = CPR < 8 ? CPR - 1 : 7;
    constexpr int FIT = (int)sizeof(s0) / (32 * RB);   // wavefronts' rows in a stage
    static_assert(L::WAVES <= 2 * FIT, "and in two");
    uint8_t* mine = (wave < FIT ? s0.a : s1.a) + wave % FIT * 32 * RB;
    // (rows past the last token lie past the resource's end: such stores are dropped)
    const int g_row = (int)(c.g_ld * ES);
    const int64_t bytes = min(tokens - n0, (int64_t)L::BN) * g_row - (vw - c.v0) * ES;
    const __amdgpu_buffer_rsrc_t rs = resource((elem*)c.g + n0 * c.g_ld + (vw - c.v0), bytes);
    const int halves = uniform(halves_of((int)tokens, c.held));
    const int left = edge ? (int)(c.v1 - vw) : L::TM * 32;   // rows of the vocabulary
    const auto half_of_g = [&](auto second, const __amdgpu_buffer_rsrc_t& rs) {
#pragma unroll 1
      for (int b = 0; b < L::TN; ++b) {
        const int64_t i = n0 + (wn * L::TN + b) * 32 + (lane & 31);
        const bool real = i < tokens;
        // (beside the largest logit, whose distance is exact where weights are large: log of the sum alone is off by 2^-21)
        const float top = real ? c.lse[i] : 0.f;
        const float lift = (c.factor && real ? c.factor[i] : 1.f) * OP::LIFT, over = real ? c.lse[c.tokens + i] * lift : 0.f;
        const int64_t t = real ? c.targets[c.rows[ROWS_HEAD + i]] - vw : -1;
        const int tl = t >= 0 && t < L::TM * 32 ? (int)t : -1;
        uint8_t* to = mine + (lane & 31) * RB;
#pragma unroll
        for (int a = 0; a < L::TM; ++a)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float p[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int row = a * 32 + 8 * q + 4 * h + r;
              float x = l.acc[a][0][4 * q + r];
#pragma unroll
              for (int o = 1; o < L::TN; ++o) x = b == o ? l.acc[a][o][4 * q + r] : x;
              x = __builtin_amdgcn_exp2f((x - top) * LOG2E) * over;
              x = tl == row ? x - lift : x;
              if constexpr (second) x -= stored(x, OP::CODE);   // (an infinity: a NaN, in a row that has them already)
              p[r] = row < left ? x : 0.f;
            }
            const int byte = (a * 32 + 8 * q + 4 * h) * ES;
            put<true>(to + (((byte >> 4) ^ (lane & TURN)) << 4) + (byte & 15), OP::CODE, 0, 1, 4, p);
          }
        __asm__ volatile("" ::: "memory");   // (a wavefront's own LDS accesses run in order)
#pragma unroll
        for (int k = 0; k < 32 * CPR / 64; ++k) {
          const int slot = k * 64 + lane, r = slot / CPR, ch = slot % CPR;
          const u32x4 v = *reinterpret_cast<const u32x4*>(mine + r * RB + ((ch ^ (r & TURN)) << 4));
          __builtin_amdgcn_raw_buffer_store_b128(v, rs, r * g_row + ch * 16, (wn * L::TN + b) * 32 * g_row, 0);
        }
        __asm__ volatile("" ::: "memory");
      }
    };
    half_of_g(std::false_type{}, rs);
    if constexpr (L::TWO_NUMBERS)
      if (halves == 2) half_of_g(std::true_type{}, resource((elem*)c.g + (tokens + n0) * c.g_ld + (vw - c.v0), bytes));
  }
}

template <class OP, class L>
__global__ __launch_bounds__(L::THREADS, L::WAVES >= 8 ? 2 : 1) void xent_logits_kernel(LogitsCall c) {
  __shared__ typename L::Stage s0, s1, s2, s3;
  logits_tile<OP, L, false>(c, blockIdx.x, s0, s1, s2, s3);
}

// A token's statistics over the mt tiles joined: `TOKENS` tokens a workgroup, NTHREADS / TOKENS lanes each. What the backward pass takes of them, the loss, and
// the workgroup's sum of losses. (32 tokens where there are many, four where a few tokens' 400 tiles are all there is to
// read: 8 tokens of 50304 words 8.1 us with 8 lanes each, 4.7 with 64.)
template <int TOKENS>
__global__ __launch_bounds__(NTHREADS) void xent_join_kernel(LogitsCall c, float* lse, float* each, float* sums, int64_t ignore) {
  constexpr int LANES = NTHREADS / TOKENS;
  __shared__ float tm[LANES][TOKENS + 1], ts[LANES][TOKENS + 1], out[TOKENS];
  const int64_t tokens = c.rows ? c.rows[0] : c.tokens;
  const int x = threadIdx.x % TOKENS, k = threadIdx.x / TOKENS;
  float total = 0.f;
  for (int64_t i0 = (int64_t)blockIdx.x * TOKENS; i0 < tokens; i0 += (int64_t)gridDim.x * TOKENS) {
    const int64_t i = i0 + x;
    float mx = -INFINITY, s = 0.f;
    if (i < tokens) {
#pragma unroll 8
      for (int m = k; m < c.mt; m += LANES) {
        const float a = c.top[m * c.tokens + i], b = c.sum[m * c.tokens + i];
        const float up = fmaxf(mx, a), ref = up == -INFINITY ? 0.f : up;
        s = s * __builtin_amdgcn_exp2f((mx - ref) * LOG2E) + b * __builtin_amdgcn_exp2f((a - ref) * LOG2E);
        mx = up;
      }
    }
    __syncthreads();
    tm[k][x] = mx, ts[k][x] = s;
    __syncthreads();
    if (k == 0 && i < tokens) {
      for (int w = 1; w < LANES; ++w) mx = fmaxf(mx, tm[w][x]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      s = 0.f;
      for (int w = 0; w < LANES; ++w) s += ts[w][x] * __builtin_amdgcn_exp2f((tm[w][x] - ref) * LOG2E);
      const int64_t token = c.rows ? c.rows[ROWS_HEAD + i] : i;
      const int64_t t = c.targets[token];
      // (a target outside the vocabulary has no logit: its loss and gradients become NaN)
      const bool real = t >= 0 && t < c.vocab;
      const float nan = __uint_as_float(0x7fc00000u);
      float loss = real ? (mx - c.at[i]) + logf(s) : nan;
      if (!c.rows && t == ignore) loss = 0.f;
      if (lse) lse[i] = mx, lse[c.tokens + i] = real ? 1.f / s : nan;
      if (each) each[token] = loss;
      total += loss;
    }
  }
  if (!sums) return;
  if (k == 0) out[x] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < TOKENS; ++w) total += out[w];
    sums[blockIdx.x] = total;
  }
}

// The workgroups' sums added in a fixed order, over the tokens kept where a mean is asked for (none: 0 / 0, a NaN).
__global__ __launch_bounds__(1024) void xent_sum_kernel(const float* sums, int n, const int* rows, float* loss) {
  __shared__ float acc[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) s += sums[i];
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if (lane == 0) acc[wave] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = 0.f;
  for (int w = 0; w < 16; ++w) s += acc[w];
  *loss = rows ? s / (float)rows[0] : s;
}

// ---------------------------------------------------------------------------------------------
// The backward pass's factors. w and x: the units that the products with G hold weight and x in, powers of two (`scaled`; x's with `power`, too),
// from_w and from_x back from them. g multiplies the sums of both products.
// Reduction none: g is the power of two at or below the largest |g_i| that is a number, for dW's sums. With `power` that at or below each kept
// token's own |g_i| goes there, for its dX, and g_i over it to `factor`, for its row of G before it is rounded: so G_i has all its bits
// whatever the others are (with one unit for all a row of 1e-8 of the largest was off by 1.8%). Without (fp32's range needs none)
// factor is g_i / g.
__device__ __forceinline__ uint32_t exponent_of(float x) { return (__float_as_uint(x) >> 23) & 0xff; }
__global__ __launch_bounds__(1024) void xent_factors_kernel(const float* dloss, const int* rows, int reduction, bool scaled, Factors* out,
                                                            float* factor, float* power) {
  __shared__ float acc[16], maxima[2];
  const int tokens = rows[0];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (scaled || power) {   // half of the threads look at either matrix's largest magnitudes
    float most = scaled || threadIdx.x >= MAXIMA ? __uint_as_float((uint32_t)rows[64 + threadIdx.x]) : 0.f;
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    if (lane == 0) acc[wave] = most;
    __syncthreads();
    if (threadIdx.x < 2) {
      most = 0.f;
      for (int w = 0; w < 8; ++w) most = fmaxf(most, acc[threadIdx.x * 8 + w]);
      maxima[threadIdx.x] = most;
    }
    __syncthreads();
  }
  static_assert(MAXIMA == 512, "half of the threads");
  const auto below = [](float x) { return __uint_as_float(min(max(exponent_of(x), 1u), 254u) << 23); };   // a power of two
  float g;
  if (!factor) {   // (no token kept: gradients of zeros, not 0 / 0)
    g = tokens == 0 ? 0.f : reduction == SA_REDUCE_MEAN ? dloss[0] / (float)tokens : dloss[0];
  } else {
    float most = 0.f;
    for (int i = threadIdx.x; i < tokens; i += 1024) most = larger(most, dloss[rows[ROWS_HEAD + i]]);
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    if (lane == 0) acc[wave] = most;
    __syncthreads();
    for (int w = 0; w < 16; ++w) most = fmaxf(most, acc[w]);
    g = below(most);
    for (int i = threadIdx.x; i < tokens; i += 1024) {
      const float mine = dloss[rows[ROWS_HEAD + i]], to = power ? below(mine) : g;
      factor[i] = mine / to;
      if (power) power[i] = to;
    }
  }
  if (threadIdx.x) return;
  Factors f{g, 1.f, 1.f, 1.f, 1.f};
  const auto unit = [](float most, float& to, float& from) {   // the largest comes to 2^14 .. 2^15; nothing but zeros stays as it is
    const int e = most == 0.f ? 0 : min(14 - ((int)exponent_of(most) - 127), 126);
    to = __uint_as_float((uint32_t)(127 + e) << 23);
    from = __uint_as_float((uint32_t)(127 - e) << 23);
  };
  if (scaled) unit(maxima[0], f.w, f.from_w);
  if (scaled || power) unit(maxima[1], f.x, f.from_x);
  *out = f;
}

// ---------------------------------------------------------------------------------------------
// A product of the backward pass. A plain, (M, K): dX = G W; A turned, (K, M): dW = G^T X. B turned, (K, N).

struct ProductCall {
  const void *a, *b;
  int64_t a_ld, b_ld;
  const int* rows;          // kept tokens: M (dX) or K (dW), as many times over as G has numbers (halves_of, held)
  int64_t held;
  int64_t m, n, k;          // M of dW, N, K of dX
  int64_t b_cols;           // columns of b that may be read (whole 16-byte pieces)
  int mt, nt, splits;
  float* sums;              // [split][M rows][n_ld] where they go to the workspace
  int64_t n_ld, m_rows;
  int add;                  // onto what is there
  void* out;                // dW's rows, where nothing is split
  int64_t out_ld;
  int out_t;
  const Factors* units;
  float lift;
};

template <class OP, class L, bool DW>
__device__ __forceinline__ void product_tile(const ProductCall& c, int64_t id, int part, typename L::Stage& s0, typename L::Stage& s1,
                                             typename L::Stage& s2, typename L::Stage& s3) {
  typedef typename OP::elem elem;
  constexpr int ES = sizeof(elem);
  const int64_t tokens = uniform(c.rows[0] * halves_of(c.rows[0], c.held));
  const int64_t M = DW ? c.m : tokens, K = DW ? tokens : c.k;
  int m, n;
  if (!tile_of(id, DW ? c.mt : (int)((M + L::BM - 1) / L::BM), c.nt, m, n)) return;
  const int64_t m0 = (int64_t)m * L::BM, n0 = (int64_t)n * L::BN;
  const int stages = (int)((K + L::BK - 1) / L::BK);
  const int per = (stages + c.splits - 1) / c.splits;
  const int first = uniform(min(part * per, stages)), last = uniform(min(first + per, stages));
  const int64_t k0 = (int64_t)first * L::BK;   // (offsets within a split stay below 2^31 bytes)
  typename L::A oa;
  typename L::B ob;
  if constexpr (DW) oa.open((const elem*)c.a + k0 * c.a_ld + m0, ((K - k0) * c.a_ld - m0) * ES, c.a_ld);
  else oa.open((const elem*)c.a + m0 * c.a_ld + k0, ((M - m0) * c.a_ld - k0) * ES, c.a_ld);
  ob.open((const elem*)c.b + k0 * c.b_ld + n0, ((K - k0 - 1) * c.b_ld + c.b_cols - n0) * ES, c.b_ld);
  L l;
  l.run(oa, ob, s0, s1, s2, s3, last - first);
  const int lane = threadIdx.x & 63, wave = wave_index(), h = lane >> 5, wm = wave / L::WN, wn = wave % L::WN;
  // rows past M lie past the resource's end, columns past N get an offset there: such stores are dropped
  const int es = c.out ? (c.out_t == SA_DTYPE_F32 ? 4 : 2) : 4;
  const int64_t ld = c.out ? c.out_ld : c.n_ld;
  uint8_t* base = (uint8_t*)c.out + m0 * ld * es;
  if (!c.out) base = (uint8_t*)(c.sums + ((int64_t)part * c.m_rows + m0) * ld);
  const __amdgpu_buffer_rsrc_t rs = resource(base, min(M - m0, (int64_t)L::BM) * ld * es);
  // (the unit last and alone: with g it may leave fp32's range)
  const float scale = c.out ? c.units->g * c.lift : 1.f, unit = c.out ? c.units->from_x : 1.f;
  const int row_bytes = (int)ld * es;
  const auto each = [&](auto&& put_sixteen) {
#pragma unroll
    for (int b = 0; b < L::TN; ++b) {
      const int64_t col = n0 + (wn * L::TN + b) * 32 + (lane & 31);
      const int at = col < c.n ? (int)col * es + 4 * h * row_bytes : 0x7ffffff0;
#pragma unroll
      for (int a = 0; a < L::TM; ++a) put_sixteen(l.acc[a][b], at, (wm * L::TM + a) * 32);
    }
  };
  if (es == 2) {
    each([&](const f32x16& x, int at, int row) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        __builtin_amdgcn_raw_buffer_store_b16(to16(x[r] * scale * unit, c.out_t), rs, at, (row + acc_row(r, 0)) * row_bytes, 0);
    });
  } else if (c.add) {
    each([&](const f32x16& x, int at, int row) {
      float y[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) y[r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, at, (row + acc_row(r, 0)) * row_bytes, 0));
#pragma unroll
      for (int r = 0; r < 16; ++r)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y[r] + x[r]), rs, at, (row + acc_row(r, 0)) * row_bytes, 0);
    });
  } else {
    each([&](const f32x16& x, int at, int row) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[r] * scale * unit), rs, at, (row + acc_row(r, 0)) * row_bytes, 0);
    });
  }
}

// One pass of the backward over the vocabulary: dX's and dW's products of a piece and G of the next one, which do not depend on
// each other, in one launch. The products of a piece are a few hundred long tiles (dW's contract over all tokens), fewer than two rounds
// of the chip or just over one; the many short tiles of G fill what they leave idle. Workgroups start in order: the longest first.
struct PassCall {
  LogitsCall g;
  ProductCall x, w;
  int x_at, x_tiles, x_end, w_at, w_tiles, w_end, g_at;   // workgroups: of a part of the contraction, of all parts
};
template <class OP, class LG, class LX, class LW>
__global__ __launch_bounds__(LG::THREADS, LG::WAVES >= 8 ? 2 : 1) void xent_pass_kernel(PassCall c) {
  typedef typename std::conditional<(sizeof(typename LW::Stage) > sizeof(typename LG::Stage)), typename LW::Stage, typename LG::Stage>::type S;
  static_assert(sizeof(typename LX::Stage) <= sizeof(S) && LG::THREADS == LX::THREADS && LG::THREADS == LW::THREADS, "one launch for all");
  __shared__ S s0, s1, s2, s3;
  const int id = blockIdx.x;
  if (id >= c.x_at && id < c.x_end) {
    const int part = uniform((id - c.x_at) / c.x_tiles);
    typedef typename LX::Stage X;
    product_tile<OP, LX, false>(c.x, id - c.x_at - part * c.x_tiles, part, (X&)s0, (X&)s1, (X&)s2, (X&)s3);
  } else if (id >= c.w_at && id < c.w_end) {
    const int part = uniform((id - c.w_at) / c.w_tiles);
    typedef typename LW::Stage W;
    product_tile<OP, LW, true>(c.w, id - c.w_at - part * c.w_tiles, part, (W&)s0, (W&)s1, (W&)s2, (W&)s3);
  } else {
    typedef typename LG::Stage G;
    logits_tile<OP, LG, true>(c.g, id - c.g_at, (G&)s0, (G&)s1, (G&)s2, (G&)s3);
  }
}

// dX: a token's parts added (and those *kept rows behind them, where G has two numbers: halves_of, held), times g or its own power; zero rows for the tokens that are
// ignored. dW: the parts of a piece's rows.
__global__ __launch_bounds__(NTHREADS) void xent_finish_kernel(const float* sums, int splits, int64_t split_stride, int64_t n_ld,
                                                               const int* place, const Factors* units, const float* unit, float lift,
                                                               const float* power, const int* kept, int64_t held, void* out, int64_t rows,
                                                               int width, int dtype) {
  const int lane = threadIdx.x & 63;
  const bool quads = width % 4 == 0;
  const float u = *unit;
  const bool two = held && halves_of(*kept, held) == 2;
  for (int64_t row = (int64_t)blockIdx.x * NWAVES + wave_index(); row < rows; row += (int64_t)gridDim.x * NWAVES) {
    const int64_t at = place ? place[row] : row;
    const float f = (power && at >= 0 ? power[at] : units->g) * lift;
    for (int e = 4 * lane; e < width; e += 256) {
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (at >= 0) {
#pragma unroll 8
        for (int s = 0; s < splits; ++s) {
          const float4 v = *reinterpret_cast<const float4*>(sums + s * split_stride + at * n_ld + e);
          x[0] += v.x, x[1] += v.y, x[2] += v.z, x[3] += v.w;
        }
        if (two) {
          const int64_t behind = at + *kept;
#pragma unroll 8
          for (int s = 0; s < splits; ++s) {
            const float4 v = *reinterpret_cast<const float4*>(sums + s * split_stride + behind * n_ld + e);
            x[0] += v.x, x[1] += v.y, x[2] += v.z, x[3] += v.w;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = x[j] * f * u;
      }
      if (quads) put<true>(row_of(out, row, width, dtype), dtype, e, 1, width, x);
      else put<false>(row_of(out, row, width, dtype), dtype, e, 1, width, x);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Host side

template <class OP>
struct XentConfigs {   // 16-bit products
  typedef Mainloop<OP, 2, 4, 4, 2, false, false> Large;   // 256 x 256
  typedef Mainloop<OP, 2, 2, 2, 2, false, false> Middle;  // 128 x 128
  typedef Mainloop<OP, 4, 1, 1, 2, false, false> Small;   // 128 x 64
  typedef Mainloop<OP, 2, 4, 4, 2, false, true> LargeX;
  typedef Mainloop<OP, 2, 2, 2, 2, false, true> MiddleX;
  typedef Mainloop<OP, 2, 2, 1, 2, false, true> SmallX;   // 64 x 128
  typedef Mainloop<OP, 2, 4, 4, 2, true, true> LargeW;
  typedef Mainloop<OP, 2, 2, 2, 2, true, true> MiddleW;
};
template <>
struct XentConfigs<XF32> {   // (fp32 tiles are half as large in elements per stage; one size)
  typedef Mainloop<XF32, 2, 2, 2, 2, false, false> Large;
  typedef Mainloop<XF32, 2, 2, 2, 2, false, false> Middle;
  typedef Mainloop<XF32, 4, 1, 1, 2, false, false> Small;
  typedef Mainloop<XF32, 2, 2, 2, 2, false, true> LargeX;
  typedef Mainloop<XF32, 2, 2, 2, 2, false, true> MiddleX;
  typedef Mainloop<XF32, 2, 2, 1, 2, false, true> SmallX;
  typedef Mainloop<XF32, 2, 2, 2, 2, true, true> LargeW;
  typedef Mainloop<XF32, 2, 2, 2, 2, true, true> MiddleW;
};

// One tile's tokens of the smallest kernels. Us by 128 x 64 / 128 x 128: 8 tokens x 50304 x 768, no gradient, weight out of HBM 20.0 / 21.5; training,
// forward and backward: fp32 64 x 50304 x 768 67 / 109 and 183 / 323, fp16 33 x 32000 x 2048 40 / 42 and 122 / 140, bf16 64 x 50304 x 768
// 56 / 58 and 122 / 118 (backward 26 and 8 less than now that fp16's G is two numbers, and bf16's weight read in two types).
constexpr int64_t SMALL_TOKENS = 64;
constexpr int64_t IN_PLACE_TOKENS = 256;  // up to here a forward pass reads the rows as they are (250 tokens 40 us, listed and gathered 47)
constexpr int64_t PIECE_BYTES = (int64_t)256 << 20;   // of a piece's G, of which there are two at a time
constexpr int64_t JOIN_FEW = 1024;        // tokens up to which the join takes 64 lanes for each (calls, us, 64 / 8 lanes: 1000 tokens 110 / 112, 4096 345 / 340)
constexpr int64_t MAX_LD_BYTES = 1 << 22;             // of a row: 256 within a buffer resource's 2 GiB, their offsets within 31 bits

// What a call does, from its sizes alone.
template <class OP>
struct XentShape {
  static constexpr int ES = sizeof(typename OP::elem), BK = KB / ES;
  static constexpr bool SCALED = !std::is_same<OP, typename OP::Back>::value;   // weight and x have copies for the products with G
  bool train, small, large, gather, copy_w;
  int64_t padded, bm, mt, join_tokens, join_blocks;
  // backward
  int64_t held;   // rows of G
  int64_t piece, pieces;
  bool large_pass;
  int splits_x, splits_w, splits_last;   // parts of dX's contraction, of dW's, and of that in the last pass
  // workspace
  int64_t x, w, top, sum, at, sums, factors, x_back, w_back, g, g2, dx, dw, total;

  XentShape(const XentCall& c, bool backward) {
    train = c.lse != nullptr;
    padded = align_up(c.width, BK);
    small = c.tokens <= SMALL_TOKENS;
    // Tiles of 256 x 256 where every CU has one and the last tokens' are not mostly empty (four wavefronts' of 128 x 128 else).
    // Forward, us, large / middle, tokens x words x 768: 400 x 50304 58 / 64, 1000 x 16384 40 / 47, 2000 x 50304 183 / 197; 128 x 50304
    // 27 / 25 (197 tiles), 300 x 33000 54 / 42 (212 of the second 256 tokens missing).
    const bool whole = cdiv(c.tokens, 256) * 256 * 4 <= cdiv(c.tokens, 128) * 128 * 5;
    large = !small && ES == 2 && whole && cdiv(c.vocab, 256) * cdiv(c.tokens, 256) >= c.cus;
    bm = large ? 256 : 128;
    mt = cdiv(c.vocab, bm);
    const bool x_ok = c.x_t == OP::CODE && padded == c.width && (uintptr_t)c.x % 16 == 0 && c.x_ld * ES % 16 == 0 &&
                      c.x_ld >= c.width && c.x_ld * ES < MAX_LD_BYTES;
    gather = train || c.reduction != SA_REDUCE_NONE || c.tokens > IN_PLACE_TOKENS || !x_ok;
    copy_w = !(c.w_t == OP::CODE && padded == c.width && (uintptr_t)c.w % 16 == 0 && c.w_ld * ES % 16 == 0 &&
               c.w_ld >= c.width && c.w_ld * ES < MAX_LD_BYTES);
    join_tokens = c.tokens <= JOIN_FEW ? 4 : 32;
    join_blocks = std::min<int64_t>(cdiv(c.tokens, join_tokens), 4096);
    int64_t p = 0;
    const auto take = [&p](int64_t bytes) {
      const int64_t at = p;
      p += align_up(bytes, 1024);
      return at;
    };
    // (few tokens: room for two numbers of each, whatever is kept; more: where half of the rows are enough for what is kept)
    held = backward && ES == 2 && !SCALED && c.tokens <= TWICE_TOKENS ? 2 * c.tokens : c.tokens;
    x = take(gather ? held * padded * ES : 0);
    w = take(copy_w ? c.vocab * padded * ES : 0);
    if (!backward) {
      top = take(mt * c.tokens * 4);
      sum = take(mt * c.tokens * 4);
      at = take(c.tokens * 4);
      sums = take(join_blocks * 4);
    } else {
      // Pieces of the vocabulary whose G fits PIECE_BYTES (and a token's row of it MAX_LD_BYTES), in whole tiles, of about one size
      const int64_t most = std::max<int64_t>(std::min(PIECE_BYTES / (held * ES), MAX_LD_BYTES / ES) / 256 * 256, 256);
      pieces = cdiv(c.vocab, most);
      piece = align_up(cdiv(c.vocab, pieces), 256);
      pieces = cdiv(c.vocab, piece);
      // The same choice by a pass's tiles (backward, us, large / middle: 2048 x 50304 x 768 589 / 645, 4096 x 16384 x 1024 455 / 498, 500 x
      // 50304 x 768 229 / 237; 100 x 50304 x 768 143 / 117, 2000 x 4000 x 1024 109 / 95). No contraction is longer than a CU's
      // share of a pass, or twice that in the last, where no tiles of G fill up; parts' sums go through memory. dX's is held to half of
      // the share, as ignored tokens shorten everything else (5003 x 50257 x 1024, a third ignored, in 1 / 2 / 3 / 4 parts:
      // 1453 / 1201 / 1199 / 1205 us; 1000 x 16384 x 768 in 2 / 4 / 8 / 16: 217 / 151 / 130 / 136; 100 x 50304 x 768 in 4 / 8 / 16: 153 / 117 / 114).
      // dW's over few tokens is best whole (1000 x 16384 x 768 in 1 / 2 parts 136 / 175), over 16384 x 50304 the last piece's
      // in 1 / 2 / 3 / 6 4138 / 4070 / 4056 / 4063. Pieces of 64 / 128 / 256 / 512 MB there: 4405 / 4160 / 4039 / 4016.
      const int64_t k_x = cdiv(piece, BK), k_w = cdiv(held, BK), k_g = padded / BK;
      const auto tiles = [&](int64_t edge, int64_t m, int64_t n) { return cdiv(m, edge) * cdiv(n, edge); };
      large_pass = ES == 2 && whole && tiles(256, c.tokens, c.width) + tiles(256, piece, c.width) + tiles(256, c.tokens, piece) / 4 >= c.cus;
      const int64_t edge = large_pass ? 256 : 128, slots = large_pass ? c.cus : 2 * (int64_t)c.cus;
      const int64_t products = (c.dx ? tiles(edge, held, c.width) * k_x : 0) + (c.dw ? tiles(edge, piece, c.width) * k_w : 0);
      const int64_t share = cdiv(products + (pieces > 1 ? tiles(edge, c.tokens, piece) * (k_g + 8) : products / 2), slots);
      const int64_t share_last = std::max<int64_t>(cdiv(products, 2 * slots), 1);
      const auto parts = [](int64_t stages, int64_t of, int64_t most) {
        return (int)std::max<int64_t>(1, std::min<int64_t>({cdiv(stages, of), stages / 8, most}));
      };
      // A part more costs dX's sums once more through memory: up to 64 parts where they take no more than 32 MB, 16 at least (few tokens have
      // few tiles and long contractions; with the smallest tiles, fp32 3 x 68497 x 768 430 -> 242 us, 5 x 68536 x 128 311 -> 119).
      const int64_t most_x = std::min<int64_t>(std::max<int64_t>(((int64_t)32 << 20) / (held * padded * 4), 16), 64);
      splits_x = parts(k_x, pieces > 1 ? cdiv(share, 2) : 2 * share_last, most_x);
      splits_w = parts(k_w, share, 16);
      splits_last = parts(k_w, 2 * share_last, 16);
      // (a part's rows lie within 2^30 bytes)
      const int64_t w_row = (SCALED || copy_w ? padded : c.w_ld) * ES, x_row = std::max(padded, piece) * ES;
      splits_x = std::max(splits_x, (int)cdiv(piece * w_row, (int64_t)1 << 30));
      splits_w = std::max(splits_w, (int)cdiv(held * x_row, (int64_t)1 << 30));
      splits_last = std::max(splits_last, splits_w);
      factors = take((2 * c.tokens + 64) * 4);
      x_back = take(c.dw && ES == 2 ? held * padded * ES : 0);   // (many tokens, fp16: with reduction none alone, which the size's query does not know)
      w_back = take(c.dx && SCALED ? c.vocab * padded * ES : 0);
      g = take(held * piece * ES);
      g2 = take(pieces > 1 ? held * piece * ES : 0);
      dx = take(c.dx ? splits_x * held * padded * 4 : 0);
      dw = take(c.dw && splits_last > 1 ? splits_last * piece * padded * 4 : 0);
    }
    total = p;
  }
};

template <class OP, class L>
void launch_logits(LogitsCall lc, int64_t tokens, hipStream_t st) {
  lc.mt = (int)cdiv(lc.v1 - lc.v0, L::BM);
  lc.nt = (int)cdiv(tokens, L::BN);
  hipLaunchKernelGGL((xent_logits_kernel<OP, L>), dim3((unsigned)tiles_grid(lc.mt, lc.nt)), dim3(L::THREADS), 0, st, lc);
}
// g, x, w: what the pass does (null: not that)
// held: rows of G
template <class OP, class LG, class LX, class LW>
bool launch_pass(const LogitsCall* g, const ProductCall* x, const ProductCall* w, int64_t tokens, int64_t held, hipStream_t st) {
  PassCall pc{};
  int64_t at = 0;
  const auto place = [&at](ProductCall& c, int64_t m, int edge_m, int edge_n, int& begin, int& tiles, int& end) {
    c.mt = (int)cdiv(m, edge_m);
    c.nt = (int)cdiv(c.n, edge_n);
    tiles = (int)tiles_grid(c.mt, c.nt);
    begin = (int)at;
    end = (int)(at += (int64_t)tiles * c.splits);
  };
  const auto put_x = [&] {
    if (x) pc.x = *x, place(pc.x, held, LX::BM, LX::BN, pc.x_at, pc.x_tiles, pc.x_end);
  };
  const bool x_first = x && w && cdiv(x->k, x->splits) > cdiv(held, w->splits);
  if (x_first) put_x();
  if (w) pc.w = *w, place(pc.w, w->m, LW::BM, LW::BN, pc.w_at, pc.w_tiles, pc.w_end);
  if (!x_first) put_x();
  if (g) {
    pc.g = *g;
    pc.g.mt = (int)cdiv(g->v1 - g->v0, LG::BM);
    pc.g.nt = (int)cdiv(tokens, LG::BN);
    pc.g_at = (int)at;
    at += tiles_grid(pc.g.mt, pc.g.nt);
  }
  if (at * LG::THREADS >= ((int64_t)1 << 32)) return false;   // more threads than a launch takes
  hipLaunchKernelGGL((xent_pass_kernel<OP, LG, LX, LW>), dim3((unsigned)at), dim3(LG::THREADS), 0, st, pc);
  return true;
}
template <class OP>
void launch_gather(const void* from, int64_t ld, int dtype, int64_t width, const int* numbers_of, const int* count, int64_t rows, int* maxima,
                   void* to, int64_t padded, hipStream_t st, void* also = nullptr, const float* unit = nullptr, const float* power = nullptr,
                   const float* g = nullptr, int64_t held = 0) {
  const int64_t blocks = maxima ? MAXIMA : std::min<int64_t>(cdiv(rows, NWAVES), 16384);
  hipLaunchKernelGGL((xent_gather_kernel<OP>), dim3((unsigned)blocks), dim3(maxima ? 1024 : NTHREADS), 0, st, from, ld, dtype, (int)width,
                     numbers_of, count, rows, maxima, (typename OP::elem*)to, (int)padded, (typename OP::Back::elem*)also, unit, power, g, held);
}
inline void launch_finish(const float* sums, int splits, int64_t split_stride, int64_t n_ld, const int* place, const Factors* units,
                          const float* unit, float lift, const float* power, const int* kept, int64_t held, void* out, int64_t rows,
                          int64_t width, int dtype, hipStream_t st) {
  const int64_t blocks = std::min<int64_t>(cdiv(rows, NWAVES), 16384);
  hipLaunchKernelGGL(xent_finish_kernel, dim3((unsigned)blocks), dim3(NTHREADS), 0, st, sums, splits, split_stride, n_ld, place, units,
                     unit, lift, power, kept, held, out, rows, (int)width, dtype);
}

template <class OP>
int64_t xent_bytes(const XentCall& c, bool backward) {
  return XentShape<OP>(c, backward).total;
}

template <class OP>
int xent_forward(const XentCall& c) {
  typedef XentConfigs<OP> F;
  const XentShape<OP> s(c, false);
  char* ws = (char*)c.ws;
  float* each = c.reduction == SA_REDUCE_NONE ? c.loss : nullptr;
  LogitsCall lc{};
  lc.targets = c.targets;
  lc.tokens = c.tokens;
  lc.vocab = c.vocab;
  if (s.gather) {
    const bool scaled = s.train && s.SCALED;
    const bool maxima = s.train && s.ES == 2;   // of x (fp16: for a backward pass with reduction none, whatever the forward's)
    hipLaunchKernelGGL(xent_rows_kernel, dim3(scaled ? 1 + MAXIMA : 1), dim3(1024), 0, c.st, c.targets, c.tokens, c.ignore, c.rows, each,
                       Matrix{c.w, c.w_ld, c.vocab, (int)c.width, c.w_t});
    lc.rows = c.rows;
    launch_gather<OP>(c.x, c.x_ld, c.x_t, c.width, c.rows + ROWS_HEAD, c.rows, c.tokens, maxima ? c.rows + 64 + MAXIMA : nullptr,
                      ws + s.x, s.padded, c.st);
    lc.x = ws + s.x, lc.x_ld = s.padded;
  } else {
    lc.x = c.x, lc.x_ld = c.x_ld;
  }
  if (s.copy_w) {
    launch_gather<OP>(c.w, c.w_ld, c.w_t, c.width, nullptr, nullptr, c.vocab, nullptr, ws + s.w, s.padded, c.st);
    lc.w = ws + s.w, lc.w_ld = s.padded;
  } else {
    lc.w = c.w, lc.w_ld = c.w_ld;
  }
  lc.v0 = 0, lc.v1 = c.vocab;
  lc.stages = (int)(s.padded / s.BK);
  lc.top = (float*)(ws + s.top), lc.sum = (float*)(ws + s.sum), lc.at = (float*)(ws + s.at);
  if (s.small) launch_logits<OP, typename F::Small>(lc, c.tokens, c.st);
  else if (s.large) launch_logits<OP, typename F::Large>(lc, c.tokens, c.st);
  else launch_logits<OP, typename F::Middle>(lc, c.tokens, c.st);
  lc.mt = (int)s.mt;
  float* sums = each ? nullptr : (float*)(ws + s.sums);
  const dim3 joins((unsigned)s.join_blocks);
  if (s.join_tokens == 4) hipLaunchKernelGGL((xent_join_kernel<4>), joins, dim3(NTHREADS), 0, c.st, lc, c.lse, each, sums, c.ignore);
  else hipLaunchKernelGGL((xent_join_kernel<32>), joins, dim3(NTHREADS), 0, c.st, lc, c.lse, each, sums, c.ignore);
  if (sums)
    hipLaunchKernelGGL(xent_sum_kernel, dim3(1), dim3(1024), 0, c.st, sums, (int)s.join_blocks,
                       c.reduction == SA_REDUCE_MEAN ? c.rows : nullptr, c.loss);
  return launch_status();
}

template <class OP>
int xent_backward(const XentCall& c) {
  typedef typename OP::Back BACK;
  typedef XentConfigs<OP> F;
  typedef XentConfigs<BACK> B;
  constexpr int ES = sizeof(typename BACK::elem);
  const XentShape<OP> s(c, true);
  char* ws = (char*)c.ws;
  Factors* units = (Factors*)(ws + s.factors);
  float* factor = c.reduction == SA_REDUCE_NONE ? (float*)units + 64 : nullptr;
  float* power = factor && ES == 2 ? factor + c.tokens : nullptr;
  hipLaunchKernelGGL(xent_factors_kernel, dim3(1), dim3(1024), 0, c.st, c.dloss, c.rows, c.reduction, s.SCALED, units, factor, power);
  const int64_t held = ES == 2 && !s.SCALED ? s.held : 0;   // (0: G in one number)
  const bool two = s.SCALED || power;
  const char* x_back = ws + (two ? s.x_back : s.x);   // dW's
  launch_gather<OP>(c.x, c.x_ld, c.x_t, c.width, c.rows + ROWS_HEAD, c.rows, c.tokens, nullptr, ws + s.x, s.padded, c.st,
                    c.dw && two ? ws + s.x_back : nullptr, &units->x, power, &units->g, held);
  const char *w = s.copy_w ? ws + s.w : (const char*)c.w, *w_back = s.SCALED ? ws + s.w_back : w;   // dX's
  const int64_t w_ld = s.copy_w ? s.padded : c.w_ld, w_back_ld = s.SCALED ? s.padded : w_ld;
  void* const scaled_w = s.SCALED && c.dx ? ws + s.w_back : nullptr;
  if (s.copy_w || scaled_w)
    launch_gather<OP>(c.w, c.w_ld, c.w_t, c.width, nullptr, nullptr, c.vocab, nullptr, s.copy_w ? ws + s.w : nullptr, s.padded, c.st, scaled_w,
                      &units->w);
  // pass p: G of piece p, and the products of piece p - 1
  for (int64_t p = 0; p <= s.pieces; ++p) {
    LogitsCall g{};
    if (p < s.pieces) {
      g.w = w, g.w_ld = w_ld, g.x = ws + s.x, g.x_ld = s.padded, g.targets = c.targets, g.rows = c.rows, g.tokens = c.tokens;
      g.vocab = c.vocab, g.v0 = p * s.piece, g.v1 = std::min(g.v0 + s.piece, c.vocab), g.stages = (int)(s.padded / s.BK);
      g.lse = c.lse, g.factor = factor, g.held = held, g.g = ws + (p & 1 ? s.g2 : s.g), g.g_ld = s.piece;
    }
    ProductCall px{}, pw{};
    const int64_t v0 = (p - 1) * s.piece, v1 = std::min(v0 + s.piece, c.vocab);
    char* out = (char*)c.dw + v0 * c.width * lm_elem_size(c.w_t);
    if (p > 0) {
      px.a = pw.a = ws + (p & 1 ? s.g : s.g2), px.a_ld = pw.a_ld = s.piece, px.rows = pw.rows = c.rows, px.held = pw.held = held;
      px.b = w_back + v0 * w_back_ld * ES, px.b_ld = w_back_ld, px.n = px.b_cols = s.padded, px.k = v1 - v0;
      px.splits = s.splits_x, px.sums = (float*)(ws + s.dx), px.n_ld = s.padded, px.m_rows = s.held, px.add = p > 1;
      pw.b = x_back, pw.b_ld = pw.b_cols = s.padded, pw.m = v1 - v0, pw.n = c.width;
      pw.splits = p == s.pieces ? s.splits_last : s.splits_w, pw.lift = 1.f / BACK::LIFT, pw.units = units;
      if (pw.splits == 1) pw.out = out, pw.out_ld = c.width, pw.out_t = c.w_t;
      else pw.sums = (float*)(ws + s.dw), pw.n_ld = s.padded, pw.m_rows = s.piece;
    }
    const LogitsCall* pg = p < s.pieces ? &g : nullptr;
    const ProductCall *x = p > 0 && c.dx ? &px : nullptr, *y = p > 0 && c.dw ? &pw : nullptr;
    if (!(s.small        ? launch_pass<BACK, typename F::Small, typename B::SmallX, typename B::MiddleW>(pg, x, y, c.tokens, s.held, c.st)
          : s.large_pass ? launch_pass<BACK, typename F::Large, typename B::LargeX, typename B::LargeW>(pg, x, y, c.tokens, s.held, c.st)
                         : launch_pass<BACK, typename F::Middle, typename B::MiddleX, typename B::MiddleW>(pg, x, y, c.tokens, s.held, c.st)))
      return SA_ERR_ARGUMENT;
    if (y && pw.splits > 1)
      launch_finish(pw.sums, pw.splits, s.piece * s.padded, s.padded, nullptr, units, &units->from_x, 1.f / BACK::LIFT, nullptr, nullptr, 0, out, v1 - v0, c.width, c.w_t, c.st);
  }
  if (c.dx)
    launch_finish((float*)(ws + s.dx), s.splits_x, s.held * s.padded, s.padded, c.rows + ROWS_HEAD + c.tokens, units, &units->from_w,
                  1.f / BACK::LIFT, power, c.rows, held, c.dx, c.tokens, c.width, c.x_t, c.st);
  return launch_status();
}

}  // namespace
