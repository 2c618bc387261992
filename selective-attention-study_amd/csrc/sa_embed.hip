// Embedding lookup and its gradient (include/sa.h: sa_embedding).
//
//   y_i = a W[t_i];   dW_v = a (sum of dy_i over the tokens i with t_i = v), zero rows for ids that no token has
//
// The gradient goes by sorted tokens, so that each row is summed in token order by whoever owns it: no atomics, equal calls give
// equal bits, and an id that half of a batch has (padding, a frequent word) is summed by many wavefronts.
//   embed_sort   a workgroup owns RANGE ids and reads every token's id twice: to count its own (and the smaller ids, which
//                is where its part of the order begins), and to put its tokens' numbers in place. A count per id and
//                wavefront, each wavefront on a contiguous run of tokens, makes the order that of the tokens. No step needs
//                another workgroup's result, so there is one launch and no wait between workgroups; the price is that every
//                workgroup reads all ids (out of L2).
//   embed_sum    a wavefront sums CHUNK consecutive tokens of the order over 256 columns: ids that begin and end in the chunk
//                are written, what reaches over an end goes to the workspace; other workgroups of the launch clear the
//                rows of ids without tokens
//   embed_join   ids that reach over chunks: their parts, added in a fixed order
// Bound by memory: dy read once, dW written once.

#include "sa_lm.h"

namespace {

constexpr int RANGE = 256;       // ids of a sorting workgroup
constexpr int SORT_WAVES = 16;
constexpr int CHUNK = 32;        // tokens of a summing wavefront
constexpr int COLUMNS = 256;     // and its columns: four per lane

struct EmbedCall {
  const void* ids;
  const void* w;      // (forward) rows w_ld apart
  void* y;
  int64_t w_ld, dy_ld, tokens, vocab;
  const void* dy;
  void* dw;
  int* offsets;       // (vocab + 1) where each id's tokens begin in the order
  int* order;         // (tokens) token numbers by id, then by number
  float* part;        // [chunk][2][width]: what reaches in from the chunk before; what begins here and reaches on
  int width, dtype, ids64, chunks;
  float scale;
};

__device__ __forceinline__ int64_t id_at(const EmbedCall& c, int64_t i) {
  return c.ids64 ? ((const int64_t*)c.ids)[i] : (int64_t)((const int32_t*)c.ids)[i];
}

// ---------------------------------------------------------------------------------------------

// A thread per four elements; an id outside the table gives a row of NaN, as there is no row to read and nothing on the
// host knows of it.
template <bool VEC>
__global__ __launch_bounds__(NTHREADS) void embed_kernel(EmbedCall c) {
  const int per = (c.width + 3) / 4;
  const int64_t n = c.tokens * per;
  for (int64_t k = (int64_t)blockIdx.x * NTHREADS + threadIdx.x; k < n; k += (int64_t)gridDim.x * NTHREADS) {
    const int64_t i = k / per;
    const int q = (int)(k - i * per);
    const int e = VEC ? 4 * q : q, gap = VEC ? 1 : per;
    const int64_t id = id_at(c, i);
    float x[4];
    if (id >= 0 && id < c.vocab) {
      numbers<VEC>(fetch<VEC>(row_of(c.w, id, c.w_ld, c.dtype), c.dtype, e, gap, c.width), c.dtype, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] *= c.scale;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(0x7fc00000u);
    }
    put<VEC>(row_of(c.y, i, c.width, c.dtype), c.dtype, e, gap, c.width, x);
  }
}

// ---------------------------------------------------------------------------------------------

__global__ __launch_bounds__(64 * SORT_WAVES) void embed_sort_kernel(EmbedCall c) {
  __shared__ int count[SORT_WAVES][RANGE];   // tokens of an id in a wavefront's run; then where the next of them goes
  __shared__ int below[SORT_WAVES];
  __shared__ int scan[RANGE / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t lo = (int64_t)blockIdx.x * RANGE;
  const int ids = (int)min((int64_t)RANGE, c.vocab - lo);
  for (int k = threadIdx.x; k < SORT_WAVES * RANGE; k += 64 * SORT_WAVES) count[0][k] = 0;
  __syncthreads();
  const int run = (int)((c.tokens + 64 * SORT_WAVES - 1) / (64 * SORT_WAVES)) * 64;
  const int64_t first = (int64_t)wave * run, last = min(first + run, c.tokens);
  constexpr int AHEAD = 8;   // loads in flight
  int less = 0;
  for (int64_t i0 = first; i0 < last; i0 += 64 * AHEAD) {
    int64_t id[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int64_t i = i0 + 64 * u + lane;
      id[u] = i < last ? id_at(c, i) : -1;
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      less += id[u] >= 0 && id[u] < lo;
      if (id[u] >= lo && id[u] < lo + ids) atomicAdd(&count[wave][id[u] - lo], 1);   // (whole numbers: any order)
    }
  }
#pragma unroll
  for (int m = 32; m; m >>= 1) less += __shfl_xor(less, m);
  if (lane == 0) below[wave] = less;
  __syncthreads();
  // threads 0 .. RANGE - 1, an id each: where its tokens begin, and each wavefront's of them
  int total = 0, upto = 0;
  if (threadIdx.x < RANGE) {
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) total += count[w][threadIdx.x];
    upto = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    if (lane == 63) scan[wave] = upto;
  }
  __syncthreads();
  if (threadIdx.x < RANGE) {
    int at = upto - total;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) at += below[w];
    for (int w = 0; w < wave; ++w) at += scan[w];
    if ((int)threadIdx.x < ids) c.offsets[lo + threadIdx.x] = at;
    if (lo + ids == c.vocab && (int)threadIdx.x == ids - 1) c.offsets[c.vocab] = at + total;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      const int n = count[w][threadIdx.x];
      count[w][threadIdx.x] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int64_t i0 = first; i0 < last; i0 += 64 * AHEAD) {
    int64_t id[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int64_t i = i0 + 64 * u + lane;
      id[u] = i < last ? id_at(c, i) : -1;
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const bool mine = id[u] >= lo && id[u] < lo + ids;
      const int x = mine ? (int)(id[u] - lo) : -1;
      // the wavefront's tokens of one id at a time, in lane order
      for (uint64_t left = __ballot(mine); left;) {
        const int y = __builtin_amdgcn_readlane(x, (int)__builtin_ctzll(left));
        const uint64_t same = __ballot(x == y);
        const int at = count[wave][y];
        if (x == y) c.order[at + (int)__popcll(same & (((uint64_t)1 << lane) - 1))] = (int)(i0 + 64 * u + lane);
        if (lane == (int)__builtin_ctzll(same)) count[wave][y] = at + (int)__popcll(same);
        __asm__ volatile("" ::: "memory");   // (a wavefront's own LDS accesses run in order)
        left &= ~same;
      }
    }
  }
}

// Sums of CHUNK tokens; blockIdx.x counts wavefront-sized pieces of work: chunks x column blocks, then rows to clear.
template <bool VEC>
__global__ __launch_bounds__(NTHREADS) void embed_sum_kernel(EmbedCall c, int blocks, int64_t pieces) {
  const int lane = threadIdx.x & 63;
  const int64_t piece = (int64_t)blockIdx.x * NWAVES + (threadIdx.x >> 6);
  if (piece >= pieces) {   // clear the rows of 64 ids that have no token
    const int64_t v0 = (piece - pieces) * 64;
    if (v0 >= c.vocab) return;
    const int64_t v = min(v0 + lane, c.vocab - 1);
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint64_t none = __ballot(v0 + lane < c.vocab && c.offsets[v] == c.offsets[v + 1]); none; none &= none - 1) {
      void* row = row_of(c.dw, v0 + (int)__builtin_ctzll(none), c.width, c.dtype);
      for (int e = VEC ? 4 * lane : lane; e < c.width; e += 256) put<VEC>(row, c.dtype, e, 64, c.width, zero);
    }
    return;
  }
  const int chunk = (int)(piece / blocks), block = (int)(piece - (int64_t)chunk * blocks);
  const int total = c.offsets[c.vocab];
  const int a = chunk * CHUNK, b = min(a + CHUNK, total);
  if (a >= b) return;
  const int e = block * COLUMNS + (VEC ? 4 * lane : lane);
  // lane l < CHUNK looks up token l of the chunk and its id's bounds
  int token = 0, id = -1, begin = 0, end = 0;
  if (a + lane < b) {
    token = c.order[a + lane];
    id = (int)id_at(c, token);
    begin = c.offsets[id], end = c.offsets[id + 1];
  }
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  constexpr int AHEAD = 8;
  for (int k0 = 0; k0 < b - a; k0 += AHEAD) {
    Quad q[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int t = __builtin_amdgcn_readlane(token, min(k0 + u, CHUNK - 1));
      q[u] = fetch<VEC>(row_of(c.dy, t, c.dy_ld, c.dtype), c.dtype, e, 64, k0 + u < b - a ? c.width : 0);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = k0 + u;
      if (k >= b - a) break;
      float x[4];
      numbers<VEC>(q[u], c.dtype, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += x[j];
      const int i = __builtin_amdgcn_readlane(id, k), s0 = __builtin_amdgcn_readlane(begin, k), s1 = __builtin_amdgcn_readlane(end, k);
      if (a + k + 1 < min(s1, b)) continue;   // the id goes on
      if (s0 >= a && s1 <= b) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] *= c.scale;
        put<VEC>(row_of(c.dw, i, c.width, c.dtype), c.dtype, e, 64, c.width, sum);
      } else {
        put<VEC>(c.part + ((int64_t)chunk * 2 + (s0 >= a)) * c.width, SA_DTYPE_F32, e, 64, c.width, sum);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = 0.f;
    }
  }
}

// The id that begins in chunk blockIdx.x and reaches past its end: its parts here and in the chunks it reaches into, every
// JOIN_WAVES-th by one wavefront, then added in order.
constexpr int JOIN_WAVES = 8;
template <bool VEC>
__global__ __launch_bounds__(64 * JOIN_WAVES) void embed_join_kernel(EmbedCall c, int blocks) {
  __shared__ float acc[JOIN_WAVES][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int chunk = blockIdx.x / blocks, block = blockIdx.x - chunk * blocks;
  const int total = c.offsets[c.vocab];
  const int a = chunk * CHUNK, b = a + CHUNK;
  if (b >= total) return;
  const int id = (int)id_at(c, c.order[b - 1]);
  const int begin = c.offsets[id], end = c.offsets[id + 1];
  if (begin < a || end <= b) return;
  const int parts = 1 + (end - b + CHUNK - 1) / CHUNK;   // part 0: this chunk's second, then the first of those that follow
  const int e = block * COLUMNS + (VEC ? 4 * lane : lane);
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  constexpr int AHEAD = 8;
  for (int k0 = wave; k0 < parts; k0 += JOIN_WAVES * AHEAD) {
    Quad q[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = k0 + u * JOIN_WAVES;
      q[u] = fetch<VEC>(c.part + ((int64_t)(chunk + min(k, parts - 1)) * 2 + (k == 0)) * c.width, SA_DTYPE_F32, e, 64, k < parts ? c.width : 0);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      float x[4];
      numbers<VEC>(q[u], SA_DTYPE_F32, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += x[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[wave][j][lane] = sum[j];
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < JOIN_WAVES; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] += acc[w][j][lane];
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] *= c.scale;
  put<VEC>(row_of(c.dw, id, c.width, c.dtype), c.dtype, e, 64, c.width, sum);
}

bool embed_sizes_ok(int64_t tokens, int64_t vocab, int64_t width) {
  return tokens >= 0 && tokens < ((int64_t)1 << 30) && vocab >= 1 && vocab < ((int64_t)1 << 28) && width >= 1 && width < ((int64_t)1 << 24);
}

struct EmbedSpace {
  int64_t offsets, order, part, total, chunks;
  EmbedSpace(int64_t tokens, int64_t vocab, int64_t width) {
    chunks = cdiv(tokens, CHUNK);
    offsets = 0;
    order = offsets + align_up(4 * (vocab + 1), 256);
    part = order + align_up(4 * tokens, 256);
    total = part + align_up(chunks * 2 * width * 4, 256);
  }
};

}  // namespace

extern "C" {

int sa_embedding(const void* ids, int ids_bytes, const void* weight, int64_t weight_ld, void* out, int64_t tokens, int64_t vocab,
                 int64_t width, float scale, int dtype, void* stream) {
  const int64_t es = lm_elem_size(dtype);
  if (!es) return SA_ERR_DTYPE;
  if (!embed_sizes_ok(tokens, vocab, width) || (ids_bytes != 4 && ids_bytes != 8) || weight_ld < 0 || weight_ld >= ((int64_t)1 << 31))
    return SA_ERR_ARGUMENT;
  if (tokens == 0) return SA_OK;
  if (!ids || (uintptr_t)ids % ids_bytes || !weight || !out || (uintptr_t)weight % es || (uintptr_t)out % es) return SA_ERR_ARGUMENT;
  EmbedCall c{};
  c.ids = ids, c.ids64 = ids_bytes == 8, c.w = weight, c.w_ld = weight_ld, c.y = out, c.tokens = tokens, c.vocab = vocab;
  c.width = (int)width, c.scale = scale, c.dtype = dtype;
  const bool vec = width % 4 == 0 && quads_ok(weight, weight_ld, dtype) && quads_ok(out, width, dtype);
  const int64_t blocks = std::min<int64_t>(cdiv(tokens * cdiv(width, 4), NTHREADS), LAUNCH_BLOCKS);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (vec) hipLaunchKernelGGL((embed_kernel<true>), dim3((unsigned)blocks), dim3(NTHREADS), 0, st, c);
  else hipLaunchKernelGGL((embed_kernel<false>), dim3((unsigned)blocks), dim3(NTHREADS), 0, st, c);
  return launch_status();
}

int64_t sa_embedding_backward_workspace_bytes(int64_t tokens, int64_t vocab, int64_t width) {
  if (!embed_sizes_ok(tokens, vocab, width)) return -1;
  return EmbedSpace(tokens, vocab, width).total;
}

int sa_embedding_backward(const void* ids, int ids_bytes, const void* dout, int64_t dout_ld, void* dweight, void* workspace,
                          int64_t workspace_bytes, int64_t tokens, int64_t vocab, int64_t width, float scale, int dtype,
                          void* stream) {
  const int64_t es = lm_elem_size(dtype);
  if (!es) return SA_ERR_DTYPE;
  if (!embed_sizes_ok(tokens, vocab, width) || (ids_bytes != 4 && ids_bytes != 8) || dout_ld < 0 || dout_ld >= ((int64_t)1 << 31))
    return SA_ERR_ARGUMENT;
  if (!dweight || (uintptr_t)dweight % es || (tokens > 0 && (!ids || (uintptr_t)ids % ids_bytes || !dout || (uintptr_t)dout % es)))
    return SA_ERR_ARGUMENT;
  const EmbedSpace ws(tokens, vocab, width);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < ws.total) return SA_ERR_WORKSPACE;
  const int64_t blocks = cdiv(width, COLUMNS), pieces = ws.chunks * blocks, clears = cdiv(vocab, 64);
  if (cdiv(pieces + clears, NWAVES) >= ((int64_t)1 << 24) || pieces >= ((int64_t)1 << 23)) return SA_ERR_ARGUMENT;   // 2^32 threads
  EmbedCall c{};
  c.ids = ids, c.ids64 = ids_bytes == 8, c.dy = dout, c.dy_ld = dout_ld, c.dw = dweight, c.tokens = tokens, c.vocab = vocab;
  c.width = (int)width, c.scale = scale, c.dtype = dtype, c.chunks = (int)ws.chunks;
  c.offsets = (int*)((char*)workspace + ws.offsets);
  c.order = (int*)((char*)workspace + ws.order);
  c.part = (float*)((char*)workspace + ws.part);
  const bool vec = width % 4 == 0 && quads_ok(dout, dout_ld, dtype) && quads_ok(dweight, width, dtype);
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(embed_sort_kernel, dim3((unsigned)cdiv(vocab, RANGE)), dim3(64 * SORT_WAVES), 0, st, c);
  const dim3 sums((unsigned)cdiv(pieces + clears, NWAVES));
  if (vec) hipLaunchKernelGGL((embed_sum_kernel<true>), sums, dim3(NTHREADS), 0, st, c, (int)blocks, pieces);
  else hipLaunchKernelGGL((embed_sum_kernel<false>), sums, dim3(NTHREADS), 0, st, c, (int)blocks, pieces);
  if (tokens > CHUNK) {
    const dim3 joins((unsigned)pieces);
    if (vec) hipLaunchKernelGGL((embed_join_kernel<true>), joins, dim3(64 * JOIN_WAVES), 0, st, c, (int)blocks);
    else hipLaunchKernelGGL((embed_join_kernel<false>), joins, dim3(64 * JOIN_WAVES), 0, st, c, (int)blocks);
  }
  return launch_status();
}

}  // extern "C"
