// Embedding lookup and its gradient (include/sa.h: sa_embedding).
//
//   y_i = a W[t_i];   dW_v = a (sum of dy_i over the tokens i with t_i = v), zero rows for ids that no token has
//
// The gradient goes by sorted tokens, so that each row is summed in token order by whoever owns it: no atomics, equal calls give
// equal bits, and an id that half of a batch has (padding, a frequent word) is summed by many wavefronts.
//   embed_split  pieces of SPLIT tokens, each put in the order of the last 8 bits of its ids (256 buckets: neighbouring ids, whose
//                frequencies are alike in most vocabularies, fall into different ones)
//   embed_place  a workgroup per bucket (and RANGE ids of it) takes that bucket's tokens of all pieces, a contiguous run of pieces per
//                wavefront, counts each id's per wavefront, and puts the tokens' numbers in place, each id's in token order
//   embed_sum    a wavefront sums CHUNK consecutive tokens of the order over 256 columns: ids that begin and end in the chunk
//                are written, what reaches over an end goes to the workspace; other workgroups of the launch clear the
//                rows of ids without tokens
//   embed_join   ids that reach over chunks: their parts, added in a fixed order
// Bound by memory: dy read once, dW written once. Measured, us, lookup / split / place / sum / join: 16384 tokens of a text, 50304 x 768
// fp32 17 / 7 / 8 / 43 (4.8 TB/s) / 4; 50003 tokens, half of them one id, 50304 x 512 bf16 18 / 6 / 28 / 21 / 13.

#include "sa_lm.h"

namespace {

constexpr int BUCKETS = 256;
constexpr int SPLIT = 2048;      // tokens of a piece that embed_split orders
constexpr int RANGE = 1024;      // ids of an embed_place workgroup
constexpr int PLACE_WAVES = 16;
constexpr int CHUNK = 32;        // tokens of a summing wavefront
constexpr int COLUMNS = 256;     // and its columns: four per lane

struct EmbedCall {
  const void* ids;
  const void* w;      // (forward) rows w_ld apart
  void* y;
  int64_t w_ld, dy_ld, tokens, vocab;
  const void* dy;
  void* dw;
  int* heads;         // [piece][BUCKETS + 1] where a bucket's tokens begin in the piece
  int2* pairs;        // (id / BUCKETS, token) by piece and bucket
  int2* spans;        // (vocab) where each id's tokens begin and end in the order
  int* order;         // (tokens) token numbers, each id's together and in order; then how many there are
  float* part;        // [chunk][2][width]: what reaches in from the chunk before; what begins here and reaches on
  int width, dtype, ids64, chunks, splits;
  float scale;
};

__device__ __forceinline__ int64_t id_at(const EmbedCall& c, int64_t i) {
  return c.ids64 ? ((const int64_t*)c.ids)[i] : (int64_t)((const int32_t*)c.ids)[i];
}

// ---------------------------------------------------------------------------------------------

// 1 << shift lanes a row (as many as have four elements each, up to a wavefront); an id outside the table gives a row of NaN, as
// there is no row to read and nothing on the host knows of it.
template <bool VEC>
__global__ __launch_bounds__(NTHREADS) void embed_kernel(EmbedCall c, int shift) {
  const int lanes = 1 << shift, lane = threadIdx.x & (lanes - 1);
  const int rows = NTHREADS >> shift;
  for (int64_t i = (int64_t)blockIdx.x * rows + (threadIdx.x >> shift); i < c.tokens; i += (int64_t)gridDim.x * rows) {
    const int64_t id = id_at(c, i);
    const bool real = id >= 0 && id < c.vocab;
    const void* from = row_of(c.w, real ? id : 0, c.w_ld, c.dtype);
    void* to = row_of(c.y, i, c.width, c.dtype);
    constexpr int AHEAD = 4;   // loads in flight
    for (int e0 = VEC ? 4 * lane : lane; e0 < c.width; e0 += 4 * lanes * AHEAD) {
      Quad q[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) q[u] = fetch<VEC>(from, c.dtype, e0 + 4 * lanes * u, lanes, real ? c.width : 0);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        float x[4];
        numbers<VEC>(q[u], c.dtype, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = real ? x[j] * c.scale : __uint_as_float(0x7fc00000u);
        put<VEC>(to, c.dtype, e0 + 4 * lanes * u, lanes, c.width, x);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------

__global__ __launch_bounds__(NTHREADS) void embed_split_kernel(EmbedCall c) {
  __shared__ int count[NWAVES][BUCKETS];   // a wavefront's tokens of a bucket so far; then where its first goes
  __shared__ int scan[NWAVES];
  static_assert(NTHREADS == BUCKETS, "a thread per bucket");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int EACH = SPLIT / NTHREADS;
  const int64_t first = (int64_t)blockIdx.x * SPLIT + wave * (64 * EACH) + lane;
  int64_t id[EACH];
#pragma unroll
  for (int u = 0; u < EACH; ++u) id[u] = first + 64 * u < c.tokens ? id_at(c, first + 64 * u) : -1;
  for (int k = threadIdx.x; k < NWAVES * BUCKETS; k += NTHREADS) count[0][k] = 0;
  __syncthreads();
  int bucket[EACH], rank[EACH];
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    const bool real = id[u] >= 0 && id[u] < c.vocab;
    const int b = (int)id[u] & (BUCKETS - 1);
    uint64_t same = __ballot(real);   // the lanes of the same bucket
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const uint64_t ones = __ballot((b >> bit) & 1);
      same &= (b >> bit) & 1 ? ones : ~ones;
    }
    const uint64_t before = same & (((uint64_t)1 << lane) - 1);
    bucket[u] = real ? b : -1;
    if (real) rank[u] = count[wave][b] + (int)__popcll(before);
    __asm__ volatile("" ::: "memory");   // (a wavefront's own LDS accesses run in order)
    if (real && before == 0) count[wave][b] += (int)__popcll(same);
    __asm__ volatile("" ::: "memory");
  }
  __syncthreads();
  const int b = threadIdx.x;
  int total = 0;
#pragma unroll
  for (int w = 0; w < NWAVES; ++w) total += count[w][b];
  int upto = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(upto, d);
    if (lane >= d) upto += v;
  }
  if (lane == 63) scan[wave] = upto;
  __syncthreads();
  int at = upto - total;
  for (int w = 0; w < wave; ++w) at += scan[w];
  int* heads = c.heads + (int64_t)blockIdx.x * (BUCKETS + 1);
  heads[b] = at;
  if (b == BUCKETS - 1) heads[BUCKETS] = at + total;
#pragma unroll
  for (int w = 0; w < NWAVES; ++w) {
    const int n = count[w][b];
    count[w][b] = at;
    at += n;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < EACH; ++u)
    if (bucket[u] >= 0)
      c.pairs[(int64_t)blockIdx.x * SPLIT + count[wave][bucket[u]] + rank[u]] = make_int2((int)(id[u] >> 8), (int)(first + 64 * u));
}

__global__ __launch_bounds__(64 * PLACE_WAVES) void embed_place_kernel(EmbedCall c) {
  __shared__ int count[PLACE_WAVES][RANGE];   // tokens of an id in a wavefront's pieces; then where the next of them goes
  __shared__ int below[PLACE_WAVES], scan[PLACE_WAVES];
  static_assert(RANGE == 64 * PLACE_WAVES, "a thread per id");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int bucket = blockIdx.x, lo = blockIdx.y * RANGE;
  for (int k = threadIdx.x; k < PLACE_WAVES * RANGE; k += 64 * PLACE_WAVES) count[0][k] = 0;
  __syncthreads();
  const int per = (c.splits + PLACE_WAVES - 1) / PLACE_WAVES;
  const int first = wave * per, last = min(first + per, c.splits);
  // visit(pair, real): the wavefront's tokens of the bucket in order, 64 at a time. 64 pieces a round: lane l holds piece l's
  // part, and the lanes find the piece of their token among the parts' ends.
  constexpr int AHEAD = 8;   // loads in flight
  const auto walk = [&](auto&& visit, int& less) {
    for (int p0 = first; p0 < last; p0 += 64) {
      const int pieces = min(64, last - p0);
      int begin = 0, n = 0;
      if (lane < pieces) {
        const int* heads = c.heads + (int64_t)(p0 + lane) * (BUCKETS + 1) + bucket;
        begin = heads[0];
        n = heads[1] - begin;
        less += begin;   // (the piece's tokens of the buckets before)
      }
      int ends = n;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(ends, d);
        if (lane >= d) ends += v;
      }
      const int all = __builtin_amdgcn_readlane(ends, 63);
      const int offset = (p0 + lane) * SPLIT + begin - (ends - n);   // of the flat numbers of this piece's tokens
      for (int k0 = 0; k0 < all; k0 += 64 * AHEAD) {
        int2 pair[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          if (k0 + 64 * u >= all) break;
          const int k = k0 + 64 * u + lane;
          int piece = 0;
          for (int j = 0; j < pieces - 1; ++j) piece += k >= __builtin_amdgcn_readlane(ends, j);
          const int at = __shfl(offset, piece) + k;
          pair[u] = k < all ? c.pairs[at] : make_int2(0, 0);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          if (k0 + 64 * u >= all) break;
          visit(pair[u], k0 + 64 * u + lane < all);
        }
      }
    }
  };
  int less = 0;   // tokens of ids that come before this workgroup's
  walk([&](int2 pair, bool real) {
    less += real && pair.x < lo;
    const int x = real && pair.x >= lo && pair.x < lo + RANGE ? pair.x - lo : -1;
    // the first token's id at once (additions to one number run one after the other: 50003 tokens of
    // one id took 73 us instead of 47), the others' by additions of whole numbers, whose order does not matter
    const uint64_t some = __ballot(x >= 0);
    if (!some) return;
    const int leader = (int)__builtin_ctzll(some), y = __builtin_amdgcn_readlane(x, leader);
    const uint64_t same = __ballot(x == y);
    if (lane == leader) atomicAdd(&count[wave][y], (int)__popcll(same));
    else if (x >= 0 && x != y) atomicAdd(&count[wave][x], 1);
  }, less);
#pragma unroll
  for (int m = 32; m; m >>= 1) less += __shfl_xor(less, m);
  if (lane == 0) below[wave] = less;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < PLACE_WAVES; ++w) total += count[w][threadIdx.x];
  int upto = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(upto, d);
    if (lane >= d) upto += v;
  }
  if (lane == 63) scan[wave] = upto;
  __syncthreads();
  int at = upto - total;
#pragma unroll
  for (int w = 0; w < PLACE_WAVES; ++w) at += below[w] + (w < wave ? scan[w] : 0);
  const int64_t id = ((int64_t)lo + threadIdx.x) * BUCKETS + bucket;
  if (id < c.vocab) c.spans[id] = make_int2(at, at + total);
  if (bucket == BUCKETS - 1 && blockIdx.y == gridDim.y - 1 && threadIdx.x == RANGE - 1) c.order[c.tokens] = at + total;
#pragma unroll
  for (int w = 0; w < PLACE_WAVES; ++w) {
    const int n = count[w][threadIdx.x];
    count[w][threadIdx.x] = at;
    at += n;
  }
  __syncthreads();
  walk([&](int2 pair, bool real) {
    const int x = real && pair.x >= lo && pair.x < lo + RANGE ? pair.x - lo : -1;
    // the tokens of one id at a time, in lane order
    for (uint64_t left = __ballot(x >= 0); left;) {
      const int leader = (int)__builtin_ctzll(left), y = __builtin_amdgcn_readlane(x, leader);
      const uint64_t same = __ballot(x == y);
      const int to = count[wave][y];
      if (x == y) c.order[to + (int)__popcll(same & (((uint64_t)1 << lane) - 1))] = pair.y;
      __asm__ volatile("" ::: "memory");   // (a wavefront's own LDS accesses run in order)
      if (lane == leader) count[wave][y] = to + (int)__popcll(same);
      __asm__ volatile("" ::: "memory");
      left &= ~same;
    }
  }, less);
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
    const int2 span = c.spans[v];
    for (uint64_t none = __ballot(v0 + lane < c.vocab && span.x == span.y); none; none &= none - 1) {
      void* row = row_of(c.dw, v0 + (int)__builtin_ctzll(none), c.width, c.dtype);
      for (int e = VEC ? 4 * lane : lane; e < c.width; e += 256) put<VEC>(row, c.dtype, e, 64, c.width, zero);
    }
    return;
  }
  const int chunk = (int)(piece / blocks), block = (int)(piece - (int64_t)chunk * blocks);
  const int total = c.order[c.tokens];
  const int a = chunk * CHUNK, b = min(a + CHUNK, total);
  if (a >= b) return;
  const int e = block * COLUMNS + (VEC ? 4 * lane : lane);
  // lane l < CHUNK looks up token l of the chunk and its id's bounds
  int token = 0, id = -1, begin = 0, end = 0;
  if (a + lane < b) {
    token = c.order[a + lane];
    id = (int)id_at(c, token);
    const int2 span = c.spans[id];
    begin = span.x, end = span.y;
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
  const int total = c.order[c.tokens];
  const int a = chunk * CHUNK, b = a + CHUNK;
  if (b >= total) return;
  const int id = (int)id_at(c, c.order[b - 1]);
  const int2 span = c.spans[id];
  const int begin = span.x, end = span.y;
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
  int64_t heads, pairs, spans, order, part, total, chunks, splits;
  EmbedSpace(int64_t tokens, int64_t vocab, int64_t width) {
    chunks = cdiv(tokens, CHUNK);
    splits = cdiv(tokens, SPLIT);
    heads = 0;
    pairs = heads + align_up(splits * (BUCKETS + 1) * 4, 256);
    spans = pairs + splits * SPLIT * 8;
    order = spans + align_up(8 * vocab, 256);
    part = order + align_up(4 * (tokens + 1), 256);
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
  int shift = 0;
  while (shift < 6 && (4 << shift) < width) ++shift;
  const int64_t blocks = std::min<int64_t>(cdiv(tokens, NTHREADS >> shift), LAUNCH_BLOCKS);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (vec) hipLaunchKernelGGL((embed_kernel<true>), dim3((unsigned)blocks), dim3(NTHREADS), 0, st, c, shift);
  else hipLaunchKernelGGL((embed_kernel<false>), dim3((unsigned)blocks), dim3(NTHREADS), 0, st, c, shift);
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
  c.splits = (int)ws.splits;
  c.heads = (int*)((char*)workspace + ws.heads);
  c.pairs = (int2*)((char*)workspace + ws.pairs);
  c.spans = (int2*)((char*)workspace + ws.spans);
  c.order = (int*)((char*)workspace + ws.order);
  c.part = (float*)((char*)workspace + ws.part);
  const bool vec = width % 4 == 0 && quads_ok(dout, dout_ld, dtype) && quads_ok(dweight, width, dtype);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (tokens > 0) hipLaunchKernelGGL(embed_split_kernel, dim3((unsigned)ws.splits), dim3(NTHREADS), 0, st, c);
  hipLaunchKernelGGL(embed_place_kernel, dim3(BUCKETS, (unsigned)cdiv(cdiv(vocab, BUCKETS), RANGE)), dim3(64 * PLACE_WAVES), 0, st, c);
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
