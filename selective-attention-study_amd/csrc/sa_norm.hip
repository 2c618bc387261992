// Layer norm over rows, alone or after a residual addition, and its backward pass (include/sa.h: sa_layer_norm).
//
//   s = x + branch (rounded to x's type: it is the next block's stream, and the norm is that stream's), s = x without one
//   y = w h + b,  h = (s - mean) r,  r = 1 / sqrt(var + eps)
//   dx = dbranch = r (u - mean(u) - h mean(u h)) + ds,  u = dy w;   dw = sum over rows of dy h,  db = sum of dy
//
// Bound by memory: the forward reads x and branch and writes y and s once, the backward reads s, dy and ds and writes dx once. A row
// stays in the registers of the lanes that loaded it (a wavefront up to 1024 wide, a workgroup of 4 to 16 wavefronts beyond), so its mean
// and the sum of its squared deviations are two exact passes over registers, not a difference of sums. Everything is fp32 in
// between; outputs are rounded once.
//
// The weights' gradients: a workgroup walks over rows a fixed stride apart and keeps its sums in registers, its wavefronts'
// are added in LDS, and norm_join adds the workgroups' rows of sums in a fixed order. No atomics: equal calls give equal bits.
//
// Measured: 16384 x 768, fp32 stream, bf16 branch and result, forward 31 us (4.8 TB/s), backward 44 (4.6 TB/s) and 4 for the join; 2048 x 8192 bf16
// 30, 38 and 4; 5003 x 1001 fp32 13, 22 and 4. A copy of 4 GiB runs at 4.7 TB/s. Wider than 8192, 1024 threads leave 128 registers each and the rest
// spills: 2048 x 12000 bf16 70 and with gradients 268, 1024 x 32768 127 and 613 (their bytes at that rate 42 and 84, 57 and 114).

#include <math.h>

#include "sa_lm.h"

namespace {

struct NormCall {
  const void *x, *branch, *w, *b, *dy, *ds;
  void *y, *s, *dx, *dbranch;
  float *mean, *rstd, *part;
  int64_t x_ld, branch_ld, dy_ld, ds_ld, rows;
  int width, x_t, branch_t, y_t, w_t, sums;   // sums: rows of part (dw, db)
  float eps;
};

// the sum over the G lanes that share a row
template <int G>
__device__ __forceinline__ float row_sum(float x, float* red) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
  if constexpr (G > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();   // (the sums of the call before have been read)
    if ((threadIdx.x & 63) == 0) red[wave] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int i = 0; i < G / 64; ++i) x += red[i];
  }
  return x;
}

template <int G>
constexpr int norm_threads() { return G == 64 ? NTHREADS : G; }

// Element indices of lane `lane`'s quad v among G lanes: neighbours (VEC), or G apart.
template <int G, bool VEC>
__device__ __forceinline__ int first_of(int v, int lane) { return VEC ? (v * G + lane) * 4 : v * 4 * G + lane; }

// Rows that a workgroup shares: as many workgroups as fit on the chip walk over them with the weights in registers and the next row's
// loads under way (us, with a workgroup per row: 2048 x 8192 bf16 30, 44; 4096 x 4096 29, 34; up to 2048 wide and for a wavefront's rows
// there are enough of them on a CU without: 8192 and 16384 x 2048 together 42, 39).
template <int G, int V>
constexpr bool norm_walks() { return (G == 256 || G == 512) && V == 4; }

template <int G, int V, bool VEC>
__global__ __launch_bounds__(norm_threads<G>(), (norm_walks<G, V>() ? 4 : 1)) void norm_kernel(NormCall c) {
  __shared__ float red[G / 64];
  constexpr int PER = norm_threads<G>() / G;
  constexpr bool WALK = norm_walks<G, V>();
  const int lane = threadIdx.x % G;
  const int64_t stride = (int64_t)gridDim.x * PER;
  Quad qx[V], qb[V];
  const auto load = [&](int64_t row) {
    const void* xr = row_of(c.x, row, c.x_ld, c.x_t);
#pragma unroll
    for (int v = 0; v < V; ++v) qx[v] = fetch<VEC>(xr, c.x_t, first_of<G, VEC>(v, lane), G, c.width);
    if (c.branch) {
      const void* br = row_of(c.branch, row, c.branch_ld, c.branch_t);
#pragma unroll
      for (int v = 0; v < V; ++v) qb[v] = fetch<VEC>(br, c.branch_t, first_of<G, VEC>(v, lane), G, c.width);
    }
  };
  int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / G;
  float w[V][4], b[V][4];
  const auto weights = [&](int v) {
    const int e = first_of<G, VEC>(v, lane);
    numbers<VEC>(fetch<VEC>(c.w, c.w_t, e, G, c.width), c.w_t, w[v]);
#pragma unroll
    for (int j = 0; j < 4; ++j) b[v][j] = 0.f;
    if (c.b) numbers<VEC>(fetch<VEC>(c.b, c.w_t, e, G, c.width), c.w_t, b[v]);
  };
  if constexpr (WALK) {
    if (row < c.rows) load(row);
#pragma unroll
    for (int v = 0; v < V; ++v) weights(v);
  }
  for (; row < c.rows; row += stride) {
    if constexpr (!WALK) load(row);
    float s[V][4];
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      numbers<VEC>(qx[v], c.x_t, s[v]);
      if (c.branch) {
        float d[4];
        numbers<VEC>(qb[v], c.branch_t, d);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[v][j] = stored(s[v][j] + d[j], c.x_t);
        put<VEC>(row_of(c.s, row, c.width, c.x_t), c.x_t, first_of<G, VEC>(v, lane), G, c.width, s[v]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += s[v][j];
    }
    if (WALK && row + stride < c.rows) load(row + stride);
    const float mean = row_sum<G>(sum, red) / (float)c.width;
    float square = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = first_of<G, VEC>(v, lane) + (VEC ? j : j * G);
        s[v][j] -= mean;
        square += e < c.width ? s[v][j] * s[v][j] : 0.f;
      }
    const float r = 1.f / sqrtf(row_sum<G>(square, red) / (float)c.width + c.eps);
    if (c.mean && lane == 0) c.mean[row] = mean, c.rstd[row] = r;
    void* yr = row_of(c.y, row, c.width, c.y_t);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if constexpr (!WALK) weights(v);
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = s[v][j] * r * w[v][j] + b[v][j];
      put<VEC>(yr, c.y_t, first_of<G, VEC>(v, lane), G, c.width, y);
    }
  }
}

template <int G, int V, bool VEC>
__global__ __launch_bounds__(norm_threads<G>()) void norm_backward_kernel(NormCall c) {
  __shared__ float red[G / 64];
  constexpr int PER = norm_threads<G>() / G;
  const int lane = threadIdx.x % G;
  float w[V][4], dw[V][4], db[V][4];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    numbers<VEC>(fetch<VEC>(c.w, c.w_t, first_of<G, VEC>(v, lane), G, c.width), c.w_t, w[v]);
#pragma unroll
    for (int j = 0; j < 4; ++j) dw[v][j] = db[v][j] = 0.f;
  }
  Quad qs[V], qy[V], qd[V];
  const auto load = [&](int64_t row) {
    const void *sr = row_of(c.x, row, c.x_ld, c.x_t), *yr = row_of(c.dy, row, c.dy_ld, c.y_t);
#pragma unroll
    for (int v = 0; v < V; ++v) qs[v] = fetch<VEC>(sr, c.x_t, first_of<G, VEC>(v, lane), G, c.width);
#pragma unroll
    for (int v = 0; v < V; ++v) qy[v] = fetch<VEC>(yr, c.y_t, first_of<G, VEC>(v, lane), G, c.width);
    if (c.ds) {
      const void* dr = row_of(c.ds, row, c.ds_ld, c.x_t);
#pragma unroll
      for (int v = 0; v < V; ++v) qd[v] = fetch<VEC>(dr, c.x_t, first_of<G, VEC>(v, lane), G, c.width);
    }
  };
  // Rows that a workgroup shares: the next one's loads are under way while one is worked on (2048 x 8192 bf16: 53 -> 38 us). Rows of
  // a wavefront have other wavefronts for that, and lose more of them to the registers (16384 x 768: 43 -> 52 us).
  constexpr bool AHEAD = G > 64 && G < 1024;
  const int64_t stride = (int64_t)gridDim.x * PER;
  int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / G;
  if (AHEAD && row < c.rows) load(row);
  for (; row < c.rows; row += stride) {
    if (!AHEAD) load(row);
    const float mean = c.mean[row], r = c.rstd[row];
    float h[V][4], u[V][4], d[V][4];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      numbers<VEC>(qs[v], c.x_t, h[v]);
      numbers<VEC>(qy[v], c.y_t, u[v]);
#pragma unroll
      for (int j = 0; j < 4; ++j) d[v][j] = 0.f;
      if (c.ds) numbers<VEC>(qd[v], c.x_t, d[v]);
    }
    if (AHEAD && row + stride < c.rows) load(row + stride);
    float su = 0.f, suh = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = first_of<G, VEC>(v, lane) + (VEC ? j : j * G);
        h[v][j] = e < c.width ? (h[v][j] - mean) * r : 0.f;
        dw[v][j] += u[v][j] * h[v][j];
        db[v][j] += u[v][j];
        u[v][j] *= w[v][j];
        su += u[v][j];
        suh += u[v][j] * h[v][j];
      }
    }
    const float mu = row_sum<G>(su, red) / (float)c.width, muh = row_sum<G>(suh, red) / (float)c.width;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = first_of<G, VEC>(v, lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) d[v][j] += r * (u[v][j] - mu - h[v][j] * muh);
      if (c.dx) put<VEC>(row_of(c.dx, row, c.width, c.x_t), c.x_t, e, G, c.width, d[v]);
      if (c.dbranch) put<VEC>(row_of(c.dbranch, row, c.width, c.branch_t), c.branch_t, e, G, c.width, d[v]);
    }
  }
  if (!c.part) return;
  // part[workgroup][sums][width]: the wavefronts' sums are added in order
  float* mine = c.part + (int64_t)blockIdx.x * c.sums * c.width;
  if constexpr (PER == 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      put<VEC>(mine, SA_DTYPE_F32, first_of<G, VEC>(v, lane), G, c.width, dw[v]);
      if (c.sums > 1) put<VEC>(mine + c.width, SA_DTYPE_F32, first_of<G, VEC>(v, lane), G, c.width, db[v]);
    }
  } else {
    __shared__ float acc[2][V * 4][64];
    for (int k = 0; k < PER; ++k) {
      if ((int)threadIdx.x / G == k) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[0][v * 4 + j][lane] = k ? acc[0][v * 4 + j][lane] + dw[v][j] : dw[v][j];
            acc[1][v * 4 + j][lane] = k ? acc[1][v * 4 + j][lane] + db[v][j] : db[v][j];
          }
      }
      __syncthreads();
    }
    if (threadIdx.x < G) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a[4], b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = acc[0][v * 4 + j][lane], b[j] = acc[1][v * 4 + j][lane];
        put<VEC>(mine, SA_DTYPE_F32, first_of<G, VEC>(v, lane), G, c.width, a);
        if (c.sums > 1) put<VEC>(mine + c.width, SA_DTYPE_F32, first_of<G, VEC>(v, lane), G, c.width, b);
      }
    }
  }
}

// dw, db from the workgroups' sums: 16 rows of lanes take every 16th workgroup each, and are added in order.
__global__ __launch_bounds__(1024) void norm_join_kernel(const float* part, int parts, int width, void* dw, void* db, int w_t) {
  __shared__ float acc[16][64];
  const int x = threadIdx.x & 63, k = threadIdx.x >> 6;
  const int e = blockIdx.x * 64 + x;
  float sum = 0.f;
  if (e < width) {
    const float* p = part + (int64_t)blockIdx.y * width + e;
#pragma unroll 8
    for (int i = k; i < parts; i += 16) sum += p[(int64_t)i * gridDim.y * width];
  }
  acc[k][x] = sum;
  __syncthreads();
  if (k != 0 || e >= width) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += acc[i][x];
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  if (w_t == SA_DTYPE_F32) ((float*)out)[e] = sum;
  else ((uint16_t*)out)[e] = to16(sum, w_t);
}

constexpr int64_t MAX_WIDTH = 32768;

// Workgroups of the backward: enough to fill every CU, few enough that their sums are little beside the rows, of which
// there is one at a time and wavefront up to 1024 wide, and one a workgroup beyond.
int64_t norm_parts(int64_t rows, int64_t width) {
  return std::max<int64_t>(1, width <= 1024 ? std::min<int64_t>(512, cdiv(rows, 4)) : std::min<int64_t>(width <= 4096 ? 512 : 256, rows));
}

// Lanes of a row and quads of a lane by width.
template <int G, int V, bool VEC>
void launch_norm(const NormCall& c, bool backward, hipStream_t st) {
  const dim3 threads(norm_threads<G>());
  if (backward) {
    hipLaunchKernelGGL((norm_backward_kernel<G, V, VEC>), dim3((unsigned)norm_parts(c.rows, c.width)), threads, 0, st, c);
  } else {
    const int64_t most = norm_walks<G, V>() ? (int64_t)device_cus() * (1024 / G) : LAUNCH_BLOCKS;
    const int64_t blocks = std::min<int64_t>(cdiv(c.rows, norm_threads<G>() / G), most);
    hipLaunchKernelGGL((norm_kernel<G, V, VEC>), dim3((unsigned)blocks), threads, 0, st, c);
  }
}
template <bool VEC>
void launch_norm(const NormCall& c, bool backward, hipStream_t st) {
  const int w = c.width;
  if (w <= 256) launch_norm<64, 1, VEC>(c, backward, st);
  else if (w <= 512) launch_norm<64, 2, VEC>(c, backward, st);
  else if (w <= 768) launch_norm<64, 3, VEC>(c, backward, st);
  else if (w <= 1024) launch_norm<64, 4, VEC>(c, backward, st);
  else if (w <= 2048) launch_norm<256, 2, VEC>(c, backward, st);
  else if (w <= 4096) launch_norm<256, 4, VEC>(c, backward, st);
  else if (w <= 8192) launch_norm<512, 4, VEC>(c, backward, st);
  else if (w <= 16384) launch_norm<1024, 4, VEC>(c, backward, st);
  else launch_norm<1024, 8, VEC>(c, backward, st);
}

bool norm_sizes_ok(int64_t rows, int64_t width) { return rows >= 0 && rows < ((int64_t)1 << 40) && width >= 1 && width <= MAX_WIDTH; }
bool ld_ok(int64_t ld) { return ld >= 0 && ld < ((int64_t)1 << 40); }
bool of_type(const void* p, int dtype) { return (uintptr_t)p % lm_elem_size(dtype) == 0; }

}  // namespace

extern "C" {

int sa_layer_norm(const void* x, int64_t x_ld, const void* branch, int64_t branch_ld, const void* weight, const void* bias, void* y,
                  void* sum, float* mean, float* rstd, int64_t rows, int64_t width, float eps, int x_dtype, int branch_dtype,
                  int y_dtype, int weight_dtype, void* stream) {
  if (!lm_elem_size(x_dtype) || !lm_elem_size(y_dtype) || !lm_elem_size(weight_dtype) || (branch && !lm_elem_size(branch_dtype)))
    return SA_ERR_DTYPE;
  if (!norm_sizes_ok(rows, width) || !ld_ok(x_ld) || !ld_ok(branch_ld) || !(eps >= 0.f) || !(eps < INFINITY)) return SA_ERR_ARGUMENT;
  if (rows == 0) return SA_OK;
  if (!x || !weight || !y || (branch && !sum) || !mean != !rstd) return SA_ERR_ARGUMENT;
  if (!of_type(x, x_dtype) || !of_type(y, y_dtype) || !of_type(weight, weight_dtype) || !of_type(bias, weight_dtype) ||
      !of_type(sum, x_dtype) || (branch && !of_type(branch, branch_dtype)))
    return SA_ERR_ARGUMENT;
  NormCall c{};
  c.x = x, c.branch = branch, c.w = weight, c.b = bias, c.y = y, c.s = sum, c.mean = mean, c.rstd = rstd;
  c.x_ld = x_ld, c.branch_ld = branch_ld, c.rows = rows, c.width = (int)width, c.eps = eps;
  c.x_t = x_dtype, c.branch_t = branch ? branch_dtype : x_dtype, c.y_t = y_dtype, c.w_t = weight_dtype;
  const bool vec = width % 4 == 0 && quads_ok(x, x_ld, x_dtype) && quads_ok(branch, branch_ld, c.branch_t) &&
                   quads_ok(weight, 0, weight_dtype) && quads_ok(bias, 0, weight_dtype) && quads_ok(y, width, y_dtype) &&
                   quads_ok(sum, width, x_dtype);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (vec) launch_norm<true>(c, false, st);
  else launch_norm<false>(c, false, st);
  return launch_status();
}

int64_t sa_layer_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
  if (!norm_sizes_ok(rows, width)) return -1;
  return align_up(norm_parts(rows, width) * 2 * width * 4, 256);
}

int sa_layer_norm_backward(const void* s, int64_t s_ld, const void* dy, int64_t dy_ld, const void* ds, int64_t ds_ld,
                           const void* weight, const float* mean, const float* rstd, void* dx, void* dbranch, void* dweight,
                           void* dbias, void* workspace, int64_t workspace_bytes, int64_t rows, int64_t width, int s_dtype,
                           int branch_dtype, int y_dtype, int weight_dtype, void* stream) {
  if (!lm_elem_size(s_dtype) || !lm_elem_size(y_dtype) || !lm_elem_size(weight_dtype) || (dbranch && !lm_elem_size(branch_dtype)))
    return SA_ERR_DTYPE;
  if (!norm_sizes_ok(rows, width) || !ld_ok(s_ld) || !ld_ok(dy_ld) || !ld_ok(ds_ld)) return SA_ERR_ARGUMENT;
  if (!weight || (rows > 0 && (!s || !dy || !mean || !rstd))) return SA_ERR_ARGUMENT;
  if (!of_type(s, s_dtype) || !of_type(dy, y_dtype) || !of_type(ds, s_dtype) || !of_type(weight, weight_dtype) ||
      !of_type(dx, s_dtype) || (dbranch && !of_type(dbranch, branch_dtype)) || !of_type(dweight, weight_dtype) ||
      !of_type(dbias, weight_dtype))
    return SA_ERR_ARGUMENT;
  const bool sums = dweight || dbias;
  if (sums && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < sa_layer_norm_backward_workspace_bytes(rows, width)))
    return SA_ERR_WORKSPACE;
  NormCall c{};
  c.x = s, c.dy = dy, c.ds = ds, c.w = weight, c.mean = const_cast<float*>(mean), c.rstd = const_cast<float*>(rstd);
  c.dx = dx, c.dbranch = dbranch, c.part = sums ? (float*)workspace : nullptr, c.sums = dbias ? 2 : 1;
  c.x_ld = s_ld, c.dy_ld = dy_ld, c.ds_ld = ds_ld, c.rows = rows, c.width = (int)width;
  c.x_t = s_dtype, c.branch_t = dbranch ? branch_dtype : s_dtype, c.y_t = y_dtype, c.w_t = weight_dtype;
  const bool vec = width % 4 == 0 && quads_ok(s, s_ld, s_dtype) && quads_ok(dy, dy_ld, y_dtype) && quads_ok(ds, ds_ld, s_dtype) &&
                   quads_ok(weight, 0, weight_dtype) && quads_ok(dx, width, s_dtype) && quads_ok(dbranch, width, c.branch_t);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (vec) launch_norm<true>(c, true, st);   // (no rows: sums of nothing)
  else launch_norm<false>(c, true, st);
  if (sums)
    hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)cdiv(width, 64), (unsigned)c.sums), dim3(1024), 0, st, c.part,
                       (int)norm_parts(rows, width), (int)width, dweight, dbias, weight_dtype);
  return launch_status();
}

}  // extern "C"
