// Layer norm over the last axis, forward and backward.
//
//   h = (x - mean) r,  r = (var + eps)^-1/2,  y = h w + b
//   g = dy w,  dx = r (g - mean(g) - h mean(g h)),  dw = sum over rows of dy h,  db = sum over rows of dy
//
// The variance is taken about the mean (two passes over a row), so rows far from zero lose nothing.
#include "inputs.cuh"

namespace evo {
namespace {

struct NormArgs {
  long long rows;
  long long n1, n2;  // rows are (n0, n1, n2)
  int C;
  float eps;
  int w_dtype, b_dtype;
  const void* x;
  Str3 sx;
  const void* w;
  const void* b;
  void* y;
  float* stats;
  const void* dy;
  Str3 sdy;
  void* dx;
  void* dw;
  void* db;
  float* partial;  // [blocks][2][C]
  int blocks;
};

__device__ __forceinline__ long long row_offset(const NormArgs& a, const Str3& s, long long n) {
  const long long q = n / a.n2, k = n - q * a.n2, i = q / a.n1, j = q - i * a.n1;
  return i * s.a + j * s.b + k * s.c;
}

// A block walks rows, reading each three times (the second and third time from L1 or L2): any C, any alignment.
template <class T>
__global__ void __launch_bounds__(256) norm_fwd_any(NormArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  __shared__ float sm[32];
  for (long long n = blockIdx.x; n < a.rows; n += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row_offset(a, a.sx, n);
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < a.C; c += 256) s[0] += to_float<T>(x[c]);
    block_sum(s, sm);
    const float mean = s[0] / a.C;
    s[0] = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float d = to_float<T>(x[c]) - mean;
      s[0] = fmaf(d, d, s[0]);
    }
    block_sum(s, sm);
    const float r = rsqrtf(s[0] / a.C + a.eps);
    if (a.stats && threadIdx.x == 0) reinterpret_cast<float2*>(a.stats)[n] = make_float2(mean, r);
    T* y = static_cast<T*>(a.y) + n * a.C;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float h = (to_float<T>(x[c]) - mean) * r;
      y[c] = from_float<T>(fmaf(h, a.w ? load_any(a.w, a.w_dtype, c) : 1.f, a.b ? load_any(a.b, a.b_dtype, c) : 0.f));
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256) norm_dx_any(NormArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  __shared__ float sm[64];
  for (long long n = blockIdx.x; n < a.rows; n += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row_offset(a, a.sx, n);
    const T* dy = static_cast<const T*>(a.dy) + row_offset(a, a.sdy, n);
    const float2 st = reinterpret_cast<const float2*>(a.stats)[n];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float g = to_float<T>(dy[c]) * (a.w ? load_any(a.w, a.w_dtype, c) : 1.f);
      s[0] += g;
      s[1] = fmaf(g, (to_float<T>(x[c]) - st.x) * st.y, s[1]);
    }
    block_sum(s, sm);
    const float m1 = s[0] / a.C, m2 = s[1] / a.C;
    T* dx = static_cast<T*>(a.dx) + n * a.C;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float g = to_float<T>(dy[c]) * (a.w ? load_any(a.w, a.w_dtype, c) : 1.f);
      dx[c] = from_float<T>(st.y * (g - m1 - (to_float<T>(x[c]) - st.x) * st.y * m2));
    }
  }
}

// dw and db over the rows blockIdx.y, blockIdx.y + gridDim.y, ... of 32 columns a block; eight rows at a time.
template <class T>
__global__ void __launch_bounds__(256) norm_columns_any(NormArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  __shared__ float sm[2][8][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float dw = 0.f, db = 0.f;
  if (c < a.C)
    for (long long n = (long long)blockIdx.y * 8 + part; n < a.rows; n += (long long)gridDim.y * 8) {
      const float2 st = reinterpret_cast<const float2*>(a.stats)[n];
      const float dy = to_float<T>(static_cast<const T*>(a.dy)[row_offset(a, a.sdy, n) + c]);
      const float x = to_float<T>(static_cast<const T*>(a.x)[row_offset(a, a.sx, n) + c]);
      dw = fmaf(dy, (x - st.x) * st.y, dw);
      db += dy;
    }
  sm[0][part][lane] = dw;
  sm[1][part][lane] = db;
  __syncthreads();
  if (part < 2 && c < a.C) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += sm[part][i][lane];
    a.partial[((long long)blockIdx.y * 2 + part) * a.C + c] = s;
  }
}

// The partial sums of all blocks, added in order.
__global__ void __launch_bounds__(256) norm_sum_partials(NormArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  __shared__ float sm[8][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, which = blockIdx.y;
  float s = 0.f;
  if (c < a.C)
    for (int k = part; k < a.blocks; k += 8) s += a.partial[((long long)k * 2 + which) * a.C + c];
  sm[part][lane] = s;
  __syncthreads();
  if (part == 0 && c < a.C) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += sm[i][lane];
    if (which == 0 && a.dw) store_any(a.dw, a.w_dtype, c, s);
    if (which == 1 && a.db) store_any(a.db, a.b_dtype, c, s);
  }
}

// Blocks that take a share of the rows for the columns' sums.
int row_shares(long long rows) { return (int)(rows < 8 * 148 ? (rows + 7) / 8 : 148); }

int validate(const evoattn_layer_norm_params* p) {
  if (!p) return EVOATTN_ERR_NULL;
  if (!known_dtype(p->dtype)) return EVOATTN_ERR_DTYPE;
  if ((p->weight || p->dweight) && !known_dtype(p->weight_dtype)) return EVOATTN_ERR_DTYPE;
  if ((p->bias || p->dbias) && !known_dtype(p->bias_dtype)) return EVOATTN_ERR_DTYPE;
  if (p->C <= 0 || !(p->eps >= 0.f)) return EVOATTN_ERR_SHAPE;
  long long rows = 1;
  for (int i = 0; i < 3; ++i) {
    if (p->n[i] < 0) return EVOATTN_ERR_SHAPE;
    if (p->n[i] > 0 && rows > (1LL << 48) / p->n[i]) return EVOATTN_ERR_SHAPE;
    rows *= p->n[i];
  }
  if (rows > (1LL << 48) / p->C) return EVOATTN_ERR_SHAPE;
  return EVOATTN_OK;
}

NormArgs args_of(const evoattn_layer_norm_params* p) {
  NormArgs a{};
  a.rows = (long long)p->n[0] * p->n[1] * p->n[2];
  a.n1 = p->n[1]; a.n2 = p->n[2];
  a.C = p->C; a.eps = p->eps;
  a.w_dtype = p->weight_dtype; a.b_dtype = p->bias_dtype;
  a.x = p->x; a.sx = Str3{p->x_stride[0], p->x_stride[1], p->x_stride[2]};
  a.w = p->weight; a.b = p->bias; a.y = p->y; a.stats = p->stats;
  a.dy = p->d_y; a.sdy = Str3{p->d_y_stride[0], p->d_y_stride[1], p->d_y_stride[2]};
  a.dx = p->dx; a.dw = p->dweight; a.db = p->dbias;
  return a;
}

unsigned row_blocks(long long rows) { return (unsigned)(rows < (1LL << 30) ? rows : (1LL << 30)); }

}  // namespace
}  // namespace evo

extern "C" {

int evoattn_layer_norm_fwd(const evoattn_layer_norm_params* p, void* cuda_stream) {
  using namespace evo;
  if (const int rc = validate(p)) return rc;
  NormArgs a = args_of(p);
  if (a.rows == 0) return EVOATTN_OK;
  if (!a.x || !a.y) return EVOATTN_ERR_NULL;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  return with_dtype(p->dtype, [&](auto e) {
    using T = decltype(e);
    return launch_dependent(norm_fwd_any<T>, dim3(row_blocks(a.rows)), 256, 0, st, a) == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
  });
}

size_t evoattn_layer_norm_bwd_workspace_bytes(const evoattn_layer_norm_params* p) {
  using namespace evo;
  if (validate(p) || !(p->dweight || p->dbias)) return 0;
  const NormArgs a = args_of(p);
  return (size_t)row_shares(a.rows) * 2 * a.C * sizeof(float);
}

int evoattn_layer_norm_bwd(const evoattn_layer_norm_params* p, void* cuda_stream) {
  using namespace evo;
  if (const int rc = validate(p)) return rc;
  NormArgs a = args_of(p);
  const bool columns = a.dw || a.db;
  if (a.rows > 0 && (!a.x || !a.dy || !a.stats)) return EVOATTN_ERR_NULL;
  const size_t need = evoattn_layer_norm_bwd_workspace_bytes(p);
  if (need && (!p->workspace || p->workspace_bytes < need)) return EVOATTN_ERR_WORKSPACE;
  if ((uintptr_t)p->workspace & 15) return EVOATTN_ERR_ALIGN;
  a.partial = static_cast<float*>(p->workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t rc = cudaSuccess;
  if (a.dx && a.rows > 0)
    with_dtype(p->dtype, [&](auto e) {
      rc = launch_dependent(norm_dx_any<decltype(e)>, dim3(row_blocks(a.rows)), 256, 0, st, a);
      return 0;
    });
  if (rc == cudaSuccess && columns) {
    a.blocks = row_shares(a.rows);
    const unsigned strips = (unsigned)((a.C + 31) / 32);
    if (a.blocks)
      with_dtype(p->dtype, [&](auto e) {
        rc = launch_dependent(norm_columns_any<decltype(e)>, dim3(strips, (unsigned)a.blocks), 256, 0, st, a);
        return 0;
      });
    if (rc == cudaSuccess) rc = launch_dependent(norm_sum_partials, dim3(strips, 2), 256, 0, st, a);
  }
  return rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

}  // extern "C"
