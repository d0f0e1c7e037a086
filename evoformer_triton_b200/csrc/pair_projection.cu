// The pair representation's layer norm and its projection to a pair bias, heads first, in one pass:
//
//   xh = (z - mean) r,  G[h,c] = weight[h,c] g[c],  out[b,h,i,j] = sum_c G[h,c] xh[c] + sum_c weight[h,c] b[c]
//
// Backward, with u[c] = sum_h d[h] G[h,c], M[h,c] = sum over rows of d[h] xh[c] and s[h] = sum over rows of d[h]:
//
//   dz = r (u - mean(u) - xh mean(u xh))
//   dweight[h,c] = g[c] M[h,c] + b[c] s[h],  dg[c] = sum_h weight[h,c] M[h,c],  db[c] = sum_h weight[h,c] s[h]
//
// so the gradients of all three weights come from sums that do not depend on them.
#include "inputs.cuh"

namespace evo {
namespace {

struct ProjArgs {
  int B, Ri, Rj, C, H;
  float eps;
  int w_dtype, g_dtype, b_dtype;
  const void* z;
  Str3 sz;
  const void* w;
  const void* g;
  const void* b;
  void* out;        // forward: out; backward: d_out
  Str3 sout;
  void* dz;
  void* dw;
  void* dg;
  void* db;
  float* stats;     // [rows][2]
  float* partial;   // [blocks][H][C + 1]: M and s
  int blocks;
};

constexpr int kMaxPerLane = EVOATTN_PROJECTION_MAX_C / 32;

__device__ __forceinline__ float gain(const ProjArgs& a, int c) { return a.g ? load_any(a.g, a.g_dtype, c) : 1.f; }

struct Row {
  int b, i, j;
  __device__ __forceinline__ Row(const ProjArgs& a, long long n) {
    j = (int)(n % a.Rj);
    const long long q = n / a.Rj;
    i = (int)(q % a.Ri);
    b = (int)(q / a.Ri);
  }
  __device__ __forceinline__ long long at(const Str3& s) const { return b * s.a + i * s.b + j * s.c; }
  __device__ __forceinline__ long long at(const Str3& s, int h) const { return b * s.a + h * s.b + i * s.c + j; }
};

// A warp a row, lane l the channels l, l + 32, ...
template <class T>
__device__ __forceinline__ void normalise(const ProjArgs& a, const Row& row, float (&x)[kMaxPerLane], float& mean, float& r) {
  const T* z = static_cast<const T*>(a.z) + row.at(a.sz);
  const int lane = threadIdx.x & 31;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < kMaxPerLane; ++k) {
    x[k] = lane + 32 * k < a.C ? to_float<T>(z[lane + 32 * k]) : 0.f;
    s += x[k];
  }
  mean = warp_sum(s) / a.C;
  s = 0.f;
#pragma unroll
  for (int k = 0; k < kMaxPerLane; ++k) {
    x[k] = lane + 32 * k < a.C ? x[k] - mean : 0.f;
    s = fmaf(x[k], x[k], s);
  }
  r = rsqrtf(warp_sum(s) / a.C + a.eps);
#pragma unroll
  for (int k = 0; k < kMaxPerLane; ++k) x[k] *= r;
}

template <class T>
__global__ void __launch_bounds__(256) projection_fwd(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  extern __shared__ float sm[];  // [H][C] and [H]
  float* sm_t = sm + a.H * a.C;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < a.H * a.C; i += 256) sm[i] = load_any(a.w, a.w_dtype, i) * gain(a, i % a.C);
  for (int h = warp; h < a.H; h += 8) {
    float t = 0.f;
    if (a.b)
      for (int c = lane; c < a.C; c += 32) t = fmaf(load_any(a.w, a.w_dtype, h * a.C + c), load_any(a.b, a.b_dtype, c), t);
    t = warp_sum(t);
    if (lane == 0) sm_t[h] = t;
  }
  __syncthreads();
  const long long rows = (long long)a.B * a.Ri * a.Rj;
  for (long long n = (long long)blockIdx.x * 8 + warp; n < rows; n += (long long)gridDim.x * 8) {
    const Row row(a, n);
    float x[kMaxPerLane], mean, r;
    normalise<T>(a, row, x, mean, r);
    for (int h = 0; h < a.H; ++h) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kMaxPerLane; ++k)
        if (lane + 32 * k < a.C) s = fmaf(x[k], sm[h * a.C + lane + 32 * k], s);
      s = warp_sum(s);
      if (lane == 0) static_cast<T*>(a.out)[row.at(a.sout, h)] = from_float<T>(s + sm_t[h]);
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256) projection_dz(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  extern __shared__ float sm[];  // [H][C]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < a.H * a.C; i += 256) sm[i] = load_any(a.w, a.w_dtype, i) * gain(a, i % a.C);
  __syncthreads();
  const long long rows = (long long)a.B * a.Ri * a.Rj;
  for (long long n = (long long)blockIdx.x * 8 + warp; n < rows; n += (long long)gridDim.x * 8) {
    const Row row(a, n);
    float x[kMaxPerLane], mean, r;
    normalise<T>(a, row, x, mean, r);
    if (a.stats && lane == 0) reinterpret_cast<float2*>(a.stats)[n] = make_float2(mean, r);
    if (!a.dz) continue;
    float u[kMaxPerLane] = {};
    for (int h = 0; h < a.H; ++h) {
      const float d = to_float<T>(static_cast<const T*>(a.out)[row.at(a.sout, h)]);
#pragma unroll
      for (int k = 0; k < kMaxPerLane; ++k)
        if (lane + 32 * k < a.C) u[k] = fmaf(d, sm[h * a.C + lane + 32 * k], u[k]);
    }
    float m1 = 0.f, m2 = 0.f;
#pragma unroll
    for (int k = 0; k < kMaxPerLane; ++k) {
      m1 += u[k];
      m2 = fmaf(u[k], x[k], m2);
    }
    m1 = warp_sum(m1) / a.C;
    m2 = warp_sum(m2) / a.C;
#pragma unroll
    for (int k = 0; k < kMaxPerLane; ++k)
      if (lane + 32 * k < a.C) static_cast<T*>(a.dz)[n * a.C + lane + 32 * k] = from_float<T>(r * (u[k] - m1 - x[k] * m2));
  }
}

// M and s of a share of the rows: a thread a channel (the one behind the last: s), eight heads a block.
template <class T>
__global__ void __launch_bounds__(128) projection_sums(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int c = blockIdx.y * 128 + threadIdx.x, h0 = blockIdx.z * 8, nh = min(8, a.H - h0);
  if (c > a.C) return;
  float m[8] = {};
  const long long rows = (long long)a.B * a.Ri * a.Rj;
  for (long long n = blockIdx.x; n < rows; n += gridDim.x) {
    const Row row(a, n);
    const float2 st = reinterpret_cast<const float2*>(a.stats)[n];
    const float x = c < a.C ? (to_float<T>(static_cast<const T*>(a.z)[row.at(a.sz) + c]) - st.x) * st.y : 1.f;
#pragma unroll
    for (int h = 0; h < 8; ++h)
      if (h < nh) m[h] = fmaf(to_float<T>(static_cast<const T*>(a.out)[row.at(a.sout, h0 + h)]), x, m[h]);
  }
  for (int h = 0; h < nh; ++h) a.partial[((long long)blockIdx.x * a.H + h0 + h) * (a.C + 1) + c] = m[h];
}

// The blocks' sums added in order, a thread an element of the first block's place.
__global__ void __launch_bounds__(256) projection_sum_partials(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long size = (long long)a.H * (a.C + 1), e = (long long)blockIdx.x * 256 + threadIdx.x;
  if (e >= size) return;
  float s = 0.f;
  for (int k = 0; k < a.blocks; ++k) s += a.partial[k * size + e];
  a.partial[a.blocks * size + e] = s;
}

__global__ void __launch_bounds__(128) projection_weights(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= a.C) return;
  const float* m = a.partial + (long long)a.blocks * a.H * (a.C + 1);
  const float g = gain(a, c), b = a.b ? load_any(a.b, a.b_dtype, c) : 0.f;
  float dg = 0.f, db = 0.f;
  for (int h = 0; h < a.H; ++h) {
    const float w = load_any(a.w, a.w_dtype, h * a.C + c), mh = m[h * (a.C + 1) + c], s = m[h * (a.C + 1) + a.C];
    if (a.dw) store_any(a.dw, a.w_dtype, h * a.C + c, fmaf(g, mh, b * s));
    dg = fmaf(w, mh, dg);
    db = fmaf(w, s, db);
  }
  if (a.dg) store_any(a.dg, a.g_dtype, c, dg);
  if (a.db) store_any(a.db, a.b_dtype, c, db);
}

int validate(const evoattn_pair_projection_params* p) {
  if (!p) return EVOATTN_ERR_NULL;
  if (!known_dtype(p->dtype) || !known_dtype(p->weight_dtype)) return EVOATTN_ERR_DTYPE;
  if ((p->norm_weight || p->dnorm_weight) && !known_dtype(p->norm_weight_dtype)) return EVOATTN_ERR_DTYPE;
  if ((p->norm_bias || p->dnorm_bias) && !known_dtype(p->norm_bias_dtype)) return EVOATTN_ERR_DTYPE;
  if (p->B < 0 || p->Ri < 0 || p->Rj < 0 || p->C <= 0 || p->H <= 0 || !(p->eps >= 0.f)) return EVOATTN_ERR_SHAPE;
  if (p->C > EVOATTN_PROJECTION_MAX_C || p->H > EVOATTN_PROJECTION_MAX_H) return EVOATTN_ERR_UNSUPPORTED;
  if (p->Ri > (1 << 20) || p->Rj > (1 << 20) || p->B > (1 << 20)) return EVOATTN_ERR_SHAPE;
  if ((long long)p->B * p->Ri > (1LL << 48) / (p->Rj > 0 ? p->Rj : 1) / p->C) return EVOATTN_ERR_SHAPE;
  return EVOATTN_OK;
}

ProjArgs args_of(const evoattn_pair_projection_params* p) {
  ProjArgs a{};
  a.B = p->B; a.Ri = p->Ri; a.Rj = p->Rj; a.C = p->C; a.H = p->H; a.eps = p->eps;
  a.w_dtype = p->weight_dtype; a.g_dtype = p->norm_weight_dtype; a.b_dtype = p->norm_bias_dtype;
  a.z = p->pair; a.sz = Str3{p->pair_stride[0], p->pair_stride[1], p->pair_stride[2]};
  a.w = p->weight; a.g = p->norm_weight; a.b = p->norm_bias;
  a.dz = p->dpair; a.dw = p->dweight; a.dg = p->dnorm_weight; a.db = p->dnorm_bias;
  const long long rows = (long long)p->B * p->Ri * p->Rj;
  a.blocks = (int)(rows < 592 ? rows : 592);
  return a;
}
long long rows_of(const ProjArgs& a) { return (long long)a.B * a.Ri * a.Rj; }
size_t stats_bytes(const ProjArgs& a) { return (size_t)((rows_of(a) * 8 + 15) / 16 * 16); }
int weights_smem(const ProjArgs& a) { return a.H * (a.C + 1) * (int)sizeof(float); }

}  // namespace
}  // namespace evo

extern "C" {

int evoattn_pair_projection_fwd(const evoattn_pair_projection_params* p, void* cuda_stream) {
  using namespace evo;
  if (const int rc = validate(p)) return rc;
  ProjArgs a = args_of(p);
  const long long rows = rows_of(a);
  if (rows == 0) return EVOATTN_OK;
  if (!a.z || !a.w || !p->out) return EVOATTN_ERR_NULL;
  a.out = p->out;
  a.sout = Str3{p->out_stride[0], p->out_stride[1], p->out_stride[2]};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  const unsigned grid = (unsigned)((rows + 7) / 8 < 148 * 4 ? (rows + 7) / 8 : 148 * 4);
  return with_dtype(p->dtype, [&](auto e) {
    const auto kern = projection_fwd<decltype(e)>;
    if (!kernel_ready(reinterpret_cast<const void*>(kern), weights_smem(a), nullptr)) return (int)EVOATTN_ERR_CUDA;
    return (int)(launch_dependent(kern, dim3(grid), 256, (size_t)weights_smem(a), st, a) == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA);
  });
}

size_t evoattn_pair_projection_bwd_workspace_bytes(const evoattn_pair_projection_params* p) {
  using namespace evo;
  if (validate(p) || !(p->dweight || p->dnorm_weight || p->dnorm_bias)) return 0;
  const ProjArgs a = args_of(p);
  return stats_bytes(a) + (size_t)(a.blocks + 1) * a.H * (a.C + 1) * sizeof(float);
}

int evoattn_pair_projection_bwd(const evoattn_pair_projection_params* p, void* cuda_stream) {
  using namespace evo;
  if (const int rc = validate(p)) return rc;
  ProjArgs a = args_of(p);
  const long long rows = rows_of(a);
  if (!a.w || (rows > 0 && (!a.z || !p->d_out))) return EVOATTN_ERR_NULL;
  const size_t need = evoattn_pair_projection_bwd_workspace_bytes(p);
  if (need && (!p->workspace || p->workspace_bytes < need)) return EVOATTN_ERR_WORKSPACE;
  if ((uintptr_t)p->workspace & 15) return EVOATTN_ERR_ALIGN;
  a.out = const_cast<void*>(p->d_out);
  a.sout = Str3{p->d_out_stride[0], p->d_out_stride[1], p->d_out_stride[2]};
  const bool sums = a.dw || a.dg || a.db;
  if (sums) {
    a.stats = static_cast<float*>(p->workspace);
    a.partial = reinterpret_cast<float*>(static_cast<unsigned char*>(p->workspace) + stats_bytes(a));
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t rc = cudaSuccess;
  if (rows > 0 && (a.dz || sums)) {
    const int bad = with_dtype(p->dtype, [&](auto e) {
      using T = decltype(e);
      const auto kern = projection_dz<T>;
      if (!kernel_ready(reinterpret_cast<const void*>(kern), weights_smem(a), nullptr)) return 1;
      rc = launch_dependent(kern, dim3((unsigned)((rows + 7) / 8 < 148 * 4 ? (rows + 7) / 8 : 148 * 4)), 256, (size_t)weights_smem(a), st, a);
      if (rc == cudaSuccess && sums)
        rc = launch_dependent(projection_sums<T>, dim3((unsigned)a.blocks, (unsigned)((a.C + 128) / 128), (unsigned)((a.H + 7) / 8)), 128, 0, st, a);
      return 0;
    });
    if (bad) return EVOATTN_ERR_CUDA;
  }
  if (rc == cudaSuccess && sums) {
    rc = launch_dependent(projection_sum_partials, dim3((unsigned)((a.H * (a.C + 1) + 255) / 256)), 256, 0, st, a);
    if (rc == cudaSuccess) rc = launch_dependent(projection_weights, dim3((unsigned)((a.C + 127) / 128)), 128, 0, st, a);
  }
  return rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

}  // extern "C"
