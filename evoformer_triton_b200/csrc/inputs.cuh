// What the kernels of layer norm, the relative position bias and the pair-bias projection share.
#pragma once
#include "common.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace evo {

inline bool known_dtype(int t) { return t == EVOATTN_BF16 || t == EVOATTN_FP16 || t == EVOATTN_FP32; }
inline int dtype_bytes(int t) { return t == EVOATTN_FP32 ? 4 : 2; }

// Calls f with a value of the element type of `dtype`.
template <class F>
inline int with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case EVOATTN_BF16: return f(__nv_bfloat16());
    case EVOATTN_FP16: return f(__half());
    default: return f(float());
  }
}

// A value of a small tensor (weights) whose type is known when the kernel runs.
__device__ __forceinline__ float load_any(const void* p, int dtype, long long i) {
  if (dtype == EVOATTN_FP32) return static_cast<const float*>(p)[i];
  if (dtype == EVOATTN_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dtype, long long i, float v) {
  if (dtype == EVOATTN_FP32) static_cast<float*>(p)[i] = v;
  else if (dtype == EVOATTN_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// The sum over a block of up to 1024 threads, the same for all of them; `sm` holds 32 floats a value.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* sm) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return;
  __syncthreads();  // (the values of the call before have been read)
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) sm[i * 32 + (threadIdx.x >> 5)] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
    for (int w = 0; w < warps; ++w) s += sm[i * 32 + w];
    v[i] = s;
  }
}

}  // namespace evo
