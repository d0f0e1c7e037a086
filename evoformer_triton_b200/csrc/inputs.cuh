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

// Division of 0 <= n < 2^31 by a number that is the same for a whole launch: n * ceil(2^p / d) >> p with p = 31 + ceil(log2 d);
// the rounded-up factor is off by less than d <= 2^(p - 31), so n < 2^31 leaves the quotient as it is.
struct FastDiv {
  uint32_t d = 1, m = 1u << 31;
  int p = 31;
  FastDiv() = default;
  explicit FastDiv(uint32_t by) : d(by) {
    while ((1ull << (p - 31)) < by) ++p;
    m = (uint32_t)(((1ull << p) + by - 1) / by);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> p); }
};

// Sixteen bytes of T as floats and back.
template <class T> constexpr int kPer16 = 16 / (int)sizeof(T);
template <class T>
__device__ __forceinline__ void unpack16(const uint4& w, float* v) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
  } else {
    unpack2<T>(w.x, v[0], v[1]); unpack2<T>(w.y, v[2], v[3]); unpack2<T>(w.z, v[4], v[5]); unpack2<T>(w.w, v[6], v[7]);
  }
}
template <class T>
__device__ __forceinline__ uint4 pack16(const float* v) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else
    return make_uint4(Pack2<T>::pack(v[0], v[1]), Pack2<T>::pack(v[2], v[3]), Pack2<T>::pack(v[4], v[5]), Pack2<T>::pack(v[6], v[7]));
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
