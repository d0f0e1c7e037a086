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
#include <type_traits>

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
  FastDiv by_Ri, by_Rj;  // rows below 2^31
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

// ---------------------------------------------------------------- on tensor cores
//
// Few heads make the products thin (N = 8 heads or K = 8 heads), and the kernels are bound by the pair representation's way
// through memory; warp-level MMAs take their operands from the registers that the rows were loaded into, with no staging.
//
// A warp takes 16 rows.  Four lanes share a row: lane t of them loads channels 8 t .. 8 t + 7 of every 32, sixteen bytes in
// 16-bit types.  What a lane holds is at once the A operand of rows x channels (the channels that the MMA calls 2t, 2t + 1 and
// 2t + 8, 2t + 9 of a step are 8t + 4s .. 8t + 4s + 3 here; G is laid out to match), the accumulator layout of heads x
// channels products, and, transposed 8 x 8 at a time by movmatrix, the A operand of channels x rows.  The sums over a
// row are two exchanges.
//
// Products are of bf16 pieces with fp32 sums: an fp32 factor is the sum of three (24 bits), an fp16 one of two, a bf16 one
// is one.  z enters as it is: sum_c G z[c] - mean sum_c G, with both sums over the same pieces of G, and M likewise from d r z
// and d r mean.  G is two pieces (2^-17 of it is left out) where results are rounded to 16 bits, else three; d r always
// three, since the weights' gradients may be fp32.

__device__ __forceinline__ void mma_k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_k8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Two floats as N bf16 pieces each, packed by piece.
template <int N>
__device__ __forceinline__ void split2(float lo, float hi, uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = Pack2<__nv_bfloat16>::pack(lo, hi);
    if (i + 1 < N) {
      float a, b;
      unpack2<__nv_bfloat16>(w[i], a, b);
      lo -= a;
      hi -= b;
    }
  }
}

template <class T> struct Pieces;  // pieces of a value of type T, and of G beside it; products of pieces i + j < kTerms
template <> struct Pieces<__nv_bfloat16> { static constexpr int kX = 1, kG = 2, kTerms = 2; };
template <> struct Pieces<__half> { static constexpr int kX = 2, kG = 2, kTerms = 3; };
template <> struct Pieces<float> { static constexpr int kX = 3, kG = 3, kTerms = 3; };

// Eight channels of a row.
template <class T>
struct Eight {
  static constexpr int kWords = sizeof(T) / 2;
  uint4 w[kWords];
  __device__ __forceinline__ void load(const T* p, bool on) {
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = on ? reinterpret_cast<const uint4*>(p)[k] : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void floats(float (&v)[8]) const {
#pragma unroll
    for (int k = 0; k < kWords; ++k) unpack16<T>(w[k], v + k * kPer16<T>);
  }
  // [pair of channels][piece]
  __device__ __forceinline__ void pieces(uint32_t (&p)[4][Pieces<T>::kX]) const {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      p[0][0] = w[0].x; p[1][0] = w[0].y; p[2][0] = w[0].z; p[3][0] = w[0].w;
    } else {
      float v[8];
      floats(v);
#pragma unroll
      for (int k = 0; k < 4; ++k) split2<Pieces<T>::kX>(v[2 * k], v[2 * k + 1], p[k]);
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < kWords; ++k) reinterpret_cast<uint4*>(p)[k] = pack16<T>(v + k * kPer16<T>);
  }
};

__device__ __forceinline__ float g_of(const ProjArgs& a, int h, int c) {
  return h < a.H && c < a.C ? load_any(a.w, a.w_dtype, h * a.C + c) * gain(a, c) : 0.f;
}

// A lane's two rows of a tile: g and g + 8.
struct Rows2 {
  long long z[2], o[2];
  uint32_t n[2];
  bool on[2];
  __device__ __forceinline__ Rows2(const ProjArgs& a, uint32_t n0, uint32_t rows) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      n[k] = n0 + (threadIdx.x & 31) / 4 + 8 * k;
      on[k] = n[k] < rows;
      const uint32_t m = on[k] ? n[k] : 0, q = a.by_Rj.div(m), j = m - q * a.Rj, b = a.by_Ri.div(q), i = q - b * a.Ri;
      z[k] = b * a.sz.a + i * a.sz.b + j * a.sz.c;
      o[k] = b * a.sout.a + i * a.sout.c + j;
    }
  }
};

template <class T, int KC>
struct Tile {
  Eight<T> x[2][KC];
  float mean[2], r[2];
  __device__ __forceinline__ void load(const ProjArgs& a, const Rows2& row) {
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int c = 0; c < KC; ++c) x[k][c].load(static_cast<const T*>(a.z) + row.z[k] + c * 32 + t * 8, row.on[k] && c * 32 + t * 8 < a.C);
  }
  // Mean and 1 / deviation, the latter about the mean; a row that is not there has r = 0 and adds nothing.
  __device__ __forceinline__ void statistics(const ProjArgs& a, const Rows2& row) {
    const float by_C = 1.f / a.C;
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        float v[8];
        x[k][c].floats(v);
        s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      }
      mean[k] = quad_sum(s) * by_C;
      s = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        if (c * 32 + t * 8 >= a.C) continue;
        float v[8];
        x[k][c].floats(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(v[e] - mean[k], v[e] - mean[k], s);
      }
      s = quad_sum(s);  // (all lanes, rows that are not there too)
      r[k] = row.on[k] ? rsqrtf(s * by_C + a.eps) : 0.f;
    }
  }
};

template <class T, int KC, int NT>
__global__ void __launch_bounds__(256) projection_fwd_mma(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int GP = Pieces<T>::kG, XP = Pieces<T>::kX;
  extern __shared__ __align__(16) uint4 sm_g[];  // [KC][NT][GP][32 lanes]
  __shared__ float sm_sum[NT * 8], sm_t[NT * 8];  // sum_c of the pieces of G; sum_c weight b
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t rows = (uint32_t)((long long)a.B * a.Ri * a.Rj), step = gridDim.x * 128;
  uint32_t n0 = (blockIdx.x * 8 + warp) * 16;
  Tile<T, KC> x;
  if (n0 < rows) x.load(a, Rows2(a, n0, rows));
  for (int i = threadIdx.x; i < KC * NT * 32; i += 256) {
    const int l = i & 31, nt = (i >> 5) % NT, kc = (i >> 5) / NT, h = nt * 8 + l / 4, c = kc * 32 + (l & 3) * 8;
    uint32_t p[4][GP];
#pragma unroll
    for (int k = 0; k < 4; ++k) split2<GP>(g_of(a, h, c + 2 * k), g_of(a, h, c + 2 * k + 1), p[k]);
#pragma unroll
    for (int j = 0; j < GP; ++j) sm_g[((kc * NT + nt) * GP + j) * 32 + l] = make_uint4(p[0][j], p[1][j], p[2][j], p[3][j]);
  }
  for (int h = warp; h < NT * 8; h += 8) {
    float s = 0.f, tb = 0.f;
    for (int c = lane; c < a.C; c += 32) {
      uint32_t p[GP];
      split2<GP>(g_of(a, h, c), 0.f, p);
      float v = 0.f;
#pragma unroll
      for (int j = GP - 1; j >= 0; --j) {
        float lo, hi;
        unpack2<__nv_bfloat16>(p[j], lo, hi);
        v += lo;
      }
      s += v;
      if (a.b && h < a.H) tb = fmaf(load_any(a.w, a.w_dtype, h * a.C + c), load_any(a.b, a.b_dtype, c), tb);
    }
    s = warp_sum(s);
    tb = warp_sum(tb);
    if (lane == 0) sm_sum[h] = s, sm_t[h] = tb;
  }
  __syncthreads();
  for (; n0 < rows; n0 += step) {
    const Rows2 row(a, n0, rows);
    x.statistics(a, row);
    float acc[NT][4] = {};
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      uint32_t lo[4][XP], hi[4][XP];
      x.x[0][kc].pieces(lo);
      x.x[1][kc].pieces(hi);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < GP; ++j) {
          const uint4 gw = sm_g[((kc * NT + nt) * GP + j) * 32 + lane];
#pragma unroll
          for (int i = 0; i < XP; ++i) {
            if (i + j >= Pieces<T>::kTerms) continue;
            mma_k16(acc[nt], lo[0][i], hi[0][i], lo[1][i], hi[1][i], gw.x, gw.y);
            mma_k16(acc[nt], lo[2][i], hi[2][i], lo[3][i], hi[3][i], gw.z, gw.w);
          }
        }
    }
    const float mean[2] = {x.mean[0], x.mean[1]}, r[2] = {x.r[0], x.r[1]};
    if (n0 + step < rows) x.load(a, Rows2(a, n0 + step, rows));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = nt * 8 + 2 * t + e;
        if (h >= a.H) continue;
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (row.on[k])
            static_cast<T*>(a.out)[row.o[k] + h * a.sout.b] = from_float<T>(fmaf(acc[nt][2 * k + e] - mean[k] * sm_sum[h], r[k], sm_t[h]));
      }
  }
}

// Backward in one pass over z: dz, and M and s of the block's rows.
template <class T, int KC, int NT>
__global__ void __launch_bounds__(256) projection_bwd_mma(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int GP = Pieces<T>::kG, XP = Pieces<T>::kX, AP = 3;
  extern __shared__ __align__(16) uint4 sm_g[];  // [KC][NT][GP][32 lanes]; behind the rows, [H][C + 1] sums
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t rows = (uint32_t)((long long)a.B * a.Ri * a.Rj), step = gridDim.x * 128;
  if (a.dz) {
    for (int i = threadIdx.x; i < KC * NT * 32; i += 256) {
      const int l = i & 31, nt = (i >> 5) % NT, kc = (i >> 5) / NT, h = nt * 8 + (l & 3) * 2, c = kc * 32 + l / 8 * 8 + (l / 4 & 1);
      uint32_t p[4][GP];
#pragma unroll
      for (int q = 0; q < 4; ++q) split2<GP>(g_of(a, h, c + 2 * q), g_of(a, h + 1, c + 2 * q), p[q]);
#pragma unroll
      for (int j = 0; j < GP; ++j) sm_g[((kc * NT + nt) * GP + j) * 32 + l] = make_uint4(p[0][j], p[1][j], p[2][j], p[3][j]);
    }
  }
  __syncthreads();
  const float by_C = 1.f / a.C;
  float m_acc[KC][2][NT][4] = {}, s_acc[NT] = {}, q_acc[NT] = {};  // sums of d r z, of d, of d r mean
  for (uint32_t n0 = (blockIdx.x * 8 + warp) * 16; n0 < rows; n0 += step) {
    const Rows2 row(a, n0, rows);
    Tile<T, KC> x;
    x.load(a, row);
    float d[NT][2][2];  // [row g, g + 8][head 2t, 2t + 1]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int h = nt * 8 + 2 * t + e;
          d[nt][k][e] = row.on[k] && h < a.H ? to_float<T>(static_cast<const T*>(a.out)[row.o[k] + h * a.sout.b]) : 0.f;
        }
    uint32_t dp[NT][2][XP];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) split2<XP>(d[nt][k][0], d[nt][k][1], dp[nt][k]);
    x.statistics(a, row);

    if (a.partial) {
      // r and mean of rows 2t, 2t + 1, 2t + 8, 2t + 9, which the lanes 4 (2t) and 4 (2t + 1) hold
      float r[2][2], mean[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          r[k][e] = __shfl_sync(0xffffffffu, x.r[k], 8 * t + 4 * e);
          mean[k][e] = __shfl_sync(0xffffffffu, x.mean[k], 8 * t + 4 * e);
        }
      uint32_t ap[NT][2][AP];  // pieces of d r, [rows x heads] transposed
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float d0 = 0.f, d1 = 0.f;
#pragma unroll
          for (int i = XP - 1; i >= 0; --i) {
            float lo, hi;
            unpack2<__nv_bfloat16>(transposed(dp[nt][k][i]), lo, hi);
            d0 += lo;
            d1 += hi;
          }
          s_acc[nt] += d0 + d1;
          d0 *= r[k][0];
          d1 *= r[k][1];
          q_acc[nt] = fmaf(d0, mean[k][0], fmaf(d1, mean[k][1], q_acc[nt]));
          split2<AP>(d0, d1, ap[nt][k]);
        }
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) {
        uint32_t lo[4][XP], hi[4][XP];
        x.x[0][kc].pieces(lo);
        x.x[1][kc].pieces(hi);
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < XP; ++i) {
            const uint32_t a0 = transposed(lo[2 * p][i]), a1 = transposed(lo[2 * p + 1][i]), a2 = transposed(hi[2 * p][i]), a3 = transposed(hi[2 * p + 1][i]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j + i < AP; ++j) mma_k16(m_acc[kc][p][nt], a0, a1, a2, a3, ap[nt][0][j], ap[nt][1][j]);
          }
      }
    }
    if (!a.dz) continue;
    const auto u_of = [&](int kc, float (&u)[2][8]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float acc[4] = {};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < GP; ++j) {
            const uint32_t gw = reinterpret_cast<const uint32_t*>(sm_g + ((kc * NT + nt) * GP + j) * 32 + lane)[q];
#pragma unroll
            for (int i = 0; i < XP; ++i)
              if (i + j < Pieces<T>::kTerms) mma_k8(acc, dp[nt][0][i], dp[nt][1][i], gw);
          }
        u[0][2 * q] = acc[0]; u[0][2 * q + 1] = acc[1]; u[1][2 * q] = acc[2]; u[1][2 * q + 1] = acc[3];
      }
    };
    constexpr bool kKeep = KC <= 4 && sizeof(T) == 2;  // u stays in registers, else it is worked out twice
    float u_all[kKeep ? KC : 1][2][8], m1[2] = {}, m2[2] = {};
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      float(&u)[2][8] = u_all[kKeep ? kc : 0];
      u_of(kc, u);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float v[8];
        x.x[k][kc].floats(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          m1[k] += u[k][e];
          m2[k] = fmaf(u[k][e], v[e] - x.mean[k], m2[k]);  // (channels that are not there have u = 0)
        }
      }
    }
    // dz = r u - r m1 - (z - mean) r^2 mean(u (z - mean) r)
    float c0[2], c1[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      c0[k] = x.r[k] * quad_sum(m1[k]) * by_C;
      c1[k] = x.r[k] * x.r[k] * x.r[k] * quad_sum(m2[k]) * by_C;
    }
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      float(&u)[2][8] = u_all[kKeep ? kc : 0];
      if (!kKeep) u_of(kc, u);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (!row.on[k] || kc * 32 + t * 8 >= a.C) continue;
        float v[8];
        x.x[k][kc].floats(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(x.r[k], u[k][e], -fmaf(v[e] - x.mean[k], c1[k], c0[k]));
        Eight<T>::store(static_cast<T*>(a.dz) + (long long)row.n[k] * a.C + kc * 32 + t * 8, v);
      }
    }
  }
  if (!a.partial) return;
  // The warps add their sums in turn; q is the same for all channels.
  float* sums = reinterpret_cast<float*>(sm_g);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    s_acc[nt] = quad_sum(s_acc[nt]);
    q_acc[nt] = quad_sum(q_acc[nt]);
  }
  for (int w = 0; w < 8; ++w) {
    __syncthreads();
    if (warp != w) continue;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // head 8 nt + g is what the lane's s and q are of; its part of M is heads 2t, 2t + 1
      const float q0 = __shfl_sync(0xffffffffu, q_acc[nt], 8 * t), q1 = __shfl_sync(0xffffffffu, q_acc[nt], 8 * t + 4);
#pragma unroll
      for (int kc = 0; kc < KC; ++kc)
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int h = nt * 8 + 2 * t + e, c = kc * 32 + g / 2 * 8 + 2 * (2 * p + k) + (g & 1);
              if (h >= a.H || c >= a.C) continue;
              float& to = sums[h * (a.C + 1) + c];
              const float v = m_acc[kc][p][nt][2 * k + e] - (e ? q1 : q0);
              to = w ? to + v : v;
            }
      const int h = nt * 8 + g;
      if (t == 0 && h < a.H) {
        float& to = sums[h * (a.C + 1) + a.C];
        to = w ? to + s_acc[nt] : s_acc[nt];
      }
    }
  }
  __syncthreads();
  const int size = a.H * (a.C + 1);
  for (int i = threadIdx.x; i < size; i += 256) a.partial[(long long)blockIdx.x * size + i] = sums[i];
}

// ---------------------------------------------------------------- any call

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

// The blocks' sums, added in order, and the gradients of the weights from them.  A block has eight channels: 128 shares of
// the sums of eight heads at a time, a warp four of them.
__global__ void __launch_bounds__(1024) projection_weights(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  __shared__ float sm[32][8][9], sm_m[EVOATTN_PROJECTION_MAX_H][9];  // [..][8]: s
  const long long size = (long long)a.H * (a.C + 1);
  const int c0 = blockIdx.x * 8;
  for (int h0 = 0; h0 < a.H; h0 += 8) {
    // 32 shares of 8 heads x 4 pairs of channels would leave s out: 72 values, each summed by 14 threads
    for (int i = threadIdx.x; i < 72 * 32; i += 1024) {
      const int share = i / 72, v = i - share * 72, hh = v / 9, cc = v - hh * 9, h = h0 + hh, c = cc == 8 ? a.C : c0 + cc;
      float s = 0.f;
      if (h < a.H && c <= a.C && (cc == 8 || c < a.C)) {
        const float* p = a.partial + h * (a.C + 1) + c;
#pragma unroll 4
        for (int k = share; k < a.blocks; k += 32) s += p[k * size];
      }
      sm[share][hh][cc] = s;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 72; i += 1024) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) s += sm[k][i / 9][i % 9];
      if (h0 + i / 9 < a.H) sm_m[h0 + i / 9][i % 9] = s;
    }
    __syncthreads();
  }
  const int c = c0 + (int)threadIdx.x % 8;
  if (c >= a.C) return;
  if (a.dw && threadIdx.x / 8 < a.H) {
    const int h = threadIdx.x / 8;
    const float b = a.b ? load_any(a.b, a.b_dtype, c) : 0.f;
    store_any(a.dw, a.w_dtype, h * a.C + c, fmaf(gain(a, c), sm_m[h][threadIdx.x % 8], b * sm_m[h][8]));
  }
  if (threadIdx.x >= 8) return;
  float dg = 0.f, db = 0.f;
  for (int h = 0; h < a.H; ++h) {
    const float w = load_any(a.w, a.w_dtype, h * a.C + c);
    dg = fmaf(w, sm_m[h][threadIdx.x], dg);
    db = fmaf(w, sm_m[h][8], db);
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
  if (p->Ri > 0 && p->Rj > 0) {
    a.by_Ri = FastDiv((uint32_t)p->Ri);
    a.by_Rj = FastDiv((uint32_t)p->Rj);
  }
  return a;
}
long long rows_of(const ProjArgs& a) { return (long long)a.B * a.Ri * a.Rj; }
size_t stats_bytes(const ProjArgs& a) { return (size_t)((rows_of(a) * 8 + 15) / 16 * 16); }
int weights_smem(const ProjArgs& a) { return a.H * (a.C + 1) * (int)sizeof(float); }

// Whether the tensor-core kernels take a call: rows in pieces of eight channels and 16 bytes.  The backward holds M of all
// channels and heads in registers, which bounds their product.
bool rows_in_pieces(const ProjArgs& a, int es) {
  return a.C % 8 == 0 && rows_of(a) < (1LL << 31) && ((uintptr_t)a.z & 15) == 0 && a.sz.a * es % 16 == 0 && a.sz.b * es % 16 == 0 && a.sz.c * es % 16 == 0;
}
bool mma_fwd(const ProjArgs& a, int es) { return rows_in_pieces(a, es) && a.C <= (es == 2 ? 512 : 256); }
bool mma_bwd(const ProjArgs& a, int es) {
  if (!rows_in_pieces(a, es) || ((uintptr_t)a.dz & 15)) return false;
  if (es == 4) return a.C <= 128 && a.H <= 8;
  return (a.C <= 256 && a.H <= 8) || (a.C <= 128 && a.H <= 16);
}
template <int KC_, int NT_> struct Shape { static constexpr int KC = KC_, NT = NT_; };
template <class T, class F>
void with_fwd_shape(const ProjArgs& a, F&& f) {
  const auto heads = [&](auto kc) {
    constexpr int KC = decltype(kc)::value;
    if (a.H <= 8) f(Shape<KC, 1>());
    else if (a.H <= 16) f(Shape<KC, 2>());
    else if (a.H <= 32) f(Shape<KC, 4>());
    else f(Shape<KC, 8>());
  };
  if (a.C <= 64) heads(std::integral_constant<int, 2>());
  else if (a.C <= 128) heads(std::integral_constant<int, 4>());
  else if (a.C <= 256) heads(std::integral_constant<int, 8>());
  else if constexpr (sizeof(T) == 2) heads(std::integral_constant<int, 16>());
}
template <class T, class F>
void with_bwd_shape(const ProjArgs& a, F&& f) {
  if (a.H <= 8) {
    if (a.C <= 64) f(Shape<2, 1>());
    else if (a.C <= 128) f(Shape<4, 1>());
    else if constexpr (sizeof(T) == 2) f(Shape<8, 1>());
  } else if constexpr (sizeof(T) == 2) {
    if (a.C <= 64) f(Shape<2, 2>());
    else f(Shape<4, 2>());
  }
}
// Blocks of the backward, each of which leaves sums of H (C + 1) floats.
int bwd_blocks(const ProjArgs& a, bool mma) {
  const long long rows = rows_of(a), want = mma ? (rows + 127) / 128 : rows, most = mma ? 148 : 592;
  return (int)(want < most ? want : most);
}

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
  return with_dtype(p->dtype, [&](auto e) {
    using T = decltype(e);
    cudaError_t rc = cudaErrorUnknown;
    if (mma_fwd(a, (int)sizeof(T))) {
      with_fwd_shape<T>(a, [&](auto sh) {
        using Sh = decltype(sh);
        const auto kern = projection_fwd_mma<T, Sh::KC, Sh::NT>;
        const int smem = Sh::KC * Sh::NT * Pieces<T>::kG * 512;
        int regs = 0;
        if (!kernel_ready(reinterpret_cast<const void*>(kern), smem, &regs)) return;
        const int by_regs = 65536 / ((regs + 7) / 8 * 8 * 256), by_smem = 220 * 1024 / (smem + 2048);
        const long long blocks = (rows + 127) / 128, most = 148LL * (by_regs < by_smem ? by_regs : by_smem);
        rc = launch_dependent(kern, dim3((unsigned)(blocks < most ? blocks : most)), 256, (size_t)smem, st, a);
      });
    } else {
      const auto kern = projection_fwd<T>;
      if (!kernel_ready(reinterpret_cast<const void*>(kern), weights_smem(a), nullptr)) return (int)EVOATTN_ERR_CUDA;
      rc = launch_dependent(kern, dim3((unsigned)((rows + 7) / 8 < 148 * 4 ? (rows + 7) / 8 : 148 * 4)), 256, (size_t)weights_smem(a), st, a);
    }
    return (int)(rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA);
  });
}

size_t evoattn_pair_projection_bwd_workspace_bytes(const evoattn_pair_projection_params* p) {
  using namespace evo;
  if (validate(p) || !(p->dweight || p->dnorm_weight || p->dnorm_bias)) return 0;
  const ProjArgs a = args_of(p);
  const bool mma = mma_bwd(a, dtype_bytes(p->dtype));
  return (mma ? 0 : stats_bytes(a)) + (size_t)bwd_blocks(a, mma) * a.H * (a.C + 1) * sizeof(float);
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
  const bool sums = a.dw || a.dg || a.db, mma = mma_bwd(a, dtype_bytes(p->dtype));
  a.blocks = bwd_blocks(a, mma);
  if (sums) {
    unsigned char* ws = static_cast<unsigned char*>(p->workspace);
    if (!mma) a.stats = reinterpret_cast<float*>(ws);
    a.partial = reinterpret_cast<float*>(ws + (mma ? 0 : stats_bytes(a)));
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t rc = cudaSuccess;
  if (rows > 0 && (a.dz || sums))
    with_dtype(p->dtype, [&](auto e) {
      using T = decltype(e);
      rc = cudaErrorUnknown;
      if (mma) {
        with_bwd_shape<T>(a, [&](auto sh) {
          using Sh = decltype(sh);
          const auto kern = projection_bwd_mma<T, Sh::KC, Sh::NT>;
          const int pieces = Sh::KC * Sh::NT * Pieces<T>::kG * 512, smem = pieces > weights_smem(a) ? pieces : weights_smem(a);
          if (!kernel_ready(reinterpret_cast<const void*>(kern), smem, nullptr)) return;
          rc = launch_dependent(kern, dim3((unsigned)a.blocks), 256, (size_t)smem, st, a);
        });
        return 0;
      }
      const auto kern = projection_dz<T>;
      if (!kernel_ready(reinterpret_cast<const void*>(kern), weights_smem(a), nullptr)) return 0;
      rc = launch_dependent(kern, dim3((unsigned)((rows + 7) / 8 < 148 * 4 ? (rows + 7) / 8 : 148 * 4)), 256, (size_t)weights_smem(a), st, a);
      if (rc == cudaSuccess && sums)
        rc = launch_dependent(projection_sums<T>, dim3((unsigned)a.blocks, (unsigned)((a.C + 128) / 128), (unsigned)((a.H + 7) / 8)), 128, 0, st, a);
      return 0;
    });
  if (rc == cudaSuccess && sums) rc = launch_dependent(projection_weights, dim3((unsigned)((a.C + 7) / 8)), 1024, 0, st, a);
  return rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

}  // extern "C"
