// The pair representation's layer norm and its projection to a pair bias, heads first, in one pass:
//
//   xh = (z - mean) r,  G[h,c] = weight[h,c] g[c],  out[b,h,i,j] = sum_c G[h,c] xh[c] + sum_c weight[h,c] b[c]
//
// Backward, with u[c] = sum_h d[h] G[h,c], M[h,c] = sum over rows of d[h] xh[c] and s[h] = sum over rows of d[h]:
//
//   dz = r (u - mean(u) - xh mean(u xh))
//   dweight[h,c] = g[c] M[h,c] + b[c] s[h],  dg[c] = sum_h weight[h,c] M[h,c],  db[c] = sum_h weight[h,c] s[h]
//
// so the gradients of all three weights come from sums that do not depend on them.  [2,768,768,128] to 8 heads, bf16: 67 us (4.8 TB/s)
// and 144 (4.3 TB/s) on a card whose copies run at 6.5.  What is short is warps that cover the latency of loads and of one
// MMA after another, for want of registers: 22 of 64 warps an SM forward, with 58 % of DRAM and 59 % of the issue slots busy, and 16 of 64
// backward, with 49 and 55 %.
#include <string.h>

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
  FastDiv by_Ri, by_Rj;
  int z_dense;      // rows of z one after another
  int small;        // offsets of rows fit 32 bits
};

__device__ __forceinline__ float gain(const ProjArgs& a, int c) { return a.g ? load_any(a.g, a.g_dtype, c) : 1.f; }

// Few heads make the products thin (N = 8 heads or K = 8 heads), and the kernels are bound by the pair representation's way
// through memory; warp-level MMAs take their operands from the registers that the rows were loaded into, with no staging.
//
// A warp takes 16 rows.  Four lanes share a row: lane t of them loads channels 8 t .. 8 t + 7 of every 32, sixteen bytes in
// 16-bit types.  What a lane holds is at once the A operand of rows x channels (the channels that the MMA calls 2t, 2t + 1 and
// 2t + 8, 2t + 9 of a step are 8t + 4s .. 8t + 4s + 3 here; G is laid out to match), the accumulator layout of heads x
// channels products, and, transposed 8 x 8 at a time by movmatrix, the A operand of channels x rows.
//
// Products are of bf16 pieces with fp32 sums: an fp32 factor is the sum of three (24 bits), an fp16 one of two, a bf16 one
// is one.  z enters as it is: sum_c G z[c] - mean sum_c G, with both sums over the same pieces of G, and M likewise from d r z
// and d r mean.  G is two pieces (2^-17 of it is left out) where results are rounded to 16 bits, else three; d r always
// three, since the weights' gradients may be fp32.  The rows x channels product of fp16 rows takes them as they are, with G in
// two fp16 pieces, each head's times a power of two that brings its largest to 8 .. 16, so that no piece is too small for
// the type.  An MMA cuts its sums off where fp32 additions round: a sum that ends in fp32 is
// one of few MMAs, the products of low pieces first, and is added to the others in fp32.

__device__ __forceinline__ void mma_k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_k16_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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

// Two floats as N pieces of 16 bits each, packed by piece.
template <int N, class P = __nv_bfloat16>
__device__ __forceinline__ void split2(float lo, float hi, uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = Pack2<P>::pack(lo, hi);
    if (i + 1 < N) {
      float a, b;
      unpack2<P>(w[i], a, b);
      lo -= a;
      hi -= b;
    }
  }
}

template <class T> struct Pieces;  // pieces of a value of type T, and of G beside it; products of pieces i + j < kTerms
template <> struct Pieces<__nv_bfloat16> { static constexpr int kX = 1, kG = 2, kTerms = 2; };
template <> struct Pieces<__half> { static constexpr int kX = 2, kG = 2, kTerms = 3; };
template <> struct Pieces<float> { static constexpr int kX = 3, kG = 3, kTerms = 3; };
template <class T> constexpr bool kNativeRows = std::is_same<T, __half>::value;

// Eight channels of a row, the first `count` of which are there.
template <class T>
struct Eight {
  static constexpr int kWords = sizeof(T) / 2;
  uint4 w[kWords];
  // VEC: C and all rows are in pieces of as many channels (8: 16 bytes; 4: 8 bytes, fp32 16; else 1).
  template <int VEC>
  __device__ __forceinline__ void load(const T* p, int count) {
    if constexpr (VEC == 4) {
      using Four = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
      Four h[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        h[k] = Four();
        if (count > 4 * k) h[k] = reinterpret_cast<const Four*>(p)[k];
      }
      memcpy(w, h, sizeof(h));
    } else if constexpr (VEC == 8) {
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = count > 0 ? reinterpret_cast<const uint4*>(p)[k] : make_uint4(0, 0, 0, 0);
    } else {
      T v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < count ? p[e] : from_float<T>(0.f);
      memcpy(w, v, sizeof(v));
    }
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
  template <int VEC>
  static __device__ __forceinline__ void store(T* p, const float (&v)[8], int count) {
    if constexpr (VEC == 4) {
      using Four = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
      uint4 packed[kWords];
      Four h[2];
#pragma unroll
      for (int k = 0; k < kWords; ++k) packed[k] = pack16<T>(v + k * kPer16<T>);
      memcpy(h, packed, sizeof(h));
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (count > 4 * k) reinterpret_cast<Four*>(p)[k] = h[k];
    } else if constexpr (VEC == 8) {
#pragma unroll
      for (int k = 0; k < kWords; ++k)
        if (count > 0) reinterpret_cast<uint4*>(p)[k] = pack16<T>(v + k * kPer16<T>);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) p[e] = from_float<T>(v[e]);
    }
  }
};

// Weights first + lane, first + lane + 32, ... as they lie, and then as floats: a warp's loads all go out before one is used.
template <int KC>
__device__ __forceinline__ void load_bits(const void* p, int dtype, long long first, int n, uint32_t (&bits)[KC]) {
  const int lane = threadIdx.x & 31;
  if (dtype == EVOATTN_FP32) {
#pragma unroll
    for (int k = 0; k < KC; ++k) bits[k] = lane + 32 * k < n ? static_cast<const uint32_t*>(p)[first + lane + 32 * k] : 0;
  } else {
#pragma unroll
    for (int k = 0; k < KC; ++k) bits[k] = lane + 32 * k < n ? static_cast<const uint16_t*>(p)[first + lane + 32 * k] : 0;
  }
}
__device__ __forceinline__ float of_bits(int dtype, uint32_t bits) {
  return dtype == EVOATTN_FP32 ? __uint_as_float(bits) : dtype == EVOATTN_BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits));
}

// A kernel's weights: G in pieces as B operands of rows x channels products, and as those of heads x channels products, both
// [KC][NT][pieces][lane] (null: not wanted); the sum over the channels of the pieces of G and that of weight b for every
// head.  Eight heads at a time, one a warp.  Ends with a barrier.
// sm_scale: what products by rows are to be multiplied by (null: 1).
template <class T, int KC, int NT>
__device__ __forceinline__ void prepare_weights(const ProjArgs& a, uint4* by_rows, uint4* by_heads, float* sm_sum, float* sm_t, float* sm_scale) {
  constexpr int GP = Pieces<T>::kG;
  using P = typename std::conditional<kNativeRows<T>, __half, __nv_bfloat16>::type;  // pieces of products by rows
  __shared__ float sm_G[8][32 * KC + 4];  // (4 floats apart: eight heads in different banks)
  __shared__ float sm_up[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int nt = 0; nt < NT; ++nt) {
    const int h = nt * 8 + warp;
    const bool biased = a.b && sm_t;
    uint32_t w[KC], gains[KC], biases[KC];
    load_bits<KC>(a.w, a.w_dtype, (long long)h * a.C, h < a.H ? a.C : 0, w);
    if (a.g) load_bits<KC>(a.g, a.g_dtype, 0, a.C, gains);
    if (biased) load_bits<KC>(a.b, a.b_dtype, 0, a.C, biases);
    if (nt) __syncthreads();
    float s = 0.f, tb = 0.f, G[KC], most = 0.f;
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      const float weight = of_bits(a.w_dtype, w[k]);
      G[k] = a.g ? weight * of_bits(a.g_dtype, gains[k]) : weight;
      if (biased) tb = fmaf(weight, of_bits(a.b_dtype, biases[k]), tb);
      sm_G[warp][lane + 32 * k] = G[k];
      most = fmaxf(most, fabsf(G[k]));
    }
    if constexpr (kNativeRows<T>) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      int up = most > 0.f && most < INFINITY ? 3 - ilogbf(most) : 0;
      up = min(max(up, -100), 100);
      if (lane == 0) sm_up[warp] = scalbnf(1.f, up);
      if (sm_scale && lane == 0) sm_scale[h] = scalbnf(1.f, -up);
      __syncwarp();
    }
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      uint32_t p[GP];
      split2<GP, P>(kNativeRows<T> ? G[k] * sm_up[warp] : G[k], 0.f, p);
      float v = 0.f;
#pragma unroll
      for (int j = GP - 1; j >= 0; --j) {
        float lo, hi;
        unpack2<P>(p[j], lo, hi);
        v += lo;
      }
      s += v;
    }
    if (sm_sum) {
      s = warp_sum(s);
      if (biased) tb = warp_sum(tb);
      if (lane == 0) {
        sm_sum[h] = kNativeRows<T> && sm_scale ? s * sm_scale[h] : s;
        if (sm_t) sm_t[h] = tb;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < KC * 32; i += blockDim.x) {
      const int l = i & 31, kc = i >> 5;
      const auto write = [&](uint4* sm, const float (&v)[8], auto piece) {
        uint32_t p[4][GP];
#pragma unroll
        for (int k = 0; k < 4; ++k) split2<GP, decltype(piece)>(v[2 * k], v[2 * k + 1], p[k]);
#pragma unroll
        for (int j = 0; j < GP; ++j) sm[((kc * NT + nt) * GP + j) * 32 + l] = make_uint4(p[0][j], p[1][j], p[2][j], p[3][j]);
      };
      float v[8];
      if (by_rows) {  // eight channels of head l / 4
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = sm_G[l / 4][kc * 32 + (l & 3) * 8 + k] * (kNativeRows<T> ? sm_up[l / 4] : 1.f);
        write(by_rows, v, P());
      }
      if (by_heads) {  // pairs of heads of the four channels of a lane's accumulators
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = sm_G[(l & 3) * 2 + (k & 1)][kc * 32 + l / 8 * 8 + (l / 4 & 1) + (k & ~1)];
        write(by_heads, v, __nv_bfloat16());
      }
    }
  }
  __syncthreads();
}

// A lane's two rows of a tile: g and g + 8.
struct Rows2 {
  long long z[2], o[2];
  uint32_t n0;
  bool on[2];
  __device__ __forceinline__ Rows2(const ProjArgs& a, uint32_t first, uint32_t rows) : n0(first) {
    const uint32_t q0 = a.by_Rj.div(first), j0 = first - q0 * a.Rj, b0 = a.by_Ri.div(q0), i0 = q0 - b0 * a.Ri;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t n = row(k);
      uint32_t j = j0 + (n - first), i = i0, b = b0;
      on[k] = n < rows;
      while (j >= (uint32_t)a.Rj) {
        j -= a.Rj;
        if (++i == (uint32_t)a.Ri) i = 0, ++b;
      }
      if (a.small) {
        z[k] = (int)(a.z_dense ? n * (int)a.sz.c : b * (int)a.sz.a + i * (int)a.sz.b + j * (int)a.sz.c);
        o[k] = (int)(b * (int)a.sout.a + i * (int)a.sout.c + j);
      } else {
        z[k] = b * a.sz.a + i * a.sz.b + j * a.sz.c;
        o[k] = b * a.sout.a + i * a.sout.c + j;
      }
    }
  }
  __device__ __forceinline__ uint32_t row(int k) const { return n0 + (threadIdx.x & 31) / 4 + 8 * k; }
};

// 16 rows, 32 KC channels.  KEEP: in registers; else read again (from L1 or L2) by every use.
template <class T, int KC, bool KEEP, int VEC_>
struct Tile {
  static constexpr int VEC = VEC_;
  static constexpr int kUnroll = KEEP ? KC : 1;
  static_assert(KC % 2 == 0, "statistics() takes two times 32 channels at once");
  Eight<T> x[2][KEEP ? KC : 1];
  const T* at[2];
  bool on[2];
  float mean[2], r[2];
  __device__ __forceinline__ int count(const ProjArgs& a, int c) const { return a.C - c * 32 - (int)(threadIdx.x & 3) * 8; }
  __device__ __forceinline__ void load(const ProjArgs& a, const Rows2& row) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      at[k] = static_cast<const T*>(a.z) + row.z[k] + (threadIdx.x & 3) * 8;
      on[k] = row.on[k];
      if constexpr (KEEP) {
#pragma unroll
        for (int c = 0; c < KC; ++c) x[k][c].template load<VEC>(at[k] + c * 32, on[k] ? count(a, c) : 0);
      }
    }
  }
  __device__ __forceinline__ Eight<T> get(const ProjArgs& a, int k, int c) const {
    if constexpr (KEEP) return x[k][c];
    Eight<T> e;
    e.template load<VEC>(at[k] + c * 32, on[k] ? count(a, c) : 0);
    return e;
  }
  // Mean and 1 / deviation, the latter about the mean; a row that is not there has r = 0 and adds nothing.
  __device__ __forceinline__ void about_the_mean(const ProjArgs& a) {
    const float by_C = 1.f / a.C;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float s = 0.f;
#pragma unroll kUnroll
      for (int c = 0; c < KC; ++c) {
        float v[8];
        get(a, k, c).floats(v);
        s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      }
      mean[k] = quad_sum(s) * by_C;
      s = 0.f;
#pragma unroll kUnroll
      for (int c = 0; c < KC; ++c) {
        float v[8];
        get(a, k, c).floats(v);
        const int there = count(a, c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float d = e < there ? v[e] - mean[k] : 0.f;
          s = fmaf(d, d, s);
        }
      }
      s = quad_sum(s);  // (all lanes, rows that are not there too)
      r[k] = on[k] ? rsqrtf(s * by_C + a.eps) : 0.f;
    }
  }
  // In 16-bit types both sums come from MMAs: with a column of ones, and the diagonal of rows x rows (the registers of the A
  // operand are those of its transpose as B).  The variance is then a difference: where the mean is at most twice the deviation, five
  // times as far off, relative to it, as the mean square is; other rows are done the other way.  What MMAs cut off always makes a
  // sum of squares smaller, so a sum is of four (64 channels), 2.5 * 2^-23 of it at most, and these are added in fp32.  One sum over all
  // channels had r up to 3.8e-6 too large (512 channels, fp16), these 2.6e-7; 32 channels a sum cost registers: forward of
  // [2,768,768,128] to 8 heads, bf16, 72 -> 78 us, backward 144 -> 154.
  __device__ __forceinline__ void statistics(const ProjArgs& a) {
    if constexpr (sizeof(T) == 4) {
      about_the_mean(a);
    } else {
      constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
      constexpr uint32_t ones = bf ? 0x3f803f80u : 0x3c003c00u;
      const auto mma = [](float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        if constexpr (bf) mma_k16(d, a0, a1, a2, a3, b0, b1);
        else mma_k16_f16(d, a0, a1, a2, a3, b0, b1);
      };
      const float by_C = 1.f / a.C;
      const int lane = threadIdx.x & 31, g = lane >> 2, diagonal = (lane & ~3) | (g >> 1);
      float total[2] = {}, square[2] = {};
#pragma unroll kUnroll
      for (int c0 = 0; c0 < KC; c0 += 2) {
        float sum[4] = {}, lo[4] = {}, hi[4] = {};
#pragma unroll
        for (int c = c0; c < c0 + 2; ++c) {
          const uint4 l = get(a, 0, c).w[0], h = get(a, 1, c).w[0];
          mma(sum, l.x, h.x, l.y, h.y, ones, ones);
          mma(lo, l.x, h.x, l.y, h.y, l.x, l.y);
          mma(hi, l.x, h.x, l.y, h.y, h.x, h.y);
          mma(sum, l.z, h.z, l.w, h.w, ones, ones);
          mma(lo, l.z, h.z, l.w, h.w, l.z, l.w);
          mma(hi, l.z, h.z, l.w, h.w, h.z, h.w);
        }
        total[0] += sum[0];
        total[1] += sum[2];
        square[0] += g & 1 ? lo[1] : lo[0];  // (on the diagonal in one of the row's four lanes)
        square[1] += g & 1 ? hi[3] : hi[2];
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) square[k] = __shfl_sync(0xffffffffu, square[k], diagonal);
      float quick_mean[2], quick_r[2];
      bool fine[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        quick_mean[k] = total[k] * by_C;
        const float var = fmaf(-quick_mean[k], quick_mean[k], square[k] * by_C);
        fine[k] = quick_mean[k] * quick_mean[k] <= 4.f * var;
        quick_r[k] = on[k] ? rsqrtf(var + a.eps) : 0.f;
      }
      if (!__all_sync(0xffffffffu, fine[0] && fine[1])) about_the_mean(a);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (fine[k]) mean[k] = quick_mean[k], r[k] = quick_r[k];  // (what a row gets does not depend on its neighbours)
    }
  }
};

// acc[nt] += rows x channels of the tile with G (laid out by rows).
template <class T, int KC, int NT, class TileT>
__device__ __forceinline__ void product_by_rows(const ProjArgs& a, const TileT& x, const uint4* sm_g, float (&acc)[NT][4]) {
  constexpr int GP = Pieces<T>::kG, XP = Pieces<T>::kX;
  const int lane = threadIdx.x & 31;
#pragma unroll TileT::kUnroll
  for (int kc = 0; kc < KC; ++kc) {
    if constexpr (kNativeRows<T>) {
      const uint4 l = x.get(a, 0, kc).w[0], h = x.get(a, 1, kc).w[0];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = GP - 1; j >= 0; --j) {
          const uint4 gw = sm_g[((kc * NT + nt) * GP + j) * 32 + lane];
          mma_k16_f16(acc[nt], l.x, h.x, l.y, h.y, gw.x, gw.y);
          mma_k16_f16(acc[nt], l.z, h.z, l.w, h.w, gw.z, gw.w);
        }
      continue;
    }
    uint32_t lo[4][XP], hi[4][XP];
    x.get(a, 0, kc).pieces(lo);
    x.get(a, 1, kc).pieces(hi);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float chunk[4] = {};
      float(&sum)[4] = sizeof(T) == 4 ? chunk : acc[nt];
      uint4 gw[GP];
#pragma unroll
      for (int j = 0; j < GP; ++j) gw[j] = sm_g[((kc * NT + nt) * GP + j) * 32 + lane];
#pragma unroll
      for (int order = Pieces<T>::kTerms - 1; order >= 0; --order)
#pragma unroll
        for (int i = 0; i < XP; ++i) {
          const int j = order - i;
          if (j < 0 || j >= GP) continue;
          mma_k16(sum, lo[0][i], hi[0][i], lo[1][i], hi[1][i], gw[j].x, gw[j].y);
          mma_k16(sum, lo[2][i], hi[2][i], lo[3][i], hi[3][i], gw[j].z, gw[j].w);
        }
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][e] += chunk[e];
      }
    }
  }
}

// Three blocks an SM where the registers allow it: [1,768,768,128] to 8 heads 47 -> 43 us, fp16 56 -> 51.
template <class T, int KC, int NT, bool KEEP, int VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && KC <= 4 && NT <= 2 && VEC == 8 && KEEP ? 3 : 0) projection_fwd(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  extern __shared__ __align__(16) uint4 sm_g[];  // [KC][NT][GP][32 lanes]
  __shared__ float sm_sum[NT * 8], sm_t[NT * 8], sm_scale[NT * 8];
  const int warp = threadIdx.x >> 5, t = threadIdx.x & 3;
  const uint32_t rows = (uint32_t)((long long)a.B * a.Ri * a.Rj), step = gridDim.x * 128;
  Rows2 next(a, (blockIdx.x * 8 + warp) * 16, rows);
  Tile<T, KC, KEEP, VEC> x;
  x.load(a, next);
  prepare_weights<T, KC, NT>(a, sm_g, nullptr, sm_sum, sm_t, sm_scale);
  while (next.n0 < rows) {
    const Rows2 row = next;
    x.statistics(a);
    float acc[NT][4] = {};
    product_by_rows<T, KC, NT>(a, x, sm_g, acc);
    const float mean[2] = {x.mean[0], x.mean[1]}, r[2] = {x.r[0], x.r[1]};
    next = Rows2(a, row.n0 + step, rows);
    x.load(a, next);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = nt * 8 + 2 * t + e;
        if (h >= a.H) continue;
        const float sum = sm_sum[h], tb = sm_t[h], scale = kNativeRows<T> ? sm_scale[h] : 1.f;
        T* out = static_cast<T*>(a.out) + h * a.sout.b;
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (row.on[k]) out[row.o[k]] = from_float<T>(fmaf(fmaf(-mean[k], sum, acc[nt][2 * k + e] * scale), r[k], tb));
      }
  }
}

// d of a lane's two rows and heads 8 nt + 2t, 8 nt + 2t + 1, as pieces.
template <class T, int NT>
__device__ __forceinline__ void load_d(const ProjArgs& a, const Rows2& row, int nt0, float (&d)[NT][2][2], uint32_t (&dp)[NT][2][Pieces<T>::kX]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int h = (nt0 + nt) * 8 + 2 * (threadIdx.x & 3) + e;
      const T* p = static_cast<const T*>(a.out) + h * a.sout.b;
#pragma unroll
      for (int k = 0; k < 2; ++k) d[nt][k][e] = row.on[k] && h < a.H ? to_float<T>(p[row.o[k]]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) split2<Pieces<T>::kX>(d[nt][k][0], d[nt][k][1], dp[nt][k]);
  }
}

// Sums over the rows: M before the mean is taken out (d r z), s (d) and q (d r mean), of 32 KC channels and 8 NT heads.
template <class T, int KC, int NT>
struct RowSums {
  static constexpr int XP = Pieces<T>::kX, AP = 3;
  float m[KC][2][NT][4] = {}, s[NT] = {}, q[NT] = {};
  template <class TileT>
  __device__ __forceinline__ void add(const ProjArgs& a, const TileT& x, const uint32_t (&dp)[NT][2][XP]) {
    const int t = threadIdx.x & 3;
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
        s[nt] += d0 + d1;
        d0 *= r[k][0];
        d1 *= r[k][1];
        q[nt] = fmaf(d0, mean[k][0], fmaf(d1, mean[k][1], q[nt]));
        split2<AP>(d0, d1, ap[nt][k]);
      }
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      uint32_t lo[4][XP], hi[4][XP];
      x.get(a, 0, kc).pieces(lo);
      x.get(a, 1, kc).pieces(hi);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint32_t at[XP][4];
#pragma unroll
        for (int i = 0; i < XP; ++i) {
          at[i][0] = transposed(lo[2 * p][i]);
          at[i][1] = transposed(lo[2 * p + 1][i]);
          at[i][2] = transposed(hi[2 * p][i]);
          at[i][3] = transposed(hi[2 * p + 1][i]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float sum[4] = {};
#pragma unroll
          for (int order = AP - 1; order >= 0; --order)
#pragma unroll
            for (int i = 0; i < XP; ++i)
              if (order - i >= 0) mma_k16(sum, at[i][0], at[i][1], at[i][2], at[i][3], ap[nt][0][order - i], ap[nt][1][order - i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) m[kc][p][nt][e] += sum[e];
        }
      }
    }
  }
  // The block's sums in shared memory, [8 NT heads][32 KC + 1]: its warps add theirs in turn.  q is the same for all channels.
  __device__ __forceinline__ void leave(float* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, pitch = 32 * KC + 1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      s[nt] = quad_sum(s[nt]);
      q[nt] = quad_sum(q[nt]);
    }
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
      __syncthreads();
      if (warp != w) continue;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // head 8 nt + g is what the lane's s and q are of; its part of M is heads 2t, 2t + 1
        const float q0 = __shfl_sync(0xffffffffu, q[nt], 8 * t), q1 = __shfl_sync(0xffffffffu, q[nt], 8 * t + 4);
#pragma unroll
        for (int kc = 0; kc < KC; ++kc)
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float& to = sums[(nt * 8 + 2 * t + e) * pitch + kc * 32 + g / 2 * 8 + 2 * (2 * p + k) + (g & 1)];
                const float v = m[kc][p][nt][2 * k + e] - (e ? q1 : q0);
                to = w ? to + v : v;
              }
        float& to = sums[(nt * 8 + g) * pitch + 32 * KC];
        if (t == 0) to = w ? to + s[nt] : s[nt];
      }
    }
    __syncthreads();
  }
};
// From there to the block's partial sums [H][C + 1]: heads h0 .. and channels c0 .. of them, s by the first channels' block.
template <int KC, int NT>
__device__ __forceinline__ void write_partial(const ProjArgs& a, const float* sums, int block, int h0, int c0) {
  constexpr int pitch = 32 * KC + 1;
  float* out = a.partial + (long long)block * a.H * (a.C + 1);
  for (int i = threadIdx.x; i < 8 * NT * pitch; i += blockDim.x) {
    const int h = h0 + i / pitch, k = i % pitch, c = c0 + k;
    if (h >= a.H) break;
    if (k == 32 * KC) {
      if (c0 == 0) out[h * (a.C + 1) + a.C] = sums[i];
    } else if (c < a.C) {
      out[h * (a.C + 1) + c] = sums[i];
    }
  }
}

// u[c] = sum_h d[h] G[h,c] of chunk kc in the layout of the lane's eight channels.  With d in one piece, its products with both
// pieces of G are one MMA: K = 8 heads with the first and the same 8 heads with the second.
template <class T, int NT>
__device__ __forceinline__ void product_by_heads(const uint4* sm_u, int kc, const uint32_t (&dp)[NT][2][Pieces<T>::kX], float (&u)[2][8]) {
  constexpr int GP = Pieces<T>::kG, XP = Pieces<T>::kX;
  const int lane = threadIdx.x & 31;
  float acc[4][4] = {};
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    uint32_t gw[GP][4];
#pragma unroll
    for (int j = 0; j < GP; ++j) *reinterpret_cast<uint4*>(gw[j]) = sm_u[((kc * NT + nt) * GP + j) * 32 + lane];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (XP == 1) {
        mma_k16(acc[q], dp[nt][0][0], dp[nt][1][0], dp[nt][0][0], dp[nt][1][0], gw[0][q], gw[1][q]);
      } else {
#pragma unroll
        for (int order = Pieces<T>::kTerms - 1; order >= 0; --order)
#pragma unroll
          for (int i = 0; i < XP; ++i) {
            const int j = order - i;
            if (j >= 0 && j < GP) mma_k8(acc[q], dp[nt][0][i], dp[nt][1][i], gw[j][q]);
          }
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    u[0][2 * q] = acc[q][0]; u[0][2 * q + 1] = acc[q][1]; u[1][2 * q] = acc[q][2]; u[1][2 * q + 1] = acc[q][3];
  }
}

// dz = r (u - c0 - (z - mean) c1) with c0 = mean(u), c1 = r^2 mean(u (z - mean)), two channels an instruction.  Powers of r are never
// formed by themselves, and r comes last: each factor is of the size of a result then, where r^3 alone, or r c1, leaves
// fp32's range in rows that deviate by 10^14 or by 10^-14.  (One multiplication more: backward of [2,768,768,128] to 8 heads, bf16, 141 -> 143 us.)
template <class T, int KC, int NT, class TileT>
__device__ __forceinline__ void write_dz(const ProjArgs& a, const TileT& x, const Rows2& row, const uint4* sm_u, const uint32_t (&dp)[NT][2][Pieces<T>::kX],
                                         const float (&c0)[2], const float (&c1)[2]) {
  ptx::F2 by_r[2], by_z[2], rest[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float more = fmaf(x.mean[k], c1[k], -c0[k]);
    by_r[k] = ptx::f2_make(x.r[k], x.r[k]);
    by_z[k] = ptx::f2_make(-c1[k], -c1[k]);
    rest[k] = ptx::f2_make(more, more);
  }
#pragma unroll TileT::kUnroll
  for (int kc = 0; kc < KC; ++kc) {
    float u[2][8];
    product_by_heads<T, NT>(sm_u, kc, dp, u);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float v[8];
      x.get(a, k, kc).floats(v);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const ptx::F2 z = ptx::f2_fma(ptx::f2_make(v[e], v[e + 1]), by_z[k], rest[k]);
        ptx::f2_get(ptx::f2_mul(ptx::f2_add(ptx::f2_make(u[k][e], u[k][e + 1]), z), by_r[k]), v[e], v[e + 1]);
      }
      if (row.on[k])
        Eight<T>::template store<TileT::VEC>(static_cast<T*>(a.dz) + (long long)row.row(k) * a.C + kc * 32 + (threadIdx.x & 3) * 8, v, x.count(a, kc));
    }
  }
}

// c0 = sum_c u and c1 = sum_c u (z - mean) of a lane's two rows, as far as the lane's heads go:
//   sum_c u = sum_h d[h] sum_c G[h,c],   sum_c u (z - mean) = sum_h d[h] (sum_c G[h,c] z[c] - mean sum_c G[h,c]),
// the latter with the product that the forward takes.
template <class T, int KC, int NT, class TileT>
__device__ __forceinline__ void sums_over_heads(const ProjArgs& a, const TileT& x, const uint4* by_rows, const float* sm_sum, const float* sm_scale, const float (&d)[NT][2][2],
                                                float (&c0)[2], float (&c1)[2]) {
  float acc[NT][4] = {};
  product_by_rows<T, KC, NT>(a, x, by_rows, acc);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int h = nt * 8 + 2 * (threadIdx.x & 3) + e;
      const float sum = sm_sum[h], scale = kNativeRows<T> ? sm_scale[h] : 1.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        c0[k] = fmaf(d[nt][k][e], sum, c0[k]);
        c1[k] = fmaf(d[nt][k][e], fmaf(-x.mean[k], sum, acc[nt][2 * k + e] * scale), c1[k]);
      }
    }
}

// Backward in one pass over z: dz, and M and s of the block's rows.
// Two blocks an SM where the registers allow it (bf16, 128 channels, 8 heads: one block of 148 registers 116 us, two of 128 95 us).
template <class T, int KC, int NT, int VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && KC <= 4 && NT == 1 && VEC == 8 ? 2 : 1) projection_bwd(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int kG = KC * NT * Pieces<T>::kG * 32;
  extern __shared__ __align__(16) uint4 sm_g[];  // G by rows, G by heads; behind the rows' loop, the sums
  __shared__ float sm_sum[NT * 8], sm_scale[NT * 8];
  const int warp = threadIdx.x >> 5;
  const uint32_t rows = (uint32_t)((long long)a.B * a.Ri * a.Rj), step = gridDim.x * 128;
  if (a.dz) prepare_weights<T, KC, NT>(a, sm_g, sm_g + kG, sm_sum, nullptr, sm_scale);
  const float by_C = 1.f / a.C;
  RowSums<T, KC, NT> sums;
  for (uint32_t n0 = (blockIdx.x * 8 + warp) * 16; n0 < rows; n0 += step) {
    const Rows2 row(a, n0, rows);
    Tile<T, KC, true, VEC> x;
    x.load(a, row);
    float d[NT][2][2];
    uint32_t dp[NT][2][Pieces<T>::kX];
    load_d<T, NT>(a, row, 0, d, dp);
    x.statistics(a);
    if (a.partial) sums.add(a, x, dp);
    if (!a.dz) continue;
    float c0[2] = {}, c1[2] = {};
    sums_over_heads<T, KC, NT>(a, x, sm_g, sm_sum, sm_scale, d, c0, c1);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      c0[k] = quad_sum(c0[k]) * by_C;
      c1[k] = x.r[k] * (x.r[k] * (quad_sum(c1[k]) * by_C));
    }
    write_dz<T, KC, NT>(a, x, row, sm_g + kG, dp, c0, c1);
  }
  if (!a.partial) return;
  sums.leave(reinterpret_cast<float*>(sm_g));
  write_partial<KC, NT>(a, reinterpret_cast<const float*>(sm_g), blockIdx.x, 0, 0);
}

// Whether the sums over heads are taken (with G in both layouts) where rows are kept: [1,512,512,256] to 16 heads, bf16, backward 198 ->
// 169 us.  Rows that are read again for every use are better off with u worked out twice ([1,768,768,384] to 8 531, not 596).
template <class T>
__host__ __device__ constexpr bool both_layouts(int KC, int NT, bool keep) { return keep && KC * NT * Pieces<T>::kG <= 192; }

// More channels and heads than one block can hold the sums of: dz and the rows' statistics in one kernel ...
// Up to 16 heads of 512 channels the compiler would otherwise spill for a fourth block an SM: backward of [1,768,768,512] to 16, bf16, 739 us
// with three, 830 with four.
template <class T, int KC, int NT, bool KEEP, int VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && KC == 16 && NT == 2 && VEC == 8 ? 3 : 0) projection_dz(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr bool kBoth = both_layouts<T>(KC, NT, KEEP);
  constexpr int kG = KC * NT * Pieces<T>::kG * 32;
  extern __shared__ __align__(16) uint4 sm_g[];  // G by heads, and by rows if kBoth
  __shared__ float sm_sum[NT * 8], sm_scale[NT * 8];
  const int warp = threadIdx.x >> 5;
  const uint32_t rows = (uint32_t)((long long)a.B * a.Ri * a.Rj), step = gridDim.x * 128;
  if (a.dz) prepare_weights<T, KC, NT>(a, kBoth ? sm_g + kG : nullptr, sm_g, sm_sum, nullptr, sm_scale);
  const float by_C = 1.f / a.C;
  for (uint32_t n0 = (blockIdx.x * 8 + warp) * 16; n0 < rows; n0 += step) {
    const Rows2 row(a, n0, rows);
    Tile<T, KC, KEEP, VEC> x;
    x.load(a, row);
    x.statistics(a);
    if (a.stats && (threadIdx.x & 3) == 0) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (row.on[k]) reinterpret_cast<float2*>(a.stats)[row.row(k)] = make_float2(x.mean[k], x.r[k]);
    }
    if (!a.dz) continue;
    float d[NT][2][2], c0[2] = {}, c1[2] = {};
    uint32_t dp[NT][2][Pieces<T>::kX];
    load_d<T, NT>(a, row, 0, d, dp);
    if constexpr (kBoth) {
      sums_over_heads<T, KC, NT>(a, x, sm_g + kG, sm_sum, sm_scale, d, c0, c1);
    } else {
#pragma unroll KEEP ? KC : 1
      for (int kc = 0; kc < KC; ++kc) {
        float u[2][8];
        product_by_heads<T, NT>(sm_g, kc, dp, u);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float v[8];
          x.get(a, k, kc).floats(v);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            c0[k] += u[k][e];
            c1[k] = fmaf(u[k][e], v[e] - x.mean[k], c1[k]);  // (channels that are not there have u = 0)
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      c0[k] = quad_sum(c0[k]) * by_C;
      c1[k] = x.r[k] * (x.r[k] * (quad_sum(c1[k]) * by_C));
    }
    write_dz<T, KC, NT>(a, x, row, sm_g, dp, c0, c1);
  }
}

// ... and M and s of 128 channels and 16 heads a block in another, with those statistics.
constexpr int kSumChannels = 128, kSumHeads = 16;
template <class T, int VEC>
__global__ void __launch_bounds__(256) projection_sums(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int KC = kSumChannels / 32, NT = kSumHeads / 8;
  __shared__ float sm[kSumHeads * (kSumChannels + 1)];
  const int warp = threadIdx.x >> 5, c0 = blockIdx.y * kSumChannels, h0 = blockIdx.z * kSumHeads;
  const uint32_t rows = (uint32_t)((long long)a.B * a.Ri * a.Rj), step = gridDim.x * 128;
  ProjArgs part = a;  // these channels of z
  part.z = static_cast<const T*>(a.z) + c0;
  part.C = a.C - c0;
  RowSums<T, KC, NT> sums;
  for (uint32_t n0 = (blockIdx.x * 8 + warp) * 16; n0 < rows; n0 += step) {
    const Rows2 row(a, n0, rows);
    Tile<T, KC, true, VEC> x;
    x.load(part, row);
    float d[NT][2][2];
    uint32_t dp[NT][2][Pieces<T>::kX];
    load_d<T, NT>(a, row, h0 / 8, d, dp);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float2 st = row.on[k] ? reinterpret_cast<const float2*>(a.stats)[row.row(k)] : make_float2(0.f, 0.f);
      x.mean[k] = st.x;
      x.r[k] = st.y;
    }
    sums.add(part, x, dp);
  }
  sums.leave(sm);
  write_partial<KC, NT>(a, sm, blockIdx.x, h0, c0);
}

// The blocks' sums, added in order, and the gradients of the weights from them.  A block has two channels and sums eight heads
// at a time: 24 values (the third of a head: s), each in 42 shares, so that a thread's few loads go out at once.
constexpr int kWeightChannels = 2, kShares = 42;
__global__ void __launch_bounds__(1024) projection_weights(ProjArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int V = kWeightChannels + 1;
  __shared__ float sm[kShares][8 * V], sm_m[EVOATTN_PROJECTION_MAX_H][V];
  const long long size = (long long)a.H * (a.C + 1);
  const int c0 = blockIdx.x * kWeightChannels, share = threadIdx.x / (8 * V), v = threadIdx.x % (8 * V), hh = v / V, cc = v % V;
  for (int h0 = 0; h0 < a.H; h0 += 8) {
    const int h = h0 + hh, c = cc == kWeightChannels ? a.C : c0 + cc;
    if (share < kShares) {
      float s = 0.f;
      if (h < a.H && (cc == kWeightChannels || c < a.C)) {
        const float* p = a.partial + h * (a.C + 1) + c;
#pragma unroll 8
        for (int k = share; k < a.blocks; k += kShares) s += p[k * size];
      }
      sm[share][v] = s;
    }
    __syncthreads();
    if (threadIdx.x < 8 * V && h < a.H) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kShares; ++k) s += sm[k][v];
      sm_m[h][cc] = s;
    }
    __syncthreads();
  }
  const int mine = threadIdx.x % kWeightChannels, c = c0 + mine, h = threadIdx.x / kWeightChannels;
  if (c >= a.C) return;
  if (a.dw && h < a.H) {
    const float b = a.b ? load_any(a.b, a.b_dtype, c) : 0.f;
    store_any(a.dw, a.w_dtype, h * a.C + c, fmaf(gain(a, c), sm_m[h][mine], b * sm_m[h][kWeightChannels]));
  }
  if (threadIdx.x >= kWeightChannels) return;
  float dg = 0.f, db = 0.f;
#pragma unroll 8
  for (int k = 0; k < a.H; ++k) {
    const float w = load_any(a.w, a.w_dtype, k * a.C + c);
    dg = fmaf(w, sm_m[k][mine], dg);
    db = fmaf(w, sm_m[k][kWeightChannels], db);
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
  if ((long long)p->B * p->Ri > 0x7fffffffLL / (p->Rj > 0 ? p->Rj : 1)) return EVOATTN_ERR_SHAPE;  // rows are counted in 32 bits
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
// The channels of a piece in which rows of z (and dz) can be read and written: 8 (16 bytes, fp32 twice), 4 or 1.
int vector_of(const ProjArgs& a, int es) {
  for (int vec = 8; vec >= 4; vec /= 2) {
    const int bytes = vec * es < 16 ? vec * es : 16;
    if (a.C % vec == 0 && ((uintptr_t)a.z | (uintptr_t)a.dz | (uintptr_t)(a.sz.a * es) | (uintptr_t)(a.sz.b * es) | (uintptr_t)(a.sz.c * es)) % bytes == 0) return vec;
  }
  return 1;
}
void look_at_rows(ProjArgs* a) {
  const auto reach = [](const Str3& s, long long x, long long y, long long z) {
    const auto size = [](long long v) { return (double)(v < 0 ? -v : v); };
    return size(s.a) * x + size(s.b) * y + size(s.c) * z;
  };
  a->z_dense = a->sz.b == a->Rj * a->sz.c && a->sz.a == a->Ri * a->sz.b;
  // (sout.b is the heads', which are not part of a row's offset; row numbers run up to a tile beyond the last)
  a->small = reach(a->sz, a->B + 1, a->Ri, a->Rj + 64) < 2147483647.0 && reach(Str3{a->sout.a, a->sout.c, 1}, a->B + 1, a->Ri, a->Rj) < 2147483647.0;
}

template <int KC_, int NT_, bool KEEP_, int VEC_> struct Shape { static constexpr int KC = KC_, NT = NT_, VEC = VEC_; static constexpr bool KEEP = KEEP_; };
// 32 KC channels and 8 NT heads for a call; rows stay in registers up to 256 channels (fp32, 256 to 8 heads, [1,512,512,256]: forward 73
// us, read again for every use 126), with more than 16 heads up to 8 words a lane and row.
template <class T, class F>
void with_shape(const ProjArgs& a, F&& f) {
  const int vec = vector_of(a, (int)sizeof(T));
  if (vec < 8) {  // fewer shapes
    if (a.C <= 128 && a.H <= 8 && vec == 4) f(Shape<4, 1, true, 4>());
    else if (a.C <= 128 && a.H <= 8) f(Shape<4, 1, true, 1>());
    else if (a.C <= 128 && a.H <= 16 && vec == 4) f(Shape<4, 2, true, 4>());
    else if (a.C <= 128 && a.H <= 16) f(Shape<4, 2, true, 1>());
    else if (a.H <= 16) f(Shape<16, 2, false, 1>());
    else f(Shape<16, 8, false, 1>());
    return;
  }
  const auto heads = [&](auto kc) {
    constexpr int KC = decltype(kc)::value;
    constexpr bool keep = KC <= 8;
    if (a.H <= 8) f(Shape<KC, 1, keep, 8>());
    else if (a.H <= 16) f(Shape<KC, 2, keep, 8>());
    else f(Shape<KC, 8, KC * (int)sizeof(T) <= 8, 8>());
  };
  if (a.C <= 64) heads(std::integral_constant<int, 2>());
  else if (a.C <= 128) heads(std::integral_constant<int, 4>());
  else if (a.C <= 256) heads(std::integral_constant<int, 8>());
  else heads(std::integral_constant<int, 16>());
}
// Whether the backward is one kernel, which holds M of all channels and heads in registers beside the rows.
bool one_pass(const ProjArgs& a, int es) {
  if (es == 4 || vector_of(a, es) < 8) return a.C <= 128 && a.H <= 8;
  return (a.C <= 256 && a.H <= 8) || (a.C <= 128 && a.H <= 16);
}
template <class T, class F>
void with_one_pass_shape(const ProjArgs& a, F&& f) {
  const int vec = vector_of(a, (int)sizeof(T));
  if (vec == 4) {
    f(Shape<4, 1, true, 4>());
  } else if (vec == 1) {
    f(Shape<4, 1, true, 1>());
  } else if (a.H <= 8) {
    if (a.C <= 64) f(Shape<2, 1, true, 8>());
    else if (a.C <= 128) f(Shape<4, 1, true, 8>());
    else if constexpr (sizeof(T) == 2) f(Shape<8, 1, true, 8>());
  } else if constexpr (sizeof(T) == 2) {
    if (a.C <= 64) f(Shape<2, 2, true, 8>());
    else f(Shape<4, 2, true, 8>());
  }
}
// The same of the shapes that with_shape() gives: those whose backward is one kernel need none of the two.
template <class T>
constexpr bool one_pass_shape(int KC, int NT, int VEC) {
  return sizeof(T) == 4 || VEC < 8 ? KC <= 4 && NT == 1 : (KC <= 8 && NT == 1) || (KC <= 4 && NT <= 2);
}
// Blocks of 128 rows that run at once.
template <class K>
bool blocks_of(K kern, long long rows, int smem, unsigned* blocks) {
  int regs = 0;
  if (!kernel_ready(reinterpret_cast<const void*>(kern), smem, &regs)) return false;
  const int by_regs = 65536 / ((regs + 7) / 8 * 8 * 256), by_smem = 220 * 1024 / (smem + 2048);
  const long long want = (rows + 127) / 128, most = 148LL * (by_regs < by_smem ? by_regs : by_smem);
  *blocks = (unsigned)(want < most ? want : most);
  return true;
}
// Blocks that leave partial sums of H (C + 1) floats: as many as run at once.
int sum_blocks(const ProjArgs& a, int es) {
  const long long want = (rows_of(a) + 127) / 128, most = es == 2 && a.C <= 128 && a.H <= 8 && vector_of(a, es) == 8 ? 296 : 148;
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
  a.dz = nullptr;
  look_at_rows(&a);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t rc = cudaErrorUnknown;
  with_dtype(p->dtype, [&](auto e) {
    using T = decltype(e);
    with_shape<T>(a, [&](auto sh) {
      using Sh = decltype(sh);
      const auto kern = projection_fwd<T, Sh::KC, Sh::NT, Sh::KEEP, Sh::VEC>;
      const int smem = Sh::KC * Sh::NT * Pieces<T>::kG * 512;
      unsigned blocks;
      if (blocks_of(kern, rows, smem, &blocks)) rc = launch_dependent(kern, dim3(blocks), 256, (size_t)smem, st, a);
    });
    return 0;
  });
  return rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

size_t evoattn_pair_projection_bwd_workspace_bytes(const evoattn_pair_projection_params* p) {
  using namespace evo;
  if (validate(p) || !(p->dweight || p->dnorm_weight || p->dnorm_bias)) return 0;
  const ProjArgs a = args_of(p);
  return (one_pass(a, dtype_bytes(p->dtype)) ? 0 : stats_bytes(a)) + (size_t)sum_blocks(a, dtype_bytes(p->dtype)) * a.H * (a.C + 1) * sizeof(float);
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
  look_at_rows(&a);
  const bool sums = a.dw || a.dg || a.db, one = one_pass(a, dtype_bytes(p->dtype));
  a.blocks = sum_blocks(a, dtype_bytes(p->dtype));
  if (sums) {
    unsigned char* ws = static_cast<unsigned char*>(p->workspace);
    if (!one) a.stats = reinterpret_cast<float*>(ws);
    a.partial = reinterpret_cast<float*>(ws + (one ? 0 : stats_bytes(a)));
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t rc = cudaSuccess;
  if (rows > 0 && (a.dz || sums))
    with_dtype(p->dtype, [&](auto e) {
      using T = decltype(e);
      rc = cudaErrorUnknown;
      if (one) {
        with_one_pass_shape<T>(a, [&](auto sh) {
          using Sh = decltype(sh);
          const auto kern = projection_bwd<T, Sh::KC, Sh::NT, Sh::VEC>;
          const int pieces = 2 * Sh::KC * Sh::NT * Pieces<T>::kG * 512, left = 8 * Sh::NT * (32 * Sh::KC + 1) * (int)sizeof(float), smem = pieces > left ? pieces : left;
          if (kernel_ready(reinterpret_cast<const void*>(kern), smem, nullptr)) rc = launch_dependent(kern, dim3((unsigned)a.blocks), 256, (size_t)smem, st, a);
        });
        return 0;
      }
      with_shape<T>(a, [&](auto sh) {
        using Sh = decltype(sh);
        if constexpr (!one_pass_shape<T>(Sh::KC, Sh::NT, Sh::VEC)) {
          const auto kern = projection_dz<T, Sh::KC, Sh::NT, Sh::KEEP, Sh::VEC>;
          const int smem = (both_layouts<T>(Sh::KC, Sh::NT, Sh::KEEP) ? 2 : 1) * Sh::KC * Sh::NT * Pieces<T>::kG * 512;
          unsigned blocks;
          if (blocks_of(kern, rows, smem, &blocks)) rc = launch_dependent(kern, dim3(blocks), 256, (size_t)smem, st, a);
        }
      });
      if (rc == cudaSuccess && sums) {
        const dim3 grid((unsigned)a.blocks, (unsigned)((a.C + kSumChannels - 1) / kSumChannels), (unsigned)((a.H + kSumHeads - 1) / kSumHeads));
        const int vec = vector_of(a, (int)sizeof(T));
        rc = launch_dependent(vec == 8 ? projection_sums<T, 8> : vec == 4 ? projection_sums<T, 4> : projection_sums<T, 1>, grid, 256, 0, st, a);
      }
      return 0;
    });
  if (rc == cudaSuccess && sums) rc = launch_dependent(projection_weights, dim3((unsigned)((a.C + kWeightChannels - 1) / kWeightChannels)), 1024, 0, st, a);
  return rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

}  // extern "C"
