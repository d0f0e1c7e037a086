// Attention over packed sequences on CUDA cores, forward and backward: fp32, head dimensions that are not in eights or
// above 128, and tensors off 16 bytes.  Everything in fp32.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j - lse_i) over the keys j of i's sequence (causal: j <= i + nk - nq)
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i v_j - delta_i),  delta_i = do_i o_i,  dq_i = scale sum_j ds_ij k_j,
//   dk_j = scale sum_i ds_ij q_i
//
// Tiles of TILE queries by TILE keys, 256 threads as 16 x 16, each with TILE / 16 rows and as many columns of the scores
// and as many rows of every product.  Keys and queries of a thread are 16 apart, so that its rows of DP + 4 floats lie in
// other banks than its neighbours'.  The backward is two kernels, one that walks the queries of a key tile (all heads of
// the group in turn) and one that walks the keys of a query tile: the scores are formed twice, and no sum depends on the
// order in which blocks run; they run beside one another where there is room.
//
// Bound by FMA issue and shared-memory loads, where it is large (fp32, [8192] causal, 8 heads of 64: 2.6 ms forward, 26 TFLOP/s),
// and by the latency of a block's tiles, 2.5 us each, where it is small ([437 300 129], 4 heads of 64: 112 us forward and backward).
#include <math.h>

#include <type_traits>

#include "packed.cuh"

namespace evo {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

// TILE is 64, or 32 where that makes more blocks than an SM's worth of work each (and above D = 128, where four tiles of 64
// rows would not fit).
template <int DP, int TILE_>
struct GenericCfg {
  static constexpr int TILE = TILE_;
  static constexpr int NR = TILE / 16, NC = DP / 64, LD = DP + 4, LP = TILE + 4;
  static constexpr size_t bytes(int tiles, int scores) { return sizeof(float) * ((size_t)tiles * TILE * LD + (size_t)scores * TILE * LP + 2 * TILE); }
};

// Rows [from, n) of a tile on their way to shared memory as floats, zeros before, beyond n and beyond D: get() asks for all of them at once (one
// at a time they took 9 of a tile's 11 us), put() stores them.  VEC: 16 bytes at a time.
template <class T, int DP, int TILE, bool VEC>
struct Rows {
  static constexpr int LD = GenericCfg<DP, TILE>::LD, V = VEC ? kPer16<T> : 1, PER = DP / V, N = TILE * PER / kThreads;
  using Raw = typename std::conditional<VEC, uint4, T>::type;
  Raw raw[N];
  __device__ __forceinline__ void get(const void* src, long long stride, int n, int D, int from = 0) {
    const T* p = static_cast<const T*>(src);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = threadIdx.x + u * kThreads, r = i / PER, d = i % PER * V;
      raw[u] = Raw{};
      if (r >= from && r < n && d < D) raw[u] = *reinterpret_cast<const Raw*>(p + r * stride + d);
    }
  }
  __device__ __forceinline__ void put(float* dst) const {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = threadIdx.x + u * kThreads;
      float* to = dst + i / PER * LD + i % PER * V;
      if constexpr (VEC) {
        float f[V];
        unpack16<T>(raw[u], f);
#pragma unroll
        for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(to + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
      } else {
        *to = to_float(raw[u]);
      }
    }
  }
};
__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float dot4(float4 a, float4 b, float s) { return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, s)))); }

// s[r][c] = row (ty + 16 r) of x times row (tx + 16 c) of y.
template <class C, int DP>
__device__ __forceinline__ void products(const float* x, const float* y, int ty, int tx, float (&s)[C::NR][C::NR]) {
  constexpr int NR = C::NR, LD = C::LD;
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int c = 0; c < NR; ++c) s[r][c] = 0.f;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 u[NR], w[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) u[r] = ld4(x + (ty + 16 * r) * LD + d);
#pragma unroll
    for (int c = 0; c < NR; ++c) w[c] = ld4(y + (tx + 16 * c) * LD + d);
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int c = 0; c < NR; ++c) s[r][c] = dot4(u[r], w[c], s[r][c]);
  }
}
// acc[r][.] += sum_j p[ty + 16 r][j] * y[j][4 tx + 64 c ..].
template <class C>
__device__ __forceinline__ void accumulate(const float* p, const float* y, int ty, int tx, float4 (&acc)[C::NR][C::NC]) {
#pragma unroll 2
  for (int j = 0; j < C::TILE; j += 4) {
    float4 w[C::NR];
#pragma unroll
    for (int r = 0; r < C::NR; ++r) w[r] = ld4(p + (ty + 16 * r) * C::LP + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int c = 0; c < C::NC; ++c) {
        const float4 v = ld4(y + (j + e) * C::LD + 4 * tx + 64 * c);
#pragma unroll
        for (int r = 0; r < C::NR; ++r) {
          const float f = e == 0 ? w[r].x : e == 1 ? w[r].y : e == 2 ? w[r].z : w[r].w;
          acc[r][c].x = fmaf(f, v.x, acc[r][c].x); acc[r][c].y = fmaf(f, v.y, acc[r][c].y);
          acc[r][c].z = fmaf(f, v.z, acc[r][c].z); acc[r][c].w = fmaf(f, v.w, acc[r][c].w);
        }
      }
    }
  }
}
template <class T>
__device__ __forceinline__ void store_row(T* row, int tx, int c, float4 v, float by, int D) {
  const float f[4] = {v.x * by, v.y * by, v.z * by, v.w * by};
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (4 * tx + 64 * c + u < D) row[4 * tx + 64 * c + u] = from_float<T>(f[u]);
}
__device__ __forceinline__ float max16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <class T, int DP, int TILE, bool VEC>
__global__ void __launch_bounds__(kThreads) packed_generic_fwd_kernel(const PackedArgs a) {
  using C = GenericCfg<DP, TILE>;
  constexpr int NR = C::NR, NC = C::NC;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sK = sQ + TILE * C::LD, *sV = sK + TILE * C::LD, *sP = sV + TILE * C::LD;
  __shared__ int place[34];
  const int h = blockIdx.y, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  T* o = static_cast<T*>(a.o);
  if (h == 0) zero_outside(a.offsets, a.wide, a.B, a.Tq, a.o, (long long)a.H * a.D * sizeof(T), blockIdx.x, gridDim.x);
  auto count = [&](int b) { return query_span(a, b).n; };
  const Place at = locate(a.B, blockIdx.x, TILE, place, count);
  if (at.seq < 0) return;
  // Offsets that do not ascend may make sequences that overlap, and more tiles than there are blocks: then the last one zeroes the
  // head's rows, so that nothing comes back as memory was.
  if (blockIdx.x + 1 == gridDim.x && locate(a.B, (int)gridDim.x, TILE, place, count).seq >= 0) {
    for (long long i = threadIdx.x; i < (long long)a.Tq * a.D; i += kThreads) o[(i / a.D * a.H + h) * a.D + i % a.D] = from_float<T>(0.f);
    return;
  }
  const Span qs = query_span(a, at.seq), ks = key_span(a, at.seq);
  const int i0 = at.tile * TILE, rows = min(TILE, qs.n - i0), shift = ks.n - qs.n, hk = h / a.G;
  const int seen = keys_seen(a, qs.n, ks.n, i0, TILE);
  Rows<T, DP, TILE, VEC> x, y;
  x.get(static_cast<const T*>(a.q) + (long long)(qs.begin + i0) * a.sq[0] + (long long)h * a.sq[1], a.sq[0], rows, a.D);
  x.put(sQ);
  auto fetch = [&](int j0) {
    const long long row = ks.begin + j0;
    x.get(static_cast<const T*>(a.k) + row * a.sk[0] + (long long)hk * a.sk[1], a.sk[0], ks.n - j0, a.D);
    y.get(static_cast<const T*>(a.v) + row * a.sv[0] + (long long)hk * a.sv[1], a.sv[0], ks.n - j0, a.D);
  };
  if (seen > 0) fetch(0);
  const float c = a.scale * kLog2e;
  float m[NR], l[NR];
  float4 acc[NR][NC];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) acc[r][k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int j0 = 0; j0 < seen; j0 += TILE) {
    __syncthreads();
    x.put(sK);
    y.put(sV);
    __syncthreads();
    if (j0 + TILE < seen) fetch(j0 + TILE);  // (the next tile's rows are on their way under this one's arithmetic)
    float s[NR][NR];
    products<C, DP>(sQ, sK, ty, tx, s);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int last = a.causal ? min(ks.n - 1, i0 + ty + 16 * r + shift) : ks.n - 1;  // the last key of this row
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        s[r][k] = j0 + tx + 16 * k <= last ? s[r][k] * c : -INFINITY;
        mx = fmaxf(mx, s[r][k]);
      }
      const float up = fmaxf(m[r], max16(mx));
      const float from = up == -INFINITY ? 0.f : up;  // (a row that has seen no key: all exponentials are 0)
      const float alpha = exp2f(m[r] - from);
      m[r] = up;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        const float p = exp2f(s[r][k] - from);
        sum += p;
        sP[(ty + 16 * r) * C::LP + tx + 16 * k] = p;
      }
      l[r] = l[r] * alpha + sum16(sum);
#pragma unroll
      for (int k = 0; k < NC; ++k) { acc[r][k].x *= alpha; acc[r][k].y *= alpha; acc[r][k].z *= alpha; acc[r][k].w *= alpha; }
    }
    __syncthreads();
    accumulate<C>(sP, sV, ty, tx, acc);
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int i = ty + 16 * r;
    if (i >= rows) continue;
    const float inv = l[r] != 0.f ? 1.f / l[r] : 0.f;  // (0: no key; NaN where a score is infinite or NaN)
    T* out = o + ((long long)(qs.begin + i0 + i) * a.H + h) * a.D;
#pragma unroll
    for (int k = 0; k < NC; ++k) store_row(out, tx, k, acc[r][k], inv, a.D);
    if (a.o_rest) {
      T* rest = static_cast<T*>(a.o_rest) + (out - o);
      auto left = [&](float v) { return v * inv - to_float(from_float<T>(v * inv)); };
#pragma unroll
      for (int k = 0; k < NC; ++k) store_row(rest, tx, k, make_float4(left(acc[r][k].x), left(acc[r][k].y), left(acc[r][k].z), left(acc[r][k].w)), 1.f, a.D);
    }
    if (tx == 0 && a.lse) a.lse[(long long)h * a.lse_ld + qs.begin + i0 + i] = l[r] == 0.f ? -INFINITY : m[r] + log2f(l[r]);
  }
}

// p and ds of a tile, in place of the scores and of dO V^T.
template <int NR>
__device__ __forceinline__ void p_and_ds(const PackedArgs& a, float (&s)[NR][NR], float (&dp)[NR][NR], const float* lse, const float* delta, int i0, int j0, int nq, int nk, int ty, int tx) {
  const float c = a.scale * kLog2e;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int i = ty + 16 * r;
    const int last = i0 + i >= nq ? -1 : a.causal ? min(nk - 1, i0 + i + nk - nq) : nk - 1;
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const bool seen = j0 + tx + 16 * k <= last;
      s[r][k] = seen ? exp2f(s[r][k] * c - lse[i]) : 0.f;
      dp[r][k] = seen ? s[r][k] * (dp[r][k] - delta[i]) : 0.f;
    }
  }
}
template <int TILE>
__device__ __forceinline__ void load_statistics(const PackedArgs& a, float* lse, float* delta, int h, int row, int rows) {
  for (int i = threadIdx.x; i < TILE; i += kThreads) {
    lse[i] = i < rows ? a.lse[(long long)h * a.lse_ld + row + i] : 0.f;
    delta[i] = i < rows ? a.delta[(long long)h * a.lse_ld + row + i] : 0.f;
  }
}

template <class T, int DP, int TILE, bool VEC>
__global__ void __launch_bounds__(kThreads) packed_generic_dq_kernel(const PackedArgs a, const int follows) {
  using C = GenericCfg<DP, TILE>;
  constexpr int NR = C::NR, NC = C::NC;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sO = sQ + TILE * C::LD, *sK = sO + TILE * C::LD, *sV = sK + TILE * C::LD, *sS = sV + TILE * C::LD;
  float *lse = sS + TILE * C::LP, *delta = lse + TILE;
  __shared__ int place[34];
  const int h = blockIdx.y, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const bool overlap = __ldcg(a.overlap) != 0;
  if (h == 0) zero_outside(a.offsets, a.wide, a.B, a.Tq, a.dq, (long long)a.H * a.D * sizeof(T), blockIdx.x, gridDim.x, overlap);
  const Place at = overlap ? Place{-1, 0} : locate(a.B, blockIdx.x, TILE, place, [&](int b) { return query_span(a, b).n; });
  if (at.seq < 0) {
    if (follows) ptx::grid_dependency_wait();
    return;
  }
  const Span qs = query_span(a, at.seq), ks = key_span(a, at.seq);
  const int i0 = at.tile * TILE, rows = min(TILE, qs.n - i0), hk = h / a.G, seen = keys_seen(a, qs.n, ks.n, i0, TILE);
  const long long row = qs.begin + i0;
  Rows<T, DP, TILE, VEC> x, y;
  x.get(static_cast<const T*>(a.q) + row * a.sq[0] + (long long)h * a.sq[1], a.sq[0], rows, a.D);
  y.get(static_cast<const T*>(a.d_o) + row * a.sdo[0] + (long long)h * a.sdo[1], a.sdo[0], rows, a.D);
  x.put(sQ);
  y.put(sO);
  auto fetch = [&](int j0) {
    const long long key = ks.begin + j0;
    x.get(static_cast<const T*>(a.k) + key * a.sk[0] + (long long)hk * a.sk[1], a.sk[0], ks.n - j0, a.D);
    y.get(static_cast<const T*>(a.v) + key * a.sv[0] + (long long)hk * a.sv[1], a.sv[0], ks.n - j0, a.D);
  };
  if (seen > 0) fetch(0);
  load_statistics<TILE>(a, lse, delta, h, (int)row, rows);
  float4 acc[NR][NC];
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int k = 0; k < NC; ++k) acc[r][k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j0 = 0; j0 < seen; j0 += TILE) {
    __syncthreads();
    x.put(sK);
    y.put(sV);
    __syncthreads();
    if (j0 + TILE < seen) fetch(j0 + TILE);
    float s[NR][NR], dp[NR][NR];
    products<C, DP>(sQ, sK, ty, tx, s);
    products<C, DP>(sO, sV, ty, tx, dp);
    p_and_ds(a, s, dp, lse, delta, i0, j0, qs.n, ks.n, ty, tx);
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int k = 0; k < NR; ++k) sS[(ty + 16 * r) * C::LP + tx + 16 * k] = dp[r][k];
    __syncthreads();
    accumulate<C>(sS, sK, ty, tx, acc);
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (ty + 16 * r >= rows) continue;
    T* out = static_cast<T*>(a.dq) + ((row + ty + 16 * r) * a.H + h) * a.D;
#pragma unroll
    for (int k = 0; k < NC; ++k) store_row(out, tx, k, acc[r][k], a.scale, a.D);
  }
  if (follows) ptx::grid_dependency_wait();
}

template <class T, int DP, int TILE, bool VEC>
__global__ void __launch_bounds__(kThreads) packed_generic_dkv_kernel(const PackedArgs a) {
  using C = GenericCfg<DP, TILE>;
  constexpr int NR = C::NR, NC = C::NC;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sO = sQ + TILE * C::LD, *sK = sO + TILE * C::LD, *sV = sK + TILE * C::LD, *sP = sV + TILE * C::LD, *sS = sP + TILE * C::LP;
  float *lse = sS + TILE * C::LP, *delta = lse + TILE;
  __shared__ int place[34];
  ptx::grid_launch_dependents();
  const int hk = blockIdx.y, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const long long row_bytes = (long long)a.Hk * a.D * sizeof(T);
  const bool overlap = __ldcg(a.overlap) || __ldcg(a.overlap + 1);
  if (hk == 0) {
    zero_outside(a.key_offsets, a.wide, a.B, a.Tk, a.dk, row_bytes, blockIdx.x, gridDim.x, overlap);
    zero_outside(a.key_offsets, a.wide, a.B, a.Tk, a.dv, row_bytes, blockIdx.x, gridDim.x, overlap);
  }
  if (overlap) return;
  const Place at = locate(a.B, blockIdx.x, TILE, place, [&](int b) { return key_span(a, b).n; });
  if (at.seq < 0) return;
  const Span qs = query_span(a, at.seq), ks = key_span(a, at.seq);
  const int j0 = at.tile * TILE, keys = min(TILE, ks.n - j0);
  const long long key = ks.begin + j0;
  Rows<T, DP, TILE, VEC> x, y;
  x.get(static_cast<const T*>(a.k) + key * a.sk[0] + (long long)hk * a.sk[1], a.sk[0], keys, a.D);
  y.get(static_cast<const T*>(a.v) + key * a.sv[0] + (long long)hk * a.sv[1], a.sv[0], keys, a.D);
  x.put(sK);
  y.put(sV);
  float4 dk[NR][NC], dv[NR][NC];
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int k = 0; k < NC; ++k) dk[r][k] = dv[r][k] = make_float4(0.f, 0.f, 0.f, 0.f);
  // the first query that sees a key of this tile
  const int first = a.causal ? max(0, j0 - (ks.n - qs.n)) : 0;
  const int i_first = first / TILE * TILE, blind = a.causal ? qs.n - ks.n : 0;  // (the queries before `blind` see no key: whatever they hold)
  auto fetch = [&](int h, int i0) {
    const long long row = qs.begin + i0;
    const int rows = min(TILE, qs.n - i0);
    x.get(static_cast<const T*>(a.q) + row * a.sq[0] + (long long)h * a.sq[1], a.sq[0], rows, a.D, blind - i0);
    y.get(static_cast<const T*>(a.d_o) + row * a.sdo[0] + (long long)h * a.sdo[1], a.sdo[0], rows, a.D, blind - i0);
  };
  if (i_first < qs.n) fetch(hk * a.G, i_first);
  for (int g = 0; g < a.G; ++g) {
    const int h = hk * a.G + g;
    for (int i0 = i_first; i0 < qs.n; i0 += TILE) {
      __syncthreads();
      const long long row = qs.begin + i0;
      const int rows = min(TILE, qs.n - i0);
      x.put(sQ);
      y.put(sO);
      load_statistics<TILE>(a, lse, delta, h, (int)row, rows);
      __syncthreads();
      if (i0 + TILE < qs.n) fetch(h, i0 + TILE);
      else if (g + 1 < a.G) fetch(h + 1, i_first);
      float s[NR][NR], dp[NR][NR];
      products<C, DP>(sQ, sK, ty, tx, s);
      products<C, DP>(sO, sV, ty, tx, dp);
      p_and_ds(a, s, dp, lse, delta, i0, j0, qs.n, ks.n, ty, tx);
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int k = 0; k < NR; ++k) {
          sP[(tx + 16 * k) * C::LP + ty + 16 * r] = s[r][k];  // (by keys)
          sS[(tx + 16 * k) * C::LP + ty + 16 * r] = dp[r][k];
        }
      __syncthreads();
      accumulate<C>(sP, sO, ty, tx, dv);
      accumulate<C>(sS, sQ, ty, tx, dk);
    }
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (ty + 16 * r >= keys) continue;
    const long long at_row = ((key + ty + 16 * r) * a.Hk + hk) * a.D;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      store_row(static_cast<T*>(a.dk) + at_row, tx, k, dk[r][k], a.scale, a.D);
      store_row(static_cast<T*>(a.dv) + at_row, tx, k, dv[r][k], 1.f, a.D);
    }
  }
}

template <class K, class... X>
int run(K kern, const PackedArgs& a, long long rows, int tile, int heads, size_t smem, cudaStream_t st, int* launches, bool early, X... x) {
  if (!kernel_ready(reinterpret_cast<const void*>(kern), (int)smem, nullptr)) return EVOATTN_ERR_CUDA;
  const dim3 grid((unsigned)(rows / tile + a.B), (unsigned)heads);
  if (early) launch_dependent(kern, grid, kThreads, smem, st, a, x...);
  else kern<<<grid, kThreads, smem, st>>>(a, x...);
  *launches += 1;
  return cudaGetLastError() == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}
template <class T, int DP, int TILE, bool VEC>
int both(bool back, const PackedArgs& a, cudaStream_t st, int* launches) {
  using C = GenericCfg<DP, TILE>;
  if (!back) return run(packed_generic_fwd_kernel<T, DP, TILE, VEC>, a, a.Tq, TILE, a.H, C::bytes(3, 1), st, launches, false);
  if (a.dk) {
    const int rc = run(packed_generic_dkv_kernel<T, DP, TILE, VEC>, a, a.Tk, TILE, a.Hk, C::bytes(4, 2), st, launches, false);
    if (rc) return rc;
  }
  // (dQ needs nothing of the kernel before it, which began when the statistics were complete: it runs beside it, and waits for
  // it at its end)
  return a.dq ? run(packed_generic_dq_kernel<T, DP, TILE, VEC>, a, a.Tq, TILE, a.H, C::bytes(4, 1), st, launches, a.dk != nullptr, (int)(a.dk != nullptr)) : EVOATTN_OK;
}
template <class T>
bool vectors(const PackedArgs& a, bool bwd) {
  constexpr int V = kPer16<T>;
  const auto ok = [](const void* p, const long long* st) { return ((uintptr_t)p & 15) == 0 && st[0] % V == 0 && st[1] % V == 0; };
  return a.D % V == 0 && ok(a.q, a.sq) && ok(a.k, a.sk) && ok(a.v, a.sv) && (!bwd || ok(a.d_o, a.sdo));
}
template <class T, int DP>
int launch(bool back, const PackedArgs& a, cudaStream_t st, int* launches) {
  const bool vec = vectors<T>(a, back);
  if constexpr (DP <= 128) {
    const long long blocks = (a.Tq / 64 + a.B) * (long long)(back ? a.Hk : a.H);
    if (blocks > 3LL * sm_count()) return vec ? both<T, DP, 64, true>(back, a, st, launches) : both<T, DP, 64, false>(back, a, st, launches);
  }
  return vec ? both<T, DP, 32, true>(back, a, st, launches) : both<T, DP, 32, false>(back, a, st, launches);
}
int launch_any(int dtype, bool back, const PackedArgs& a, cudaStream_t st, int* launches) {
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return a.D <= 64 ? launch<T, 64>(back, a, st, launches) : a.D <= 128 ? launch<T, 128>(back, a, st, launches) : launch<T, 256>(back, a, st, launches);
  });
}

}  // namespace

int launch_packed_generic_fwd(int dtype, const PackedArgs& a, cudaStream_t st, int* launches) { return launch_any(dtype, false, a, st, launches); }
int launch_packed_generic_bwd(int dtype, const PackedArgs& a, cudaStream_t st, int* launches) { return launch_any(dtype, true, a, st, launches); }

}  // namespace evo
