// Layer norm over the last axis, forward and backward.
//
//   h = (x - mean) r,  r = (var + eps)^-1/2,  y = h w + b
//   g = dy w,  dx = r (g - mean(g) - h mean(g h)),  dw = sum over rows of dy h,  db = sum over rows of dy
//
// The variance is taken about the mean (two passes over a row), so rows far from zero lose nothing.  Bound by memory: two
// passes over the rows forward, three backward.  [2,512,768,256] bf16, transposed rows: forward 145 us (5.5 TB/s), backward
// 219 (5.5), on a card whose copies run at 6.5.
#include <type_traits>

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
  // rows below 2^31: the same division without dividing
  FastDiv by_n1, by_n2;
  int one_axis;    // n0 = n1 = 1
};

__device__ __forceinline__ long long row_offset(const NormArgs& a, const Str3& s, long long n) {
  const long long q = n / a.n2, k = n - q * a.n2, i = q / a.n1, j = q - i * a.n1;
  return i * s.a + j * s.b + k * s.c;
}

__device__ __forceinline__ long long row_offset32(const NormArgs& a, const Str3& s, uint32_t n) {
  if (a.one_axis) return (long long)n * s.c;
  const uint32_t q = a.by_n2.div(n), k = n - q * (uint32_t)a.n2, i = a.by_n1.div(q), j = q - i * (uint32_t)a.n1;
  return i * s.a + j * s.b + k * s.c;
}

// ---------------------------------------------------------------- rows in registers
//
// A team of G lanes (G = 0: the whole block) takes a row: K pieces of V values a lane, piece k of lane l being values
// (k G + l) V ..., so that a team reads G pieces next to each other.  V is 16 bytes, or one value where C, strides or
// addresses are not whole pieces.  Few lanes and more values a lane make the sums over a row cheap: eight lanes with 16
// values of 128 take three exchanges for four rows of a warp.  The next D rows are on their way while one is used.
template <class T, int V, int K>
struct Pieces {
  using Raw = typename std::conditional<V == 1, T, uint4>::type;
  Raw raw[K];
  __device__ __forceinline__ void load(const T* row, int lane, int lanes, int C) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      if constexpr (V == 1) raw[k] = c < C ? row[c] : from_float<T>(0.f);
      else raw[k] = c < C ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void floats(float (&v)[K * V]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if constexpr (V == 1) v[k] = to_float<T>(raw[k]);
      else unpack16<T>(raw[k], v + k * V);
    }
  }
  static __device__ __forceinline__ void store(T* row, const float (&v)[K * V], int lane, int lanes, int C) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      if (c >= C) continue;
      if constexpr (V == 1) row[c] = from_float<T>(v[k]);
      else *reinterpret_cast<uint4*>(row + c) = pack16<T>(v + k * V);
    }
  }
};

constexpr int kMostWarps = 16;  // of a block that is one team

// Sums over a team, in all of its lanes.  Between warps they go through one of two buffers in turn: a buffer is written
// again only after everyone has passed the barrier of the sum in between, and so has read it.
template <int G, int N>
struct TeamSum {
  float (*sm)[N][kMostWarps];
  int turn = 0;
  __device__ __forceinline__ explicit TeamSum(float (*buffers)[N][kMostWarps]) : sm(buffers) {}
  template <int M>
  __device__ __forceinline__ void operator()(float (&v)[M]) {
#pragma unroll
    for (int o = (G ? G : 32) / 2; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < M; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (G == 0) {
      const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
      if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int i = 0; i < M; ++i) sm[turn][i][warp] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < M; ++i) {
        v[i] = 0.f;
        for (int w = 0; w < warps; ++w) v[i] += sm[turn][i][w];
      }
      turn ^= 1;
    }
  }
};

// The team of a thread and the rows it takes: first, first + step, ... ; teams of a warp go on together.
template <int G>
struct Team {
  int lane, lanes;
  uint32_t first, step, offset;  // offset: of this team among those that go on together
  __device__ __forceinline__ Team() {
    if constexpr (G == 0) {
      lane = threadIdx.x; lanes = blockDim.x;
      first = blockIdx.x; step = gridDim.x; offset = 0;
    } else {
      const uint32_t per_warp = 32 / G, warps = blockDim.x >> 5;
      lane = threadIdx.x & (G - 1); lanes = G;
      first = (blockIdx.x * warps + (threadIdx.x >> 5)) * per_warp;
      step = gridDim.x * warps * per_warp;
      offset = (threadIdx.x & 31) / G;
    }
  }
};

template <int V, int K>
__device__ __forceinline__ void load_weights(const void* p, int dtype, float other, int lane, int lanes, int C, float (&v)[K * V]) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int c = (k * lanes + lane) * V + u;
      v[k * V + u] = c < C ? (p ? load_any(p, dtype, c) : other) : 0.f;
    }
}

// Threads of a block: 256 in teams, or one team of up to 512.
template <int G, int K, int V> constexpr int kThreads = G ? 256 : 512;

template <class T, int V, int G, int K, int D>
__global__ void __launch_bounds__(kThreads<G, K, V>) norm_fwd_rows(NormArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  __shared__ float sm[2][1][kMostWarps];
  TeamSum<G, 1> sum(sm);
  const Team<G> t;
  const uint32_t rows = (uint32_t)a.rows;
  const float by_C = 1.f / a.C;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  Pieces<T, V, K> next[D];
  const auto fetch = [&](Pieces<T, V, K>& to, uint32_t n) {
    if (n < rows) to.load(x + row_offset32(a, a.sx, n), t.lane, t.lanes, a.C);
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(next[d], t.first + t.offset + d * t.step);
  float w[K * V], b[K * V];
  load_weights<V, K>(a.w, a.w_dtype, 1.f, t.lane, t.lanes, a.C, w);
  load_weights<V, K>(a.b, a.b_dtype, 0.f, t.lane, t.lanes, a.C, b);
  bool on[K];
#pragma unroll
  for (int k = 0; k < K; ++k) on[k] = (k * t.lanes + t.lane) * V < a.C;
  for (uint32_t base = t.first; base < rows; base += D * t.step) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (d && base + d * t.step >= rows) break;
      const uint32_t n = base + t.offset + d * t.step;
      float v[K * V];
      next[d].floats(v);
      fetch(next[d], n + D * t.step);
      float s[1] = {0.f};
#pragma unroll
      for (int e = 0; e < K * V; ++e) s[0] += v[e];
      sum(s);
      const float mean = s[0] * by_C;
      s[0] = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (on[k]) {
#pragma unroll
          for (int e = k * V; e < k * V + V; ++e) {
            v[e] -= mean;
            s[0] = fmaf(v[e], v[e], s[0]);
          }
        }
      sum(s);
      const float r = rsqrtf(s[0] * by_C + a.eps);
      if (n >= rows) continue;
      if (a.stats && t.lane == 0) reinterpret_cast<float2*>(a.stats)[n] = make_float2(mean, r);
#pragma unroll
      for (int e = 0; e < K * V; ++e) v[e] = fmaf(v[e] * r, w[e], b[e]);
      Pieces<T, V, K>::store(y + (long long)n * a.C, v, t.lane, t.lanes, a.C);
    }
  }
}

// dx of the rows, and the sums over them of dy h and dy: in registers over a team's rows, then over the block's teams in order
// (no atomics: the same bits every time).
template <class T, int V, int G, int K, int D>
__global__ void __launch_bounds__(kThreads<G, K, V>) norm_bwd_rows(NormArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int kSlots = G ? 256 / (G ? G : 1) : 1;
  __shared__ float sm[2][2][kMostWarps];
  __shared__ float sm_cols[G ? 256 * K * V : 1];
  TeamSum<G, 2> sum(sm);
  const Team<G> t;
  const uint32_t rows = (uint32_t)a.rows;
  const float by_C = 1.f / a.C;
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  T* dx = static_cast<T*>(a.dx);
  Pieces<T, V, K> next_x[D], next_d[D];
  float2 next_st[D];
  const auto fetch = [&](int d, uint32_t n) {
    if (n >= rows) return;
    next_x[d].load(x + row_offset32(a, a.sx, n), t.lane, t.lanes, a.C);
    next_d[d].load(dy + row_offset32(a, a.sdy, n), t.lane, t.lanes, a.C);
    next_st[d] = reinterpret_cast<const float2*>(a.stats)[n];
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(d, t.first + t.offset + d * t.step);
  float w[K * V], dw[K * V], db[K * V];
  load_weights<V, K>(a.w, a.w_dtype, 1.f, t.lane, t.lanes, a.C, w);
#pragma unroll
  for (int e = 0; e < K * V; ++e) dw[e] = db[e] = 0.f;
  for (uint32_t base = t.first; base < rows; base += D * t.step) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (d && base + d * t.step >= rows) break;
      const uint32_t n = base + t.offset + d * t.step;
      float h[K * V], g[K * V];
      next_x[d].floats(h);
      next_d[d].floats(g);
      const float2 st = next_st[d];
      fetch(d, n + D * t.step);
      const bool on = n < rows;
      float s[2] = {0.f, 0.f};
      if (on) {
#pragma unroll
        for (int e = 0; e < K * V; ++e) {
          h[e] = (h[e] - st.x) * st.y;
          dw[e] = fmaf(g[e], h[e], dw[e]);
          db[e] += g[e];
          g[e] *= w[e];
          s[0] += g[e];
          s[1] = fmaf(g[e], h[e], s[1]);
        }
      }
      if (!dx) continue;
      sum(s);
      if (!on) continue;
      const float m1 = s[0] * by_C, m2 = s[1] * by_C;
#pragma unroll
      for (int e = 0; e < K * V; ++e) g[e] = st.y * (g[e] - m1 - h[e] * m2);
      Pieces<T, V, K>::store(dx + (long long)n * a.C, g, t.lane, t.lanes, a.C);
    }
  }
  if (!a.partial) return;
  float* out = a.partial + (long long)blockIdx.x * 2 * a.C;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float(&v)[K * V] = which ? db : dw;
    if constexpr (G == 0) {
#pragma unroll
      for (int e = 0; e < K * V; ++e) {
        const int c = (e / V * t.lanes + t.lane) * V + e % V;
        if (c < a.C) out[which * a.C + c] = v[e];
      }
    } else {
      constexpr int kCols = G * K * V;
      if (which) __syncthreads();
#pragma unroll
      for (int e = 0; e < K * V; ++e) sm_cols[threadIdx.x / G * kCols + (e / V * G + t.lane) * V + e % V] = v[e];
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += 256) {
        float s = 0.f;
#pragma unroll 8
        for (int i = 0; i < kSlots; ++i) s += sm_cols[i * kCols + c];
        out[which * a.C + c] = s;
      }
    }
  }
}

// ---------------------------------------------------------------- any row

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

// The partial sums of all blocks, added in order: 32 columns a block, 32 shares of the partial sums.
__global__ void __launch_bounds__(1024) norm_sum_partials(NormArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  __shared__ float sm[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, which = blockIdx.y;
  float s = 0.f;
  if (c < a.C) {
#pragma unroll 10
    for (int k = part; k < a.blocks; k += 32) s += a.partial[((long long)k * 2 + which) * a.C + c];
  }
  sm[part][lane] = s;
  __syncthreads();
  s = warp_sum(sm[lane][part]);  // (a warp a column)
  const int out = blockIdx.x * 32 + part;
  if (lane == 0 && out < a.C) {
    if (which == 0 && a.dw) store_any(a.dw, a.w_dtype, out, s);
    if (which == 1 && a.db) store_any(a.db, a.b_dtype, out, s);
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
  a.one_axis = p->n[0] == 1 && p->n[1] == 1;
  if (a.rows > 0 && a.rows < (1LL << 31)) {
    a.by_n1 = FastDiv((uint32_t)a.n1);
    a.by_n2 = FastDiv((uint32_t)a.n2);
  }
  return a;
}

bool whole_pieces(const void* p, const Str3& s, int es) {
  return ((uintptr_t)p & 15) == 0 && s.a * es % 16 == 0 && s.b * es % 16 == 0 && s.c * es % 16 == 0;
}
bool whole_pieces(const NormArgs& a, int es, bool backward) {
  if ((long long)a.C * es % 16 || !whole_pieces(a.x, a.sx, es)) return false;
  if (!backward) return ((uintptr_t)a.y & 15) == 0;
  return whole_pieces(a.dy, a.sdy, es) && ((uintptr_t)a.dx & 15) == 0;
}

// Which form takes rows of C values; false: the kernels for any row.  What counts is some 32 KB on their way an SM.
// Forward, 16-bit: eight values a lane and four rows on the way (64 M values of rows of 256: 53 us; sixteen values and one row
// 64); fp32: one row (91 us; four rows 107: registers).  Backward, 16-bit: sixteen values (75 us; eight, at as many
// blocks, 106); fp32: eight (128 us).  Rows of 513 .. 1024: 32 values rather than two barriers a row (1024 bf16, forward 62 us;
// a block of 16 values a lane 76).  Beyond, a block a row (2048 bf16: 74 and 93 us); above 8192 its registers spill.
template <int V_, int G_, int K_, int D_> struct Form { static constexpr int V = V_, G = G_, K = K_, D = D_; };
template <class T, class F>
bool with_fwd_form(long long rows, int C, bool pieces, F&& f) {
  if (rows >= (1LL << 31)) return false;
  if (pieces) {
    constexpr int P = kPer16<T>, K = 8 / P;
    constexpr int D8 = sizeof(T) == 2 ? 4 : 1, D16 = sizeof(T) == 2 ? 2 : 1;
    if (C <= 32) f(Form<P, 4, K, D8>());
    else if (C <= 64) f(Form<P, 8, K, D8>());
    else if (C <= 128) f(Form<P, 16, K, D8>());
    else if (C <= 256) f(Form<P, 32, K, D8>());
    else if (C <= 512) f(Form<P, 32, 2 * K, D16>());
    else if (C <= 1024) f(Form<P, 32, 4 * K, 1>());
    else if (C <= 8192) f(Form<P, 0, 2 * K, D16>());
    else return false;
  } else {
    if (C <= 16) f(Form<1, 8, 2, 1>());
    else if (C <= 64) f(Form<1, 8, 8, 1>());
    else if (C <= 256) f(Form<1, 32, 8, 1>());
    else if (C <= 512) f(Form<1, 32, 16, 1>());
    else if (C <= 1024) f(Form<1, 32, 32, 1>());
    else if (C <= 8192) f(Form<1, 0, 16, 1>());
    else return false;
  }
  return true;
}
template <class T, class F>
bool with_bwd_form(long long rows, int C, bool pieces, F&& f) {
  if (rows >= (1LL << 31)) return false;
  if (pieces) {
    constexpr int P = kPer16<T>, K = 8 / P;
    if (sizeof(T) == 2) {
      if (C <= 64) f(Form<P, 4, 2 * K, 1>());
      else if (C <= 128) f(Form<P, 8, 2 * K, 1>());
      else if (C <= 256) f(Form<P, 16, 2 * K, 1>());
      else if (C <= 512) f(Form<P, 32, 2 * K, 1>());
      else if (C <= 1024) f(Form<P, 32, 4 * K, 1>());
      else if (C <= 8192) f(Form<P, 0, 2 * K, 1>());
      else return false;
    } else {
      if (C <= 32) f(Form<P, 4, K, 1>());
      else if (C <= 64) f(Form<P, 8, K, 1>());
      else if (C <= 128) f(Form<P, 16, K, 1>());
      else if (C <= 256) f(Form<P, 32, K, 1>());
      else if (C <= 512) f(Form<P, 32, 2 * K, 1>());
      else if (C <= 1024) f(Form<P, 32, 4 * K, 1>());
      else if (C <= 8192) f(Form<P, 0, 2 * K, 1>());
      else return false;
    }
  } else {
    if (C <= 16) f(Form<1, 8, 2, 1>());
    else if (C <= 64) f(Form<1, 8, 8, 1>());
    else if (C <= 256) f(Form<1, 32, 8, 1>());
    else if (C <= 512) f(Form<1, 32, 16, 1>());
    else if (C <= 1024) f(Form<1, 32, 32, 1>());
    else if (C <= 8192) f(Form<1, 0, 16, 1>());
    else return false;
  }
  return true;
}
// Blocks and threads of a launch, as many blocks as there are rows for.
template <class Fm>
void shape_of(const NormArgs& a, int* threads, long long* blocks) {
  *threads = Fm::G ? 256 : (int)(((a.C + Fm::V * Fm::K - 1) / (Fm::V * Fm::K) + 31) / 32 * 32);
  const int rows_at_once = Fm::G ? 256 / (Fm::G ? Fm::G : 1) : 1;
  *blocks = (a.rows + rows_at_once - 1) / rows_at_once;
}
// Blocks of the backward: as many as run at once (by the registers of the form), each leaving a partial sum of 2 C floats.
template <class Fm>
long long bwd_blocks(long long wanted, int threads) {
  const int at_once = Fm::K * Fm::V <= 8 ? 768 : Fm::K * Fm::V <= 16 ? 512 : 256;
  const long long most = 148LL * (threads >= at_once ? 1 : at_once / threads);
  return wanted < most ? wanted : most;
}

unsigned row_blocks(long long rows) { return (unsigned)(rows < (1LL << 30) ? rows : (1LL << 30)); }

// What a backward call launches: the form's blocks, or those of the kernels for any row.
int plan_bwd(const NormArgs& a, int dtype, bool pieces) {
  int blocks = 0;
  with_dtype(dtype, [&](auto e) {
    using T = decltype(e);
    const bool ok = with_bwd_form<T>(a.rows, a.C, pieces, [&](auto fm) {
      int threads;
      long long n;
      shape_of<decltype(fm)>(a, &threads, &n);
      blocks = (int)bwd_blocks<decltype(fm)>(n, threads);
    });
    if (!ok) blocks = row_shares(a.rows);
    return 0;
  });
  return blocks;
}

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
    cudaError_t rc = cudaSuccess;
    const bool ok = with_fwd_form<T>(a.rows, a.C, whole_pieces(a, (int)sizeof(T), false), [&](auto fm) {
      using Fm = decltype(fm);
      int threads;
      long long blocks;
      shape_of<Fm>(a, &threads, &blocks);
      const long long most = 148LL * (2048 / threads);
      rc = launch_dependent(norm_fwd_rows<T, Fm::V, Fm::G, Fm::K, Fm::D>, dim3((unsigned)(blocks < most ? blocks : most)), threads, 0, st, a);
    });
    if (!ok) rc = launch_dependent(norm_fwd_any<T>, dim3(row_blocks(a.rows)), 256, 0, st, a);
    return rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
  });
}

size_t evoattn_layer_norm_bwd_workspace_bytes(const evoattn_layer_norm_params* p) {
  using namespace evo;
  if (validate(p) || !(p->dweight || p->dbias)) return 0;
  const NormArgs a = args_of(p);
  const int blocks = plan_bwd(a, p->dtype, whole_pieces(a, dtype_bytes(p->dtype), true));
  return (size_t)blocks * 2 * a.C * sizeof(float);
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
  if (columns) a.partial = static_cast<float*>(p->workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t rc = cudaSuccess;
  const bool pieces = whole_pieces(a, dtype_bytes(p->dtype), true);
  a.blocks = plan_bwd(a, p->dtype, pieces);
  const unsigned strips = (unsigned)((a.C + 31) / 32);
  if (a.rows > 0 && (a.dx || columns))
    with_dtype(p->dtype, [&](auto e) {
      using T = decltype(e);
      const bool ok = with_bwd_form<T>(a.rows, a.C, pieces, [&](auto fm) {
        using Fm = decltype(fm);
        int threads;
        long long blocks;
        shape_of<Fm>(a, &threads, &blocks);
        rc = launch_dependent(norm_bwd_rows<T, Fm::V, Fm::G, Fm::K, Fm::D>, dim3((unsigned)a.blocks), threads, 0, st, a);
      });
      if (ok) return 0;
      if (a.dx) rc = launch_dependent(norm_dx_any<T>, dim3(row_blocks(a.rows)), 256, 0, st, a);
      if (rc == cudaSuccess && columns) rc = launch_dependent(norm_columns_any<T>, dim3(strips, (unsigned)a.blocks), 256, 0, st, a);
      return 0;
    });
  if (rc == cudaSuccess && columns) rc = launch_dependent(norm_sum_partials, dim3(strips, 2), 1024, 0, st, a);
  return rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

}  // extern "C"
