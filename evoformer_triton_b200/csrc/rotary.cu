// Rotary positions: pairs (a, b) of a head's values turned by angle = position * frequency of the pair,
//   (a, b) -> amplitude (a cos - b sin, a sin + b cos),
// over q and k in one launch; the gradient is the same with the angle's sign changed.  "half": pair i is (x_i, x_{i+n}) of
// the 2 n rotated values, else (x_{2i}, x_{2i+1}).  Values behind them are copied.
//
// Angles: a position of 10^6 times a frequency of 1 rounded to fp32 is off by 0.03 of a radian.  Here turns = position *
// (frequency / 2 pi) are formed in fp64 (off by 2^-53 of them), whole turns are taken off there, and sine and cosine are of
// the fraction, which fp32 holds to 2^-26 of a turn.
//
// Bound by memory.  A block takes a strip of tokens: their sines and cosines once, into shared memory; then a thread keeps one
// piece of a head (16 bytes, or two of them that make pairs), with its sines and cosines in registers, and walks heads.
#include "inputs.cuh"

namespace evo {
namespace {

struct RotaryArgs {
  const void* x[2];     // q, k (or null)
  void* y[2];
  long long sx[2][4];   // element strides of the three token axes and the head
  int heads[2];
  const void* positions;
  long long sp[3];
  const void* frequencies;
  int wide, f64, half, D, n;  // n = pairs
  float amplitude, sign;
  long long tokens;
  FastDiv inner, middle;      // tokens -> three axes
};

// Two heads' loads at once a thread and some five heads a thread, four blocks an SM.  16 384 tokens of 40 heads of 128 bf16
// values take 58 us (5.7 TB/s) so, 61 with one head at once, 63 with four (and two blocks), 61 with ten heads a thread.
// Before, a thread took whatever pieces came, with the index arithmetic and the sines and cosines read again for each: 64.
constexpr int kThreads = 256, kAtOnce = 2, kHeads = 5;
constexpr int kMinBlocks = 6, kMostTokens = 16;  // blocks that every SM gets before they grow, up to this many tokens

// 16 bytes of values, or one.
template <class T, int V>
struct Piece {
  using Raw = uint4;
  static __device__ __forceinline__ void get(const uint4& r, float* f) { unpack16<T>(r, f); }
  static __device__ __forceinline__ uint4 put(const float* f) { return pack16<T>(f); }
};
template <class T>
struct Piece<T, 1> {
  using Raw = T;
  static __device__ __forceinline__ void get(const T& r, float* f) { *f = to_float(r); }
  static __device__ __forceinline__ T put(const float* f) { return from_float<T>(*f); }
};

struct Shape {
  FastDiv head, lanes, pairs;  // pieces of a head; threads that share a token's heads; pairs of a token
  int per, strip, side;        // pieces of a head that are turned; tokens of a block, and of a pass over its threads
};

// A piece is V values of the turned ones (half: two of them, n apart) or of the others.
template <class T, int V, bool HALF>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const RotaryArgs a, const Shape g) {
  extern __shared__ __align__(16) float2 turn[];  // [strip][n]: cos and sin, times the amplitude
  constexpr bool kTwo = HALF || V == 1;  // (one value at a time, neighbours are two pieces that are one apart)
  constexpr int P = kTwo ? V : V / 2;    // pairs of a piece
  using Chunk = typename Piece<T, V>::Raw;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long t0 = (long long)blockIdx.x * g.strip;
  const int tokens = (int)(a.tokens - t0 < g.strip ? a.tokens - t0 : g.strip);
  const int apart = HALF ? a.n : 1;
  auto axes = [&](int t, uint32_t& i0, uint32_t& i1, uint32_t& i2) {
    const uint32_t x = (uint32_t)(t0 + t), u = a.inner.div(x);
    i2 = x - u * a.inner.d;
    i0 = a.middle.div(u);
    i1 = u - i0 * a.middle.d;
  };
  for (int i = threadIdx.x; i < tokens * a.n; i += kThreads) {
    const int t = (int)g.pairs.div((uint32_t)i), p = i - t * a.n;
    uint32_t i0, i1, i2;
    axes(t, i0, i1, i2);
    const long long at = i0 * a.sp[0] + i1 * a.sp[1] + i2 * a.sp[2];
    const double pos = (double)(a.wide ? static_cast<const long long*>(a.positions)[at] : (long long)static_cast<const int*>(a.positions)[at]);
    const double f = a.f64 ? static_cast<const double*>(a.frequencies)[p] : (double)static_cast<const float*>(a.frequencies)[p];
    const double turns = pos * (f * 0.15915494309189533577);
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    turn[i] = make_float2(c * a.amplitude, s * a.amplitude * a.sign);
  }
  __syncthreads();
  const int heads = a.heads[0] + a.heads[1], lanes = (int)g.lanes.d;
  // (a head may have more pieces than a block has threads: they take turns)
  for (int first = 0; first < (int)g.head.d; first += kThreads) {
    const int wide = min((int)g.head.d - first, kThreads);
    const int group = first == 0 ? (int)g.head.div(threadIdx.x) : 0, step = first + (int)threadIdx.x - group * (int)g.head.d;
    const int ti = (int)g.lanes.div((uint32_t)group), hl = group - ti * lanes;
    if (ti >= g.side || step >= first + wide) continue;
    const bool turned = step < g.per;
    const int d = turned ? (kTwo && V == 1 && !HALF ? 2 * step : step * V) : 2 * a.n + (step - g.per) * V;
    for (int t = ti; t < tokens; t += g.side) {
      uint32_t i0, i1, i2;
      axes(t, i0, i1, i2);
      float2 cs[P];
#pragma unroll
      for (int e = 0; e < P; ++e) cs[e] = turned ? turn[t * a.n + step * P + e] : make_float2(1.f, 0.f);
      const T* x[2];
      T* y[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        x[w] = static_cast<const T*>(a.x[w]) + i0 * a.sx[w][0] + i1 * a.sx[w][1] + i2 * a.sx[w][2] + d;
        y[w] = static_cast<T*>(a.y[w]) + (t0 + t) * a.heads[w] * a.D + d;
      }
      for (int h0 = hl; h0 < heads; h0 += lanes * kAtOnce) {
        Chunk u[kAtOnce], w[kAtOnce];
        T* to[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          int h = h0 + k * lanes;
          to[k] = nullptr;
          if (h >= heads) continue;
          const bool second = h >= a.heads[0];
          h -= second ? a.heads[0] : 0;
          const T* from = second ? x[1] + h * a.sx[1][3] : x[0] + h * a.sx[0][3];
          to[k] = (second ? y[1] : y[0]) + h * a.D;
          u[k] = *reinterpret_cast<const Chunk*>(from);
          if (kTwo && turned) w[k] = *reinterpret_cast<const Chunk*>(from + apart);
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          if (to[k] == nullptr) continue;
          if (turned) {
            float p[V], q[V];
            Piece<T, V>::get(u[k], p);
            if (kTwo) Piece<T, V>::get(w[k], q);
#pragma unroll
            for (int e = 0; e < P; ++e) {
              float &lo = p[kTwo ? e : 2 * e], &hi = kTwo ? q[e] : p[V > 1 ? 2 * e + 1 : 0];
              const float x0 = lo, x1 = hi;
              lo = x0 * cs[e].x - x1 * cs[e].y;
              hi = x0 * cs[e].y + x1 * cs[e].x;
            }
            u[k] = Piece<T, V>::put(p);
            if (kTwo) *reinterpret_cast<Chunk*>(to[k] + apart) = Piece<T, V>::put(q);
          }
          *reinterpret_cast<Chunk*>(to[k]) = u[k];
        }
      }
    }
  }
}

template <class T, int V, bool HALF>
int launch(const RotaryArgs& a, cudaStream_t st) {
  const int sms = sm_count();
  if (sms <= 0) return EVOATTN_ERR_CUDA;
  Shape g;
  g.per = a.n / (HALF || V == 1 ? V : V / 2);
  const int head = g.per + (a.D - 2 * a.n) / V, heads = a.heads[0] + a.heads[1];
  g.head = FastDiv((uint32_t)head);
  g.pairs = FastDiv((uint32_t)a.n);
  // a thread has kHeads heads of a token or so, fewer where there are few tokens
  const int groups = head < kThreads ? kThreads / head : 1;
  const long long few = a.tokens / (sms * (long long)kMinBlocks);  // tokens of a block that leave every SM some blocks
  int lanes = (heads + kHeads - 1) / kHeads;
  if (few * lanes < groups) lanes = (int)(groups / (few > 0 ? few : 1));
  lanes = lanes > groups ? groups : lanes > heads ? heads : lanes;
  g.lanes = FastDiv((uint32_t)lanes);
  g.side = groups / lanes;
  const int most = g.side > kMostTokens ? g.side : kMostTokens / g.side * g.side;
  g.strip = (int)(few < g.side ? g.side : few < most ? few / g.side * g.side : most);
  const size_t smem = (size_t)g.strip * a.n * sizeof(float2);
  auto kern = rotary_kernel<T, V, HALF>;
  if (!kernel_ready(reinterpret_cast<const void*>(kern), (int)smem, nullptr)) return EVOATTN_ERR_CUDA;
  launch_dependent(kern, dim3((unsigned)((a.tokens + g.strip - 1) / g.strip)), kThreads, smem, st, a, g);
  return cudaGetLastError() == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

int validate(const evoattn_rotary_params* p) {
  if (!p || !p->positions || !p->frequencies || (!p->q && !p->k)) return EVOATTN_ERR_NULL;
  if ((p->q && !p->q_out) || (p->k && !p->k_out)) return EVOATTN_ERR_NULL;
  if (!known_dtype(p->dtype) || (p->layout != EVOATTN_ROTARY_HALF && p->layout != EVOATTN_ROTARY_INTERLEAVED)) return EVOATTN_ERR_DTYPE;
  if (p->D < 1 || p->D > EVOATTN_ROTARY_MAX_D || p->rotary < 2 || p->rotary % 2 || p->rotary > p->D) return EVOATTN_ERR_SHAPE;
  if ((p->q && p->H < 1) || (p->k && p->Hk < 1) || p->H > 65536 || p->Hk > 65536) return EVOATTN_ERR_SHAPE;
  long long tokens = 1;
  for (int i = 0; i < 3; ++i) {
    if (p->n[i] < 1 || p->n[i] > 0x7fffffffLL || (tokens *= p->n[i]) > 0x7fffffffLL) return EVOATTN_ERR_SHAPE;
  }
  if (!(p->amplitude == p->amplitude)) return EVOATTN_ERR_SHAPE;
  return EVOATTN_OK;
}

}  // namespace
}  // namespace evo

extern "C" int evoattn_rotary(const evoattn_rotary_params* p, void* cuda_stream) {
  using namespace evo;
  const int rc = validate(p);
  if (rc) return rc;
  RotaryArgs a{};
  a.x[0] = p->q; a.x[1] = p->k;
  a.y[0] = p->q_out; a.y[1] = p->k_out;
  a.heads[0] = p->q ? p->H : 0;
  a.heads[1] = p->k ? p->Hk : 0;
  for (int i = 0; i < 4; ++i) a.sx[0][i] = p->q_stride[i], a.sx[1][i] = p->k_stride[i];
  a.positions = p->positions;
  for (int i = 0; i < 3; ++i) a.sp[i] = p->position_stride[i];
  a.frequencies = p->frequencies;
  a.wide = p->positions64; a.f64 = p->frequencies64; a.half = p->layout == EVOATTN_ROTARY_HALF;
  a.D = p->D; a.n = p->rotary / 2;
  a.amplitude = p->amplitude; a.sign = p->inverse ? -1.f : 1.f;
  a.tokens = (long long)p->n[0] * p->n[1] * p->n[2];
  a.middle = FastDiv((uint32_t)p->n[1]);
  a.inner = FastDiv((uint32_t)p->n[2]);
  // 16 bytes at a time where every row, the rotated values and (half) the second of each pair begin on such boundaries
  const int es = dtype_bytes(p->dtype), v = 16 / es;
  bool wide = a.D % v == 0 && (a.half ? a.n : 2 * a.n) % v == 0;
  for (int w = 0; w < 2; ++w) {
    if (!a.x[w]) continue;
    wide = wide && (((uintptr_t)a.x[w] | (uintptr_t)a.y[w]) & 15) == 0;
    for (int i = 0; i < 4; ++i) wide = wide && a.sx[w][i] % v == 0;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  return with_dtype(p->dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / (int)sizeof(T);
    if (wide) return a.half ? launch<T, V, true>(a, st) : launch<T, V, false>(a, st);
    return a.half ? launch<T, 1, true>(a, st) : launch<T, 1, false>(a, st);
  });
}
