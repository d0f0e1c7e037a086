// Rotary positions: pairs (a, b) of a head's values turned by angle = position * frequency of the pair,
//   (a, b) -> amplitude (a cos - b sin, a sin + b cos),
// over q and k in one launch; the gradient is the same with the angle's sign changed.  "half": pair i is (x_i, x_{i+n}) of
// the 2 n rotated values, else (x_{2i}, x_{2i+1}).  Values behind them are copied.
//
// Angles: a position of 10^6 times a frequency of 1 rounded to fp32 is off by 0.03 of a radian.  Here turns = position *
// (frequency / 2 pi) are formed in fp64 (off by 2^-53 of them), whole turns are taken off there, and sine and cosine are of
// the fraction, which fp32 holds to 2^-26 of a turn.
//
// Bound by memory.  A block takes the tokens of a strip: sines and cosines of each once, into shared memory, then all
// heads of q and k, 16 bytes at a time.
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

constexpr int kThreads = 256;

// V values are handled at once: V pairs (half) or V / 2 (neighbours).
template <class T, int V>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a, const int strip) {
  extern __shared__ float2 turn[];  // [strip][n]: cos and sin, times the amplitude
  const long long t0 = (long long)blockIdx.x * strip;
  const int tokens = (int)(a.tokens - t0 < strip ? a.tokens - t0 : strip);
  auto axes = [&](long long t, uint32_t& i0, uint32_t& i1, uint32_t& i2) {
    const uint32_t u = a.inner.div((uint32_t)t);
    i2 = (uint32_t)t - u * a.inner.d;
    i0 = a.middle.div(u);
    i1 = u - i0 * a.middle.d;
  };
  for (int i = threadIdx.x; i < tokens * a.n; i += kThreads) {
    const int t = i / a.n, p = i - t * a.n;
    uint32_t i0, i1, i2;
    axes(t0 + t, i0, i1, i2);
    const long long at = i0 * a.sp[0] + i1 * a.sp[1] + i2 * a.sp[2];
    const double pos = (double)(a.wide ? static_cast<const long long*>(a.positions)[at] : (long long)static_cast<const int*>(a.positions)[at]);
    const double f = a.f64 ? static_cast<const double*>(a.frequencies)[p] : (double)static_cast<const float*>(a.frequencies)[p];
    const double turns = pos * (f * 0.15915494309189533577);
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    turn[i] = make_float2(c * a.amplitude, s * a.amplitude * a.sign);
  }
  __syncthreads();
  const int pairs_at_once = a.half || V == 1 ? V : V / 2;
  const int per = a.n / pairs_at_once;                        // steps of a head's rotated values
  const int all = per + (a.D - 2 * a.n) / V;                  // ... and of its others
  const int heads = a.heads[0] + a.heads[1], per_token = heads * all;
  for (int i = threadIdx.x; i < tokens * per_token; i += kThreads) {
    const int t = i / per_token, r = i - t * per_token;
    int h = r / all;
    const int step = r - h * all;
    const int which = h >= a.heads[0];
    h -= which ? a.heads[0] : 0;
    uint32_t i0, i1, i2;
    axes(t0 + t, i0, i1, i2);
    const T* x = static_cast<const T*>(a.x[which]) + i0 * a.sx[which][0] + i1 * a.sx[which][1] + i2 * a.sx[which][2] + h * a.sx[which][3];
    T* y = static_cast<T*>(a.y[which]) + ((t0 + t) * a.heads[which] + h) * a.D;
    struct alignas(sizeof(T) * V) Chunk { T v[V]; };
    auto load = [&](int d) { return *reinterpret_cast<const Chunk*>(x + d); };
    auto store = [&](int d, const Chunk& c) { *reinterpret_cast<Chunk*>(y + d) = c; };
    if (step >= per) {
      const int d = 2 * a.n + (step - per) * V;
      store(d, load(d));
    } else if (a.half || V == 1) {
      const int d = a.half ? step * V : 2 * step, apart = a.half ? a.n : 1;  // (one pair at a time: neighbours are one apart)
      Chunk u = load(d), w = load(d + apart);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 cs = turn[t * a.n + step * V + e];
        const float p = to_float(u.v[e]), q = to_float(w.v[e]);
        u.v[e] = from_float<T>(p * cs.x - q * cs.y);
        w.v[e] = from_float<T>(p * cs.y + q * cs.x);
      }
      store(d, u);
      store(d + apart, w);
    } else if constexpr (V > 1) {
      const int d = step * V;
      Chunk u = load(d);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 cs = turn[t * a.n + (d + e) / 2];
        const float p = to_float(u.v[e]), q = to_float(u.v[e + 1]);
        u.v[e] = from_float<T>(p * cs.x - q * cs.y);
        u.v[e + 1] = from_float<T>(p * cs.y + q * cs.x);
      }
      store(d, u);
    }
  }
}

template <class T, int V>
int launch(const RotaryArgs& a, cudaStream_t st) {
  const int sms = sm_count();
  if (sms <= 0) return EVOATTN_ERR_CUDA;
  long long strip = a.tokens / (sms * 16LL);
  strip = strip < 1 ? 1 : strip > 8 ? 8 : strip;
  const size_t smem = (size_t)strip * a.n * sizeof(float2);
  auto kern = rotary_kernel<T, V>;
  if (!kernel_ready(reinterpret_cast<const void*>(kern), (int)smem, nullptr)) return EVOATTN_ERR_CUDA;
  kern<<<(unsigned)((a.tokens + strip - 1) / strip), kThreads, smem, st>>>(a, (int)strip);
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
    if (wide) return launch<T, 16 / (int)sizeof(T)>(a, st);
    return launch<T, 1>(a, st);
  });
}
