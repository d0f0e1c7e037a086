// Attention over packed sequences for few query rows against many keys (new tokens against a cache), forward only: bf16
// and fp16, head dimensions in eights up to 128.
//
// The rows of a sequence that read the same key head (its queries times the heads of a group) are taken 16 at a time:
// a unit is 16 rows, one key head and the keys that they see in blocks of 64.  All units' blocks lie one behind another
// and every CTA gets an equal share of that line, so that no CTA waits for another whatever the lengths are; a unit that
// ends up with several CTAs is joined by a second kernel (each CTA can leave two parts at most, at the ends of its
// share).  Where every unit is short, CTAs get whole ones and nothing is joined.
//
// Bound by reading K and V once.  A CTA is four warps, each with its own ring of tiles of 16 keys, filled by TMA by
// the warp itself, and its own running maximum, sum and O; they meet at the end of a unit.  Products of 16 rows are
// warp-level MMAs: tcgen05 would work on 128.
#include <math.h>

#include "packed_sm100.cuh"

namespace evo {
namespace {

using namespace ptx;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kRows = 16, kKeys = 16, kBlock = kWarps * kKeys;
constexpr int kFewMaxSequences = 2048;  // of a launch
constexpr int kShort = 8;  // blocks of a unit up to which CTAs take whole units: a CTA is through with 512 keys in the time that joining takes

template <int DP>
struct FewCfg {
  static constexpr int kPanel = kKeys * 128, kTile = DP / 64 * kPanel;  // K or V of a warp
  static constexpr int kStages = DP == 128 ? 3 : 6;
  static constexpr int offRing = 0, offSum = kWarps * kStages * 2 * kTile, offMl = offSum + kRows * DP * 4;
  static constexpr int offBars = offMl + kWarps * kRows * 8, offTable = offBars + kWarps * kStages * 8 + 64;
  static constexpr size_t bytes(int B) { return 1024 + offTable + (size_t)(B + 1) * 12 + 64; }
};

// Where units lie: blocks and units of the sequences before b, and the share of a CTA.
struct Line {
  long long* blocks;  // [B + 1], shared memory
  int* units;         // [B + 1]
  int B, Hk;
  long long share;    // blocks of a CTA; 0: whole units
};
struct UnitAt {
  int b, unit;               // sequence, unit of it: 16 rows (unit / Hk), key head (unit % Hk)
  long long begin, end;      // blocks
};
__device__ __forceinline__ int rows_of(const PackedArgs& a, int b) {
  const int n = query_span(a, b).n;
  return n > a.few_tokens ? 0 : n * a.G;  // (longer sequences are the tile kernel's)
}
// For all threads of a block.  sums: 3 long longs a warp.
__device__ __forceinline__ Line make_line(const PackedArgs& a, long long* blocks, int* units, long long* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long before_b = 0;
  int before_u = 0, most = 0;
  for (int b0 = 0; b0 < a.B; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    int u = 0, nb = 0;
    if (b < a.B) {
      u = (rows_of(a, b) + kRows - 1) / kRows * a.Hk;
      nb = u ? max(1, (key_span(a, b).n + kBlock - 1) / kBlock) : 0;
    }
    long long sb = (long long)u * nb;
    int su = u, mx = nb;
    const long long own_b = sb;
    const int own_u = su;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long xb = __shfl_up_sync(0xffffffffu, sb, o);
      const int xu = __shfl_up_sync(0xffffffffu, su, o);
      if (lane >= o) { sb += xb; su += xu; }
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    __syncthreads();
    if (lane == 31) { sums[3 * warp] = sb; sums[3 * warp + 1] = su; sums[3 * warp + 2] = mx; }
    __syncthreads();
    long long all_b = 0;
    int all_u = 0;
    for (int w = 0; w < warps; ++w) {
      if (w == warp) { sb += all_b; su += all_u; }
      all_b += sums[3 * w];
      all_u += (int)sums[3 * w + 1];
      most = max(most, (int)sums[3 * w + 2]);
    }
    if (b < a.B) { blocks[b] = before_b + sb - own_b; units[b] = before_u + su - own_u; }
    before_b += all_b;
    before_u += all_u;
  }
  if (threadIdx.x == 0) { blocks[a.B] = before_b; units[a.B] = before_u; }
  __syncthreads();
  return Line{blocks, units, a.B, a.Hk, most <= kShort ? 0 : (long long)most};
}
__device__ __forceinline__ void set_share(Line& l, int ctas) {
  if (l.share) l.share = max((long long)kShort / 2, (l.blocks[l.B] + ctas - 1) / ctas);
}
template <class V>
__device__ __forceinline__ int last_not_above(const V* p, int n, V x) {  // the last b < n with p[b] <= x (p ascends; empty ones repeat)
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ int blocks_each(const Line& l, int b) { return (int)((l.blocks[b + 1] - l.blocks[b]) / (l.units[b + 1] - l.units[b])); }
__device__ __forceinline__ UnitAt unit_of_block(const Line& l, long long x) {
  UnitAt u;
  u.b = last_not_above(l.blocks, l.B, x);
  const int each = blocks_each(l, u.b);
  u.unit = (int)((x - l.blocks[u.b]) / each);
  u.begin = l.blocks[u.b] + (long long)u.unit * each;
  u.end = u.begin + each;
  return u;
}
__device__ __forceinline__ UnitAt unit_at(const Line& l, int n) {
  UnitAt u;
  u.b = last_not_above(l.units, l.B, n);
  u.unit = n - l.units[u.b];
  const int each = blocks_each(l, u.b);
  u.begin = l.blocks[u.b] + (long long)u.unit * each;
  u.end = u.begin + each;
  return u;
}

struct Parts {
  float* o;    // [CTA][2][16][DP]
  float2* ml;  // [CTA][2][16]: reference (a power of two) and sum
};

template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

template <class T, int DP>
__global__ void __launch_bounds__(kThreads)
packed_few_kernel(const PackedArgs a, const Parts parts, const int clear, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV) {
  using C = FewCfg<DP>;
  constexpr int NS = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t ring = smem_u32(smem) + C::offRing + warp * (NS * 2 * C::kTile);
  const uint32_t bars = smem_u32(smem + C::offBars) + warp * NS * 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::offBars + kWarps * NS * 8);
  const uint32_t abort_s = smem_u32(const_cast<int*>(abort_flag));
  long long* t_blocks = reinterpret_cast<long long*>(smem + C::offTable);
  int* t_units = reinterpret_cast<int*>(t_blocks + a.B + 1);
  __shared__ long long scan[3 * kWarps];
  if (lane == 0) {
    for (int i = 0; i < NS; ++i) mbar_init_s(bars + 8 * i, 1);
    fence_mbar_init();
  }
  if (tid == 0) { prefetch_tmap(&tmK); prefetch_tmap(&tmV); }
  grid_dependency_wait();
  grid_launch_dependents();
  if (tid == 0) *abort_flag = (a.status && *reinterpret_cast<volatile int*>(a.status) != 0) ? 1 : 0;
  Line line = make_line(a, t_blocks, t_units, scan);  // (synchronises)
  if (*abort_flag) return;
  set_share(line, gridDim.x);
  if (clear) zero_outside(a.offsets, a.wide, clear, a.Tq, a.o, (long long)a.H * a.D * 2, blockIdx.x, gridDim.x);

  const long long n_blocks = line.blocks[a.B];
  long long x0, x1;
  if (line.share) {
    x0 = min(n_blocks, blockIdx.x * line.share);
    x1 = min(n_blocks, x0 + line.share);
  } else {
    const long long n = line.units[a.B];
    const int u0 = (int)(n * blockIdx.x / gridDim.x), u1 = (int)(n * (blockIdx.x + 1) / gridDim.x);
    x0 = u0 < u1 ? unit_at(line, u0).begin : 0;
    x1 = u0 < u1 ? unit_at(line, u1 - 1).end : 0;
  }
  const float c = a.scale * kLog2e;

  // The warp's tiles along the share: a cursor that loads, NS - 1 tiles ahead of the one that computes.
  struct Cursor {
    long long x, end;   // block; end of the unit
    int key0, nk, hk;   // of the unit's sequence and head
    int j;              // first key of the warp's tile
  };
  auto enter = [&](Cursor& k) {
    const UnitAt u = unit_of_block(line, k.x);
    const Span ks = key_span(a, u.b);
    k.end = min(u.end, x1);
    k.key0 = ks.begin;
    k.nk = ks.n;
    k.hk = u.unit % a.Hk;
    k.j = (int)(k.x - u.begin) * kBlock + warp * kKeys;
  };
  Cursor ld{x0, x0, 0, 0, 0, 0};
  uint32_t ls = 0;  // stage that is loaded next
  auto load_next = [&] {  // the next tile that has a key
    while (ld.x < x1) {
      if (ld.x == ld.end) enter(ld);
      const bool any = ld.j < ld.nk;
      if (any && lane == 0) {
        const uint32_t dst = ring + ls * (2 * C::kTile), bar = bars + 8 * ls;
        mbar_expect_tx_s(bar, 2 * C::kTile);
#pragma unroll
        for (int p = 0; p < DP / 64; ++p) {
          tma_load_3d_s(dst + p * C::kPanel, &tmK, bar, 64 * p, ld.key0 + ld.j, ld.hk);
          tma_load_3d_s(dst + C::kTile + p * C::kPanel, &tmV, bar, 64 * p, ld.key0 + ld.j, ld.hk);
        }
      }
      ++ld.x;
      ld.j += kBlock;
      if (any) {
        if (++ls == NS) ls = 0;
        return;
      }
    }
  };
  for (int i = 0; i < NS - 1; ++i) load_next();

  uint32_t st = 0, par = 0;
  for (long long x = x0; x < x1;) {
    const UnitAt u = unit_of_block(line, x);
    const Span qs = query_span(a, u.b), ks = key_span(a, u.b);
    const int hk = u.unit % a.Hk, r0 = u.unit / a.Hk * kRows, n_rows = qs.n * a.G;
    const long long end = min(u.end, x1);
    // Rows lane / 4 and lane / 4 + 8 of the unit: where they lie, and the last key they see.
    int last[2];
    const T* q[2];
    bool valid[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = r0 + lane / 4 + 8 * e;
      valid[e] = r < n_rows;
      const int i = valid[e] ? r / a.G : 0, g = valid[e] ? r - i * a.G : 0;
      last[e] = a.causal ? min(ks.n - 1, i + ks.n - qs.n) : ks.n - 1;
      q[e] = static_cast<const T*>(a.q) + (long long)(qs.begin + i) * a.sq[0] + (long long)(hk * a.G + g) * a.sq[1];
    }
    uint32_t qa[DP / 16][4];
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
      for (int f = 0; f < 4; ++f) {  // (rows lane / 4, + 8; values 2 (lane % 4), + 8)
        const int d = 16 * k + 2 * (lane & 3) + 8 * (f >> 1);
        qa[k][f] = valid[f & 1] && d < a.D ? *reinterpret_cast<const uint32_t*>(q[f & 1] + d) : 0u;
      }
    }
    float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    for (int j = (int)(x - u.begin) * kBlock + warp * kKeys; x < end; ++x, j += kBlock) {
      if (j >= ks.n) continue;
      load_next();
      mbar_wait_s(bars + 8 * st, par, abort_s, DEV_TIMEOUT_TMA);
      const uint32_t kt = ring + st * (2 * C::kTile), vt = kt + C::kTile;
      if (++st == NS) { st = 0; par ^= 1; }
      const int real = ks.n - j;
      if (real < kKeys) {  // rows behind the end may hold anything, and P = 0 times infinity is not 0
        for (int y = real * 128 + lane * 16; y < C::kPanel; y += 512)
#pragma unroll
          for (int p = 0; p < DP / 64; ++p) sts_v4(vt + p * C::kPanel + y, 0, 0, 0, 0);
        fence_async_shared();
        __syncwarp();
      }
      float s[2][4] = {};
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        uint32_t b[4];
        const int r = (lane & 7) + 8 * (lane >> 4), ch = 2 * (k & 3) + ((lane >> 3) & 1);
        ldmatrix4(b, kt + (k >> 2) * C::kPanel + r * 128 + ((ch ^ (r & 7)) << 4));
        mma16816<T>(s[0], qa[k], b[0], b[1]);
        mma16816<T>(s[1], qa[k], b[2], b[3]);
      }
      uint32_t pa[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v[4], mx = -INFINITY;
#pragma unroll
        for (int f = 0; f < 4; ++f) {  // key 8 (f / 2) + 2 (lane % 4) + f % 2
          const int key = j + 8 * (f >> 1) + 2 * (lane & 3) + (f & 1);
          v[f] = key <= last[e] ? s[f >> 1][2 * e + (f & 1)] * c : -INFINITY;
          mx = fmaxf(mx, v[f]);
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float up = fmaxf(m[e], mx), from = up == -INFINITY ? 0.f : up;
        const float alpha = ex2(m[e] - from);
        if (__any_sync(0xffffffffu, up != m[e])) {
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) { o[i][2 * e] *= alpha; o[i][2 * e + 1] *= alpha; }
        }
        m[e] = up;
        float p[4];
#pragma unroll
        for (int f = 0; f < 4; ++f) p[f] = ex2(v[f] - from);
        l[e] = l[e] * alpha + ((p[0] + p[1]) + (p[2] + p[3]));
        pa[e] = Pack2<T>::pack(p[0], p[1]);
        pa[2 + e] = Pack2<T>::pack(p[2], p[3]);
      }
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        uint32_t b[4];
        const int r = (lane & 7) + 8 * ((lane >> 3) & 1), ch = 2 * (i & 3) + (lane >> 4);
        ldmatrix4_t(b, vt + (i >> 2) * C::kPanel + r * 128 + ((ch ^ (r & 7)) << 4));
        mma16816<T>(o[2 * i], pa, b[0], b[1]);
        mma16816<T>(o[2 * i + 1], pa, b[2], b[3]);
      }
      __syncwarp();  // (every lane has read the tile)
    }

    // The warps' parts of the unit: to one reference, then added up from the last warp to the first.
    float2* ml = reinterpret_cast<float2*>(smem + C::offMl);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if ((lane & 3) == 0) ml[warp * kRows + lane / 4 + 8 * e] = make_float2(m[e], l[e]);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float up = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) up = fmaxf(up, ml[w * kRows + lane / 4 + 8 * e].x);
      const float from = up == -INFINITY ? 0.f : up;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 t = ml[w * kRows + lane / 4 + 8 * e];
        sum += t.y * ex2(t.x - from);
      }
      const float f = ex2(m[e] - from);
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) { o[i][2 * e] *= f; o[i][2 * e + 1] *= f; }
      m[e] = up;
      l[e] = sum;
    }
    float* sum = reinterpret_cast<float*>(smem + C::offSum);
#pragma unroll 1
    for (int w = kWarps - 1; w > 0; --w) {
      if (warp == w) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
          for (int f = 0; f < 4; ++f) sum[(4 * i + f) * 32 + lane] = o[i][f];
      }
      __syncthreads();
      if (warp == w - 1) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
          for (int f = 0; f < 4; ++f) o[i][f] += sum[(4 * i + f) * 32 + lane];
      }
      __syncthreads();
    }
    if (warp == 0) {
      const bool whole = u.begin >= x0 && u.end <= x1;
      const int slot = blockIdx.x * 2 + (u.begin > x0 ? 1 : 0);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (!valid[e]) continue;
        const int r = r0 + lane / 4 + 8 * e, i = r / a.G, h = hk * a.G + r - i * a.G;
        if (whole) {
          const float inv = l[e] > 0.f ? 1.f / l[e] : 0.f;
          T* out = static_cast<T*>(a.o) + ((long long)(qs.begin + i) * a.H + h) * a.D;
#pragma unroll
          for (int n = 0; n < DP / 8; ++n)
            if (8 * n < a.D) *reinterpret_cast<uint32_t*>(out + 8 * n + 2 * (lane & 3)) = Pack2<T>::pack(o[n][2 * e] * inv, o[n][2 * e + 1] * inv);
        } else {
          const int row = lane / 4 + 8 * e;
          float* out = parts.o + ((long long)slot * kRows + row) * DP;
#pragma unroll
          for (int n = 0; n < DP / 8; ++n) *reinterpret_cast<float2*>(out + 8 * n + 2 * (lane & 3)) = make_float2(o[n][2 * e], o[n][2 * e + 1]);
          if ((lane & 3) == 0) parts.ml[slot * kRows + row] = make_float2(m[e], l[e]);
        }
      }
    }
  }
  __syncthreads();
  if (*abort_flag) report_abort(*abort_flag, a.status);
}

// Units that lie in several CTAs' shares: a block per row of one, its threads over the values.
template <class T, int DP>
__global__ void __launch_bounds__(128) packed_join_kernel(const PackedArgs a, const Parts parts, const int ctas) {
  extern __shared__ uint8_t smem_raw[];
  long long* t_blocks = reinterpret_cast<long long*>(smem_raw);
  int* t_units = reinterpret_cast<int*>(t_blocks + a.B + 1);
  float* weight = reinterpret_cast<float*>(t_units + a.B + 1);  // [ctas]
  __shared__ long long scan[12];
  __shared__ float red[8];
  grid_dependency_wait();
  grid_launch_dependents();
  Line line = make_line(a, t_blocks, t_units, scan);
  set_share(line, ctas);
  if (!line.share) return;
  const long long items = (long long)line.units[a.B] * kRows;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const UnitAt u = unit_at(line, (int)(item / kRows));
    const int row = (int)(item % kRows);
    const Span qs = query_span(a, u.b);
    const int hk = u.unit % a.Hk, r = u.unit / a.Hk * kRows + row;
    const int c0 = (int)(u.begin / line.share), c1 = (int)((u.end - 1) / line.share);
    if (c0 == c1 || r >= qs.n * a.G) continue;
    auto slot = [&](int c) { return c * 2 + (u.begin > c * line.share ? 1 : 0); };
    float mx = -INFINITY;
    for (int c = c0 + threadIdx.x; c <= c1; c += 128) mx = fmaxf(mx, parts.ml[slot(c) * kRows + row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    __syncthreads();
    if (lane == 0) red[warp] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float from = mx == -INFINITY ? 0.f : mx;
    float l = 0.f;
    for (int c = c0 + threadIdx.x; c <= c1; c += 128) {
      const float2 t = parts.ml[slot(c) * kRows + row];
      const float f = exp2f(t.x - from);
      weight[c - c0] = f;
      l += t.y * f;
    }
    l = warp_sum(l);
    if (lane == 0) red[4 + warp] = l;
    __syncthreads();
    l = (red[4] + red[5]) + (red[6] + red[7]);
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int i = r / a.G, h = hk * a.G + r - i * a.G, d = threadIdx.x;
    if (d < a.D) {
      float s = 0.f;
#pragma unroll 4
      for (int c = c0; c <= c1; ++c) s = fmaf(weight[c - c0], parts.o[((long long)slot(c) * kRows + row) * DP + d], s);
      static_cast<T*>(a.o)[((long long)(qs.begin + i) * a.H + h) * a.D + d] = from_float<T>(s * inv);
    }
  }
}

int ctas_an_sm(const PackedArgs& a, int B) {
  const size_t need = a.D <= 64 ? FewCfg<64>::bytes(B) : FewCfg<128>::bytes(B);
  return need + 1024 <= 114 * 1024 ? 2 : 1;
}
int padded(const PackedArgs& a) { return a.D <= 64 ? 64 : 128; }

template <class T, int DP>
int launch(const PackedArgs& args, bool clear, void* ws, cudaStream_t st, int* launches) {
  const int sms = sm_count();
  if (sms <= 0) return EVOATTN_ERR_CUDA;
  CUtensorMap tk, tv;
  if (!make_packed_map(&tk, args.k, args.sk, args.Tk, args.Hk, args.D, kKeys) || !make_packed_map(&tv, args.v, args.sv, args.Tk, args.Hk, args.D, kKeys)) return EVOATTN_ERR_CUDA;
  auto kern = packed_few_kernel<T, DP>;
  auto join = packed_join_kernel<T, DP>;
  const int es = args.wide ? 8 : 4;
  for (int b0 = 0; b0 < args.B; b0 += kFewMaxSequences) {
    PackedArgs a = args;
    a.B = args.B - b0 < kFewMaxSequences ? args.B - b0 : kFewMaxSequences;
    a.offsets = static_cast<const unsigned char*>(args.offsets) + (long long)b0 * es;
    a.key_offsets = static_cast<const unsigned char*>(args.key_offsets) + (long long)b0 * es * (args.ranges ? 2 : 1);
    const int ctas = sms * ctas_an_sm(a, a.B);
    Parts parts{static_cast<float*>(ws), nullptr};
    parts.ml = reinterpret_cast<float2*>(parts.o + (size_t)ctas * 2 * kRows * DP);
    const size_t smem = FewCfg<DP>::bytes(a.B);
    if (!kernel_ready(reinterpret_cast<const void*>(kern), (int)smem, nullptr)) return EVOATTN_ERR_CUDA;
    launch_dependent(kern, dim3((unsigned)ctas), kThreads, smem, st, a, parts, clear && b0 == 0 ? args.B : 0, tk, tv);
    *launches += 1;
    // (keys in fewer blocks than kShort leave nothing to join, wherever they lie)
    if (args.Tk > kShort * kBlock) {
      const size_t jsmem = (size_t)(a.B + 1) * 12 + (size_t)ctas * 4 + 16;
      if (!kernel_ready(reinterpret_cast<const void*>(join), (int)jsmem, nullptr)) return EVOATTN_ERR_CUDA;
      const long long rows = ((long long)args.Tq * a.G / kRows + a.B) * a.Hk * kRows;
      launch_dependent(join, dim3((unsigned)(rows < 8LL * sms ? rows : 8LL * sms)), 128, jsmem, st, a, parts, ctas);
      *launches += 1;
    }
  }
  return cudaGetLastError() == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

}  // namespace

size_t packed_few_workspace_bytes(const PackedArgs& a) {
  const int sms = sm_count();
  return (size_t)(sms > 0 ? sms : 1) * 2 * 2 * kRows * ((size_t)padded(a) * 4 + 8);
}
int launch_packed_few(int dtype, const PackedArgs& a, bool clear, void* ws, cudaStream_t st, int* launches) {
  if (dtype == EVOATTN_BF16) return a.D <= 64 ? launch<__nv_bfloat16, 64>(a, clear, ws, st, launches) : launch<__nv_bfloat16, 128>(a, clear, ws, st, launches);
  return a.D <= 64 ? launch<__half, 64>(a, clear, ws, st, launches) : launch<__half, 128>(a, clear, ws, st, launches);
}

}  // namespace evo
