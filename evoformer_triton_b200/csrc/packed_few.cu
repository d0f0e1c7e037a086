// Attention over packed sequences for few query rows against many keys (new tokens against a cache), forward only: bf16
// and fp16, head dimensions in eights up to 128.
//
// The rows of a sequence that read the same key head (its queries times the heads of a group) are taken 16 at a time: a
// unit is 16 such rows of each of up to four neighbouring key heads, and the keys that they see in blocks.  All units'
// blocks (and, before them, two for the time that a unit takes by itself) lie one behind another and every CTA gets an
// equal share of that line, so that no CTA waits for another whatever the lengths are; a unit that ends up with several
// CTAs is joined by a second kernel (each CTA can leave two parts at most, at the ends of its share), in a fixed order.
// Where every unit is short, CTAs get whole ones and nothing is joined.
//
// Bound by reading K and V once.  A CTA is four warps, each with its own ring of tiles of 16 keys (D <= 64: 32), filled by
// TMA by the warp itself, and its own running maximum, sum and O.  Where there are four key heads or more, a warp has
// one each and all four read the same keys, which lie side by side in memory; else two or four warps share the keys of a
// head and meet at the end of a unit.  Products of 16 rows are warp-level MMAs: tcgen05 would work on 128.  P enters its
// product in two pieces of the type, itself rounded and what that left: a second MMA a tile, which costs nothing beside the
// loads (86.4 us for the case below, 87.7 with one, the same minute), and results are off by their own rounding only (bf16, of the norm: 0.0016
// for one token, 0.0022 with one piece).
//
// 32 sequences of 1 to 8 191 keys, 32 heads of 128 over 8: 86 us, the 465 MB at 5.4 TB/s (with one piece of P 89, 118 with units weighed by
// their keys alone, one head a CTA and exchanges in every tile); even ones of 4 096 keys 98 us, 5.5 TB/s; 16 heads of 64, 16
// key heads, 32 of 4 096: 98 us, 151 with one head a CTA (rows of 128 bytes, 2 KB apart).  Some 10 us of that are the start,
// the end and the joining.
#include <math.h>

#include "packed_sm100.cuh"

namespace evo {
namespace {

using namespace ptx;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kRows = 16;
constexpr int kFewMaxSequences = 2048;  // of a launch
constexpr int kUnitCost = 2;           // blocks of keys that beginning and ending a unit takes the time of (CTAs with ten short units took 98 us where others took 70)
constexpr int kShort = 8;              // blocks of a unit up to which CTAs take whole units: a CTA is through with them in the time that joining takes

template <int DP>
struct FewCfg {
  static constexpr int kKeys = DP == 128 ? 16 : 32;                           // of a warp's tile
  static constexpr int kPanel = kKeys * 128, kTile = DP / 64 * kPanel;        // K or V of a warp
  static constexpr int kStages = 3;
  static constexpr int offRing = 0, offMl = kWarps * kStages * 2 * kTile;
  static constexpr int offBars = offMl + kWarps * kRows * 8, offTable = (offBars + kWarps * kStages * 8 + 64 + 15) / 16 * 16;
  static_assert(2 * kTile >= kRows * DP * 4, "a stage holds a warp's O");
  static constexpr size_t bytes(int B) { return 1024 + offTable + (size_t)(B + 1) * 28 + 64; }
};

// Key heads of a unit, and keys of a block.  Where a CTA gets few keys, it is latency that counts, and all four warps
// work on one head's.
int heads_of(const PackedArgs& a, int ctas) {
  if ((long long)a.Tk * a.Hk < 512LL * ctas) return 1;
  return a.Hk % 4 == 0 ? 4 : a.Hk % 2 == 0 ? 2 : 1;
}
template <int DP>
__host__ __device__ __forceinline__ int block_of(int heads) { return kWarps / heads * FewCfg<DP>::kKeys; }

// Where units lie: blocks and units of the sequences before b, and the share of a CTA.
struct Line {
  int4* spans;        // [B + 1], shared memory: first query, queries, first key, keys
  long long* blocks;  // [B + 1]
  int* units;         // [B + 1]
  int B;
  long long share;    // blocks of a CTA; 0: whole units
};
struct UnitAt {
  int b, unit;               // sequence, unit of it: 16 rows (unit / groups), group of key heads (unit % groups)
  long long begin, end;      // blocks
};
// For all threads of a block; table: 28 (B + 1) bytes, sums: 3 long longs a warp.
__device__ __forceinline__ Line make_line(const PackedArgs& a, int block, int groups, void* table, long long* sums) {
  Line line;
  line.spans = static_cast<int4*>(table);
  line.blocks = reinterpret_cast<long long*>(line.spans + a.B + 1);
  line.units = reinterpret_cast<int*>(line.blocks + a.B + 1);
  line.B = a.B;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long before_b = 0;
  int before_u = 0, most = 0;
  for (int b0 = 0; b0 < a.B; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    int u = 0, nb = 0;
    if (b < a.B) {
      const Span q = query_span(a, b), k = key_span(a, b);
      line.spans[b] = make_int4(q.begin, q.n, k.begin, k.n);
      if (q.n <= a.few_tokens) u = (q.n * a.G + kRows - 1) / kRows * groups;  // (longer sequences are the tile kernel's)
      nb = u ? kUnitCost + (k.n + block - 1) / block : 0;
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
    if (b < a.B) { line.blocks[b] = before_b + sb - own_b; line.units[b] = before_u + su - own_u; }
    before_b += all_b;
    before_u += all_u;
  }
  if (threadIdx.x == 0) { line.blocks[a.B] = before_b; line.units[a.B] = before_u; }
  __syncthreads();
  line.share = most - kUnitCost <= kShort ? 0 : 1;
  return line;
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
  float* o;    // [CTA][2][heads of a unit][16][DP]
  float2* ml;  // [CTA][2][heads of a unit][16]: reference (a power of two) and sum
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
__global__ void __launch_bounds__(kThreads, 2)
packed_few_kernel(const PackedArgs a, const Parts parts, const int clear, const int nh, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV) {
  using C = FewCfg<DP>;
  constexpr int NS = C::kStages, kKeys = C::kKeys;
  const int groups = a.Hk / nh, block = block_of<DP>(nh);
  constexpr float kRise = std::is_same<T, __nv_bfloat16>::value ? 30.f : 14.f;  // powers of two by which a score may lie above the reference
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t ring = smem_u32(smem) + C::offRing + warp * (NS * 2 * C::kTile);
  const uint32_t bars = smem_u32(smem + C::offBars) + warp * NS * 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::offBars + kWarps * NS * 8);
  const uint32_t abort_s = smem_u32(const_cast<int*>(abort_flag));
  __shared__ long long scan[3 * kWarps];
  __shared__ uint32_t where[kWarps];
  if (lane == 0) {
    for (int i = 0; i < NS; ++i) mbar_init_s(bars + 8 * i, 1);
    fence_mbar_init();
  }
  if (tid == 0) { prefetch_tmap(&tmK); prefetch_tmap(&tmV); }
  grid_dependency_wait();
  grid_launch_dependents();
  if (tid == 0) *abort_flag = (a.status && *reinterpret_cast<volatile int*>(a.status) != 0) ? 1 : 0;
  Line line = make_line(a, block, groups, smem + C::offTable, scan);  // (synchronises)
  if (*abort_flag) return;
  set_share(line, gridDim.x);
  const int sub = warp / nh * kKeys, head = warp % nh;  // the warp's first key in a block; its head in a unit
  if (clear && (clear > a.B || line.spans[a.B - 1].x + line.spans[a.B - 1].y - line.spans[0].x < a.Tq))
    zero_outside(a.offsets, a.wide, clear, a.Tq, a.o, (long long)a.H * a.D * 2, blockIdx.x, gridDim.x);

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
    const int4 sp = line.spans[u.b];
    k.end = min(u.end, x1);
    k.key0 = sp.z;
    k.nk = sp.w;
    k.hk = u.unit % groups * nh + head;
    k.x = max(k.x, u.begin + kUnitCost);
    k.j = (int)(k.x - u.begin - kUnitCost) * block + sub;
  };
  Cursor ld{x0, x0, 0, 0, 0, 0};
  uint32_t ls = 0;  // stage that is loaded next
  auto load_next = [&] {  // the next tile that has a key
    while (ld.x < x1) {
      if (ld.x == ld.end) {
        enter(ld);
        if (ld.x >= ld.end) {  // (the share ends before the unit's first block, or the unit has none)
          ld.x = ld.end;
          continue;
        }
      }
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
      ld.j += block;
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
    const int4 sp = line.spans[u.b];
    const Span qs{sp.x, sp.y}, ks{sp.z, sp.w};
    const int hk = u.unit % groups * nh + head, r0 = u.unit / groups * kRows, n_rows = qs.n * a.G;
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
    float o[DP / 8][4], m[2], l[2] = {0.f, 0.f};  // (a row that is none needs no reference)
    m[0] = valid[0] ? -INFINITY : 0.f;
    m[1] = valid[1] ? -INFINITY : 0.f;
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    x = max(x, u.begin + kUnitCost);
    for (int j = (int)(x - u.begin - kUnitCost) * block + sub; x < end; ++x, j += block) {
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
      // S in two chains of MMAs a tile of 8 keys: what a warp waits for is their latency
      float s[2][kKeys / 8][4] = {};
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
        for (int n = 0; n < kKeys / 16; ++n) {
          uint32_t b[4];
          const int r = 16 * n + (lane & 7) + 8 * (lane >> 4), ch = 2 * (k & 3) + ((lane >> 3) & 1);
          ldmatrix4(b, kt + (k >> 2) * C::kPanel + r * 128 + ((ch ^ (r & 7)) << 4));
          mma16816<T>(s[k & 1][2 * n], qa[k], b[0], b[1]);
          mma16816<T>(s[k & 1][2 * n + 1], qa[k], b[2], b[3]);
        }
      }
      // Exponentials against the reference of the tiles before; only where a score lies too far above it (or there is none
      // yet) is the tile's maximum taken, which costs a row's lanes two exchanges.
      float v[2][kKeys / 4];
      bool far = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int f = 0; f < kKeys / 4; ++f) {  // key 8 (f / 2) + 2 (lane % 4) + f % 2
          const int key = j + 8 * (f >> 1) + 2 * (lane & 3) + (f & 1), at = 2 * e + (f & 1);
          v[e][f] = key <= last[e] ? (s[0][f >> 1][at] + s[1][f >> 1][at]) * c : -INFINITY;
          far |= v[e][f] > m[e] + kRise;
        }
      }
      if (__any_sync(0xffffffffu, far)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = v[e][0];
#pragma unroll
          for (int f = 1; f < kKeys / 4; ++f) mx = fmaxf(mx, v[e][f]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float up = fmaxf(m[e], mx), alpha = up > m[e] ? ex2(m[e] - up) : 1.f;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) { o[i][2 * e] *= alpha; o[i][2 * e + 1] *= alpha; }
          l[e] *= alpha;
          m[e] = up;
        }
      }
      uint32_t pa[kKeys / 16][4], pl[kKeys / 16][4];  // P rounded, and what rounding left
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float nm = m[e] == -INFINITY ? 0.f : m[e];
        float p[kKeys / 4];
#pragma unroll
        for (int f = 0; f < kKeys / 4; ++f) p[f] = ex2(v[e][f] - nm);
#pragma unroll
        for (int f = 0; f < kKeys / 4; f += 2) {
          l[e] += p[f] + p[f + 1];
          const int at = (f / 2 & 1) * 2 + e;
          float r0, r1;
          pa[f / 4][at] = Pack2<T>::pack(p[f], p[f + 1]);
          unpack2<T>(pa[f / 4][at], r0, r1);
          pl[f / 4][at] = Pack2<T>::pack(p[f] - r0, p[f + 1] - r1);
        }
      }
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
        for (int n = 0; n < kKeys / 16; ++n) {
          uint32_t b[4];
          const int r = 16 * n + (lane & 7) + 8 * ((lane >> 3) & 1), ch = 2 * (i & 3) + (lane >> 4);
          ldmatrix4_t(b, vt + (i >> 2) * C::kPanel + r * 128 + ((ch ^ (r & 7)) << 4));
          mma16816<T>(o[2 * i], pa[n], b[0], b[1]);
          mma16816<T>(o[2 * i + 1], pa[n], b[2], b[3]);
          mma16816<T>(o[2 * i], pl[n], b[0], b[1]);
          mma16816<T>(o[2 * i + 1], pl[n], b[2], b[3]);
        }
      }
      __syncwarp();  // (every lane has read the tile)
    }

    x = end;

    const bool whole = u.begin >= x0 && u.end <= x1;
    const int slot = (blockIdx.x * 2 + (u.begin > x0 ? 1 : 0)) * nh + head;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    // Columns 8 (i0 + n) + 2 (lane % 4) .. of a row to where they go.
    auto store = [&](const auto& r, int i0, int e, bool with_ml) {
      constexpr int N = sizeof(r) / sizeof(r[0]);
      if (!valid[e]) return;
      const int row = r0 + lane / 4 + 8 * e, i = row / a.G, h = hk * a.G + row - i * a.G, d0 = i0 * 8 + 2 * (lane & 3);
      if (whole) {
        const float inv = l[e] != 0.f ? 1.f / l[e] : 0.f;
        T* out = static_cast<T*>(a.o) + ((long long)(qs.begin + i) * a.H + h) * a.D + d0;
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (8 * n + d0 < a.D) *reinterpret_cast<uint32_t*>(out + 8 * n) = Pack2<T>::pack(r[n][2 * e] * inv, r[n][2 * e + 1] * inv);
      } else {
        const long long at = (long long)slot * kRows + lane / 4 + 8 * e;
        float* out = parts.o + at * DP + d0;
#pragma unroll
        for (int n = 0; n < N; ++n) *reinterpret_cast<float2*>(out + 8 * n) = make_float2(r[n][2 * e], r[n][2 * e + 1]);
        if (with_ml && (lane & 3) == 0) parts.ml[at] = make_float2(m[e], l[e]);
      }
    };
    if (nh == kWarps) {
      store(o, 0, 0, true);
      store(o, 0, 1, true);
      continue;
    }
    // The warps of a head: each leaves its part in the stage that it loads next, and takes a share of the columns.
    float2* ml = reinterpret_cast<float2*>(smem + C::offMl);
    float* mine = reinterpret_cast<float*>(smem + C::offRing + (warp * NS + ls) * (2 * C::kTile));
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if ((lane & 3) == 0) ml[warp * kRows + lane / 4 + 8 * e] = make_float2(m[e], l[e]);
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int f = 0; f < 4; ++f) mine[(4 * i + f) * 32 + lane] = o[i][f];
    if (lane == 0) where[warp] = ls;
    __syncthreads();
    float weight[2][kWarps];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float2 t[kWarps];
      m[e] = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        t[w] = w % nh == head ? ml[w * kRows + lane / 4 + 8 * e] : make_float2(-INFINITY, 0.f);
        m[e] = fmaxf(m[e], t[w].x);
      }
      const float from = m[e] == -INFINITY ? 0.f : m[e];
      l[e] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        weight[e][w] = ex2(t[w].x - from);
        l[e] += t[w].y * weight[e][w];
      }
    }
    // (of two warps a head each takes half of the columns, in two quarters as of four)
    constexpr int kEach = DP / 8 / kWarps;
    const int per = nh;  // quarters of a warp
#pragma unroll 1
    for (int part = 0; part < per; ++part) {
      const int i0 = (warp / nh * per + part) * kEach;
      float r[kEach][4] = {};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w % nh != head) continue;
        const float* in = reinterpret_cast<const float*>(smem + C::offRing + (w * NS + where[w]) * (2 * C::kTile)) + i0 * 128 + lane;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
#pragma unroll
          for (int f = 0; f < 4; ++f) r[i][f] = fmaf(in[(4 * i + f) * 32], weight[f >> 1][w], r[i][f]);
      }
      store(r, i0, 0, i0 == 0);
      store(r, i0, 1, i0 == 0);
    }
    fence_async_shared();  // (what was written here goes before the next TMA copy to it)
    __syncthreads();
  }
  __syncthreads();
  if (*abort_flag) report_abort(*abort_flag, a.status);
}

// Rows whose unit lies in several CTAs' shares: a block per query and head, its warps over the parts and a warp's lanes over
// the values.  What a part weighs is worked out by every warp for itself.
template <class T, int DP>
__global__ void __launch_bounds__(kThreads) packed_join_kernel(const PackedArgs a, const Parts parts, const int ctas, const int nh) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long scan[3 * kWarps];
  __shared__ float sums[kWarps][DP];
  const int groups = a.Hk / nh, block = block_of<DP>(nh);
  // (offsets were complete before the kernel before this one began to read them)
  Line line = make_line(a, block, groups, smem_raw, scan);
  set_share(line, ctas);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (!line.share) return;
  constexpr int V = DP / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long items = (long long)a.Tq * a.H;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const int t = (int)(item / a.H), h = (int)(item - (long long)t * a.H);
    int lo = 0, hi = a.B - 1;  // the last sequence that begins at t or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (line.spans[mid].x <= t) lo = mid;
      else hi = mid - 1;
    }
    const int i = t - line.spans[lo].x, n_units = line.units[lo + 1] - line.units[lo];
    if (i < 0 || i >= line.spans[lo].y || n_units == 0) continue;
    const int hk = h / a.G, r = i * a.G + h - hk * a.G;
    const int each = (int)((line.blocks[lo + 1] - line.blocks[lo]) / n_units);
    const long long begin = line.blocks[lo] + (long long)(r / kRows * groups + hk / nh) * each;
    const int c0 = (int)(begin / line.share), c1 = (int)((begin + each - 1) / line.share);
    if (c0 == c1) continue;
    auto place = [&](int c) { return (((long long)c * 2 + (begin > c * line.share ? 1 : 0)) * nh + hk % nh) * kRows + r % kRows; };
    float mx = -INFINITY, l = 0.f;
    for (int c = c0 + lane; c <= c1; c += 32) mx = fmaxf(mx, parts.ml[place(c)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float from = mx == -INFINITY ? 0.f : mx;
    for (int c = c0 + lane; c <= c1; c += 32) {
      const float2 x = parts.ml[place(c)];
      l += x.y * ptx::ex2(x.x - from);
    }
    l = warp_sum(l);
    float s[V] = {};
#pragma unroll 4
    for (int c = c0 + warp; c <= c1; c += kWarps) {
      const long long at = place(c);
      const float f = ptx::ex2(parts.ml[at].x - from);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] = fmaf(f, parts.o[at * DP + 32 * e + lane], s[e]);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) sums[warp][32 * e + lane] = s[e];
    __syncthreads();
    const int d = threadIdx.x;
    if (d < a.D) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += sums[w][d];
      static_cast<T*>(a.o)[((long long)t * a.H + h) * a.D + d] = from_float<T>(l != 0.f ? v / l : 0.f);
    }
  }
}

int ctas_an_sm(const PackedArgs& a, int B) {
  const size_t need = a.D <= 64 ? FewCfg<64>::bytes(B) : FewCfg<128>::bytes(B);
  return need + 1024 <= 114 * 1024 ? 2 : 1;
}
int padded(const PackedArgs& a) { return a.D <= 64 ? 64 : 128; }
// Few keys leave nothing to join, wherever they lie.
bool may_split(const PackedArgs& a, int ctas) {
  const int nh = heads_of(a, ctas), block = a.D <= 64 ? block_of<64>(nh) : block_of<128>(nh);
  return (a.Tk + block - 1LL) / block > kShort;
}

template <class T, int DP>
int launch(const PackedArgs& args, bool clear, void* ws, cudaStream_t st, int* launches) {
  const int sms = sm_count();
  if (sms <= 0) return EVOATTN_ERR_CUDA;
  CUtensorMap tk, tv;
  if (!make_packed_map(&tk, args.k, args.sk, args.Tk, args.Hk, args.D, FewCfg<DP>::kKeys) || !make_packed_map(&tv, args.v, args.sv, args.Tk, args.Hk, args.D, FewCfg<DP>::kKeys)) return EVOATTN_ERR_CUDA;
  auto kern = packed_few_kernel<T, DP>;
  auto join = packed_join_kernel<T, DP>;
  const int es = args.wide ? 8 : 4;
  for (int b0 = 0; b0 < args.B; b0 += kFewMaxSequences) {
    PackedArgs a = args;
    a.B = args.B - b0 < kFewMaxSequences ? args.B - b0 : kFewMaxSequences;
    a.offsets = static_cast<const unsigned char*>(args.offsets) + (long long)b0 * es;
    a.key_offsets = static_cast<const unsigned char*>(args.key_offsets) + (long long)b0 * es * (args.ranges ? 2 : 1);
    const int ctas = sms * ctas_an_sm(a, a.B), nh = heads_of(a, ctas);
    Parts parts{static_cast<float*>(ws), nullptr};
    parts.ml = reinterpret_cast<float2*>(parts.o + (size_t)ctas * 2 * nh * kRows * DP);
    const size_t smem = FewCfg<DP>::bytes(a.B);
    if (!kernel_ready(reinterpret_cast<const void*>(kern), (int)smem, nullptr)) return EVOATTN_ERR_CUDA;
    launch_dependent(kern, dim3((unsigned)ctas), kThreads, smem, st, a, parts, clear && b0 == 0 ? args.B : 0, nh, tk, tv);
    *launches += 1;
    if (may_split(a, ctas)) {
      const size_t jsmem = (size_t)(a.B + 1) * 28 + 16;
      if (!kernel_ready(reinterpret_cast<const void*>(join), (int)jsmem, nullptr)) return EVOATTN_ERR_CUDA;
      const long long rows = (long long)args.Tq * a.H;
      launch_dependent(join, dim3((unsigned)(rows < 16LL * sms ? rows : 16LL * sms)), kThreads, jsmem, st, a, parts, ctas, nh);
      *launches += 1;
    }
  }
  return cudaGetLastError() == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

}  // namespace

size_t packed_few_workspace_bytes(const PackedArgs& a) {
  const int sms = sm_count();
  if (sms <= 0 || !may_split(a, sms * ctas_an_sm(a, a.B < kFewMaxSequences ? a.B : kFewMaxSequences))) return 0;
  return (size_t)sms * 2 * 2 * kWarps * kRows * ((size_t)padded(a) * 4 + 8);
}
int launch_packed_few(int dtype, const PackedArgs& a, bool clear, void* ws, cudaStream_t st, int* launches) {
  if (dtype == EVOATTN_BF16) return a.D <= 64 ? launch<__nv_bfloat16, 64>(a, clear, ws, st, launches) : launch<__nv_bfloat16, 128>(a, clear, ws, st, launches);
  return a.D <= 64 ? launch<__half, 64>(a, clear, ws, st, launches) : launch<__half, 128>(a, clear, ws, st, launches);
}

}  // namespace evo
