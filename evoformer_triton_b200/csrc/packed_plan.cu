// What precedes the tensor-core kernels of attention over packed sequences: the lists of tiles that they walk, made on the
// device, where the offsets are, and the row sums of dO * O for the backward, in one launch.
#include "packed_sm100.cuh"

namespace evo {
namespace {

constexpr int kThreads = 512;
constexpr int kClasses = kThreads;  // by work, in steps that are as wide as the longest tile makes them

constexpr int kKept = 1024;

struct Sums {
  int4 spans[kKept];
  int first[kClasses];
  int warps[kThreads / 32 + 1];
  long long steps;
  long long rows;
  int slots, joins, most;
};

// The tiles of all sequences, a warp per sequence and its lanes over the tiles; called several times, so the spans of the
// first kKept sequences are kept in shared memory.
struct Tiles {
  const int4* kept;
  __device__ __forceinline__ Tiles(const PackedArgs& a, int4* keep) : kept(keep) {
    for (int b = threadIdx.x; b < a.B && b < kKept; b += kThreads) {
      const Span q = query_span(a, b), k = key_span(a, b);
      keep[b] = make_int4(q.begin, q.n, k.begin, k.n);
    }
    __syncthreads();
  }
  template <class F>
  __device__ __forceinline__ void each(const PackedArgs& a, bool queries, int unit, F&& f) const {
    for (int b = threadIdx.x >> 5; b < a.B; b += kThreads / 32) {
      Span qs, ks;
      if (b < kKept) {
        const int4 x = kept[b];
        qs = Span{x.x, x.y};
        ks = Span{x.z, x.w};
      } else {
        qs = query_span(a, b);
        ks = key_span(a, b);
      }
      const int n = !queries ? ks.n : qs.n > a.few_tokens ? qs.n : 0;
      for (int x = (threadIdx.x & 31) * unit; x < n; x += 32 * unit) {
        PackedTile t{};
        t.rows = min(unit, n - x);
        t.parts = 1;
        if (queries) {
          t.row = qs.begin + x;
          t.other = ks.begin;
          t.n = ks.n;
          t.shift = x + ks.n - qs.n;
          t.tiles = (keys_seen(a, qs.n, ks.n, x, unit) + kTileRows - 1) / kTileRows;
          t.steps = t.tiles;
        } else {
          t.row = ks.begin + x;
          t.other = qs.begin;
          t.n = qs.n;
          t.shift = x + qs.n - ks.n;
          const int first = a.causal ? max(0, t.shift) : 0;  // the first query that sees a key of the tile
          t.tiles = first < qs.n ? (qs.n + kTileRows - 1) / kTileRows - first / kTileRows : 0;
          t.steps = t.tiles * a.G;
          t.blind = a.causal ? max(0, qs.n - ks.n) : 0;
        }
        f(t);
      }
    }
  }
};

// A list by a counting sort, most work first, so that what a persistent grid ends with is short.  Tiles with more steps than a
// share of those of an SM are cut into parts, which leave fp32 sums to be joined: a group of heads or a long
// sequence makes single tiles that would outlast everything else.
__device__ __forceinline__ void make_list(const PackedArgs& a, const PackedPlan& plan, bool queries, int unit, int sms, const PackedCut& c, Sums& s) {
  const Tiles tiles(a, s.spans);
  PackedTile* out = queries ? plan.queries : plan.keys;
  for (int i = threadIdx.x; i < kClasses; i += kThreads) s.first[i] = 0;
  if (queries)
    for (int i = threadIdx.x; i < plan.n_arrived; i += kThreads) plan.arrived[i] = 0;
  if (threadIdx.x == 0) { s.steps = 0; s.slots = 0; s.joins = 0; s.rows = 0; s.most = 0; }
  __syncthreads();
  long long work = 0, n = 0;
  int most = 0;
  tiles.each(a, queries, unit, [&](const PackedTile& t) {
    work += t.steps;
    most = max(most, t.steps);
    n += t.rows;
  });
  most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    work += __shfl_xor_sync(0xffffffffu, work, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if ((threadIdx.x & 31) == 0 && n) {
    atomicAdd(reinterpret_cast<unsigned long long*>(&s.steps), (unsigned long long)work);
    atomicAdd(reinterpret_cast<unsigned long long*>(&s.rows), (unsigned long long)n);
    atomicMax(&s.most, most);
  }
  __syncthreads();
  // (offsets that do not ascend may make sequences that overlap, and more tiles than there is room for: none are listed.  Where rows
  // are no more than there are, tiles are none but a sequence's last more than rows / unit)
  const bool overlap = s.rows > (queries ? a.Tq : a.Tk);
  if (threadIdx.x == 0) plan.counts[queries ? 6 : 7] = overlap;
  if (overlap) {
    if (threadIdx.x == 0) {
      plan.counts[queries ? 0 : 1] = plan.counts[queries ? 4 : 5] = 0;
      if (!queries) plan.counts[2] = plan.counts[3] = 0;
    }
    return;
  }
  const int longest = c.heads ? part_steps(s.steps, sms, c) : 0x7fffffff;
  // (parts are of up to one and a half times `longest`; 9 bits for 512 classes)
  const int shift = max(0, 32 - __clz((int)min((long long)s.most, longest + longest / 2LL)) - 9);
  auto place = [&](int steps) { return steps == 0 ? kClasses - 1 : kClasses - 2 - min(steps >> shift, kClasses - 2); };
  auto cut = [&](const PackedTile& t) { return t.steps - longest > longest / 2 ? (t.steps + longest / 2) / longest : 1; };
  tiles.each(a, queries, unit, [&](const PackedTile& t) {
    const int parts = cut(t);
    atomicAdd(&s.first[place((t.steps + parts - 1) / parts)], parts);
  });
  __syncthreads();
  // exclusive sums of the classes, one a thread
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, own = s.first[threadIdx.x];
  int sum = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 31) s.warps[warp] = sum;
  __syncthreads();
  int before = sum - own, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += s.warps[w];
    all += s.warps[w];
  }
  s.first[threadIdx.x] = before;
  if (threadIdx.x == kClasses - 1) {  // (its class: tiles without a step)
    plan.counts[queries ? 0 : 1] = queries ? all : before;
    if (!queries) plan.counts[3] = own;
    plan.counts[queries ? 4 : 5] = 0;
  }
  __syncthreads();
  tiles.each(a, queries, unit, [&](PackedTile t) {
    const int steps = t.steps, parts = cut(t);
    if (parts > 1) {
      t.slot = atomicAdd(&s.slots, parts);
      if (!queries) plan.joins[atomicAdd(&s.joins, 1)] = PackedJoin{t.row, t.rows, t.slot, parts};
    }
    const int at = atomicAdd(&s.first[place((steps + parts - 1) / parts)], parts);
    t.parts = parts;
    for (int p = 0; p < parts; ++p) {
      t.part = p;
      t.begin = (int)((long long)steps * p / parts);
      t.steps = (int)((long long)steps * (p + 1) / parts) - t.begin;
      out[at + p] = t;
      ++t.slot;
    }
  });
  __syncthreads();
  if (threadIdx.x == 0 && !queries) plan.counts[2] = s.joins;
}

// Without lists (the kernels on CUDA cores look their tiles up): whether sequences overlap, by a block.
__device__ __forceinline__ void find_overlap(const PackedArgs& a, const PackedPlan& plan) {
  __shared__ unsigned long long rows[2];
  if (threadIdx.x < 2) rows[threadIdx.x] = 0;
  __syncthreads();
  long long q = 0, k = 0;
  for (int b = threadIdx.x; b < a.B; b += kThreads) {
    q += query_span(a, b).n;
    k += key_span(a, b).n;
  }
  atomicAdd(&rows[0], (unsigned long long)q);
  atomicAdd(&rows[1], (unsigned long long)k);
  __syncthreads();
  if (threadIdx.x == 0) {
    plan.counts[6] = (long long)rows[0] > a.Tq;
    plan.counts[7] = (long long)rows[1] > a.Tk;
  }
}

// delta: VEC values of 16 bytes at a time, `lanes` lanes a row (a power of two), two rows of a lane on their way.  NORMS: the largest
// |dO_i|^2 of queries that see a key and |V_j|^2 of keys of a sequence as well (those that are not finite have no say: theirs are the
// only rows that they reach).
template <class T, bool VEC, bool NORMS>
__device__ __forceinline__ void row_sums(const PackedArgs& a, const PackedPlan& plan, long long block, long long blocks, int lanes, const FastDiv& heads, const FastDiv& key_heads) {
  const int team = threadIdx.x / lanes, lane = threadIdx.x % lanes, teams = kThreads / lanes;
  const int ahead = (threadIdx.x & 31) / lanes;  // teams of the warp before this one
  const long long items = (long long)a.Tq * a.H;
  const T* o = static_cast<const T*>(a.o);
  const T* d_o = static_cast<const T*>(a.d_o);
  const T* rest = static_cast<const T*>(a.o_rest);
  constexpr int V = VEC ? kPer16<T> : 1, U = 2;
  const Span queries = NORMS ? clamped(packed_offset(a.offsets, a.wide, 0), packed_offset(a.offsets, a.wide, a.B), a.Tq) : Span{0, 0};
  float most_do = 0.f, most_v = 0.f;
  auto larger = [](float a, float b) { return b > a && b < INFINITY ? b : a; };
  // (the teams of a warp meet in shuffles: as long as the first of them has a row, all go on, the others with a row that
  // is there and nothing to store)
  for (long long i0 = block * teams * U + team; i0 - ahead < items; i0 += blocks * teams * U) {
    float s[U] = {}, sq[U] = {};
    long long to[U];
    float lse[U] = {};
    bool in[U] = {};
    const T* d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = i0 + (long long)u * teams;
      const long long t = i < items ? (items <= 0x7fffffffLL ? (long long)heads.div((uint32_t)i) : i / a.H) : 0;
      const int h = i < items ? (int)(i - t * a.H) : 0;
      d[u] = d_o + t * a.sdo[0] + (long long)h * a.sdo[1];
      to[u] = (long long)h * a.lse_ld + t;
      if constexpr (NORMS) {
        lse[u] = a.lse[to[u]];  // (compared when the rows are there: a branch around it would keep them waiting)
        in[u] = i < items && t >= queries.begin && t - queries.begin < queries.n;
      }
    }
    for (int x = lane * V; x < a.D; x += lanes * V) {
      if constexpr (VEC) {
        uint4 w[U], y[U], z[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const long long i = min(i0 + (long long)u * teams, items - 1);
          w[u] = *reinterpret_cast<const uint4*>(o + i * a.D + x);
          z[u] = *reinterpret_cast<const uint4*>(d[u] + x);
          y[u] = rest ? *reinterpret_cast<const uint4*>(rest + i * a.D + x) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[V], h[V], g[V];
          unpack16<T>(w[u], f);
          unpack16<T>(y[u], h);
          unpack16<T>(z[u], g);
#pragma unroll
          for (int e = 0; e < V; ++e) f[e] += h[e];
#pragma unroll
          for (int e = 0; e < V; ++e) s[u] = fmaf(f[e], g[e], s[u]);
          if constexpr (NORMS) {
#pragma unroll
            for (int e = 0; e < V; ++e) sq[u] = fmaf(g[e], g[e], sq[u]);
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const long long i = min(i0 + (long long)u * teams, items - 1);
          const float g = to_float(d[u][x]);
          s[u] = fmaf(to_float(o[i * a.D + x]) + (rest ? to_float(rest[i * a.D + x]) : 0.f), g, s[u]);
          if constexpr (NORMS) sq[u] = fmaf(g, g, sq[u]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      for (int m = lanes / 2; m > 0; m >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], m);
      if (lane == 0 && i0 + (long long)u * teams < items) a.delta[to[u]] = s[u];
      if constexpr (NORMS) {
        for (int m = lanes / 2; m > 0; m >>= 1) sq[u] += __shfl_xor_sync(0xffffffffu, sq[u], m);
        if (in[u] && lse[u] != -INFINITY) most_do = larger(most_do, sq[u]);
      }
    }
  }
  if constexpr (NORMS) {
    const T* v = static_cast<const T*>(a.v);
    // (keys of packed sequences lie one behind another, those in ranges anywhere: one after another, by all blocks)
    for (int b = 0; b < (a.ranges ? a.B : 1); ++b) {
      const Span keys = a.ranges ? key_span(a, b) : clamped(packed_offset(a.key_offsets, a.wide, 0), packed_offset(a.key_offsets, a.wide, a.B), a.Tk);
      const long long key_items = (long long)keys.n * a.Hk;
      // (the last blocks first: there may be some without rows of dO)
      for (long long i0 = (blocks - 1 - block) * teams * U + team; i0 - ahead < key_items; i0 += blocks * teams * U) {
        float sq[U] = {};
        const T* from[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const long long i = min(i0 + (long long)u * teams, key_items - 1);
          const long long t = key_items <= 0x7fffffffLL ? (long long)key_heads.div((uint32_t)i) : i / a.Hk;
          from[u] = v + (keys.begin + t) * a.sv[0] + (i - t * a.Hk) * a.sv[1];
        }
        for (int x = lane * V; x < a.D; x += lanes * V) {
          if constexpr (VEC) {
            uint4 w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = *reinterpret_cast<const uint4*>(from[u] + x);
#pragma unroll
            for (int u = 0; u < U; ++u) {
              float f[V];
              unpack16<T>(w[u], f);
#pragma unroll
              for (int e = 0; e < V; ++e) sq[u] = fmaf(f[e], f[e], sq[u]);
            }
          } else {
#pragma unroll
            for (int u = 0; u < U; ++u) sq[u] = fmaf(to_float(from[u][x]), to_float(from[u][x]), sq[u]);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          for (int m = lanes / 2; m > 0; m >>= 1) sq[u] += __shfl_xor_sync(0xffffffffu, sq[u], m);
          most_v = larger(most_v, sq[u]);
        }
      }
    }
    __shared__ uint32_t both[2][kThreads / 32];
    const uint32_t m0 = __reduce_max_sync(0xffffffffu, __float_as_uint(most_do)), m1 = __reduce_max_sync(0xffffffffu, __float_as_uint(most_v));
    if ((threadIdx.x & 31) == 0) { both[0][threadIdx.x >> 5] = m0; both[1][threadIdx.x >> 5] = m1; }
    __syncthreads();
    if (threadIdx.x < 32) {
      const uint32_t x = threadIdx.x < kThreads / 32 ? both[0][threadIdx.x] : 0, y = threadIdx.x < kThreads / 32 ? both[1][threadIdx.x] : 0;
      const float2 most = make_float2(__uint_as_float(__reduce_max_sync(0xffffffffu, x)), __uint_as_float(__reduce_max_sync(0xffffffffu, y)));
      if (threadIdx.x == 0) plan.norms[block] = most;
    }
  }
}

// Block 0 makes the list of queries, block 1 (or 0) that of keys, the others the row sums; without lists block 0 looks for overlaps.
template <class T, bool VEC, bool NORMS>
__global__ void __launch_bounds__(kThreads, 2) packed_prepare_kernel(const PackedArgs a, const PackedPlan plan, const int queries, const int unit, const int keys,
                                                                  const int sms, const PackedCut qcut, const PackedCut kcut, const int lanes, const FastDiv heads, const FastDiv key_heads) {
  __shared__ Sums s;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int lists = max(queries + keys, 1);
  if (queries + keys == 0 && blockIdx.x == 0) {
    find_overlap(a, plan);
  } else if ((int)blockIdx.x < lists) {
    const bool q = queries && blockIdx.x == 0;
    make_list(a, plan, q, q ? unit : kTileRows, sms, q ? qcut : kcut, s);
  } else {
    row_sums<T, VEC, NORMS>(a, plan, blockIdx.x - lists, gridDim.x - lists, lanes, heads, key_heads);
  }
}

}  // namespace

int launch_packed_prepare(int dtype, const PackedArgs& a, PackedPlan& plan, bool queries, int unit, bool keys, bool delta, cudaStream_t st, int* launches,
                          const PackedCut& qcut) {
  const int sms = sm_count();
  if (sms <= 0) return EVOATTN_ERR_CUDA;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = kPer16<T>;
    const bool norms = std::is_same<T, __half>::value && delta && keys;
    bool vec = delta && a.D % V == 0 && ((reinterpret_cast<uintptr_t>(a.o) | reinterpret_cast<uintptr_t>(a.o_rest) | reinterpret_cast<uintptr_t>(a.d_o)) & 15) == 0 && a.sdo[0] % V == 0 && a.sdo[1] % V == 0;
    if (norms) vec = vec && (reinterpret_cast<uintptr_t>(a.v) & 15) == 0 && a.sv[0] % V == 0 && a.sv[1] % V == 0;
    int lanes = 1;
    while (lanes < 32 && lanes * (vec ? V : 1) < a.D) lanes *= 2;
    // (with norms as many as are resident beside the lists' two: a block has three waits of its own then, 33 us with eight an SM and 27
    // so for [8192], 16 heads of 128)
    const long long each = kThreads / lanes * 2, most = norms ? 2LL * sms - 2 : (long long)sms * kSumBlocks;
    const long long rows = ((long long)a.Tq * a.H + each - 1) / each + (norms ? ((long long)a.Tk * a.Hk + each - 1) / each : 0);
    const int sums = delta ? (int)(rows < most ? rows : most) : 0, blocks = (queries && keys ? 2 : 1) + sums;
    plan.n_norms = norms ? sums : 0;
    auto kern = vec ? packed_prepare_kernel<T, true, false> : packed_prepare_kernel<T, false, false>;
    if constexpr (std::is_same<T, __half>::value)
      if (norms) kern = vec ? packed_prepare_kernel<T, true, true> : packed_prepare_kernel<T, false, true>;
    launch_dependent(kern, dim3((unsigned)blocks), kThreads, 0, st, a, plan, (int)queries, unit, (int)keys,
                     sms, qcut, key_cut(a), lanes, FastDiv((uint32_t)a.H), FastDiv((uint32_t)a.Hk));
    *launches += 1;
    return cudaGetLastError() == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
  });
}

}  // namespace evo
