// The lists of tiles that the tensor-core kernels of attention over packed sequences walk, made on the device, where the
// offsets are: a counting sort by the work of a tile, most first, so that what a persistent grid ends with is short.
#include "packed_sm100.cuh"

namespace evo {
namespace {

constexpr int kThreads = 1024, kClasses = 2048;  // tiles that meet more than kClasses others are of one class

// A warp per sequence, its lanes over the tiles.
template <class F>
__device__ __forceinline__ void each_tile(const PackedArgs& a, bool queries, int unit, F&& f) {
  for (int b = threadIdx.x >> 5; b < a.B; b += kThreads / 32) {
    const Span q = query_span(a, b), k = key_span(a, b);
    const int n = !queries ? k.n : q.n > a.few_tokens ? q.n : 0;
    for (int x = (threadIdx.x & 31) * unit; x < n; x += 32 * unit) {
      PackedTile t{};
      t.rows = min(unit, n - x);
      if (queries) {
        t.row = q.begin + x;
        t.other = k.begin;
        t.n = k.n;
        t.shift = x + k.n - q.n;
        t.tiles = (keys_seen(a, q.n, k.n, x, unit) + kTileRows - 1) / kTileRows;
      } else {
        t.row = k.begin + x;
        t.other = q.begin;
        t.n = q.n;
        t.shift = x + q.n - k.n;
        const int first = a.causal ? max(0, t.shift) : 0;  // the first query that sees a key of the tile
        t.tiles = first < q.n ? (q.n + kTileRows - 1) / kTileRows - first / kTileRows : 0;
      }
      f(t);
    }
  }
}

__global__ void __launch_bounds__(kThreads) packed_plan_kernel(const PackedArgs a, const PackedPlan plan, const int queries, const int unit, const int keys) {
  __shared__ int first[kClasses];
  __shared__ int sums[33];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  for (int list = 0; list < 2; ++list) {
    if (!(list == 0 ? queries : keys)) continue;
    const int u = list == 0 ? unit : kTileRows;
    PackedTile* out = list == 0 ? plan.queries : plan.keys;
    __syncthreads();
    for (int i = threadIdx.x; i < kClasses; i += kThreads) first[i] = 0;
    __syncthreads();
    auto place = [](const PackedTile& t) { return kClasses - 1 - min(t.tiles, kClasses - 1); };
    each_tile(a, list == 0, u, [&](const PackedTile& t) { atomicAdd(&first[place(t)], 1); });
    __syncthreads();
    // exclusive sums of the classes: two a thread
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int x0 = first[2 * threadIdx.x], x1 = first[2 * threadIdx.x + 1];
    int sum = x0 + x1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      int s = sums[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += up;
      }
      sums[lane] = s;
    }
    __syncthreads();
    const int before = sum - x0 - x1 + (warp ? sums[warp - 1] : 0);
    first[2 * threadIdx.x] = before;
    first[2 * threadIdx.x + 1] = before + x0;
    if (threadIdx.x == 0) plan.counts[list] = sums[31];
    __syncthreads();
    each_tile(a, list == 0, u, [&](const PackedTile& t) { out[atomicAdd(&first[place(t)], 1)] = t; });
  }
}

}  // namespace

int launch_packed_plan(const PackedArgs& a, const PackedPlan& plan, bool queries, int unit, bool keys, cudaStream_t st, int* launches) {
  launch_dependent(packed_plan_kernel, dim3(1), kThreads, 0, st, a, plan, (int)queries, unit, (int)keys);
  *launches += 1;
  return cudaGetLastError() == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

}  // namespace evo
