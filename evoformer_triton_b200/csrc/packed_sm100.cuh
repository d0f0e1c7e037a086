// What the tensor-core kernels of attention over packed sequences share: the list of their tiles, tensor maps of rows,
// and the shape of a staged tile.
#pragma once
#include <type_traits>

#include "packed.cuh"
#include "tmap.h"

namespace evo {

constexpr int kTileRows = 128;
constexpr float kLog2e = 1.4426950408889634f;

// A tile of queries with the keys that it meets, or of keys (or a part of one) with the queries.
struct PackedTile {
  int row, rows;    // first row of the tile in its tensor, rows of the sequence from there on (at most the tile's)
  int other, n;     // first row of the sequence in the other tensor, its rows there
  int shift;        // position of the tile's first row as the other tensor counts: query i sees the keys up to i + shift,
                    // key j is seen by the queries from j + shift on
  int tiles;        // tiles of 128 rows of the other tensor that it meets: the first ones of the keys; the last ones of the queries
  int begin, steps; // of the steps of a key tile (the tiles of the group's heads, one after another) this part's
  int parts, part;  // parts of the tile, and which this is
  int slot;         // where it leaves its sums (those of part 0 lie `part` slots before)
  int blind;        // of key tiles: queries at the start of the sequence that see no key at all
};
static_assert(sizeof(PackedTile) == 48, "three 16-byte loads");
struct PackedJoin {
  int row, rows, slot, parts;
};

// Where lists lie in a workspace: 256 bytes with their lengths, the tiles, the key tiles whose parts are to be joined and the parts.
struct PackedPlan {
  int* counts;               // [0] query units, [1] key tiles and parts that have steps, [2] joins, [3] key tiles that no query sees, behind those;
                             // [4], [5] items that have been taken of the two lists; [6], [7] whether queries, and keys, of sequences overlap:
                             // then nothing is listed, and results are zeros
  PackedTile *queries, *keys;
  PackedJoin* joins;
  float* sums;               // key tiles: [slot][Hk][dV, dK][DP / 4][128 rows][4]; query units: [slot][units of heads][2 tiles][DP / 4][128][4]
  float4* ml;                // [slot][units of heads][2 tiles][128 rows]: reference, sum of P as rounded, and as it is
  int *arrived, n_arrived;   // [slot][units of heads][2 tiles]: parts that are through, of the tile whose first part has that slot
  float2* norms;             // fp16 backward: the largest |dO_i|^2 and |V_j|^2 that a block of the row sums has met
  int n_norms;
};
constexpr int kSumBlocks = 8;  // of the row sums an SM, at most
// What a list cuts: tiles of one and a half times as many steps and more as `part` hundredths of what an SM has to do, and as
// `least`; `heads` is how many of each there are on the list.
struct PackedCut {
  int part, least, heads;
};
// Steps of a part: a share of what an SM has to do, and no fewer than what a part costs by itself.
__host__ __device__ inline int part_steps(long long steps, int sms, const PackedCut& c) {
  const long long n = (steps * c.heads * c.part + 100LL * sms - 1) / (100LL * sms);
  return n < c.least ? c.least : n > 0x7fffffff ? 0x7fffffff : (int)n;
}
inline PackedCut key_cut(const PackedArgs& a) { return PackedCut{50, 4, a.Hk}; }
inline long long query_units(const PackedArgs& a, int unit) { return a.Tq / unit + a.B; }
inline long long key_tiles(const PackedArgs& a) { return a.Tk / kTileRows + a.B; }
// A tile of 3 n / 2 steps or more, n = part_steps(), makes at most steps / n + 1 / 2 < 2 steps / n parts, and all heads' steps are at most
// 100 sms n / part: so all heads' slots are fewer than 200 sms / part, and no more than `least` allows.  The same bounds what
// parts add to the list.
inline long long most_slots(long long tiles, long long steps, int sms, const PackedCut& c) {
  const long long each = (steps + c.least - 1) / c.least, all = tiles * each, most = (200LL * sms / c.part + c.heads - 1) / c.heads;
  return each < 2 ? 0 : all < most ? all : most;
}
inline long long key_slots(const PackedArgs& a, int sms) { return most_slots(key_tiles(a), (a.Tq / kTileRows + 1LL) * a.G, sms, key_cut(a)); }
inline long long query_slots(const PackedArgs& a, int unit, int sms, const PackedCut& c) { return most_slots(query_units(a, unit), a.Tk / kTileRows + 1LL, sms, c); }
inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }
struct PlanBytes {
  size_t queries, keys, joins, sums, ml, arrived, norms;
  size_t all() const { return 256 + queries + keys + joins + sums + ml + arrived + norms; }
};
// qcut.heads = 0: the query units are not cut.
inline PlanBytes plan_bytes(const PackedArgs& a, bool queries, int unit, bool keys, int sms, const PackedCut& qcut = PackedCut{100, 1, 0}) {
  const long long ks = keys ? key_slots(a, sms) : 0, qs = queries && qcut.heads ? query_slots(a, unit, sms, qcut) : 0;
  const size_t tile = (size_t)kTileRows * (a.D <= 64 ? 64 : 128) * sizeof(float), tiles = (size_t)qs * qcut.heads * 2;
  return PlanBytes{queries ? round256((query_units(a, unit) + qs) * sizeof(PackedTile)) : 0, keys ? round256((key_tiles(a) + ks) * sizeof(PackedTile)) : 0,
                   round256(ks * sizeof(PackedJoin)), round256(tile * (ks * a.Hk * 2 + tiles)), round256(tiles * kTileRows * sizeof(float4)), round256(tiles * sizeof(int)),
                   keys ? round256((size_t)sms * 2 * sizeof(float2)) : 0};
}
inline PackedPlan place_plan(const PackedArgs& a, int unit, void* ws, const PlanBytes& n) {
  unsigned char* p = static_cast<unsigned char*>(ws);
  PackedPlan plan{};
  plan.counts = reinterpret_cast<int*>(p);
  plan.queries = reinterpret_cast<PackedTile*>(p += 256);
  plan.keys = reinterpret_cast<PackedTile*>(p += n.queries);
  plan.joins = reinterpret_cast<PackedJoin*>(p += n.keys);
  plan.sums = reinterpret_cast<float*>(p += n.joins);
  plan.ml = reinterpret_cast<float4*>(p += n.sums);
  plan.arrived = reinterpret_cast<int*>(p += n.ml);
  plan.norms = reinterpret_cast<float2*>(p + n.arrived);
  plan.n_arrived = (int)(n.arrived / sizeof(int));
  return plan;
}
// Writes the lists, those with the most work first, and the row sums of dO * O (with both lists and fp16 the norms too, whose number
// it sets), in one launch (packed_plan.cu).
int launch_packed_prepare(int dtype, const PackedArgs& a, PackedPlan& plan, bool queries, int unit, bool keys, bool delta, cudaStream_t st, int* launches,
                          const PackedCut& qcut = PackedCut{100, 1, 0});

// [T][heads][D] rows of 16 bits as a 3-D map (D, T, heads) with boxes of 64 values (128 bytes, swizzled) by `rows`;
// values beyond D and rows beyond T read as zero.
bool make_packed_map(CUtensorMap* out, const void* base, const long long* stride, int T, int heads, int D, int rows = kTileRows);
// Whether such a map can be made (strides are in elements of 16 bits).
inline bool packed_map_ok(const void* base, const long long* stride, int T, int heads) {
  if (reinterpret_cast<uintptr_t>(base) & 15) return false;
  const long long most = 1LL << 38;
  const bool rows = T == 1 || (stride[0] > 0 && stride[0] % 8 == 0 && stride[0] < most);
  return rows && (heads == 1 || (stride[1] > 0 && stride[1] % 8 == 0 && stride[1] < most));
}

bool sm100_packed_supported(int dtype, const PackedArgs& a);
bool sm100_packed_bwd_supported(int dtype, const PackedArgs& a);
size_t sm100_packed_fwd_workspace_bytes(const PackedArgs& a);
int launch_sm100_packed_fwd(int dtype, const PackedArgs& a, void* workspace, cudaStream_t st, int* launches);
size_t sm100_packed_bwd_workspace_bytes(const PackedArgs& a);
int launch_sm100_packed_bwd(int dtype, const PackedArgs& a, void* workspace, cudaStream_t st, int* launches);

// Few query rows against many keys (packed_few.cu): sequences of up to a.few_tokens queries; `clear`: the rows of no sequence too.
size_t packed_few_workspace_bytes(const PackedArgs& a);
int launch_packed_few(int dtype, const PackedArgs& a, bool clear, void* workspace, cudaStream_t st, int* launches);

// 2^x of two values on the FMA pipes, for a part of the exponentials of a tile: the special-function units make 16 a cycle
// and SM, which is as long as the tile's MMAs take (head dimension 128) or twice that (64).  x = n + f with n whole (by
// adding and taking off 1.5 2^23) and |f| <= 1/2; 2^f by a polynomial whose largest relative error is the smallest there
// is for its degree (fitted by exchange): 7.5e-5 of degree 3, 2.6e-6 of degree 4, a fiftieth and a two-hundredth of half a step of bf16 and fp16;
// n is added to the exponent's bits.  Exponents below -126 count as that; with BOTH those above 126 too.  NaN makes the largest
// number there is (the sum of its bits), which no 16-bit type holds and no sum of exponentials reaches.
template <class T, bool BOTH>
__device__ __forceinline__ void exp2_fma(ptx::F2 x, float& p0, float& p1) {
  using namespace ptx;
  float x0, x1;
  f2_get(x, x0, x1);
  x0 = max_nan(x0, -126.f);
  x1 = max_nan(x1, -126.f);
  if constexpr (BOTH) {
    x0 = min_nan(x0, 126.f);
    x1 = min_nan(x1, 126.f);
  }
  x = f2_make(x0, x1);
  const F2 t = f2_add(x, f2_make(12582912.f, 12582912.f));
  const F2 f = f2_fma(f2_add(t, f2_make(-12582912.f, -12582912.f)), f2_make(-1.f, -1.f), x);
  F2 p;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    p = f2_fma(f, f2_make(0.055171669f, 0.055171669f), f2_make(0.24261112f, 0.24261112f));
    p = f2_fma(p, f, f2_make(0.69326099f, 0.69326099f));
    p = f2_fma(p, f, f2_make(0.99992807f, 0.99992807f));
  } else {
    p = f2_fma(f, f2_make(0.0095701019f, 0.0095701019f), f2_make(0.05591786f, 0.05591786f));
    p = f2_fma(p, f, f2_make(0.24024745f, 0.24024745f));
    p = f2_fma(p, f, f2_make(0.69312181f, 0.69312181f));
    p = f2_fma(p, f, f2_make(0.99999926f, 0.99999926f));
  }
  float t0, t1;
  f2_get(t, t0, t1);
  f2_get(p, p0, p1);
  p0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
  p1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}

// DP columns of an accumulator, times f, as 16-bit values to the rows of a warp: lane i has row i, of which the first `rows`
// are stored, at out + i ld and, as the map has it, at (row0, head); zeros where `any` is not set.  By way of 4 KB of
// shared memory a warp, 64 columns at a time, which leave by one TMA store where all 32 rows are the sequence's (what is
// behind it belongs to the next one).  An SM takes more than a microsecond to get rid of a 128 x 128 tile: as plain stores
// that is waited for at the end of every item (2.0 us from the lanes, 1.6 by way of shared memory).
constexpr int kStageBytes = 32 * 128;
// REST: what rounding leaves of them instead.
template <class T, int DP, bool REST = false>
__device__ __forceinline__ void store_rows_staged(uint32_t stage_s, uint32_t t_src, const CUtensorMap* map, int row0, int head, T* out, long long ld, int rows, int D,
                                                  float f, bool any) {
  using namespace ptx;
  const int lane = threadIdx.x & 31;
  const bool whole = rows >= 32;
#pragma unroll 1
  for (int c0 = 0; c0 < DP; c0 += 32) {
    const int half = (c0 >> 5) & 1;
    uint32_t r[32];
    if (any) {
      tmem_ld32(t_src + c0, r);
      tmem_wait_ld();
    }
    if (half == 0) {
      if (lane == 0) tma_wait_group_read0();
      __syncwarp();  // (what the stage held before has been read)
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float x0 = __uint_as_float(r[8 * i + 2 * u]) * f, x1 = __uint_as_float(r[8 * i + 2 * u + 1]) * f;
        p[u] = Pack2<T>::pack(x0, x1);
        if constexpr (REST) {
          float y0, y1;
          unpack2<T>(p[u], y0, y1);
          p[u] = Pack2<T>::pack(x0 - y0, x1 - y1);
        }
        if (!any) p[u] = 0u;
      }
      sts_v4(stage_s + lane * 128 + (((4 * half + i) ^ (lane & 7)) << 4), p[0], p[1], p[2], p[3]);
    }
    if (half == 0) continue;
    if (whole) {
      fence_async_shared();
      __syncwarp();
      if (lane == 0) {
        tma_store_3d_s(map, stage_s, c0 - 32, row0, head);
        tma_commit_group();
      }
      continue;
    }
    __syncwarp();
    const int c = lane & 7, d = c0 - 32 + 8 * c;
#pragma unroll 1
    for (int i = lane >> 3; i < rows; i += 4)
      if (d < D) *reinterpret_cast<uint4*>(out + i * ld + d) = lds_v4(stage_s + i * 128 + ((c ^ (i & 7)) << 4));
    __syncwarp();
  }
}
// What the stores of a warp still read or write, at the end of a kernel.
__device__ __forceinline__ void stores_done() {
  if ((threadIdx.x & 31) == 0) ptx::tma_wait_group0();
  __syncwarp();
}

__device__ __forceinline__ PackedTile load_tile(const PackedTile* p) {
  const uint4* x = reinterpret_cast<const uint4*>(p);
  const uint4 u = __ldcg(x), v = __ldcg(x + 1), w = __ldcg(x + 2);
  return PackedTile{(int)u.x, (int)u.y, (int)u.z, (int)u.w, (int)v.x, (int)v.y, (int)v.z, (int)v.w, (int)w.x, (int)w.y, (int)w.z, (int)w.w};
}
// Which item a CTA works on next: the first is its own, the others it takes from a counter, the most work first as the list
// has them.  The warp that loads takes one when it has asked for all tiles of the item before (no sooner: who has the
// longest item should not have the next as well), and hands it to the other warps by way of two words of shared memory.
struct Schedule {
  uint32_t full, empty, words;  // shared addresses: two barriers each (empty: of all other warps that work on items), two words
  uint32_t abort_s;
  int* counter;
  int n_items;
  uint32_t n = 0;
  __device__ __forceinline__ int first() const { return (int)blockIdx.x; }
  __device__ __forceinline__ bool over(int idx) const { return idx >= n_items; }
  __device__ __forceinline__ int take() {  // the warp that loads
    int idx = 0;
    if ((threadIdx.x & 31) == 0) idx = (int)gridDim.x + atomicAdd(counter, 1);
    idx = __shfl_sync(0xffffffffu, idx, 0);
    const uint32_t at = n & 1;
    ptx::mbar_wait_s(empty + 8 * at, ((n >> 1) & 1) ^ 1, abort_s, DEV_TIMEOUT_SYNC);
    if ((threadIdx.x & 31) == 0) {
      ptx::sts_u32(words + 4 * at, (uint32_t)idx);
      ptx::mbar_arrive_s(full + 8 * at);
    }
    __syncwarp();
    ++n;
    return stopped() ? n_items : idx;
  }
  __device__ __forceinline__ int next() {  // the others
    const uint32_t at = n & 1;
    ptx::mbar_wait_s(full + 8 * at, (n >> 1) & 1, abort_s, DEV_TIMEOUT_SYNC);
    const int idx = (int)ptx::lds_u32(words + 4 * at);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) ptx::mbar_arrive_s(empty + 8 * at);
    ++n;
    return stopped() ? n_items : idx;
  }
  // (a wait that gave up hands on no item)
  __device__ __forceinline__ bool stopped() const { return __any_sync(0xffffffffu, ptx::lds_u32(abort_s) != 0); }
};

}  // namespace evo
