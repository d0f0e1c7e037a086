// What the tensor-core kernels of attention over packed sequences share: the list of their tiles, tensor maps of rows,
// and the shape of a staged tile.
#pragma once
#include <type_traits>

#include "packed.cuh"
#include "tmap.h"

namespace evo {

constexpr int kTileRows = 128;
constexpr float kLog2e = 1.4426950408889634f;

// A tile of queries with the keys that it meets, or of keys with the queries.
struct PackedTile {
  int row, rows;    // first row of the tile in its tensor, rows of the sequence from there on (at most the tile's)
  int other, n;     // first row of the sequence in the other tensor, its rows there
  int shift;        // position of the tile's first row as the other tensor counts: query i sees the keys up to i + shift,
                    // key j is seen by the queries from j + shift on
  int tiles;        // tiles of 128 rows of the other tensor that it meets: [0, tiles) of the keys; the last ones of the queries
  int pad[2];
};
static_assert(sizeof(PackedTile) == 32, "two 16-byte loads");

// Where lists lie in a workspace: 256 bytes with their lengths, then the tiles.
struct PackedPlan {
  int* counts;               // [0] query units, [1] key tiles
  PackedTile *queries, *keys;
};
inline long long query_units(const PackedArgs& a, int unit) { return a.Tq / unit + a.B; }
inline long long key_tiles(const PackedArgs& a) { return a.Tk / kTileRows + a.B; }
inline size_t plan_bytes(const PackedArgs& a, bool queries, int unit, bool keys) {
  const size_t n = (queries ? query_units(a, unit) : 0) + (keys ? key_tiles(a) : 0);
  return (256 + n * sizeof(PackedTile) + 255) / 256 * 256;
}
inline PackedPlan place_plan(const PackedArgs& a, void* ws, bool queries, int unit) {
  unsigned char* p = static_cast<unsigned char*>(ws);
  PackedTile* q = reinterpret_cast<PackedTile*>(p + 256);
  return PackedPlan{reinterpret_cast<int*>(p), q, q + (queries ? query_units(a, unit) : 0)};
}
// Writes the lists, those with the most work first (packed_plan.cu).
int launch_packed_plan(const PackedArgs& a, const PackedPlan& plan, bool queries, int unit, bool keys, cudaStream_t st, int* launches);

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

__device__ __forceinline__ PackedTile load_tile(const PackedTile* p) {
  const uint4 u = __ldcg(reinterpret_cast<const uint4*>(p)), w = __ldcg(reinterpret_cast<const uint4*>(p) + 1);
  return PackedTile{(int)u.x, (int)u.y, (int)u.z, (int)u.w, (int)w.x, (int)w.y, {0, 0}};
}
// The items of a CTA in turns that go back and forth over the CTAs, so that the last one to get a long item is the first
// to get a short one.
__device__ __forceinline__ int item_of(int turn) {
  return turn * (int)gridDim.x + (turn & 1 ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
}

}  // namespace evo
