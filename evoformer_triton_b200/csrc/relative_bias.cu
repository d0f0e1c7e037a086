// Learned relative position bias by buckets, forward and backward.
//
//   out[b,h,i,j] = table[row(k_j - q_i), h] (+ base[b,h,i,j]),   dtable[r,h] = sum of d_out over (b,i,j) with row r
//
// Memory bound both ways: one write (and one read of the base) of B H Rq Rk values, one read of them.  A warp
// walks rows of a strip of keys whose positions stay in registers, so the bucket of a score is worked out
// once for all heads (forward), or not at all where a whole strip falls into one bucket, as it does away from
// the diagonal.  [2,16,2048,2048] bf16, 32 logarithmic buckets: forward 47 us (5.7 TB/s), backward 82 (3.3 TB/s; its items
// without their data are 27 of them: positions to read, buckets to find).  Far from memory's time: tables of more than 128 rows in the
// backward (a pass per 128: [1,16,2048,2048] bf16, 601 rows, 193 us for 20), rows of the gradient off 16 bytes
// ([1,8,2047,2047] bf16 43 us for 10) and an added bias forward ([1,8,2048,2048] bf16 39 us for 20).
#include <string.h>

#include "inputs.cuh"

namespace evo {
namespace {

constexpr int kLogEdges = EVOATTN_MAX_BUCKET_EDGES;

struct RelArgs {
  int B, H, Rq, Rk;
  int buckets, scheme, exact, n_edges;
  int positions64, table_dtype, base_dtype;
  const void* table;
  const void* q_pos;
  const void* k_pos;
  long long sq, sk;
  const void* base;
  Str3 sbase;
  void* out;
  Str3 sout;
  // backward
  float* partial;     // [H][blocks][buckets]
  void* dtable;
  int blocks;         // per head
  int item_rows;      // rows a warp takes at a time
  int window;         // table rows a block keeps sums of
  int edges[kLogEdges];
};

__device__ __forceinline__ long long position(const void* p, bool wide, long long i) {
  return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

constexpr int kNear = 1024;               // differences up to here are looked up
constexpr int kFarthest = 1 << 28;        // no edge lies beyond

// Positions are 64-bit; differences beyond +-2^30 are all the same to a bucket.
__device__ __forceinline__ int difference(long long key, long long query) {
  const long long d = key - query;
  return (int)max(-(1ll << 30), min(1ll << 30, d));
}

// The table's row for a key `rel` ahead of the query.
__device__ __forceinline__ int bucket_row(const RelArgs& a, int rel) {
  const bool ahead = rel > 0;
  const int d = ahead ? rel : -rel;
  if (a.scheme == EVOATTN_BUCKETS_CLIP) {
    const int f = min(d, a.exact);
    return ahead ? a.exact - f : a.exact + f;
  }
  if (a.scheme == EVOATTN_BUCKETS_LOG_CAUSAL && ahead) return 0;
  int f = d;
  if (d >= a.exact) {
    int lo = 0, hi = a.n_edges;  // the number of edges that are <= d
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.edges[mid] <= d) lo = mid + 1;
      else hi = mid;
    }
    f = a.exact + lo;
  }
  return ahead ? (a.buckets >> 1) + f : f;
}

// The same looked up, as MAP puts it: differences beyond `far` have the bucket of `far`.  Edges beyond kNear are searched.
template <class MAP>
struct Buckets {
  const RelArgs& a;
  const uint16_t* near;  // shared memory, [2 far + 1]
  int far;               // 0: not looked up
  __device__ __forceinline__ Buckets(const RelArgs& args, uint16_t* sm_near) : a(args), near(sm_near) {
    const int last = a.scheme == EVOATTN_BUCKETS_CLIP ? a.exact : a.n_edges ? a.edges[a.n_edges - 1] : a.exact;
    far = last <= kNear ? max(last, 1) : 0;
    if (far)
      for (int i = threadIdx.x; i < 2 * far + 1; i += blockDim.x) sm_near[i] = (uint16_t)MAP::of(bucket_row(a, i - far));
  }  // (the caller synchronises)
  __device__ __forceinline__ int operator()(int rel) const {
    return far ? near[min(max(rel, -far), far) + far] : MAP::of(bucket_row(a, rel));
  }
};

// The keys of a strip of L V keys that L lanes hold, V each: consecutive ones (WIDE), or L apart; other lanes of the warp
// hold the same.  Positions are kept relative to the least one of the strip, in 32 bits: where they span 2^29 or more, which
// no sequence does, they are read again for every row.  least - query clamped to +-2^30 plus an offset below 2^29 is on
// the right side of every edge.
template <int V, int L, bool WIDE>
struct Strip {
  int j0, off[V];
  long long least, most;         // where near_together
  bool near_together, in_order;  // in_order: every lane's keys ascend, so those of one bucket are next to each other
  __device__ __forceinline__ int col(int u) const { return WIDE ? j0 + (threadIdx.x & (L - 1)) * V + u : j0 + u * L + (threadIdx.x & (L - 1)); }
  __device__ __forceinline__ void load(const RelArgs& a, int b, int first) {
    j0 = first;
    const long long at = b * a.sk, origin = position(a.k_pos, a.positions64, at + first);
    int lo = 0, hi = 0;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      off[u] = col(u) < a.Rk ? difference(position(a.k_pos, a.positions64, at + col(u)), origin) : 0x7fffffff;
      lo = min(lo, off[u]);
      if (off[u] != 0x7fffffff) hi = max(hi, off[u]);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    near_together = (long long)hi - lo < 1 << 29;  // (one that was clamped is too far from the origin, which is at 0)
    least = origin + lo;
    most = origin + hi;
    bool ascending = near_together;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      off[u] = (off[u] == 0x7fffffff ? hi : off[u]) - lo;
      ascending = ascending && (u == 0 || off[u] >= off[u ? u - 1 : 0]);
    }
    in_order = __all_sync(0xffffffffu, ascending);
  }
  // The rows of the table for the query at q, from = difference(least, q).
  template <class MAP>
  __device__ __forceinline__ void rows(const RelArgs& a, const Buckets<MAP>& bucket, int b, long long q, int from, int (&r)[V]) const {
    if (near_together && bucket.far) {
      from += bucket.far;
#pragma unroll
      for (int u = 0; u < V; ++u) r[u] = bucket.near[min(max(from + off[u], 0), 2 * bucket.far)];
    } else {
      // A place without a key has the row of the lane's key before it: equal rows of keys in order stay next to each other.
      int row = 0;
      for (int u = 0; u < V; ++u) {
        const int c = WIDE ? j0 + (int)(threadIdx.x & (L - 1)) * V + u : j0 + u * L + (int)(threadIdx.x & (L - 1));
        if (c < a.Rk) row = bucket(difference(position(a.k_pos, a.positions64, b * a.sk + c), q));
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (k == u) r[k] = row;
      }
    }
  }
};

// Heads that a block of the forward holds the table of: the work on a row's buckets is shared by as many.
constexpr int kHeads = 8;
// A row of the table in shared memory.  Lanes read rows that lie V = 4 or 8 apart (consecutive keys): one
// float of padding every eight rows keeps them in different banks.
__host__ __device__ constexpr int slot(int row) { return row + (row >> 3); }
struct Slot { static __device__ __forceinline__ int of(int row) { return slot(row); } };
struct Same { static __device__ __forceinline__ int of(int row) { return row; } };

// V values of the base, in pieces of up to 16 bytes.
template <int V>
__device__ __forceinline__ void add_base(const RelArgs& a, long long at, float (&v)[V]) {
  if (a.base_dtype == EVOATTN_FP32) {
    const float* p = static_cast<const float*>(a.base) + at;
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
      const float4 w = *reinterpret_cast<const float4*>(p + 4 * k);
      v[4 * k] += w.x; v[4 * k + 1] += w.y; v[4 * k + 2] += w.z; v[4 * k + 3] += w.w;
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(a.base) + at;
    uint32_t w[V / 2];
    if constexpr (V == 8) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      float lo, hi;
      if (a.base_dtype == EVOATTN_BF16) unpack2<__nv_bfloat16>(w[k], lo, hi);
      else unpack2<__half>(w[k], lo, hi);
      v[2 * k] += lo;
      v[2 * k + 1] += hi;
    }
  }
}

template <class T> __device__ __forceinline__ uint32_t same2(float v) {  // a 16-bit value twice
  if constexpr (sizeof(T) == 2) return Pack2<T>::pack(v, v);
  return 0;
}

// A block of eight warps takes a strip of 32 V keys and kHeads heads and walks rows; with fewer rows than warps, the warps
// share the heads of a row.  A row whose strip is one bucket, as away from the diagonal, is one value a head.
template <class T, bool WIDE, bool BASE>
__global__ void __launch_bounds__(256, 4) relative_fwd(RelArgs a, int rows_per_block, int row_warps) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int V = kPer16<T>;
  extern __shared__ float sm_table[];  // [kHeads][slot(buckets)]
  __shared__ uint16_t sm_near[2 * kNear + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = (a.H + kHeads - 1) / kHeads;
  const int b = blockIdx.z / groups, h0 = (blockIdx.z - b * groups) * kHeads, nh = min(kHeads, a.H - h0);
  const int pitch = slot(a.buckets) + 1;
  Strip<V, 32, WIDE> strip;
  strip.load(a, b, blockIdx.x * 32 * V);
  // lane l: the warp's l-th row (at most 32 of them)
  const int i0 = blockIdx.y * rows_per_block + warp % row_warps, i_end = (int)min((long long)a.Rq, ((long long)blockIdx.y + 1) * rows_per_block);
  const int my_i = i0 + lane * row_warps;
  const long long my_q = my_i < i_end ? position(a.q_pos, a.positions64, b * a.sq + my_i) : 0;
  const Buckets<Slot> bucket(a, sm_near);
  for (int i = threadIdx.x; i < a.buckets * nh; i += 256) {
    const int r = i / nh, h = i - r * nh;
    sm_table[h * pitch + slot(r)] = load_any(a.table, a.table_dtype, (long long)r * a.H + h0 + h);
  }
  __syncthreads();
  const int lo = bucket(difference(strip.least, my_q)), hi = bucket(difference(strip.most, my_q));
  const int my_kind = strip.near_together && lo == hi ? lo : -1;  // (rows are in the order of distances on either side, so all between are the same)
  const int first_head = warp / row_warps, head_step = 8 / row_warps;
  for (int k = 0, i = i0; i < i_end; ++k, i += row_warps) {
    const int kind = __shfl_sync(0xffffffffu, my_kind, k);
    const long long q = __shfl_sync(0xffffffffu, my_q, k);
    int s[V];
    if (kind < 0) {
      strip.rows(a, bucket, b, q, difference(strip.least, q), s);
    }
    T* o = static_cast<T*>(a.out) + b * a.sout.a + (h0 + first_head) * a.sout.b + (long long)i * a.sout.c;
    const long long down = head_step * a.sout.b;
    const float* t = sm_table + first_head * pitch;
    const int down_t = head_step * pitch;
    const bool whole = WIDE && strip.col(V - 1) < a.Rk;
    if constexpr (!BASE) {
      if (whole) {  // the common cases: a row is one value a head, or V of them
        o += strip.col(0);
        if (kind >= 0) {
          t += kind;
          for (int h = first_head; h < nh; h += head_step, o += down, t += down_t) {
            const uint32_t w = sizeof(T) == 4 ? __float_as_uint(*t) : same2<T>(*t);
            *reinterpret_cast<uint4*>(o) = make_uint4(w, w, w, w);
          }
        } else {
          for (int h = first_head; h < nh; h += head_step, o += down, t += down_t) {
            float v[V];
#pragma unroll
            for (int u = 0; u < V; ++u) v[u] = t[s[u]];
            *reinterpret_cast<uint4*>(o) = pack16<T>(v);
          }
        }
        continue;
      }
    }
    long long at = b * a.sbase.a + (h0 + first_head) * a.sbase.b + (long long)i * a.sbase.c;
    for (int h = first_head; h < nh; h += head_step, o += down, t += down_t, at += head_step * a.sbase.b) {
      float v[V];
      if (kind >= 0) {
        v[0] = t[kind];
#pragma unroll
        for (int u = 1; u < V; ++u) v[u] = v[0];
      } else {
#pragma unroll
        for (int u = 0; u < V; ++u) v[u] = t[s[u]];
      }
      if (BASE && whole) {  // (WIDE: the base's rows are whole pieces too)
        add_base<V>(a, at + strip.col(0), v);
        *reinterpret_cast<uint4*>(o + strip.col(0)) = pack16<T>(v);
        continue;
      }
      if constexpr (BASE) {
        uint32_t w[V];
        if (a.base_dtype == EVOATTN_FP32) {
#pragma unroll
          for (int u = 0; u < V; ++u) w[u] = strip.col(u) < a.Rk ? static_cast<const uint32_t*>(a.base)[at + strip.col(u)] : 0;
        } else {
#pragma unroll
          for (int u = 0; u < V; ++u) w[u] = strip.col(u) < a.Rk ? static_cast<const uint16_t*>(a.base)[at + strip.col(u)] : 0;
        }
#pragma unroll
        for (int u = 0; u < V; ++u)
          v[u] += a.base_dtype == EVOATTN_FP32 ? __uint_as_float(w[u])
                  : a.base_dtype == EVOATTN_BF16 ? __uint_as_float(w[u] << 16) : __half2float(__ushort_as_half((unsigned short)w[u]));
      }
#pragma unroll
      for (int u = 0; u < V; ++u)
        if (strip.col(u) < a.Rk) o[strip.col(u)] = from_float<T>(v[u]);
    }
  }
}

// Backward: a warp takes item_rows rows of a strip of keys of one (b, h) at a time and adds every value to the sum of its
// bucket.  Every lane has sums of its own (no two lanes add to one address, and the order of the additions is fixed).  A
// load is 64 keys of 4 rows (fp32: 2), whole cache lines of each: as near to a square as those go, so that few loads lie across the
// diagonal; the others are one bucket and are added up in a register.  A block keeps the sums of `window` table rows
// (blockIdx.z says which); loads that cannot touch them are left out.  Loads of one row of 256 keys took 196 us where these take
// 82 ([2,16,2048,2048] bf16, graph replay); fp32 loads of 32 keys by 4 rows 88 where 64 by 2 take 74 ([1,16,2048,2048]).
template <class T> constexpr int kLanes = 64 / kPer16<T>;
template <class T> constexpr int kTall = 32 / kLanes<T>;
constexpr int kLoads = 16;  // of an item, at most (8: 110 us, 32: as fast, but clipped buckets 54 us for 50)

template <class T, bool WIDE>
struct RowPiece {  // V values of a row
  static constexpr int V = kPer16<T>;
  uint4 w;
  T e[V];
  __device__ __forceinline__ void load(const RelArgs& a, const Strip<V, kLanes<T>, WIDE>& strip, const T* row) {
    if (WIDE && strip.col(V - 1) < a.Rk) {
      w = *reinterpret_cast<const uint4*>(row + strip.col(0));
    } else {
#pragma unroll
      for (int u = 0; u < V; ++u) e[u] = strip.col(u) < a.Rk ? row[strip.col(u)] : from_float<T>(0.f);
      if constexpr (WIDE) memcpy(&w, e, 16);
    }
  }
  __device__ __forceinline__ void clear() {
    w = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < V; ++u) e[u] = from_float<T>(0.f);
  }
  __device__ __forceinline__ void floats(float (&v)[V]) const {
    if constexpr (WIDE) unpack16<T>(w, v);
    else {
#pragma unroll
      for (int u = 0; u < V; ++u) v[u] = to_float<T>(e[u]);
    }
  }
  __device__ __forceinline__ float sum() const {
    float v[V];
    floats(v);
#pragma unroll
    for (int n = V / 2; n > 0; n /= 2)
#pragma unroll
      for (int u = 0; u < n; ++u) v[u] += v[u + n];
    return v[0];
  }
};

template <class T, bool WIDE>
__global__ void __launch_bounds__(128, 5) relative_bwd(RelArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int V = kPer16<T>, L = kLanes<T>, TALL = kTall<T>, U = WIDE ? 8 : 4;  // U: loads on the way at once
  extern __shared__ float sm_sums[];  // [4 warps][window + 1][32 lanes]
  __shared__ uint16_t sm_near[2 * kNear + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, my_row = lane / L;
  const int h = blockIdx.y, first = blockIdx.z * a.window, count = min(a.window, a.buckets - first);
  const Buckets<Same> bucket(a, sm_near);
  const int per_warp = (a.window + 1) * 32;  // (one more row, for what is not of this block's)
  for (int i = threadIdx.x; i < 4 * per_warp; i += 128) sm_sums[i] = 0.f;
  __syncthreads();
  float* sums = sm_sums + warp * per_warp + lane;
  const unsigned strips = (a.Rk + L * V - 1) / (L * V), chunks = (a.Rq + a.item_rows - 1) / a.item_rows;
  const unsigned items = a.B * strips * chunks;
  // What all scores of keys least .. most and queries q0 .. q1 have in common: their bucket (>= 0), that none is of this
  // block's (-2), or nothing (-1).  Between the buckets of the two ends are those of all others, but for LOG, whose
  // upper half begins behind the query.
  const auto kind_of = [&](long long least, long long most, long long q0, long long q1) {
    const int from = difference(least, q1), to = difference(most, q0);
    const int lo = bucket(from), hi = bucket(to);
    const bool ordered = a.scheme != EVOATTN_BUCKETS_LOG || from > 0 || to <= 0;
    return ordered && (max(lo, hi) < first || min(lo, hi) >= first + count) ? -2 : lo == hi ? lo : -1;
  };
  for (unsigned item = blockIdx.x * 4 + warp; item < items; item += gridDim.x * 4) {
    const unsigned rest = item / chunks, b = rest / strips;
    const int i0 = (int)(item - rest * chunks) * a.item_rows, ni = min(a.item_rows, a.Rq - i0), loads = (ni + TALL - 1) / TALL;
    Strip<V, L, WIDE> strip;
    strip.load(a, b, (int)(rest - b * strips) * L * V);
    const long long q_at = b * a.sq + i0, q_origin = position(a.q_pos, a.positions64, q_at);
    int q0 = 0x7fffffff, q1 = -q0;  // relative to q_origin, over the rows of load `lane`
#pragma unroll
    for (int k = 0; k < TALL; ++k) {  // (rows behind the last: the last one, which changes no least or greatest)
      const int q = difference(position(a.q_pos, a.positions64, q_at + min(lane * TALL + k, ni - 1)), q_origin);
      q0 = min(q0, q);
      q1 = max(q1, q);
    }
    const T* d = static_cast<const T*>(a.out) + b * a.sout.a + h * a.sout.b + (long long)(i0 + my_row) * a.sout.c;
    const long long down = TALL * a.sout.c;
    const int all0 = __reduce_min_sync(0xffffffffu, q0), all1 = __reduce_max_sync(0xffffffffu, q1);
    // (positions that span 2^29 or more are looked at one by one)
    const bool can_tell = strip.near_together && (long long)all1 - all0 < 1 << 29;
    const int kind = can_tell ? kind_of(strip.least, strip.most, q_origin + all0, q_origin + all1) : -1;
    if (kind == -2) continue;
    if (kind >= 0) {  // one bucket altogether
      float acc = 0.f;
      int l = 0;
      for (; (l + U) * TALL <= ni; l += U) {
        RowPiece<T, WIDE> p[U];
#pragma unroll
        for (int k = 0; k < U; ++k, d += down) p[k].load(a, strip, d);
#pragma unroll
        for (int k = 0; k < U; ++k) acc += p[k].sum();
      }
      for (; l * TALL + my_row < ni; ++l, d += down) {
        RowPiece<T, WIDE> p;
        p.load(a, strip, d);
        acc += p.sum();
      }
      sums[(kind - first) * 32] += acc;
      continue;
    }
    // Load by load: the lines are asked for first, since there is room for no more than the next load in registers.
    const int my_kind = lane >= loads ? -2 : can_tell ? kind_of(strip.least, strip.most, q_origin + q0, q_origin + q1) : -1;
    for (int l = 0; l < loads; ++l)
      if (lane % L == 0 && l * TALL + my_row < ni) ptx::prefetch_l2(d + l * down + strip.col(0));
    RowPiece<T, WIDE> next;
    long long next_q = 0;
    const auto fetch = [&](int l) {
      const int i = l * TALL + my_row;
      if (i < ni) {
        next.load(a, strip, d + l * down);
        next_q = position(a.q_pos, a.positions64, q_at + i);
      } else {
        next.clear();
      }
    };
    float acc = 0.f;
    int acc_row = -1;
    fetch(0);
#pragma unroll 1
    for (int l = 0; l < loads; ++l) {
      const int of_load = __shfl_sync(0xffffffffu, my_kind, l);
      const RowPiece<T, WIDE> now = next;
      const long long q = next_q;
      if (l + 1 < loads) fetch(l + 1);
      if (of_load >= 0) {
        if (of_load != acc_row) {
          if (acc_row >= 0) sums[(acc_row - first) * 32] += acc;
          acc_row = of_load;
          acc = 0.f;
        }
        acc += now.sum();
      } else if (of_load == -1) {
        float v[V];
        int r[V];
        now.floats(v);
        strip.rows(a, bucket, b, q, difference(strip.least, q), r);
#pragma unroll
        for (int u = 0; u < V; ++u) r[u] = (int)min((unsigned)(r[u] - first), (unsigned)count) * 32;
        if (strip.in_order) {  // values of one bucket first, then all sums at once
          bool last[V];
          float old[V];
#pragma unroll
          for (int u = 0; u < V; ++u) {
            last[u] = u == V - 1 || r[u + 1 < V ? u + 1 : u] != r[u];
            if (!last[u]) v[u + 1 < V ? u + 1 : u] += v[u];
          }
#pragma unroll
          for (int u = 0; u < V; ++u) old[u] = last[u] ? sums[r[u]] : 0.f;
#pragma unroll
          for (int u = 0; u < V; ++u)
            if (last[u]) sums[r[u]] = old[u] + v[u];
        } else {
#pragma unroll
          for (int u = 0; u < V; ++u) sums[r[u]] += v[u];  // (where there is no key: zero)
        }
      }
    }
    if (acc_row >= 0) sums[(acc_row - first) * 32] += acc;
  }
  __syncthreads();
  for (int r = warp; r < count; r += 4) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) s += sm_sums[w * per_warp + r * 32 + lane];
    s = warp_sum(s);
    if (lane == 0) a.partial[((long long)h * a.blocks + blockIdx.x) * a.buckets + first + r] = s;
  }
}

// The blocks' sums of a head, added in order: 32 table rows a block, 32 shares of the sums.
__global__ void __launch_bounds__(1024) relative_sum_partials(RelArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  __shared__ float sm[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, r = blockIdx.x * 32 + lane, h = blockIdx.y;
  float s = 0.f;
  if (r < a.buckets) {
#pragma unroll 8
    for (int k = part; k < a.blocks; k += 32) s += a.partial[((long long)h * a.blocks + k) * a.buckets + r];
  }
  sm[part][lane] = s;
  __syncthreads();
  s = warp_sum(sm[lane][part]);  // (a warp a table row)
  const int out = blockIdx.x * 32 + part;
  if (lane == 0 && out < a.buckets) store_any(a.dtable, a.table_dtype, (long long)out * a.H + h, s);
}

int validate(const evoattn_relative_bias_params* p) {
  if (!p) return EVOATTN_ERR_NULL;
  if (!known_dtype(p->dtype) || !known_dtype(p->table_dtype) || (p->base && !known_dtype(p->base_dtype))) return EVOATTN_ERR_DTYPE;
  if (p->B < 0 || p->H <= 0 || p->Rq < 0 || p->Rk < 0 || p->B > 65535 || p->H > 4096) return EVOATTN_ERR_SHAPE;
  if (p->Rq > (1 << 23) || p->Rk > (1 << 23)) return EVOATTN_ERR_SHAPE;
  if ((long long)p->B * ((p->H + kHeads - 1) / kHeads) > 65535) return EVOATTN_ERR_SHAPE;
  if ((long long)p->B * ((p->Rk + 63) / 64) * ((p->Rq + 7) / 8) > 0x7fffffffLL) return EVOATTN_ERR_SHAPE;
  if (p->buckets <= 0 || p->buckets > EVOATTN_MAX_BUCKETS || p->n_edges < 0 || p->n_edges > kLogEdges || p->exact < 0) return EVOATTN_ERR_SHAPE;
  if (p->n_edges > 0 && !p->edges) return EVOATTN_ERR_NULL;
  for (int i = 0; i < p->n_edges; ++i)  // a distance finds its bucket by bisection
    if (p->edges[i] < p->exact || p->edges[i] > kFarthest || (i && p->edges[i] < p->edges[i - 1])) return EVOATTN_ERR_SHAPE;
  const int most = p->exact + p->n_edges;  // the largest f
  switch (p->scheme) {
    case EVOATTN_BUCKETS_CLIP: return p->n_edges == 0 && p->buckets == 2 * p->exact + 1 ? EVOATTN_OK : EVOATTN_ERR_SHAPE;
    case EVOATTN_BUCKETS_LOG: return p->buckets % 2 == 0 && most < p->buckets / 2 ? EVOATTN_OK : EVOATTN_ERR_SHAPE;
    case EVOATTN_BUCKETS_LOG_CAUSAL: return most < p->buckets ? EVOATTN_OK : EVOATTN_ERR_SHAPE;
    default: return EVOATTN_ERR_SHAPE;
  }
}

RelArgs args_of(const evoattn_relative_bias_params* p) {
  RelArgs a{};
  a.B = p->B; a.H = p->H; a.Rq = p->Rq; a.Rk = p->Rk;
  a.buckets = p->buckets; a.scheme = p->scheme; a.exact = p->exact; a.n_edges = p->n_edges;
  a.positions64 = p->positions64; a.table_dtype = p->table_dtype; a.base_dtype = p->base_dtype;
  a.table = p->table; a.q_pos = p->q_pos; a.k_pos = p->k_pos; a.sq = p->q_pos_stride; a.sk = p->k_pos_stride;
  for (int i = 0; i < p->n_edges; ++i) a.edges[i] = p->edges[i];
  return a;
}

bool rows_of_16_bytes(const void* p, const int64_t* stride, int es) {
  return ((uintptr_t)p & 15) == 0 && stride[0] * es % 16 == 0 && stride[1] * es % 16 == 0 && stride[2] * es % 16 == 0;
}

// How the backward is cut: rows a warp takes at a time, blocks of four warps a head, table rows a block sums.
void plan_bwd(RelArgs* a, int es) {
  a->window = a->buckets < 128 ? a->buckets : 128;
  const int tall = es == 4 ? kTall<float> : kTall<__half>, strips = (a->Rk + 63) / 64;
  a->item_rows = kLoads * tall;
  const auto items = [&] { return (long long)a->B * strips * ((a->Rq + a->item_rows - 1) / a->item_rows); };
  while (a->item_rows > 4 * tall && items() * a->H < 148 * 20 * 2) a->item_rows /= 2;
  const long long blocks = (items() + 3) / 4, most = 148 * 5 / a->H > 1 ? 148 * 5 / a->H : 1;
  a->blocks = (int)(blocks < most ? blocks : most);
}

}  // namespace
}  // namespace evo

extern "C" {

int evoattn_relative_bias_fwd(const evoattn_relative_bias_params* p, void* cuda_stream) {
  using namespace evo;
  if (const int rc = validate(p)) return rc;
  if (p->B == 0 || p->Rq == 0 || p->Rk == 0) return EVOATTN_OK;
  if (!p->table || !p->q_pos || !p->k_pos || !p->out) return EVOATTN_ERR_NULL;
  RelArgs a = args_of(p);
  a.base = p->base;
  a.sbase = Str3{p->base_stride[0], p->base_stride[1], p->base_stride[2]};
  a.out = p->out;
  a.sout = Str3{p->out_stride[0], p->out_stride[1], p->out_stride[2]};
  const int es = dtype_bytes(p->dtype);
  const int strips = (a.Rk + 512 / es - 1) / (512 / es), groups = (a.H + kHeads - 1) / kHeads;
  int rows = 64;
  while (rows > 8 && (long long)strips * ((a.Rq + rows - 1) / rows) * a.B * groups < 148 * 4) rows /= 2;
  while ((a.Rq + rows - 1) / rows > 65535) rows *= 2;
  int row_warps = 8;
  while (row_warps > 1 && a.Rq <= row_warps / 2) row_warps /= 2;
  const dim3 grid((unsigned)strips, (unsigned)((a.Rq + rows - 1) / rows), (unsigned)(a.B * groups));
  const size_t smem = (size_t)(a.H < kHeads ? a.H : kHeads) * (slot(a.buckets) + 1) * sizeof(float);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  return with_dtype(p->dtype, [&](auto e) {
    using T = decltype(e);
    bool base_pieces = false;
    if (p->base) {  // V values of a lane in whole pieces of the base, too
      const int piece = (int)(kPer16<T> * dtype_bytes(p->base_dtype) < 16 ? kPer16<T> * dtype_bytes(p->base_dtype) : 16);
      base_pieces = ((uintptr_t)p->base | (uintptr_t)(p->base_stride[0] * dtype_bytes(p->base_dtype)) | (uintptr_t)(p->base_stride[1] * dtype_bytes(p->base_dtype)) |
                       (uintptr_t)(p->base_stride[2] * dtype_bytes(p->base_dtype))) % piece == 0;
    }
    const bool wide = rows_of_16_bytes(p->out, p->out_stride, (int)sizeof(T)) && (!p->base || base_pieces);
    const auto kern = p->base ? (wide ? relative_fwd<T, true, true> : relative_fwd<T, false, true>) : wide ? relative_fwd<T, true, false> : relative_fwd<T, false, false>;
    const cudaError_t rc = launch_dependent(kern, grid, 256, smem, st, a, rows, row_warps);
    return rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
  });
}

size_t evoattn_relative_bias_bwd_workspace_bytes(const evoattn_relative_bias_params* p) {
  using namespace evo;
  if (validate(p)) return 0;
  RelArgs a = args_of(p);
  plan_bwd(&a, dtype_bytes(p->dtype));
  return (size_t)a.H * a.blocks * a.buckets * sizeof(float);
}

int evoattn_relative_bias_bwd(const evoattn_relative_bias_params* p, void* cuda_stream) {
  using namespace evo;
  if (const int rc = validate(p)) return rc;
  RelArgs a = args_of(p);
  const int es = dtype_bytes(p->dtype);
  plan_bwd(&a, es);
  if (!p->dtable) return EVOATTN_ERR_NULL;
  if (a.blocks && (!p->q_pos || !p->k_pos || !p->d_out)) return EVOATTN_ERR_NULL;
  const size_t need = evoattn_relative_bias_bwd_workspace_bytes(p);
  if (need && (!p->workspace || p->workspace_bytes < need)) return EVOATTN_ERR_WORKSPACE;
  if ((uintptr_t)p->workspace & 15) return EVOATTN_ERR_ALIGN;
  a.partial = static_cast<float*>(p->workspace);
  a.dtable = p->dtable;
  a.out = const_cast<void*>(p->d_out);
  a.sout = Str3{p->d_out_stride[0], p->d_out_stride[1], p->d_out_stride[2]};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t rc = cudaSuccess;
  if (a.blocks) {
    const dim3 grid((unsigned)a.blocks, (unsigned)a.H, (unsigned)((a.buckets + a.window - 1) / a.window));
    const int smem = 4 * (a.window + 1) * 32 * (int)sizeof(float);
    const bool wide = rows_of_16_bytes(p->d_out, p->d_out_stride, es);
    const int bad = with_dtype(p->dtype, [&](auto e) {
      using T = decltype(e);
      const auto kern = wide ? relative_bwd<T, true> : relative_bwd<T, false>;
      if (!kernel_ready(reinterpret_cast<const void*>(kern), smem, nullptr)) return 1;
      rc = launch_dependent(kern, grid, 128, (size_t)smem, st, a);
      return 0;
    });
    if (bad) return EVOATTN_ERR_CUDA;
  }
  if (rc == cudaSuccess) rc = launch_dependent(relative_sum_partials, dim3((unsigned)((a.buckets + 31) / 32), (unsigned)a.H), 1024, 0, st, a);
  return rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

}  // extern "C"
