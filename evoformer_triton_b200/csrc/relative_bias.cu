// Learned relative position bias by buckets, forward and backward.
//
//   out[b,h,i,j] = table[row(k_j - q_i), h] (+ base[b,h,i,j]),   dtable[r,h] = sum of d_out over (b,i,j) with row r
//
// Memory bound both ways: one write (and one read of the base) of B H Rq Rk values, one read of them.  A warp
// walks rows of a strip of keys whose positions stay in registers, so the bucket of a score is worked out
// once for all heads (forward), or not at all where a whole strip of a row falls into one bucket, as
// it does away from the diagonal (backward).
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

// The table's row for a key `rel` ahead of the query.  edges: shared memory.
struct Buckets {
  int scheme, exact, n_edges, half;
  const int* edges;
  __device__ __forceinline__ Buckets(const RelArgs& a, const int* sm_edges)
      : scheme(a.scheme), exact(a.exact), n_edges(a.n_edges), half(a.buckets >> 1), edges(sm_edges) {}
  __device__ __forceinline__ int operator()(long long rel) const {
    const bool ahead = rel > 0;
    if (scheme == EVOATTN_BUCKETS_LOG_CAUSAL && ahead) return 0;
    const unsigned long long far = ahead ? (unsigned long long)rel : 0ull - (unsigned long long)rel;
    const int a = far > 0x3fffffffull ? 0x3fffffff : (int)far;
    int f = a;
    if (a >= exact) {
      int lo = 0, hi = n_edges;  // the number of edges that are <= a
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (edges[mid] <= a) lo = mid + 1;
        else hi = mid;
      }
      f = exact + lo;
    }
    if (scheme == EVOATTN_BUCKETS_CLIP) return ahead ? exact - f : exact + f;
    return scheme == EVOATTN_BUCKETS_LOG && ahead ? half + f : f;
  }
};

// Heads that a block of the forward holds the table of.
constexpr int kHeads = 8;
// A row of the table in shared memory.  Lanes read rows that lie V = 4 or 8 apart (consecutive keys): one
// float of padding every eight rows keeps them in different banks.
__host__ __device__ constexpr int slot(int row) { return row + (row >> 3); }

// A block of eight warps takes a strip of 32 V keys and kHeads heads and walks rows, one a warp.  V
// consecutive keys a lane where rows are 16-byte aligned (WIDE), else keys 32 apart.
template <class T, bool WIDE>
__global__ void __launch_bounds__(256) relative_fwd(RelArgs a, int rows_per_block) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int V = kPer16<T>;
  extern __shared__ float sm_table[];  // [kHeads][slot(buckets)]
  __shared__ int sm_edges[kLogEdges];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = (a.H + kHeads - 1) / kHeads;
  const int b = blockIdx.z / groups, h0 = (blockIdx.z - b * groups) * kHeads, nh = min(kHeads, a.H - h0);
  const int pitch = slot(a.buckets) + 1;
  for (int i = threadIdx.x; i < a.n_edges; i += 256) sm_edges[i] = a.edges[i];
  for (int i = threadIdx.x; i < a.buckets * nh; i += 256) {
    const int r = i / nh, h = i - r * nh;
    sm_table[h * pitch + slot(r)] = load_any(a.table, a.table_dtype, (long long)r * a.H + h0 + h);
  }
  const Buckets bucket(a, sm_edges);
  const int j0 = blockIdx.x * 32 * V;
  long long key[V];
  int col[V];
#pragma unroll
  for (int u = 0; u < V; ++u) {
    col[u] = WIDE ? j0 + lane * V + u : j0 + u * 32 + lane;
    key[u] = col[u] < a.Rk ? position(a.k_pos, a.positions64, b * a.sk + col[u]) : 0;
  }
  __syncthreads();
  const int i_end = (int)min((long long)a.Rq, ((long long)blockIdx.y + 1) * rows_per_block);
  for (int i = blockIdx.y * rows_per_block + warp; i < i_end; i += 8) {
    const long long q = position(a.q_pos, a.positions64, b * a.sq + i);
    int s[V];
    bool same = true;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      s[u] = slot(bucket(key[u] - q));
      same = same && s[u] == s[0];
    }
    for (int h = 0; h < nh; ++h) {
      const float* t = sm_table + h * pitch;
      float v[V];
      if (same) {
        v[0] = t[s[0]];
#pragma unroll
        for (int u = 1; u < V; ++u) v[u] = v[0];
      } else {
#pragma unroll
        for (int u = 0; u < V; ++u) v[u] = t[s[u]];
      }
      if (a.base) {
        const long long at = b * a.sbase.a + (h0 + h) * a.sbase.b + (long long)i * a.sbase.c;
#pragma unroll
        for (int u = 0; u < V; ++u)
          if (col[u] < a.Rk) v[u] += load_any(a.base, a.base_dtype, at + col[u]);
      }
      T* o = static_cast<T*>(a.out) + b * a.sout.a + (h0 + h) * a.sout.b + (long long)i * a.sout.c;
      if (WIDE && col[V - 1] < a.Rk) {
        *reinterpret_cast<uint4*>(o + col[0]) = pack16<T>(v);
      } else {
#pragma unroll
        for (int u = 0; u < V; ++u)
          if (col[u] < a.Rk) o[col[u]] = from_float<T>(v[u]);
      }
    }
  }
}

// Backward: a warp takes item_rows rows of a strip of 32 V keys of one (b, h) at a time and adds every value to
// the sum of its bucket.  Every lane has sums of its own (no two lanes add to one address, and the order
// of the additions is fixed); a row whose strip is one bucket is added up in a register first.  A block keeps
// the sums of `window` table rows (blockIdx.z says which); strips that cannot touch them are not read.
template <class T, bool WIDE>
__global__ void __launch_bounds__(128) relative_bwd(RelArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int V = kPer16<T>;
  extern __shared__ float sm_sums[];  // [4 warps][window][32 lanes]
  __shared__ int sm_edges[kLogEdges];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, first = blockIdx.z * a.window, count = min(a.window, a.buckets - first);
  for (int i = threadIdx.x; i < a.n_edges; i += 128) sm_edges[i] = a.edges[i];
  for (int i = threadIdx.x; i < 4 * a.window * 32; i += 128) sm_sums[i] = 0.f;
  __syncthreads();
  const Buckets bucket(a, sm_edges);
  float* sums = sm_sums + warp * a.window * 32 + lane;
  const int strips = (a.Rk + 32 * V - 1) / (32 * V), chunks = (a.Rq + a.item_rows - 1) / a.item_rows;
  const long long items = (long long)a.B * strips * chunks;
  for (long long item = (long long)blockIdx.x * 4 + warp; item < items; item += (long long)gridDim.x * 4) {
    const int chunk = (int)(item % chunks);
    const long long rest = item / chunks;
    const int strip = (int)(rest % strips), b = (int)(rest / strips);
    const int j0 = strip * 32 * V, i0 = chunk * a.item_rows, ni = min(a.item_rows, a.Rq - i0);
    long long key[V], least = 0x7fffffffffffffffll, most = -0x7fffffffffffffffll - 1;
    int col[V];
#pragma unroll
    for (int u = 0; u < V; ++u) {
      col[u] = WIDE ? j0 + lane * V + u : j0 + u * 32 + lane;
      key[u] = 0;
      if (col[u] < a.Rk) {
        key[u] = position(a.k_pos, a.positions64, b * a.sk + col[u]);
        least = min(least, key[u]);
        most = max(most, key[u]);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    // lane l: what row i0 + l of the strip is: one bucket (>= 0), several (-1), none of this block's (-2)
    const long long my_q = lane < ni ? position(a.q_pos, a.positions64, b * a.sq + i0 + lane) : 0;
    int my_kind = -2;
    if (lane < ni) {
      const int lo = bucket(least - my_q), hi = bucket(most - my_q);
      my_kind = lo == hi ? (lo >= first && lo < first + count ? lo : -2) : -1;
    }
    const T* d = static_cast<const T*>(a.out) + b * a.sout.a + h * a.sout.b + (long long)i0 * a.sout.c;
    float acc = 0.f;
    int acc_row = -1;
    for (int i = 0; i < ni; ++i) {
      const int kind = __shfl_sync(0xffffffffu, my_kind, i);
      const long long q = __shfl_sync(0xffffffffu, my_q, i);
      if (kind == -2) continue;
      const T* row = d + i * a.sout.c;
      float v[V];
      if (WIDE && col[V - 1] < a.Rk) {
        unpack16<T>(*reinterpret_cast<const uint4*>(row + col[0]), v);
      } else {
#pragma unroll
        for (int u = 0; u < V; ++u) v[u] = col[u] < a.Rk ? to_float<T>(row[col[u]]) : 0.f;
      }
      if (kind >= 0) {
        if (kind != acc_row) {
          if (acc_row >= 0) sums[(acc_row - first) * 32] += acc;
          acc_row = kind;
          acc = 0.f;
        }
#pragma unroll
        for (int u = 0; u < V; ++u) acc += v[u];
      } else {
#pragma unroll
        for (int u = 0; u < V; ++u) {
          const int r = bucket(key[u] - q) - first;
          if (col[u] < a.Rk && r >= 0 && r < count) sums[r * 32] += v[u];
        }
      }
    }
    if (acc_row >= 0) sums[(acc_row - first) * 32] += acc;
  }
  __syncthreads();
  for (int r = warp; r < count; r += 4) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) s += sm_sums[(w * a.window + r) * 32 + lane];
    s = warp_sum(s);
    if (lane == 0) a.partial[((long long)h * a.blocks + blockIdx.x) * a.buckets + first + r] = s;
  }
}

// The blocks' sums of a head, added in order: a warp for 32 table rows, eight shares of the blocks.
__global__ void __launch_bounds__(256) relative_sum_partials(RelArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  __shared__ float sm[8][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, r = blockIdx.x * 32 + lane, h = blockIdx.y;
  float s = 0.f;
  if (r < a.buckets)
    for (int k = part; k < a.blocks; k += 8) s += a.partial[((long long)h * a.blocks + k) * a.buckets + r];
  sm[part][lane] = s;
  __syncthreads();
  if (part == 0 && r < a.buckets) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += sm[i][lane];
    store_any(a.dtable, a.table_dtype, (long long)r * a.H + h, s);
  }
}

int validate(const evoattn_relative_bias_params* p) {
  if (!p) return EVOATTN_ERR_NULL;
  if (!known_dtype(p->dtype) || !known_dtype(p->table_dtype) || (p->base && !known_dtype(p->base_dtype))) return EVOATTN_ERR_DTYPE;
  if (p->B < 0 || p->H <= 0 || p->Rq < 0 || p->Rk < 0 || p->B > 65535 || p->H > 4096) return EVOATTN_ERR_SHAPE;
  if (p->Rq > (1 << 24) || p->Rk > (1 << 24)) return EVOATTN_ERR_SHAPE;
  if ((long long)p->B * ((p->H + kHeads - 1) / kHeads) > 65535) return EVOATTN_ERR_SHAPE;
  if (p->buckets <= 0 || p->buckets > EVOATTN_MAX_BUCKETS || p->n_edges < 0 || p->n_edges > kLogEdges || p->exact < 0) return EVOATTN_ERR_SHAPE;
  if (p->n_edges > 0 && !p->edges) return EVOATTN_ERR_NULL;
  for (int i = 0; i < p->n_edges; ++i)  // a distance finds its bucket by bisection
    if (p->edges[i] < p->exact || (i && p->edges[i] < p->edges[i - 1])) return EVOATTN_ERR_SHAPE;
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
  const int strips = (a->Rk + 512 / es - 1) / (512 / es);
  a->item_rows = 32;
  const auto items = [&] { return (long long)a->B * strips * ((a->Rq + a->item_rows - 1) / a->item_rows); };
  while (a->item_rows > 4 && items() * a->H < 148 * 16) a->item_rows /= 2;
  const long long blocks = (items() + 3) / 4, most = (148 * 6 + a->H - 1) / a->H;
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
  const bool wide = rows_of_16_bytes(p->out, p->out_stride, es);
  const int strips = (a.Rk + 512 / es - 1) / (512 / es), groups = (a.H + kHeads - 1) / kHeads;
  int rows = 64;
  while (rows > 8 && (long long)strips * ((a.Rq + rows - 1) / rows) * a.B * groups < 148 * 4) rows /= 2;
  if ((a.Rq + rows - 1) / rows > 65535) rows = (a.Rq + 65534) / 65535;
  const dim3 grid((unsigned)strips, (unsigned)((a.Rq + rows - 1) / rows), (unsigned)(a.B * groups));
  const size_t smem = (size_t)(a.H < kHeads ? a.H : kHeads) * (slot(a.buckets) + 1) * sizeof(float);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  return with_dtype(p->dtype, [&](auto e) {
    using T = decltype(e);
    const cudaError_t rc = wide ? launch_dependent(relative_fwd<T, true>, grid, 256, smem, st, a, rows) : launch_dependent(relative_fwd<T, false>, grid, 256, smem, st, a, rows);
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
    const int smem = 4 * a.window * 32 * (int)sizeof(float);
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
  if (rc == cudaSuccess) rc = launch_dependent(relative_sum_partials, dim3((unsigned)((a.buckets + 31) / 32), (unsigned)a.H), 256, 0, st, a);
  return rc == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

}  // extern "C"
