// What the kernels of attention over packed sequences share: the arguments, and where a sequence's rows lie.
//
// q [Tq,H,D] and k, v [Tk,Hk,D] hold the rows of B sequences one behind another; offsets on the device say where
// each begins.  The host does not know them (reading them would wait for the device), so grids are sized by what is
// possible: rows cut into tiles of n make at most T / n + B tiles.  Whatever the offsets hold, no row outside the
// tensors is touched: they are clamped where they are read, and a sequence that would end before it begins is empty.
#pragma once
#include "inputs.cuh"

namespace evo {

struct PackedArgs {
  const void *q, *k, *v;
  void* o;             // [Tq,H,D] dense; backward: in
  void* o_rest;        // what rounding left of o, or null
  float* lse;          // [H][lse_ld]: log2 of a row's sum of exp2(score * scale * log2 e); -inf: no key
  const void *d_o;     // backward
  void *dq, *dk, *dv;  // dense, as q, k, v
  float* delta;        // [H][lse_ld]: the row sums of dO * O
  const int* overlap;  // backward on CUDA cores: whether queries, and keys, of sequences overlap (then gradients are zeros)
  long long sq[2], sk[2], sv[2], sdo[2];  // element strides of (row, head)
  const void *offsets, *key_offsets;
  int B, H, Hk, D, G;  // G = H / Hk
  int causal, wide, ranges;  // offsets are int64; key_offsets is [B][2] (begin, end)
  int Tq, Tk, lse_ld;
  int few_tokens;  // sequences of up to this many queries are left to packed_few.cu; 0: none
  float scale;
  int* status;
};

struct Span {
  int begin, n;
};
__device__ __forceinline__ long long packed_offset(const void* p, int wide, long long i) {
  return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}
__device__ __forceinline__ Span clamped(long long begin, long long end, int rows) {
  begin = begin < 0 ? 0 : begin > rows ? rows : begin;
  end = end < begin ? begin : end > rows ? rows : end;
  return Span{(int)begin, (int)(end - begin)};
}
__device__ __forceinline__ Span query_span(const PackedArgs& a, int b) {
  return clamped(packed_offset(a.offsets, a.wide, b), packed_offset(a.offsets, a.wide, b + 1), a.Tq);
}
__device__ __forceinline__ Span key_span(const PackedArgs& a, int b) {
  if (a.ranges) return clamped(packed_offset(a.key_offsets, a.wide, 2LL * b), packed_offset(a.key_offsets, a.wide, 2LL * b + 1), a.Tk);
  return clamped(packed_offset(a.key_offsets, a.wide, b), packed_offset(a.key_offsets, a.wide, b + 1), a.Tk);
}
// Keys that the queries [i, i + rows) of a sequence see between them: [0, this).
__device__ __forceinline__ int keys_seen(const PackedArgs& a, int nq, int nk, int i, int rows) {
  if (!a.causal) return nk;
  const int last = i + rows < nq ? i + rows : nq;
  const int n = nk - nq + last;
  return n < 0 ? 0 : n < nk ? n : nk;
}

// The sequence and tile of the t-th tile of all sequences whose rows count(b) are cut into tiles of `tile`; seq = -1
// behind the last.  For all threads of a block (a multiple of 32, at most 1024); sm: 34 ints.
struct Place {
  int seq, tile;
};
template <class F>
__device__ __forceinline__ Place locate(int B, int t, int tile, int* sm, F&& count) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int before = 0;
  if (threadIdx.x == 0) sm[32] = -1;
  for (int b0 = 0; b0 < B; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    const int n = b < B ? (count(b) + tile - 1) / tile : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    __syncthreads();
    if (lane == 31) sm[warp] = sum;
    __syncthreads();
    int base = before, all = 0;
    for (int w = 0; w < warps; ++w) {
      if (w == warp) base += all;
      all += sm[w];
    }
    const int first = base + sum - n;
    if (t >= first && t < first + n) {
      sm[32] = b;
      sm[33] = t - first;
    }
    before += all;
    if (t < before) break;  // (the same for all threads)
  }
  __syncthreads();
  const Place p{sm[32], sm[33]};
  __syncthreads();
  return p;
}

// Zeros in the rows of a dense tensor [rows][row_bytes] that belong to no sequence, those before the first and behind
// the last (or in all of them), shared out over the blocks.
__device__ __forceinline__ void zero_outside(const void* offsets, int wide, int B, int rows, void* dst, long long row_bytes, long long block, long long blocks, bool overlap = false) {
  const Span all = overlap ? Span{0, 0} : clamped(packed_offset(offsets, wide, 0), packed_offset(offsets, wide, B), rows);
  const long long outside = rows - all.n;
  for (long long i = block; i < outside; i += blocks) {
    const long long r = i < all.begin ? i : i + all.n;
    unsigned char* p = static_cast<unsigned char*>(dst) + r * row_bytes;
    for (long long x = threadIdx.x * 2; x < row_bytes; x += blockDim.x * 2) *reinterpret_cast<unsigned short*>(p + x) = 0;
  }
}

// The forward and backward on CUDA cores (packed_generic.cu).
int launch_packed_generic_fwd(int dtype, const PackedArgs& a, cudaStream_t st, int* launches);
int launch_packed_generic_bwd(int dtype, const PackedArgs& a, cudaStream_t st, int* launches);
}  // namespace evo
