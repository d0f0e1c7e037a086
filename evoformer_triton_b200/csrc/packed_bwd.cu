// Attention over packed sequences, backward, on the 5th-generation tensor cores: bf16 and fp16, head dimensions in eights
// up to 128.
//
//   p_ij = 2^(c q_i k_j - lse_i),  ds_ij = p_ij (do_i v_j - delta_i)
//   dv_j = sum_i p_ij do_i,  dk_j = scale sum_i ds_ij q_i,  dq_i = scale sum_j ds_ij k_j
//
// Two kernels, each of which forms the scores: one walks the queries that see a tile of 128 keys (all heads of the group in
// turn) and keeps dK and dV in tensor memory, one walks the keys of a tile of 128 queries and keeps dQ there.  That is
// seven products where five would do, but no partial dQ leaves an SM, nothing is summed by atomics (the same bits in every
// run, no fp32 buffer to clear, add up in and convert), P and dS never pass through shared memory, and the sum over a
// group's heads costs nothing.
//
// Both: persistent CTAs of 12 warps.  Warp 0 loads tiles by TMA, warp 1 issues the MMAs, warps 2 and 3 see each tile
// land before the MMAs do and clear what lies behind the end of the sequence in it, and queries that see no key (0 times infinity is not 0), warps 4
// to 11 compute: a thread has one row of the 128 x 128 scores and half of its columns, P in registers from S to dS.
//
// Items are handed out as in the forward.  A key tile of long sequences or many heads is cut into parts, whose fp32 sums
// the second kernel adds up, in their order, before it ends ([5 sequences of up to 1 499, 12 heads of 96 over 2]: dK and dV
// 124 us whole, 38 in parts).  The second kernel begins as CTAs of the first leave, and waits for it only at its end.
//
// Bound by the tensor cores and the shared memory that feeds them: a step of the first kernel (four products of 128 x 128 x
// DP) needs 1.1 us of either and takes 1.75, one of the second 0.8 and 1.35.  [8192] causal, 16 heads of 128: 403 and 321 us, 1.36
// and 1.28 PFLOP/s of the products that are formed, 950 TFLOP/s of the five that a gradient cannot do without.  With 16 compute warps
// instead of 8 (a quarter of a row each) 442 and 322.
//
// dK, dV: tensor memory holds S^T, dP^T (128 columns each), dV and dK (DP each).  P^T goes back over S^T and dS^T over dP^T,
// as the A operands of dV += P^T dO and dK += dS^T Q.  The MMAs go in the order dV(n), S(n + 1), dK(n), dP(n + 1): while the
// exponentials of a step run, its dP^T and the products of the step before are on the tensor cores.
#include "packed_sm100.cuh"

namespace evo {
namespace {

using namespace ptx;

constexpr int BT = kTileRows;
constexpr int kThreads = 384, kServiceRegs = 56, kComputeRegs = 224;

// Which pairs of values go to the FMA pipes: four of sixteen.  Both kernels at D = 64, [8192] causal, 16 heads, us, with none,
// two, four and six: 583, 594, 561, 571; at D = 128 all alike.
__device__ __forceinline__ constexpr bool on_fma(int pair) { return pair % 4 == 3; }

template <int DP>
struct Tiles {
  static constexpr int kPanels = DP / 64, kPanel = BT * 128, kTile = kPanels * kPanel;
};
template <int DP>
struct DkvCfg : Tiles<DP> {
  using Tiles<DP>::kTile;
  static constexpr int kStages = DP == 128 ? 2 : 3;
  static constexpr int offK = 0, offV = kTile, offQ = 2 * kTile, offD = offQ + kStages * kTile, offStats = offD + kStages * kTile;
  static constexpr int offOut = offStats + kStages * 2 * BT * 4, offBars = offOut + 8 * kStageBytes, kBars = 4 + 6 * kStages + 5 + 4;
  // What aligning the tiles to 1024 bytes may take: less than that would leave no room at DP = 128, where the kernel checks that
  // it is enough (the dynamic shared memory of a kernel without static shared memory starts on such a boundary here).
  static constexpr int kSlack = DP == 128 ? 512 : 1024;
  static constexpr size_t bytes = offBars + kBars * 8 + 64 + kSlack;
  static_assert(bytes <= 232448, "shared memory of one CTA");
  static constexpr int colS = 0, colP = BT, colDV = 2 * BT, colDK = colDV + DP;
  static_assert(colDK + DP <= 512, "tensor memory");
};
template <int DP>
struct DqCfg : Tiles<DP> {
  using Tiles<DP>::kTile;
  static constexpr int kK = 3, kV = 2;
  static constexpr int offQ = 0, offD = kTile, offK = 2 * kTile, offV = offK + kK * kTile;
  static constexpr int offBars = offV + kV * kTile, kBars = 2 + 3 * (kK + kV) + 5 + 4;
  static constexpr size_t bytes = offBars + kBars * 8 + 64 + 1024;
  static_assert(bytes <= 232448, "shared memory of one CTA");
  static constexpr int colS = 0, colP = 2 * BT, colDQ = 3 * BT;
  static_assert(colDQ + DP <= 512, "tensor memory");
};

template <int DP>
__device__ __forceinline__ void load_tile_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int h) {
#pragma unroll
  for (int p = 0; p < DP / 64; ++p) tma_load_3d_s(dst + p * Tiles<DP>::kPanel, map, bar, 64 * p, row, h);
}
// Zeros in the rows of a staged tile from `real` on, and in those before `blind`, by a warp.
template <int DP>
__device__ __forceinline__ void clear_rows(uint32_t tile_s, int real, int lane, int blind = 0) {
  if (real >= BT && blind <= 0) return;
#pragma unroll 1
  for (int p = 0; p < DP / 64; ++p) {
    for (int x = real * 128 + lane * 16; x < Tiles<DP>::kPanel; x += 512) sts_v4(tile_s + p * Tiles<DP>::kPanel + x, 0, 0, 0, 0);
    for (int x = lane * 16; x < min(blind, BT) * 128; x += 512) sts_v4(tile_s + p * Tiles<DP>::kPanel + x, 0, 0, 0, 0);
  }
  fence_async_shared();
}

constexpr uint32_t kHi = static_cast<uint32_t>(make_sdesc_const(16, 1024, SWZ_128B) >> 32);
constexpr uint32_t kLoK = static_cast<uint32_t>(make_sdesc_const(16, 0, 0) & 0xffffffffu);                  // K-major
constexpr uint32_t kLoMN = static_cast<uint32_t>(make_sdesc_const(Tiles<64>::kPanel, 0, 0) & 0xffffffffu);  // MN-major: to the next 64 columns

// D[128 x 128] = A B^T of two staged tiles.
template <class T, int DP>
__device__ __forceinline__ void issue_product(uint32_t el, uint32_t d_tmem, uint32_t a_tile_s, uint32_t b_tile_s) {
  constexpr uint32_t kIdesc = make_idesc(std::is_same<T, __nv_bfloat16>::value, false, false, BT, BT);
  const uint32_t a = (a_tile_s >> 4) | kLoK, b = (b_tile_s >> 4) | kLoK;
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const uint32_t o = (kk / 4) * (Tiles<DP>::kPanel >> 4) + (kk % 4) * 2;
    mma_ss_e(el, d_tmem, pack_desc(a + o, kHi), pack_desc(b + o, kHi), kIdesc, kk > 0 ? 1u : 0u);
  }
}
// D[128 x DP] (+)= A B, A 16-bit in tensor memory (columns 0..63 of the products' lie at 0, 64..127 at 64), B a staged tile.
template <class T, int DP>
__device__ __forceinline__ void issue_sum(uint32_t el, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_tile_s, bool first) {
  constexpr uint32_t kIdesc = make_idesc(std::is_same<T, __nv_bfloat16>::value, false, true, BT, DP);
  const uint32_t b = (b_tile_s >> 4) | kLoMN;
#pragma unroll
  for (int kk = 0; kk < BT / 16; ++kk)
    mma_ts_e(el, d_tmem, a_tmem + (kk < 4 ? 8 * kk : 64 + 8 * (kk - 4)), pack_desc(b + kk * 128, kHi), kIdesc, (kk > 0 || !first) ? 1u : 0u);
}

// dS of 32 columns from P and dP, packed: dS = P (dP + nd), nd = -delta of the column or the row.
template <class T, class Nd>
__device__ __forceinline__ void scores_gradient(const uint32_t (&d)[32], const F2* p, Nd nd, uint32_t (&out)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float d0, d1;
    f2_get(f2_mul(p[e], f2_add(f2_from_bits(d[2 * e], d[2 * e + 1]), nd(e))), d0, d1);
    out[e] = Pack2<T>::pack(d0, d1);
  }
}

// fp16 ends at 2^16 and has steps of 2^-24 below 2^-14: dS = P (dP - delta) of a long row or a small dO would lose its bits, or all of
// it, although the sums that it enters are ordinary numbers, and that of a large dO v would overflow.  So dS is formed times 2^e, which
// its products carry to the end.  dS_ij = P_ij sum_k P_ik dO_i (V_j - V_k) is P (1 - P) 2 |dO| |V| at most, half of the largest |dO| times
// the largest |V|; e takes that to 2^15.5 at most (what is left is for the roundings of P, O and delta).  It is in the exponent of P, for
// nothing; P itself enters dV times 2^14.  One power for a call, from maxima that the row sums leave: forward and backward of
// [3088 in 5], 12 heads of 96 over 2, 117 -> 120 us, [8192] of 16 heads of 128 over 4, 1 117 -> 1 130.  bf16 has the exponents of fp32.
template <class T>
struct Lift {
  static constexpr bool kAny = std::is_same<T, __half>::value;
  static constexpr float kDv = kAny ? 0x1p-14f : 1.f;  // of dV
  float e = 0.f;     // in the exponent of P
  float p = 1.f;     // of that P where it enters dV
  float back = 1.f;  // of dK and dQ
};
__device__ __forceinline__ float exp2_whole(int e) { return __int_as_float((e + 127) << 23); }
// The words begin as zeros; every thread of a CTA brings its share of the maxima to them.
__device__ __forceinline__ void bring_norms(const PackedPlan& plan, uint32_t* words) {
  uint32_t m0 = 0, m1 = 0;
  for (int i = threadIdx.x; i < plan.n_norms; i += kThreads) {
    const uint2 x = __ldcg(reinterpret_cast<const uint2*>(plan.norms + i));
    m0 = max(m0, x.x);
    m1 = max(m1, x.y);
  }
  m0 = __reduce_max_sync(0xffffffffu, m0);
  m1 = __reduce_max_sync(0xffffffffu, m1);
  if ((threadIdx.x & 31) == 0) {
    atomicMax(words, m0);
    atomicMax(words + 1, m1);
  }
}
template <class T>
__device__ __forceinline__ Lift<T> lift_of(const uint32_t* words) {
  Lift<T> l;
  if constexpr (Lift<T>::kAny) {
    const uint32_t b = __float_as_uint(__uint_as_float(words[0]) * __uint_as_float(words[1]));  // |dO|^2 |V|^2 < 2^(k + 1)
    const int k = (int)(b >> 23) - 127;
    const int e = b == 0 ? 0 : (32 - k) >> 1;  // (a quarter of 2^(k + 1) 4^e is 2^31 at most)
    l.e = (float)e;
    l.p = exp2_whole(14 - e);
    l.back = exp2_whole(-e);
  }
  return l;
}

// Rows of no sequence in a dense tensor of 16-bit values (all of them where sequences overlap), by a warp.
__device__ __forceinline__ void clear_outside(const void* offsets, int wide, int B, int rows, void* dst, int row16, int lane, bool overlap) {
  const Span all = overlap ? Span{0, 0} : clamped(packed_offset(offsets, wide, 0), packed_offset(offsets, wide, B), rows);
#pragma unroll 1
  for (int i = blockIdx.x; i < rows - all.n; i += gridDim.x) {
    uint4* p = static_cast<uint4*>(dst) + (long long)(i < all.begin ? i : i + all.n) * row16;
    for (int x = lane; x < row16; x += 32) p[x] = make_uint4(0, 0, 0, 0);
  }
}

// The same for keys that no query sees: the tiles [begin, begin + n) of a list.
__device__ __forceinline__ void clear_tiles(const PackedTile* list, int begin, int n, void* dst, int row16, int lane) {
#pragma unroll 1
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const PackedTile t = load_tile(list + begin + i);
    uint4* p = static_cast<uint4*>(dst) + (long long)t.row * row16;
    for (int x = lane; x < t.rows * row16; x += 32) p[x] = make_uint4(0, 0, 0, 0);
  }
}

// COLS columns of an accumulator, times f, to a row of 16-bit values; zeros where `any` is not set, and in rows that are not `seen`.
template <class T, int COLS>
__device__ __forceinline__ void store_rows(uint32_t t_src, T* out, int d0, int D, float f, bool valid, bool any, bool seen) {
#pragma unroll
  for (int c = 0; c < COLS; c += 32) {
    uint32_t r[32];
    if (any) {
      tmem_ld32(t_src + c, r);
      tmem_wait_ld();
    }
#pragma unroll
    for (int e = 0; e < 32; e += 8) {
      if (valid && d0 + c + e < D) {
        uint32_t p[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) p[u] = any && seen ? Pack2<T>::pack(__uint_as_float(r[e + 2 * u]) * f, __uint_as_float(r[e + 2 * u + 1]) * f) : 0u;
        *reinterpret_cast<uint4*>(out + d0 + c + e) = make_uint4(p[0], p[1], p[2], p[3]);
      }
    }
  }
}

template <class T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
packed_dkv_sm100_kernel(const PackedArgs a, const PackedPlan plan, const FastDiv heads, const __grid_constant__ CUtensorMap tmQ,
                        const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmD,
                        const __grid_constant__ CUtensorMap tmDK, const __grid_constant__ CUtensorMap tmDV) {
  using C = DkvCfg<DP>;
  constexpr int NS = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (static_cast<int>(smem - smem_raw) > C::kSlack) {  // the same for every thread of every CTA
    if (threadIdx.x == 0 && a.status) atomicCAS(a.status, 0, DEV_TIMEOUT_SYNC);
    return;
  }
  const uint32_t smem_s = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::offBars);
  const uint32_t b0 = smem_u32(bars);
  const uint32_t k_full = b0, k_empty = b0 + 8, v_full = b0 + 16, v_empty = b0 + 24;
  auto q_in = [&](uint32_t s) { return b0 + 8 * (4 + s); };                // Q has landed
  auto q_full = [&](uint32_t s) { return b0 + 8 * (4 + NS + s); };         // ... is clean, and its statistics are there
  auto q_empty = [&](uint32_t s) { return b0 + 8 * (4 + 2 * NS + s); };    // the dK MMAs have read it
  auto d_in = [&](uint32_t s) { return b0 + 8 * (4 + 3 * NS + s); };       // the same for dO
  auto d_full = [&](uint32_t s) { return b0 + 8 * (4 + 4 * NS + s); };
  auto d_empty = [&](uint32_t s) { return b0 + 8 * (4 + 5 * NS + s); };
  const uint32_t s_full = b0 + 8 * (4 + 6 * NS), p_full = s_full + 8, dp_full = s_full + 16, ds_full = s_full + 24, out_full = s_full + 32, sched = s_full + 40;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + C::kBars + 1);
  const uint32_t abort_s = smem_u32(const_cast<int*>(abort_flag));
  uint32_t* norm_words = reinterpret_cast<uint32_t*>(bars + C::kBars + 3);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

  if (tid == 0) {
    for (int i = 0; i < C::kBars; ++i) mbar_init_s(b0 + 8 * i, b0 + 8 * i == p_full || b0 + 8 * i == ds_full ? 8 : b0 + 8 * i >= sched + 16 ? 11 : 1);
    fence_mbar_init();
    if constexpr (Lift<T>::kAny) norm_words[0] = norm_words[1] = 0u;
    prefetch_tmap(&tmQ); prefetch_tmap(&tmK); prefetch_tmap(&tmV); prefetch_tmap(&tmD);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if constexpr (Lift<T>::kAny) __syncthreads();
  grid_dependency_wait();
  grid_launch_dependents();
  if (tid == 0) *abort_flag = (a.status && *reinterpret_cast<volatile int*>(a.status) != 0) ? 1 : 0;
  if constexpr (Lift<T>::kAny) bring_norms(plan, norm_words);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const bool failed = *abort_flag != 0;
  const Lift<T> lift = lift_of<T>(norm_words);
  const bool overlap = __ldcg(plan.counts + 6) || __ldcg(plan.counts + 7);
  const int tiles = failed || overlap ? 0 : __ldcg(plan.counts + 1);
  Schedule todo{sched, sched + 16, abort_s + 4, abort_s, plan.counts + 5, tiles * (int)heads.d};

  // The steps of a CTA, one after another over its items: head g of the group, query tile i, `left` of the item from here on.
  struct Step {
    PackedTile t;
    int hk, g, i, end, left;
    __device__ __forceinline__ bool first() const { return left == t.steps; }
    __device__ __forceinline__ bool last() const { return left == 1; }
    __device__ __forceinline__ int real() const { return t.n - i * BT; }
    __device__ __forceinline__ int blind() const { return t.blind - i * BT; }
    __device__ __forceinline__ void next() {
      --left;
      if (++i == end) { i = end - t.tiles; ++g; }
    }
  };
  auto item = [&](int idx, Step& s) {
    const int tile = (int)heads.div((uint32_t)idx);
    s.hk = idx - tile * (int)heads.d;
    s.t = load_tile(plan.keys + tile);
    s.left = s.t.steps;
    s.end = (s.t.n + BT - 1) / BT;
    s.g = s.t.tiles ? s.t.begin / s.t.tiles : 0;
    s.i = s.end - s.t.tiles + s.t.begin - s.g * s.t.tiles;
  };
  // The first step of that item.  Every item has one: the MMAs are a step ahead, and what they asked for behind an item without
  // steps would wait for the warps that compute, and these for the MMAs' word that the item before is done.
  auto begin = [&](Step& s, int idx) {
    if (todo.over(idx)) return false;
    item(idx, s);
    return true;
  };
  auto advance = [&](Step& s) {
    s.next();
    return s.left > 0 || begin(s, warp == 0 ? todo.take() : todo.next());
  };

  if (warp < 4) {
    setmaxnreg_dec<kServiceRegs>();
    Step s;
    bool more = begin(s, todo.first());
    uint32_t st = 0, par = 0;
    auto next = [&] { if (++st == NS) { st = 0; par ^= 1; } };
    if (warp == 0) {
      // =============================== TMA producer ===============================
      uint32_t n = 0;
#pragma unroll 1
      while (more) {
        const int row = s.t.other + s.i * BT, h = s.hk * a.G + s.g;
        if (s.first()) {
          mbar_wait_s(k_empty, (n & 1) ^ 1, abort_s, DEV_TIMEOUT_SYNC);
          if (elect_one()) {
            mbar_expect_tx_s(k_full, C::kTile);
            load_tile_rows<DP>(smem_s + C::offK, &tmK, k_full, s.t.row, s.hk);
          }
          __syncwarp();
        }
        mbar_wait_s(q_empty(st), par ^ 1, abort_s, DEV_TIMEOUT_SYNC);
        if (elect_one()) {
          mbar_expect_tx_s(q_in(st), C::kTile);
          load_tile_rows<DP>(smem_s + C::offQ + st * C::kTile, &tmQ, q_in(st), row, h);
        }
        __syncwarp();
        if (s.first()) {
          mbar_wait_s(v_empty, (n & 1) ^ 1, abort_s, DEV_TIMEOUT_SYNC);
          ++n;
          if (elect_one()) {
            mbar_expect_tx_s(v_full, C::kTile);
            load_tile_rows<DP>(smem_s + C::offV, &tmV, v_full, s.t.row, s.hk);
          }
          __syncwarp();
        }
        mbar_wait_s(d_empty(st), par ^ 1, abort_s, DEV_TIMEOUT_SYNC);
        if (elect_one()) {
          mbar_expect_tx_s(d_in(st), C::kTile);
          load_tile_rows<DP>(smem_s + C::offD + st * C::kTile, &tmD, d_in(st), row, h);
        }
        __syncwarp();
        next();
        more = advance(s);
      }
    } else if (warp == 1) {
      // =============================== MMA issuer ===============================
      const uint32_t tS = tmem + C::colS, tP = tmem + C::colP, tV = tmem + C::colDV, tK = tmem + C::colDK;
      uint32_t n = 0, kv = 0;  // steps; items
      auto scores = [&](const Step& x, uint32_t stage, uint32_t parity) {
        if (x.first()) mbar_wait_s(k_full, kv & 1, abort_s, DEV_TIMEOUT_TMA);
        mbar_wait_s(q_full(stage), parity, abort_s, DEV_TIMEOUT_TMA);
        tc_fence_after();
        const uint32_t el = elect_one();
        issue_product<T, DP>(el, tS, smem_s + C::offK, smem_s + C::offQ + stage * C::kTile);
        mma_commit_if_s(el, s_full);
        if (x.last()) mma_commit_if_s(el, k_empty);
      };
      auto gradients = [&](const Step& x, uint32_t stage, uint32_t parity) {
        if (x.first()) {
          mbar_wait_s(v_full, kv & 1, abort_s, DEV_TIMEOUT_TMA);
          ++kv;
        }
        mbar_wait_s(d_full(stage), parity, abort_s, DEV_TIMEOUT_TMA);
        tc_fence_after();
        const uint32_t el = elect_one();
        issue_product<T, DP>(el, tP, smem_s + C::offV, smem_s + C::offD + stage * C::kTile);
        mma_commit_if_s(el, dp_full);
        if (x.last()) mma_commit_if_s(el, v_empty);
      };
      if (more) {
        scores(s, st, par);
        gradients(s, st, par);
      }
#pragma unroll 1
      while (more) {
        const bool first = s.first(), end = s.last();
        const uint32_t cs = st;
        next();
        more = advance(s);  // (s, st, par: the step after this one)
        mbar_wait_s(p_full, n & 1, abort_s, DEV_TIMEOUT_SYNC);
        tc_fence_after();
        uint32_t el = elect_one();
        issue_sum<T, DP>(el, tV, tS, smem_s + C::offD + cs * C::kTile, first);
        mma_commit_if_s(el, d_empty(cs));
        if (more) scores(s, st, par);
        mbar_wait_s(ds_full, n & 1, abort_s, DEV_TIMEOUT_SYNC);
        tc_fence_after();
        el = elect_one();
        issue_sum<T, DP>(el, tK, tP, smem_s + C::offQ + cs * C::kTile, first);
        mma_commit_if_s(el, q_empty(cs));
        if (end) mma_commit_if_s(el, out_full);
        if (more) gradients(s, st, par);
        ++n;
      }
    } else if (warp == 2) {
      // =============================== Q: its end, and the statistics of its rows ===============================
#pragma unroll 1
      while (more) {
        const int h = s.hk * a.G + s.g, real = s.real(), blind = s.blind();
        const long long at = (long long)h * a.lse_ld + s.t.other + s.i * BT;
        float nl[4], nd[4];  // (rows behind the end, or without a key: 2^e of queries and gradients that are zero)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int r = lane + 32 * u;
          const bool seen = r >= blind && r < real;
          nl[u] = (seen ? -__ldcg(a.lse + at + r) : 0.f) + lift.e;
          nd[u] = seen ? -__ldcg(a.delta + at + r) : 0.f;
        }
        mbar_wait_s(q_empty(st), par ^ 1, abort_s, DEV_TIMEOUT_SYNC);
        const uint32_t stats = smem_s + C::offStats + st * (2 * BT * 4);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          sts_f32(stats + (lane + 32 * u) * 4, nl[u]);
          sts_f32(stats + (BT + lane + 32 * u) * 4, nd[u]);
        }
        mbar_wait_s(q_in(st), par, abort_s, DEV_TIMEOUT_TMA);
        clear_rows<DP>(smem_s + C::offQ + st * C::kTile, real, lane, blind);
        __syncwarp();
        if (lane == 0) mbar_arrive_s(q_full(st));
        next();
        more = advance(s);
      }
    } else {
      // =============================== dO: its end; rows of no sequence ===============================
      if (!failed) {
        clear_outside(a.key_offsets, a.wide, a.B, a.Tk, a.dk, a.Hk * a.D / 8, lane, overlap);
        clear_outside(a.key_offsets, a.wide, a.B, a.Tk, a.dv, a.Hk * a.D / 8, lane, overlap);
        const int unseen = overlap ? 0 : __ldcg(plan.counts + 3);
        clear_tiles(plan.keys, tiles, unseen, a.dk, a.Hk * a.D / 8, lane);
        clear_tiles(plan.keys, tiles, unseen, a.dv, a.Hk * a.D / 8, lane);
      }
#pragma unroll 1
      while (more) {
        mbar_wait_s(d_in(st), par, abort_s, DEV_TIMEOUT_TMA);
        clear_rows<DP>(smem_s + C::offD + st * C::kTile, s.real(), lane, s.blind());
        __syncwarp();
        if (lane == 0) mbar_arrive_s(d_full(st));
        next();
        more = advance(s);
      }
    }
  } else {
    // =============================== compute warps ===============================
    setmaxnreg_inc<kComputeRegs>();
    const int w = (warp >> 2) - 1, row = (warp & 3) * 32 + lane;  // queries 64 w .. of a tile; the key
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t tS = t_lane + C::colS + 64 * w, tP = t_lane + C::colP + 64 * w;
    const float c = a.scale * kLog2e;
    const F2 c2 = f2_make(c, c);
    const float kInf = __int_as_float(0x7f800000);
    uint32_t n = 0, kv = 0, st = 0, par = 0;
#pragma unroll 1
    for (int idx = todo.first(); !todo.over(idx); idx = todo.next()) {
      Step s;
      item(idx, s);
#pragma unroll 1
      for (; s.left > 0; s.next(), ++n) {
        // queries of this half before `lo` do not see the key
        const int lo = a.causal ? s.t.shift + row - s.i * BT - 64 * w : 0;
        const bool cut = __any_sync(0xffffffffu, lo > 0);
        const int hidden = __shfl_sync(0xffffffffu, lo, 0) >> 5;  // pieces of 32 queries that do not see any key of the warp
        const uint32_t stats = smem_s + C::offStats + st * (2 * BT * 4) + 64 * w * 4;
        mbar_wait_s(q_full(st), par, abort_s, DEV_TIMEOUT_SYNC);
        mbar_wait_s(s_full, n & 1, abort_s, DEV_TIMEOUT_MMA);
        tc_fence_after();
        F2 p[32];
        auto exps = [&](auto with_mask) {
          constexpr bool kMask = decltype(with_mask)::value;
          uint32_t sr[2][32];
          if (!kMask) tmem_ld32(tS, sr[0]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t pk[16];
            if (kMask && k < hidden) {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                p[16 * k + e] = f2_make(0.f, 0.f);
                pk[e] = 0u;
              }
              tmem_st16(tS + 16 * k, pk);
              continue;
            }
            if (kMask) tmem_ld32(tS + 32 * k, sr[k]);
            tmem_wait_ld();
            if (!kMask && k == 0) tmem_ld32(tS + 32, sr[1]);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 nl = lds_v4f(stats + (32 * k + e) * 4);
              const F2 nl2[2] = {f2_make(nl.x, nl.y), f2_make(nl.z, nl.w)};
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const F2 x = f2_fma(f2_from_bits(sr[k][e + 2 * u], sr[k][e + 2 * u + 1]), c2, nl2[u]);
                float p0, p1;
                if (!kMask && on_fma(e / 2 + u)) {
                  exp2_fma<T, false>(x, p0, p1);
                } else {
                  float x0, x1;
                  f2_get(x, x0, x1);
                  if constexpr (kMask) {
                    x0 = 32 * k + e + 2 * u >= lo ? x0 : -kInf;
                    x1 = 32 * k + e + 2 * u + 1 >= lo ? x1 : -kInf;
                  }
                  p0 = ex2(x0);
                  p1 = ex2(x1);
                }
                p[16 * k + e / 2 + u] = f2_make(p0, p1);
                if constexpr (Lift<T>::kAny) f2_get(f2_mul(f2_make(p0, p1), f2_make(lift.p, lift.p)), p0, p1);
                pk[e / 2 + u] = Pack2<T>::pack(p0, p1);
              }
            }
            tmem_st16(tS + 16 * k, pk);
          }
        };
        if (cut) exps(std::true_type{});
        else exps(std::false_type{});
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_s(p_full);
        mbar_wait_s(dp_full, n & 1, abort_s, DEV_TIMEOUT_MMA);
        tc_fence_after();
        {
          uint32_t dr[2][32];
          tmem_ld32(tP, dr[0]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            tmem_wait_ld();
            if (k == 0) tmem_ld32(tP + 32, dr[1]);
            uint32_t dk[16];
            scores_gradient<T>(dr[k], p + 16 * k, [&](int e) {
              const float2 nd = lds_v2f(stats + (BT + 32 * k + 2 * e) * 4);
              return f2_make(nd.x, nd.y);
            }, dk);
            tmem_st16(tP + 16 * k, dk);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_s(ds_full);
        if (++st == NS) { st = 0; par ^= 1; }
      }
      mbar_wait_s(out_full, kv & 1, abort_s, DEV_TIMEOUT_MMA);
      ++kv;
      tc_fence_after();
      const uint32_t src = t_lane + (w == 0 ? C::colDV : C::colDK);
      if (s.t.parts == 1) {
        const int first = (warp & 3) * 32;  // row of the warp's first lane
        const int at = s.t.row + first;
        store_rows_staged<T, DP>(smem_s + C::offOut + (warp - 4) * kStageBytes, src, w == 0 ? &tmDV : &tmDK, at, s.hk,
                                 static_cast<T*>(w == 0 ? a.dv : a.dk) + ((long long)at * a.Hk + s.hk) * a.D, (long long)a.Hk * a.D, s.t.rows - first, a.D,
                                 w == 0 ? Lift<T>::kDv : a.scale * lift.back, true);
      } else {
        float4* out = reinterpret_cast<float4*>(plan.sums) + (((long long)s.t.slot * a.Hk + s.hk) * 2 + w) * (DP / 4 * BT) + row;
#pragma unroll
        for (int d = 0; d < DP; d += 32) {
          uint32_t r[32];
          tmem_ld32(src + d, r);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            out[(d + e) / 4 * BT] = make_float4(__uint_as_float(r[e]), __uint_as_float(r[e + 1]), __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
        }
      }
      tc_fence_before();  // (the next item's first MMAs into them follow a later arrival)
    }
    stores_done();
  }

  end_of_cta(abort_flag, a.status);
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// dQ: tensor memory holds two S, dP and dQ.  S is formed two steps ahead; the MMAs go in the order dQ(n), dP(n + 1), S(n + 2),
// so that the exponentials of a step run while the dP of that step is formed.
template <class T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
packed_dq_sm100_kernel(const PackedArgs a, const PackedPlan plan, const FastDiv heads, const int follows, const __grid_constant__ CUtensorMap tmQ,
                       const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmD) {
  using C = DqCfg<DP>;
  constexpr int NK = C::kK, NV = C::kV;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_s = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::offBars);
  const uint32_t b0 = smem_u32(bars);
  const uint32_t q_full = b0, q_empty = b0 + 8;  // Q and dO
  auto k_in = [&](uint32_t s) { return b0 + 8 * (2 + s); };
  auto k_full = [&](uint32_t s) { return b0 + 8 * (2 + NK + s); };
  auto k_empty = [&](uint32_t s) { return b0 + 8 * (2 + 2 * NK + s); };
  auto v_in = [&](uint32_t s) { return b0 + 8 * (2 + 3 * NK + s); };
  auto v_full = [&](uint32_t s) { return b0 + 8 * (2 + 3 * NK + NV + s); };
  auto v_empty = [&](uint32_t s) { return b0 + 8 * (2 + 3 * NK + 2 * NV + s); };
  const uint32_t s_full = b0 + 8 * (2 + 3 * (NK + NV)), dp_full = s_full + 16, ds_full = s_full + 24, out_full = s_full + 32, sched = s_full + 40;  // (s_full: two)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + C::kBars + 1);
  const uint32_t abort_s = smem_u32(const_cast<int*>(abort_flag));
  uint32_t* norm_words = reinterpret_cast<uint32_t*>(bars + C::kBars + 3);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

  if (tid == 0) {
    for (int i = 0; i < C::kBars; ++i) mbar_init_s(b0 + 8 * i, b0 + 8 * i == ds_full ? 8 : b0 + 8 * i >= sched + 16 ? 11 : 1);
    fence_mbar_init();
    if constexpr (Lift<T>::kAny) norm_words[0] = norm_words[1] = 0u;
    prefetch_tmap(&tmQ); prefetch_tmap(&tmK); prefetch_tmap(&tmV); prefetch_tmap(&tmD);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if constexpr (Lift<T>::kAny) __syncthreads();
  // Behind the kernel for dK and dV this one begins as its CTAs leave: it reads nothing of theirs before the end, and what it
  // reads was complete before they began.
  if (!follows) grid_dependency_wait();
  grid_launch_dependents();
  if (tid == 0) *abort_flag = (a.status && *reinterpret_cast<volatile int*>(a.status) != 0) ? 1 : 0;
  if constexpr (Lift<T>::kAny) bring_norms(plan, norm_words);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const bool failed = *abort_flag != 0;
  const Lift<T> lift = lift_of<T>(norm_words);
  Schedule todo{sched, sched + 16, abort_s + 4, abort_s, plan.counts + 4, failed || !a.dq ? 0 : __ldcg(plan.counts) * (int)heads.d};
  auto item = [&](int idx, int& h) {
    const int tile = (int)heads.div((uint32_t)idx);
    h = idx - tile * (int)heads.d;
    return load_tile(plan.queries + tile);
  };

  if (warp < 4) {
    setmaxnreg_dec<kServiceRegs>();
    uint32_t ks = 0, kp = 0, vs = 0, vp = 0;
    auto next_k = [&] { if (++ks == NK) { ks = 0; kp ^= 1; } };
    auto next_v = [&] { if (++vs == NV) { vs = 0; vp ^= 1; } };
    if (warp == 0) {
      // =============================== TMA producer ===============================
      uint32_t n = 0;
#pragma unroll 1
      for (int idx = todo.first(); !todo.over(idx); idx = todo.take()) {
        int h;
        const PackedTile t = item(idx, h);
        if (t.tiles == 0) continue;
        const int hk = h / a.G;
        mbar_wait_s(q_empty, (n & 1) ^ 1, abort_s, DEV_TIMEOUT_SYNC);
        ++n;
        if (elect_one()) {
          mbar_expect_tx_s(q_full, 2 * C::kTile);
          load_tile_rows<DP>(smem_s + C::offQ, &tmQ, q_full, t.row, h);
          load_tile_rows<DP>(smem_s + C::offD, &tmD, q_full, t.row, h);
        }
        __syncwarp();
        auto load_k = [&](int x) {
          mbar_wait_s(k_empty(ks), kp ^ 1, abort_s, DEV_TIMEOUT_SYNC);
          if (elect_one()) {
            mbar_expect_tx_s(k_in(ks), C::kTile);
            load_tile_rows<DP>(smem_s + C::offK + ks * C::kTile, &tmK, k_in(ks), t.other + x * BT, hk);
          }
          __syncwarp();
          next_k();
        };
        load_k(t.tiles - 1);
#pragma unroll 1
        for (int x = t.tiles - 1; x >= 0; --x) {  // (what the MMAs wait for in this order: K, K, V, then V and K in turn)
          if (x == t.tiles - 1 && x > 0) load_k(x - 1);
          mbar_wait_s(v_empty(vs), vp ^ 1, abort_s, DEV_TIMEOUT_SYNC);
          if (elect_one()) {
            mbar_expect_tx_s(v_in(vs), C::kTile);
            load_tile_rows<DP>(smem_s + C::offV + vs * C::kTile, &tmV, v_in(vs), t.other + x * BT, hk);
          }
          __syncwarp();
          next_v();
          if (x > 1) load_k(x - 2);
        }
      }
    } else if (warp == 1) {
      // =============================== MMA issuer ===============================
      const uint32_t tP = tmem + C::colP, tQ = tmem + C::colDQ;
      uint32_t n = 0, n_item = 0, sn = 0;  // steps, items, scores
      uint32_t cs = 0;                     // K stage of the step whose dQ is next
#pragma unroll 1
      for (int idx = todo.first(); !todo.over(idx); idx = todo.next()) {
        int h;
        const PackedTile t = item(idx, h);
        if (t.tiles == 0) continue;
        auto scores = [&] {
          mbar_wait_s(k_full(ks), kp, abort_s, DEV_TIMEOUT_TMA);
          tc_fence_after();
          const uint32_t el = elect_one();
          issue_product<T, DP>(el, tmem + C::colS + (sn & 1) * BT, smem_s + C::offQ, smem_s + C::offK + ks * C::kTile);
          mma_commit_if_s(el, s_full + 8 * (sn & 1));
          ++sn;
          next_k();
        };
        auto gradients = [&](bool end) {
          mbar_wait_s(v_full(vs), vp, abort_s, DEV_TIMEOUT_TMA);
          tc_fence_after();
          const uint32_t el = elect_one();
          issue_product<T, DP>(el, tP, smem_s + C::offD, smem_s + C::offV + vs * C::kTile);
          mma_commit_if_s(el, dp_full);
          mma_commit_if_s(el, v_empty(vs));
          if (end) mma_commit_if_s(el, q_empty);  // (the item's last S came before)
          next_v();
        };
        mbar_wait_s(q_full, n_item & 1, abort_s, DEV_TIMEOUT_TMA);
        ++n_item;
        scores();
        if (t.tiles > 1) scores();
        gradients(t.tiles == 1);
#pragma unroll 1
        for (int x = 0; x < t.tiles; ++x, ++n) {
          mbar_wait_s(ds_full, n & 1, abort_s, DEV_TIMEOUT_SYNC);
          tc_fence_after();
          const uint32_t el = elect_one();
          issue_sum<T, DP>(el, tQ, tP, smem_s + C::offK + cs * C::kTile, x == 0);
          mma_commit_if_s(el, k_empty(cs));
          if (++cs == NK) cs = 0;
          if (x + 1 == t.tiles) {
            mma_commit_if_s(el, out_full);
          } else {
            gradients(x + 2 == t.tiles);
            if (x + 2 < t.tiles) scores();  // (its buffer was read before dS of this step was there)
          }
        }
      }
    } else {
      // =============================== K (warp 2) and V (warp 3): what lies behind the end; rows of no sequence ===============================
      if (warp == 3 && !failed && a.dq) clear_outside(a.offsets, a.wide, a.B, a.Tq, a.dq, a.H * a.D / 8, lane, __ldcg(plan.counts + 6) != 0);
#pragma unroll 1
      for (int idx = todo.first(); !todo.over(idx); idx = todo.next()) {
        int h;
        const PackedTile t = item(idx, h);
#pragma unroll 1
        for (int x = t.tiles - 1; x >= 0; --x) {
          const int real = t.n - x * BT;
          if (warp == 2) {
            mbar_wait_s(k_in(ks), kp, abort_s, DEV_TIMEOUT_TMA);
            clear_rows<DP>(smem_s + C::offK + ks * C::kTile, real, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive_s(k_full(ks));
            next_k();
          } else {
            mbar_wait_s(v_in(vs), vp, abort_s, DEV_TIMEOUT_TMA);
            clear_rows<DP>(smem_s + C::offV + vs * C::kTile, real, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive_s(v_full(vs));
            next_v();
          }
        }
      }
    }
  } else {
    // =============================== compute warps ===============================
    setmaxnreg_inc<kComputeRegs>();
    const int w = (warp >> 2) - 1, row = (warp & 3) * 32 + lane;  // keys 64 w .. of a tile; the query
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t tP = t_lane + C::colP + 64 * w;
    const float c = a.scale * kLog2e;
    const F2 c2 = f2_make(c, c);
    const float kInf = __int_as_float(0x7f800000);
    uint32_t n = 0, n_item = 0;
#pragma unroll 1
    for (int idx = todo.first(); !todo.over(idx); idx = todo.next()) {
      int h;
      const PackedTile t = item(idx, h);
      const bool valid = row < t.rows;
      const long long at = (long long)h * a.lse_ld + t.row + row;
      float nl = valid ? -__ldcg(a.lse + at) : 0.f;
      const float nd = valid ? -__ldcg(a.delta + at) : 0.f;
      nl = nl == kInf ? 0.f : nl + lift.e;  // (a row without a key: the mask hides all of it)
      const F2 nl2 = f2_make(nl, nl), nd2 = f2_make(nd, nd);
      const bool seen = !a.causal || t.shift + row >= 0;  // (a query without a key: whatever q and dO hold there)
      const int last = (a.causal ? min(t.n - 1, t.shift + row) : t.n - 1) - 64 * w;
      const int warp_last = __shfl_sync(0xffffffffu, last, 0);
#pragma unroll 1
      for (int x = t.tiles - 1; x >= 0; --x, ++n) {
        const uint32_t tS = t_lane + C::colS + (n & 1) * BT + 64 * w;
        const int lim = last - x * BT;
        mbar_wait_s(s_full + 8 * (n & 1), (n >> 1) & 1, abort_s, DEV_TIMEOUT_MMA);
        tc_fence_after();
        F2 p[32];
        auto exps = [&](auto with_mask) {
          uint32_t sr[2][32];
          tmem_ld32(tS, sr[0]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            tmem_wait_ld();
            if (k == 0) tmem_ld32(tS + 32, sr[1]);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const F2 v = f2_fma(f2_from_bits(sr[k][e], sr[k][e + 1]), c2, nl2);
              float p0, p1;
              if (!decltype(with_mask)::value && on_fma(e / 2)) {
                exp2_fma<T, false>(v, p0, p1);
              } else {
                float x0, x1;
                f2_get(v, x0, x1);
                if constexpr (decltype(with_mask)::value) {
                  x0 = 32 * k + e <= lim ? x0 : -kInf;
                  x1 = 32 * k + e + 1 <= lim ? x1 : -kInf;
                }
                p0 = ex2(x0);
                p1 = ex2(x1);
              }
              p[16 * k + e / 2] = f2_make(p0, p1);
            }
          }
        };
        if (warp_last - x * BT < 63) exps(std::true_type{});
        else exps(std::false_type{});
        mbar_wait_s(dp_full, n & 1, abort_s, DEV_TIMEOUT_MMA);
        tc_fence_after();
        {
          uint32_t dr[2][32];
          tmem_ld32(tP, dr[0]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            tmem_wait_ld();
            if (k == 0) tmem_ld32(tP + 32, dr[1]);
            uint32_t dk[16];
            scores_gradient<T>(dr[k], p + 16 * k, [&](int) { return nd2; }, dk);
            tmem_st16(tP + 16 * k, dk);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_s(ds_full);
      }
      const bool any = t.tiles > 0;
      if (any) {
        mbar_wait_s(out_full, n_item & 1, abort_s, DEV_TIMEOUT_MMA);
        ++n_item;
        tc_fence_after();
      }
      store_rows<T, DP / 2>(t_lane + C::colDQ + w * (DP / 2), static_cast<T*>(a.dq) + ((long long)(t.row + row) * a.H + h) * a.D, w * (DP / 2), a.D, a.scale * lift.back, valid, any, seen);
      tc_fence_before();  // (the next item's first dQ follows a later arrival)
    }
    if (follows) {
      // The parts of dK and dV, in order: 8 columns of a row a thread, neighbours have neighbouring rows.
      grid_dependency_wait();
      const int joins = failed || __ldcg(plan.counts + 6) || __ldcg(plan.counts + 7) ? 0 : __ldcg(plan.counts + 2);
      constexpr int kPieces = 2 * DP / 8;  // of (dV, dK)
      const int at = (warp - 4) * 32 + lane;
#pragma unroll 1
      for (int x = blockIdx.x * 2 + at / BT; x < joins * a.Hk * kPieces; x += gridDim.x * 2) {
        const int piece = x % kPieces, hk = x / kPieces % a.Hk, r = at % BT, d = piece % (DP / 8) * 8;
        const uint4 j = __ldcg(reinterpret_cast<const uint4*>(plan.joins + x / kPieces / a.Hk));  // row, rows, slot, parts
        const bool is_dk = piece >= DP / 8;
        if (r >= (int)j.y || d >= a.D) continue;
        const float4* in = reinterpret_cast<const float4*>(plan.sums) + (((long long)j.z * a.Hk + hk) * 2 + is_dk) * (DP / 4 * BT) + d / 4 * BT + r;
        float f[8] = {};
#pragma unroll 4
        for (int p = 0; p < (int)j.w; ++p) {
          const float4 u = __ldcg(in), v = __ldcg(in + BT);
          f[0] += u.x; f[1] += u.y; f[2] += u.z; f[3] += u.w;
          f[4] += v.x; f[5] += v.y; f[6] += v.z; f[7] += v.w;
          in += (long long)a.Hk * 2 * (DP / 4 * BT);
        }
        const float by = is_dk ? a.scale * lift.back : Lift<T>::kDv;
        uint32_t o[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) o[u] = Pack2<T>::pack(f[2 * u] * by, f[2 * u + 1] * by);
        *reinterpret_cast<uint4*>(static_cast<T*>(is_dk ? a.dk : a.dv) + ((long long)(j.x + r) * a.Hk + hk) * a.D + d) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }

  end_of_cta(abort_flag, a.status);
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <class K>
int prepare(K kern, size_t bytes) {
  int regs = 0;
  if (!kernel_ready(reinterpret_cast<const void*>(kern), (int)bytes, &regs)) return EVOATTN_ERR_CUDA;
  // (setmaxnreg.inc would wait for registers that the launch does not have)
  return kThreads * regs < 256 * kComputeRegs + 128 * kServiceRegs ? EVOATTN_ERR_UNSUPPORTED : EVOATTN_OK;
}

template <class T, int DP>
int launch(const PackedArgs& a, const PackedPlan& plan, cudaStream_t st, int* launches) {
  CUtensorMap tq, tk, tv, td;
  if (!make_packed_map(&tq, a.q, a.sq, a.Tq, a.H, a.D) || !make_packed_map(&tk, a.k, a.sk, a.Tk, a.Hk, a.D) || !make_packed_map(&tv, a.v, a.sv, a.Tk, a.Hk, a.D) ||
      !make_packed_map(&td, a.d_o, a.sdo, a.Tq, a.H, a.D))
    return EVOATTN_ERR_CUDA;
  const int sms = sm_count();
  if (sms <= 0) return EVOATTN_ERR_CUDA;
  if (a.dk) {
    auto kern = packed_dkv_sm100_kernel<T, DP>;
    CUtensorMap tdk, tdv;
    const long long sk[2] = {(long long)a.Hk * a.D, a.D};
    if (!make_packed_map(&tdk, a.dk, sk, a.Tk, a.Hk, a.D, 32) || !make_packed_map(&tdv, a.dv, sk, a.Tk, a.Hk, a.D, 32)) return EVOATTN_ERR_CUDA;
    const int rc = prepare(kern, DkvCfg<DP>::bytes);
    if (rc) return rc;
    const long long most = (key_tiles(a) + key_slots(a, sms)) * a.Hk;
    launch_dependent(kern, dim3((unsigned)(most < sms ? most : sms)), kThreads, DkvCfg<DP>::bytes, st, a, plan, FastDiv((uint32_t)a.Hk), tq, tk, tv, td, tdk, tdv);
    *launches += 1;
  }
  // (also where no dQ is wanted, if there may be parts of dK and dV to join)
  if (a.dq || key_slots(a, sms) > 0) {
    auto kern = packed_dq_sm100_kernel<T, DP>;
    const int rc = prepare(kern, DqCfg<DP>::bytes);
    if (rc) return rc;
    const long long most = a.dk ? sms : query_units(a, BT) * a.H;
    launch_dependent(kern, dim3((unsigned)(most < sms ? most : sms)), kThreads, DqCfg<DP>::bytes, st, a, plan, FastDiv((uint32_t)a.H), (int)(a.dk != nullptr), tq, tk, tv, td);
    *launches += 1;
  }
  return cudaGetLastError() == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}

size_t delta_bytes(const PackedArgs& a) { return ((size_t)a.H * a.Tq * sizeof(float) + 255) / 256 * 256; }

}  // namespace

bool sm100_packed_bwd_supported(int dtype, const PackedArgs& a) {
  return sm100_packed_supported(dtype, a) && packed_map_ok(a.d_o, a.sdo, a.Tq, a.H) && ((reinterpret_cast<uintptr_t>(a.dq) | reinterpret_cast<uintptr_t>(a.dk) | reinterpret_cast<uintptr_t>(a.dv)) & 15) == 0;
}
size_t sm100_packed_bwd_workspace_bytes(const PackedArgs& a) { return delta_bytes(a) + plan_bytes(a, true, BT, true, sm_count()).all(); }
int launch_sm100_packed_bwd(int dtype, const PackedArgs& args, void* ws, cudaStream_t st, int* launches) {
  PackedArgs a = args;
  a.delta = static_cast<float*>(ws);
  PackedPlan plan = place_plan(a, BT, static_cast<unsigned char*>(ws) + delta_bytes(a), plan_bytes(a, true, BT, true, sm_count()));
  const int rc = launch_packed_prepare(dtype, a, plan, true, BT, true, true, st, launches);
  if (rc) return rc;
  if (dtype == EVOATTN_BF16) return a.D <= 64 ? launch<__nv_bfloat16, 64>(a, plan, st, launches) : launch<__nv_bfloat16, 128>(a, plan, st, launches);
  return a.D <= 64 ? launch<__half, 64>(a, plan, st, launches) : launch<__half, 128>(a, plan, st, launches);
}

}  // namespace evo
