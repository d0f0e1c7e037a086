// Attention over packed sequences, forward, on the 5th-generation tensor cores: bf16 and fp16, head dimensions in eights
// up to 128.
//
//   o_i = sum_j p_ij v_j / l_i,  p_ij = 2^(c q_i k_j - m_i),  l_i = sum_j p_ij,  c = scale log2 e
//
// in one pass over the keys.  Persistent CTAs of 12 warps: warp 0 loads tiles by TMA, warp 1 issues the MMAs, warp 2
// writes zeros where no sequence lies, warps 4 to 11 are two warpgroups with a tile of 128 queries each, a thread a
// query.  The two tiles are those of two heads that read the same keys (an even number of heads a group), or two
// neighbouring ones of one head: one load of K and V serves both, and while one warpgroup's MMAs run, the other has the
// exponentials.  Keys in tiles of 128, the last first: those are the ones that a mask cuts, and the others take a loop
// without it.  Items (a unit of tiles, a head or two) go out most work first from a counter; with long rows of key tiles and
// few items, an item is a part of a row, and the last part to arrive adds them up in their order (the same bits in
// every run): [512 512 300 77] queries against up to 6 001 keys, 16 heads of 64, 99 us whole, 59 in parts.
//
// S = Q K^T lands in tensor memory (128 columns a warpgroup); P goes back over it in 16 bits, from where it is the A
// operand of P V; O accumulates next to it (DP columns): with DP = 128 that is all of tensor memory.  The MMAs of a
// warpgroup are issued by one thread in the order P V of tile n, S of tile n - 1, so that S lands when O is complete up
// to tile n and may be rescaled.
//
// m is not the maximum but a reference that the exponentials of a tile are taken against straight from the scores, without
// looking for their maximum: any m gives the same o as long as nothing leaves the range of P's type.  It is 0 to begin with; if
// a tile's sum shows that some p may be too large, or a row's first sum that all of them are too small, the tile's maximum
// is taken, O and l follow it, and the tile is done again (P is kept in registers until then).  A score that is infinite or NaN
// comes this way too, since its p is, and makes l, and with it the row, NaN.  O is divided by the sum of the
// P that it was made of, rounded (with that of the unrounded values it was off by 0.0023 instead of 0.0021 of its norm, where
// its own rounding makes 0.0016, and a forward took 4 % less); the log-sum-exp is that of the unrounded ones.
//
// Bound at D = 128 by the chain of a warpgroup's tile: 0.7 us of softmax, 0.27 us each for P V and S, and three hand-overs;
// 1.9 us for a tile of each, of which the tensor cores work 1.1 and shared memory feeds them without a pause (S reads
// both operands there).  [16384] causal, 16 heads of 128 over 4: 894 us, 1.23 PFLOP/s; under the power cap, calls back to
// back, 1 055.  At D = 64 by the issue slots and units of the exponentials: 16 heads 740 us.  An item costs some 3 us besides.
#include "packed_sm100.cuh"

namespace evo {
namespace {

using namespace ptx;

constexpr int BM = kTileRows, BN = kTileRows;
constexpr int kThreads = 384, kServiceRegs = 56, kSoftmaxRegs = 224;

// kMaxSum: sum of a tile's exponentials up to which they serve (fp16 ends at 2^16; bf16 and the fp32 sums hold any); kMinSum:
// the least first sum of a row (fp16 has steps of 2^-24: against a sum of 2^-4 that is what rounding P costs at 2^-10
// of it); kRise: rise of a tile's maximum, in powers of two, up to which the sum of its 128 cannot be more.
template <class T> struct Lag;
template <> struct Lag<__half> { static constexpr float kMaxSum = 32768.f, kMinSum = 0.0625f, kRise = 8.f; };
template <> struct Lag<__nv_bfloat16> { static constexpr float kMaxSum = 4294967296.f, kMinSum = 0x1p-40f, kRise = 25.f; };

// Which pairs of values go to the FMA pipes: four of sixteen.  Forward of [16384] causal, 16 heads, us, with none, two, four,
// six and eight: D = 128 (4 key heads) 923, 876, 852, 913, 973; D = 64 818, 759, 712, 737, 811.
__device__ __forceinline__ constexpr bool on_fma(int pair) { return pair % 4 == 3; }

template <int DP>
struct FwdCfg {
  static constexpr int kPanels = DP / 64;             // of 64 values: 128 bytes a row, swizzled
  static constexpr int kPanel = BM * 128, kTile = kPanels * kPanel;
  static constexpr int kStages = DP == 128 ? 4 : 8;   // K and V tiles in the order of their use
  static constexpr int offQ = 0, offKV = 2 * kTile, offOut = offKV + kStages * kTile, offBars = offOut + 8 * kStageBytes;
  static constexpr int kBars = 2 * kStages + 2 + 6 + 4 + 2;
  static constexpr size_t bytes = offBars + kBars * 8 + 64 + 1024;
  static_assert(bytes <= 232448, "shared memory of one CTA");
  static constexpr int colO = 2 * BN;                 // S of both warpgroups, then O of both
  static_assert(colO + 2 * DP <= 512, "tensor memory");
};

template <class T, int DP, bool PAIR, bool LSE>  // PAIR: two query tiles of one head, else one tile of two heads; LSE: for a backward pass
__global__ void __launch_bounds__(kThreads, 1)
packed_fwd_sm100_kernel(const PackedArgs a, const PackedPlan plan, const FastDiv units, const __grid_constant__ CUtensorMap tmQ,
                        const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmR) {
  using C = FwdCfg<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int NS = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ volatile int arrived[2];
  const uint32_t smem_s = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::offBars);
  const uint32_t bars_s = smem_u32(bars);
  auto t_full = [&](uint32_t st) { return bars_s + 8 * st; };            // a K or V tile has landed
  auto t_empty = [&](uint32_t st) { return bars_s + 8 * (NS + st); };    // ... and has been read
  const uint32_t q_full = bars_s + 8 * (2 * NS), q_empty = q_full + 8;
  auto s_full = [&](int w) { return q_full + 8 * (2 + w); };             // S of a tile (and O up to the tile before)
  auto p_full = [&](int w) { return q_full + 8 * (4 + w); };             // P of a tile is in tensor memory
  auto o_full = [&](int w) { return q_full + 8 * (6 + w); };             // O of an item
  const uint32_t sched = q_full + 8 * 8;
  auto together = [&](int w) { return q_full + 8 * (12 + w); };          // the warps of a warpgroup (where parts are joined)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + C::kBars + 1);
  const uint32_t abort_s = smem_u32(const_cast<int*>(abort_flag));
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) { mbar_init_s(t_full(i), 1); mbar_init_s(t_empty(i), 1); }
    mbar_init_s(q_full, 1);
    mbar_init_s(q_empty, 1);
    for (int w = 0; w < 2; ++w) { mbar_init_s(s_full(w), 1); mbar_init_s(p_full(w), 4); mbar_init_s(o_full(w), 1); mbar_init_s(together(w), 4); }
    for (int i = 0; i < 2; ++i) { mbar_init_s(sched + 8 * i, 1); mbar_init_s(sched + 16 + 8 * i, 9); }
    fence_mbar_init();
    prefetch_tmap(&tmQ); prefetch_tmap(&tmK); prefetch_tmap(&tmV);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  grid_dependency_wait();
  grid_launch_dependents();
  // A launch that follows a failed one returns at once (one reader, so the CTA agrees).
  if (tid == 0) *abort_flag = (a.status && *reinterpret_cast<volatile int*>(a.status) != 0) ? 1 : 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const bool failed = *abort_flag != 0;
  Schedule todo{sched, sched + 16, abort_s + 4, abort_s, plan.counts + 4, failed ? 0 : __ldcg(plan.counts) * (int)units.d};

  // An item: its tile and first head, and of warpgroup w the valid rows, the last key of row 0 and the tiles of keys.
  struct Item {
    PackedTile t;
    int h;
  };
  auto item_at = [&](int idx) {
    Item it;
    const int tile = (int)units.div((uint32_t)idx), u = idx - tile * (int)units.d;
    it.t = load_tile(plan.queries + tile);
    it.h = PAIR ? u : 2 * u;
    return it;
  };
  auto rows_of = [&](const Item& it, int w) { return PAIR ? max(0, min(BM, it.t.rows - w * BM)) : it.t.rows; };
  // (key tiles [begin, this) are those of the item that it works on)
  auto end_of = [&](const Item& it, int w) {
    const int end = it.t.begin + it.t.steps;
    if (!PAIR || rows_of(it, 1) == 0) return PAIR && w == 1 ? it.t.begin : end;
    if (w == 1 || !a.causal) return end;
    return max(it.t.begin, min(end, (min(it.t.n, it.t.shift + BM) + BN - 1) / BN));
  };

  if (warp < 4) {
    setmaxnreg_dec<kServiceRegs>();
    if (warp == 0) {
      // =============================== TMA producer ===============================
      uint32_t st = 0, par = 1, n = 0;
      auto load = [&](const CUtensorMap* map, int row, int h) {
        mbar_wait_s(t_empty(st), par, abort_s, DEV_TIMEOUT_SYNC);
        if (elect_one()) {
          mbar_expect_tx_s(t_full(st), C::kTile);
#pragma unroll
          for (int p = 0; p < C::kPanels; ++p) tma_load_3d_s(smem_s + C::offKV + st * C::kTile + p * C::kPanel, map, t_full(st), 64 * p, row, h);
        }
        __syncwarp();
        if (++st == NS) { st = 0; par ^= 1; }
      };
#pragma unroll 1
      for (int idx = todo.first(); !todo.over(idx); idx = todo.take()) {
        const Item it = item_at(idx);
        if (it.t.steps == 0) continue;
        const int hk = it.h / a.G, first = it.t.begin, end = first + it.t.steps;
        mbar_wait_s(q_empty, (n & 1) ^ 1, abort_s, DEV_TIMEOUT_SYNC);
        ++n;
        if (elect_one()) {
          mbar_expect_tx_s(q_full, 2 * C::kTile);
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int p = 0; p < C::kPanels; ++p)
              tma_load_3d_s(smem_s + C::offQ + w * C::kTile + p * C::kPanel, &tmQ, q_full, 64 * p, it.t.row + (PAIR ? w * BM : 0), it.h + (PAIR ? 0 : w));
        }
        __syncwarp();
        load(&tmK, it.t.other + (end - 1) * BN, hk);
#pragma unroll 1
        for (int t = end - 1; t >= first; --t) {
          load(&tmV, it.t.other + t * BN, hk);
          if (t > first) load(&tmK, it.t.other + (t - 1) * BN, hk);
        }
      }
    } else if (warp == 1) {
      // =============================== MMA issuer ===============================
      constexpr uint32_t kIdescS = make_idesc(kBf16, false, false, BM, BN), kIdescO = make_idesc(kBf16, false, true, BM, DP);
      constexpr uint32_t kHi = static_cast<uint32_t>(make_sdesc_const(16, 1024, SWZ_128B) >> 32);
      constexpr uint32_t kLoK = static_cast<uint32_t>(make_sdesc_const(16, 0, 0) & 0xffffffffu);            // K-major
      constexpr uint32_t kLoMN = static_cast<uint32_t>(make_sdesc_const(C::kPanel, 0, 0) & 0xffffffffu);    // MN-major: to the next 64 columns
      const uint32_t q_lo = ((smem_s + C::offQ) >> 4) | kLoK, kv = (smem_s + C::offKV) >> 4;
      uint32_t st = 0, par = 0, n = 0, np[2] = {0, 0};
      auto next = [&] { if (++st == NS) { st = 0; par ^= 1; } };
      auto scores = [&](int w, uint32_t at) {
        const uint32_t el = elect_one(), ka = (kv + at * (C::kTile >> 4)) | kLoK, qa = q_lo + w * (C::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t o = (kk / 4) * (C::kPanel >> 4) + (kk % 4) * 2;
          mma_ss_e(el, tmem + w * BN, pack_desc(qa + o, kHi), pack_desc(ka + o, kHi), kIdescS, kk > 0 ? 1u : 0u);
        }
        mma_commit_if_s(el, s_full(w));
      };
#pragma unroll 1
      for (int idx = todo.first(); !todo.over(idx); idx = todo.next()) {
        const Item it = item_at(idx);
        const int first = it.t.begin, end = first + it.t.steps, tw[2] = {end_of(it, 0), end_of(it, 1)};
        if (it.t.steps == 0) continue;
        mbar_wait_s(q_full, n & 1, abort_s, DEV_TIMEOUT_TMA);
        ++n;
        mbar_wait_s(t_full(st), par, abort_s, DEV_TIMEOUT_TMA);
        tc_fence_after();
#pragma unroll
        for (int w = 0; w < 2; ++w)
          if (tw[w] == end) scores(w, st);
        uint32_t el = elect_one();
        mma_commit_if_s(el, t_empty(st));
        if (it.t.steps == 1) mma_commit_if_s(el, q_empty);
        next();
#pragma unroll 1
        for (int t = end - 1; t >= first; --t) {
          const uint32_t vs = st, vpar = par;
          next();
          const uint32_t ks = st, kpar = par;
          mbar_wait_s(t_full(vs), vpar, abort_s, DEV_TIMEOUT_TMA);
          const int real = it.t.n - t * BN;
          if (real < BN) {
            // rows behind the sequence may hold anything, and P = 0 times infinity is not 0
            const uint32_t v_s = smem_s + C::offKV + vs * C::kTile;
#pragma unroll 1
            for (int p = 0; p < C::kPanels; ++p)
              for (int x = real * 128 + lane * 16; x < C::kPanel; x += 512) sts_v4(v_s + p * C::kPanel + x, 0, 0, 0, 0);
            fence_async_shared();
            __syncwarp();
          }
          if (t > first) mbar_wait_s(t_full(ks), kpar, abort_s, DEV_TIMEOUT_TMA);
          const uint32_t va = (kv + vs * (C::kTile >> 4)) | kLoMN;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (t < tw[w]) {
              mbar_wait_s(p_full(w), np[w] & 1, abort_s, DEV_TIMEOUT_SYNC);
              ++np[w];
              tc_fence_after();
              el = elect_one();
#pragma unroll
              for (int kk = 0; kk < BN / 16; ++kk)  // 16 keys: 8 packed columns of P, 16 rows of V
                mma_ts_e(el, tmem + C::colO + w * DP, tmem + w * BN + 8 * kk, pack_desc(va + kk * 128, kHi), kIdescO, (kk > 0 || t < tw[w] - 1) ? 1u : 0u);
              if (t == first) mma_commit_if_s(el, o_full(w));
            }
            if (t > first && t - 1 < tw[w]) scores(w, ks);
          }
          el = elect_one();
          mma_commit_if_s(el, t_empty(vs));
          if (t > first) {
            mma_commit_if_s(el, t_empty(ks));
            next();
            if (t == first + 1) mma_commit_if_s(el, q_empty);
          }
        }
      }
    } else if (warp == 2 && !failed) {
      // =============================== rows of no sequence ===============================
      const Span all = __ldcg(plan.counts + 6) ? Span{0, 0} : clamped(packed_offset(a.offsets, a.wide, 0), packed_offset(a.offsets, a.wide, a.B), a.Tq);
      const int row16 = a.H * a.D / 8;
#pragma unroll 1
      for (int i = blockIdx.x; i < a.Tq - all.n; i += gridDim.x) {
        uint4* p = static_cast<uint4*>(a.o) + (long long)(i < all.begin ? i : i + all.n) * row16;
        for (int x = lane; x < row16; x += 32) p[x] = make_uint4(0, 0, 0, 0);
      }
    }
  } else {
    // =============================== softmax warpgroups ===============================
    setmaxnreg_inc<kSoftmaxRegs>();
    const int w = (warp >> 2) - 1, row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t tS = t_lane + w * BN, tO = t_lane + C::colO + w * DP;
    const float c = a.scale * kLog2e;
    const F2 c2 = f2_make(c, c);
    const float kInf = __int_as_float(0x7f800000);
    uint32_t g = 0, n = 0, met = 0;  // tiles, items with any, meetings of the warpgroup
    auto meet = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive_s(together(w));
      mbar_wait_s(together(w), met++ & 1, abort_s, DEV_TIMEOUT_SYNC);
    };
#pragma unroll 1
    for (int idx = todo.first(); !todo.over(idx); idx = todo.next()) {
      const Item it = item_at(idx);
      const int rows = rows_of(it, w), first_tile = it.t.begin, end = end_of(it, w);
      const bool valid = row < rows;
      // the last key that this row sees, and the first one that some row of the warp does not
      const int last = a.causal ? min(it.t.n - 1, it.t.shift + (PAIR ? w * BM : 0) + row) : it.t.n - 1;
      const int warp_last = __shfl_sync(0xffffffffu, last, 0), warp_most = __shfl_sync(0xffffffffu, last, 31);
      float m = 0.f, l = 0.f, lu = 0.f;  // l of P as rounded, lu of P as it is
      bool steep = false;
#pragma unroll 1
      for (int t = end - 1; t >= first_tile; --t, ++g) {
        mbar_wait_s(s_full(w), g & 1, abort_s, DEV_TIMEOUT_MMA);
        tc_fence_after();
        const int lim = last - t * BN;  // columns beyond are not seen
        const bool cut = warp_last - t * BN < BN - 1;
        const int pieces = (warp_most - t * BN + 16) >> 4;  // of 16 keys, those that some row sees
        uint32_t pk[BN / 2];
        float lsum = 0.f, lsum_u = 0.f;
        bool go = !__any_sync(0xffffffffu, steep), settled = false;
#pragma unroll 1
        for (;;) {
          bool bad = true;
          if (go) {
            const F2 nm2 = f2_make(-m, -m);
            F2 ls[4], lsu[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) ls[u] = lsu[u] = f2_make(0.f, 0.f);
            auto exps = [&](auto with_mask) {
              constexpr bool kMask = decltype(with_mask)::value;
              uint32_t sr[2][16];
              if (!kMask) tmem_ld16(tS, sr[0]);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                if (kMask && k >= pieces) {
#pragma unroll
                  for (int e = 0; e < 8; ++e) pk[8 * k + e] = 0u;
                  continue;
                }
                if (kMask) tmem_ld16(tS + 16 * k, sr[k & 1]);
                tmem_wait_ld();
                if (!kMask && k < 7) tmem_ld16(tS + 16 * (k + 1), sr[(k + 1) & 1]);
                const uint32_t* s = sr[k & 1];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                  const F2 x = f2_fma(f2_from_bits(s[e], s[e + 1]), c2, nm2);
                  float p0, p1;
                  if (!kMask && on_fma(e / 2)) {
                    exp2_fma<T, true>(x, p0, p1);
                  } else {
                    float x0, x1;
                    f2_get(x, x0, x1);
                    if constexpr (kMask) {
                      x0 = 16 * k + e <= lim ? x0 : -kInf;
                      x1 = 16 * k + e + 1 <= lim ? x1 : -kInf;
                    }
                    p0 = ex2(x0);
                    p1 = ex2(x1);
                  }
                  if constexpr (LSE) lsu[(e / 2) & 3] = f2_add(lsu[(e / 2) & 3], f2_make(p0, p1));
                  const uint32_t both = Pack2<T>::pack(p0, p1);
                  pk[8 * k + e / 2] = both;
                  unpack2<T>(both, p0, p1);
                  ls[(e / 2) & 3] = f2_add(ls[(e / 2) & 3], f2_make(p0, p1));
                }
              }
            };
            if (cut) exps(std::true_type{});
            else exps(std::false_type{});
            auto total = [](const F2 (&x)[4]) {
              float s0, s1;
              f2_get(f2_add(f2_add(x[0], x[1]), f2_add(x[2], x[3])), s0, s1);
              return s0 + s1;
            };
            lsum = total(ls);
            if constexpr (LSE) lsum_u = total(lsu);
            bad = __any_sync(0xffffffffu, valid && !(lsum <= Lag<T>::kMaxSum && (l > 0.f || lim < 0 || lsum >= Lag<T>::kMinSum)));
          }
          if (__builtin_expect(!bad || settled, 1)) break;
          // The tile's own maximum, and the reference follows it.
          float mx = -kInf;
          {
            uint32_t sr[2][32];
            tmem_ld32(tS, sr[0]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              tmem_wait_ld();
              if (k < 3) tmem_ld32(tS + 32 * (k + 1), sr[(k + 1) & 1]);
              const uint32_t* s = sr[k & 1];
              if (cut) {
#pragma unroll
                for (int e = 0; e < 32; e += 2)
                  mx = max3_nan(mx, 32 * k + e <= lim ? __uint_as_float(s[e]) : -kInf, 32 * k + e + 1 <= lim ? __uint_as_float(s[e + 1]) : -kInf);
              } else {
#pragma unroll
                for (int e = 0; e < 32; e += 2) mx = max3_nan(mx, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
              }
            }
          }
          const float m_old = m;
          mx *= c;
          const bool odd = valid && !(mx < kInf);
          if (odd) l = lu = __int_as_float(0x7fffffff);
          const bool fresh = l == 0.f;  // (nothing of the row is in O yet)
          if (valid && !odd && mx != -kInf) m = fresh ? mx : fmaxf(m, mx);
          if (t < end - 1 && __any_sync(0xffffffffu, !fresh && m > m_old)) {
            const float alpha = !fresh && m > m_old ? ex2(m_old - m) : 1.f;
            l *= alpha;
            lu *= alpha;
#pragma unroll 1
            for (int d0 = 0; d0 < DP; d0 += 16) {
              uint32_t o[16];
              tmem_ld16(tO + d0, o);
              tmem_wait_ld();
#pragma unroll
              for (int u = 0; u < 16; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * alpha);
              tmem_st16(tO + d0, o);
            }
          }
          // (scores that rise from tile to tile: the next one's maximum is taken first, and its exponentials once)
          steep = valid && !fresh && m > m_old + Lag<T>::kRise;
          go = settled = true;
        }
        l += lsum;
        lu += lsum_u;
        tmem_st32(tS, *reinterpret_cast<uint32_t(*)[32]>(&pk[0]));
        tmem_st32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&pk[32]));
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_s(p_full(w));
      }
      if (rows == 0) continue;
      const int h = it.h + (PAIR ? 0 : w);
      const long long out_row = it.t.row + (PAIR ? w * BM : 0) + row;
      bool some = end > first_tile;  // there is something in O
      if (some) {
        mbar_wait_s(o_full(w), n & 1, abort_s, DEV_TIMEOUT_MMA);
        ++n;
        tc_fence_after();
      }
      if (it.t.parts > 1) {
        // A part leaves O, m and l; the last part of a tile to arrive adds them up, in their order, back into tensor memory.
        const int u = PAIR ? it.h : it.h / 2;
        auto place = [&](int slot) { return ((long long)slot * units.d + u) * 2 + w; };
        const long long at = place(it.t.slot);
        float4* to = reinterpret_cast<float4*>(plan.sums) + at * (DP / 4 * BM) + row;
#pragma unroll 1
        for (int d = 0; some && d < DP; d += 32) {
          uint32_t r[32];
          tmem_ld32(tO + d, r);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4) to[(d + e) / 4 * BM] = make_float4(__uint_as_float(r[e]), __uint_as_float(r[e + 1]), __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
        }
        plan.ml[at * BM + row] = make_float4(m, some ? l : 0.f, lu, 0.f);
        __threadfence();
        meet();
        if (row == 0) arrived[w] = atomicAdd(plan.arrived + place(it.t.slot - it.t.part), 1);
        meet();
        if (arrived[w] != it.t.parts - 1) {
          tc_fence_before();
          continue;
        }
        __threadfence();
        some = true;
        m = -kInf;
        l = 0.f;
        const int slot0 = it.t.slot - it.t.part;
#pragma unroll 1
        for (int p = 0; p < it.t.parts; ++p) {
          const float4 x = __ldcg(plan.ml + place(slot0 + p) * BM + row);
          if (x.y != 0.f) m = fmaxf(m, x.x);
        }
        if (m == -kInf) m = 0.f;
#pragma unroll 1
        for (int d = 0; d < DP; d += 16) {
          float acc[16] = {};
          l = lu = 0.f;
#pragma unroll 1
          for (int p = 0; p < it.t.parts; ++p) {
            const float4 x = __ldcg(plan.ml + place(slot0 + p) * BM + row);
            const float f = x.y != 0.f ? ex2(x.x - m) : 0.f;
            const float4* from = reinterpret_cast<const float4*>(plan.sums) + place(slot0 + p) * (DP / 4 * BM) + d / 4 * BM + row;
            l = fmaf(x.y, f, l);
            lu = fmaf(x.z, f, lu);
            if (f > 0.f) {  // (a part that this row sees nothing of may have left nothing)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 v = __ldcg(from + e * BM);
                acc[4 * e] = fmaf(v.x, f, acc[4 * e]); acc[4 * e + 1] = fmaf(v.y, f, acc[4 * e + 1]);
                acc[4 * e + 2] = fmaf(v.z, f, acc[4 * e + 2]); acc[4 * e + 3] = fmaf(v.w, f, acc[4 * e + 3]);
              }
            }
          }
          uint32_t r[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(acc[e]);
          tmem_st16(tO + d, r);
        }
        tmem_wait_st();
      }
      const bool any = l != 0.f;
      const int first = (warp & 3) * 32;  // row of the warp's first lane
      store_rows_staged<T, DP>(smem_s + C::offOut + (warp - 4) * kStageBytes, tO, &tmO, (int)(out_row - lane), h, static_cast<T*>(a.o) + ((out_row - lane) * a.H + h) * a.D,
                               (long long)a.H * a.D, rows - first, a.D, any ? 1.f / l : 0.f, some);
      if constexpr (LSE) {
        if (a.o_rest)
          store_rows_staged<T, DP, true>(smem_s + C::offOut + (warp - 4) * kStageBytes, tO, &tmR, (int)(out_row - lane), h,
                                         static_cast<T*>(a.o_rest) + ((out_row - lane) * a.H + h) * a.D, (long long)a.H * a.D, rows - first, a.D, any ? 1.f / l : 0.f, some);
        if (valid) a.lse[(long long)h * a.lse_ld + out_row] = any ? m + log2f(lu) : -kInf;
      }
      tc_fence_before();  // (the next item's first P V, which overwrites O, follows a later arrival)
    }
    stores_done();
  }

  end_of_cta(abort_flag, a.status);
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// Two heads of a group where there are pairs of them, else two query tiles of one head.
bool head_pairs(const PackedArgs& a) { return a.G % 2 == 0; }
PackedCut query_cut(const PackedArgs& a, bool pair) { return PackedCut{100, 10, pair ? a.H : a.H / 2}; }

template <class T, int DP, bool PAIR, bool LSE>
int launch(const PackedArgs& a, void* ws, cudaStream_t st, int* launches) {
  using C = FwdCfg<DP>;
  constexpr int unit = PAIR ? 2 * BM : BM;
  CUtensorMap tq, tk, tv, to, tr;
  const long long so[2] = {(long long)a.H * a.D, a.D};
  if (!make_packed_map(&tq, a.q, a.sq, a.Tq, a.H, a.D) || !make_packed_map(&tk, a.k, a.sk, a.Tk, a.Hk, a.D) || !make_packed_map(&tv, a.v, a.sv, a.Tk, a.Hk, a.D) ||
      !make_packed_map(&to, a.o, so, a.Tq, a.H, a.D, 32) || !make_packed_map(&tr, a.o_rest ? a.o_rest : a.o, so, a.Tq, a.H, a.D, 32))
    return EVOATTN_ERR_CUDA;
  const int sms = sm_count();
  if (sms <= 0) return EVOATTN_ERR_CUDA;
  auto kern = packed_fwd_sm100_kernel<T, DP, PAIR, LSE>;
  int regs = 0;
  if (!kernel_ready(reinterpret_cast<const void*>(kern), (int)C::bytes, &regs)) return EVOATTN_ERR_CUDA;
  // (setmaxnreg.inc would wait for registers that the launch does not have)
  if (kThreads * regs < 256 * kSoftmaxRegs + 128 * kServiceRegs) return EVOATTN_ERR_UNSUPPORTED;
  const PackedCut cut = query_cut(a, PAIR);
  PackedPlan plan = place_plan(a, unit, ws, plan_bytes(a, true, unit, false, sms, cut));
  const int rc = launch_packed_prepare(std::is_same<T, __nv_bfloat16>::value ? EVOATTN_BF16 : EVOATTN_FP16, a, plan, true, unit, false, false, st, launches, cut);
  if (rc) return rc;
  const int heads = PAIR ? a.H : a.H / 2;
  const long long most = (query_units(a, unit) + query_slots(a, unit, sms, cut)) * heads;
  launch_dependent(kern, dim3((unsigned)(most < sms ? most : sms)), kThreads, C::bytes, st, a, plan, FastDiv((uint32_t)heads), tq, tk, tv, to, tr);
  *launches += 1;
  return cudaGetLastError() == cudaSuccess ? EVOATTN_OK : EVOATTN_ERR_CUDA;
}
template <class T, int DP>
int launch_d(const PackedArgs& a, void* ws, cudaStream_t st, int* launches) {
  if (a.lse) return head_pairs(a) ? launch<T, DP, false, true>(a, ws, st, launches) : launch<T, DP, true, true>(a, ws, st, launches);
  return head_pairs(a) ? launch<T, DP, false, false>(a, ws, st, launches) : launch<T, DP, true, false>(a, ws, st, launches);
}

}  // namespace

bool sm100_packed_supported(int dtype, const PackedArgs& a) {
  if (dtype == EVOATTN_FP32 || a.D % 8 || a.D > 128 || !(a.scale > 0.f)) return false;
  // (numbers of items fit 31 bits)
  if ((a.Tq / kTileRows + a.B) * (long long)a.H >= 1LL << 31 || (a.Tk / kTileRows + a.B) * (long long)a.Hk >= 1LL << 31) return false;
  if ((reinterpret_cast<uintptr_t>(a.o) | reinterpret_cast<uintptr_t>(a.o_rest)) & 15) return false;
  return packed_map_ok(a.q, a.sq, a.Tq, a.H) && packed_map_ok(a.k, a.sk, a.Tk, a.Hk) && packed_map_ok(a.v, a.sv, a.Tk, a.Hk);
}
size_t sm100_packed_fwd_workspace_bytes(const PackedArgs& a) { return plan_bytes(a, true, head_pairs(a) ? BM : 2 * BM, false, sm_count(), query_cut(a, !head_pairs(a))).all(); }
int launch_sm100_packed_fwd(int dtype, const PackedArgs& a, void* ws, cudaStream_t st, int* launches) {
  if (dtype == EVOATTN_BF16) return a.D <= 64 ? launch_d<__nv_bfloat16, 64>(a, ws, st, launches) : launch_d<__nv_bfloat16, 128>(a, ws, st, launches);
  return a.D <= 64 ? launch_d<__half, 64>(a, ws, st, launches) : launch_d<__half, 128>(a, ws, st, launches);
}

}  // namespace evo
