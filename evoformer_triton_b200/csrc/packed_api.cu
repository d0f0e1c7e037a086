// Attention over packed sequences: what a request has to hold, and which kernels serve it.
#include "packed_sm100.cuh"

namespace evo {
namespace {

constexpr long long kMaxRows = 1LL << 30;

int validate(const evoattn_packed_params* p, bool bwd) {
  if (!p || !p->q || !p->k || !p->v || !p->offsets || !p->o) return EVOATTN_ERR_NULL;
  if (!known_dtype(p->dtype)) return EVOATTN_ERR_DTYPE;
  if (p->B < 1 || p->H < 1 || p->Hk < 1 || p->H % p->Hk || p->H > 65535 || p->D < 1) return EVOATTN_ERR_SHAPE;
  if (p->Tq < 1 || p->Tk < 1 || p->Tq > kMaxRows || p->Tk > kMaxRows || p->B > kMaxRows || p->Tq * p->H > 8 * kMaxRows) return EVOATTN_ERR_SHAPE;
  if (p->D > EVOATTN_PACKED_MAX_D) return EVOATTN_ERR_UNSUPPORTED;
  if (p->key_form != EVOATTN_PACKED_KEY_OFFSETS && p->key_form != EVOATTN_PACKED_KEY_RANGES) return EVOATTN_ERR_DTYPE;
  if (p->key_form == EVOATTN_PACKED_KEY_RANGES && !p->key_offsets) return EVOATTN_ERR_NULL;
  if (!(p->scale - p->scale == 0.f)) return EVOATTN_ERR_SHAPE;  // (NaN or infinite)
  if (p->o_rest && !p->lse) return EVOATTN_ERR_NULL;  // (only the kernels for training leave it)
  if (!bwd) return EVOATTN_OK;
  if (!p->lse || !p->d_o || !p->dk != !p->dv) return EVOATTN_ERR_NULL;
  if (p->dk && p->key_form != EVOATTN_PACKED_KEY_OFFSETS) return EVOATTN_ERR_UNSUPPORTED;
  return EVOATTN_OK;
}

PackedArgs arguments(const evoattn_packed_params* p) {
  PackedArgs a{};
  a.q = p->q; a.k = p->k; a.v = p->v; a.o = p->o; a.o_rest = p->o_rest; a.lse = p->lse;
  a.d_o = p->d_o; a.dq = p->dq; a.dk = p->dk; a.dv = p->dv;
  for (int i = 0; i < 2; ++i) a.sq[i] = p->q_stride[i], a.sk[i] = p->k_stride[i], a.sv[i] = p->v_stride[i], a.sdo[i] = p->do_stride[i];
  a.offsets = p->offsets;
  a.key_offsets = p->key_offsets ? p->key_offsets : p->offsets;
  a.B = p->B; a.H = p->H; a.Hk = p->Hk; a.D = p->D; a.G = p->H / p->Hk;
  a.causal = p->causal != 0; a.wide = p->offsets64 != 0; a.ranges = p->key_form == EVOATTN_PACKED_KEY_RANGES;
  a.Tq = (int)p->Tq; a.Tk = (int)p->Tk; a.lse_ld = (int)p->Tq;
  a.scale = p->scale;
  a.status = p->status;
  return a;
}

bool tensor_cores(const evoattn_packed_params* p, const PackedArgs& a, bool bwd) {
  return !(p->flags & EVOATTN_FLAG_FORCE_GENERIC) && (bwd ? sm100_packed_bwd_supported(p->dtype, a) : sm100_packed_supported(p->dtype, a));
}
// Which kernels a forward takes, and their scratch.  The host knows how many sequences and queries there are, not how they
// fall.  Sequences of a few queries against keys of their own go to packed_few.cu, the others to the tiles; calls whose
// queries are few altogether go there as a whole (the worst is that all queries are one sequence's: 64 units then),
// which saves the launches for the tiles.
struct Forward {
  bool generic, few, tiles;
  size_t few_bytes, tile_bytes;
  size_t bytes() const { return few_bytes + tile_bytes; }
};
int few_tokens(const PackedArgs& a) { return a.G > 16 ? 2 : 32 / a.G; }
Forward forward_plan(const evoattn_packed_params* p, const PackedArgs& a) {
  Forward f{!tensor_cores(p, a, false), false, false, 0, 0};
  if (f.generic) return f;
  const bool own_keys = p->key_offsets && !p->lse;
  const bool all_few = own_keys && a.Tq <= (long long)few_tokens(a) * a.B && (long long)a.Tq * a.G <= 1024;
  f.few = own_keys && (a.B > 1 || all_few);
  f.tiles = !all_few;
  if (f.few) f.few_bytes = (packed_few_workspace_bytes(a) + 255) / 256 * 256;
  if (f.tiles) f.tile_bytes = sm100_packed_fwd_workspace_bytes(a);
  return f;
}
int check_workspace(const evoattn_packed_params* p, size_t need) {
  if (!need) return EVOATTN_OK;
  if (!p->workspace || p->workspace_bytes < need) return EVOATTN_ERR_WORKSPACE;
  return (uintptr_t)p->workspace & 255 ? EVOATTN_ERR_ALIGN : EVOATTN_OK;
}

}  // namespace
}  // namespace evo

extern "C" {

using namespace evo;

size_t evoattn_packed_fwd_workspace_bytes(const evoattn_packed_params* p) {
  if (validate(p, false)) return 0;
  const PackedArgs a = arguments(p);
  return forward_plan(p, a).bytes();
}

int evoattn_packed_fwd(const evoattn_packed_params* p, void* cuda_stream) {
  int rc = validate(p, false);
  if (rc) return rc;
  PackedArgs a = arguments(p);
  const Forward f = forward_plan(p, a);
  rc = check_workspace(p, f.bytes());
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  bind_context_once();
  int launches = 0;
  if (f.generic) {
    rc = launch_packed_generic_fwd(p->dtype, a, st, &launches);
  } else {
    if (f.few) {
      a.few_tokens = f.tiles ? few_tokens(a) : a.Tq;
      rc = launch_packed_few(p->dtype, a, !f.tiles, p->workspace, st, &launches);
    }
    if (!rc && f.tiles) rc = launch_sm100_packed_fwd(p->dtype, a, static_cast<unsigned char*>(p->workspace) + f.few_bytes, st, &launches);
  }
  note_call(f.generic ? EVOATTN_PATH_GENERIC : EVOATTN_PATH_TCGEN05, launches);
  return rc;
}

size_t evoattn_packed_bwd_workspace_bytes(const evoattn_packed_params* p) {
  if (validate(p, true)) return 0;
  const PackedArgs a = arguments(p);
  return tensor_cores(p, a, true) ? sm100_packed_bwd_workspace_bytes(a) : 256 + (size_t)p->H * p->Tq * sizeof(float);
}

int evoattn_packed_bwd(const evoattn_packed_params* p, void* cuda_stream) {
  int rc = validate(p, true);
  if (rc) return rc;
  rc = check_workspace(p, evoattn_packed_bwd_workspace_bytes(p));
  if (rc) return rc;
  PackedArgs a = arguments(p);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  bind_context_once();
  int launches = 0;
  const bool fast = tensor_cores(p, a, true);
  if (fast) {
    rc = launch_sm100_packed_bwd(p->dtype, a, p->workspace, st, &launches);
  } else {
    PackedPlan plan{};
    plan.counts = static_cast<int*>(p->workspace);
    a.overlap = plan.counts + 6;
    a.delta = reinterpret_cast<float*>(static_cast<unsigned char*>(p->workspace) + 256);
    rc = launch_packed_prepare(p->dtype, a, plan, false, 0, false, true, st, &launches);
    if (!rc) rc = launch_packed_generic_bwd(p->dtype, a, st, &launches);
  }
  note_call(fast ? EVOATTN_PATH_TCGEN05 : EVOATTN_PATH_GENERIC, launches);
  return rc;
}

}  // extern "C"
