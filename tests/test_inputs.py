"""CPU: the operators before the attention, as far as they go without a GPU: the borders of logarithmic buckets, what
the entry points refuse, the C ABI's structs and status codes."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from oracle import inputs_oracle as oc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("scheme", ["log", "log_causal"])
@pytest.mark.parametrize("n,M", [(4, 2), (8, 5), (32, 128), (32, 127), (64, 1000), (256, 100000)])
def test_log_edges_are_the_borders_of_the_buckets(scheme, n, M):
    from evoformer_triton_b200.inputs import _log_buckets
    exact, edges = _log_buckets(n, M, scheme == "log_causal")
    side = n if scheme == "log_causal" else n // 2
    assert len(edges) == side - exact - 1 and edges == sorted(edges)
    for a in sorted({d + k for d in edges + [exact, M] for k in (-1, 0, 1)} | set(range(40))):
        want = oc.bucket(-a, scheme, n, M)
        assert (a if a < exact else exact + sum(e <= a for e in edges)) == want, a


def test_powers_of_two_begin_a_bucket():
    """32 buckets up to 128: 8 * 2 ** (k / 2), whole for even k, where a logarithm in floating point may say less."""
    from evoformer_triton_b200.inputs import _log_buckets
    assert _log_buckets(32, 128, False) == (8, [12, 16, 23, 32, 46, 64, 91])


def test_structs_match_the_header(tmp_path):
    from evoformer_triton_b200 import _lib
    pairs = (("evoattn_layer_norm_params", _lib.LayerNormParams), ("evoattn_relative_bias_params", _lib.RelativeBiasParams),
             ("evoattn_pair_projection_params", _lib.PairProjectionParams))
    rows = [(c, f[0]) for c, p in pairs for f in p._fields_]
    src = tmp_path / "sz.c"
    src.write_text('#include "evoattn.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){' +
                   "".join(f'printf("%zu\\n", sizeof({c}));' for c, _ in pairs) +
                   "".join(f'printf("%zu\\n", offsetof({c}, {f}));' for c, f in rows) + "return 0;}\n")
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    assert got == [C.sizeof(p) for _, p in pairs] + [getattr(p, f[0]).offset for _, p in pairs for f in p._fields_]


def test_c_entries_refuse_without_a_gpu(built_library):
    """Addresses are made up: none of these calls gets as far as a launch."""
    from evoformer_triton_b200 import _lib
    lib = _lib.load()
    n = _lib.LayerNormParams(n=(2, 3, 4), C=8, eps=1e-5, x=256, y=512)
    assert lib.evoattn_layer_norm_fwd(None, None) == 1 and lib.evoattn_layer_norm_bwd(None, None) == 1
    assert lib.evoattn_layer_norm_bwd_workspace_bytes(None) == 0
    for field, value, rc in (("dtype", 3, 3), ("dtype", -1, 3), ("C", 0, 2), ("eps", -1.0, 2), ("eps", float("nan"), 2), ("x", None, 1), ("y", None, 1)):
        keep = getattr(n, field)
        setattr(n, field, value)
        assert lib.evoattn_layer_norm_fwd(C.byref(n), None) == rc, field
        setattr(n, field, keep)
    n.n[1] = -1
    assert lib.evoattn_layer_norm_fwd(C.byref(n), None) == 2
    n.n[1] = 1 << 50
    assert lib.evoattn_layer_norm_fwd(C.byref(n), None) == 2
    n.n[1] = 0
    assert lib.evoattn_layer_norm_fwd(C.byref(n), None) == 0  # no rows: nothing to do
    n.n[1] = 3
    n.dweight, n.d_y, n.stats, n.weight = 1024, 2048, 4096, 8192
    assert lib.evoattn_layer_norm_bwd(C.byref(n), None) == 7
    n.workspace, n.workspace_bytes = 260, lib.evoattn_layer_norm_bwd_workspace_bytes(C.byref(n))
    assert lib.evoattn_layer_norm_bwd(C.byref(n), None) == 4
    n.workspace, n.stats = 256, None
    assert lib.evoattn_layer_norm_bwd(C.byref(n), None) == 1

    r = _lib.RelativeBiasParams(B=1, H=2, Rq=3, Rk=4, buckets=65, exact=32, table=256, q_pos=256, k_pos=256, out=512)
    assert lib.evoattn_relative_bias_fwd(None, None) == 1
    for field, value, rc in (("dtype", 9, 3), ("table_dtype", 9, 3), ("H", 0, 2), ("Rq", -1, 2), ("buckets", 64, 2), ("buckets", 1025, 2),
                             ("scheme", 3, 2), ("n_edges", 1, 1), ("n_edges", 129, 2), ("exact", -1, 2), ("table", None, 1), ("out", None, 1)):
        keep = getattr(r, field)
        setattr(r, field, value)
        assert lib.evoattn_relative_bias_fwd(C.byref(r), None) == rc, field
        setattr(r, field, keep)
    r.edges, r.n_edges, r.scheme, r.exact, r.buckets = (C.c_int32 * 2)(9, 8), 2, 1, 8, 32
    assert lib.evoattn_relative_bias_fwd(C.byref(r), None) == 2      # edges go down
    r.edges = (C.c_int32 * 2)(7, 9)
    assert lib.evoattn_relative_bias_fwd(C.byref(r), None) == 2      # an edge below the exact distances
    r.edges, r.buckets = (C.c_int32 * 2)(8, 9), 20
    assert lib.evoattn_relative_bias_fwd(C.byref(r), None) == 2      # 8 + 2 is no row of ten
    r.buckets = 32
    assert lib.evoattn_relative_bias_bwd(C.byref(r), None) == 1      # no dtable
    r.dtable, r.d_out = 512, 512
    assert lib.evoattn_relative_bias_bwd(C.byref(r), None) == 7

    p = _lib.PairProjectionParams(B=1, Ri=2, Rj=3, C=8, H=2, eps=1e-5, pair=256, weight=256, out=512)
    assert lib.evoattn_pair_projection_fwd(None, None) == 1
    for field, value, rc in (("dtype", 5, 3), ("weight_dtype", 5, 3), ("C", 0, 2), ("C", 513, 5), ("H", 65, 5), ("H", 0, 2), ("Ri", -1, 2), ("eps", -1.0, 2),
                             ("pair", None, 1), ("weight", None, 1), ("out", None, 1)):
        keep = getattr(p, field)
        setattr(p, field, value)
        assert lib.evoattn_pair_projection_fwd(C.byref(p), None) == rc, field
        setattr(p, field, keep)
    p.d_out, p.dweight = 512, 512
    assert lib.evoattn_pair_projection_bwd(C.byref(p), None) == 7


def test_operators_refuse_tensors_without_a_gpu():
    import evoformer_triton_b200 as evo
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        evo.layer_norm(torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        evo.relative_position_bias(torch.zeros(65, 3), torch.arange(3), max_distance=32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        evo.pair_bias_projection(torch.zeros(1, 2, 2, 4), torch.zeros(2, 4))


@pytest.mark.parametrize("rows,kw", [(64, dict(max_distance=32)), (1025, dict(max_distance=512)), (1, dict(max_distance=-1)),
                                     (30, dict(max_distance=128, buckets="log")), (31, dict(max_distance=128, buckets="log_causal")),
                                     (260, dict(max_distance=1024, buckets="log")), (32, dict(max_distance=8, buckets="log")),
                                     (32, dict(max_distance=1 << 20, buckets="log")), (32, dict(max_distance=16, buckets="log_causal")),
                                     (65, dict(max_distance=32, buckets="other"))])
def test_bucket_parameters_that_do_not_fit(rows, kw):
    import evoformer_triton_b200 as evo
    with pytest.raises(ValueError):
        evo.relative_position_bias(torch.zeros(rows, 2), torch.arange(3), **kw)


@pytest.mark.parametrize("scheme,n,M", [("clip", 9, 4), ("log", 12, 20), ("log_causal", 10, 30)])
def test_oracle_gradients_against_differences(scheme, n, M):
    """The oracle's closed forms against differences of its forward, in 64 bits."""
    g = torch.Generator().manual_seed(n)
    draw = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731

    def differences(f, x, e=1e-6):
        out = torch.zeros_like(x)
        for i in range(x.numel()):
            up, down = x.clone(), x.clone()
            up.view(-1)[i] += e
            down.view(-1)[i] -= e
            out.view(-1)[i] = (f(up) - f(down)) / (2 * e)
        return out

    x, w, b, d = draw(3, 5), draw(5), draw(5), draw(3, 5)
    got = oc.layer_norm(x, w, b, 1e-3, d)
    for k, f in ((1, lambda t: oc.layer_norm(t, w, b, 1e-3)[0][0]), (2, lambda t: oc.layer_norm(x, t, b, 1e-3)[0][0]), (3, lambda t: oc.layer_norm(x, w, t, 1e-3)[0][0])):
        assert torch.allclose(got[k][0], differences(lambda t: (f(t) * d).sum(), (None, x, w, b)[k]), atol=1e-7)
    z, W, dz = draw(1, 2, 3, 5), draw(2, 5), draw(1, 1, 2, 2, 3)
    got = oc.pair_projection(z, W, w, b, 1e-3, dz)
    for k in range(4):
        def f(t, k=k):
            a = [z, W, w, b]
            a[k] = t
            return (oc.pair_projection(*a, 1e-3)[0][0] * dz).sum()
        assert torch.allclose(got[k + 1][0], differences(f, (z, W, w, b)[k]), atol=1e-7), k
    rows = oc.bucket_rows([[0, 1, 7]], [[0, 3, 9, 40]], scheme, n, M)
    table, d = draw(n, 2), draw(1, 1, 2, 3, 4)
    lookup = lambda t: (t[rows].permute(0, 3, 1, 2).unsqueeze(1) * d).sum()  # noqa: E731
    assert torch.allclose(oc.relative_bias(table, rows, None, torch.float64, d)[1][0], differences(lookup, table), atol=1e-7)
