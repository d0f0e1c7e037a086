"""CPU: rotary positions and packed attention as far as they go without a GPU: the frequencies, the oracle against
differentiation, what the entry points refuse, the C ABI's structs and status codes."""
import ctypes as C
import math
import os
import subprocess

import pytest
import torch

from oracle import sequences_oracle as oc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_frequencies():
    import evoformer_triton_b200 as evo
    f = evo.rotary_frequencies(64, 500.0)
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1
    assert torch.allclose(f, torch.tensor([500.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-14)
    assert torch.allclose(evo.rotary_frequencies(64, 500.0, scaling="linear", factor=4.0), f / 4)
    g = evo.rotary_frequencies(64, 500.0, scaling="base", factor=4.0)
    assert g[0] == 1 and math.isclose(float(g[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    b = evo.rotary_frequencies(64, 500.0, scaling="bands", factor=4.0, original_length=1000)
    turns = 1000 * f / (2 * math.pi)
    assert (turns < 1).any() and (turns > 4).any() and ((turns > 1) & (turns < 4)).any()
    assert torch.allclose(b[turns < 1], f[turns < 1] / 4) and torch.equal(b[turns > 4], f[turns > 4])
    mid = (turns > 1) & (turns < 4)
    assert ((b[mid] > f[mid] / 4) & (b[mid] < f[mid])).all()
    assert evo.rotary_frequencies(2, scaling="base", factor=8.0).tolist() == [1.0]


@pytest.mark.parametrize("kw", [dict(dim=3), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, factor=-1.0), dict(dim=8, scaling="other"),
                                dict(dim=8, scaling="bands"), dict(dim=8, scaling="bands", original_length=10, slow=4.0, fast=4.0),
                                dict(dim=8, base=math.nan)], ids=str)
def test_frequencies_refuse(kw):
    import evoformer_triton_b200 as evo
    with pytest.raises(ValueError):
        evo.rotary_frequencies(**kw)


@pytest.mark.parametrize("causal", [True, False])
def test_oracle_gradients_are_those_of_its_output(causal):
    """The formulas of the backward against differentiating the forward, and against differences."""
    g = torch.Generator().manual_seed(1)
    spans = [(1, 3, 0, 5), (4, 4, 5, 2), (8, 1, 7, 1), (9, 0, 8, 2), (9, 2, 10, 0), (11, 3, 11, 3)]
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((15, 4, 6), (15, 2, 6), (15, 2, 6)))
    d = torch.randn(q.shape, generator=g, dtype=torch.float64)

    def forward(q, k, v):
        out = torch.zeros_like(q)
        for i0, nq, j0, nk in spans:
            for h in range(4):
                for i in range(nq):
                    n = min(nk, max(0, i + nk - nq + 1)) if causal else nk
                    if n:
                        w = torch.softmax(q[i0 + i, h] @ k[j0:j0 + n, h // 2].t() / math.sqrt(6), -1)
                        out[i0 + i, h] = w @ v[j0:j0 + n, h // 2]
        return out

    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = forward(*leaves)
    want = [out, *torch.autograd.grad(out, leaves, d)]
    # (the oracle's bounds are of the storage types: values only, here)
    got = [t for t, _ in oc.attention(q, k, v, spans, causal, d=d)]
    for a, b in zip(got, want):
        assert torch.allclose(a, b.detach(), rtol=1e-11, atol=1e-12)
    for n, grad in enumerate(got[1:]):
        step = torch.randn((q, k, v)[n].shape, generator=g, dtype=torch.float64)
        args = lambda x: [t + x * step if m == n else t for m, t in enumerate((q, k, v))]  # noqa: E731
        slope = ((forward(*args(1e-5)) - forward(*args(-1e-5))) * d).sum() / 2e-5
        assert torch.allclose(slope, (grad * step).sum(), rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_oracle_turns(layout):
    """A turn by a whole number of quarter turns, and back."""
    x = torch.arange(1.0, 7.0, dtype=torch.float64).reshape(1, 1, 6)
    f = torch.tensor([math.pi / 2, math.pi], dtype=torch.float64)
    y, _ = oc.rotary(x, torch.tensor([1]), f, layout)
    want = [-3.0, -2, 1, -4, 5, 6] if layout == "half" else [-2.0, 1, -3, -4, 5, 6]
    assert torch.allclose(y.flatten(), torch.tensor(want, dtype=torch.float64))
    z, _ = oc.rotary(y, torch.tensor([1]), f, layout, inverse=True)
    assert torch.allclose(z, x)


def test_structs_match_the_header(tmp_path):
    from evoformer_triton_b200 import _lib
    pairs = (("evoattn_rotary_params", _lib.RotaryParams), ("evoattn_packed_params", _lib.PackedParams))
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

    def refused(fn, p, cases):
        for field, value, rc in cases:
            keep = getattr(p, field)
            setattr(p, field, value)
            assert fn(C.byref(p), None) == rc, (field, value)
            setattr(p, field, keep)

    r = _lib.RotaryParams(n=(1, 1, 4), H=2, Hk=1, D=8, rotary=8, q=256, q_out=512, k=768, k_out=1024, positions=256, frequencies=256, amplitude=1.0)
    assert lib.evoattn_rotary(None, None) == 1
    refused(lib.evoattn_rotary, r, [("dtype", 3, 3), ("dtype", -1, 3), ("positions", None, 1), ("frequencies", None, 1), ("q_out", None, 1), ("k_out", None, 1),
                                    ("D", 0, 2), ("D", 1025, 2), ("rotary", 7, 2), ("rotary", 10, 2), ("rotary", 0, 2), ("H", 0, 2), ("Hk", 0, 2),
                                    ("amplitude", math.nan, 2), ("layout", 2, 3), ("layout", -1, 3)])
    r.n[1] = 0
    assert lib.evoattn_rotary(C.byref(r), None) == 2
    r.n[1] = 1 << 30
    assert lib.evoattn_rotary(C.byref(r), None) == 2

    p = _lib.PackedParams(B=2, H=4, Hk=2, D=64, Tq=10, Tk=10, scale=1.0, q=256, k=256, v=256, o=256, offsets=256)
    assert lib.evoattn_packed_fwd(None, None) == 1 and lib.evoattn_packed_bwd(None, None) == 1
    assert lib.evoattn_packed_fwd_workspace_bytes(None) == 0 and lib.evoattn_packed_bwd_workspace_bytes(None) == 0
    refused(lib.evoattn_packed_fwd, p, [("dtype", 3, 3), ("q", None, 1), ("k", None, 1), ("v", None, 1), ("o", None, 1), ("offsets", None, 1), ("B", 0, 2),
                                        ("H", 0, 2), ("H", 3, 2), ("Hk", 0, 2), ("H", 65536, 2), ("D", 0, 2), ("D", 257, 5), ("Tq", 0, 2), ("Tk", (1 << 30) + 1, 2),
                                        ("key_form", 2, 3), ("key_form", 1, 1), ("scale", math.nan, 2), ("scale", math.inf, 2)])
    assert lib.evoattn_packed_bwd(C.byref(p), None) == 1  # no lse
    p.lse = p.d_o = p.dq = p.dk = p.dv = 256
    assert lib.evoattn_packed_bwd(C.byref(p), None) == 7  # no workspace
    need = lib.evoattn_packed_bwd_workspace_bytes(C.byref(p))
    assert need >= 4 * 10 * 4
    p.workspace, p.workspace_bytes = 256, need - 1
    assert lib.evoattn_packed_bwd(C.byref(p), None) == 7
    p.workspace, p.workspace_bytes = 128, need
    assert lib.evoattn_packed_bwd(C.byref(p), None) == 4
    p.workspace = 256
    refused(lib.evoattn_packed_bwd, p, [("dk", None, 1), ("dv", None, 1), ("d_o", None, 1)])
    p.key_form, p.key_offsets = 1, 256
    assert lib.evoattn_packed_bwd(C.byref(p), None) == 5  # ranges have no gradient


def test_cpu_tensors_and_names_are_refused(built_library):
    import evoformer_triton_b200 as evo
    x, off = torch.zeros(4, 2, 8), torch.tensor([0, 4])
    with pytest.raises(RuntimeError, match="CUDA"):
        evo.packed_attention(x, x, x, off)
    with pytest.raises(RuntimeError, match="CUDA"):
        evo.rotary_embedding(x, x, torch.arange(4), torch.ones(4))
    with pytest.raises(ValueError, match="layout"):
        evo.rotary_embedding(x, x, torch.arange(4), torch.ones(4), layout="other")
