"""GPU: the pair-bias projection against its definition in 64 bits, and the three operators together with the attention."""
import pytest
import torch

from oracle import evo_oracle, inputs_oracle as oc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _draw(shape, dtype, seed, std=1.0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)


def _against_oracle(z, W, g, b, d=None, eps=1e-5):
    import evoformer_triton_b200 as evo
    leaves = [t.requires_grad_() for t in (z, W, g, b) if t is not None]
    out = evo.pair_bias_projection(z, W, g, b, eps=eps)
    B, I, J, C = z.shape
    assert out.shape == (B, 1, W.shape[0], I, J) and out.dtype == z.dtype
    es = out.element_size()
    assert out.data_ptr() % 16 == 0 and all(s * es % 16 == 0 for s in out.stride()[:4])
    with torch.no_grad():
        assert torch.equal(evo.pair_bias_projection(z, W, g, b, eps=eps), out)
    if d is None:
        d = _draw(out.shape, out.dtype, 9)
    grads = torch.autograd.grad(out, leaves, d)
    plain = [t if t is None else t.detach() for t in (z, W, g, b)]
    want = oc.pair_projection(*plain, eps, d)
    oc.check("out", out, want[0])
    for name, t, got, w in zip(("dpair", "dweight", "dnorm_weight", "dnorm_bias"), leaves, grads, [w for w in want[1:] if w is not None]):
        assert got.dtype == t.dtype and got.shape == t.shape
        oc.check(name, got, w)


def _weights(H, C, dtype=F32, affine=True):
    return _draw((H, C), dtype, 2, C ** -0.5), _draw((C,), dtype, 3, 0.2, 1.0) if affine else None, _draw((C,), dtype, 4, 0.2) if affine else None


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,I,J,C,H", [(1, 1, 1, 1, 1), (1, 1, 1, 128, 8), (1, 3, 5, 7, 3), (2, 9, 9, 32, 4), (1, 17, 17, 64, 1), (1, 31, 33, 128, 4), (2, 40, 40, 128, 8),
                                       (1, 20, 50, 100, 5), (1, 24, 24, 256, 8), (1, 16, 16, 192, 16), (1, 12, 12, 384, 12), (1, 10, 14, 512, 64), (1, 7, 200, 130, 9),
                                       (1, 64, 64, 48, 32), (1, 101, 101, 128, 4), (1, 300, 260, 32, 2), (1, 30, 41, 100, 12), (1, 30, 41, 99, 16),
                                       (1, 9, 30, 300, 10), (1, 9, 30, 301, 40)], ids=str)
def test_sizes(B, I, J, C, H, dtype):
    _against_oracle(_draw((B, I, J, C), dtype, 1, 2.0, 0.3), *_weights(H, C))


@pytest.mark.parametrize("weights", [BF, HF, F32, "none", "gain", "bias"], ids=str)
def test_weights_of_other_types_or_none(weights):
    W, g, b = _weights(8, 128, weights if isinstance(weights, torch.dtype) else BF)
    _against_oracle(_draw((1, 33, 40, 128), BF, 1), W, None if weights in ("none", "bias") else g, None if weights in ("none", "gain") else b)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
def test_weights_of_any_size(dtype):
    """Heads whose weights differ by twelve orders of magnitude, zero among them, and gains that differ by four."""
    W, g, b = _weights(8, 128)
    W = W * torch.tensor([1e-9, 1e-6, 1e-3, 1.0, 30.0, 1e3, 0.0, -1.0], device=DEV)[:, None]
    g = g * torch.logspace(-2, 2, 128, device=DEV)
    _against_oracle(_draw((1, 20, 33, 128), dtype, 1), W, g, b, d=_draw((1, 1, 8, 20, 33), dtype, 5) * 0.01)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("C", [64, 50])
def test_pair_is_read_where_it_lies(C, dtype):
    W, g, b = _weights(4, C)
    for z in (_draw((2, 21, 18, C), dtype, 1).transpose(1, 2), _draw((2, 21, 18, 2 * C), dtype, 1)[..., C:], _draw((2, 21, 18, C + 1), dtype, 1)[..., 1:],
              _draw((2, C, 21, 18), dtype, 1).permute(0, 2, 3, 1), _draw((4, 42, 36, C), dtype, 1)[::2, ::2, ::2], _draw((1, 1, 18, C), dtype, 1).expand(2, 21, 18, C)):
        _against_oracle(z.detach(), W.detach(), g.detach(), b.detach())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_gradients_of_any_layout(dtype):
    B, R, C, H = 2, 37, 64, 4
    full = _draw((B, 1, H, R, R), dtype, 5)
    for d in (full.transpose(3, 4), full.permute(0, 1, 3, 4, 2).contiguous().permute(0, 1, 4, 2, 3), _draw((1,), dtype, 4).expand(B, 1, H, R, R),
              _draw((B, 1, H, R, 48), dtype, 5)[..., :R], _draw((B, 1, H, R, 49), dtype, 5)[..., 3:R + 3]):
        _against_oracle(_draw((B, R, R, C), dtype, 1), *_weights(H, C), d=d)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("C", [128, 320])
def test_rows_far_from_zero_constant_rows_and_large_values(C, dtype):
    z = _draw((1, 4, 12, C), dtype, 1)
    z[0, 0, 0:3] = _draw((3, C), dtype, 2, 1.0, 1000.0)
    z[0, 1, 3], z[0, 1, 4] = 7.0, 0.0
    z[0, 2, 5] = _draw((C,), dtype, 3, 1e4 if dtype == HF else 1e8)
    z[0, 3, 6] = _draw((C,), dtype, 3, 1e-4)
    _against_oracle(z, *_weights(8, C))


def test_values_that_are_not_finite_stay_in_their_rows():
    import evoformer_triton_b200 as evo
    z, (W, g, b) = _draw((1, 30, 30, 128), BF, 1), _weights(8, 128)
    clean = evo.pair_bias_projection(z, W, g, b)
    z[0, 3, 4, 5], z[0, 17, 29, 127], z[0, 29, 29, 0] = float("nan"), float("inf"), float("-inf")
    bad = torch.zeros(30, 30, dtype=torch.bool, device=DEV)
    bad[[3, 17, 29], [4, 29, 29]] = True
    zr = z.requires_grad_()
    out = evo.pair_bias_projection(zr, W, g, b)
    assert torch.equal(out[0, 0][:, ~bad], clean[0, 0][:, ~bad]) and torch.isnan(out[0, 0][:, bad]).all()
    dz, = torch.autograd.grad(out, zr, torch.ones_like(out))
    assert torch.isfinite(dz[0][~bad]).all() and torch.isnan(dz[0][bad]).all()


@pytest.mark.parametrize("shape", [(0, 5, 5, 64), (2, 0, 0, 64), (1, 3, 0, 64)], ids=str)
def test_nothing_to_project(shape):
    import evoformer_triton_b200 as evo
    z = torch.zeros(shape, device=DEV, requires_grad=True)
    leaves = [z] + [t.requires_grad_() for t in _weights(4, 64)]
    out = evo.pair_bias_projection(*leaves)
    assert out.shape == (shape[0], 1, 4, shape[1], shape[2])
    grads = torch.autograd.grad(out, leaves, torch.zeros_like(out))
    assert grads[0].shape == shape and not any(t.any() for t in grads[1:])


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (3,), (0, 1), (1, 3)], ids=str)
def test_only_the_gradients_that_are_wanted(wanted):
    import evoformer_triton_b200 as evo
    a = [_draw((1, 50, 50, 128), BF, 1), *_weights(8, 128)]
    for i in wanted:
        a[i].requires_grad_()
    d = _draw((1, 1, 8, 50, 50), BF, 9)
    got = torch.autograd.grad(evo.pair_bias_projection(*a), [a[i] for i in wanted], d)
    want = oc.pair_projection(*[t.detach() for t in a], 1e-5, d)
    for i, t in zip(wanted, got):
        oc.check(str(i), t, want[1 + i])


def test_refusals():
    import evoformer_triton_b200 as evo
    z, (W, g, b) = _draw((1, 4, 4, 64), F32, 1), _weights(4, 64)
    for bad in (lambda: evo.pair_bias_projection(z.double(), W), lambda: evo.pair_bias_projection(z, W.double()), lambda: evo.pair_bias_projection(z, W, g.double())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: evo.pair_bias_projection(z[0], W), lambda: evo.pair_bias_projection(z, W[:, :63]), lambda: evo.pair_bias_projection(z, W[0]),
                lambda: evo.pair_bias_projection(z, W, g[:63]), lambda: evo.pair_bias_projection(z, W, g, b[None]), lambda: evo.pair_bias_projection(z, W, eps=-1.0),
                lambda: evo.pair_bias_projection(z, torch.zeros(65, 64, device=DEV)), lambda: evo.pair_bias_projection(torch.zeros(1, 2, 2, 513, device=DEV), torch.zeros(1, 513, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        evo.pair_bias_projection(z, W.cpu())
    z.requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(evo.pair_bias_projection(z, W).sum(), z, create_graph=True)


# ---------------------------------------------------------------- together, as a block runs them

def _block(p, m, z, pos, mask):
    """MSA row attention with pair bias: norms, projections, the relative bias added to the pair bias, attention."""
    import evoformer_triton_b200 as evo
    B, S, R, _ = m.shape
    x = evo.layer_norm(m, p["m_w"], p["m_b"])
    H = p["table"].shape[1]
    q, k, v, gate = ((x @ p[n]).view(B, S, R, H, -1) for n in ("q", "k", "v", "gate"))
    bias = evo.pair_bias_projection(z, p["w"], p["z_w"], p["z_b"])
    bias = evo.relative_position_bias(p["table"], pos, max_distance=32, pair_bias=bias)
    return evo.evoformer_attention(q, k, v, [mask, bias], gate=gate)


def _parameters(C, Cz, H, D, seed, dtype=BF):
    p = {n: _draw((C, H * D), dtype, seed + i, C ** -0.5) for i, n in enumerate(("q", "k", "v", "gate"))}
    p.update(m_w=_draw((C,), F32, seed + 5, 0.2, 1.0), m_b=_draw((C,), F32, seed + 6, 0.2), w=_draw((H, Cz), F32, seed + 7, Cz ** -0.5),
             z_w=_draw((Cz,), F32, seed + 8, 0.2, 1.0), z_b=_draw((Cz,), F32, seed + 9, 0.2), table=_draw((65, H), F32, seed + 10))
    return {n: t.requires_grad_() for n, t in p.items()}


@pytest.mark.parametrize("R", [64, 77])
def test_together_with_the_attention(R):
    """Against the same block in fp32 (fp64 where that is at hand) on the same values.  Each of its five 16-bit steps (norm,
    product, bias, sum of biases, attention with P rounded too) is off by 2^-8 of its size at most; a gradient passes
    as many again: 1.5 % and 3 % of the largest value leave a factor of two."""
    B, S, H, D, C, Cz = 2, 5, 4, 32, 64, 128
    p = _parameters(C, Cz, H, D, 20)
    m, z = _draw((B, S, R, C), BF, 1).requires_grad_(), _draw((B, R, R, Cz), BF, 2, 2.0).requires_grad_()
    pos = torch.arange(R, device=DEV) + (torch.arange(R, device=DEV) > 20) * 15
    keep = torch.rand((B, S, 1, 1, R), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) < 0.8
    keep[..., 0] = True
    d = _draw((B, S, R, H, D), BF, 3)
    out = _block(p, m, z, pos, keep)
    leaves = [m, z] + list(p.values())
    got = torch.autograd.grad(out, leaves, d)

    f = [t.detach().double().requires_grad_() for t in leaves]
    fp = dict(zip(p, f[2:]))
    norm = lambda t, w, b: torch.nn.functional.layer_norm(t, t.shape[-1:], w, b)  # noqa: E731
    x = norm(f[0], fp["m_w"], fp["m_b"])
    q, k, v, gate = ((x @ fp[n]).view(B, S, R, H, D).permute(0, 3, 1, 2, 4) for n in ("q", "k", "v", "gate"))
    rows = oc.bucket_rows([pos.tolist()], [pos.tolist()], "clip", 65, 32).to(DEV)
    bias = torch.einsum("bijc,hc->bhij", norm(f[1], fp["z_w"], fp["z_b"]), fp["w"]) + fp["table"][rows].permute(0, 3, 1, 2)
    s = (q @ k.transpose(-1, -2) * D ** -0.5 + bias.unsqueeze(2)).masked_fill(~keep.view(B, 1, S, 1, R), -1e30)
    want = (torch.sigmoid(gate) * (s.softmax(-1) @ v)).permute(0, 2, 3, 1, 4)
    *wants, d_bias = torch.autograd.grad(want, f + [bias], d.double())
    assert evo_oracle.rel_err(out.float(), want.float()) < 1.5e-2
    for n, a, b in zip(["m", "z"] + list(p), got, wants):
        if n == "z_b":
            # z_b adds one number to all scores of a row, which softmax does not see: the gradient is zero.  What is left
            # are roundings of d(bias), 2^-8 each in the attention (dS), in its result and in the two sums over MSA rows.
            noise = 4 * 2.0 ** -8 * d_bias.abs().sum((0, 2, 3)) @ fp["w"].abs()
            assert b.abs().max() < 1e-10 and (a.abs() < noise).all()
            continue
        assert a.shape == b.shape and torch.isfinite(a).all() and evo_oracle.rel_err(a.float(), b.float()) < 3e-2, n


@pytest.mark.parametrize("R", [64, 77])
def test_one_bias_for_a_batch(R):
    """A bias of positions that the batch shares, expanded: the attention reads it in place, and its gradient is summed over the
    batch.  As with the bias copied out, to the roundings of d(bias) and of sums in no fixed order."""
    import evoformer_triton_b200 as evo
    B, S, H, D = 3, 4, 4, 32
    q, k, v, d = (_draw((B, S, R, H, D), BF, i) for i in range(4))
    table = _draw((65, H), F32, 5).requires_grad_()
    pos = torch.arange(R, device=DEV)
    res = []
    for copied in (False, True):
        bias = evo.relative_position_bias(table, pos, max_distance=32, dtype=BF).expand(B, 1, H, R, R)
        bias = bias.clone(memory_format=torch.contiguous_format) if copied else bias
        out = evo.evoformer_attention(q, k, v, [None, bias])
        res.append((out.detach(), torch.autograd.grad(out, table, d)[0]))
    assert torch.equal(res[0][0], res[1][0])
    assert evo_oracle.rel_err(res[0][1], res[1][1]) < 4e-3


def test_together_in_a_cuda_graph():
    """A block's forward and backward captured once and replayed on other values, beside a second captured block."""
    B, S, R, H, D, C, Cz = 1, 3, 77, 4, 32, 64, 128
    pos = torch.arange(R, device=DEV)

    def program(seed):
        p = _parameters(C, Cz, H, D, seed)
        m, z = _draw((B, S, R, C), BF, seed).requires_grad_(), _draw((B, R, R, Cz), BF, seed + 1).requires_grad_()
        d = _draw((B, S, R, H, D), BF, seed + 2)

        def run():
            out = _block(p, m, z, pos, None)
            return [out.detach()] + list(torch.autograd.grad(out, [m, z] + list(p.values()), d))

        return p, m, z, run

    programs = [program(100), program(200)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for *_, run in programs:
            run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for *_, run in programs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = run()
        graphs.append((graph, res))
    with torch.no_grad():
        for i, (p, m, z, _) in enumerate(programs):
            m.copy_(_draw(m.shape, BF, 300 + i))
            z.copy_(_draw(z.shape, BF, 310 + i))
            p["table"].copy_(_draw(p["table"].shape, F32, 320 + i))
    for graph, _ in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    for (*_, run), (_, res) in zip(programs, graphs):
        for k, (a, b) in enumerate(zip(res, run())):
            # dQ of the attention is summed in no fixed order: what follows it is equal to rounding
            assert torch.equal(a, b) if k == 0 else evo_oracle.rel_err(a, b) < 1e-2, k
