"""GPU: rotary positions against their definition in 64 bits, value by value within the roundings that are made."""
import pytest
import torch

from oracle import sequences_oracle as oc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
IDS = {BF: "bf16", HF: "fp16", F32: "fp32"}


def _draw(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def _against_oracle(q, k, positions, f, layout="half", amplitude=1.0, seed=3):
    import evoformer_triton_b200 as evo
    q.requires_grad_()
    k.requires_grad_()
    out = evo.rotary_embedding(q, k, positions, f, layout=layout, amplitude=amplitude)
    with torch.no_grad():
        for a, b in zip(out, evo.rotary_embedding(q, k, positions, f, layout=layout, amplitude=amplitude)):
            assert torch.equal(a, b) and a.is_contiguous()
        assert torch.equal(evo.rotary_embedding(k, None, positions, f, layout=layout, amplitude=amplitude), out[1])
    d = [_draw(o.shape, o.dtype, seed + n) for n, o in enumerate(out)]
    grads = torch.autograd.grad(out, (q, k), d)
    pos = positions.expand(q.shape[:-2])
    for name, x, y, g, dx in zip("qk", (q, k), out, d, grads):
        oc.check(name, y, oc.rotary(x.detach(), pos, f, layout, amplitude))
        oc.check("d" + name, dx, oc.rotary(g, pos, f, layout, amplitude, inverse=True))


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,Hk,D,rotary", [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (8, 32, 8, 128, 128), (37, 3, 1, 64, 64), (300, 12, 2, 96, 64), (129, 5, 5, 80, 40),
                                             (41, 2, 1, 33, 32), (41, 2, 1, 7, 6), (5, 1, 2, 1024, 1024), (2049, 4, 4, 64, 16), (5000, 6, 3, 128, 128), (23, 4, 2, 192, 100)])
def test_sizes(T, H, Hk, D, rotary, layout, dtype):
    import evoformer_triton_b200 as evo
    f = evo.rotary_frequencies(rotary, device=DEV)
    _against_oracle(_draw((T, H, D), dtype, 1), _draw((T, Hk, D), dtype, 2), torch.arange(T, device=DEV), f, layout)


@pytest.mark.parametrize("start", [0, 4095, 10 ** 6, 2 ** 31 - 100, 10 ** 12, -50, -10 ** 9])
def test_far_positions_are_as_exact(start):
    import evoformer_triton_b200 as evo
    f = evo.rotary_frequencies(64, device=DEV)
    pos = torch.arange(100, device=DEV) + start
    _against_oracle(_draw((100, 2, 64), F32, 1), _draw((100, 2, 64), F32, 2), pos, f)
    if abs(start) < 2 ** 31 - 100:
        _against_oracle(_draw((100, 2, 64), F32, 1), _draw((100, 2, 64), F32, 2), pos.int(), f.float(), "interleaved")


def test_positions_that_jump_and_repeat():
    import evoformer_triton_b200 as evo
    g = torch.Generator(device=DEV).manual_seed(5)
    pos = torch.randint(-5000, 5000, (777,), generator=g, device=DEV)
    _against_oracle(_draw((777, 4, 64), BF, 1), _draw((777, 2, 64), BF, 2), pos, evo.rotary_frequencies(64, device=DEV), amplitude=1.3)


def _layouts():
    return {
        "slices of one projection": lambda dt: (lambda x: (x[:, :4], x[:, 4:6]))(_draw((50, 8, 64), dt, 1)),
        "heads before tokens": lambda dt: (_draw((4, 50, 64), dt, 1).transpose(0, 1), _draw((2, 50, 64), dt, 2).transpose(0, 1)),
        "rows of an odd pitch": lambda dt: (_draw((50, 4, 65), dt, 1)[..., :64], _draw((50, 2, 67), dt, 2)[..., 1:65]),
        "values not contiguous": lambda dt: (_draw((50, 64, 4), dt, 1).transpose(1, 2), _draw((50, 2, 64), dt, 2)),
        "one head for all": lambda dt: (_draw((50, 1, 64), dt, 1).expand(50, 4, 64), _draw((1, 2, 64), dt, 2).expand(50, 2, 64)),
        "backwards through a buffer": lambda dt: (_draw((50, 4, 64), dt, 1).flip(0), _draw((100, 2, 64), dt, 2)[::2]),
    }


@pytest.mark.parametrize("dtype", [BF, F32], ids=IDS.get)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("name", sorted(_layouts()))
def test_rows_are_read_where_they_lie(name, layout, dtype):
    import evoformer_triton_b200 as evo
    q, k = (t.detach() for t in _layouts()[name](dtype))
    _against_oracle(q, k, torch.arange(50, device=DEV), evo.rotary_frequencies(48, device=DEV), layout)


@pytest.mark.parametrize("shape,positions", [((3, 20), (20,)), ((3, 20), (3, 20)), ((3, 20), (1, 20)), ((2, 3, 20), (2, 3, 20)), ((2, 3, 20), (2, 1, 20)), ((2, 3, 20), (1, 3, 20)),
                                             ((2, 3, 20), (20,))], ids=str)
def test_axes_before_the_tokens(shape, positions):
    import evoformer_triton_b200 as evo
    g = torch.Generator(device=DEV).manual_seed(5)
    pos = torch.randint(0, 1000, positions, generator=g, device=DEV)
    _against_oracle(_draw((*shape, 4, 32), BF, 1), _draw((*shape, 2, 32), BF, 2), pos, evo.rotary_frequencies(32, device=DEV))
    turned = pos.unsqueeze(-1).expand(*positions, 2)[..., 1]  # (positions that are not dense)
    _against_oracle(_draw((*shape, 4, 32), BF, 1), _draw((*shape, 2, 32), BF, 2), turned, evo.rotary_frequencies(32, device=DEV))


def test_nothing_in_nothing_out():
    import evoformer_triton_b200 as evo
    x = torch.empty(0, 4, 32, device=DEV, requires_grad=True)
    f = evo.rotary_frequencies(32, device=DEV)
    y, z = evo.rotary_embedding(x, x, torch.empty(0, dtype=torch.long, device=DEV), f)
    (y.sum() + z.sum()).backward()
    assert y.shape == z.shape == x.grad.shape == (0, 4, 32)


def test_gradients_of_one_or_none():
    import evoformer_triton_b200 as evo
    f, pos = evo.rotary_frequencies(32, device=DEV), torch.arange(9, device=DEV)
    q, k = _draw((9, 4, 32), F32, 1).requires_grad_(), _draw((9, 2, 32), F32, 2)
    y, z = evo.rotary_embedding(q, k, pos, f)
    d = _draw(y.shape, F32, 3)
    (g,) = torch.autograd.grad(y, q, d)
    oc.check("dq", g, oc.rotary(d, pos, f, "half", inverse=True))
    y, z = evo.rotary_embedding(k, q, pos, f)  # only the second has one
    (g,) = torch.autograd.grad(z, q, d)
    oc.check("dk", g, oc.rotary(d, pos, f, "half", inverse=True))
    x = q.detach().clone().requires_grad_()
    y, z = evo.rotary_embedding(x, x, pos, f)  # the same tensor twice: both gradients
    (g,) = torch.autograd.grad([y, z], x, [d, d])
    assert torch.allclose(g, 2 * oc.rotary(d, pos, f, "half", inverse=True)[0].float(), atol=1e-5)


def test_graph_and_side_stream():
    """Captured with its backward and replayed on other values; and called on another stream than the current."""
    import evoformer_triton_b200 as evo
    f, pos = evo.rotary_frequencies(64, device=DEV), torch.arange(33, device=DEV)
    q, k = _draw((33, 4, 64), BF, 1), _draw((33, 2, 64), BF, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = evo.rotary_embedding(q, k, pos, f)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, evo.rotary_embedding(q, k, pos, f)))
    sq, sk = torch.zeros_like(q).requires_grad_(), torch.zeros_like(k).requires_grad_()
    spos, d = torch.zeros_like(pos), [_draw(t.shape, BF, 5) for t in (q, k)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = evo.rotary_embedding(sq, sk, spos, f)
        grads = torch.autograd.grad(out, (sq, sk), d)
    for shift in (0, 7):
        with torch.no_grad():
            sq.copy_(q + shift), sk.copy_(k - shift), spos.copy_(pos + shift)
        graph.replay()
        for x, y, g, dx in zip((sq, sk), out, d, grads):
            oc.check("replayed", y, oc.rotary(x.detach(), spos, f, "half"))
            oc.check("replayed gradient", dx, oc.rotary(g, spos, f, "half", inverse=True))


def test_refusals():
    import evoformer_triton_b200 as evo
    q, k = _draw((6, 4, 32), BF, 1), _draw((6, 2, 32), BF, 2)
    f, pos = evo.rotary_frequencies(32, device=DEV), torch.arange(6, device=DEV)
    call = evo.rotary_embedding
    bad = [
        (ValueError, lambda: call(q[0], k, pos, f)), (ValueError, lambda: call(q[None, None, None], None, pos, f)),
        (ValueError, lambda: call(q, k[:5], pos, f)), (ValueError, lambda: call(q, k[..., :30], pos, f)), (TypeError, lambda: call(q, k.float(), pos, f)),
        (TypeError, lambda: call(q.double(), None, pos, f)), (ValueError, lambda: call(q, k, pos[:5], f)), (ValueError, lambda: call(q, k, pos[None], f)),
        (TypeError, lambda: call(q, k, pos.float(), f)), (RuntimeError, lambda: call(q, k, pos.cpu(), f)), (RuntimeError, lambda: call(q, k.cpu(), pos, f)),
        (TypeError, lambda: call(q, k, pos, f.bfloat16())), (RuntimeError, lambda: call(q, k, pos, f.cpu())), (ValueError, lambda: call(q, k, pos, f[None])),
        (ValueError, lambda: call(q[..., :30], None, pos, f)), (ValueError, lambda: call(q, k, pos, f[:0])), (ValueError, lambda: call(q, k, pos, f.clone().requires_grad_())),
        (ValueError, lambda: call(q, k, pos, f, amplitude=float("nan"))), (ValueError, lambda: call(q, k, pos, f, amplitude=1e300)),
    ]
    for kind, fn in bad:
        with pytest.raises(kind):
            fn()
    x = q.float().requires_grad_()
    y = call(x, None, pos, f)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
        call(fwad.make_dual(q.float(), q.float()), None, pos, f)
