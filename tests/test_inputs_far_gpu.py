"""GPU: the operators before the attention on tensors whose offsets pass 32 bits."""
import pytest
import torch

from oracle import inputs_oracle as oc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _give_memory_back():
    yield
    torch.cuda.empty_cache()


def _draw(shape, dtype, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _apart(values, far=2 ** 31 + 64):
    """The same values with the two batch entries 2^31 elements from one another."""
    buf = torch.empty(far + values[0].numel(), dtype=values.dtype, device=DEV)
    view = buf.as_strided(values.shape, (far, *values[0].contiguous().stride()))
    view.copy_(values)
    return view


@pytest.mark.parametrize("C", [64, 50])
def test_far_apart(C):
    """Every strided operand of the three operators; the results are those of the same values next to each other, to the bit."""
    import evoformer_triton_b200 as evo
    R, H = 37, 4
    pos = torch.arange(R, device=DEV)

    def run(place):
        x, dy = place(_draw((2, R, C), BF, 1)).requires_grad_(), place(_draw((2, R, C), BF, 2))
        y = evo.layer_norm(x)
        z, W = place(_draw((2, R, R, C), BF, 3)).requires_grad_(), _draw((H, C), F32, 4).requires_grad_()
        out, d = evo.pair_bias_projection(z, W), place(_draw((2, 1, H, R, R), BF, 5))
        table, base = _draw((65, H), F32, 6).requires_grad_(), place(_draw((2, 1, H, R, R), BF, 7))
        bias = evo.relative_position_bias(table, pos, max_distance=32, pair_bias=base)
        return [y.detach(), *torch.autograd.grad(y, x, dy), out.detach(), *torch.autograd.grad(out, (z, W), d), bias.detach(), *torch.autograd.grad(bias, table, d)]

    for a, b in zip(run(_apart), run(lambda t: t)):
        assert torch.equal(a, b)


def test_layer_norm_of_more_than_2_31_values():
    import evoformer_triton_b200 as evo
    C, N = 128, 2 ** 24 + 1000
    x = torch.empty(N, C, dtype=BF, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    w = _draw((C,), F32, 2).requires_grad_()
    x.requires_grad_()
    y = evo.layer_norm(x, w)
    dy = torch.empty_like(y).normal_(generator=torch.Generator(device=DEV).manual_seed(3))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for rows in (slice(0, 100), slice(N - 1100, N)):
        want = oc.layer_norm(x.detach()[rows], w.detach(), None, 1e-5, dy[rows])
        oc.check("y", y[rows], want[0])
        oc.check("dx", dx[rows], want[1])
    want = torch.zeros(C, dtype=torch.float64, device=DEV)
    size = want.clone()
    for part in range(0, N, 2 ** 20):
        h, _ = oc.normalise(x.detach()[part:part + 2 ** 20].double(), 1e-5)
        p = dy[part:part + 2 ** 20].double() * h
        want += p.sum(0)
        size += p.abs().sum(0)
    # a lane adds 1 / 4 736 of the rows (296 blocks of 16 teams) one after another: 3 543 of them, and then the lanes' sums
    assert ((dw.double() - want).abs() <= 4000 * oc.UNIT32 * size).all()


def test_relative_bias_of_more_than_2_31_values():
    import evoformer_triton_b200 as evo
    R, H = 8200, 32
    pos = torch.arange(R, device=DEV)
    table = _draw((65, H), F32, 1).requires_grad_()
    out = evo.relative_position_bias(table, pos, max_distance=32, dtype=BF)
    assert out.numel() > 2 ** 31
    t = table.detach()
    for h, i in ((0, 0), (H - 1, R - 1), (H - 1, R - 40), (17, 4000)):
        assert torch.equal(out[0, 0, h, i], t[(i - pos).clamp(-32, 32) + 32, h].to(BF))
    g, = torch.autograd.grad(out, table, torch.ones_like(out))
    away = torch.arange(-32, 33, device=DEV).abs()
    count = (R - away).double()
    count[0] = count[64] = (R - 32) * (R - 31) / 2
    assert ((g.double() - count[:, None]).abs() <= 2000 * oc.UNIT32 * count[:, None]).all()


def test_pair_projection_of_more_than_2_31_values():
    import evoformer_triton_b200 as evo
    R, C, H = 4100, 128, 2
    z = torch.empty(1, R, R, C, dtype=BF, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(1)).requires_grad_()
    W = _draw((H, C), F32, 2, 0.1).requires_grad_()
    out = evo.pair_bias_projection(z, W)
    d = _draw((1, 1, H, R, R), BF, 3)
    dz, dW = torch.autograd.grad(out, (z, W), d)
    for i in (0, R - 1):
        want = oc.pair_projection(z.detach()[:, i:i + 1], W.detach(), None, None, 1e-5, d[:, :, :, i:i + 1])
        oc.check("out", out[:, :, :, i:i + 1], want[0])
        oc.check("dpair", dz[:, i:i + 1], want[1])
    want, size = torch.zeros(H, C, dtype=torch.float64, device=DEV), torch.zeros(H, C, dtype=torch.float64, device=DEV)
    for i in range(0, R, 100):
        h, _ = oc.normalise(z.detach()[0, i:i + 100].double(), 1e-5)
        part = d[0, 0, :, i:i + 100].double()
        want += torch.einsum("hij,ijc->hc", part, h)
        size += torch.einsum("hij,ijc->hc", part.abs(), h.abs())
    # a warp (296 blocks of 8) takes 444 tiles of 16 rows one after another, and is off by 2^-17 of a product of pieces at most
    assert ((dW.double() - want).abs() <= (600 * oc.UNIT32 + 2.0 ** -16) * size).all()
