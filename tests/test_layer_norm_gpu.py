"""GPU: layer norm against its definition in 64 bits, value by value within the roundings that fp32 arithmetic makes."""
import pytest
import torch

from oracle import inputs_oracle as oc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _draw(shape, dtype, seed, std=1.0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)


def _against_oracle(x, w, b, dy, eps=1e-5):
    import evoformer_triton_b200 as evo
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = evo.layer_norm(x, w, b, eps=eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(evo.layer_norm(x, w, b, eps=eps), y)
    grads = iter(torch.autograd.grad(y, leaves, dy))
    C = x.shape[-1]
    flat = lambda t: t.detach().reshape(-1, C)  # noqa: E731
    want = oc.layer_norm(flat(x), w if w is None else w.detach(), b if b is None else b.detach(), eps, flat(dy))
    oc.check("y", flat(y), want[0])
    oc.check("dx", flat(next(grads)), want[1])
    for name, t, z in (("dweight", w, want[2]), ("dbias", b, want[3])):
        if t is not None:
            got = next(grads)
            assert got.dtype == t.dtype
            oc.check(name, got, z)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", [(1,), (1, 1), (5, 7), (1, 256), (3, 4, 64), (2, 33, 96), (4, 9, 128), (3, 1, 255), (3, 5, 256), (17, 260), (9, 384), (7, 512),
                                   (5, 1000), (33, 1111), (6, 1024), (5, 2048), (3, 4097), (3, 8192), (2, 16384), (2, 16400), (2, 40000), (1500, 24), (70001, 16), (4000, 130)], ids=str)
def test_sizes(shape, dtype):
    C = shape[-1]
    _against_oracle(_draw(shape, dtype, 1, 1.5, 0.3), _draw((C,), F32, 2, 0.2, 1.0), _draw((C,), F32, 3, 0.2), _draw(shape, dtype, 4))


@pytest.mark.parametrize("weights", [(None, None), (BF, None), (None, HF), (BF, BF), (F32, HF), (HF, F32)], ids=str)
@pytest.mark.parametrize("C", [128, 37])
def test_weights_of_other_types_or_none(weights, C):
    wt, bt = weights
    w, b = None if wt is None else _draw((C,), wt, 2, 0.2, 1.0), None if bt is None else _draw((C,), bt, 3)
    _against_oracle(_draw((4, 50, C), BF, 1), w, b, _draw((4, 50, C), BF, 4))


def _layouts():
    wide = lambda *s: (lambda dt: _draw(s, dt, 1))  # noqa: E731
    return {
        "turned": lambda dt: wide(2, 7, 5, 64)(dt).transpose(1, 2),
        "sliced": lambda dt: wide(3, 5, 256)(dt)[..., :128],
        "sliced, unaligned": lambda dt: wide(3, 5, 131)(dt)[..., 1:129],
        "rows of an odd pitch": lambda dt: wide(6, 129)(dt)[:, :128],
        "every other row": lambda dt: wide(8, 6, 128)(dt)[::2, ::3],
        "four axes that do not fold": lambda dt: wide(4, 6, 4, 6, 64)(dt)[::2, ::2, ::2, ::2],
        "channels not contiguous": lambda dt: wide(5, 64, 9)(dt).transpose(1, 2),
        "one row for all": lambda dt: wide(1, 1, 128)(dt).expand(4, 3, 128),
        "one channel, strided": lambda dt: wide(6, 4)(dt)[:, 1:2],
    }


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("dy_layout", ["dense", "turned", "expanded"])
@pytest.mark.parametrize("name", sorted(_layouts()))
def test_rows_are_read_where_they_lie(name, dy_layout, dtype):
    x = _layouts()[name](dtype).detach()
    C = x.shape[-1]
    dy = _draw(x.shape, dtype, 4)
    if dy_layout == "turned":
        dy = dy.transpose(0, 1).contiguous().transpose(0, 1)
    elif dy_layout == "expanded":
        dy = _draw((1,), dtype, 5).expand(x.shape)
    _against_oracle(x, _draw((C,), F32, 2, 0.2, 1.0), _draw((C,), F32, 3), dy)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("C", [128, 256, 1500])
def test_rows_far_from_zero_constant_rows_and_large_values(C, dtype):
    x = _draw((12, C), dtype, 1)
    x[0:3] = _draw((3, C), dtype, 2, 1.0, 1000.0)
    x[3] = 7.0
    x[4] = 0.0
    x[5] = _draw((C,), dtype, 3, 1e4 if dtype == HF else 1e8)
    x[6] = _draw((C,), dtype, 3, 1e-4)
    _against_oracle(x, _draw((C,), F32, 2, 0.2, 1.0), _draw((C,), F32, 3), _draw((12, C), dtype, 4))


def test_values_that_are_not_finite_stay_in_their_rows():
    import evoformer_triton_b200 as evo
    x = _draw((40, 128), BF, 1)
    clean = evo.layer_norm(x)
    x[3, 5], x[17, 0], x[33, 127] = float("nan"), float("inf"), float("-inf")
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 17, 33]] = True
    xr = x.requires_grad_()
    y = evo.layer_norm(xr)
    dx, = torch.autograd.grad(y, xr, torch.ones_like(y))
    assert torch.equal(y[~bad], clean[~bad]) and torch.isfinite(dx[~bad]).all()
    assert torch.isnan(y[bad]).all() and torch.isnan(dx[bad]).all()


@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 33)], ids=str)
def test_no_rows(shape):
    import evoformer_triton_b200 as evo
    x, w, b = torch.zeros(shape, device=DEV, requires_grad=True), torch.ones(shape[-1], device=DEV, requires_grad=True), torch.ones(shape[-1], device=DEV, requires_grad=True)
    y = evo.layer_norm(x, w, b)
    assert y.shape == shape
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (0, 2), (1, 2)], ids=str)
def test_only_the_gradients_that_are_wanted(wanted):
    import evoformer_triton_b200 as evo
    a = [_draw((300, 128), BF, 1), _draw((128,), F32, 2, 0.2, 1.0), _draw((128,), F32, 3)]
    for i in wanted:
        a[i].requires_grad_()
    dy = _draw((300, 128), BF, 4)
    got = torch.autograd.grad(evo.layer_norm(*a), [a[i] for i in wanted], dy)
    want = oc.layer_norm(a[0].detach(), a[1].detach(), a[2].detach(), 1e-5, dy)
    for i, t in zip(wanted, got):
        oc.check(str(i), t, want[1 + i])
    assert all(a[i].grad is None for i in range(3))


def test_same_bits_every_time_and_on_another_stream():
    import evoformer_triton_b200 as evo
    x, w, b, dy = _draw((2, 99, 77, 256), BF, 1), _draw((256,), F32, 2), _draw((256,), F32, 3), _draw((2, 99, 77, 256), BF, 4)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def once():
        y = evo.layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = once()
    torch.cuda.current_stream().wait_stream(s)
    for a, b, c in zip(first, once(), other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals():
    import evoformer_triton_b200 as evo
    x, w = _draw((3, 8), F32, 1), _draw((8,), F32, 2)
    for bad in (lambda: evo.layer_norm(x.double()), lambda: evo.layer_norm(x, w.double()), lambda: evo.layer_norm(x.long())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: evo.layer_norm(x, w[:7]), lambda: evo.layer_norm(x, w, w[None]), lambda: evo.layer_norm(x[0, 0]), lambda: evo.layer_norm(x[:, :0]),
                lambda: evo.layer_norm(x, eps=-1.0), lambda: evo.layer_norm(x, eps=float("nan"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        evo.layer_norm(x, w.cpu())
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(evo.layer_norm(x, w).sum(), x, create_graph=True)
