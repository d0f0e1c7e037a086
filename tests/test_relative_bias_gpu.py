"""GPU: the relative position bias: the forward to the bit, the gradient of the table within the roundings of its sums."""
import pytest
import torch

from oracle import inputs_oracle as oc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
CLIP, LOG, CAUSAL = ("clip", 65, 32), ("log", 32, 128), ("log_causal", 32, 128)


def _draw(shape, dtype, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _residues(B, n, seed):
    """Numbers of residues: consecutive runs, gaps, a jump to another chain and back."""
    g = torch.Generator().manual_seed(seed)
    step = 1 + (torch.rand((B, n), generator=g) < 0.05) * torch.randint(0, 30, (B, n), generator=g)
    pos = torch.cumsum(step, 1)
    pos[:, n // 2:] -= int(pos[0, n // 2]) if n > 40 else 0
    return pos


def _run(table, q, k, kind, base=None, dtype=None, d=None):
    import evoformer_triton_b200 as evo
    scheme, n, M = kind
    leaves = [t.requires_grad_() for t in (table, base) if t is not None]
    out = evo.relative_position_bias(table, q, k, max_distance=M, buckets=scheme, pair_bias=base, dtype=dtype)
    with torch.no_grad():
        assert torch.equal(out, evo.relative_position_bias(table, q, k, max_distance=M, buckets=scheme, pair_bias=base, dtype=dtype))
    if d is None:
        d = _draw(out.shape, out.dtype, 9)
    grads = torch.autograd.grad(out, leaves, d)
    key = q if k is None else k
    two = lambda t: (t if t.dim() == 2 else t[None]).tolist()  # noqa: E731
    B = out.shape[0]
    ql, kl = two(q), two(key)
    rows = oc.bucket_rows(ql * (B if len(ql) == 1 else 1), kl * (B if len(kl) == 1 else 1), scheme, n, M).to(DEV)
    want, dtable = oc.relative_bias(table.detach(), rows, None if base is None else base.detach(), out.dtype, d)
    assert out.shape == want.shape and torch.equal(out, want)
    es = out.element_size()
    assert out.data_ptr() % 16 == 0 and all(s * es % 16 == 0 for s in out.stride()[:4])
    assert grads[0].dtype == table.dtype
    oc.check("dtable", grads[0], dtable)
    if base is not None:
        assert torch.equal(grads[1], d.to(base.dtype))
    return out


@pytest.mark.parametrize("kind", [CLIP, LOG, CAUSAL], ids=lambda k: k[0])
@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,H,R", [(1, 1, 1), (1, 2, 2), (2, 3, 31), (1, 8, 100), (2, 4, 257), (1, 9, 384), (1, 2, 437), (1, 1, 1025)], ids=str)
def test_sizes(B, H, R, dtype, kind):
    pos = _residues(B, R, R).to(DEV)
    _run(_draw((kind[1], H), dtype, 1), pos, None, kind)


@pytest.mark.parametrize("kind", [("clip", 1, 0), ("clip", 3, 1), ("clip", 257, 128), ("clip", 1023, 511), ("log", 4, 2), ("log", 8, 5), ("log", 64, 1000),
                                  ("log", 256, 700), ("log_causal", 2, 4), ("log_causal", 256, 100000)], ids=str)
def test_buckets(kind):
    """Few and many buckets, more than a block of the backward keeps sums of; keys from far before to far behind."""
    q = torch.arange(150, device=DEV) * 3
    k = torch.arange(-700, 1300, 2, device=DEV)[None]
    _run(_draw((kind[1], 2), F32, 1), q, k, kind, dtype=BF)


def test_borders_of_logarithmic_buckets():
    """Every distance up to beyond the last border, both ways."""
    q, k = torch.zeros(1, dtype=torch.int64, device=DEV), torch.arange(-1100, 1101, device=DEV)
    for kind in (LOG, CAUSAL, ("log", 32, 127), ("log", 64, 1000)):
        _run(_draw((kind[1], 1), F32, 1), q, k, kind)


@pytest.mark.parametrize("kind", [CLIP, LOG, CAUSAL], ids=lambda k: k[0])
def test_positions_of_any_order_size_and_type(kind):
    g = torch.Generator().manual_seed(3)
    table = _draw((kind[1], 3), BF, 1)
    mixed = torch.randint(-300, 300, (2, 140), generator=g).to(DEV)
    _run(table, mixed, None, kind)
    _run(table, mixed.int(), mixed, kind)
    _run(table, mixed.int(), mixed.int(), kind, dtype=F32)
    _run(table, torch.zeros(70, dtype=torch.int32, device=DEV), None, kind)              # all the same residue
    far = torch.tensor([-2 ** 62, -2 ** 40, -2 ** 31, -5, 0, 1, 2 ** 31, 2 ** 33 + 1, 2 ** 62 - 1], device=DEV)
    _run(table, far, None, kind)
    _run(table, torch.tensor([-2 ** 31, -1, 0, 2 ** 31 - 1], dtype=torch.int32, device=DEV), None, kind)
    _run(table, torch.arange(400, device=DEV).flip(0)[::2], None, kind)                  # downwards, and strided
    _run(table, mixed.t().contiguous().t(), None, kind)                                  # positions that are not contiguous


@pytest.mark.parametrize("Rq,Rk", [(1, 1), (1, 2048), (1, 77), (5, 1000), (300, 1), (64, 9)], ids=str)
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_queries_and_keys_of_their_own(Rq, Rk, dtype):
    k = _residues(2, Rk, 5).to(DEV)
    q = torch.arange(Rq, device=DEV)[None] + Rk - Rq
    for kind in (CLIP, CAUSAL):
        _run(_draw((kind[1], 12), F32, 1), q, k, kind, dtype=dtype)                       # q shared over the batch
        _run(_draw((kind[1], 12), F32, 1), q[0].expand(2, Rq), k[0], kind, dtype=dtype)   # k shared


@pytest.mark.parametrize("table,base,out", [(F32, F32, None), (BF, BF, None), (F32, BF, None), (BF, F32, None), (F32, BF, F32), (HF, F32, HF)], ids=str)
@pytest.mark.parametrize("R", [64, 101])
def test_added_to_a_pair_bias(R, table, base, out):
    pos = torch.arange(R, device=DEV)
    pb = _draw((2, 1, 4, R, R), base, 3)
    _run(_draw((65, 4), table, 1), pos, None, CLIP, pb, out)
    view = _draw((2, 1, R, R, 4), base, 3).permute(0, 1, 4, 2, 3)                         # heads last
    _run(_draw((65, 4), table, 1), pos, None, CLIP, view, out)
    padded = _draw((2, 1, 4, R, R + 11), base, 3)[..., 3:R + 3]                            # rows of an odd pitch, off their start
    _run(_draw((65, 4), table, 1), pos, None, CLIP, padded, out)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_gradients_of_any_layout(dtype):
    R = 133
    pos = _residues(2, R, 1).to(DEV)
    full = _draw((2, 1, 4, R, R), dtype, 3)
    for d in (full, full.transpose(3, 4), full.permute(0, 1, 3, 4, 2).contiguous().permute(0, 1, 4, 2, 3), _draw((1,), dtype, 4).expand(2, 1, 4, R, R),
              _draw((2, 1, 4, R, 160), dtype, 5)[..., :R], _draw((2, 1, 4, R, 161), dtype, 5)[..., 5:R + 5], full[:1].expand(2, 1, 4, R, R)):
        _run(_draw((65, 4), F32, 1), pos, None, CLIP, dtype=dtype, d=d)


def test_values_that_are_not_finite_stay_in_their_bucket():
    import evoformer_triton_b200 as evo
    table = _draw((65, 2), F32, 1)
    table[10, 0], table[64, 1] = float("nan"), float("-inf")
    pos = torch.arange(200, device=DEV)
    out = evo.relative_position_bias(table, pos, max_distance=32)
    i, j = torch.meshgrid(pos, pos, indexing="ij")
    assert torch.equal(torch.isnan(out[0, 0, 0]), i - j == -22) and not torch.isnan(out[0, 0, 1]).any()
    assert torch.equal(torch.isinf(out[0, 0, 1]), i - j >= 32)
    table = _draw((65, 2), F32, 1).requires_grad_()
    d = _draw((1, 1, 2, 200, 200), F32, 2)
    d[0, 0, 0, 60, 50] = float("nan")
    dt, = torch.autograd.grad(evo.relative_position_bias(table, pos, max_distance=32), table, d)
    bad = torch.zeros(65, 2, dtype=torch.bool, device=DEV)
    bad[42, 0] = True
    assert torch.equal(torch.isnan(dt), bad)


@pytest.mark.parametrize("B,Rq,Rk", [(1, 0, 0), (2, 0, 5), (2, 5, 0), (0, 4, 4)], ids=str)
def test_nothing_to_look_up(B, Rq, Rk):
    import evoformer_triton_b200 as evo
    table = torch.ones(65, 2, device=DEV, requires_grad=True)
    out = evo.relative_position_bias(table, torch.zeros(B, Rq, dtype=torch.int64, device=DEV), torch.zeros(B, Rk, dtype=torch.int64, device=DEV), max_distance=32)
    assert out.shape == (B, 1, 2, Rq, Rk)
    dt, = torch.autograd.grad(out, table, torch.zeros_like(out))
    assert not dt.any()


def test_same_bits_every_time():
    import evoformer_triton_b200 as evo
    pos = torch.randint(0, 500, (2, 700), device=DEV)
    for kind in (CLIP, LOG, ("clip", 401, 200)):
        table, d = _draw((kind[1], 8), F32, 1).requires_grad_(), _draw((2, 1, 8, 700, 700), BF, 2)
        runs = [torch.autograd.grad(evo.relative_position_bias(table, pos, max_distance=kind[2], buckets=kind[0], dtype=BF), table, d)[0] for _ in range(3)]
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_gradient_only_of_what_wants_one():
    import evoformer_triton_b200 as evo
    pos, base, table = torch.arange(50, device=DEV), _draw((1, 1, 2, 50, 50), BF, 1), _draw((65, 2), F32, 2)
    d = _draw((1, 1, 2, 50, 50), BF, 3)
    b = base.clone().requires_grad_()
    g, = torch.autograd.grad(evo.relative_position_bias(table, pos, max_distance=32, pair_bias=b), b, d)
    assert torch.equal(g, d)
    t = table.clone().requires_grad_()
    g, = torch.autograd.grad(evo.relative_position_bias(t, pos, max_distance=32, pair_bias=base), t, d)
    rows = oc.bucket_rows([pos.tolist()], [pos.tolist()], *CLIP).to(DEV)
    oc.check("dtable", g, oc.relative_bias(table, rows, base, BF, d)[1])


def test_refusals():
    import evoformer_triton_b200 as evo
    table, pos = _draw((65, 2), F32, 1), torch.arange(7, device=DEV)
    call = lambda t=table, p=pos, k=None, **kw: evo.relative_position_bias(t, p, k, max_distance=32, **kw)  # noqa: E731
    base = _draw((1, 1, 2, 7, 7), BF, 1)
    for bad in (lambda: call(p=pos.float()), lambda: call(k=pos.short()), lambda: call(table.double()), lambda: call(dtype=torch.float64), lambda: call(pair_bias=base.double())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: call(p=pos[None, None]), lambda: call(p=pos.expand(2, 7), k=pos.expand(3, 7)), lambda: call(pair_bias=base[..., :6]), lambda: call(pair_bias=base[:, 0]),
                lambda: call(p=pos.expand(2, 7), pair_bias=base), lambda: call(table[0]), lambda: call(table[:64])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: call(p=pos.cpu()), lambda: call(k=pos.cpu()), lambda: call(pair_bias=base.cpu())):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(RuntimeError, match="differentiated once"):
        t = table.clone().requires_grad_()
        torch.autograd.grad(call(t).sum(), t, create_graph=True)

