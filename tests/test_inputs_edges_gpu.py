"""GPU: the operators before the attention at the edges of what they take."""
import ctypes as C

import pytest
import torch

from oracle import inputs_oracle as oc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _draw(shape, dtype, seed, std=1.0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)


# ---------------------------------------------------------------- relative position bias

def _keys_that_jump_back(n, apart):
    """Two chains far from each other in pieces of `apart` keys, the last of which may be cut short: a piece is one chain up to the
    length of the short one, and the other one, but for the first of every 64 keys, behind that."""
    i = torch.arange(n)
    return torch.where((i % apart < n % apart) | (i % 64 < apart), 5, 2000)


@pytest.mark.parametrize("kind", [("log_causal", 32, 4096), ("log", 64, 5000), ("log_causal", 32, 128)], ids=str)
@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Rk", [3, 18, 34, 77, 437])
def test_relative_gradient_of_keys_in_no_order(Rk, dtype, kind):
    """The gradient of ones counts the keys of a bucket, exactly (whole numbers below 2^24): rows on 16 bytes and off them, a last strip
    that ends anywhere, borders beyond those that are looked up and within."""
    import evoformer_triton_b200 as evo
    scheme, n, M = kind
    H, q = 2, torch.tensor([3000, 2000, 5, 0, 1999])
    for keys in (_keys_that_jump_back(Rk, 8), _keys_that_jump_back(Rk, 16), torch.arange(Rk).flip(0) * 7, (torch.arange(Rk) * 37) % 3001):
        rows = oc.bucket_rows([q.tolist()], [keys.tolist()], scheme, n, M).reshape(-1)
        want = torch.bincount(rows, minlength=n).to(F32).unsqueeze(1).expand(n, H)
        table = _draw((n, H), F32, 1).requires_grad_()
        out = evo.relative_position_bias(table, q.to(DEV), keys.to(DEV), max_distance=M, buckets=scheme, dtype=dtype)
        for pitch in (out.stride(3), Rk + 1 - Rk % 2):
            d = torch.ones((1, 1, H, len(q), pitch), dtype=dtype, device=DEV)[..., :Rk]
            g, = torch.autograd.grad(out, table, d, retain_graph=True)
            assert torch.equal(g.cpu(), want), (pitch, (g.cpu() - want)[:, 0].nonzero().flatten().tolist())


# ---------------------------------------------------------------- pair-bias projection

@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("C_,H", [(128, 8), (64, 16), (256, 16), (384, 4), (100, 5), (130, 20)], ids=str)
def test_projection_of_rows_of_any_scale(C_, H, dtype):
    """Rows that deviate by 10^-17 to 10^17 (fp16: as far as it goes), with no eps that would hide the small ones, and gradients
    of any size: rows scaled by s have the result of s = 1 and dpair / s."""
    import evoformer_triton_b200 as evo
    exps = torch.arange(-17, 18, device=DEV).double() if dtype != HF else torch.linspace(-2, 4, 35, device=DEV).double()
    z = (_draw((1, 35, 6, C_), F32, 1).double() * (10.0 ** exps)[None, :, None, None]).to(dtype).requires_grad_()
    W, g, b = _draw((H, C_), F32, 2, C_ ** -0.5), _draw((C_,), F32, 3, 0.2, 1.0), _draw((C_,), F32, 4, 0.2)
    for size in (1.0, 1e-3) if dtype == HF else (1.0, 1e-10, 1e10):
        d = (_draw((1, 1, H, 35, 6), F32, 5) * size).to(dtype)
        out = evo.pair_bias_projection(z, W, g, b, eps=0.0)
        dz, = torch.autograd.grad(out, z, d)
        want = oc.pair_projection(z.detach(), W, g, b, 0.0, d)
        oc.check("out", out, want[0])
        oc.check("dpair", dz, want[1])


# ---------------------------------------------------------------- derivatives that are not there

def test_forward_derivatives_are_refused():
    import evoformer_triton_b200 as evo
    from torch.autograd import forward_ad
    z, W, table, pos = _draw((1, 4, 4, 64), F32, 1), _draw((4, 64), F32, 2), _draw((65, 4), F32, 3), torch.arange(4, device=DEV)
    base = _draw((1, 1, 4, 4, 4), F32, 4)
    calls = ((evo.layer_norm, [z, z[0, 0, 0], z[0, 0, 1]], {}), (evo.pair_bias_projection, [z, W, z[0, 0, 0], z[0, 0, 1]], {}),
             (lambda t, p: evo.relative_position_bias(t, pos, max_distance=32, pair_bias=p), [table, base], {}))
    for fn, args, kw in calls:
        for i in range(len(args)):
            for grads in (False, True):
                with forward_ad.dual_level(), torch.set_grad_enabled(grads):
                    a = list(args)
                    a[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i]))
                    with pytest.raises(RuntimeError, match="forward mode"):
                        fn(*a, **kw)
        fn(*args, **kw)
        # the gradient of a result, asked for with a gradient that has a derivative itself
        leaf = args[0].clone().requires_grad_()
        out = fn(leaf, *args[1:], **kw)
        with forward_ad.dual_level():
            d = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward mode"):
                torch.autograd.grad(out, leaf, d, retain_graph=True)
        torch.autograd.grad(out, leaf, torch.ones_like(out))


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("C_,H", [(128, 8), (256, 8), (256, 16), (512, 8), (500, 16)], ids=str)
def test_spread_of_rows_off_zero_does_not_lean(C_, H, dtype):
    """Rows whose mean is 1.9 deviations, and the sum of an fp32 gain's gradient, all of whose terms (a row's d . out) are positive. A
    rounding goes either way and averages out over 2 304 rows and C channels; what is cut off does not.  An MMA cuts off less
    than a unit of its sum, half of one on average; of 64 channels, four MMAs at 1/4, 2/4, 3/4 and the whole of the sum of squares cut
    off 2.5 * 2^-24 of it.  The variance is 1 / 4.61 of the mean square, r half as far off as it: 2.5 * 2^-24 * 4.61 / 2 = 3.5e-7.
    The MMA of the sums over rows cuts off less than a unit again, 1.2e-7.  (One chain over 512 channels: 3.8e-6.)"""
    import evoformer_triton_b200 as evo
    R = 48
    z = _draw((1, R, R, C_), dtype, 1, 1.0, 1.9)
    W = _draw((H, C_), F32, 2, C_ ** -0.5).requires_grad_()
    g = torch.ones(C_, device=DEV, requires_grad=True)
    out = evo.pair_bias_projection(z, W, g)
    d = out.detach()
    dg, = torch.autograd.grad(out, g, d)
    want = oc.pair_projection(z, W.detach(), g.detach(), None, 1e-5, d)[3][0]
    assert abs(float(dg.double().sum() / want.sum()) - 1) < 5.4e-7


# ---------------------------------------------------------------- sizes that no counter holds

def test_sizes_beyond_the_counters_are_refused():
    """Views of one value: 2^32 + 1 of them along an axis are not one."""
    import evoformer_triton_b200 as evo
    far = 2 ** 32 + 1
    pos, W, table = torch.zeros(1, dtype=torch.int64, device=DEV), _draw((2, 8), F32, 1), _draw((65, 2), F32, 2)
    for bad in (lambda: evo.pair_bias_projection(torch.zeros(1, 1, 1, 8, device=DEV).expand(far, 1, 1, 8), W),
                lambda: evo.pair_bias_projection(torch.zeros(1, 1, 1, 8, device=DEV).expand(1, far, 1, 8), W),
                lambda: evo.pair_bias_projection(torch.zeros(1, 1, 1, 8, device=DEV).expand(1, 1, far, 8), W),
                lambda: evo.relative_position_bias(table, pos.expand(far), pos, max_distance=32),
                lambda: evo.relative_position_bias(table, pos, pos.expand(far), max_distance=32),
                lambda: evo.relative_position_bias(table, pos[None].expand(far, 1), pos, max_distance=32),
                lambda: evo.relative_position_bias(table[:, :1].expand(65, far), pos, max_distance=32),
                lambda: evo.relative_position_bias(table, pos, max_distance=32, pair_bias=torch.zeros(1, 1, 2, 1, 1, device=DEV).expand(far, 1, 2, 1, 1))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("scheme,exact,edges,buckets", [(2, 300, list(range(310, 1010, 50)), 400), (1, 260, [270, 700, 3000], 900), (2, 1000, [], 1024)], ids=str)
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_many_distances_with_a_bucket_of_their_own(scheme, exact, edges, buckets, dtype):
    """More than a byte counts, through the C ABI: the forward to the bit, the gradient of ones exactly."""
    from evoformer_triton_b200 import _lib
    lib = _lib.load()
    Rq, Rk = 7, 1201
    q, k = torch.tensor([0, 1, 900, 1800, 2400, 2399, 1200], device=DEV), torch.arange(0, 2 * Rk, 2, device=DEV)
    rel = k[None] - q[:, None]
    a = rel.abs()
    f = torch.where(a < exact, a, exact + torch.bucketize(a, torch.tensor(edges, dtype=torch.int64, device=DEV), right=True))
    rows = torch.where(rel > 0, 0 * f, f) if scheme == 2 else f + (rel > 0) * (buckets // 2)
    table = _draw((buckets, 1), F32, 1)
    out = torch.empty((1, 1, Rq, Rk), dtype=dtype, device=DEV)
    strides = (C.c_int64 * 3)(Rq * Rk, Rq * Rk, Rk)
    code = 0 if dtype == BF else 2
    p = _lib.RelativeBiasParams(table_dtype=2, dtype=code, B=1, H=1, Rq=Rq, Rk=Rk, buckets=buckets, scheme=scheme, exact=exact, n_edges=len(edges), positions64=1,
                                edges=(C.c_int32 * max(1, len(edges)))(*edges), table=table.data_ptr(), q_pos=q.data_ptr(), k_pos=k.data_ptr(),
                                out=out.data_ptr(), out_stride=strides)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.evoattn_relative_bias_fwd(C.byref(p), stream) == 0
    assert torch.equal(out[0, 0], table[rows, 0].to(dtype))
    d, dtable = torch.ones_like(out), torch.empty_like(table)
    p.d_out, p.d_out_stride, p.dtable = d.data_ptr(), strides, dtable.data_ptr()
    need = lib.evoattn_relative_bias_bwd_workspace_bytes(C.byref(p))
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    p.workspace, p.workspace_bytes = ws.data_ptr(), need
    assert lib.evoattn_relative_bias_bwd(C.byref(p), stream) == 0
    assert torch.equal(dtable[:, 0], torch.bincount(rows.reshape(-1), minlength=buckets).to(F32))


def test_layer_norm_leaves_what_is_not_wanted():
    """Through the C ABI: with no place for a gradient given, the others are written and nothing beside them."""
    from evoformer_triton_b200 import _lib
    lib = _lib.load()
    N, C_ = 70, 96
    x, dy, w = _draw((N, C_), BF, 1), _draw((N, C_), BF, 2), _draw((C_,), F32, 3)
    h, r = oc.normalise(x.double(), 1e-5)
    stats = torch.stack([x.double().mean(-1), r[:, 0]], 1).float()
    want = oc.layer_norm(x, w, w, 1e-5, dy)
    for names in (("dx",), ("dweight",), ("dbias",), ("dx", "dbias"), ("dweight", "dbias")):
        got = {"dx": torch.full((N + 2, C_), 7.0, dtype=BF, device=DEV), "dweight": torch.full((3, C_), 7.0, device=DEV), "dbias": torch.full((3, C_), 7.0, device=DEV)}
        p = _lib.LayerNormParams(dtype=0, weight_dtype=2, bias_dtype=2, eps=1e-5, n=(1, 1, N), C=C_, x=x.data_ptr(), x_stride=(0, 0, C_), weight=w.data_ptr(), bias=w.data_ptr(),
                                 stats=stats.data_ptr(), d_y=dy.data_ptr(), d_y_stride=(0, 0, C_), **{n: got[n][1].data_ptr() for n in names})
        need = lib.evoattn_layer_norm_bwd_workspace_bytes(C.byref(p))
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
        p.workspace, p.workspace_bytes = ws.data_ptr(), need
        assert lib.evoattn_layer_norm_bwd(C.byref(p), C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        for k, (n, t) in enumerate(got.items()):
            if n not in names:
                assert (t == 7.0).all(), n
                continue
            assert (t[0] == 7.0).all() and (t[-1] == 7.0).all()
            oc.check(n, t[1:-1] if n == "dx" else t[1], want[1 + k])
