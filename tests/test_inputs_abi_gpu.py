"""GPU: the operators before the attention through the C ABI, where a caller may place results anywhere: rows of an odd pitch that
begin off a 16-byte boundary, nothing written between or behind them; and several calls at once on streams of their own."""
import ctypes as C

import pytest
import torch

from oracle import inputs_oracle as oc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MARK = 7.0


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _draw(shape, dtype, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _strides(t, axes):
    return (C.c_int64 * 3)(*(t.stride(a) for a in axes))


def _odd_rows(shape, dtype):
    """A buffer of MARKs and a view of `shape` in it whose rows have an odd pitch and an odd start."""
    n = shape[-1]
    pitch = n + 5 + n % 2
    rows = 1
    for s in shape[:-1]:
        rows *= s
    buf = torch.full((rows * pitch + 8,), MARK, dtype=dtype, device=DEV)
    st, step = [], pitch
    for s in reversed(shape[:-1]):
        st.insert(0, step)
        step *= s
    view = buf[3:].as_strided(shape, (*st, 1))
    return buf, view


def _check_untouched(buf, view):
    seen = torch.zeros_like(buf, dtype=torch.bool)
    seen[3:].as_strided(view.shape, view.stride()).fill_(True)
    assert (buf[~seen] == MARK).all()


@pytest.mark.parametrize("dtype", list(CODES), ids=str)
@pytest.mark.parametrize("Rq,Rk", [(70, 70), (5, 601), (1, 33)])
def test_relative_bias_anywhere(Rq, Rk, dtype):
    from evoformer_triton_b200 import _lib
    lib = _lib.load()
    H = 9
    table = _draw((65, H), torch.float32, 1)
    q, k = torch.arange(Rq, dtype=torch.int32, device=DEV) * 2, torch.arange(Rk, dtype=torch.int32, device=DEV)
    buf, out = _odd_rows((1, H, Rq, Rk), dtype)
    p = _lib.RelativeBiasParams(table_dtype=2, dtype=CODES[dtype], B=1, H=H, Rq=Rq, Rk=Rk, buckets=65, scheme=0, exact=32,
                                table=table.data_ptr(), q_pos=q.data_ptr(), k_pos=k.data_ptr(), out=out.data_ptr(), out_stride=_strides(out, (0, 1, 2)))
    assert lib.evoattn_relative_bias_fwd(C.byref(p), _stream()) == 0
    rows = oc.bucket_rows([q.tolist()], [k.tolist()], "clip", 65, 32).to(DEV)
    d = _draw((1, 1, H, Rq, Rk), dtype, 2)
    want, dtable = oc.relative_bias(table, rows, None, dtype, d)
    assert torch.equal(out, want[:, 0])
    _check_untouched(buf, out)
    # the gradient from rows placed as oddly
    _, view = _odd_rows((1, H, Rq, Rk), dtype)
    view.copy_(d[:, 0])
    got = torch.full_like(table, MARK)
    p.d_out, p.d_out_stride, p.dtable = view.data_ptr(), _strides(view, (0, 1, 2)), got.data_ptr()
    need = lib.evoattn_relative_bias_bwd_workspace_bytes(C.byref(p))
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    p.workspace, p.workspace_bytes = ws.data_ptr(), need
    assert lib.evoattn_relative_bias_bwd(C.byref(p), _stream()) == 0
    oc.check("dtable", got, dtable)


@pytest.mark.parametrize("dtype", list(CODES), ids=str)
@pytest.mark.parametrize("I,J,C_,H", [(3, 21, 64, 8), (11, 5, 100, 3), (2, 40, 37, 20)])
def test_pair_projection_anywhere(I, J, C_, H, dtype):
    from evoformer_triton_b200 import _lib
    lib = _lib.load()
    z, W = _draw((1, I, J, C_), dtype, 1, 2.0), _draw((H, C_), torch.float32, 2, C_ ** -0.5)
    buf, out = _odd_rows((1, H, I, J), dtype)
    dbuf, dz = _odd_rows((I * J, C_), dtype)
    p = _lib.PairProjectionParams(dtype=CODES[dtype], weight_dtype=2, eps=1e-5, B=1, Ri=I, Rj=J, C=C_, H=H, pair=z.data_ptr(),
                                  pair_stride=_strides(z, (0, 1, 2)), weight=W.data_ptr(), out=out.data_ptr(), out_stride=_strides(out, (0, 1, 2)))
    assert lib.evoattn_pair_projection_fwd(C.byref(p), _stream()) == 0
    d = _draw((1, 1, H, I, J), dtype, 3)
    want = oc.pair_projection(z, W, None, None, 1e-5, d)
    oc.check("out", out, (want[0][0][:, 0], want[0][1][:, 0]))
    _check_untouched(buf, out)
    # dpair is dense, but may begin anywhere
    flat = dbuf[3:3 + I * J * C_]
    dW = torch.full_like(W, MARK)
    p.d_out, p.d_out_stride, p.dpair, p.dweight = d.data_ptr(), _strides(d[:, 0], (0, 1, 2)), flat.data_ptr(), dW.data_ptr()
    need = lib.evoattn_pair_projection_bwd_workspace_bytes(C.byref(p))
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    p.workspace, p.workspace_bytes = ws.data_ptr(), need
    assert lib.evoattn_pair_projection_bwd(C.byref(p), _stream()) == 0
    oc.check("dpair", flat.view(1, I, J, C_), want[1])
    oc.check("dweight", dW, want[2])
    assert (dbuf[:3] == MARK).all() and (dbuf[3 + I * J * C_:] == MARK).all()


@pytest.mark.parametrize("dtype", list(CODES), ids=str)
@pytest.mark.parametrize("N,C_", [(37, 128), (6, 1000), (4, 9000)])
def test_layer_norm_anywhere(N, C_, dtype):
    from evoformer_triton_b200 import _lib
    lib = _lib.load()
    x, dy = _draw((N, C_), dtype, 1), _draw((N, C_), dtype, 2)
    buf, dbuf = (torch.full((N * C_ + 8,), MARK, dtype=dtype, device=DEV) for _ in range(2))
    stats = torch.empty(N, 2, device=DEV)
    p = _lib.LayerNormParams(dtype=CODES[dtype], eps=1e-5, n=(1, 1, N), C=C_, x=x.data_ptr(), x_stride=(0, 0, C_), y=buf[3:].data_ptr(), stats=stats.data_ptr(),
                             d_y=dy.data_ptr(), d_y_stride=(0, 0, C_), dx=dbuf[3:].data_ptr())
    assert lib.evoattn_layer_norm_fwd(C.byref(p), _stream()) == 0
    assert lib.evoattn_layer_norm_bwd_workspace_bytes(C.byref(p)) == 0
    assert lib.evoattn_layer_norm_bwd(C.byref(p), _stream()) == 0
    want = oc.layer_norm(x, None, None, 1e-5, dy)
    for name, b, w in (("y", buf, want[0]), ("dx", dbuf, want[1])):
        oc.check(name, b[3:3 + N * C_].view(N, C_), w)
        assert (b[:3] == MARK).all() and (b[3 + N * C_:] == MARK).all()


def test_several_calls_at_once():
    """Forward and backward of all three on four streams at the same time, each with workspaces of its own: the bits of calls
    made one after another."""
    import evoformer_triton_b200 as evo
    R, Cz, H = 150, 128, 8
    pos = torch.arange(R, device=DEV)

    def inputs(seed):
        leaves = [_draw((4, R, 256), torch.bfloat16, seed), _draw((256,), torch.float32, seed + 1), _draw((256,), torch.float32, seed + 2),
                  _draw((1, R, R, Cz), torch.bfloat16, seed + 3), _draw((H, Cz), torch.float32, seed + 4, 0.1), _draw((65, H), torch.float32, seed + 5)]
        return [t.requires_grad_() for t in leaves], _draw((4, R, 256), torch.bfloat16, seed + 6), _draw((1, 1, H, R, R), torch.bfloat16, seed + 7)

    def run(x):
        (m, w, b, z, W, table), dy, d = x
        y = evo.layer_norm(m, w, b)
        bias = evo.relative_position_bias(table, pos, max_distance=32, pair_bias=evo.pair_bias_projection(z, W))
        return [y.detach(), bias.detach(), *torch.autograd.grad([y, bias], [m, w, b, z, W, table], [dy, d])]

    all_inputs = [inputs(100 * i) for i in range(4)]
    want = [run(x) for x in all_inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in all_inputs]
    for _ in range(3):
        got = []
        for s, x in zip(streams, all_inputs):
            with torch.cuda.stream(s):
                got.append(run(x))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for u, v in zip(a, b):
                assert torch.equal(u, v)
