"""GPU: attention over packed sequences against its definition in 64 bits, value by value within the roundings that are
made, on the kernels that a call takes by itself and on the CUDA-core ones."""
import itertools

import pytest
import torch

from oracle import sequences_oracle as oc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
IDS = {BF: "bf16", HF: "fp16", F32: "fp32"}


def _draw(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * std).to(dtype)


def _sums(lengths, start=0):
    return list(itertools.accumulate(lengths, initial=start))


def _spans(nq, nk, q0=0, k0=0):
    return [(i, n, j, m) for i, n, j, m in zip(_sums(nq, q0), nq, _sums(nk, k0), nk)]


def _check(q, k, v, nq, nk=None, causal=True, scale=None, train=True, wide=False, before=0, seed=9):
    """A call whose sequences begin `before` rows into the tensors, against the oracle; twice to the same bits."""
    import evoformer_triton_b200 as evo
    typed = lambda x: torch.tensor(x, dtype=torch.long if wide else torch.int32, device=DEV)  # noqa: E731
    off, koff = typed(_sums(nq, before)), None if nk is None else typed(_sums(nk, before))
    spans = _spans(nq, nq if nk is None else nk, before, before)
    with torch.no_grad():
        out = evo.packed_attention(q, k, v, off, koff, causal=causal, scale=scale)
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
    if not train:
        oc.check("o", out, oc.attention(q.detach(), k.detach(), v.detach(), spans, causal, scale)[0])
        return out
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    d = _draw(q.shape, q.dtype, seed)
    again = evo.packed_attention(*leaves, off, koff, causal=causal, scale=scale)
    grads = torch.autograd.grad(again, leaves, d, retain_graph=True)
    for a, b in zip(grads, torch.autograd.grad(again, leaves, d)):
        assert torch.equal(a, b)
    want = oc.attention(q.detach(), k.detach(), v.detach(), spans, causal, scale, d)
    for name, got, w in zip(("o of training", "dq", "dk", "dv"), (again, *grads), want):
        oc.check(name, got, w)
    oc.check("o", out, want[0])
    return out


def _qkv(T, Tk, H, Hk, D, dtype, seed=1, std=1.0):
    return _draw((T, H, D), dtype, seed, std), _draw((Tk, Hk, D), dtype, seed + 1, std), _draw((Tk, Hk, D), dtype, seed + 2)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("lengths", [[1], [2, 1, 1], [63, 64, 65], [127], [128], [129], [255, 257], [300, 1, 130, 5], [384, 512], [640]], ids=str)
def test_lengths(lengths, causal, dtype):
    _check(*_qkv(sum(lengths), sum(lengths), 4, 2, 64, dtype), lengths, causal=causal)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("D", [1, 7, 8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 120, 128, 136, 192, 256])
def test_head_dimensions(D, dtype):
    _check(*_qkv(290, 290, 2, 1, D, dtype), [150, 11, 129])


@pytest.mark.parametrize("dtype", [BF, F32], ids=IDS.get)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 3), (2, 1), (3, 1), (8, 2), (12, 4), (6, 3), (40, 8), (16, 1), (33, 1), (71, 71)])
def test_heads(H, Hk, D, dtype):
    _check(*_qkv(210, 210, H, Hk, D, dtype), [140, 70])


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("nq,nk", [([5], [300]), ([130, 1], [257, 64]), ([1, 1, 1], [1, 129, 640]), ([128], [129]), ([300], [100]), ([7, 200, 3], [0, 50, 3]), ([0, 3, 0], [5, 0, 9]),
                                   ([256, 128], [1000, 128]), ([64], [1000]), ([129], [1])], ids=str)
def test_queries_and_keys_of_different_lengths(nq, nk, causal, dtype):
    """Fewer queries than keys (the last query sees all), more (the first ones see none), none of either."""
    _check(*_qkv(sum(nq), sum(nk), 4, 2, 64, dtype), nq, nk, causal)


@pytest.mark.parametrize("dtype", [BF, F32], ids=IDS.get)
@pytest.mark.parametrize("D", [64, 128])
def test_many_sequences(D, dtype):
    """More sequences than a block has threads, empty ones among them."""
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 9, (700,), generator=g).tolist() + [140]
    _check(*_qkv(sum(lengths), sum(lengths), 2, 1, D, dtype), lengths, wide=True)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("D", [64, 128])
def test_many_tiles_of_keys_that_no_query_sees(D, dtype):
    """Far more of them than there are SMs, behind and between tiles with queries: their rows of dK and dV are zero."""
    nq, nk = [130, 0, 300] + [0] * 200 + [5], [260, 700, 1] + [130] * 200 + [140]
    _check(*_qkv(sum(nq) + 6, sum(nk) + 6, 8, 4, D, dtype), nq, nk, before=3)
    _check(*_qkv(sum(nq), sum(nk), 8, 4, D, dtype), nq, nk, causal=False)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("nk", [1, 15, 16, 17, 64, 65, 500, 5000])
@pytest.mark.parametrize("H,Hk,D", [(8, 8, 64), (32, 8, 128), (12, 2, 96), (40, 2, 32), (4, 1, 256), (3, 1, 20)])
def test_single_tokens(H, Hk, D, nk, dtype):
    _check(*_qkv(3, 3 * nk + 7, H, Hk, D, dtype), [1, 1, 1], [nk, nk + 7, nk], train=False)


@pytest.mark.parametrize("dtype", [BF, F32], ids=IDS.get)
def test_a_few_tokens_each_and_one_long(dtype):
    nq, nk = [2, 4, 1, 3, 2], [800, 4, 3000, 65, 1]
    _check(*_qkv(sum(nq), sum(nk), 8, 2, 64, dtype), nq, nk, train=False)
    _check(*_qkv(sum(nq), sum(nk), 8, 2, 64, dtype), nq, nk, causal=False, train=False)
    nq, nk = [1] * 30 + [300], [40] * 30 + [2000]
    _check(*_qkv(sum(nq), sum(nk), 8, 2, 128, dtype), nq, nk, train=False)


@pytest.mark.parametrize("dtype", [BF, HF], ids=IDS.get)
@pytest.mark.parametrize("nq,nk", [([300], [9000]), ([129, 40, 7], [5000, 40, 6100]), ([256], [4000]), ([1000], None), ([2500], None)], ids=str)
def test_long_rows_of_tiles_are_cut(nq, nk, dtype):
    """Few queries against many keys, and few heads: parts of a tile that are joined, in both directions."""
    for H, Hk, D in ((2, 1, 64), (1, 1, 128), (3, 1, 128), (6, 1, 96)):
        for causal in (True, False):
            _check(*_qkv(sum(nq), sum(nk or nq), H, Hk, D, dtype), nq, nk, causal)


def test_thousands_of_tokens():
    """More sequences than a launch of the kernel for few rows takes; empty ones, sequences without keys, rows of none."""
    import evoformer_triton_b200 as evo
    g = torch.Generator().manual_seed(3)
    nk = torch.randint(0, 70, (5000,), generator=g).tolist()
    nq = [int(i % 7 != 3) for i in range(5000)]
    nq[4990], nk[4990] = 40, 3000
    _check(*_qkv(sum(nq), sum(nk), 2, 1, 64, BF), nq, nk, train=False)
    q, k, v = _qkv(sum(nq) + 9, sum(nk), 2, 1, 64, BF)
    off = torch.tensor(_sums(nq, 4), device=DEV)
    out = evo.packed_attention(q, k, v, off, torch.tensor(_sums(nk), device=DEV))
    assert not out[:4].any() and not out[-5:].any() and out[4:-5].any(-1).any()


@pytest.mark.parametrize("nq", [[1] * 6 + [64, 1], [3, 2, 1, 200, 4]], ids=["one of many", "mixed"])
def test_tokens_beside_prompts(nq):
    """New tokens and prompts in one call, each to its kernel."""
    nk = [900, 33, 64, 1, 4000, 129, 700, 17][:len(nq)]
    for H, Hk, D in ((8, 2, 64), (6, 1, 128), (40, 1, 64)):
        for causal in (True, False):
            _check(*_qkv(sum(nq), sum(nk), H, Hk, D, BF), nq, nk, causal, train=False)


@pytest.mark.parametrize("dtype", [BF, HF], ids=IDS.get)
@pytest.mark.parametrize("nk", [[100_000], [70_000, 64, 513, 512], [5000] * 40], ids=["one long", "uneven", "even"])
def test_long_rows_of_keys_are_shared_out(nk, dtype):
    for H, Hk, D in ((4, 4, 128), (16, 1, 64)):
        _check(*_qkv(len(nk), sum(nk), H, Hk, D, dtype), [1] * len(nk), nk, train=False)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("nq", [[1, 1, 1, 1, 1], [100, 1, 140, 37, 3]], ids=["tokens", "pieces"])
def test_keys_in_slots(nq, dtype):
    """Key ranges in any order, shared, with whatever in between; ranges that leave the tensor are cut."""
    import evoformer_triton_b200 as evo
    q, k, v = _qkv(sum(nq), 1000, 4, 2, 64, dtype)
    ranges = [(500, 1000), (0, 1), (20, 270), (20, 270), (300, 340)]
    used = torch.zeros(1000, dtype=torch.bool, device=DEV)
    for a, b in ranges:
        used[a:b] = True
    for bad in (float("nan"), float("inf")):
        k2, v2 = (torch.where(used[:, None, None], t, bad) for t in (k, v))
        for wide in (torch.int32, torch.int64):
            out = evo.packed_attention(q, k2, v2, torch.tensor(_sums(nq), dtype=torch.int32, device=DEV), torch.tensor(ranges, dtype=wide, device=DEV))
            spans = [(i, n, a, b - a) for i, n, (a, b) in zip(_sums(nq), nq, ranges)]
            oc.check("o", out, oc.attention(q, k, v, spans, True)[0])
    cut = [(500, 4000), (-10, 1), (20, 270), (270, 20), (1000, 1040)]
    out = evo.packed_attention(q, k, v, torch.tensor(_sums(nq), device=DEV), torch.tensor(cut, device=DEV))
    spans = [(i, n, a, b - a) for i, n, (a, b) in zip(_sums(nq), nq, [(500, 1000), (0, 1), (20, 270), (0, 0), (0, 0)])]
    oc.check("o", out, oc.attention(q, k, v, spans, True)[0])


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("D", [64, 96, 128])
def test_rows_outside_the_sequences(D, dtype):
    """Rows before the first and behind the last sequence hold infinities and NaN: they come back as zeros, gradients too."""
    import evoformer_triton_b200 as evo
    for nq, nk in (([70, 130], None), ([3, 200], [60, 290])):
        T, Tk = 40 + sum(nq) + 90, 40 + sum(nk or nq) + 90
        q, k, v = _qkv(T, Tk, 4, 2, D, dtype)
        d = _draw(q.shape, dtype, 4)
        for t, n in ((q, nq), (k, nk or nq), (v, nk or nq), (d, nq)):
            t[:40], t[40 + sum(n):] = float("nan"), float("-inf")
        off = torch.tensor(_sums(nq, 40), device=DEV)
        koff = None if nk is None else torch.tensor(_sums(nk, 40), device=DEV)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = evo.packed_attention(*leaves, off, koff)
        got = [out, *torch.autograd.grad(out, leaves, d)]
        clean = [torch.nan_to_num(t.detach(), 0.0, 0.0, 0.0) for t in (q, k, v, d)]
        want = oc.attention(*clean[:3], _spans(nq, nk or nq, 40, 40), True, d=clean[3])
        for name, g, w in zip(("o", "dq", "dk", "dv"), got, want):
            oc.check(name, g, w)
            n = sum(nq) if name in ("o", "dq") else sum(nk or nq)
            assert not g[:40].any() and not g[40 + n:].any()


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
def test_a_sequence_does_not_see_its_neighbour(dtype):
    """NaN and infinities in one sequence stay there, also where its rows lie in a tile of the next one's."""
    import evoformer_triton_b200 as evo
    lengths = [50, 77, 200, 3]
    for bad in (0, 1, 2, 3):
        q, k, v = _qkv(330, 330, 4, 2, 64, dtype)
        d = _draw(q.shape, dtype, 4)
        rows = slice(sum(lengths[:bad]), sum(lengths[:bad + 1]))
        for t, x in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (d, float("-inf"))):
            t[rows] = x
        off = torch.tensor(_sums(lengths), device=DEV)
        for causal in (True, False):
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            out = evo.packed_attention(*leaves, off, causal=causal)
            got = [out, *torch.autograd.grad(out, leaves, d)]
            clean = [torch.nan_to_num(t, 0.0, 0.0, 0.0) for t in (q, k, v, d)]
            spans = [s for n, s in enumerate(_spans(lengths, lengths)) if n != bad]
            keep = torch.ones(330, dtype=torch.bool, device=DEV)
            keep[rows] = False
            for name, g, (w, e) in zip(("o", "dq", "dk", "dv"), got, oc.attention(*clean[:3], spans, causal, d=clean[3])):
                oc.check(name, g.detach()[keep], (w[keep], e[keep]))


def _layouts():
    return {
        "slices of one projection": lambda dt: (lambda x: (x[:, :4], x[:, 4:6], x[:, 6:]))(_draw((200, 8, 64), dt, 1)),
        "heads before rows": lambda dt: tuple(_draw((h, 200, 64), dt, n).transpose(0, 1) for n, h in enumerate((4, 2, 2))),
        "rows of an odd pitch": lambda dt: tuple(_draw((200, h, 65), dt, n)[..., 1:] for n, h in enumerate((4, 2, 2))),
        "values not contiguous": lambda dt: tuple(_draw((200, 64, h), dt, n).transpose(1, 2) for n, h in enumerate((4, 2, 2))),
        "every other row": lambda dt: tuple(_draw((400, h, 64), dt, n)[::2] for n, h in enumerate((4, 2, 2))),
        "one key head for all": lambda dt: (_draw((200, 4, 64), dt, 1), *(_draw((200, 1, 64), dt, n).expand(200, 2, 64) for n in (2, 3))),
        "one row for all": lambda dt: (_draw((1, 4, 64), dt, 1).expand(200, 4, 64), _draw((200, 2, 64), dt, 2), _draw((1, 2, 64), dt, 3).expand(200, 2, 64)),
        "a base off 16 bytes": lambda dt: tuple(_draw((200 * h * 64 + 1,), dt, n)[1:].view(200, h, 64) for n, h in enumerate((4, 2, 2))),
    }


@pytest.mark.parametrize("dtype", [BF, F32], ids=IDS.get)
@pytest.mark.parametrize("name", sorted(_layouts()))
def test_rows_are_read_where_they_lie(name, dtype):
    import evoformer_triton_b200 as evo
    q, k, v = (t.detach() for t in _layouts()[name](dtype))
    lengths = [129, 71]
    d = _draw((4, 200, 64), dtype, 8).transpose(0, 1)  # (a gradient that is not dense either)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = evo.packed_attention(*leaves, torch.tensor(_sums(lengths), device=DEV))
    got = [out, *torch.autograd.grad(out, leaves, d)]
    for n, g, w in zip(("o", "dq", "dk", "dv"), got, oc.attention(q.detach(), k.detach(), v.detach(), _spans(lengths, lengths), True, d=d)):
        oc.check(n, g, w)
    with torch.no_grad():
        tokens = evo.packed_attention(q[:2], k, v, torch.tensor([0, 1, 2], device=DEV), torch.tensor([0, 90, 200], device=DEV))
    oc.check("tokens", tokens, oc.attention(q.detach()[:2], k.detach(), v.detach(), [(0, 1, 0, 90), (1, 1, 90, 110)], True)[0])


def test_gradient_of_one_value_for_all():
    """What .sum() hands over: a gradient whose strides are zero."""
    import evoformer_triton_b200 as evo
    for dtype in (BF, F32):
        leaves = [t.requires_grad_() for t in _qkv(150, 150, 4, 2, 64, dtype)]
        out = evo.packed_attention(*leaves, torch.tensor([0, 150], device=DEV))
        grads = torch.autograd.grad(out.sum(), leaves)
        want = oc.attention(*(t.detach() for t in leaves), [(0, 150, 0, 150)], True, d=torch.ones_like(out))
        for n, g, w in zip(("dq", "dk", "dv"), grads, want[1:]):
            oc.check(n, g, w)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-3, 3.0])
def test_scales(scale, dtype):
    _check(*_qkv(200, 200, 2, 1, 32, dtype), [200], scale=scale)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rise", ["up", "down", "steps", "spike"])
def test_scores_that_rise_along_the_keys(rise, D, dtype):
    """Maxima that a running maximum has to follow, tile after tile or at once, and rows that one key dominates."""
    T = 700
    g = torch.arange(T, device=DEV, dtype=torch.float32)
    w = {"up": g / 20, "down": (T - g) / 20, "steps": (g // 128) * 12, "spike": (g == 500) * 60.0 + (g == 3) * 30.0}[rise]
    q, k, v = _qkv(T, T, 2, 1, D, dtype, std=0.2)
    q, k = q.clone(), k.clone()
    q[..., 0], k[..., 0] = 1.0, w[:, None].to(dtype)  # scores: w of the key, next to a little noise
    for causal in (True, False):
        _check(q, k, v, [T], causal=causal, scale=1.0)
    with torch.no_grad():
        _check(q[:2], k, v, [1, 1], [600, 100], scale=1.0, train=False)


@pytest.mark.parametrize("dtype", [BF, HF], ids=IDS.get)
def test_cuda_core_kernels_agree(dtype):
    import evoformer_triton_b200 as evo
    evo.force_generic(True)
    try:
        _check(*_qkv(400, 400, 4, 2, 128, dtype), [260, 140])
        _check(*_qkv(2, 400, 4, 2, 128, dtype), [1, 1], [260, 140], train=False)
    finally:
        evo.force_generic(False)


def test_which_kernels_a_call_takes():
    from evoformer_triton_b200 import _lib, attention
    for dtype, D, want in ((BF, 64, _lib.PATH_TCGEN05), (HF, 128, _lib.PATH_TCGEN05), (BF, 8, _lib.PATH_TCGEN05), (F32, 64, _lib.PATH_GENERIC), (BF, 136, _lib.PATH_GENERIC), (BF, 20, _lib.PATH_GENERIC)):
        _check(*_qkv(150, 150, 2, 1, D, dtype), [150])
        assert attention.last_path["fwd"] == attention.last_path["bwd"] == want


def test_gradients_against_differences():
    import evoformer_triton_b200 as evo
    off = torch.tensor([0, 40, 97], device=DEV)
    x = [t.requires_grad_() for t in _qkv(97, 97, 4, 2, 16, F32)]
    d = _draw((97, 4, 16), F32, 5)
    grads = torch.autograd.grad(evo.packed_attention(*x, off), x, d)
    for n, g in enumerate(grads):
        step = _draw(x[n].shape, F32, 6 + n)
        with torch.no_grad():
            at = lambda h: (evo.packed_attention(*(t + h * step if m == n else t for m, t in enumerate(x)), off).double() * d).sum()  # noqa: E731
            slope = (at(1e-2) - at(-1e-2)) / 2e-2
        # third derivatives of a smooth function of size one: 1e-4 of the slope's terms; outputs to 1e-6 over 2e-2
        assert abs(float(slope - (g.double() * step).sum())) < 1e-2 * float((g.double() * step).abs().sum()) ** 0.5


def test_gradients_of_some():
    import evoformer_triton_b200 as evo
    off = torch.tensor([0, 150], device=DEV)
    for dtype in (BF, F32):
        q, k, v = _qkv(150, 150, 4, 2, 64, dtype)
        d = _draw(q.shape, dtype, 5)
        want = oc.attention(q, k, v, [(0, 150, 0, 150)], True, d=d)[1:]
        for which in ((0,), (1,), (2,), (0, 2), (1, 2)):
            x = [t.detach().requires_grad_(n in which) for n, t in enumerate((q, k, v))]
            got = torch.autograd.grad(evo.packed_attention(*x, off), [x[n] for n in which], d)
            for n, g in zip(which, got):
                oc.check(str(n), g, want[n])
        x = q.detach().requires_grad_()  # one tensor as all three
        out = evo.packed_attention(x, x, x, off)
        (g,) = torch.autograd.grad(out, x, d)
        w = oc.attention(q, q, q, [(0, 150, 0, 150)], True, d=d)[1:]
        # three results of the type added in it: each of them rounded, and twice the sum
        e = sum(t[1] for t in w) + 4 * torch.finfo(dtype).eps * sum(t[0].abs() for t in w)
        oc.check("one for all", g, (sum(t[0] for t in w), e))


@pytest.mark.parametrize("nq,nk,train", [([200, 60], None, True), ([1, 1], [300, 50], False)], ids=["training", "tokens"])
def test_graph_with_other_lengths(nq, nk, train):
    """Captured once; replayed with other values and other lengths in the same tensors."""
    import evoformer_triton_b200 as evo
    T, Tk = sum(nq), sum(nk or nq)
    q, k, v = (t.requires_grad_(train) for t in _qkv(T, Tk, 4, 2, 64, BF))
    d = _draw(q.shape, BF, 5)
    off = torch.tensor(_sums(nq), device=DEV)
    koff = None if nk is None else torch.tensor(_sums(nk), device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = evo.packed_attention(q, k, v, off, koff)
        grads = torch.autograd.grad(out, (q, k, v), d) if train else ()
    others = [(nq, nk), ([90, 100], None) if nk is None else ([1, 1], [3, 340])]
    for seed, (n, m) in enumerate(others):
        with torch.no_grad():
            for t, s in zip((q, k, v), _qkv(T, Tk, 4, 2, 64, BF, seed=20 + 3 * seed)):
                t.copy_(s)
            off.copy_(torch.tensor(_sums(n)))
            if koff is not None:
                koff.copy_(torch.tensor(_sums(m)))
        graph.replay()
        want = oc.attention(q.detach(), k.detach(), v.detach(), _spans(n, m or n), True, d=d if train else None)
        for g, w in zip((out, *grads), want):
            oc.check("replayed", g, w)


def test_two_calls_at_once():
    """Two streams: nothing is shared between calls."""
    import evoformer_triton_b200 as evo
    sets = [(_qkv(600, 600, 8, 2, 64, BF, seed=s), torch.tensor([0, 250, 600], device=DEV)) for s in (1, 11)]
    tok = [(_qkv(4, 8000, 8, 2, 64, BF, seed=s), torch.arange(5, device=DEV), torch.tensor([0, 1000, 3000, 7000, 8000], device=DEV)) for s in (1, 11)]
    want = [evo.packed_attention(*x, o) for x, o in sets] + [evo.packed_attention(*x, o, c) for x, o, c in tok]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(20):
        got = []
        for st, call in zip(streams, [lambda x=x, o=o: evo.packed_attention(*x, o) for x, o in sets] + [lambda x=x, o=o, c=c: evo.packed_attention(*x, o, c) for x, o, c in tok]):
            with torch.cuda.stream(st):
                got.append(call())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_nothing_in():
    import evoformer_triton_b200 as evo
    for T, Tk, B in ((0, 0, 0), (5, 5, 0), (0, 5, 1), (5, 0, 1)):
        q, k, v = (t.requires_grad_() for t in _qkv(T, Tk, 4, 2, 64, BF))
        off = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
        out = evo.packed_attention(q, k, v, off, off)
        assert out.shape == q.shape and not out.any()
        for t, g in zip((q, k, v), torch.autograd.grad(out.sum(), (q, k, v))):
            assert g.shape == t.shape and not g.any()


def test_offsets_that_make_no_sense_touch_nothing():
    """Descending, negative and far offsets: rows outside the tensors are not touched, and the next call is right."""
    import evoformer_triton_b200 as evo
    q, k, v = (t.requires_grad_() for t in _qkv(200, 200, 4, 2, 64, BF))
    for bad in ([0, 10 ** 12, 200], [-5, 50, 10 ** 6], [150, 20, 90], [300, 400, 500], [-2 ** 60, 2 ** 60, 0], [0, 200] * 40, [200, 0] * 300):
        out = evo.packed_attention(q, k, v, torch.tensor(bad, device=DEV))
        torch.autograd.grad(out.sum(), (q, k, v))
        few = torch.arange(len(bad), device=DEV).clamp(max=2)
        evo.packed_attention(q[:2].detach(), k.detach(), v.detach(), few, torch.tensor(bad, device=DEV))
        evo.packed_attention(q.detach(), k.detach(), v.detach(), torch.tensor(bad, device=DEV), torch.tensor(bad, device=DEV))
    torch.cuda.synchronize()
    evo.check_device_status()
    _check(q, k, v, [60, 140])


def test_refusals():
    import evoformer_triton_b200 as evo
    q, k, v = _qkv(6, 6, 4, 2, 32, BF)
    off = torch.tensor([0, 2, 6], device=DEV)
    call = evo.packed_attention
    big = torch.zeros(6, 2, 260, dtype=BF, device=DEV)
    bad = [
        (TypeError, lambda: call(q.double(), k, v, off)), (TypeError, lambda: call(q, k.float(), v, off)), (TypeError, lambda: call(q, k, v.half(), off)),
        (ValueError, lambda: call(q[0], k, v, off)), (ValueError, lambda: call(q, k[..., 0], v, off)), (ValueError, lambda: call(q[:, :3], k, v, off)),
        (ValueError, lambda: call(q, k, v[:5], off)), (ValueError, lambda: call(q, k[..., :16], v[..., :16], off)), (ValueError, lambda: call(big, big, big, off)),
        (ValueError, lambda: call(q[:4], k, v, off)), (ValueError, lambda: call(q, k[:, :0], v[:, :0], off)), (RuntimeError, lambda: call(q, k.cpu(), v, off)),
        (RuntimeError, lambda: call(q, k, v, off.cpu())), (TypeError, lambda: call(q, k, v, off.float())), (ValueError, lambda: call(q, k, v, off[None])),
        (ValueError, lambda: call(q, k, v, off[:0])), (ValueError, lambda: call(q, k, v, off, off[:2])), (ValueError, lambda: call(q, k, v, off, off[None].expand(3, 3))),
        (RuntimeError, lambda: call(q, k, v, off, off.cpu())), (TypeError, lambda: call(q, k, v, off, off.short())),
        (ValueError, lambda: call(q, k, v, off, scale=float("nan"))), (ValueError, lambda: call(q, k, v, off, scale=float("inf"))), (ValueError, lambda: call(q, k, v, off, scale=1e300)),
        (ValueError, lambda: call(q, k.clone().requires_grad_(), v, off, torch.tensor([[0, 2], [2, 6]], device=DEV))),
    ]
    for kind, fn in bad:
        with pytest.raises(kind):
            fn()
    # a gradient of q alone with keys in ranges is one that there is
    x = q.clone().requires_grad_()
    out = call(x, k, v, off, torch.tensor([[0, 2], [1, 6]], device=DEV))
    (g,) = torch.autograd.grad(out.sum(), x)
    oc.check("dq", g, oc.attention(q, k, v, [(0, 2, 0, 2), (2, 4, 1, 5)], True, d=torch.ones_like(q))[1])
    x = q.float().requires_grad_()
    out = call(x, k.float(), v.float(), off)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(out.sum(), x, create_graph=True)
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
        call(fwad.make_dual(q.float(), q.float()), k.float(), v.float(), off)


@pytest.mark.parametrize("dtype", [BF, F32], ids=IDS.get)
def test_a_trunk_in_training_and_token_by_token(dtype):
    """The operators as they are used together: a projection, its q and k turned, attention over packed sequences; the
    same written one token at a time into a cache, which has to agree with the whole."""
    import evoformer_triton_b200 as evo
    lengths, H, Hk, D, C = [37, 5, 130], 4, 2, 64, 96
    T = sum(lengths)
    w = _draw(((H + 2 * Hk) * D, C), dtype, 1, C ** -0.5)
    x = _draw((T, C), dtype, 2)
    f = evo.rotary_frequencies(D, scaling="bands", factor=4.0, original_length=64, device=DEV)
    pos = torch.cat([torch.arange(n) for n in lengths]).to(DEV)
    off = torch.tensor(_sums(lengths), device=DEV)

    def qkv(x, pos):
        y = torch.nn.functional.linear(x, w).view(-1, H + 2 * Hk, D)
        q, k = evo.rotary_embedding(y[:, :H], y[:, H:H + Hk], pos, f)
        return q, k, y[:, H + Hk:]

    xg = x.clone().requires_grad_()
    q, k, v = qkv(xg, pos)
    out = evo.packed_attention(q, k, v, off)
    d = _draw(out.shape, dtype, 3)
    (dx,) = torch.autograd.grad(out, xg, d)
    oc.check("o", out, oc.attention(q.detach(), k.detach(), v.detach(), _spans(lengths, lengths), True)[0])
    # the same in 64 bits, differentiated
    x64 = x.double().requires_grad_()
    y = (x64 @ w.double().t()).view(T, H + 2 * Hk, D)
    n = D // 2
    ang = pos.double()[:, None, None] * f
    turn = lambda t: torch.cat([t[..., :n] * ang.cos() - t[..., n:] * ang.sin(), t[..., :n] * ang.sin() + t[..., n:] * ang.cos()], -1)  # noqa: E731
    q64, k64, v64 = turn(y[:, :H]), turn(y[:, H:H + Hk]).repeat_interleave(H // Hk, 1), y[:, H + Hk:].repeat_interleave(H // Hk, 1)
    o64 = torch.cat([torch.nn.functional.scaled_dot_product_attention(q64[a:b].transpose(0, 1), k64[a:b].transpose(0, 1), v64[a:b].transpose(0, 1), is_causal=True).transpose(0, 1)
                     for a, b in zip(_sums(lengths), _sums(lengths)[1:])])
    (dx64,) = torch.autograd.grad(o64, x64, d.double())
    # every step of the chain rounds to the type: five roundings forward and back, of vectors of independent errors
    tol = 8 * torch.finfo(dtype).eps if dtype == BF else 1e-5
    assert float((dx.double() - dx64).norm() / dx64.norm()) < tol
    assert float((out.detach().double() - o64.detach()).norm() / o64.detach().norm()) < tol
    # token by token: slots of a cache, one new token of each sequence a step
    slots = 160
    kc, vc = (torch.full((len(lengths) * slots, Hk, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    got = torch.empty_like(out)
    begin = _sums(lengths)[:-1]
    with torch.no_grad():
        for t in range(max(lengths)):
            live = [b for b, n in enumerate(lengths) if t < n]
            rows = torch.tensor([begin[b] + t for b in live], device=DEV)
            qt, kt, vt = qkv(x[rows], torch.full((len(live),), t, device=DEV))
            at = torch.tensor([b * slots + t for b in live], device=DEV)
            kc[at], vc[at] = kt, vt
            got[rows] = evo.packed_attention(qt, kc, vc, torch.arange(len(live) + 1, device=DEV), torch.tensor([[b * slots, b * slots + t + 1] for b in live], device=DEV))
    assert float((got.double() - o64.detach()).norm() / o64.detach().norm()) < tol


def test_a_long_cache_whose_offsets_pass_32_bits():
    """More than 2^32 values of keys: the last slot's lie behind them."""
    import evoformer_triton_b200 as evo
    rows, Hk, D = 2_150_000, 16, 128  # 4.4e9 values, 8.8 GB each
    if torch.cuda.mem_get_info()[0] < 24e9:
        pytest.skip("needs 24 GB")
    k, v = (torch.empty(rows, Hk, D, dtype=BF, device=DEV) for _ in range(2))
    for nq in ([1, 1], [200, 1]):
        q = _draw((sum(nq), 2 * Hk, D), BF, 1)
        spans = [(0, nq[0], rows - 700, 700), (nq[0], nq[1], 3, 300)]
        for n, (_, _, j, m) in enumerate(spans):
            k[j:j + m], v[j:j + m] = _draw((m, Hk, D), BF, 2 + n), _draw((m, Hk, D), BF, 5 + n)
        ranges = torch.tensor([[j, j + m] for _, _, j, m in spans], device=DEV)
        out = evo.packed_attention(q, k, v, torch.tensor(_sums(nq), device=DEV), ranges)
        for i, n, j, m in spans:
            oc.check("o", out[i:i + n], oc.attention(q[i:i + n], k[j:j + m], v[j:j + m], [(0, n, 0, m)], True)[0])
