"""GPU: attention over packed sequences where little or nothing is left: single rows, values that are not finite, gradients near the
ends of a type, offsets that overlap."""
import pytest
import torch

from oracle import sequences_oracle as oc
from test_packed_attention_gpu import BF, DEV, F32, HF, IDS, _check, _draw, _qkv, _spans, _sums

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("D", [1, 8, 20, 32, 64, 128, 256])
@pytest.mark.parametrize("T,H", [(1, 1), (1, 2), (3, 1), (1, 5), (7, 1), (9, 3)])
def test_gradients_of_a_few_rows(T, H, D, dtype):
    """Fewer rows of dO * O than a warp adds up at once, and numbers of them that it does not divide."""
    _check(*_qkv(T, T, H, 1, D, dtype), [T])


@pytest.mark.parametrize("dtype", [BF, HF], ids=IDS.get)
@pytest.mark.parametrize("H,Hk,D", [(8, 8, 64), (32, 8, 128), (12, 2, 96), (6, 1, 64)])
@pytest.mark.parametrize("nk", [[1], [130], [700, 64, 5000, 33]], ids=str)
def test_tokens_lose_only_the_rounding_of_their_results(nk, H, Hk, D, dtype):
    """P enters its product in two pieces of the type.  What is left of its rounding is half a step of half a step."""
    import evoformer_triton_b200 as evo
    q, k, v = _qkv(len(nk), sum(nk), H, Hk, D, dtype)
    spans = _spans([1] * len(nk), nk)
    out = evo.packed_attention(q, k, v, torch.tensor(_sums([1] * len(nk)), device=DEV), torch.tensor(_sums(nk), device=DEV))
    value, bound = oc.attention(q.float(), k.float(), v.float(), spans, True)[0]  # (that of sums and exponentials in fp32)
    big = oc.attention(q.float(), k.float(), v.float().abs(), spans, True)[0][0]  # sums of p |v|
    u = torch.finfo(dtype).eps / 2
    # the second piece rounded (fp16: by half of its smallest step too, against a sum of one or more)
    bound = bound + u * u * big + (max(nk) * 2.0 ** -25 * v.abs().max().double() if dtype == HF else 0.0)
    oc.check("o", out, (value, bound + oc.rounding(dtype, value.abs() + bound)))


HALF_LENGTHS = [[1500], [700, 37, 900]]


def _half_gradients(q, k, v, d, lengths, causal):
    import evoformer_triton_b200 as evo
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    return torch.autograd.grad(evo.packed_attention(*leaves, torch.tensor(_sums(lengths), device=DEV), causal=causal), leaves, d)


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("lengths", HALF_LENGTHS, ids=str)
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (2, 1, 96), (2, 2, 128)])
def test_fp16_gradients_of_a_gradient_of_any_size(H, Hk, D, lengths, causal):
    """A gradient times a power of two makes gradients times that power but for the rounding of the results: dS neither
    loses its bits at the lower end of fp16 nor passes its upper end.  Roundings are even over a step: half a step over the root
    of three each, which is 0.58 of it; the rest is for the few dS that round to the other side."""
    q, k, v = _qkv(sum(lengths), sum(lengths), H, Hk, D, HF)
    d = (_draw(q.shape, F32, 5) * 64).round() / 64  # (multiples of 2^-6, which fp16 holds exactly times 2^-18 as well)
    base = _half_gradients(q, k, v, d.to(HF), lengths, causal)
    for power in (-18, -12, -8, 5, 12):
        got = _half_gradients(q, k, v, (d * 2.0 ** power).to(HF), lengths, causal)
        for name, g, b in zip(("dq", "dk", "dv"), got, base):
            want = b.double() * 2.0 ** power
            off = torch.where(want.abs() < 65000, g.double() - want, 0.0)
            steps = float(oc.rounding(HF, b.double()).norm()) * 2.0 ** power + float(oc.rounding(HF, want).norm())
            assert float(off.norm()) <= 0.65 * steps, (name, power, float(off.norm()) / steps)
            assert torch.equal(torch.isfinite(g), torch.isfinite(want.to(HF))) or power == 12


@pytest.mark.parametrize("std", [1.0, 1e-3, 1e-4, 3000.0])
@pytest.mark.parametrize("H,Hk,D", [(4, 1, 64), (2, 1, 96)])
def test_fp16_gradients_by_their_norm(H, Hk, D, std):
    """Of far rows too: what rounding the results makes (half a step over the root of three, 0.58 of it), and half a step more for
    those of P and dS, which are as independent."""
    T = 1600
    q, k, v = _qkv(T, T, H, Hk, D, HF)
    d = _draw(q.shape, HF, 5, std)
    want = oc.attention(q, k, v, [(0, T, 0, T)], True, d=d)[1:]
    for name, g, (w, _) in zip(("dq", "dk", "dv"), _half_gradients(q, k, v, d, [T], True), want):
        for rows in (slice(0, 400), slice(400, 1000), slice(1000, T)):
            x = w[rows]
            assert float((g[rows].double() - x).norm()) <= 0.65 * float(oc.rounding(HF, x).norm()) + torch.finfo(HF).eps / 2 * float(x.norm()), (name, rows)


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 6e4])
def test_fp16_gradients_beside_ones_of_another_size(bad):
    """Sequences, and rows of none, whose gradients or values are huge or not finite say nothing about the others."""
    lengths, D = [300, 200, 129], 64
    T = sum(lengths) + 9
    q, k, v = _qkv(T, T, 4, 2, D, HF)
    d = _draw(q.shape, HF, 5)
    for t in (q, k, v, d):
        t[:4], t[-5:] = bad, float("nan")
    d[4 + 300:4 + 500] = bad
    spans = _spans(lengths, lengths, 4, 4)
    import evoformer_triton_b200 as evo
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(evo.packed_attention(*leaves, torch.tensor(_sums(lengths, 4), device=DEV)), leaves, d)
    clean = [torch.nan_to_num(t, 0.0, 0.0, 0.0) for t in (q, k, v, d)]
    keep = torch.zeros(T, dtype=torch.bool, device=DEV)
    keep[4:304] = keep[504:-5] = True
    for name, g, (w, e) in zip(("dq", "dk", "dv"), got, oc.attention(*clean[:3], spans, True, d=clean[3])[1:]):
        if bad < 1e5:
            oc.check(name, g, (w, e))
        oc.check(name, g[keep], (w[keep], e[keep]))


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (3, 1, 128), (2, 2, 20)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_queries_without_a_key_may_hold_anything(bad, H, Hk, D, dtype):
    """q and the gradient of queries that the mask leaves no key (more queries than keys, or no keys at all): zeros come back, and
    nothing of them reaches the other rows."""
    import evoformer_triton_b200 as evo
    nq, nk = [300, 7, 129, 40, 260], [100, 0, 1, 40, 132]
    q, k, v = _qkv(sum(nq), sum(nk), H, Hk, D, dtype)
    d = _draw(q.shape, dtype, 5)
    blind = torch.zeros(sum(nq), dtype=torch.bool, device=DEV)
    for i, n, _, m in _spans(nq, nk):
        blind[i:i + max(0, n - m)] = True
    dirty = [torch.where(blind[:, None, None], bad, t) for t in (q, d)]
    leaves = [t.detach().requires_grad_() for t in (dirty[0], k, v)]
    out = evo.packed_attention(*leaves, torch.tensor(_sums(nq), device=DEV), torch.tensor(_sums(nk), device=DEV))
    grads = torch.autograd.grad(out, leaves, dirty[1])
    assert not out[blind].any() and not grads[0][blind].any()
    for name, g, w in zip(("o", "dq", "dk", "dv"), (out, *grads), oc.attention(q, k, v, _spans(nq, nk), True, d=d)):
        oc.check(name, g, w)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("H,Hk,D", [(2, 1, 64), (3, 1, 128), (2, 1, 20)])
@pytest.mark.parametrize("bad", ["nan", "inf", "overflow"])
def test_scores_that_are_not_finite_show(bad, H, Hk, D, dtype):
    """One key whose scores are NaN or plus infinity, at every place of eight and in a tile that no mask cuts: the rows that see it
    are not finite, whichever kernel and however the keys are cut up, nor are their gradients; the others are."""
    import evoformer_triton_b200 as evo
    if bad == "overflow" and dtype == HF:
        return  # (65 504 squared is a number)
    for nq, nk in ((400, 400), (300, 9000)):
        q, k, v = _qkv(nq, nk, H, Hk, D, dtype)
        q[..., 0] = q[..., 0].abs() + 0.5
        off, koff = torch.tensor([0, nq], device=DEV), torch.tensor([0, nk], device=DEV)
        for place in range(8):
            at = nk - nq + 40 + place
            k2 = k.clone()
            k2[at, :, 0] = {"nan": float("nan"), "inf": float("inf"), "overflow": 3e38}[bad]
            q2 = q * 20 if bad == "overflow" else q
            leaves = [t.detach().requires_grad_() for t in (q2, k2, v)]
            out = evo.packed_attention(*leaves, off, koff)
            (dq,) = torch.autograd.grad(out, leaves[:1], torch.ones_like(out))
            with torch.no_grad():
                infer = evo.packed_attention(q2, k2, v, off, koff)
                tokens = evo.packed_attention(q2[-3:], k2, v, torch.arange(4, device=DEV), torch.tensor([[0, nk], [at, at + 1], [0, at]], device=DEV))
            for t in (out, infer):
                assert torch.isfinite(t[:40 + place]).all() and not torch.isfinite(t[40 + place:]).any(), place
            assert not torch.isfinite(dq[40 + place:]).any(), place
            assert not torch.isfinite(tokens[:2]).any() and torch.isfinite(tokens[2]).all(), place


@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (F32, 64), (BF, 20)], ids=["bf16", "fp16", "fp32", "bf16 on CUDA cores"])
@pytest.mark.parametrize("bad", [[0, 200] * 40, [200, 0] * 300 + [200], [0, 200] * 3, [0, 150, 50, 200]], ids=["many", "descending", "three", "two"])
def test_offsets_that_overlap_leave_no_memory_as_it_was(bad, dtype, D):
    """Sequences that overlap are not right, but what comes back was written: blocks that held NaN before are handed out again.  The
    tensor-core kernels give zeros; on CUDA cores some rows may be those of one of the sequences."""
    import evoformer_triton_b200 as evo
    q, k, v = (t.requires_grad_() for t in _qkv(200, 200, 4, 2, D, dtype))
    off = torch.tensor(bad, device=DEV)
    d = _draw(q.shape, dtype, 5)
    for koff in (None, off, torch.tensor([0] * (len(bad) - 1) + [200], device=DEV)):
        used = [torch.full((n, 4, D), float("nan"), dtype=t, device=DEV) for n, t in ((200, dtype),) * 8 + ((400, F32),) * 4]
        del used
        out = evo.packed_attention(q, k, v, off, koff)
        grads = torch.autograd.grad(out, (q, k, v), d)
        for t in (out, *grads):
            assert torch.isfinite(t).all()
            assert not t.any() or D == 20 or dtype == F32
    _check(*_qkv(200, 200, 4, 2, D, dtype), [60, 140])


@pytest.mark.parametrize("D", [64, 128])
def test_thousands_of_tokens_between_rows_of_no_sequence(D):
    """More sequences than a launch of the kernel for few rows takes, and rows of none around them: every value, on each side of every
    border between launches."""
    g = torch.Generator().manual_seed(3)
    nk = torch.randint(0, 70, (5000,), generator=g).tolist()
    nq = [int(i % 7 != 3) for i in range(5000)]
    out = _check(*_qkv(sum(nq) + 9, sum(nk) + 9, 2, 1, D, BF), nq, nk, before=4, train=False)
    assert not out[:4].any() and not out[-5:].any()
    nq[4990], nk[4990] = 40, 3000  # one for the other kernel
    out = _check(*_qkv(sum(nq) + 9, sum(nk) + 9, 2, 1, D, BF), nq, nk, before=4, train=False)
    assert not out[:4].any() and not out[-5:].any()


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
def test_gradients_against_differences_of_the_fourth_order(causal):
    """Slopes along a direction from four points, h and 2 h to either side.  What is left out is h^4 / 30 of a fifth derivative: those of a
    softmax along scores that move by up to 3 are within 10^4 of the slope's terms, 10^-5 of them all told.  Results are off by
    some 2^-21 of the largest, independently; of the four, weighted 8, 8, 1 and 1 over 12 h, that is 95 times as much, four deviations."""
    import evoformer_triton_b200 as evo
    off, h = torch.tensor([0, 40, 97], device=DEV), 1e-2
    x = [t.requires_grad_() for t in _qkv(97, 97, 4, 2, 16, F32)]
    d = _draw((97, 4, 16), F32, 5)
    out = evo.packed_attention(*x, off, causal=causal)
    grads = torch.autograd.grad(out, x, d)
    for n, g in enumerate(grads):
        step = _draw(x[n].shape, F32, 6 + n)
        with torch.no_grad():
            at = lambda h: (evo.packed_attention(*(t + h * step if m == n else t for m, t in enumerate(x)), off, causal=causal).double() * d).sum()  # noqa: E731
            slope = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
        tol = 4 * 95 * 2.0 ** -21 * float(d.norm()) * float(out.detach().abs().max()) + 1e-5 * float((g.double() * step).abs().sum())
        assert abs(float(slope - (g.double() * step).sum())) < tol


@pytest.mark.parametrize("size", [2.0 ** -20, 1.0, 180.0, 16000.0])
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_gradients_of_the_largest_scores_gradient(D, size):
    """Two keys of equal scores and opposite values, and a gradient along them: dS is half of |dO| |V|, as large as it can be.  The sums are
    short, so dQ is dS times the keys' difference but for a rounding each of dS and dQ, and P and its sum: two steps."""
    import evoformer_triton_b200 as evo
    T = 130
    u = torch.ones(D, device=DEV)
    u[::2] = -1
    k = torch.zeros(2 * T, 1, D, device=DEV)
    k[::2, :, 0], k[1::2, :, 0] = 2.0 ** -12, -(2.0 ** -12)
    v = torch.stack([u, -u]).repeat(T, 1)[:, None] * 4
    q = torch.zeros(T, 1, D, device=DEV)  # (scores: zero)
    d = (u * size).expand(T, 1, D)
    leaves = [t.to(HF).requires_grad_() for t in (q, k, v)]
    off = torch.arange(T + 1, device=DEV)
    out = evo.packed_attention(*leaves, off, off * 2, causal=False, scale=1.0)
    dq, dk, dv = torch.autograd.grad(out, leaves, d.to(HF))
    ds = 0.25 * 2 * 4 * D * float(d.to(HF).abs()[0, 0, 0])  # P (1 - P) dO (V - V')
    want = torch.zeros(T, 1, D, device=DEV, dtype=torch.float64)
    want[..., 0] = ds * 2 * 2.0 ** -12
    oc.check("dq", dq, (want, 2 * torch.finfo(HF).eps * want + oc.rounding(HF, want)))
    assert not dk.any()
    oc.check("dv", dv, (d.to(HF).double().repeat_interleave(2, 0) / 2, oc.rounding(HF, d.to(HF).double().repeat_interleave(2, 0))))


@pytest.mark.parametrize("B", [2, 3, 5])
@pytest.mark.parametrize("power", [-18, 12])
def test_fp16_gradients_of_queries_with_keys_in_ranges(power, B):
    """The gradient of q alone, with keys that lie anywhere: rows of the cache that no range names have no say in the size of dS, those
    of every range have."""
    import evoformer_triton_b200 as evo
    nq, D = [700, 40, 129, 1, 300][:B], 64
    ranges = [(2500, 4000), (100, 400), (1000, 1130), (0, 50), (1500, 2300)][:B]
    q, k, v = _qkv(sum(nq), 4100, 4, 2, D, HF)
    used = torch.zeros(4100, dtype=torch.bool, device=DEV)
    for a, b in ranges:
        used[a:b] = True
    k[~used], v[~used] = 6e4, -6e4
    d = (_draw(q.shape, F32, 5) * 64).round() / 64 * 2.0 ** power
    x = q.clone().requires_grad_()
    out = evo.packed_attention(x, k, v, torch.tensor(_sums(nq), device=DEV), torch.tensor(ranges, device=DEV))
    (dq,) = torch.autograd.grad(out, x, d.to(HF))
    spans = [(i, n, a, b - a) for i, n, (a, b) in zip(_sums(nq), nq, ranges)]
    want = oc.attention(q, k, v, spans, True, d=d.to(HF))[1][0]
    for i, n, _, _ in spans:
        w = want[i:i + n]
        assert float((dq[i:i + n].double() - w).norm()) <= 0.65 * float(oc.rounding(HF, w).norm()) + torch.finfo(HF).eps / 2 * float(w.norm()), i
