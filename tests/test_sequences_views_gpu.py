"""GPU: rotary positions and packed attention of views that have yet to be negated."""
import pytest
import torch

import evoformer_triton_b200 as evo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _imaginary(x):
    """-x as the imaginary part of a conjugate: a view of +x."""
    y = torch.complex(torch.zeros_like(x), x).conj().imag
    assert y.is_neg()
    return y


def _draw(*shape, seed=1):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def test_rotary_of_negated_views():
    q, k, f = _draw(9, 4, 32), _draw(9, 2, 32, seed=2), evo.rotary_frequencies(32, device=DEV).float()
    pos = torch.arange(9, device=DEV)
    for freq in (f, _imaginary(-f)):
        got = evo.rotary_embedding(_imaginary(q), _imaginary(k), pos, freq)
        for a, b in zip(got, evo.rotary_embedding(-q, -k, pos, f)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("D", [1, 32])
def test_packed_attention_of_negated_views(D):
    """(With one value a head no axis has to be made dense, which would negate it.)"""
    q, k, v, off = _draw(90, 4, D), _draw(90, 2, D, seed=2), _draw(90, 2, D, seed=3), torch.tensor([0, 40, 90], device=DEV)
    assert torch.equal(evo.packed_attention(_imaginary(q), _imaginary(k), _imaginary(v), off), evo.packed_attention(-q, -k, -v, off))
    a, b = ([t.clone().requires_grad_() for t in (q, k, v)] for _ in range(2))
    got = torch.autograd.grad(evo.packed_attention(*(_imaginary(t) for t in a), off).sum(), a)
    want = torch.autograd.grad(evo.packed_attention(*(-t for t in b), off).sum(), b)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
