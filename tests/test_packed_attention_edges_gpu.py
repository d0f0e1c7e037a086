"""GPU: attention over packed sequences where little or nothing is left: single rows, values that are not finite, gradients near the
ends of a type, offsets that overlap."""
import pytest
import torch

from oracle import sequences_oracle as oc
from test_packed_attention_gpu import BF, DEV, F32, HF, IDS, _check, _qkv, _spans, _sums

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
