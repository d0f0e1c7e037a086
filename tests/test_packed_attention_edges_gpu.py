"""GPU: attention over packed sequences where little or nothing is left: single rows, values that are not finite, gradients near the
ends of a type, offsets that overlap."""
import pytest
import torch

from oracle import sequences_oracle as oc
from test_packed_attention_gpu import BF, DEV, F32, HF, IDS, _check, _qkv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=IDS.get)
@pytest.mark.parametrize("D", [1, 8, 20, 32, 64, 128, 256])
@pytest.mark.parametrize("T,H", [(1, 1), (1, 2), (3, 1), (1, 5), (7, 1), (9, 3)])
def test_gradients_of_a_few_rows(T, H, D, dtype):
    """Fewer rows of dO * O than a warp adds up at once, and numbers of them that it does not divide."""
    _check(*_qkv(T, T, H, 1, D, dtype), [T])
