"""CPU: what the operators before the attention refuse before they look at the device."""
import pytest
import torch
from torch.autograd import forward_ad


def test_forward_derivatives_are_refused():
    import evoformer_triton_b200 as evo
    z, W, w, table, base = torch.ones(1, 2, 2, 4), torch.ones(2, 4), torch.ones(4), torch.ones(65, 2), torch.ones(1, 1, 2, 2, 2)
    calls = ((evo.layer_norm, (z, w, w)), (evo.pair_bias_projection, (z, W, w, w)),
             (lambda t, p: evo.relative_position_bias(t, torch.arange(2), max_distance=32, pair_bias=p), (table, base)))
    for fn, args in calls:
        for i in range(len(args)):
            for grads in (False, True):
                with forward_ad.dual_level(), torch.set_grad_enabled(grads):
                    a = list(args)
                    a[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i]))
                    with pytest.raises(RuntimeError, match="forward mode"):
                        fn(*a)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            fn(*args)
