"""The scale of attention behind a shared prefix."""
import pytest
import torch

from .test_hybrid_kernels_gpu import DEV, _scratch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf")])
def test_a_scale_that_is_not_positive_and_finite_is_refused(scale):
    """The prefix finds the largest score before it is scaled, and what is masked is minus infinity there."""
    from llaminar_b200 import ops
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    H, Hk, D, B = 4, 2, 128, 2
    out = torch.full((B, H, D), 7.0, dtype=torch.bfloat16, device=DEV)
    for max_shared in (64, 0):
        with pytest.raises(RuntimeError, match="scale"):
            ops.attn_decode_shared(torch.zeros(B, H, D, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 2, Hk, 64, D, dtype=torch.bfloat16, device=DEV), out,
                                   it([[1, 2], [1, 3]]), it([70, 80]), it([64]), H, Hk, D, 1, scale, _scratch(), max_shared=max_shared)
    torch.cuda.synchronize()
    assert (out == 7).all()
