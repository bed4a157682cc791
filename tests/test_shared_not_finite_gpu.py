"""Keys that are not finite among those that only the later drafted rows of a sequence see."""
import pytest
import torch

from . import hybrid_oracle as oracle
from .test_hybrid_kernels_gpu import DEV, _check_attention, _scratch, _shared_problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,H", [(64, 4), (128, 4), (256, 2)])
@pytest.mark.parametrize("drafted", [0, 1])
@pytest.mark.parametrize("max_shared", [128, 0])
def test_a_drafted_key_that_is_no_number_makes_the_rows_that_see_it_so(D, H, drafted, max_shared):
    from llaminar_b200 import ops
    Hk, R, prefix = 1, 3, 128
    table, kv, q, _, total = _shared_problem(H, Hk, D, R, prefix, [20, 64], False)
    key = total[0] - (R - 1) + drafted                             # row r sees keys < total - (R - 1 - r): rows 1 + drafted .. R - 1
    kv[int(table[0, key // 64]), 0, 0, key % 64] = float("nan")
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    out = torch.zeros_like(q, device=DEV)
    ops.attn_decode_shared(q.to(DEV), kv.to(DEV), out, table.to(DEV), it(total), it([prefix]), H, Hk, D, R, D ** -0.5, _scratch(), max_shared=max_shared)
    assert torch.isnan(out[1 + drafted:R]).all()
    clean = kv.clone()
    clean[int(table[0, key // 64]), 0, 0, key % 64] = 0
    want, size = oracle.attention_rows(q[:R], clean, table[0], total[0], R, Hk, D ** -0.5)
    _check_attention(out[:1 + drafted], want[:1 + drafted], size[:1 + drafted])
    _check_attention(out[R:], *oracle.attention_rows(q[R:], kv, table[1], total[1], R, Hk, D ** -0.5))
