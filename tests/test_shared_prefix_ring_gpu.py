"""Parts of a shared prefix that are longer than the ring of key and value tiles behind them: one part has all tiles of the prefix (the host's bound only picks the
parts), so every place of the ring, both score tiles and every barrier is used again and again, and the last, ragged tile lies in a place that was used before."""
import pytest
import torch

from . import hybrid_oracle as oracle
from .test_hybrid_kernels_gpu import DEV, _check_attention, _clean, _scratch, _shared_problem

pytestmark = pytest.mark.gpu

RING = [
    # heads, kv heads, head size, rows per sequence, prefix, keys behind it
    (4, 2, 64, 1, 900, [5, 70]),
    (28, 4, 64, 2, 1000, [40] * 10),                           # both slots of 128 rows
    (8, 2, 128, 1, 577, [1, 63, 64]),
    (32, 8, 128, 1, 3000, [17] * 40),
    (24, 4, 256, 1, 700, [9, 100, 1]),
    (12, 2, 256, 2, 677, [200] * 11),                          # a second tile of rows
]


@pytest.mark.parametrize("H,Hk,D,R,prefix,tails", RING)
@pytest.mark.parametrize("rising", [False, True])
def test_a_part_of_many_tiles_equals_attention_over_each_table(H, Hk, D, R, prefix, tails, rising):
    """``rising``: keys that grow along the prefix, so that the running maximum is raised again and again."""
    from llaminar_b200 import ops
    table, kv, q, _, total = _shared_problem(H, Hk, D, R, prefix, tails, False)
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    if rising:
        front = table[0, :-(-prefix // 64)].long()
        grow = (1 + 3 * torch.arange(front.numel()) / front.numel()).to(torch.bfloat16)
        kv[front, 0] = kv[front, 0] * grow[:, None, None, None]
    seen = torch.zeros(kv.shape[0], 64, dtype=torch.bool)
    for b in range(len(tails)):
        for k in range(total[b]):
            seen[int(table[b, k // 64]), k % 64] = True
    kv.permute(0, 3, 1, 2, 4)[~seen] = torch.tensor([float("nan"), float("inf")] * (D // 2), dtype=torch.bfloat16)
    want = [oracle.attention_rows(q[b * R:(b + 1) * R], kv, table[b], total[b], R, Hk, D ** -0.5) for b in range(len(tails))]
    outs = []
    for max_shared in (64, 64, prefix):
        out = torch.full_like(q, float("nan"), device=DEV)
        ops.attn_decode_shared(q.to(DEV), kv.to(DEV), out, table.to(DEV), it(total), it([prefix]), H, Hk, D, R, D ** -0.5, _scratch(), max_shared=max_shared)
        torch.cuda.synchronize()
        for b in range(len(tails)):
            _check_attention(out[b * R:(b + 1) * R], *want[b])
        outs.append(out)
    assert torch.equal(outs[0], outs[1])                       # nothing depends on the order in which parts are done
    _clean()
