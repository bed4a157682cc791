"""The state of the delta rule behind a prompt: chunks on the tensor cores against the chunk-parallel form in 32 bits (models/gdn.py)."""
import pytest
import torch

from . import hybrid_oracle as oracle
from .test_hybrid_passes_gpu import D, EPS, N_K, N_V, _Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [64, 600])
def test_the_state_is_as_good_as_that_of_32_bit_products(rows):
    """Operands are two fp16 numbers, 22 bits, and the product of the two lower parts is left out: each of the three is at most four times the half step of a 32-bit
    number, 2^-24, and products of two such operands have both, so an error is at most 4 + 4 times that of 32-bit products, whose sums err alike."""
    from llaminar_b200.models import gdn
    call = _Call([rows], [9])
    call.run()
    out, _, rec = call.results()
    w, dw, C = call.w, call.dw, call.w["C"]
    conv, state = call.conv.cuda(), call.rec.cuda()
    x = call.inp.float()
    allow = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        gdn.gdn_block_rows(x[:, :C], x[:, w["z_off"]:w["z_off"] + N_V * D], x[:, w["ab_off"]:w["ab_off"] + N_V], x[:, w["ab_off"] + N_V:w["ab_off"] + 2 * N_V],
                           [(0, rows, 1, False)], conv, state, dw["conv_w"], dw["ssm_a"], dw["dt_bias"], dw["norm_w"], N_K, N_V, D, EPS)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = allow
    _, states = oracle.gdn_rows(call.buf, 0, rows, call.conv[1], call.rec[1], w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"], N_K, 0, EPS, w["z_off"], w["ab_off"])
    want = states[-1][1]
    off = lambda s: float((s.double().cpu() - want).norm() / want.norm())
    print(f"{rows} rows: kernel {off(rec[1]):.3g}, 32 bits {off(state[1]):.3g}")
    assert off(rec[1]) <= 8 * off(state[1])
