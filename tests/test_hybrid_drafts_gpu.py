"""Drafted rows of the gated delta rule at other tap counts, head sizes and row counts than test_hybrid_kernels_gpu.py (whose tolerances hold here too): every row's
output, and the state after any number of accepted rows."""
import pytest
import torch

from . import hybrid_oracle as oracle
from .test_hybrid_kernels_gpu import DEV, EPS, _check_out, _check_state, _rows_problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,n_k,n_v,v_off,K,B,R", [(32, 2, 4, 0, 4, 2, 4), (32, 1, 3, 2, 2, 3, 3), (64, 1, 2, 0, 2, 3, 8), (64, 3, 5, 1, 4, 2, 4), (128, 2, 3, 1, 3, 2, 3),
                                                  (128, 2, 2, 0, 8, 1, 7), (128, 4, 2, 0, 4, 2, 5), (128, 1, 1, 0, 4, 1, 1), (128, 2, 4, 0, 4, 40, 2)])
@pytest.mark.parametrize("long_memory", [False, True])
def test_rows_and_states_of_drafts(d, n_k, n_v, v_off, K, B, R, long_memory):
    from llaminar_b200 import ops
    buf, width, w, conv, rec = _rows_problem(7 * d + R, B * R, d, n_k, n_v, K, B + 1, long_memory)
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in w.items()}
    order = list(range(B, 0, -1))
    conv_d, rec_d = conv.to(DEV), rec.to(DEV)
    out = torch.zeros(B * R, n_v * d, dtype=torch.bfloat16, device=DEV)
    st = ops.gdn_verify(buf.to(DEV)[:, :width], w["C"], w["z_off"], w["ab_off"], dw["conv_w"], dw["ssm_a"], dw["dt_bias"], dw["norm_w"], conv_d, rec_d, it(order), out, n_k,
                        v_off, EPS)
    torch.cuda.synchronize()
    assert torch.equal(conv_d.cpu(), conv) and torch.equal(rec_d.cpu(), rec)
    wants = [oracle.gdn_rows(buf, b * R, R, conv[order[b]], rec[order[b]], w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"], n_k, v_off, EPS, w["z_off"], w["ab_off"])
             for b in range(B)]
    for b in range(B):
        _check_out(out[b * R:(b + 1) * R], wants[b][0], d)
    for accepted in range(R + 1):
        conv_a, rec_a = conv.to(DEV), rec.to(DEV)
        ops.gdn_commit(st, it([accepted] * B), conv_a, rec_a)
        for b in range(min(B, 3)):
            s = order[b]
            if accepted == 0:
                assert torch.equal(conv_a[s].cpu(), conv[s]) and torch.equal(rec_a[s].cpu(), rec[s])
                continue
            want_conv, want_rec = wants[b][1][accepted - 1]
            assert torch.equal(conv_a[s].cpu(), want_conv.float())
            _check_state(rec_a[s], want_rec, d)
