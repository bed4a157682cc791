"""Gates of the delta rule at the ends of their range: an infinite alpha forgets everything (decay 0), one of minus infinity nothing, an infinite beta writes all or
nothing.  Row by row, in chunks and for drafts; tolerances as in test_hybrid_kernels_gpu.py."""
import pytest
import torch

from . import hybrid_oracle as oracle
from .test_hybrid_kernels_gpu import DEV, EPS, _check_out, _check_state, _rows_problem

pytestmark = pytest.mark.gpu
INF = float("inf")


def _problem(T, d, n_k, n_v, slots, seed):
    buf, width, w, conv, rec = _rows_problem(seed, T, d, n_k, n_v, 4, slots, long_memory=True)
    ab = w["ab_off"]
    gates = [(ab, INF), (ab, 1e38), (ab, -INF), (ab, -1e38), (ab + n_v, INF), (ab + n_v, -INF), (ab, INF), (ab + 1, INF)]
    for i, (col, x) in enumerate(gates):                         # every seventh row, the first ones of a sequence among them; two neighbours
        for t in range(i * 7, T, 7 * len(gates)):
            buf[t, col] = x
    for t in range(17, T, 31):
        buf[t:t + 2, ab] = INF
    return buf, width, w, conv, rec


@pytest.mark.parametrize("d,n_k,n_v,lens", [(128, 2, 2, [9, 3]), (64, 1, 3, [100]), (128, 1, 2, [70, 129]), (128, 2, 4, [200])])
def test_prompts_with_gates_at_the_ends_of_their_range(d, n_k, n_v, lens):
    from llaminar_b200 import ops
    buf, width, w, conv, rec = _problem(sum(lens), d, n_k, n_v, len(lens) + 1, d + sum(lens))
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in w.items()}
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    positions = it([3 + t for n in lens for t in range(n)])
    conv_d, rec_d, out = conv.to(DEV), rec.to(DEV), torch.zeros(sum(lens), n_v * d, dtype=torch.bfloat16, device=DEV)
    ops.gdn_prefill(buf.to(DEV)[:, :width], w["C"], w["z_off"], w["ab_off"], dw["conv_w"], dw["ssm_a"], dw["dt_bias"], dw["norm_w"], conv_d, rec_d, positions, it(cu),
                    it(list(range(len(lens)))), out, n_k, 0, EPS)
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        want, states = oracle.gdn_rows(buf, cu[b], n, conv[b], rec[b], w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"], n_k, 0, EPS, w["z_off"], w["ab_off"])
        _check_out(out[cu[b]:cu[b + 1]], want, d)
        _check_state(rec_d[b], states[-1][1], d)


@pytest.mark.parametrize("d,n_k,n_v,B,R", [(128, 2, 2, 4, 3), (128, 1, 2, 2, 11), (64, 1, 2, 3, 5)])
def test_drafts_with_gates_at_the_ends_of_their_range(d, n_k, n_v, B, R):
    from llaminar_b200 import ops
    buf, width, w, conv, rec = _problem(B * R, d, n_k, n_v, B + 1, d + R)
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in w.items()}
    conv_d, rec_d, out = conv.to(DEV), rec.to(DEV), torch.zeros(B * R, n_v * d, dtype=torch.bfloat16, device=DEV)
    st = ops.gdn_verify(buf.to(DEV)[:, :width], w["C"], w["z_off"], w["ab_off"], dw["conv_w"], dw["ssm_a"], dw["dt_bias"], dw["norm_w"], conv_d, rec_d,
                        it(list(range(B))), out, n_k, 0, EPS)
    ops.gdn_commit(st, it([R] * B), conv_d, rec_d)
    torch.cuda.synchronize()
    for b in range(B):
        want, states = oracle.gdn_rows(buf, b * R, R, conv[b], rec[b], w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"], n_k, 0, EPS, w["z_off"], w["ab_off"])
        _check_out(out[b * R:(b + 1) * R], want, d)
        _check_state(rec_d[b], states[-1][1], d)
