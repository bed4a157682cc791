"""The persistent kernels of the gated delta rule with more (sequence, value head) items than CTAs: a CTA goes from item to item, the next state, rows and gates on
their way, past sequences without rows and fresh ones.  Tolerances as in test_hybrid_kernels_gpu.py; every item's arithmetic is its own, so a call of many sequences
has the bits of the calls of each alone."""
import pytest
import torch

from . import hybrid_oracle as oracle
from .test_hybrid_kernels_gpu import DEV, EPS, _check_out, _check_state, _rows_problem

pytestmark = pytest.mark.gpu


def _args(w, dw, conv_d, rec_d):
    return (w["C"], w["z_off"], w["ab_off"], dw["conv_w"], dw["ssm_a"], dw["dt_bias"], dw["norm_w"], conv_d, rec_d)


# items: 512 and 528 on 148 CTAs; 1280 on 296; 2048 on 592
@pytest.mark.parametrize("d,n_k,n_v,K,B", [(128, 2, 8, 4, 64), (128, 2, 8, 3, 66), (64, 2, 16, 4, 80), (32, 4, 16, 4, 128)])
def test_rows_one_by_one_of_many_sequences(d, n_k, n_v, K, B):
    from llaminar_b200 import ops
    lens = [(5 * b + b // 7) % 7 for b in range(B)]                # 0 .. 6 rows, empty ones between
    lens[0] = 0
    lens[B // 2:B // 2 + 3] = [0, 0, 0]
    T = sum(lens)
    assert T < ops.hybrid.GDN_CHUNK_MIN_ROWS[0] + ops.hybrid.GDN_CHUNK_MIN_ROWS[1] * B and n_v * B > 3 * 148
    buf, width, w, conv, rec = _rows_problem(d + B, T, d, n_k, n_v, K, B + 1)
    cu, positions, pos = [0], torch.zeros(T, dtype=torch.int32), [0 if b % 3 == 0 else 11 + b for b in range(B)]
    for b, n in enumerate(lens):
        cu.append(cu[-1] + n)
        positions[cu[b]:cu[b + 1]] = torch.arange(pos[b], pos[b] + n, dtype=torch.int32)
    order = torch.randperm(B + 1, generator=torch.Generator().manual_seed(3)).tolist()[:B]
    for b in range(B):
        if pos[b] == 0 and lens[b]:
            conv[order[b]], rec[order[b]] = float("nan"), float("nan")
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in w.items()}
    inp, conv_d, rec_d = buf.to(DEV)[:, :width], conv.to(DEV), rec.to(DEV)
    out = torch.full((T, n_v * d), 3.0, dtype=torch.bfloat16, device=DEV)
    ops.gdn_prefill(inp, *_args(w, dw, conv_d, rec_d), positions.to(DEV), it(cu), it(order), out, n_k, 0, EPS)
    torch.cuda.synchronize()
    conv_1, rec_1 = conv.to(DEV), rec.to(DEV)
    out_1 = torch.full_like(out, 3.0)
    for b in range(B):                                            # one sequence a call: a CTA has one item
        if lens[b]:
            r = slice(cu[b], cu[b + 1])
            ops.gdn_prefill(inp[r], *_args(w, dw, conv_1, rec_1), positions[r].to(DEV), it([0, lens[b]]), it([order[b]]), out_1[r], n_k, 0, EPS)
    torch.cuda.synchronize()
    same = lambda a, b: torch.equal(a.view(torch.int16 if a.dtype == torch.bfloat16 else torch.int32), b.view(torch.int16 if b.dtype == torch.bfloat16 else torch.int32))
    assert same(out, out_1) and same(conv_d, conv_1) and same(rec_d, rec_1)
    for b in (1, 2, 3, B // 2 + 3, B - 2, B - 1):
        if lens[b] == 0:
            assert same(rec_d[order[b]].cpu(), rec[order[b]])
            continue
        s, fresh = order[b], pos[b] == 0
        want, states = oracle.gdn_rows(buf, cu[b], lens[b], None if fresh else conv[s], None if fresh else rec[s], w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"],
                                       n_k, 0, EPS, w["z_off"], w["ab_off"])
        _check_out(out[cu[b]:cu[b + 1]], want, d)
        assert torch.equal(conv_d[s].double().cpu(), states[-1][0])
        _check_state(rec_d[s], states[-1][1], d)


# items: 544 on 148 CTAs, 9 rows (row by row); 960 on 148; 1280 on 296; 2560 on 592
@pytest.mark.parametrize("d,n_k,n_v,K,B,R", [(128, 2, 8, 4, 68, 9), (128, 4, 16, 4, 60, 3), (128, 2, 8, 3, 60, 6), (64, 2, 16, 4, 80, 4), (32, 4, 16, 4, 160, 2)])
def test_drafts_of_many_sequences(d, n_k, n_v, K, B, R):
    from llaminar_b200 import ops
    buf, width, w, conv, rec = _rows_problem(d + R, B * R, d, n_k, n_v, K, B + 1)
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in w.items()}
    inp, conv_d, rec_d, order = buf.to(DEV)[:, :width], conv.to(DEV), rec.to(DEV), list(range(B, 0, -1))
    args = _args(w, dw, conv_d, rec_d)
    out, out_1 = (torch.zeros(B * R, n_v * d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    st = ops.gdn_verify(inp, *args, it(order), out, n_k, 0, EPS)
    for b in range(B):
        r = slice(b * R, (b + 1) * R)
        one = ops.gdn_verify(inp[r], *args, it([order[b]]), out_1[r], n_k, 0, EPS)
        for x, y in ((one.decay, st.decay), (one.key, st.key), (one.correction, st.correction), (one.inputs, st.inputs)):
            assert torch.equal(x[0], y[b]), b
    assert torch.equal(out, out_1) and torch.equal(rec_d.cpu(), rec)
    accepted = [b % (R + 1) for b in range(B)]
    ops.gdn_commit(st, it(accepted), conv_d, rec_d)
    torch.cuda.synchronize()
    for b in (0, 1, B // 2, B - 2, B - 1):
        s = order[b]
        want, states = oracle.gdn_rows(buf, b * R, R, conv[s], rec[s], w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"], n_k, 0, EPS, w["z_off"], w["ab_off"])
        _check_out(out[b * R:(b + 1) * R], want, d)
        if accepted[b]:
            assert torch.equal(conv_d[s].cpu(), states[accepted[b] - 1][0].float())
            _check_state(rec_d[s], states[accepted[b] - 1][1], d)
        else:
            assert torch.equal(rec_d[s].cpu(), rec[s])
