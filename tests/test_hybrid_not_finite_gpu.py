"""Rows of a prompt whose values are not finite.  The recurrence is causal: the rows in front of such a row, the other heads and the other sequences do not see it."""
import pytest
import torch

from . import hybrid_oracle as oracle
from .test_hybrid_kernels_gpu import DEV, EPS, _check_out, _check_state, _rows_problem

pytestmark = pytest.mark.gpu
D, N_K, N_V = 128, 2, 6


def _columns(kind, w, head):
    """A column of the input rows of value head ``head`` (q and k: of its key head)."""
    kh = head % N_K
    return {"q": kh * D + 5, "k": (N_K + kh) * D + 77, "v": (2 * N_K + head) * D + 31, "z": w["z_off"] + head * D + 9, "alpha": w["ab_off"] + head,
            "beta": w["ab_off"] + N_V + head}[kind]


@pytest.mark.parametrize("kind", ["q", "k", "v", "z", "alpha", "beta"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("taps", [4, 3])
def test_rows_in_front_and_other_heads_and_sequences_do_not_see_them(kind, value, taps):
    from llaminar_b200 import ops
    if kind in ("alpha", "beta") and value == float("inf"):
        pytest.skip("a finite decay and a finite share")
    lens, bad, head = [150, 90], 83, 3                             # the first sequence's second chunk, an odd row
    buf, width, w, conv, rec = _rows_problem(17, sum(lens), D, N_K, N_V, taps, 3, long_memory=True)
    buf[bad, _columns(kind, w, head)] = value
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in w.items()}
    conv_d, rec_d, out = conv.to(DEV), rec.to(DEV), torch.zeros(sum(lens), N_V * D, dtype=torch.bfloat16, device=DEV)
    positions = it([3 + t for n in lens for t in range(n)])
    ops.gdn_prefill(buf.to(DEV)[:, :width], w["C"], w["z_off"], w["ab_off"], dw["conv_w"], dw["ssm_a"], dw["dt_bias"], dw["norm_w"], conv_d, rec_d, positions,
                    it([0, 150, 240]), it([0, 1]), out, N_K, 0, EPS)
    torch.cuda.synchronize()
    clean = buf.clone()
    clean[bad, _columns(kind, w, head)] = 0
    orc = lambda first, n, s: oracle.gdn_rows(clean, first, n, conv[s], rec[s], w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"], N_K, 0, EPS, w["z_off"], w["ab_off"])
    (want, states), (want1, states1) = orc(0, 150, 0), orc(150, 90, 1)
    _check_out(out[150:], want1, D)
    _check_state(rec_d[1], states1[-1][1], D)
    _check_out(out[:bad], want[:bad], D)                           # in front: all heads
    reads = [h for h in range(N_V) if (h == head if kind in ("v", "z", "alpha", "beta") else h % N_K == head % N_K)]
    for h in range(N_V):
        cols = slice(h * D, (h + 1) * D)
        if h not in reads:                                         # another head: all rows and the state
            _check_out(out[bad:150, cols], want[bad:, cols], D)
            _check_state(rec_d[0, h], states[-1][1][h], D)
            continue
        if kind == "z":
            assert not torch.isfinite(out[bad, cols].float()).all()
        else:
            assert torch.isnan(out[bad, cols].float()).any()
        if kind in ("z", "q"):                                     # what does not enter the state ends with its row (the convolution's reach: three more)
            _check_out(out[bad + 4:150, cols], want[bad + 4:, cols], D)
            _check_state(rec_d[0, h], states[-1][1][h], D)
        else:
            assert torch.isnan(out[bad + 1:150, cols].float()).any(1).all() and torch.isnan(rec_d[0, h]).any()
