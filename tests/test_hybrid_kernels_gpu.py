"""Kernels of the hybrid family's blocks against plain 64-bit implementations: the gated delta rule over prompts and drafted rows.

Tolerances.  Outputs are bf16: half a step, 2^-8 of the value, behind sums of d products in 32 bits, whose error is at most d 2^-24 of the
largest value; the gated norm divides by a root mean square, which is why the second part is taken relative to the largest output.  States are 32-bit sums: a
row rounds each value a few times and its correction is a sum of d products, (d + 8) 2^-24 of the state's norm; a row shrinks what came before, and the
roundings of many rows are independent, so that bound is used for any number of rows."""
import pytest
import torch

from . import hybrid_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6


def _rows_problem(seed, n_rows, d, n_k, n_v, K, slots, long_memory=False):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    C = (2 * n_k + n_v) * d
    z_off, ab_off = C, C + n_v * d
    width = ab_off + 2 * n_v
    buf = torch.zeros(n_rows, width + 7, dtype=torch.bfloat16)
    buf[:, :width] = (rnd(n_rows, width) * 1.5).to(torch.bfloat16)
    w = {"C": C, "z_off": z_off, "ab_off": ab_off, "conv_w": rnd(C, K) * 0.4, "ssm_a": -(torch.rand(n_v, generator=g) * 4 + 0.2) * (0.02 if long_memory else 1.0),
         "dt_bias": torch.rand(n_v, generator=g) * 2 - 1, "norm_w": torch.rand(d, generator=g) + 0.5}
    conv = rnd(slots, C, K - 1) * 0.5
    rec = rnd(slots, n_v, d, d) * 0.1
    return buf, width, w, conv, rec


def _check_out(got, want, d):
    got, want = got.double().cpu(), want
    bound = 2.0 ** -8 * want.abs() + 16 * d * 2.0 ** -24 * want.abs().max()
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() - bound).max())


def _check_state(got, want, d):
    got = got.double().cpu()
    assert (got - want).norm() <= (d + 8) * 2.0 ** -24 * want.norm() + 1e-30, float((got - want).norm() / want.norm())


PREFILL = [
    # d, n_k, n_v, v_off, K, rows per sequence, first positions
    (32, 2, 4, 0, 4, [1], [0]),
    (32, 2, 4, 2, 4, [3, 0, 70], [0, 5, 9]),
    (64, 3, 5, 1, 2, [9, 17], [4, 0]),
    (64, 2, 4, 0, 4, [130], [0]),
    (128, 1, 1, 0, 4, [1], [17]),
    (128, 2, 2, 1, 4, [2, 1, 3], [0, 1, 0]),
    (128, 2, 3, 0, 4, [63, 64, 65], [0, 64, 0]),
    (128, 4, 2, 3, 3, [37], [0]),
    (128, 2, 6, 0, 4, [0, 129, 5, 0], [3, 0, 8, 0]),
    (128, 1, 2, 0, 8, [200, 127], [0, 300]),
    (128, 1, 1, 0, 16, [70], [11]),
]


@pytest.mark.parametrize("d,n_k,n_v,v_off,K,lens,pos", PREFILL)
@pytest.mark.parametrize("long_memory", [False, True])
def test_gdn_prefill_follows_the_recurrence(d, n_k, n_v, v_off, K, lens, pos, long_memory):
    from llaminar_b200 import ops
    front, behind, slots_n = 2, 3, len(lens) + 2                # rows outside of all sequences, slots of nobody
    T = front + sum(lens) + behind
    buf, width, w, conv, rec = _rows_problem(d + sum(lens), T, d, n_k, n_v, K, slots_n, long_memory)
    buf[:front], buf[T - behind:] = float("nan"), float("nan")
    order = torch.randperm(slots_n, generator=torch.Generator().manual_seed(3)).tolist()[:len(lens)]
    cu = [front]
    for n in lens:
        cu.append(cu[-1] + n)
    positions = torch.full((T,), 7, dtype=torch.int32)
    for b, n in enumerate(lens):
        positions[cu[b]:cu[b + 1]] = torch.arange(pos[b], pos[b] + n, dtype=torch.int32)
        if pos[b] == 0 and n:
            conv[order[b]], rec[order[b]] = float("nan"), float("nan")      # what a fresh sequence's slot holds does not matter
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in w.items()}
    conv_d, rec_d = conv.to(DEV), rec.to(DEV)
    out = torch.full((T, n_v * d + 5), 3.0, dtype=torch.bfloat16, device=DEV)[:, :n_v * d]
    ops.gdn_prefill(buf.to(DEV)[:, :width], w["C"], w["z_off"], w["ab_off"], dw["conv_w"], dw["ssm_a"], dw["dt_bias"], dw["norm_w"], conv_d, rec_d,
                    positions.to(DEV), it(cu), it(order), out, n_k, v_off, EPS)
    torch.cuda.synchronize()
    assert (out[:front] == 3).all() and (out[T - behind:] == 3).all()
    for b, n in enumerate(lens):
        s = order[b]
        if n == 0:
            assert torch.equal(conv_d[s].cpu(), conv[s]) and torch.equal(rec_d[s].cpu(), rec[s])
            continue
        fresh = pos[b] == 0
        want, states = oracle.gdn_rows(buf, cu[b], n, None if fresh else conv[s], None if fresh else rec[s], w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"],
                                       n_k, v_off, EPS, w["z_off"], w["ab_off"])
        _check_out(out[cu[b]:cu[b + 1]], want, d)
        assert torch.equal(conv_d[s].double().cpu(), states[-1][0])
        _check_state(rec_d[s], states[-1][1], d)
    for s in set(range(slots_n)) - set(order):
        assert torch.equal(conv_d[s].cpu(), conv[s]) and torch.equal(rec_d[s].cpu(), rec[s])


@pytest.mark.parametrize("d,n_k,n_v,v_off,B,R", [(32, 2, 4, 0, 3, 1), (64, 2, 3, 1, 2, 5), (128, 2, 4, 0, 5, 3), (128, 4, 2, 2, 1, 8), (128, 1, 2, 0, 2, 19)])
def test_gdn_verify_leaves_the_state_and_commit_advances_it(d, n_k, n_v, v_off, B, R):
    from llaminar_b200 import ops
    buf, width, w, conv, rec = _rows_problem(d + R, B * R, d, n_k, n_v, 4, B + 1)
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in w.items()}
    order = list(range(B, 0, -1))
    conv_d, rec_d = conv.to(DEV), rec.to(DEV)
    out = torch.zeros(B * R, n_v * d, dtype=torch.bfloat16, device=DEV)
    inp = buf.to(DEV)[:, :width]
    st = ops.gdn_verify(inp, w["C"], w["z_off"], w["ab_off"], dw["conv_w"], dw["ssm_a"], dw["dt_bias"], dw["norm_w"], conv_d, rec_d, it(order), out, n_k, v_off, EPS)
    torch.cuda.synchronize()
    assert torch.equal(conv_d.cpu(), conv) and torch.equal(rec_d.cpu(), rec)
    inp.fill_(float("nan"))                                      # the rows are somebody else's by the time of the commit
    accepted = [b % (R + 1) for b in range(B)]
    accepted[-1] = R
    ops.gdn_commit(st, it(accepted), conv_d, rec_d)
    torch.cuda.synchronize()
    for b in range(B):
        s = order[b]
        want, states = oracle.gdn_rows(buf, b * R, R, conv[s], rec[s], w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"], n_k, v_off, EPS, w["z_off"], w["ab_off"])
        _check_out(out[b * R:(b + 1) * R], want, d)
        if accepted[b] == 0:
            assert torch.equal(conv_d[s].cpu(), conv[s]) and torch.equal(rec_d[s].cpu(), rec[s])
        else:
            assert torch.equal(conv_d[s].cpu(), states[accepted[b] - 1][0].float())
            _check_state(rec_d[s], states[accepted[b] - 1][1], d)
    assert torch.equal(rec_d[0].cpu(), rec[0])


def test_prompt_chunks_drafts_and_steps_of_one_sequence_follow_one_recurrence():
    """A prompt in two chunks, drafted rows of which two are accepted, then single steps: one long recurrence."""
    from llaminar_b200 import ops
    d, n_k, n_v = 128, 2, 4
    n = [70, 51, 3, 1, 1]
    buf, width, w, conv, rec = _rows_problem(11, sum(n), d, n_k, n_v, 4, 2)
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in w.items()}
    rows = torch.cat([buf[:123], buf[124:]])                     # the third draft is rejected: the recurrence never sees it
    want, states = oracle.gdn_rows(rows, 0, 125, None, None, w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"], n_k, 0, EPS, w["z_off"], w["ab_off"])
    conv_d, rec_d = conv.to(DEV), rec.to(DEV)
    inp = buf.to(DEV)[:, :width]
    args = lambda x: (x, w["C"], w["z_off"], w["ab_off"], dw["conv_w"], dw["ssm_a"], dw["dt_bias"], dw["norm_w"], conv_d, rec_d)
    got = []
    for a, b in ((0, 70), (70, 121)):
        out = torch.zeros(b - a, n_v * d, dtype=torch.bfloat16, device=DEV)
        ops.gdn_prefill(*args(inp[a:b]), torch.arange(a, b, dtype=torch.int32, device=DEV), it([0, b - a]), it([1]), out, n_k, 0, EPS)
        got.append(out)
    out = torch.zeros(3, n_v * d, dtype=torch.bfloat16, device=DEV)
    st = ops.gdn_verify(*args(inp[121:124]), it([1]), out, n_k, 0, EPS)
    ops.gdn_commit(st, it([2]), conv_d, rec_d)
    got.append(out[:2])
    y = torch.empty(1, w["C"], dtype=torch.float32, device=DEV)
    for r in (124, 125):
        out = torch.zeros(1, n_v * d, dtype=torch.bfloat16, device=DEV)
        ops.gdn_step(*args(inp[r:r + 1]), it([1]), y, out, n_k, 0, EPS)
        got.append(out)
    torch.cuda.synchronize()
    _check_out(torch.cat(got[:3]), want[:123], d)
    # the single-step kernels use the fast exponential, 2 ulp + 2^-21 of the exponent's size, on gates and decays: a few more 2^-20
    tail = torch.cat(got[3:]).double().cpu()
    assert ((tail - want[123:]).abs() <= 2.0 ** -8 * want[123:].abs() + 2.0 ** -14 * want.abs().max()).all()
    assert torch.equal(conv_d[1].double().cpu(), states[-1][0])


def test_gdn_calls_refuse_what_they_cannot_take():
    from llaminar_b200 import ops
    d, n_k, n_v, T = 128, 1, 1, 4
    buf, width, w, conv, rec = _rows_problem(1, T, d, n_k, n_v, 4, 2)
    dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in w.items()}
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    good = dict(inp=buf.to(DEV)[:, :width], C=w["C"], z_off=w["z_off"], ab_off=w["ab_off"], conv_w=dw["conv_w"], ssm_a=dw["ssm_a"], dt_bias=dw["dt_bias"],
                norm_w=dw["norm_w"], conv_state=conv.to(DEV), rec=rec.to(DEV), positions=torch.arange(T, dtype=torch.int32, device=DEV), cu=it([0, T]), slots=it([0]),
                out=torch.zeros(T, d, dtype=torch.bfloat16, device=DEV), n_k=1, v_head_offset=0, eps=EPS)
    ops.gdn_prefill(**good)
    bad = [dict(inp=good["inp"].float()), dict(inp=good["inp"].cpu()), dict(inp=good["inp"].t()), dict(C=w["C"] - 1), dict(z_off=width), dict(ab_off=-1), dict(conv_w=dw["conv_w"][:, :3]),
           dict(conv_w=dw["conv_w"].double()), dict(ssm_a=dw["ssm_a"].repeat(2)), dict(norm_w=dw["norm_w"][:64]), dict(conv_state=good["conv_state"][:1]), dict(rec=good["rec"].half()),
           dict(rec=torch.zeros(2, 1, 48, 48, device=DEV)), dict(positions=good["positions"][:3]), dict(positions=good["positions"].long()), dict(cu=it([0])), dict(slots=it([0, 1])),
           dict(slots=torch.tensor([0], dtype=torch.int32)), dict(out=good["out"][:3]), dict(out=good["out"].float()), dict(n_k=0), dict(n_k=2), dict(v_head_offset=-1)]
    for change in bad:
        with pytest.raises((RuntimeError, ValueError)):
            ops.gdn_prefill(**{**good, **change})
    ver = {k: v for k, v in good.items() if k not in ("positions", "cu")}
    st = ops.gdn_verify(**ver)
    for change in (dict(slots=it([0, 1, 0])), dict(slots=it([])), dict(inp=good["inp"].float())):
        with pytest.raises((RuntimeError, ValueError)):
            ops.gdn_verify(**{**ver, **change})
    with pytest.raises(RuntimeError):
        ops.gdn_commit(st, it([1, 1]), good["conv_state"], good["rec"])
    with pytest.raises(RuntimeError):
        ops.gdn_commit(st, torch.tensor([1]), good["conv_state"], good["rec"])
    with pytest.raises(RuntimeError):
        ops.gdn_commit(st, it([1]), good["conv_state"].double(), good["rec"])
    # nothing to do: no rows, no sequences
    ops.gdn_prefill(**{**good, "inp": good["inp"][:0], "out": good["out"][:0], "positions": good["positions"][:0], "cu": it([0, 0])})
    ops.gdn_prefill(**{**good, "cu": it([0]), "slots": it([])})
    torch.cuda.synchronize()
