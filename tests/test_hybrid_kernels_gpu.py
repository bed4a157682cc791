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


# -- rotation of a part of every head with the append ---------------------------------------------------------------------

ROPE = [
    # heads, kv heads, head size, pairs, gated, interleaved, norms, tokens per sequence, first positions
    (6, 2, 64, 8, True, False, True, [1], [0]),
    (4, 1, 64, 32, False, True, False, [5, 70], [0, 63]),
    (8, 8, 128, 64, False, False, True, [3, 1, 130], [200000, 7, 100]),
    (7, 1, 128, 16, True, True, True, [64], [64]),
    (24, 4, 256, 32, True, False, True, [1] * 9, [131071, 0, 1, 62, 63, 64, 65, 999, 262143]),
    (3, 1, 256, 128, False, False, True, [2], [50]),
    (2, 2, 256, 5, True, False, True, [9], [120]),             # halves that end inside a lane's values
    (5, 1, 128, 3, False, False, False, [3], [61]),
    (2, 1, 64, 0, False, False, True, [4], [10]),              # nothing turns
    (16, 2, 256, 32, True, False, True, [2500], [30]),         # a warp per token
]


@pytest.mark.parametrize("H,Hk,D,n,gated,interleaved,norms,lens,first", ROPE)
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("odd_rows", [False, True])
def test_rope_part_kv_follows_the_definition(H, Hk, D, n, gated, interleaved, norms, lens, first, q8, odd_rows):
    """Queries and bf16 entries: half a step, 2^-8 of the value, behind sums of D squares and a few products in 32 bits (an angle is 2^-22 off at most).  8-bit
    entries: half a step of the scale, which is the largest of 32 values / 127 rounded up by up to 2^-7."""
    from llaminar_b200 import ops
    if sum(lens) > 300 and odd_rows:
        pytest.skip("one form of the long case")
    g = torch.Generator().manual_seed(H * D + n)
    T, B = sum(lens), len(lens)
    width = (H * (2 if gated else 1) + 2 * Hk) * D
    buf = torch.randn(T, width + (1 if odd_rows else 0), generator=g).to(torch.bfloat16)
    q_norm, k_norm = (torch.rand(D, generator=g) + 0.5, torch.rand(D, generator=g) + 0.5) if norms else (None, None)
    freqs, magnitude = 1e6 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)), 1.25
    pos = [f + t for f, k in zip(first, lens) for t in range(k)]
    sid = [b for b, k in enumerate(lens) for _ in range(k)]
    used = sorted({(b, p // 64) for b, p in zip(sid, pos)})
    table = torch.zeros(B, max(p for _, p in used) + 1, dtype=torch.int32)
    ids = (torch.randperm(len(used), generator=g) + 1).tolist()
    for (b, p), i in zip(used, ids):
        table[b, p] = i
    n_pages = len(used) + 1
    kv = torch.zeros(n_pages, 2, Hk, 64, D, dtype=torch.bfloat16, device=DEV) if not q8 else torch.zeros(n_pages, 2 * Hk * 64 * D * 17 // 16, dtype=torch.uint8, device=DEV)
    q_out = torch.zeros(T, H, D, dtype=torch.bfloat16, device=DEV)
    dev = lambda x: None if x is None else x.to(DEV)
    ops.rope_part_kv(buf.to(DEV)[:, :width], q_out, kv, dev(q_norm), dev(k_norm), freqs.to(DEV), magnitude, torch.tensor(pos, dtype=torch.int32, device=DEV),
                     torch.tensor(sid, dtype=torch.int32, device=DEV), table.to(DEV), H, Hk, D, EPS, gated=gated, interleaved=interleaved)
    torch.cuda.synchronize()
    if T > 300:                                                  # the oracle goes pair by pair: the first, the last and some between
        some = [0, 1, 77, 1300, T - 1]
    else:
        some = list(range(T))
    q, k, v = oracle.rope_part(buf[some][:, :width], H, Hk, D, q_norm, k_norm, freqs, magnitude, [pos[t] for t in some], EPS, gated, interleaved)
    close = lambda got, want: ((got.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 64 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True) + 1e-30).all()
    assert close(q_out[some], q)
    page = torch.tensor([int(table[sid[t], pos[t] // 64]) for t in some])
    off = torch.tensor([pos[t] % 64 for t in some])
    if not q8:
        assert close(kv[page.to(DEV), 0, :, off.to(DEV)], k) and close(kv[page.to(DEV), 1, :, off.to(DEV)], v)
        mask = torch.zeros(n_pages, 64, dtype=torch.bool)
        for t in range(T):
            mask[int(table[sid[t], pos[t] // 64]), pos[t] % 64] = True
        assert (kv.cpu().permute(0, 3, 1, 2, 4)[~mask] == 0).all()       # nothing else was written
    else:
        raw = kv.cpu()
        data = raw[:, :2 * Hk * 64 * D].contiguous().view(torch.int8).view(n_pages, 2, Hk, 64, D)[page, :, :, off].double()
        sc = raw[:, 2 * Hk * 64 * D:].contiguous().view(torch.float16).view(n_pages, 2, Hk, 64, D // 32)[page, :, :, off].double()
        for i, want in enumerate((k, v)):
            blocks = want.unflatten(-1, (-1, 32))
            top = blocks.abs().amax(-1) / 127
            assert (sc[:, i] >= top * (1 - 2.0 ** -11) - 2.0 ** -24).all() and (sc[:, i] <= top * (1 + 2.0 ** -6) + 2.0 ** -24).all()
            err = (data[:, i].unflatten(-1, (-1, 32)) * sc[:, i, ..., None] - blocks).abs()
            assert (err <= sc[:, i, ..., None] * (0.5 + 2.0 ** -10)).all()


def test_rope_part_kv_writes_what_rope_kv_writes_for_whole_heads():
    """Both pages and queries of whole, plain rotations agree with the operator beside it to a step of the type (its angles are 32-bit)."""
    from llaminar_b200 import ops
    H, Hk, D, T = 8, 2, 128, 100
    g = torch.Generator(device=DEV).manual_seed(5)
    qkv = torch.randn(T, (H + 2 * Hk) * D, device=DEV, generator=g).to(torch.bfloat16)
    norm = torch.rand(D, device=DEV, generator=g) + 0.5
    pos, sid = torch.arange(T, dtype=torch.int32, device=DEV), torch.zeros(T, dtype=torch.int32, device=DEV)
    table = torch.tensor([[2, 1]], dtype=torch.int32, device=DEV)
    got = []
    for kv in (torch.zeros(3, 2, Hk, 64, D, dtype=torch.bfloat16, device=DEV), torch.zeros(3, 2, Hk, 64, D, dtype=torch.bfloat16, device=DEV)):
        q = torch.zeros(T, H, D, dtype=torch.bfloat16, device=DEV)
        if not got:
            ops.rope_kv(qkv, q, kv, norm, norm, pos, sid, table, H, Hk, D, 1e6, EPS)
        else:
            ops.rope_part_kv(qkv, q, kv, norm, norm, 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D), 1.0, pos, sid, table, H, Hk, D, EPS)
        got.append((q.float(), kv.float()))
    for a, b in zip(*got):
        assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 2.0 ** -12).all()


def test_rope_part_kv_refuses_what_it_cannot_take():
    from llaminar_b200 import ops
    H, Hk, D, T = 2, 1, 64, 3
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    good = dict(rows=torch.zeros(T, 4 * D, dtype=torch.bfloat16, device=DEV), q_out=torch.zeros(T, H, D, dtype=torch.bfloat16, device=DEV),
                kv=torch.zeros(2, 2, Hk, 64, D, dtype=torch.bfloat16, device=DEV), q_norm=torch.ones(D, device=DEV), k_norm=None,
                freqs=torch.ones(8, dtype=torch.float64, device=DEV), magnitude=1.0, positions=it([0, 1, 2]), seq_ids=it([0, 0, 0]), block_table=it([[1]]),
                n_heads=H, n_kv_heads=Hk, head_dim=D, eps=EPS)
    ops.rope_part_kv(**good)
    for change in (dict(rows=good["rows"].float()), dict(rows=good["rows"][:, :-1]), dict(rows=good["rows"].cpu()), dict(gated=True), dict(q_out=good["q_out"][:2]),
                   dict(q_out=good["q_out"].transpose(0, 1)), dict(kv=good["kv"].half()), dict(kv=good["kv"][:, :, :, :32]), dict(kv=torch.zeros(2, 100, dtype=torch.uint8, device=DEV)),
                   dict(q_norm=torch.ones(D - 1, device=DEV)), dict(k_norm=torch.ones(D, device=DEV, dtype=torch.float64)), dict(freqs=good["freqs"].float()),
                   dict(freqs=torch.ones(33, dtype=torch.float64, device=DEV)), dict(positions=it([0, 1])), dict(seq_ids=good["seq_ids"].long()), dict(block_table=it([1])),
                   dict(n_heads=0), dict(head_dim=48), dict(n_kv_heads=2)):
        with pytest.raises((RuntimeError, TypeError)):
            ops.rope_part_kv(**{**good, **change})
    ops.rope_part_kv(**{**good, "rows": good["rows"][:0], "q_out": good["q_out"][:0], "positions": it([]), "seq_ids": it([])})
    torch.cuda.synchronize()


# -- attention behind a shared prefix -------------------------------------------------------------------------------------

SHARED = [
    # heads, kv heads, head size, rows per sequence, prefix, keys behind it (or, negative, a sequence of that many keys that does not share)
    (4, 2, 64, 1, 64, [1]),
    (6, 1, 64, 2, 128, [2, 70, 64]),
    (8, 2, 128, 1, 500, [1, 63, 64, 65, 300]),                 # a prefix that ends inside a page
    (16, 1, 128, 1, 130, [5, -40, 7, 0]),                      # one shorter than the prefix, one of the prefix alone
    (28, 4, 128, 2, 1000, [30] * 20),                          # more than a tile of rows
    (2, 2, 128, 16, 200, [16, 40]),
    (24, 4, 256, 1, 700, [9, 100, 1]),
    (6, 1, 256, 2, 65, [3, -1, 66, 2]),                        # a sequence of one key and two rows
    (16, 2, 256, 1, 1, [1, 200]),
    (8, 8, 64, 1, 0, [10, 130]),                               # nothing is shared
    (32, 8, 128, 1, 3000, [17] * 40),
    (16, 4, 64, 1, 300, [2000, 3]),                            # a long tail
    (12, 2, 256, 2, 640, [200] * 30),
]


def _shared_problem(H, Hk, D, R, prefix, tails, gated):
    """The prefix's pages, the last one whole, stand in front of the tables of the sequences that share it; what a sequence has behind the prefix in a page
    where the prefix ends is then everybody's."""
    g = torch.Generator().manual_seed(H * D + prefix)
    B, pre = len(tails), -(-prefix // 64)
    total = [prefix + n if n >= 0 else -n for n in tails]
    pages = [-(-n // 64) for n in total]
    table = torch.zeros(B, max(pages + [pre]) + 1, dtype=torch.int32)
    ids = iter((torch.randperm(pre + sum(pages) + 1, generator=g) + 1).tolist())
    front = [next(ids) for _ in range(pre)]
    for b in range(B):
        mine = (front if tails[b] >= 0 else []) + [next(ids) for _ in range(pages[b])]
        table[b, :pages[b]] = torch.tensor(mine[:pages[b]], dtype=torch.int32)
    kv = torch.randn(pre + sum(pages) + 2, 2, Hk, 64, D, generator=g).to(torch.bfloat16)
    q = torch.randn(B * R, H, D, generator=g).to(torch.bfloat16)
    rows = torch.randn(B * R, H, 2, D, generator=g).to(torch.bfloat16) if gated else None
    return table, kv, q, rows, total


def _check_attention(got, want, size):
    """Probabilities enter the second product as bf16: each is off by half a step at most, 2^-8 of it, so the sum by 2^-8 sum p |v|; the result is rounded to bf16
    once more.  Scores, sums and exponentials are 32-bit: less than 2^-12 of sum p |v|."""
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * size + 1e-30
    err = (got.double().cpu() - want).abs()
    assert (err <= bound).all(), float((err - bound).max())


def _scratch():
    from llaminar_b200 import ops
    return ops.scratch_for(torch.device(DEV, torch.cuda.current_device()))


def _clean():
    assert int(_scratch().status[0]) == 0 and int(_scratch().attn_tickets.abs().sum()) == 0


@pytest.mark.parametrize("H,Hk,D,R,prefix,tails", SHARED)
@pytest.mark.parametrize("gated", [False, True])
def test_attn_decode_shared_equals_attention_over_each_table(H, Hk, D, R, prefix, tails, gated):
    from llaminar_b200 import ops
    table, kv, q, rows, total = _shared_problem(H, Hk, D, R, prefix, tails, gated)
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    # what no row sees: pages of nobody, and the keys behind each sequence
    seen = torch.zeros(kv.shape[0], 64, dtype=torch.bool)
    for b in range(len(tails)):
        for k in range(total[b]):
            seen[int(table[b, k // 64]), k % 64] = True
    if not any(t >= 0 and total[b] > 0 for b, t in enumerate(tails)):
        seen[table[0, :-(-prefix // 64)].long()] = True
    kv.permute(0, 3, 1, 2, 4)[~seen] = torch.tensor([float("nan"), float("inf")] * (D // 2), dtype=torch.bfloat16)
    scale, out = D ** -0.5, torch.empty_like(q, device=DEV)
    gate = rows.to(DEV)[:, :, 1] if gated else None
    want = [oracle.attention_rows(q[b * R:(b + 1) * R], kv, table[b], total[b], R, Hk, scale, rows[b * R:(b + 1) * R, :, 1] if gated else None) for b in range(len(tails))]
    for max_shared, max_tail in ((prefix, 0), (prefix, max(64, *tails)), (0, 0)):
        out.fill_(float("nan"))
        ops.attn_decode_shared(q.to(DEV), kv.to(DEV), out, table.to(DEV), it(total), it([prefix]), H, Hk, D, R, scale, _scratch(), gate=gate,
                               max_shared=max_shared, max_tail=max_tail)
        torch.cuda.synchronize()
        for b in range(len(tails)):
            _check_attention(out[b * R:(b + 1) * R], *want[b])
            if total[b] == 0:
                assert (out[b * R:(b + 1) * R] == 0).all()
    _clean()


def test_a_drafted_key_that_is_not_finite_reaches_the_rows_that_see_it_alone():
    from llaminar_b200 import ops
    H, Hk, D, R, prefix = 4, 1, 128, 3, 128
    table, kv, q, _, total = _shared_problem(H, Hk, D, R, prefix, [20, 64], False)
    kv[int(table[0, (total[0] - 1) // 64]), 1, 0, (total[0] - 1) % 64] = float("nan")        # the value of the first sequence's last key
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q, device=DEV)
    ops.attn_decode_shared(q.to(DEV), kv.to(DEV), out, table.to(DEV), it(total), it([prefix]), H, Hk, D, R, D ** -0.5, _scratch(), max_shared=prefix)
    assert torch.isnan(out[2]).all() and torch.isfinite(out[[0, 1, 3, 4, 5]].float()).all()
    want = oracle.attention_rows(q[3:], kv, table[1], total[1], R, Hk, D ** -0.5)
    _check_attention(out[3:], *want)


@pytest.mark.parametrize("D,gated", [(128, False), (256, True)])
def test_attn_decode_shared_is_captured_and_follows_lengths_on_the_device(D, gated):
    """One captured call: the prefix shrinks to nothing, sequences grow and end, the row that the prefix is read from stays."""
    from llaminar_b200 import ops
    H, Hk, R, prefix, tails = 8, 2, 1, 256, [40, 100, 7]
    table, kv, q, rows, total = _shared_problem(H, Hk, D, R, prefix, tails, gated)
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    lens, shared, out, qd, kvd, td = it(total), it([prefix]), torch.empty_like(q, device=DEV), q.to(DEV), kv.to(DEV), table.to(DEV)
    gate = rows.to(DEV)[:, :, 1] if gated else None
    call = lambda: ops.attn_decode_shared(qd, kvd, out, td, lens, shared, H, Hk, D, R, D ** -0.5, _scratch(), gate=gate, max_shared=prefix, max_tail=128, prefix_row=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for n, now in ((prefix, total), (128, total), (0, total), (prefix, [total[0] - 5, total[1], 0]), (prefix, [3, total[1], total[2]])):
        shared.copy_(it([n]))
        lens.copy_(it(now))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for b in range(3):
            _check_attention(out[b:b + 1], *oracle.attention_rows(q[b:b + 1], kv, table[b], now[b], R, Hk, D ** -0.5, rows[b:b + 1, :, 1] if gated else None))
    _clean()


def test_rows_are_appended_and_read_behind_a_shared_prefix():
    """A softmax block of a decode step as it is used: [query | gate] rows, norm, rotation of a quarter of each head and append, attention, gate."""
    from llaminar_b200 import ops
    H, Hk, D, prefix, tails = 6, 2, 256, 192, [1, 30, 65, 64]
    table, kv, _, _, total = _shared_problem(H, Hk, D, 1, prefix, tails, False)
    B = len(tails)
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(B, (2 * H + 2 * Hk) * D, generator=g).to(torch.bfloat16)
    gain, freqs = torch.rand(D, generator=g) + 0.5, 1e6 ** (-torch.arange(32, dtype=torch.float64) / 32)
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    pos = [n - 1 for n in total]
    kvd, q_out, rd, td = kv.to(DEV), torch.empty(B, H, D, dtype=torch.bfloat16, device=DEV), rows.to(DEV), table.to(DEV)
    ops.rope_part_kv(rd, q_out, kvd, gain.to(DEV), gain.to(DEV), freqs.to(DEV), 1.0, it(pos), it(list(range(B))), td, H, Hk, D, EPS, gated=True)
    out = torch.empty_like(q_out)
    gate = rd[:, :2 * H * D].view(B, H, 2, D)[:, :, 1]
    ops.attn_decode_shared(q_out, kvd, out, td, it(total), it([prefix]), H, Hk, D, 1, D ** -0.5, _scratch(), gate=gate, max_shared=prefix)
    torch.cuda.synchronize()
    q, k, v = oracle.rope_part(rows, H, Hk, D, gain, gain, freqs, 1.0, pos, EPS, True, False)
    for b in range(B):
        page, off = int(table[b, pos[b] // 64]), pos[b] % 64
        kv[page, 0, :, off], kv[page, 1, :, off] = k[b].to(torch.bfloat16), v[b].to(torch.bfloat16)
        want, size = oracle.attention_rows(q_out[b:b + 1].cpu(), kv, table[b], total[b], 1, Hk, D ** -0.5, gate[b:b + 1].cpu())
        # the new key may round the other way than the oracle's, a step of 2^-7 of it, which moves its score by less than 2^-7 |q||k| / 16 and its share by that much
        slack = 2.0 ** -7 * size * float((q[b].norm(dim=-1).max() * k[b].norm(dim=-1).max()) / 16) / total[b] ** 0.5
        err = (out[b].double().cpu() - want[0]).abs()
        assert (err <= 2.0 ** -8 * want[0].abs() + (2.0 ** -8 + 2.0 ** -12) * size[0] + slack[0]).all()


def test_attn_decode_shared_refuses_what_it_cannot_take():
    from llaminar_b200 import ops
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    H, Hk, D, B = 4, 2, 128, 2
    good = dict(q=torch.zeros(B, H, D, dtype=torch.bfloat16, device=DEV), kv=torch.zeros(4, 2, Hk, 64, D, dtype=torch.bfloat16, device=DEV),
                out=torch.zeros(B, H, D, dtype=torch.bfloat16, device=DEV), block_table=it([[1, 2], [1, 3]]), seq_lens=it([70, 80]), shared_len=it([64]), n_heads=H,
                n_kv_heads=Hk, head_dim=D, rows_per_seq=1, scale=0.1, scratch=_scratch(), max_shared=64)
    ops.attn_decode_shared(**good)
    for change in (dict(q=good["q"].float()), dict(q=good["q"][:1]), dict(q=good["q"].cpu()), dict(kv=good["kv"].half()), dict(kv=good["kv"][:, :1]),
                   dict(kv=torch.zeros(4, 2 * Hk * 64 * D * 17 // 16, dtype=torch.uint8, device=DEV)), dict(out=good["out"].float()), dict(out=good["out"][:, :2]),
                   dict(block_table=good["block_table"].long()), dict(block_table=good["block_table"][0]), dict(seq_lens=it([1])), dict(shared_len=it([1, 2])),
                   dict(shared_len=torch.tensor([64], dtype=torch.int32)), dict(n_heads=3), dict(n_kv_heads=3), dict(head_dim=96), dict(rows_per_seq=0), dict(rows_per_seq=2),
                   dict(gate=torch.zeros(B, H, D, device=DEV)), dict(gate=torch.zeros(B, H, D - 1, dtype=torch.bfloat16, device=DEV)), dict(max_shared=-1), dict(prefix_row=2),
                   dict(prefix_row=-1)):
        with pytest.raises((RuntimeError, TypeError)):
            ops.attn_decode_shared(**{**good, **change})
    with pytest.raises(RuntimeError):                            # 17 rows x heads of a group
        ops.attn_decode_shared(**{**good, "q": torch.zeros(2 * 17, 1, D, dtype=torch.bfloat16, device=DEV), "out": torch.zeros(2 * 17, 1, D, dtype=torch.bfloat16, device=DEV),
                                  "n_heads": 1, "n_kv_heads": 1, "kv": good["kv"][:, :, :1].contiguous(), "rows_per_seq": 17})
    ops.attn_decode_shared(**{**good, "q": good["q"][:0], "out": good["out"][:0], "block_table": good["block_table"][:0], "seq_lens": it([])})
    torch.cuda.synchronize()
    _clean()
