"""The chunk form of the gated delta rule in several passes, in captured steps and on two streams at once.

A chunk's arithmetic does not depend on the pass that it is in, and the state goes from pass to pass as 32-bit numbers, so every division into passes gives the same
bits; the division that holds all chunks at once is checked against the 64-bit recurrence in test_hybrid_kernels_gpu.py and, for a long prompt, here."""
import pytest
import torch

from . import hybrid_oracle as oracle
from .test_hybrid_kernels_gpu import DEV, EPS, _check_out, _check_state, _rows_problem

pytestmark = pytest.mark.gpu
D, N_K, N_V = 128, 16, 16


class _Call:
    def __init__(self, lens, pos, seed=5, aligned=False):
        self.lens, self.pos, T = lens, pos, sum(lens)
        self.buf, self.width, self.w, self.conv, self.rec = _rows_problem(seed, T, D, N_K, N_V, 4, len(lens) + 1)
        self.cu = [0]
        for n in lens:
            self.cu.append(self.cu[-1] + n)
        it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        self.positions = it([p + t for n, p in zip(lens, pos) for t in range(n)])
        self.cu_d, self.slots = it(self.cu), it(list(range(len(lens), 0, -1)))
        self.dw = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in self.w.items()}
        self.inp = self.buf.to(DEV)[:, :self.width]            # rows an odd number of values apart
        if aligned:
            self.inp = self.inp.contiguous()
        self.fresh_state()

    def fresh_state(self):
        self.conv_d, self.rec_d = self.conv.to(DEV), self.rec.to(DEV)
        self.out = torch.zeros(self.cu[-1], N_V * D, dtype=torch.bfloat16, device=DEV)

    def run(self):
        from llaminar_b200 import ops
        w = self.w
        ops.gdn_prefill(self.inp, w["C"], w["z_off"], w["ab_off"], self.dw["conv_w"], self.dw["ssm_a"], self.dw["dt_bias"], self.dw["norm_w"], self.conv_d,
                        self.rec_d, self.positions, self.cu_d, self.slots, self.out, N_K, 0, EPS)

    def results(self):
        torch.cuda.synchronize()
        return self.out.clone(), self.conv_d.clone(), self.rec_d.clone()


def _hold(monkeypatch, chunks):
    from llaminar_b200.ops import hybrid
    monkeypatch.setattr(hybrid, "GDN_WORKSPACE", chunks * hybrid.ext().gdn_chunk_bytes(1, N_K, N_V))


@pytest.mark.parametrize("lens,pos", [([2000], [0]), ([1300], [77]), ([700, 1, 900, 64], [0, 5, 3, 0]), ([64] * 30, [64] * 30)])
def test_every_division_into_passes_gives_the_same_bits(monkeypatch, lens, pos):
    call = _Call(lens, pos)
    _hold(monkeypatch, 10000)
    call.run()
    want = call.results()
    for chunks in (1, 2, 5, 16, 33):
        _hold(monkeypatch, chunks)
        call.fresh_state()
        call.run()
        for a, b in zip(call.results(), want):
            assert torch.equal(a, b), chunks


@pytest.mark.parametrize("aligned", [False, True])
def test_a_long_prompt_follows_the_recurrence(monkeypatch, aligned):
    call = _Call([1500], [9], aligned=aligned)
    _hold(monkeypatch, 12)
    call.run()
    out, conv, rec = call.results()
    w = call.w
    want, states = oracle.gdn_rows(call.buf, 0, 1500, call.conv[1], call.rec[1], w["conv_w"], w["ssm_a"], w["dt_bias"], w["norm_w"], N_K, 0, EPS, w["z_off"], w["ab_off"])
    _check_out(out, want, D)
    assert torch.equal(conv[1].double().cpu(), states[-1][0])
    _check_state(rec[1], states[-1][1], D)


@pytest.mark.parametrize("lens,pos", [([1500], [3]), ([100, 30], [1, 2])])
def test_a_captured_prompt_goes_on_from_replay_to_replay(monkeypatch, lens, pos):
    call = _Call(lens, pos)
    _hold(monkeypatch, 8)
    wants = []
    for _ in range(3):                                          # the state goes on from call to call
        call.run()
        wants.append(call.results())
    call.fresh_state()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call.run()                                              # warm-up
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        call.run()
    call.conv_d.copy_(call.conv), call.rec_d.copy_(call.rec), call.out.zero_()
    for want in wants:
        graph.replay()
        for a, b in zip(call.results(), want):
            assert torch.equal(a, b)


def test_two_streams_at_once(monkeypatch):
    _hold(monkeypatch, 8)
    calls = [_Call([1500], [3], 5), _Call([900, 400], [0, 6], 6)]
    wants = []
    for c in calls:
        c.run()
        wants.append(c.results())
        c.fresh_state()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for c, s in zip(calls, streams):
        with torch.cuda.stream(s):
            c.run()
    for c, want in zip(calls, wants):
        for a, b in zip(c.results(), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("lens,pos", [([37], [0]), ([63, 130, 1, 64], [2, 0, 5, 0])])
def test_rows_on_and_off_their_boundaries_give_the_same_bits(lens, pos):
    """Four taps in the same order either way."""
    results = []
    for aligned in (False, True):
        call = _Call(lens, pos, aligned=aligned)
        call.run()
        results.append(call.results())
    for a, b in zip(*results):
        assert torch.equal(a, b)
