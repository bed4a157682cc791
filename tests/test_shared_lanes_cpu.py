"""How a decode step learns which leading keys its sequences share: the number is the same on every rank that steps together, and it is looked for when the lanes change.

A captured step depends on it, and ranks that take different steps meet in different collectives.  Page ids are each rank's own (lower tiers, eviction history), so the
ranks agree on the smallest."""
import types

import torch

from llaminar_b200.engine.engine import LLMEngine, Request
from llaminar_b200.engine.kv_cache import PAGE_SIZE, SequenceKV
from llaminar_b200.engine.sampling import SamplingParams
from tests.mp_utils import run_ranks

BATCH, BUCKET, PAGES = 30, 32, 16


def _engine(common: int, group=None, shares: bool = True) -> tuple[LLMEngine, list[Request]]:
    """An engine as far as the staging of a decode step needs one, and requests of 700 tokens whose first ``common`` tokens lie in the same pages."""
    e = LLMEngine.__new__(LLMEngine)
    e.max_pages_per_seq, e._agree_group, e.stats, e.device = PAGES, group, {}, torch.device("cpu")
    e.kv = types.SimpleNamespace(hybrid=None, q8=False)
    e.model = types.SimpleNamespace(prefix_pays=lambda n_seqs, tokens: shares)
    e.prefix_cache = object()
    n = BUCKET * (2 + 1 + PAGES + 3 + 1) + 1
    e._dec_host, e._dec_dev = torch.zeros(n, dtype=torch.int32), torch.zeros(n, dtype=torch.int32)
    e._fl_host, e._seed_host = torch.zeros(2 * BUCKET), torch.zeros(BUCKET, dtype=torch.int64)
    reqs, free = [], 1000
    for i in range(BATCH):
        own = 11 - common // PAGE_SIZE
        pages = list(range(1, 1 + common // PAGE_SIZE)) + list(range(free, free + own))
        free += own
        reqs.append(Request(rid=i, prompt=[1] * 699, params=SamplingParams(temperature=0.0), output=[2], kv=SequenceKV(pages, 699)))
    return e, reqs


def _stage(e: LLMEngine, reqs: list[Request]) -> int:
    v = e._dec_views(BUCKET, 1)
    e._fill_decode_host(reqs, BUCKET, v)
    assert int(e._dec_host[v["shared"]]) == e._lane_shared
    return e._lane_shared


def _rank(rank, world, common, shares):
    import torch.distributed as dist
    e, reqs = _engine(common[rank], dist.group.WORLD, shares[rank])
    first = _stage(e, reqs)
    for r in reqs:
        r.output.append(3)
    return first, _stage(e, reqs), e.stats.get("agreements", 0)


def test_ranks_with_different_page_tables_take_the_same_step():
    """Caches that gave 384 common tokens on one rank and 640 on the other: on both sides of the threshold of 512."""
    assert [r[:2] for r in run_ranks(_rank, 2, [384, 640], [True, True])] == [(0, 0)] * 2
    got = run_ranks(_rank, 2, [576, 640], [True, True])
    assert [r[:2] for r in got] == [(576, 576)] * 2
    assert [r[2] for r in got] == [1, 1]                          # asked once for these lanes, not at every step
    assert [r[:2] for r in run_ranks(_rank, 2, [640, 640], [True, False])] == [(0, 0)] * 2      # one rank's heads have no such kernel


def test_one_rank_alone_shares_what_its_tables_have_in_common():
    for common, want in ((640, 640), (512, 512), (448, 0), (0, 0)):
        e, reqs = _engine(common)
        assert _stage(e, reqs) == want
    e, reqs = _engine(640)
    assert _stage(e, reqs[:10]) == 0                              # nine others save 5760 tokens
    assert _stage(e, reqs) == 640                                 # the lanes changed
    reqs[7].kv.pages[8] = 5
    e._lane_sig = None
    assert _stage(e, reqs) == 512


def test_a_preempted_request_is_looked_at_again():
    e, reqs = _engine(640)
    assert _stage(e, reqs) == 640
    e.running, e.waiting, e.mtp, e.stats = list(reqs), [], None, {"preemptions": 0}
    e.prefix_cache = types.SimpleNamespace(insert=lambda *a: None)
    e.kv.free_sequence = lambda s: None
    r = reqs[-1]
    e._preempt(r)
    r.kv, r.output = SequenceKV(list(range(5000, 5011)), 699), r.output + [4]        # back with pages of its own before a step without it
    assert _stage(e, reqs) == 0


def test_without_a_prefix_cache_nothing_is_looked_for():
    e, reqs = _engine(640)
    e.prefix_cache = None
    e._agree_min = None                                           # not called
    assert _stage(e, reqs) == 0


# heads, kv heads, head size, gated, sequences, shared tokens, whether a captured step was faster with the prefix taken once (by more than its spread)
MEASURED = [
    (24, 4, 256, True, 16, 512, False), (24, 4, 256, True, 3, 4096, False), (24, 4, 256, True, 16, 2048, True), (24, 4, 256, True, 32, 2048, True),
    (16, 2, 256, True, 3, 8192, False), (16, 2, 256, True, 16, 1024, False), (16, 2, 256, True, 64, 2048, True), (16, 2, 256, True, 8, 16384, True),
    (32, 8, 128, False, 4, 4096, False), (32, 8, 128, False, 2, 8192, False), (32, 8, 128, False, 6, 8192, True), (32, 8, 128, False, 32, 512, True),
    (16, 2, 128, True, 8, 8192, False), (16, 2, 128, True, 32, 1024, False), (16, 2, 128, True, 64, 8192, True),
    (16, 4, 64, False, 24, 1024, False), (32, 8, 64, False, 24, 512, False), (32, 8, 64, False, 32, 2048, True),
]


def test_a_prefix_is_taken_once_where_that_was_faster():
    """The rule on the heads' sizes against measured steps of several of them."""
    from llaminar_b200.engine.cuda_model import CudaModel
    for H, Hk, D, gated, B, tokens, faster in MEASURED:
        m = types.SimpleNamespace(cfg=types.SimpleNamespace(head_dim=D, attn_gate=gated), n_heads_local=H, n_kv_local=Hk, stack=None,
                                  PREFIX_MIN_BYTES=CudaModel.PREFIX_MIN_BYTES, PREFIX_MIN_SEQS=CudaModel.PREFIX_MIN_SEQS)
        m.shares_prefixes = lambda: CudaModel.shares_prefixes(m)
        e, reqs = _engine(640)
        e.model = types.SimpleNamespace(prefix_pays=lambda n, t: CudaModel.prefix_pays(m, n, t))
        reqs = [Request(rid=i, prompt=[1] * (tokens + 9), params=SamplingParams(temperature=0.0), output=[2], kv=SequenceKV(list(range(1, 1 + tokens // PAGE_SIZE)) + [10000 + i]))
                for i in range(B)]
        assert e._shared_tokens(reqs) == (tokens if faster else 0), (H, Hk, D, gated, B, tokens)
    m.stack = object()                                             # a model whose blocks have attention of their own
    assert not CudaModel.prefix_pays(m, 64, 8192)
