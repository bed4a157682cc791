"""Batches behind a shared prefix and the blocks of the hybrid family through the engine."""
import dataclasses

import pytest
import torch

from llaminar_b200.models.config import SHAPES
from llaminar_b200.models.reference import ReferenceModel
from llaminar_b200.models.synth import synthesize

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _tokens(n, seed, vocab=1024):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _near_the_top(ref, prompt, out):
    full, _, _ = ref.forward(torch.tensor((prompt + out)[:-1]))
    for i, t in enumerate(out):
        row = full[len(prompt) - 1 + i]
        assert row[t] >= row.max() - 0.05 * (row.max() - row.min())


@pytest.mark.parametrize("graphs", [True, False])
def test_requests_behind_a_cached_prompt_take_it_once(graphs):
    """Twenty-four requests with one system prompt of 640 tokens and questions of their own: the second batch shares the pages of the first one's prompt.  The
    tokens follow the oracle as they do without sharing."""
    from llaminar_b200.engine.engine import LLMEngine
    from llaminar_b200.engine.prefix_cache import PrefixCache, PrefixCacheConfig
    from llaminar_b200.engine.sampling import SamplingParams
    cfg = SHAPES["tiny-qwen3"].with_(d_model=512, n_heads=4, n_kv_heads=2, head_dim=128, d_ff=1024, n_layers=2)
    w = synthesize(cfg, "Q8_0", seed=5)
    system = _tokens(640, 1, cfg.vocab_size)
    prompts = [system + _tokens(5 + 3 * i, 10 + i, cfg.vocab_size) for i in range(24)]
    p = SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True)
    eng = LLMEngine(w, device=DEV, max_batch=32, max_context=1024, use_graphs=graphs, prefix_cache=PrefixCache(PrefixCacheConfig(terminal_state="off"), "fp"))
    eng.generate(prompts[:1], p)
    seen = []
    shared = eng._shared_tokens
    eng._shared_tokens = lambda reqs: seen.append(shared(reqs)) or seen[-1]
    outs = eng.generate(prompts, p)
    if graphs:
        assert 640 in seen and any(len(k) == 4 and k[3] == 1024 for k in eng._graphs)
    ref = ReferenceModel(w)
    for i in (0, 7, 23):
        _near_the_top(ref, prompts[i], outs[i])


def test_a_batch_without_a_common_page_shares_nothing():
    from llaminar_b200.engine.engine import LLMEngine
    from llaminar_b200.engine.sampling import SamplingParams
    cfg = SHAPES["tiny-qwen3"].with_(d_model=512, n_heads=4, n_kv_heads=2, head_dim=128, d_ff=1024, n_layers=2)
    eng = LLMEngine(synthesize(cfg, "Q8_0", seed=5), device=DEV, max_batch=4, max_context=1024)
    system = _tokens(640, 1, cfg.vocab_size)                    # the same words, but no cache: pages of their own
    eng.generate([system + [i] for i in range(3)], SamplingParams(temperature=0.0, max_tokens=3, ignore_eos=True))
    assert eng._graphs and all(len(k) == 3 for k in eng._graphs)


def test_published_state_and_head_sizes_of_the_hybrid_family_track_the_oracle():
    """States of 128 x 128 and heads of 256: prompts run the chunk-parallel kernels, decode steps the attention kernel for wide heads, gate included."""
    from llaminar_b200.engine.engine import LLMEngine
    from llaminar_b200.engine.sampling import SamplingParams
    cfg = dataclasses.replace(SHAPES["tiny-qwen35"], name="tiny-qwen35-wide", n_layers=4, n_heads=4, n_kv_heads=2, head_dim=256, rope_dim=64, ssm_state=128)
    w = synthesize(cfg, "Q8_0", seed=3)
    prompts = [_tokens(n, n) for n in (150, 9, 64, 65)]
    p = SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True)
    e1 = LLMEngine(w, device=DEV, max_batch=4, max_context=512, use_graphs=True, max_prefill_tokens=100)
    e2 = LLMEngine(w, device=DEV, max_batch=4, max_context=512, use_graphs=False, max_prefill_tokens=100)
    o1, o2 = e1.generate(prompts, p), e2.generate(prompts, p)
    assert o1 == o2 and e1.stats["graph_replays"] > 0
    ref = ReferenceModel(w)
    for pr, out in zip(prompts, o1):
        _near_the_top(ref, pr, out)


def test_drafts_of_a_hybrid_model_are_verified_on_the_kernels():
    """Speculative decoding: the verification pass leaves the recurrent states alone, the accepted rows advance them; every emitted token is one that the
    oracle puts at the top."""
    from llaminar_b200 import ops
    from llaminar_b200.engine.engine import LLMEngine
    from llaminar_b200.engine.mtp import MTPConfig, MTPDecoder
    from llaminar_b200.engine.sampling import SamplingParams
    w = synthesize(dataclasses.replace(SHAPES["tiny-qwen35"], nextn_layers=1, ssm_state=128), "Q8_0", seed=4)
    prompts = [_tokens(n, n) for n in (70, 12)]
    eng = LLMEngine(w, device=DEV, max_batch=2, max_context=256, mtp=MTPDecoder(MTPConfig(draft_tokens=2)))
    kept = []
    verify = ops.gdn_verify
    ops.gdn_verify = lambda *a: kept.append(1) or verify(*a)
    try:
        outs = eng.generate(prompts, SamplingParams(temperature=0.0, max_tokens=10, ignore_eos=True))
    finally:
        ops.gdn_verify = verify
    assert kept and all(len(o) == 10 for o in outs)
    ref = ReferenceModel(w)
    for pr, out in zip(prompts, outs):
        _near_the_top(ref, pr, out)
