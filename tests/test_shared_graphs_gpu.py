"""Captured decode steps behind a shared prefix beside those without one."""
import pytest
import torch

from llaminar_b200.models.config import SHAPES
from llaminar_b200.models.synth import synthesize

pytestmark = pytest.mark.gpu


def _tokens(n, seed, vocab):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def test_launches_of_a_step_are_counted_with_and_without_a_shared_prefix():
    from llaminar_b200.engine.engine import LLMEngine
    from llaminar_b200.engine.prefix_cache import PrefixCache, PrefixCacheConfig
    from llaminar_b200.engine.sampling import SamplingParams
    cfg = SHAPES["tiny-qwen3"].with_(d_model=512, n_heads=4, n_kv_heads=2, head_dim=128, d_ff=1024, n_layers=2)
    p = SamplingParams(temperature=0.0, max_tokens=4, ignore_eos=True)
    eng = LLMEngine(synthesize(cfg, "Q8_0", seed=5), device="cuda", max_batch=32, max_context=1024, prefix_cache=PrefixCache(PrefixCacheConfig(terminal_state="off"), "fp"))
    eng.generate([_tokens(9, i, cfg.vocab_size) for i in range(24)], p)
    plain = eng.launches_per_graph[(32, True)]
    system = _tokens(640, 1, cfg.vocab_size)
    eng.generate([system], p)
    eng.generate([system + [i] for i in range(24)], p)
    assert any(len(k) == 4 for k in eng._graphs)
    assert eng.launches_per_graph[(32, True)] == plain
    assert eng.launches_per_graph[(32, True, False, 1024)] == plain + cfg.n_layers      # a second launch in every block
