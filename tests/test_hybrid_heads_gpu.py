"""Softmax blocks of the hybrid family at head sizes and group sizes that their decode kernel does not have."""
import dataclasses

import pytest
import torch

from llaminar_b200.models.config import SHAPES
from llaminar_b200.models.reference import ReferenceModel
from llaminar_b200.models.synth import synthesize

from .test_shared_prefix_gpu import DEV, _near_the_top, _tokens

pytestmark = pytest.mark.gpu


def _config(**kw):
    return dataclasses.replace(SHAPES["tiny-qwen35"], name="tiny-qwen35-heads", n_layers=4, **kw)


@pytest.mark.parametrize("heads", [dict(n_heads=4, n_kv_heads=2, head_dim=96, rope_dim=32), dict(n_heads=2, n_kv_heads=1, head_dim=32, rope_dim=16),
                                   dict(n_heads=32, n_kv_heads=1, head_dim=256, rope_dim=64)])          # the last: 32 query heads of a K/V head
def test_other_heads_decode_on_pytorch_captured_and_eager(heads):
    """Norm, rotation and append on PyTorch ops (the first two) and batched attention inside the captured step; both ways agree and follow the oracle."""
    from llaminar_b200.engine import cuda_model
    from llaminar_b200.engine.engine import LLMEngine
    from llaminar_b200.engine.sampling import SamplingParams
    cfg = _config(**heads)
    w = synthesize(cfg, "Q8_0", seed=3)
    prompts = [_tokens(n, n) for n in (70, 9, 33)]
    p = SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True)
    called, real = [], cuda_model.paged_decode_attention_torch
    cuda_model.paged_decode_attention_torch = lambda *a: called.append(1) or real(*a)
    try:
        e1 = LLMEngine(w, device=DEV, max_batch=4, max_context=256, use_graphs=True)
        e2 = LLMEngine(w, device=DEV, max_batch=4, max_context=256, use_graphs=False)
        assert not e1.model.shares_prefixes()
        o1, o2 = e1.generate(prompts, p), e2.generate(prompts, p)
    finally:
        cuda_model.paged_decode_attention_torch = real
    assert called and o1 == o2 and e1.stats["graph_replays"] > 0
    ref = ReferenceModel(w)
    for pr, out in zip(prompts, o1):
        _near_the_top(ref, pr, out)


def test_too_many_query_heads_of_a_key_head_are_named():
    """64- and 128-wide heads: the decode kernels take 16 rows x query heads of a K/V head, and there is nothing behind them."""
    from llaminar_b200.engine.engine import LLMEngine
    from llaminar_b200.engine.sampling import SamplingParams
    eng = LLMEngine(synthesize(_config(n_heads=32, n_kv_heads=1, head_dim=64, rope_dim=16), "Q8_0", seed=3), device=DEV, max_batch=2, max_context=256, use_graphs=False)
    with pytest.raises(ValueError, match="16 rows x query heads of a K/V head, not 32"):
        eng.generate([_tokens(9, 1)], SamplingParams(temperature=0.0, max_tokens=3, ignore_eos=True))
