"""One scratch, and one status word, per device, however the device is named: a kernel that gave up a wait is noticed by whoever reads the word."""
import dataclasses

import pytest
import torch

from llaminar_b200 import ops
from llaminar_b200.models.config import SHAPES
from llaminar_b200.models.synth import synthesize


def test_a_device_without_a_number_is_the_current_one(monkeypatch):
    made = []
    monkeypatch.setattr(ops, "_scratch", {})
    monkeypatch.setattr(ops.Scratch, "create", staticmethod(lambda device, **kw: made.append(torch.device(device)) or object()))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    assert ops.scratch_for("cuda") is ops.scratch_for(torch.device("cuda", 1)) is ops.scratch_for("cuda:1") is ops.scratch_for(torch.device("cuda"))
    assert ops.scratch_for("cuda:0") is not ops.scratch_for("cuda") and made == [torch.device("cuda:1"), torch.device("cuda:0")]
    assert ops.scratch_for("cpu") is ops.scratch_for(torch.device("cpu")) and len(made) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [0, 2])
def test_the_engine_reads_the_word_that_the_delta_rule_writes(monkeypatch, drafts):
    from llaminar_b200.engine.engine import LLMEngine
    from llaminar_b200.engine.mtp import MTPConfig, MTPDecoder
    from llaminar_b200.engine.sampling import SamplingParams
    from llaminar_b200.ops import hybrid
    w = synthesize(dataclasses.replace(SHAPES["tiny-qwen35"], nextn_layers=1, ssm_state=128), "Q8_0", seed=4)
    eng = LLMEngine(w, device="cuda", max_batch=2, max_context=256, mtp=MTPDecoder(MTPConfig(draft_tokens=drafts)) if drafts else None)
    words, real = set(), hybrid.ext()

    class Watched:
        def __getattr__(self, name):
            def call(*a):
                if name in ("gdn_prefill", "gdn_verify") and a[-1] is not None:
                    words.add((name, a[-1].data_ptr()))
                return getattr(real, name)(*a)
            return call

    monkeypatch.setattr(hybrid, "ext", lambda: Watched())
    eng.generate([torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (100, 12)],
                 SamplingParams(temperature=0.0, max_tokens=5, ignore_eos=True))
    mine = [t.data_ptr() for t in eng._status_words()]
    assert {n for n, _ in words} == ({"gdn_prefill", "gdn_verify"} if drafts else {"gdn_prefill"})
    assert all(p in mine for _, p in words)
    assert len({s.status.data_ptr() for s in ops._scratch.values()}) == 1
