"""The history table of a rollout engine's penalties: what a step hands to the kernel."""

import pytest
import torch

from libra_b200 import ops
from libra_b200.engine.rollout.controls import LogitControls
from libra_b200.engine.rollout.sampler import SamplingParams

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


class Request:
    def __init__(self, rid, tokens, **kw):
        self.request_id, self.prompt, self.out, self.params = rid, list(tokens), [], SamplingParams(**kw)

    @property
    def n_tokens(self):
        return len(self.prompt) + len(self.out)

    def token_slice(self, a, b):
        return (self.prompt + self.out)[a:b]


@pytest.mark.parametrize("device", DEVICES)
def test_short_histories_after_a_long_one_are_counted_as_short_ones(device, monkeypatch):
    V = 3000
    seen, orig = [], ops.control_logits

    def spy(logits, **kw):
        seen.append(kw["history"].shape[1])
        return orig(logits, **kw)

    monkeypatch.setattr(ops, "control_logits", spy)
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(2, V, generator=g).to(device)
    c = LogitControls(V, 4, device)
    kw = dict(repetition_penalty=1.3, frequency_penalty=0.25)
    short = [Request("a", [5, 6, 5, 7], **kw), Request("b", range(300), **kw)]
    want = c.apply(logits, short).clone()
    c.apply(logits[:1], [Request("long", [i % V for i in range(33000)], **kw)])
    c.release("long")
    assert seen[1] >= 32768  # (the kernel needs 32-bit counters here)
    for r in short:
        c.release(r.request_id)
    again = c.apply(logits, short)
    assert torch.equal(again, want)
    assert seen[2] < 32768, "the batch's own longest history decides, not the longest one ever served"
    short[0].out.append(8)
    grown = c.apply(logits, short)
    assert torch.equal(grown[1], want[1]) and float(grown[0, 8]) != float(want[0, 8])
    ops.check_kernel_errors()
