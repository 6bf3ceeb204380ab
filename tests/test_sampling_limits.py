"""Sampling arguments at the ends of what fp32 holds, where the engine uses them."""

import asyncio
import math

import pytest

from libra_b200.engine.rollout.llm_engine import LLMEngine
from libra_b200.engine.rollout.sampler import SamplingParams

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]

REFUSED = [dict(logit_bias={5: 1e39}), dict(logit_bias={5: -1e39}), dict(logit_bias={5: 1e21}),
           dict(repetition_penalty=1e-46), dict(repetition_penalty=1e-39), dict(repetition_penalty=1e39),
           dict(repetition_penalty=1e-21), dict(repetition_penalty=1e21), dict(presence_penalty=1e39),
           dict(presence_penalty=-1e39), dict(presence_penalty=-1e21), dict(frequency_penalty=3.5e38),
           dict(frequency_penalty=-1e21)]
ACCEPTED = [dict(logit_bias={5: 1e20}), dict(logit_bias={5: -3.4e38, 6: -1e30}), dict(repetition_penalty=1e-20),
            dict(repetition_penalty=1e20), dict(presence_penalty=3.4e38, frequency_penalty=3.4e38),
            dict(presence_penalty=-1e20, frequency_penalty=-1e20), dict(presence_penalty=3.4e38, frequency_penalty=-1e20),
            dict(presence_penalty=-1e20, frequency_penalty=3.4e38, logit_bias={9: 1e20})]


def _llm(device):
    from libra_b200.engine.train_engine import B200TrainEngine

    eng = B200TrainEngine("tiny" if device == "cpu" else "tiny-gpu", device=device, seed=3)
    eng.initialize()
    return LLMEngine(eng.cfg, {k: v.detach() for k, v in eng.params.items()}, kv_blocks=64, block_size=16,
                     max_running=8)


@pytest.mark.parametrize("kw", REFUSED)
def test_controls_beyond_fp32_are_refused(kw):
    with pytest.raises(ValueError, match=next(iter(kw))):
        SamplingParams(**kw)


@pytest.mark.parametrize("device", DEVICES)
def test_controls_at_their_limits_leave_a_distribution(device):
    llm = _llm(device)
    for temperature in (0.0, 1.0, 1e-3):
        ps = [SamplingParams(max_tokens=5, temperature=temperature, seed=3, top_logprobs=4, **kw) for kw in ACCEPTED]
        for kw, r in zip(ACCEPTED, llm.generate_sync([[1, 2, 3, 1]] * len(ps), ps)):
            assert len(r.output_tokens) == 5, kw
            assert all(v == v and v < 1e-3 for v in r.output_logprobs), (kw, r.output_logprobs)
            assert all(v == v for row in r.output_top_logprobs for _, v in row), kw


@pytest.mark.parametrize("device", DEVICES)
def test_top_logprobs_is_a_whole_number(device):
    for bad in (2.5, "x", None, math.inf):
        with pytest.raises(ValueError, match="top_logprobs"):
            SamplingParams(top_logprobs=bad)
    llm = _llm(device)
    (r,) = llm.generate_sync([[1, 2, 3]], SamplingParams(max_tokens=2, temperature=0.0, top_logprobs=2.0))
    assert [len(row) for row in r.output_top_logprobs] == [2, 2]


def test_server_answers_400_for_controls_beyond_fp32():
    from libra_b200.engine.rollout_engine import HTTPRolloutEngine
    from libra_b200.engine.server import BackgroundServer, build_app

    class Tok:
        eos_token_id = None

        def encode(self, text, add_special_tokens=False):
            return [1]

        def decode(self, ids):
            return " ".join(map(str, ids))

    llm = _llm("cpu")
    srv = BackgroundServer(build_app(llm, Tok(), "tiny"))
    try:
        client = HTTPRolloutEngine(port=srv.port)

        async def go():
            for kw in REFUSED + [dict(top_logprobs=300), dict(repetition_penalty=0.0)]:
                with pytest.raises(RuntimeError, match="400"):
                    await client.generate([7, 8], max_new_tokens=2, **kw)
            out = await client.generate([7, 8], max_new_tokens=2, temperature=0.0)
            return out

        async def then_close():
            try:
                return await go()
            finally:
                await client._session.close()

        assert len(asyncio.run(then_close())["token_ids"]) == 2
    finally:
        srv.stop()
        llm.shutdown()


@pytest.mark.parametrize("device", DEVICES)
def test_extreme_temperatures_beside_a_masked_request(device):
    """A temperature that fp32 holds as 0, as a subnormal or not at all leaves no NaN, masked tokens included."""
    for bad in (dict(temperature=math.nan), dict(top_p=math.nan)):
        with pytest.raises(ValueError, match=next(iter(bad))):
            SamplingParams(**bad)
    llm = _llm(device)
    kws = [dict(temperature=t, **kw) for t in (1e-320, 1e-45, 1e-40, 1e-30, 1e30, 1e300, math.inf)
           for kw in ({}, dict(allowed_token_ids=[3, 4, 5], top_logprobs=2))]
    kws += [dict(top_p=-1.0), dict(top_p=0.0), dict(top_p=0.0, allowed_token_ids=[3, 4, 5])]
    for kw in kws:
        p = SamplingParams(max_tokens=3, **kw)
        a, b = llm.generate_sync([[1, 2], [3, 4]], [p, SamplingParams(max_tokens=3, temperature=0.0)])
        assert len(a.output_tokens) == len(b.output_tokens) == 3, kw
        assert all(v == v and -math.inf < v < 1e-3 for v in a.output_logprobs), (kw, a.output_logprobs)
        assert all(v == v for row in a.output_top_logprobs for _, v in row), kw
        if "allowed_token_ids" in kw:
            assert set(a.output_tokens) <= {3, 4, 5}
