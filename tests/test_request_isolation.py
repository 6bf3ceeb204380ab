"""A request that cannot be served ends alone: the requests beside it finish,
and what it held (KV blocks, a history row) is free again."""

import asyncio
import math

import pytest
import torch

from libra_b200.engine.rollout.controls import allow_tokens
from libra_b200.engine.rollout.llm_engine import LLMEngine
from libra_b200.engine.rollout.sampler import SamplingParams, extra_sampling


@pytest.fixture
def llm():
    from libra_b200.engine.train_engine import B200TrainEngine

    eng = B200TrainEngine("tiny", device="cpu", seed=3)
    eng.initialize()
    llm = LLMEngine(eng.cfg, {k: v.detach() for k, v in eng.params.items()}, kv_blocks=64, block_size=16,
                    max_running=4)
    yield llm
    llm.shutdown()


def _clean(llm):
    return (not llm.running and not llm.waiting and llm.kv.seqs == {} and not llm._controls._row
            and len(llm._controls._free) == llm.max_running)


def _beside_a_bystander(llm, params):
    """(bystander's result, the request's result or exception): both in flight at once."""

    async def go():
        bystander = asyncio.ensure_future(llm.generate([5, 6, 7], SamplingParams(max_tokens=40, temperature=0.0)))
        while not llm.running:
            await asyncio.sleep(0.001)
        (other,) = await asyncio.wait_for(asyncio.gather(llm.generate([1, 2, 3], params), return_exceptions=True), 30)
        return await asyncio.wait_for(bystander, 30), other

    return asyncio.run(go())


@pytest.mark.parametrize("ids", [[3, 2 ** 70], [3, -2 ** 70], [2 ** 63, 4, -1]])
def test_allowed_ids_beyond_64_bits_are_outside_the_vocabulary(llm, ids):
    bystander, res = _beside_a_bystander(llm, SamplingParams(max_tokens=3, temperature=0.0, allowed_token_ids=ids))
    assert len(bystander.output_tokens) == 40
    assert set(res.output_tokens) <= {3, 4} and len(res.output_tokens) == 3
    assert _clean(llm)


def test_allowed_ids_that_are_no_numbers_are_refused():
    for ids in ([3, None], [3, "x"], [3, [4]], [3, math.inf], [3, math.nan]):
        with pytest.raises(ValueError, match="allowed_token_ids"):
            SamplingParams(allowed_token_ids=ids)
        with pytest.raises(ValueError):
            extra_sampling({"allowed_token_ids": ids})
    for kw in ({"top_logprobs": math.inf}, {"logit_bias": {"1": 10 ** 400}}, {"frequency_penalty": 10 ** 400}):
        with pytest.raises(ValueError):
            extra_sampling(kw)


def test_a_mask_that_cannot_be_built_ends_its_request_only(llm):
    check = llm.check_params

    def then_spoil(params):  # a request changed behind every check
        check(params)
        if params.allowed_token_ids is not None:
            params.allowed_token_ids = [3, None]

    llm.check_params = then_spoil
    bystander, res = _beside_a_bystander(llm, SamplingParams(max_tokens=8, temperature=0.0, allowed_token_ids=[3, 4]))
    assert len(bystander.output_tokens) == 40 and res.finish_reason == "grammar_error" and not res.output_tokens
    assert _clean(llm)


def test_allow_tokens_ignores_ids_of_any_size():
    words = torch.zeros(2, dtype=torch.int32)
    allow_tokens(words, [0, 31, 33, 2 ** 64, -5, 40], 40)
    assert [v for v in range(64) if (int(words[v // 32]) >> (v % 32)) & 1] == [0, 31, 33]


@pytest.mark.parametrize("where", ["model", "controls", "sampler"])
def test_a_step_that_raises_answers_and_frees_the_requests_it_admitted(llm, where, monkeypatch):
    from libra_b200.engine.rollout import llm_engine

    def broken(*a, **kw):
        raise RuntimeError("broken step")

    apply = llm._controls.apply

    def apply_then_break(*a):
        apply(*a)  # (the request has its history row by then)
        broken()

    penalized = SamplingParams(max_tokens=3, temperature=0.0, frequency_penalty=0.5)
    for _ in range(llm.max_running + 1):  # more often than there are rows
        with monkeypatch.context() as m:
            if where == "model":
                m.setattr(llm.runner, "step", broken)
            elif where == "controls":
                m.setattr(llm._controls, "apply", apply_then_break)
            else:
                m.setattr(llm_engine, "sample", broken)
            with pytest.raises(RuntimeError, match="broken step"):
                asyncio.run(asyncio.wait_for(llm.generate([1, 2, 3], penalized), 30))
            llm.pause(30)
        assert _clean(llm)
        llm.resume()
    (res,) = [asyncio.run(asyncio.wait_for(llm.generate([1, 2, 3], penalized), 30))]
    assert len(res.output_tokens) == 3


def test_a_blocking_batch_that_raises_leaves_the_engine_clean(llm, monkeypatch):
    def broken(*a, **kw):
        raise RuntimeError("broken step")

    p = SamplingParams(max_tokens=3, temperature=0.0, frequency_penalty=0.5)
    with monkeypatch.context() as m:
        m.setattr(llm.runner, "step", broken)
        with pytest.raises(RuntimeError, match="broken step"):
            llm.generate_sync([[1, 2], [3, 4]], p)
    assert _clean(llm)
    assert [len(r.output_tokens) for r in llm.generate_sync([[1, 2], [3, 4]], p)] == [3, 3]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kw", [dict(top_k=2 ** 70), dict(top_k=-2 ** 70), dict(seed=2 ** 63 + 5), dict(seed=2 ** 64 - 1)])
def test_seeds_and_top_k_beyond_63_bits(device, kw):
    from libra_b200.engine.train_engine import B200TrainEngine

    eng = B200TrainEngine("tiny" if device == "cpu" else "tiny-gpu", device=device, seed=3)
    eng.initialize()
    llm = LLMEngine(eng.cfg, {k: v.detach() for k, v in eng.params.items()}, kv_blocks=64, block_size=16, max_running=4)
    plain = SamplingParams(max_tokens=6, temperature=0.0)
    for extra in ({}, {"presence_penalty": 0.1}):  # through the captured and the eager decode
        a, b = llm.generate_sync([[1, 2], [3, 4]], [plain, SamplingParams(max_tokens=6, **kw, **extra)])
        assert len(a.output_tokens) == len(b.output_tokens) == 6
    llm.add_request([1], SamplingParams(**{"seed": 1, **kw}))
    assert -2 ** 63 <= llm.waiting[0].seed < 2 ** 63
