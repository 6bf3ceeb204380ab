"""Requests with penalties, biases, allowed tokens, grammars and top logprobs
through the rollout engine, its client classes and the HTTP server, against a
plain decode loop over the same model."""

import asyncio
import math

import pytest
import torch

import vocab_oracle as oracle
from libra_b200.engine.rollout.controls import allow_tokens
from libra_b200.engine.rollout.llm_engine import LLMEngine
from libra_b200.engine.rollout.sampler import SamplingParams

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


class EveryThird:
    """A grammar: token t follows only where (t + position) % 3 == 0; nothing follows after `stop` tokens."""

    def __init__(self, vocab, stop=10 ** 9):
        self.vocab, self.stop = vocab, stop

    def allowed(self, n):
        return [] if n >= self.stop else [t for t in range(self.vocab) if (t + n) % 3 == 0]

    def fill_mask(self, output_tokens, words):
        allow_tokens(words, self.allowed(len(output_tokens)), self.vocab)


@pytest.fixture(scope="module")
def engines():
    made = {}

    def get(device):
        if device not in made:
            from libra_b200.engine.train_engine import B200TrainEngine

            eng = B200TrainEngine("tiny" if device == "cpu" else "tiny-gpu", device=device, seed=3)
            eng.initialize()
            params = {k: v.detach() for k, v in eng.params.items()}
            made[device] = LLMEngine(eng.cfg, params, kv_blocks=256, block_size=16, max_running=8)
        return made[device]

    return get


def _words(vocab, ids):
    w = torch.zeros(1, (vocab + 31) // 32, dtype=torch.int32)
    allow_tokens(w[0], ids, vocab)
    return w


def _check_greedy(llm, prompt, p, res):
    """Every output token of a greedy request is the best of its row under the plain 64-bit controls, on logits that
    a second engine call computes for the same prefix; its logprob and top logprobs are that row's."""
    V = llm.cfg.vocab_size
    toks = list(prompt)
    for n, tok in enumerate(res.output_tokens):
        got = {}
        orig = llm._controls.apply
        probe = SamplingParams(max_tokens=1, temperature=0.0, logit_bias={0: 0.0})  # (a bias of 0 changes nothing)

        def spy(logits, reqs):
            got["z"] = logits.float().cpu().clone()
            return orig(logits, reqs)

        llm._controls.apply = spy
        try:
            llm.generate_sync([toks], probe)
        finally:
            llm._controls.apply = orig
        args = dict(history=torch.tensor([toks]), history_lens=torch.tensor([len(toks)]),
                    prompt_lens=torch.tensor([len(prompt)]), repetition=torch.tensor([p.repetition_penalty]),
                    presence=torch.tensor([p.presence_penalty]), frequency=torch.tensor([p.frequency_penalty]))
        if p.logit_bias:
            args.update(bias_offsets=torch.tensor([0, len(p.logit_bias)]), bias_ids=torch.tensor(list(p.logit_bias)),
                        bias_values=torch.tensor(list(p.logit_bias.values())))
        ids = set(range(V)) if p.allowed_token_ids is None else set(p.allowed_token_ids)
        if p.grammar is not None:
            ids &= set(p.grammar.allowed(n))
        args["mask"] = _words(V, ids)
        z, _ = oracle.control(got["z"], **args)
        # the engine computed this row at another batch shape: bf16 logits may differ by a rounding of the GEMMs
        slack = 2.0 ** -6 * float(got["z"].abs().max())
        assert tok in ids
        assert float(z[0, tok]) >= float(z[0].max()) - slack, (n, tok)
        lp = torch.log_softmax(z[0], 0)
        assert abs(res.output_logprobs[n] - float(lp[tok])) < 2 * slack
        if p.top_logprobs:
            top = res.output_top_logprobs[n]
            assert len(top) == min(p.top_logprobs, len(ids)) and top[0][0] == tok
            assert abs(top[0][1] - res.output_logprobs[n]) < 1e-5
            assert all(a[1] >= b[1] for a, b in zip(top, top[1:])) and all(t in ids for t, _ in top)
            for t, v in top:
                assert abs(v - float(lp[t])) < 2 * slack
        toks.append(tok)


CASES = {
    "repetition": dict(repetition_penalty=1.8),
    "presence and frequency": dict(presence_penalty=1.5, frequency_penalty=0.7),
    "bias": dict(logit_bias={5: 4.0, 9: -100.0, 17: 3.5}),
    "allowed": dict(allowed_token_ids=[3, 4, 5, 6, 10 ** 6]),
    "grammar": dict(grammar=True),
    "all with top": dict(repetition_penalty=1.2, presence_penalty=0.3, frequency_penalty=0.2, logit_bias={8: 1.0},
                         grammar=True, top_logprobs=7),
    "more top logprobs than allowed tokens": dict(allowed_token_ids=[3, 4, 5], top_logprobs=6),
}


def _params(name, vocab, **kw):
    d = dict(CASES[name], **kw)
    if d.get("grammar"):
        d["grammar"] = EveryThird(vocab)
    return SamplingParams(max_tokens=6, temperature=0.0, **d)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", list(CASES))
def test_greedy_requests_follow_their_controls(engines, device, name):
    llm = engines(device)
    p = _params(name, llm.cfg.vocab_size)
    prompt = [7, 8, 9, 7, 7, 30]
    (res,) = llm.generate_sync([prompt], p)
    assert len(res.output_tokens) == 6 and res.finish_reason == "length"
    _check_greedy(llm, prompt, p, res)
    assert not llm._controls._row and len(llm._controls._free) == llm.max_running


@pytest.mark.parametrize("device", DEVICES)
def test_mixed_batch_and_plain_requests_unchanged(engines, device):
    llm = engines(device)
    V = llm.cfg.vocab_size
    plain = SamplingParams(max_tokens=8, temperature=0.0)
    prompts = [[11, 12, 13], [7, 8, 9, 7], [21, 22], [40, 41, 42, 43]]
    want = llm.generate_sync([prompts[0]], plain)[0]
    ps = [plain, _params("all with top", V), SamplingParams(max_tokens=4, temperature=1.0, seed=5, top_k=20,
                                                           top_p=0.9, frequency_penalty=1.0), _params("allowed", V)]
    res = llm.generate_sync(prompts, ps)
    assert res[0].output_tokens == want.output_tokens and res[0].output_top_logprobs == []
    for i in (1, 3):
        _check_greedy(llm, prompts[i], ps[i], res[i])
    assert len(res[2].output_tokens) == 4 and all(math.isfinite(v) for r in res for v in r.output_logprobs)


@pytest.mark.parametrize("device", DEVICES)
def test_long_history_grows_the_table(engines, device):
    llm = engines(device)
    c = llm._controls
    prompt = [(i * 7) % 900 for i in range(300)]
    p = SamplingParams(max_tokens=3, temperature=0.0, frequency_penalty=0.5, repetition_penalty=1.1)
    (res,) = llm.generate_sync([prompt], p)
    _check_greedy(llm, prompt, p, res)
    before = c.table.clone()
    c._grow(5000)
    assert c.table.shape[1] == 8192 and torch.equal(c.table[:, :before.shape[1]], before)
    c._grow(20000)
    assert c.table.shape[1] == 32760
    c._grow(32765)
    assert c.table.shape[1] >= 32765
    c.table = None  # (later tests start small again)


@pytest.mark.parametrize("device", DEVICES)
def test_grammar_that_ends_or_fails_finishes_its_request_only(engines, device):
    llm = engines(device)
    V = llm.cfg.vocab_size

    class Broken:
        def fill_mask(self, output_tokens, words):
            raise RuntimeError("no rule")

    plain = SamplingParams(max_tokens=5, temperature=0.0)
    res = llm.generate_sync([[1, 2], [3, 4], [5, 6], [7, 8]], [
        plain, SamplingParams(max_tokens=5, temperature=0.0, grammar=EveryThird(V, stop=2)),
        SamplingParams(max_tokens=5, grammar=Broken()),
        SamplingParams(max_tokens=5, grammar=EveryThird(V), allowed_token_ids=[1])])  # the two exclude each other
    assert [r.finish_reason for r in res] == ["length", "grammar", "grammar_error", "grammar"]
    assert [len(r.output_tokens) for r in res] == [5, 2, 0, 0]
    assert not llm.running and not llm.waiting and llm.kv.seqs == {}


def test_sampling_params_refuse_bad_controls(engines):
    for bad in (dict(repetition_penalty=0.0), dict(repetition_penalty=math.inf), dict(presence_penalty=math.nan),
                dict(frequency_penalty=math.inf), dict(logit_bias={1: math.inf}), dict(logit_bias={-1: 1.0}),
                dict(allowed_token_ids=[]), dict(top_logprobs=257), dict(top_logprobs=-1)):
        with pytest.raises(ValueError):
            SamplingParams(**bad)
    with pytest.raises(ValueError, match="vocabulary"):
        engines("cpu").add_request([1], SamplingParams(allowed_token_ids=[10 ** 7]))


def test_client_and_server_pass_controls(engines):
    from libra_b200.engine.rollout_engine import HTTPRolloutEngine, LocalRolloutEngine
    from libra_b200.engine.server import BackgroundServer, build_app

    class Tok:
        eos_token_id = None

        def encode(self, text, add_special_tokens=False):
            return [1]

        def decode(self, ids):
            return " ".join(map(str, ids))

    from libra_b200.engine.train_engine import B200TrainEngine

    eng = B200TrainEngine("tiny", device="cpu", seed=3)
    eng.initialize()
    llm = LLMEngine(eng.cfg, {k: v.detach() for k, v in eng.params.items()}, kv_blocks=64, block_size=16)
    srv = BackgroundServer(build_app(llm, Tok(), "tiny"))
    try:
        kw = dict(max_new_tokens=4, temperature=0.0, logit_bias={"5": 3.0}, allowed_token_ids=[4, 5, 6],
                  repetition_penalty=1.5, top_logprobs=2)
        client = HTTPRolloutEngine(port=srv.port)

        async def both():
            local = await LocalRolloutEngine(llm, Tok()).generate([7, 8, 9], **kw)
            remote = await client.generate([7, 8, 9], **kw)
            with pytest.raises(RuntimeError, match="400"):
                await client.generate([7, 8, 9], repetition_penalty=-1.0)
            with pytest.raises(RuntimeError, match="400"):
                await client.generate([7, 8, 9], allowed_token_ids=[10 ** 7])
            with pytest.raises(ValueError, match="in-process"):
                await client.generate([7], grammar=EveryThird(10))
            await client._session.close()
            return local, remote

        local, remote = asyncio.run(both())
        assert local["token_ids"] == remote["token_ids"] and set(local["token_ids"]) <= {4, 5, 6}
        assert [[t for t, _ in row] for row in local["top_logprobs"]] == [[t for t, _ in row]
                                                                         for row in remote["top_logprobs"]]
        assert all(len(row) == 2 for row in remote["top_logprobs"])
    finally:
        srv.stop()
        llm.shutdown()
